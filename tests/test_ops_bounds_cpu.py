"""The bounds of ops_bounds.py: the formula token by token lies within them, and outputs that are a little wrong do not."""
import math

import pytest

torch = pytest.importorskip("torch")

import ops_bounds as B          # noqa: E402
import ops_reference as R       # noqa: E402

KINDS = [torch.float16, torch.bfloat16]


def inputs(seed, n, kh, vh, d, dtype, decay=0.05):
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
    unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(dtype)  # noqa: E731
    q, k, v = unit(normal(n, kh, d)), unit(normal(n, kh, d)), normal(n, vh, d).to(dtype)
    return (q, k, v, -decay * normal(n, vh).abs(), torch.sigmoid(normal(n, vh))), normal(1, vh, d, d) * 0.1


@pytest.fixture(scope="module", params=KINDS, ids=str)
def case(request):
    x, state = inputs(3, 200, 1, 2, 128, request.param)
    scale = 128 ** -0.5
    return x, state, scale, B.delta(torch, *x, state, [0, 200], [0], scale)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("chunk", [1, 64])
def test_it_is_the_formula_token_by_token(kind, chunk):
    x, state = inputs(1, 150, 1, 3, 64, kind)
    x[3][40] = -math.inf
    out, final, *_ = B.delta(torch, *x, state, [0, 150], [0], 0.125, chunk)
    want, last, _, _ = R.delta(torch, *x, state, [0, 150], [0], 0.125)
    assert (out - want).abs().max() < 1e-12 and (final - last).abs().max() < 1e-12


def test_rounded_results_are_right(case):
    x, state, scale, bounds = case
    out = bounds[0].to(x[0].dtype)
    assert B.wrong_outputs(torch, out, bounds) is None
    for t in range(0, 200, 64):
        assert B.wrong_outputs(torch, out, bounds, slice(t, t + 64)) is None
    assert B.wrong_state(torch, bounds[1].float(), bounds) is None


@pytest.mark.parametrize("how", ["zeros", "noise of 1 %", "1 % too small", "one NaN", "one head from another"])
def test_wrong_outputs_show_in_every_block(case, how):
    x, state, scale, bounds = case
    kind, out = x[0].dtype, bounds[0]
    gen = torch.Generator().manual_seed(9)
    bad = {"zeros": torch.zeros_like(out), "noise of 1 %": out + 0.01 * out.square().mean().sqrt() * torch.randn(out.shape, generator=gen, dtype=torch.float64),
           "1 % too small": out * 0.99, "one NaN": out.clone(), "one head from another": out.clone()}[how]
    if how == "one NaN":
        bad[::64, 1, 5] = math.nan
    if how == "one head from another":
        bad[:, 1] = bad[:, 0]
    for t in range(0, 200, 64):
        assert B.wrong_outputs(torch, bad.to(kind), bounds, slice(t, t + 64)) is not None


@pytest.mark.parametrize("i,j", [(0, 0), (1, 0), (2, 1), (3, 0), (3, 3)])
def test_a_block_left_out_shows(case, i, j):
    """16 x 16 of P left out of P V', and of A out of T."""
    x, state, scale, bounds = case
    for what in ("P", "A"):
        if what == "A" and i == j:
            continue
        out = bounds[0].clone()
        for c in B.chunks(torch, *x, state[0], 0, 192, 64):
            part = c[what].clone()
            part[:, 16 * i:16 * i + 16, 16 * j:16 * j + 16] = 0
            value = c["value"] if what == "P" else torch.linalg.solve_triangular(torch.eye(64, dtype=torch.float64) + part, c["R"], upper=False, unitriangular=True)
            mix = part if what == "P" else c["P"]
            out[c["a"]:c["b"]] = (scale * (c["into"] * (c["Q"] @ c["S"]) + mix @ value)).transpose(0, 1)
        for t in range(0, 192, 64):
            assert B.wrong_outputs(torch, out.to(x[0].dtype), bounds, slice(t, t + 64)) is not None, what


def test_a_decay_left_out_shows(case):
    x, state, scale, bounds = case
    g = x[3].clone()
    g[100] = 0
    wrong = B.delta(torch, x[0], x[1], x[2], g, x[4], state, [0, 200], [0], scale)
    assert B.wrong_outputs(torch, wrong[0].to(x[0].dtype), bounds, slice(100, 164)) is not None
    assert B.wrong_outputs(torch, wrong[0].to(x[0].dtype), bounds, slice(0, 100)) is None


def test_a_part_left_out_shows():
    """float16 outputs from a state of zeros, P and V' in one part each: 1.7 roundings in place of one."""
    x, state = inputs(5, 64, 1, 2, 128, torch.float16)
    state.zero_()
    bounds = B.delta(torch, *x, state, [0, 64], [0], 1.0)
    c = next(B.chunks(torch, *x, state[0], 0, 64, 64))
    both = (c["P"] @ c["value"]).transpose(0, 1).half()
    single = (c["P"].half().double() @ c["value"].half().double()).transpose(0, 1).half()
    assert B.wrong_outputs(torch, both, bounds) is None
    assert B.wrong_outputs(torch, single, bounds) is not None


def test_a_wrong_state_shows(case):
    x, state, scale, bounds = case
    final = bounds[1]
    gen = torch.Generator().manual_seed(2)
    for bad in (torch.zeros_like(final), final * 0.998, final + 0.002 * final.square().mean().sqrt() * torch.randn(final.shape, generator=gen, dtype=torch.float64)):
        assert B.wrong_state(torch, bad.float(), bounds) is not None
    assert B.wrong_state(torch, final.half().float(), bounds) is not None


def test_a_small_column_counts_to_its_own_bound():
    """A column 2^-20 of its neighbours: errors that are small beside those, and large beside it, show."""
    x, state = inputs(7, 100, 1, 1, 64, torch.bfloat16)
    x[2][:, :, 5::16] *= 2.0 ** -20
    state[..., 5::16] *= 2.0 ** -20
    bounds = B.delta(torch, *x, state, [0, 100], [0], 0.125)
    out = bounds[0].bfloat16()
    assert B.wrong_outputs(torch, out, bounds) is None
    out[:, :, 5::16] *= 0.98
    assert B.wrong_outputs(torch, out, bounds) is not None

"""The gated delta rule against 64 bits, each output within a bound from what it is summed of (ops_bounds.py)."""
import math

import pytest

import ops_bounds as B
from test_ops_gpu import clean_status, delta_inputs, normal, run_delta, status  # noqa: F401

pytestmark = pytest.mark.gpu

KINDS = ["float16", "bfloat16"]


def check(torch, x, counts, state, lead=0, scale=None, max_tokens=None):
    first = state.clone()
    out, starts = run_delta(torch, x, state, counts, lead, scale=scale, max_tokens=max_tokens)
    assert status(torch) == 0
    starts = [int(t) for t in starts]
    bounds = B.delta(torch, *x, first, starts, list(range(len(counts))), x[0].shape[2] ** -0.5 if scale is None else scale,
                     64 if (max_tokens or max(counts)) >= 16 else 1)
    for a, b in zip(starts, starts[1:]):
        for t in range(a, b, 64):
            wrong = B.wrong_outputs(torch, out, bounds, slice(t, min(t + 64, b)))
            assert wrong is None, (a, t, wrong)
        wrong = B.wrong_outputs(torch, out, bounds, slice(a, b))
        assert wrong is None, (a, b, wrong)
    wrong = B.wrong_state(torch, state, bounds)
    assert wrong is None, wrong


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("kh,vh,d", [(2, 4, 128), (1, 3, 128), (2, 2, 64), (1, 8, 64)])
@pytest.mark.parametrize("counts", [[1], [15, 2, 7], [16], [63, 64, 65], [200], [700, 0, 3, 200]])
def test_outputs_and_states(torch_cuda, kind, kh, vh, d, counts):
    torch = torch_cuda
    x = delta_inputs(torch, 5, sum(counts), kh, vh, d, getattr(torch, kind))
    check(torch, x, counts, normal(torch, 9, len(counts), vh, d, d, scale=0.1))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vh,d,counts", [(32, 128, [190]), (48, 128, [190]), (32, 128, [70, 190]), (48, 128, [70, 129, 100]), (160, 128, [100, 30]), (32, 64, [190]), (64, 64, [190, 64, 70])])
def test_each_width(torch_cuda, kind, vh, d, counts):
    """On 148 SMs: CTAs of 32 columns, of 64 (twice), of a head (twice); of 32 and of a head of 64."""
    torch = torch_cuda
    x = delta_inputs(torch, 85, sum(counts), 16, vh, d, getattr(torch, kind))
    check(torch, x, counts, normal(torch, 86, len(counts), vh, d, d, scale=0.1))


@pytest.mark.parametrize("kind", KINDS)
def test_from_a_state_of_zeros(torch_cuda, kind):
    """All of the first chunk's output is P V'."""
    torch = torch_cuda
    for d in (64, 128):
        check(torch, delta_inputs(torch, 15, 200, 1, 2, d, getattr(torch, kind)), [200], torch.zeros(1, 2, d, d, device="cuda"), scale=1.0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count", [12, 200])
@pytest.mark.parametrize("case", ["forget now and then", "keep", "never write", "same key", "decay of 3 a token", "decay of 16 a token", "reflect"])
def test_gates(torch_cuda, kind, count, case):
    torch = torch_cuda
    q, k, v, g, beta = delta_inputs(torch, 35, count, 2, 4, 128, getattr(torch, kind))
    if case == "forget now and then":
        g[::7] = -math.inf
        g[3::11] = -200.0
    elif case == "keep":
        g.zero_()
        beta.fill_(1.0)
    elif case == "never write":
        beta.zero_()
    elif case == "same key":
        g.zero_()
        beta.fill_(0.9)
        k[:] = k[:1]
    elif case == "reflect":
        g.zero_()
        beta[:] = (2.0 / (k.float() ** 2).sum(2)).repeat_interleave(2, 1) * (1 - 2.0 ** -20)
    else:
        g.fill_(-3.0 if "3" in case else -16.0)
    check(torch, (q, k, v, g, beta), [count], normal(torch, 36, 1, 4, 128, 128, scale=0.1))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count", [12, 200])
def test_columns_of_very_different_size(torch_cuda, kind, count):
    """Neighbouring value columns down to 2^-14 of each other, and groups of 16 down to 2^-8: each to its own bound."""
    torch = torch_cuda
    q, k, v, g, beta = delta_inputs(torch, 45, count, 2, 4, 128, getattr(torch, kind))
    column = torch.arange(128, device="cuda")
    size = 2.0 ** -((column * 7 % 15) + column // 16).float()
    state = normal(torch, 46, 1, 4, 128, 128, scale=0.1) * size
    check(torch, (q, k, (v.float() * size).to(v.dtype), g, beta), [count], state, scale=16.0)


@pytest.mark.parametrize("kind", KINDS)
def test_keys_and_queries_of_other_lengths(torch_cuda, kind):
    """Keys of a tenth to 1.4 times the unit length; queries from 2^-10 of it to 2^14 in float16, 2^-30 to 2^20 in bfloat16."""
    torch = torch_cuda
    q, k, v, g, beta = delta_inputs(torch, 95, 200, 2, 4, 128, getattr(torch, kind))
    gen = torch.Generator(device="cuda").manual_seed(5)
    k = (k.float() * (torch.rand(200, 1, 1, generator=gen, device="cuda") * 1.3 + 0.1)).to(k.dtype)
    up, down = (2.0 ** 14, 2.0 ** -10) if kind == "float16" else (2.0 ** 20, 2.0 ** -30)
    q[::3] *= up
    q[1::3] *= down
    check(torch, (q, k, v, g, beta), [200], normal(torch, 96, 1, 4, 128, 128, scale=0.1), scale=2.0 ** -3)


@pytest.mark.parametrize("kind", KINDS)
def test_a_state_much_larger_and_much_smaller_than_its_tokens(torch_cuda, kind):
    torch = torch_cuda
    for size in (2.0 ** 12, 2.0 ** -20):
        q, k, v, g, beta = delta_inputs(torch, 55, 150, 1, 4, 128, getattr(torch, kind))
        check(torch, (q, k, v, g, beta), [150], normal(torch, 56, 1, 4, 128, 128, scale=size), scale=2.0 ** -3)

"""The operators on a paged cache and on state rows against plain implementations in 64 bits (ops_reference.py)."""
import math

import numpy as np
import pytest

import ops_reference as R
import oracle as O
import skv

pytestmark = pytest.mark.gpu

KINDS = ["float16", "bfloat16"]


def normal(torch, seed, *shape, dtype=None, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, generator=gen, device="cuda") * scale
    return x if dtype is None else x.to(dtype)


def make_layer(torch, seed, cells, kv=2, dim=256, page=4, int8=False, spare=3):
    """A pool of random values, and a table that puts each sequence's cells at random pages; unused entries are -1."""
    need = [(c + page - 1) // page for c in cells]
    pages = sum(need) + spare
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    table = np.full((len(cells), max(need) + 1), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    table = torch.from_numpy(table).cuda()
    shape = (pages, kv, page, dim)
    if int8:
        gen = torch.Generator(device="cuda").manual_seed(seed)
        k, v = (torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8) for _ in "kv")
        ks, vs = (normal(torch, seed + i, *shape[:3], dim // 64).abs().half() * 0.02 + 0.005 for i in (1, 2))
        return skv.KvLayer(k, v, table, k_scale=ks, v_scale=vs)
    return skv.KvLayer(normal(torch, seed, *shape, dtype=torch.float16), normal(torch, seed + 1, *shape, dtype=torch.float16), table)


def ints(torch, values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.fixture(autouse=True)
def clean_status(torch_cuda):
    torch_cuda.cuda.set_device(0)
    skv.clear_status(0)
    yield
    torch_cuda.cuda.synchronize()


def status(torch):
    torch.cuda.synchronize()
    return skv.query_status(0)


# ------------------------------------------------------------------------------------------------ append

def check_append(torch, layer, before, k, v, q, q_out, lengths, starts, inv_freq, style, untouched=()):
    """Every cell of the pool: the new ones within their bounds, the others as they were (`before`: copies)."""
    k_pool, v_pool, k_scale, v_scale, tables = layer.tensors
    size = layer.args.page_size
    rows = tables.tolist()
    written = torch.zeros(k_pool.shape[0], size, dtype=torch.bool, device="cuda")
    for s in range(len(lengths)):
        for i in range(starts[s + 1] - starts[s]):
            t, cell = starts[s] + i, lengths[s] + i
            page, slot = rows[s][cell // size], cell % size
            written[page, slot] = True
            want_k, size_k = R.rotated(torch, k[t].double(), cell, inv_freq, style)
            for pool, scale, want, mag in ((k_pool, k_scale, want_k, size_k), (v_pool, v_scale, v[t].double(), v[t].double().abs())):
                # a turned value: its angle is reduced in 64 bits, then cos and sin in 32 (2 ulp), two products, a sum
                off = 6 * 2.0 ** -24 * mag
                got = pool[page, :, slot].double()
                if scale is None:
                    off = off + want.abs() * 2.0 ** -11 * (1 + 2.0 ** -10) + 2.0 ** -25
                else:
                    top = want.unflatten(-1, (-1, 64)).abs().amax(-1)
                    step = scale[page, :, slot].double()
                    near = off.unflatten(-1, (-1, 64)).amax(-1) / 127
                    assert ((step - top / 127).abs() <= top / 127 * (2.0 ** -11 + 2.0 ** -22) + near + 2.0 ** -25).all()
                    # half a step, and where the scale was rounded down the clamp at 127: 127 of its half steps
                    step = step.repeat_interleave(64, -1)
                    got = got * step
                    off = off + step * (0.5 + 127 * 2.0 ** -11 + 127 * 2.0 ** -22) + 127 * 2.0 ** -25
                assert ((got - want).abs() <= off).all(), (s, i, cell)
            if q is not None:
                want, mag = R.rotated(torch, q[t].double(), cell, inv_freq, style)
                off = 6 * 2.0 ** -24 * mag + want.abs() * R.half(q.dtype) * (1 + 2.0 ** -7) + R.tiny(q.dtype)
                assert ((q_out[t].double() - want).abs() <= off).all(), (s, i, cell)
    old_k, old_v = before
    keep = ~written[:, None, :, None]
    assert (torch.where(keep, k_pool, old_k) == old_k).all() and (torch.where(keep, v_pool, old_v) == old_v).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("kv,heads,dim,page,rot,style", [
    (2, 24, 256, 4, 64, "half"), (2, 24, 256, 4, 64, "pairs"), (8, 8, 64, 1, 64, "half"), (1, 5, 128, 256, 128, "pairs"),
    (3, 3, 128, 16, 16, "half"), (1, 1, 256, 4, 256, "half"), (2, 4, 64, 4, 0, "half")])
def test_append_ragged(torch_cuda, kind, int8, kv, heads, dim, page, rot, style):
    """Sequences of 0, 1 and many rows, rows before the first and behind the last sequence, strided inputs."""
    torch = torch_cuda
    dt = getattr(torch, kind)
    lengths, counts, lead, trail = [5, 0, 1023, 3, 7], [1, 19, 2, 0, 6], 2, 3
    starts = list(np.cumsum([lead] + counts))
    n = starts[-1] + trail
    layer = make_layer(torch, 3, [a + c for a, c in zip(lengths, counts)], kv, dim, page, int8)
    qkv = normal(torch, 7, n, (heads + 2 * kv) * dim, dtype=dt)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([heads * dim, kv * dim, kv * dim], 1))
    q_out = torch.full((n, heads, dim), 7.0, dtype=dt, device="cuda")
    inv = 10000.0 ** (-torch.arange(rot // 2, device="cuda") / max(rot // 2, 1))
    before = [x.clone() for x in layer.tensors[:2]]
    after = ints(torch, [-9] * 5)
    skv.kv_append(layer, k, v, ints(torch, lengths), seq_starts=ints(torch, starts), q=q, q_out=q_out,
                  inv_freq=inv if rot else None, rope_style=style, lengths_out=after)
    assert status(torch) == 0
    assert after.tolist() == [a + c for a, c in zip(lengths, counts)]
    check_append(torch, layer, before, k, v, q, q_out, lengths, starts, inv, style)
    assert (q_out[:lead] == 7).all() and (q_out[starts[-1]:] == 7).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("style", ["half", "pairs"])
@pytest.mark.parametrize("scale", [1.1386294, 0.5, 0.0])
def test_append_scales_what_it_turns(torch_cuda, kind, int8, style, scale):
    """rope_scale multiplies the turned values of K and q alone: those from n_rot on and V are as without it."""
    torch = torch_cuda
    dt, n, rot, cell = getattr(torch, kind), 19, 64, 77
    layer = make_layer(torch, 5, [cell + n], 2, 128, 16, int8)
    k, v, q = (normal(torch, 70 + i, n, h, 128, dtype=dt) for i, h in enumerate((2, 2, 6)))
    q_out, inv = torch.empty_like(q), 1e4 ** (-torch.arange(rot // 2, device="cuda") / (rot // 2))
    skv.kv_append(layer, k, v, ints(torch, [cell]), seq_starts=ints(torch, [0, n]), q=q, q_out=q_out, inv_freq=inv, rope_style=style, rope_scale=scale)
    assert status(torch) == 0
    by = float(np.float32(scale))
    for t in range(n):
        at = cell + t
        page, slot = int(layer.tensors[4][0, at // 16]), at % 16
        for x, got in ((k, layer.tensors[0][page, :, slot]), (q, q_out[t]), (v, layer.tensors[1][page, :, slot])):
            want, mag = x[t].double(), x[t].double().abs()
            if x is not v:
                want, mag = R.rotated(torch, want, at, inv, style)
                want[:, :rot] *= by
                mag[:, :rot] *= by
            # cos and sin times the scale: one rounding more than a turn alone
            off = 7 * 2.0 ** -24 * mag
            if int8 and x is not q:
                steps = (layer.tensors[2] if x is k else layer.tensors[3])[page, :, slot].double().repeat_interleave(64, -1)
                got, off = got.double() * steps, off + steps * (0.5 + 127 * 2.0 ** -11 + 127 * 2.0 ** -22) + 127 * 2.0 ** -25
            else:
                # the cache holds float16, q_out its own type
                to = dt if x is q else torch.float16
                off = off + want.abs() * R.half(to) * (1 + 2.0 ** -7) + R.tiny(to)
            assert ((got.double() - want).abs() <= off).all(), (t, x is k)


@pytest.mark.parametrize("n", [1, 2, 9, 64, 300])
def test_append_one_row_each_q_in_place(torch_cuda, n):
    torch = torch_cuda
    lengths = [(37 * i) % 50 for i in range(n)]
    layer = make_layer(torch, 5, [a + 1 for a in lengths])
    k, v = normal(torch, 1, n, 2, 256, dtype=torch.bfloat16), normal(torch, 2, n, 2, 256, dtype=torch.bfloat16)
    q = normal(torch, 3, n, 24, 256, dtype=torch.bfloat16)
    was, before = q.clone(), [x.clone() for x in layer.tensors[:2]]
    inv = 1e6 ** (-torch.arange(32, device="cuda") / 32)
    skv.kv_append(layer, k, v, ints(torch, lengths), q=q, q_out=q, inv_freq=inv)
    assert status(torch) == 0
    check_append(torch, layer, before, k, v, was, q, lengths, list(range(n + 1)), inv, "half")


def test_append_turns_far_cells_exactly_and_past_4_gib(torch_cuda):
    """Cell 2^28 - 2 needs its angle in 64 bits; its page lies past 4 GiB of the pool."""
    torch = torch_cuda
    pages, page = 16500, 256
    k_pool = torch.zeros(pages, 2, page, 256, dtype=torch.float16, device="cuda")
    v_pool = torch.zeros_like(k_pool)
    assert k_pool.numel() * 2 > 2 ** 32
    cell = 2 ** 28 - 2
    table = torch.full((1, 2 ** 20), -1, dtype=torch.int32, device="cuda")
    table[0, cell // page] = pages - 1
    layer = skv.KvLayer(k_pool, v_pool, table)
    k, v = normal(torch, 1, 2, 2, 256, dtype=torch.float16), normal(torch, 2, 2, 2, 256, dtype=torch.float16)
    inv = 10000.0 ** (-torch.arange(32, device="cuda") / 32)
    skv.kv_append(layer, k, v, ints(torch, [cell]), seq_starts=ints(torch, [0, 2]), inv_freq=inv)
    assert status(torch) == 0
    for i in range(2):
        want, mag = R.rotated(torch, k[i].double(), cell + i, inv, "half")
        got = k_pool[pages - 1, :, (cell + i) % page].double()
        assert ((got - want).abs() <= 6 * 2.0 ** -24 * mag + want.abs() * 2.0 ** -11 * 1.001 + 2.0 ** -25).all()
        assert (v_pool[pages - 1, :, (cell + i) % page] == v[i]).all()
    assert int((k_pool != 0).any(-1).sum()) == 4


def test_append_refuses_cells_on_the_device_and_writes_the_others(torch_cuda):
    """A -1 entry, an entry past the pool, a cell past the table and a negative length: flagged, nothing written there."""
    torch = torch_cuda
    layer = make_layer(torch, 9, [8, 8, 8, 8, 8])
    table = layer.tensors[4]
    table[0, 0], table[1, 0] = -1, layer.tensors[0].shape[0]
    lengths = [0, 1, table.shape[1] * 4, -3, 2]
    k, v = normal(torch, 1, 5, 2, 256, dtype=torch.float16), normal(torch, 2, 5, 2, 256, dtype=torch.float16)
    before = [x.clone() for x in layer.tensors[:2]]
    after = ints(torch, [0] * 5)
    skv.kv_append(layer, k, v, ints(torch, lengths), lengths_out=after)
    assert status(torch) == skv.STATUS_BAD_DST_PAGE
    page = int(table[4, 0])
    for pool, old, rows in ((layer.tensors[0], before[0], k), (layer.tensors[1], before[1], v)):
        assert (pool[page, :, 2] == rows[4]).all()
        pool[page, :, 2] = old[page, :, 2]
        assert (pool == old).all()
    assert after.tolist() == [1, 2, lengths[2] + 1, 1, 3]


def test_append_of_nothing(torch_cuda):
    """No rows at all: the lengths still come out."""
    torch = torch_cuda
    layer = make_layer(torch, 2, [4, 9, 1])
    before = [x.clone() for x in layer.tensors[:2]]
    none, after = torch.empty(0, 2, 256, dtype=torch.float16, device="cuda"), ints(torch, [-1] * 3)
    skv.kv_append(layer, none, none, ints(torch, [4, 0, 7]), seq_starts=ints(torch, [0, 0, 0, 0]), lengths_out=after)
    assert status(torch) == 0 and after.tolist() == [4, 0, 7]
    assert torch.equal(layer.tensors[0], before[0]) and torch.equal(layer.tensors[1], before[1])


def test_append_lengths_at_the_ends_of_their_range(torch_cuda):
    """lengths_out neither wraps nor starts below zero; cells past the table are flagged and written nowhere."""
    torch = torch_cuda
    layer = make_layer(torch, 6, [4, 4, 4, 4])
    before = [x.clone() for x in layer.tensors[:2]]
    k = normal(torch, 1, 10, 2, 256, dtype=torch.float16)
    after = ints(torch, [0] * 4)
    skv.kv_append(layer, k, k, ints(torch, [2 ** 31 - 1, 2 ** 31 - 3, -2 ** 31, 2 ** 31 - 3]), seq_starts=ints(torch, [0, 1, 6, 8, 10]), lengths_out=after)
    assert status(torch) == skv.STATUS_BAD_DST_PAGE
    assert after.tolist() == [2 ** 31 - 1, 2 ** 31 - 1, 2, 2 ** 31 - 1]
    assert torch.equal(layer.tensors[0], before[0]) and torch.equal(layer.tensors[1], before[1])


def test_append_of_very_many_padding_rows(torch_cuda):
    """70 million rows, five of them a sequence's: more CTAs than 2^31 threads' worth, and only those five go anywhere."""
    torch = torch_cuda
    n = 70_000_000
    x = torch.zeros(n, 1, 64, dtype=torch.float16, device="cuda")
    x[:5] = normal(torch, 9, 5, 1, 64, dtype=torch.float16)
    k_pool, v_pool = (torch.full((4, 1, 4, 64), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    layer = skv.KvLayer(k_pool, v_pool, torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device="cuda"))
    after = torch.full((64,), -5, dtype=torch.int32, device="cuda")
    skv.kv_append(layer, x, x, ints(torch, [3, 0]), seq_starts=ints(torch, [0, 3, 5]), lengths_out=after[31:33])
    assert status(torch) == 0 and after.tolist() == [-5] * 31 + [6, 2] + [-5] * 31
    want = torch.full_like(k_pool, 7.0)
    for row, (page, cell) in enumerate(((2, 3), (0, 0), (0, 1), (1, 0), (1, 1))):
        want[page, 0, cell] = x[row, 0]
    assert torch.equal(k_pool, want) and torch.equal(v_pool, want)


def test_memory_of_another_place_is_refused(torch_cuda):
    """A pool or a state in pinned host memory never reaches a kernel."""
    torch = torch_cuda
    layer = make_layer(torch, 2, [4])
    x = normal(torch, 1, 1, 2, 256, dtype=torch.float16)
    host = torch.zeros(layer.tensors[0].shape, dtype=torch.float16).pin_memory()
    layer.args.k_pool = host.data_ptr()
    with pytest.raises(skv.SkvError, match="current device"):
        skv.kv_append(layer, x, x, ints(torch, [0]))
    q = normal(torch, 1, 1, 24, 256, dtype=torch.float16)
    with pytest.raises(skv.SkvError, match="current device"):
        run_attention(torch, layer, q, [4], 0.0625)
    assert (host == 0).all()


@pytest.mark.parametrize("part", ["k_pool", "v_pool", "k_scale", "v_scale"])
def test_each_part_of_a_layer_is_looked_at(torch_cuda, part):
    """A pool or its scales in pinned host memory (which a kernel could reach) is refused by both operators, untouched."""
    torch = torch_cuda
    layer = make_layer(torch, 2, [4], int8=True)
    like = layer.tensors[("k_pool", "v_pool", "k_scale", "v_scale").index(part)]
    host = torch.zeros(like.shape, dtype=like.dtype).pin_memory()
    setattr(layer.args, part, host.data_ptr())
    x = normal(torch, 1, 1, 2, 256, dtype=torch.float16)
    with pytest.raises(skv.SkvError, match="current device"):
        skv.kv_append(layer, x, x, ints(torch, [0]))
    with pytest.raises(skv.SkvError, match="current device"):
        run_attention(torch, layer, normal(torch, 1, 1, 24, 256, dtype=torch.float16), [4], 0.0625)
    assert status(torch) == 0 and not host.any()


def test_append_int8_edges(torch_cuda):
    """Zeros, one huge group, infinities and NaN: the other groups of the row are as without them."""
    torch = torch_cuda
    layer = make_layer(torch, 2, [4], kv=1, dim=256, int8=True)
    k = normal(torch, 1, 4, 1, 256, dtype=torch.bfloat16)
    plain = k.clone()
    k[0] = 0
    k[1, 0, 64:128] = 3e38
    k[2, 0, 70] = math.inf
    k[3, 0, 70] = math.nan
    skv.kv_append(layer, k, plain, ints(torch, [0]), seq_starts=ints(torch, [0, 4]))
    assert status(torch) == 0
    page = int(layer.tensors[4][0, 0])
    codes, scale = layer.tensors[0][page, 0], layer.tensors[2][page, 0]
    assert (codes[0] == 0).all() and (scale[0] == 0).all()
    assert (codes[1, 64:128] == 127).all() and float(scale[1, 1]) == 65504
    assert int(codes[2, 70]) == 127 and float(scale[2, 1]) == 65504
    assert int(codes[3, 70]) == 0 and math.isfinite(float(scale[3, 1]))
    for row in (1, 2, 3):
        for g in (0, 2, 3):
            assert (codes[row, g * 64:g * 64 + 64] == layer.tensors[1][page, 0, row, g * 64:g * 64 + 64]).all()
            assert scale[row, g] == layer.tensors[3][page, 0, row, g]


@pytest.mark.parametrize("kind", KINDS)
def test_append_int8_of_groups_too_small_for_a_scale(torch_cuda, kind):
    """A group whose largest value / 127 rounds to a float16 zero (below 127 * 2^-25) has scale and codes of zero, both signs,
    with and without a NaN; one just above has the smallest scale and codes of its own."""
    torch = torch_cuda
    layer = make_layer(torch, 2, [4], kv=1, dim=256, int8=True)
    sign = torch.tensor([1.0, -1.0], device="cuda").repeat(32)
    small = torch.zeros(4, 1, 256, dtype=torch.float64, device="cuda")
    for row in range(4):
        for group, size in enumerate((2.0 ** -19, 2.0 ** -24, 3e-6, 2.0 ** -18 * 1.5)):
            small[row, 0, group * 64:group * 64 + 64] = size * sign * torch.linspace(1, 0, 64, device="cuda") ** (row + 1)
    small = small.to(getattr(torch, kind))
    small[3, 0, 5] = math.nan
    skv.kv_append(layer, small, -small, ints(torch, [0]), seq_starts=ints(torch, [0, 4]))
    assert status(torch) == 0
    page = int(layer.tensors[4][0, 0])
    for codes, scale, x in ((layer.tensors[0], layer.tensors[2], small), (layer.tensors[1], layer.tensors[3], -small)):
        codes, scale = codes[page, 0].double(), scale[page, 0].double()
        assert (scale[:, :3] == 0).all() and (codes[:, :192] == 0).all()
        assert (scale[:, 3] == 2.0 ** -24).all()
        assert torch.equal(codes[:, 192:], (x[:, 0, 192:].double() / 2.0 ** -24).round().clamp(-127, 127))


# ------------------------------------------------------------------------------------------------ attention

def run_attention(torch, layer, q, lengths, scale, stream=None, workspace=None):
    out = torch.full(q.shape, 9.0, dtype=q.dtype, device="cuda")
    lse = torch.full(q.shape[:2], 9.0, device="cuda")
    if workspace is None:   # garbage: nothing may be expected of it
        workspace = torch.full((skv.decode_attention_workspace(layer, q.shape[0], q.shape[1]),), 255, dtype=torch.uint8, device="cuda")
    skv.decode_attention(layer, q, ints(torch, lengths) if isinstance(lengths, list) else lengths, out, workspace=workspace,
                         scale=scale, lse=lse, stream=stream)
    return out, lse


def check_attention(torch, layer, q, lengths, scale, got):
    out, lse, far, far_lse = R.attention(torch, layer, q, lengths, scale)
    assert ((got[0].double() - out).abs() <= far).all(), float(((got[0].double() - out).abs() / far).nan_to_num(0).max())
    empty = lse == -math.inf
    assert (got[1][empty] == -math.inf).all() and (got[0][empty] == 0).all()
    assert ((got[1].double() - lse).abs()[~empty] <= far_lse[~empty]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("kv,heads,dim,page", [(2, 24, 256, 4), (1, 16, 256, 1), (2, 34, 128, 16), (8, 8, 64, 4), (1, 3, 128, 256), (4, 20, 256, 8)])
def test_attention_ragged(torch_cuda, kind, int8, kv, heads, dim, page):
    """Lengths 0, 1 and around every tile border, groups of 1, 3, 5, 12, 16 and 17 heads per K/V head."""
    torch = torch_cuda
    lengths = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 0, 2049]
    layer = make_layer(torch, 11, lengths, kv, dim, page, int8)
    q = normal(torch, 12, len(lengths), heads, dim, dtype=getattr(torch, kind))
    got = run_attention(torch, layer, q, lengths, dim ** -0.5)
    assert status(torch) == 0
    check_attention(torch, layer, q, lengths, dim ** -0.5, got)


@pytest.mark.parametrize("kv,page,spare", [(1, 1, 0), (1, 1, 1), (3, 1, 0), (1, 2, 0)])
def test_attention_int8_to_the_last_scale_of_a_pool(torch_cuda, kv, page, spare):
    """head_dim 64 has one two-byte scale a cell, copied with the word around it: odd and even numbers of rows, the last
    page in use, what lies behind the scales full of NaN."""
    torch = torch_cuda
    lengths = [33, 70]
    layer = make_layer(torch, 13, lengths, kv, 64, page, True, spare)
    pages = layer.tensors[0].shape[0]
    if not spare:
        assert (layer.tensors[4] == pages - 1).any()
    held = []
    for i, name in ((2, "k_scale"), (3, "v_scale")):
        n = layer.tensors[i].numel()
        room = torch.full((n + 8,), math.nan, dtype=torch.float16, device="cuda")
        room[:n] = layer.tensors[i].flatten()
        setattr(layer.args, name, room.data_ptr())
        held.append(room)
    q = normal(torch, 14, 2, 3 * kv, 64, dtype=torch.float16)
    got = run_attention(torch, layer, q, lengths, 0.125)
    assert status(torch) == 0
    check_attention(torch, layer, q, lengths, 0.125, got)


@pytest.mark.parametrize("lengths", [[1], [37], [700], [5000], [40000], [20001, 3], [30] * 200, [0, 0, 0], [9000] + [1] * 40])
@pytest.mark.parametrize("int8", [False, True])
def test_attention_few_and_many(torch_cuda, lengths, int8):
    """One sequence over the whole GPU, very unequal ones, more sequences than processors, nothing at all."""
    torch = torch_cuda
    layer = make_layer(torch, 21, lengths, int8=int8)
    q = normal(torch, 22, len(lengths), 24, 256, dtype=torch.bfloat16)
    got = run_attention(torch, layer, q, lengths, 0.0625)
    assert status(torch) == 0
    check_attention(torch, layer, q, lengths, 0.0625, got)
    again = run_attention(torch, layer, q, lengths, 0.0625)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1]), "the same inputs give the same bits"


def test_attention_strides_and_a_stream_of_its_own(torch_cuda):
    torch = torch_cuda
    lengths = [100, 3, 513]
    layer = make_layer(torch, 31, lengths)
    wide = normal(torch, 32, 3, 30, 256, dtype=torch.float16)
    q = wide[:, 2:26]
    room = torch.full((3, 40, 256), 5.0, dtype=torch.float16, device="cuda")
    out = room[:, 8:32]
    work = torch.empty(skv.decode_attention_workspace(layer, 3, 24), dtype=torch.uint8, device="cuda")
    lens = ints(torch, lengths)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    skv.decode_attention(layer, q, lens, out, workspace=work, stream=side)
    side.synchronize()
    ref, _, far, _ = R.attention(torch, layer, q, lengths, 0.0625)
    assert ((out.double() - ref).abs() <= far).all()
    assert (room[:, :8] == 5).all() and (room[:, 32:] == 5).all()


def test_attention_ignores_what_lies_behind_the_length(torch_cuda):
    """NaN and infinities in cells behind the last one, in the same page."""
    torch = torch_cuda
    lengths = [5, 33, 70]
    layer = make_layer(torch, 41, [8, 36, 72])
    q = normal(torch, 42, 3, 24, 256, dtype=torch.float16)
    want = R.attention(torch, layer, q, lengths, 0.0625)
    for s, n in enumerate(lengths):
        page = int(layer.tensors[4][s, n // 4])
        layer.tensors[0][page, :, n % 4:] = math.nan
        layer.tensors[1][page, :, n % 4:] = math.inf
    got = run_attention(torch, layer, q, lengths, 0.0625)
    assert ((got[0].double() - want[0]).abs() <= want[2]).all()


def test_attention_of_70_000_sequences(torch_cuda):
    """Lengths 0, 1 and 2 over four shared pages: a single cell's value comes back as it is, two equal keys average theirs."""
    torch = torch_cuda
    n = 70_000
    k_pool = torch.zeros(4, 1, 2, 64, dtype=torch.float16, device="cuda")
    v_pool = normal(torch, 3, 4, 1, 2, 64, dtype=torch.float16)
    table = (torch.arange(n, device="cuda") % 4).to(torch.int32).view(n, 1)
    layer = skv.KvLayer(k_pool, v_pool, table)
    q = normal(torch, 4, n, 1, 64, dtype=torch.float16)
    lengths = (torch.arange(n, device="cuda") % 3).to(torch.int32)
    out, lse = run_attention(torch, layer, q, lengths, 0.125)
    assert status(torch) == 0
    v = v_pool[table[:, 0].long(), 0].double()
    two = (lengths == 2)[:, None]
    want = torch.where(two, v.mean(1), torch.where((lengths == 1)[:, None], v[:, 0], 0.0))
    # keys of zero: weights of exactly 1, their sum and its reciprocal exact; one rounding
    assert ((out[:, 0].double() - want).abs() <= want.abs() * 2.0 ** -11 + 2.0 ** -25).all()
    assert torch.equal(out[:, 0][~two[:, 0]].double(), want[~two[:, 0]])
    assert (lse[lengths == 0] == -math.inf).all() and (lse[lengths == 1] == 0).all()
    assert ((lse[lengths == 2].double() - math.log(2)).abs() <= 2.0 ** -22).all()


@pytest.mark.parametrize("int8", [False, True])
def test_attention_skips_pages_outside_the_pool(torch_cuda, int8):
    """-1 (not resident), past the pool, a whole sequence of them, a length past the table, a negative one."""
    torch = torch_cuda
    lengths = [300, 40, 64, 20, 300]
    layer = make_layer(torch, 51, lengths, int8=int8)
    table = layer.tensors[4]
    table[0, 0], table[0, 17], table[0, 74] = -1, layer.tensors[0].shape[0], 2 ** 31 - 1
    table[1, :] = -5
    asked = [300, 40, 64, -7, 2 ** 31 - 1]
    q = normal(torch, 52, 5, 24, 256, dtype=torch.bfloat16)
    got = run_attention(torch, layer, q, asked, 0.0625)
    assert status(torch) == skv.STATUS_BAD_SRC_PAGE
    check_attention(torch, layer, q, asked, 0.0625, got)
    assert (got[0][1] == 0).all() and (got[0][3] == 0).all()


def test_attention_infinities(torch_cuda):
    """Scores of minus infinity weigh nothing, a row of nothing else is empty; plus infinity or NaN gives NaN; scores
    hundreds apart leave the largest alone."""
    torch = torch_cuda
    lengths = [50, 50, 50, 50]
    layer = make_layer(torch, 61, lengths)
    k_pool, table = layer.tensors[0], layer.tensors[4]
    q = normal(torch, 62, 4, 24, 256, dtype=torch.float16).abs() + 0.5
    for cell in range(50):
        page = int(table[0, cell // 4])
        if cell != 20:
            k_pool[page, :, cell % 4] = -math.inf
        page = int(table[1, cell // 4])
        k_pool[page, :, cell % 4] = -math.inf
    k_pool[int(table[2, 3]), :, 1] = math.nan
    k_pool[int(table[3, 5]), :, 2, :] = 200.0
    got = run_attention(torch, layer, q, lengths, 0.0625)
    v = layer.tensors[1]
    assert (got[0][0].view(2, 12, 256) == v[int(table[0, 5]), :, 0][:, None]).all()
    assert (got[0][1] == 0).all() and (got[1][1] == -math.inf).all()
    assert got[0][2].isnan().all() and got[1][2].isnan().all()
    assert (got[0][3].view(2, 12, 256) == v[int(table[3, 5]), :, 2][:, None]).all()


def test_attention_of_large_and_small_queries(torch_cuda):
    """bfloat16 queries beyond the range of float16 and far below it."""
    torch = torch_cuda
    lengths = [100, 100, 100]
    layer = make_layer(torch, 71, lengths)
    q = normal(torch, 72, 3, 24, 256, dtype=torch.bfloat16)
    q[0] *= 2.0 ** 30
    q[1] *= 2.0 ** -40
    q[2, :, :128] *= 2.0 ** -30
    for s, scale in ((0, 2.0 ** -34), (1, 2.0 ** 36), (2, 0.0625)):
        got = run_attention(torch, layer, q, lengths, scale)
        want = R.attention(torch, layer, q, lengths, scale)
        # values 2^-25 of the row's largest may be rounded away: part of the bound's 2^-24 per product
        assert ((got[0][s].double() - want[0][s]).abs() <= want[2][s]).all()


@pytest.mark.parametrize("int8", [False, True])
def test_attention_through_tables_of_their_own(torch_cuda, int8):
    """A table of some of a sequence's pages, in any order, attends to their cells (the last, partly filled one at the end);
    several rows with one sequence's pages and growing lengths are several new tokens of it."""
    torch = torch_cuda
    full = make_layer(torch, 35, [333], int8=int8)
    k_pool, v_pool, k_scale, v_scale, table = full.tensors
    q = normal(torch, 36, 5, 24, 256, dtype=torch.float16)
    some = torch.from_numpy(np.random.default_rng(3).permutation(83)[:41]).cuda()    # of the 83 full pages
    picked = torch.cat([table[0][some], table[0, 83:84]])[None]
    layer = skv.KvLayer(k_pool, v_pool, picked, k_scale=k_scale, v_scale=v_scale)
    got = run_attention(torch, layer, q[:1], [41 * 4 + 1], 0.0625)
    k, v, _ = R.cells_of(torch, full, 0, 333)
    cells = torch.cat([(some[:, None] * 4 + torch.arange(4, device="cuda")).flatten(), torch.tensor([332], device="cuda")])
    k, v = (z.repeat_interleave(12, 0)[:, cells] for z in (k, v))
    score = torch.einsum("hd,hnd->hn", q[0].double(), k) * 0.0625
    want = torch.einsum("hn,hnd->hd", torch.softmax(score, -1), v)
    _, _, far, far_lse = R.attention(torch, layer, q[:1], [41 * 4 + 1], 0.0625)
    assert ((got[0][0].double() - want).abs() <= far[0]).all()
    assert ((got[1][0].double() - torch.logsumexp(score, -1)).abs() <= far_lse[0]).all()
    rows = skv.KvLayer(k_pool, v_pool, table.expand(5, -1).contiguous(), k_scale=k_scale, v_scale=v_scale)
    lengths = [329, 330, 331, 332, 333]
    check_attention(torch, rows, q, lengths, 0.0625, run_attention(torch, rows, q, lengths, 0.0625))
    assert status(torch) == 0


def test_attention_past_4_gib(torch_cuda):
    torch = torch_cuda
    pages, page, n = 16500, 256, 300
    k_pool = torch.zeros(pages, 2, page, 256, dtype=torch.float16, device="cuda")
    v_pool = torch.zeros_like(k_pool)
    table = ints(torch, [pages - 1, pages - 2]).view(1, 2)
    k_pool[pages - 2:] = normal(torch, 1, 2, 2, page, 256, dtype=torch.float16)
    v_pool[pages - 2:] = normal(torch, 2, 2, 2, page, 256, dtype=torch.float16)
    layer = skv.KvLayer(k_pool, v_pool, table)
    q = normal(torch, 3, 1, 24, 256, dtype=torch.float16)
    check_attention(torch, layer, q, [n], 0.0625, run_attention(torch, layer, q, [n], 0.0625))


def test_attention_in_a_graph_follows_its_lengths(torch_cuda):
    """Captured once, replayed with other lengths, tables and queries; two graphs with a workspace each side by side."""
    torch = torch_cuda
    cells = [600, 90, 300]
    layer = make_layer(torch, 81, cells)
    q = normal(torch, 82, 3, 24, 256, dtype=torch.bfloat16)
    lens = ints(torch, [1, 1, 1])
    run_attention(torch, layer, q, lens, 0.0625)      # sets the device up
    graphs = []
    for _ in range(2):
        out, lse = torch.empty_like(q), torch.empty(3, 24, device="cuda")
        work = torch.empty(skv.decode_attention_workspace(layer, 3, 24), dtype=torch.uint8, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            skv.decode_attention(layer, q, lens, out, workspace=work, scale=0.0625, lse=lse, stream=torch.cuda.current_stream())
        graphs.append((graph, out, lse, work))
    for step, lengths in enumerate([[600, 90, 300], [0, 1, 17], [333, 64, 0]]):
        lens.copy_(ints(torch, lengths))
        q.copy_(normal(torch, 90 + step, 3, 24, 256))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (graph, *_), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, lse, _ in graphs:
            check_attention(torch, layer, q, lengths, 0.0625, (out, lse))


# ------------------------------------------------------------------------------------------------ the gated delta rule

def delta_inputs(torch, seed, n, kh, vh, d, dtype, decay=0.05):
    unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(dtype)  # noqa: E731
    q, k = unit(normal(torch, seed, n, kh, d)), unit(normal(torch, seed + 1, n, kh, d))
    v = normal(torch, seed + 2, n, vh, d, dtype=dtype)
    g = -decay * normal(torch, seed + 3, n, vh).abs()
    beta = torch.sigmoid(normal(torch, seed + 4, n, vh))
    return q, k, v, g, beta


def run_delta(torch, x, state, counts, lead=0, state_index=None, max_tokens=None, out=None, scale=None):
    q, k, v, g, beta = x
    n, vh, d = v.shape
    starts = list(np.cumsum([lead] + counts))
    out = torch.full((n, vh, d), 9.0, dtype=q.dtype, device="cuda") if out is None else out
    most = max(counts) if max_tokens is None else max_tokens
    need = skv.gated_delta_workspace(n, len(counts), vh, d, most)
    work = torch.full((max(need, 16),), 255, dtype=torch.uint8, device="cuda")
    skv.gated_delta(q, k, v, g, beta, state, out, seq_starts=ints(torch, starts), state_index=state_index, max_tokens=most,
                    scale=d ** -0.5 if scale is None else scale, workspace=work)
    return out, starts


def check_delta(torch, x, state0, state, out, starts, rows, scale=None):
    d = x[0].shape[2]
    want, final, far, off = R.delta(torch, *x, state0, starts, rows, d ** -0.5 if scale is None else scale)
    for s in range(len(rows)):
        a, b = starts[s], starts[s + 1]
        assert ((out[a:b].double() - want[a:b]).abs() <= far[a:b]).all(), (s, float(((out[a:b].double() - want[a:b]).abs() / far[a:b]).max()))
    assert ((state.double() - final).flatten(2).norm(dim=2) <= off).all()
    assert (out[:starts[0]] == 9).all() and (out[starts[-1]:] == 9).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("kh,vh,d", [(2, 4, 128), (1, 3, 128), (2, 2, 64), (1, 8, 64)])
@pytest.mark.parametrize("counts", [[1], [2, 1, 0, 3], [15, 16, 17], [31, 33], [63, 64, 65], [0, 0], [127, 1, 130], [700, 0, 3, 200]])
def test_delta_ragged(torch_cuda, kind, kh, vh, d, counts):
    torch = torch_cuda
    lead, trail = 3, 2
    n = lead + sum(counts) + trail
    x = delta_inputs(torch, 5, n, kh, vh, d, getattr(torch, kind))
    state = normal(torch, 9, len(counts), vh, d, d, scale=0.1)
    first = state.clone()
    out, starts = run_delta(torch, x, state, counts, lead)
    assert status(torch) == 0
    check_delta(torch, x, first, state, out, starts, list(range(len(counts))))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("kh,vh,d", [(8, 24, 128), (20, 40, 64)])
def test_delta_fills_the_gpu(torch_cuda, kind, kh, vh, d):
    """More heads and sequences than fit at once: a whole head per CTA."""
    torch = torch_cuda
    counts = [130, 1, 64, 65, 0, 200, 31]
    x = delta_inputs(torch, 75, 1 + sum(counts) + 2, kh, vh, d, getattr(torch, kind))
    state = normal(torch, 79, len(counts), vh, d, d, scale=0.1)
    first = state.clone()
    out, starts = run_delta(torch, x, state, counts, 1)
    assert status(torch) == 0
    check_delta(torch, x, first, state, out, starts, list(range(len(counts))))


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("vh,d,counts", [(32, 128, [190]), (48, 128, [190]), (32, 128, [70, 190]), (48, 128, [70, 129, 100]), (32, 64, [190]), (64, 64, [190, 64, 70])])
def test_delta_of_each_width(torch_cuda, kind, vh, d, counts):
    """On 148 SMs: CTAs of 32 columns, of 64 (twice), of a head; of 32 and of a head of 64."""
    torch = torch_cuda
    x = delta_inputs(torch, 85, sum(counts), 16, vh, d, getattr(torch, kind))
    state = normal(torch, 86, len(counts), vh, d, d, scale=0.1)
    first = state.clone()
    out, starts = run_delta(torch, x, state, counts)
    assert status(torch) == 0
    check_delta(torch, x, first, state, out, starts, list(range(len(counts))))


@pytest.mark.parametrize("n,vh", [(128, 4), (129, 4), (70, 48)])
def test_delta_of_many_short_sequences(torch_cuda, n, vh):
    """By rank, too many for ranks, too short to be worth ranks; equal lengths and none among them."""
    torch = torch_cuda
    counts = [int(x) for x in np.random.default_rng(n).integers(0, 71, n)]
    counts[3], counts[5], counts[7], counts[-1] = 0, 70, 70, 64
    x = delta_inputs(torch, 87, sum(counts), 2, vh, 128, torch.bfloat16)
    state = normal(torch, 88, n, vh, 128, 128, scale=0.1)
    first = state.clone()
    out, starts = run_delta(torch, x, state, counts)
    assert status(torch) == 0
    check_delta(torch, x, first, state, out, starts, list(range(n)))


@pytest.mark.parametrize("count", [5, 200])
def test_delta_of_keys_and_queries_of_other_lengths(torch_cuda, count):
    """Keys of a tenth to twice the unit length, queries 2^20 and 2^-30 of it, large values."""
    torch = torch_cuda
    q, k, v, g, beta = delta_inputs(torch, 95, count, 2, 4, 128, torch.bfloat16)
    gen = np.random.default_rng(5)
    size = torch.from_numpy(gen.uniform(0.1, 1.4, count).astype(np.float32)).cuda()
    k = (k.float() * size[:, None, None]).to(torch.bfloat16)
    q[::3] *= 2.0 ** 20
    q[1::3] *= 2.0 ** -30
    v *= 3000.0
    state = normal(torch, 96, 1, 4, 128, 128, scale=10.0)
    first = state.clone()
    out, starts = run_delta(torch, (q, k, v, g, beta), state, [count])
    check_delta(torch, (q, k, v, g, beta), first, state, out, starts, [0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("decay", [-1.0, -16.0])
@pytest.mark.parametrize("size,strength", [(60000.0, 0.5), (1.0, 0.5), (2.0 ** -14, 0.5), (2.0 ** -20, 0.5), (30000.0, 512.0), (2.0 ** -7, 2.0 ** -7)])
@pytest.mark.parametrize("count", [12, 16])
def test_delta_of_queries_of_any_size(torch_cuda, kind, d, decay, size, strength, count):
    """Keys of four equal values each, orthogonal to each other; a token asks for the key before its own.  So what it reads
    is e^decay (q . k) v of that token and nothing else, whatever the sizes of q and k.  The sizes and the write strength
    beta = 1 / |k|^2 are powers of two or exact in both types, and scale undoes them: every output is about v.

    Bound.  The output's rounding; the decay, 2^-20 (an exponential of a difference within 2^-21 of it); two 16-bit operands
    of 2^-11 each for bfloat16 outputs, of 2^-22 for float16 ones; sums of one term, whose other terms are exact zeros; values
    of V' below 2^-39 of the largest are not kept, at most 8 here, nor decayed products of q and k below 2^-37 of d times
    the largest values of the two (2^-39 of a power of two that is at most four times that)."""
    torch = torch_cuda
    dt = getattr(torch, kind)
    if kind == "bfloat16":
        size = 2.0 ** round(math.log2(size))
    gen = torch.Generator(device="cuda").manual_seed(7)
    kh, vh = 1, 2
    q, k = (torch.zeros(count, kh, d, dtype=dt, device="cuda") for _ in "qk")
    for t in range(count):
        k[t, 0, 4 * t:4 * t + 4] = strength
        if t:
            q[t, 0, 4 * t - 4:4 * t] = size
    v = torch.randn(count, vh, d, generator=gen, device="cuda").clamp(-8, 8).to(dt)
    g = torch.full((count, vh), decay, device="cuda")
    beta = torch.full((count, vh), 0.25 / strength ** 2, device="cuda")
    state = torch.zeros(1, vh, d, d, device="cuda")
    # k beta v is read: |q . k| beta = 4 size strength / (4 strength^2)
    scale = strength / size * math.exp(-decay)
    out, _ = run_delta(torch, (q, k, v, g, beta), state, [count], scale=scale)
    assert status(torch) == 0
    assert (out[0] == 0).all()
    want = v[:-1].double() * (float(np.float32(scale)) * math.exp(decay) * size / strength)
    off = want.abs() * (R.half(dt) * (1 + 2.0 ** -7) + 2.0 ** -20 + (2.0 ** -10 if kind == "bfloat16" else 2.0 ** -21)) + 2.0 ** -36 + R.tiny(dt)
    off = off + 2.0 ** -37 * d * size * strength * (0.25 / strength ** 2) * scale * v[:-1].double().abs()
    assert ((out[1:].double() - want).abs() <= off).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("vh", [4, 160])
def test_delta_keeps_a_bad_token_to_its_heads(torch_cuda, bad, vh):
    """A NaN or an infinity in a key: other sequences, other key heads and the chunks before it as without it."""
    torch = torch_cuda
    counts = [100, 200, 70]
    x = list(delta_inputs(torch, 98, sum(counts), 2, vh, 128, torch.float16))
    state = normal(torch, 99, 3, vh, 128, 128, scale=0.1)
    clean = state.clone()
    want = run_delta(torch, x, clean, counts)[0]
    x[1] = x[1].clone()
    x[1][100 + 130, 1, 5] = bad
    got = run_delta(torch, x, state, counts)[0]
    assert torch.equal(got[:, : vh // 2], want[:, : vh // 2]) and torch.equal(state[:, : vh // 2], clean[:, : vh // 2])
    assert torch.equal(got[:228], want[:228]) and torch.equal(got[300:], want[300:])
    assert torch.equal(state[::2], clean[::2]) and not got[230, vh // 2 :].isfinite().any()


def test_delta_on_two_streams_at_once(torch_cuda):
    """Two prompts side by side, a workspace each: the bits of one after the other."""
    torch = torch_cuda
    runs = []
    for i in range(2):
        x = delta_inputs(torch, 105 + i, 400, 2, 4, 128, torch.bfloat16)
        state = normal(torch, 107 + i, 1, 4, 128, 128, scale=0.1)
        alone = state.clone()
        want = run_delta(torch, x, alone, [400])[0]
        work = torch.empty(skv.gated_delta_workspace(400, 1, 4, 128, 400), dtype=torch.uint8, device="cuda")
        runs.append((x, state, alone, want, torch.full_like(want, 9.0), ints(torch, [0, 400]), work, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for x, state, _, _, out, starts, work, stream in runs:
        skv.gated_delta(*x, state, out, seq_starts=starts, max_tokens=400, workspace=work, stream=stream)
    torch.cuda.synchronize()
    for _, state, alone, want, out, *_ in runs:
        assert torch.equal(state, alone) and torch.equal(out, want)


@pytest.mark.parametrize("n", [1, 5, 130])
def test_delta_one_token_each(torch_cuda, n):
    """The decode form: no starts; the rows' order given by an index, strided inputs and rows."""
    torch = torch_cuda
    kh, vh, d = 4, 8, 128
    q, k, v, g, beta = delta_inputs(torch, 15, n, kh, vh, d, torch.bfloat16)
    mixed = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
    q, k, v = (z.unflatten(1, (-1, d)) for z in mixed.split([kh * d, kh * d, vh * d], 1))
    gates = torch.stack([g, beta], 1)
    g, beta = gates[:, 0], gates[:, 1]
    row = vh * d * d + 1024         # a conv tail behind each state
    store = normal(torch, 16, n + 3, row, scale=0.1)
    state = store[:, :vh * d * d].view(n + 3, vh, d, d)
    first, old = state.clone(), store.clone()
    order = np.random.default_rng(1).permutation(n + 3)[:n].astype(np.int32)
    out = torch.full((n, vh, d), 9.0, dtype=torch.bfloat16, device="cuda")
    skv.gated_delta(q, k, v, g, beta, state, out, state_index=torch.from_numpy(order).cuda())
    assert status(torch) == 0
    check_delta(torch, (q, k, v, g, beta), first, state, out, list(range(n + 1)), order.tolist())
    rest = sorted(set(range(n + 3)) - set(order.tolist()))
    assert torch.equal(store[rest], old[rest]) and torch.equal(store[:, vh * d * d:], old[:, vh * d * d:])


@pytest.mark.parametrize("count", [3, 150])
def test_delta_refuses_state_rows_on_the_device(torch_cuda, count):
    torch = torch_cuda
    counts = [count] * 4
    x = delta_inputs(torch, 25, sum(counts), 1, 2, 128, torch.float16)
    state = normal(torch, 26, 4, 2, 128, 128, scale=0.1)
    first = state.clone()
    out, starts = run_delta(torch, x, state, counts, state_index=ints(torch, [2, -1, 4, 0]))
    assert status(torch) == skv.STATUS_BAD_STATE_ROW
    want, final, far, off = R.delta(torch, *x, first, [0, count], [2], 128 ** -0.5)
    assert ((out[:count].double() - want[:count]).abs() <= far[:count]).all()
    assert (out[count:3 * count] == 9).all()
    assert torch.equal(state[1], first[1]) and torch.equal(state[3], first[3]) and not torch.equal(state[0], first[0])


@pytest.mark.parametrize("count", [1, 40, 200])
@pytest.mark.parametrize("case", ["forget", "keep", "never write", "same key", "reset now and then", "deep decay"])
def test_delta_edges(torch_cuda, count, case):
    """Decays of 0 and 1, write strengths of 0 and 1, one key over and over (the triangular system at its worst)."""
    torch = torch_cuda
    q, k, v, g, beta = delta_inputs(torch, 35, count, 2, 4, 128, torch.bfloat16)
    if case == "forget":
        g.fill_(-math.inf)
    elif case == "keep":
        g.zero_()
        beta.fill_(1.0)
    elif case == "never write":
        beta.zero_()
    elif case == "same key":
        g.zero_()
        beta.fill_(1.0)
        k[:] = k[:1]
    elif case == "reset now and then":
        g[::7] = -math.inf
        g[3::11] = -200.0
    else:
        g.fill_(-30.0)
    state = normal(torch, 36, 1, 4, 128, 128, scale=0.1)
    first = state.clone()
    out, starts = run_delta(torch, (q, k, v, g, beta), state, [count])
    check_delta(torch, (q, k, v, g, beta), first, state, out, starts, [0])


@pytest.mark.parametrize("most", [5, 100])
def test_delta_cuts_at_max_tokens(torch_cuda, most):
    torch = torch_cuda
    x = delta_inputs(torch, 45, 300, 1, 2, 128, torch.bfloat16)
    state = normal(torch, 46, 2, 2, 128, 128, scale=0.1)
    first = state.clone()
    out, starts = run_delta(torch, x, state, [150, 150], max_tokens=most)
    for s, a in enumerate((0, 150)):
        want, final, far, off = R.delta(torch, *x, first, [a, a + most], [s], 128 ** -0.5)
        assert ((out[a:a + most].double() - want[a:a + most]).abs() <= far[a:a + most]).all()
        assert ((state[s].double() - final[s]).flatten(1).norm(dim=1) <= off[s]).all()
        assert (out[a + most:a + 150] == 9).all()


def test_delta_in_parts_equals_the_whole(torch_cuda):
    """A prompt in pieces of any size, the state carried between the calls; and the same bits from the same inputs."""
    torch = torch_cuda
    n = 500
    x = delta_inputs(torch, 55, n, 2, 4, 128, torch.float16)
    first = normal(torch, 56, 1, 4, 128, 128, scale=0.1)
    state, outs, at = first.clone(), [], 0
    for piece in (1, 63, 64, 2, 130, 1, 239):
        part = tuple(z[at:at + piece] for z in x)
        outs.append(run_delta(torch, part, state, [piece])[0])
        at += piece
    check_delta(torch, x, first, state, torch.cat(outs), [0, n], [0])
    one, two = first.clone(), first.clone()
    a, b = run_delta(torch, x, one, [n])[0], run_delta(torch, x, two, [n])[0]
    assert torch.equal(a, b) and torch.equal(one, two)


def test_delta_in_a_graph(torch_cuda):
    """A decode step and a prompt, captured and replayed on other inputs; the state goes on from replay to replay."""
    torch = torch_cuda
    for counts in ([1, 1, 1], [100, 70, 3]):
        n = sum(counts)
        x = delta_inputs(torch, 65, n, 1, 2, 128, torch.bfloat16)
        state = normal(torch, 66, 3, 2, 128, 128, scale=0.1)
        starts = ints(torch, list(np.cumsum([0] + counts)))
        work = torch.empty(max(16, skv.gated_delta_workspace(n, 3, 2, 128, max(counts))), dtype=torch.uint8, device="cuda")
        out = torch.empty(n, 2, 128, dtype=torch.bfloat16, device="cuda")
        call = lambda: skv.gated_delta(*x, state, out, seq_starts=starts, max_tokens=max(counts), workspace=work,  # noqa: E731
                                       stream=torch.cuda.current_stream())
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for step in range(2):
            for have, new in zip(x, delta_inputs(torch, 70 + step, n, 1, 2, 128, torch.bfloat16)):
                have.copy_(new)
            first = state.clone()
            graph.replay()
            torch.cuda.synchronize()
            check_delta(torch, x, first, state, out, starts.tolist(), [0, 1, 2])


def test_a_gradient_that_would_be_lost_is_refused(torch_cuda):
    """Each activation, gate and state of each call; without recording the results are those of plain tensors."""
    torch = torch_cuda
    layer = make_layer(torch, 2, [4])
    for name in ("q", "k", "v", "g", "beta", "state", "out"):
        x = dict(zip(("q", "k", "v", "g", "beta"), delta_inputs(torch, 3, 2, 1, 2, 64, torch.float16)))
        x["state"], x["out"] = torch.zeros(2, 2, 64, 64, device="cuda"), torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
        x[name].requires_grad_()
        with pytest.raises(TypeError, match=f"{name}: requires a gradient"):
            skv.gated_delta(**x)
        with torch.no_grad():
            skv.gated_delta(**x)
        assert x["state"].any() and x["out"].any()
    row, q = normal(torch, 4, 1, 2, 256, dtype=torch.float16), normal(torch, 5, 1, 24, 256, dtype=torch.float16)
    with pytest.raises(TypeError, match="v: requires a gradient"):
        skv.kv_append(layer, row, row.clone().requires_grad_(), ints(torch, [0]))
    with pytest.raises(TypeError, match="q: requires a gradient"):
        run_attention(torch, layer, q.clone().requires_grad_(), [4], 0.0625)
    with torch.no_grad():
        got = run_attention(torch, layer, q.clone().requires_grad_(), [4], 0.0625)
    assert torch.equal(got[0], run_attention(torch, layer, q, [4], 0.0625)[0])


# ------------------------------------------------------------------------------------------------ all of them, as a serving step uses them

def test_a_conversation_is_prefilled_handed_over_and_continued(torch_cuda):
    """Prompts fill one block pool and one set of state rows, one launch moves a conversation to other slots of another
    pool, and decoding goes on there: every token's outputs equal the 64-bit implementation's over the whole conversation."""
    torch = torch_cuda
    g = skv.KvGeometry(n_layers=4, qsa_interval=4)
    prompts, more = [517, 130], 6
    kv, heads, dim, kh, vh, d = 2, 24, 256, 2, 4, 128
    inv = 1e6 ** (-torch.arange(32, device="cuda") / 32)

    def place(seed):
        memory = torch.zeros(32 * g.block_bytes, dtype=torch.uint8, device="cuda")
        pool = skv.Pool(0, 32, g.block_bytes, memory=memory)
        pool.scramble(seed)
        blocks = [pool.alloc(g.blocks(n + more)) for n in prompts]
        tables = np.full((2, 3 * g.pages_per_block), -1, np.int32)
        for s, b in enumerate(blocks):
            tables[s, :len(b) * g.pages_per_block] = skv.layer_page_tables(g, b)[0]
        tables = torch.from_numpy(tables).cuda()
        return memory, pool, blocks, tables, skv.KvLayer.of_pool(g, pool, tables)

    src, dst = place(1), place(2)
    total = [n + more for n in prompts]
    q, k, v = (normal(torch, 100 + i, sum(total), h, dim, dtype=torch.bfloat16) for i, h in enumerate((heads, kv, kv)))
    x = delta_inputs(torch, 110, sum(total), kh, vh, d, torch.bfloat16)
    first = [0, total[0], sum(total)]
    pick = torch.cat([torch.arange(first[s], first[s] + n) for s, n in enumerate(prompts)]).cuda()
    starts = ints(torch, [0, prompts[0], sum(prompts)])

    # the prefill role
    state = torch.zeros(2, vh, d, d, device="cuda")
    lengths = [ints(torch, [0, 0]), ints(torch, [0, 0])]
    skv.kv_append(src[4], k[pick], v[pick], lengths[0], seq_starts=starts, inv_freq=inv, lengths_out=lengths[1])
    prompt_out, _ = run_delta(torch, tuple(z[pick] for z in x), state, prompts)

    # the hand-over: every page of both conversations and the state rows in one launch
    new_state = torch.zeros_like(state)
    segs = [skv.segment(state, new_state, state.numel() * 4)]
    held = []
    for s, n in enumerate(prompts):
        tabs = [[torch.from_numpy(t).cuda() for t in skv.layer_page_tables(g, side[2][s])] for side in (src, dst)]
        held.append(tabs)
        for a, b in zip(*tabs):
            segs.append(skv.segment(src[1].base, dst[1].base, g.pages(n) * g.page_bytes, src_pages=a, dst_pages=b, page_bytes=g.page_bytes,
                                    src_page_limit=32 * g.slot_pages, dst_page_limit=32 * g.slot_pages))
    skv.copy(segs)

    # the decode role
    layer = dst[4]
    outs, delta_outs = [], []
    work = torch.empty(skv.decode_attention_workspace(layer, 2, heads), dtype=torch.uint8, device="cuda")
    have, then = lengths[1], lengths[0]
    for i in range(more):
        at = torch.tensor([first[s] + n + i for s, n in enumerate(prompts)], device="cuda")
        query, out = q[at], torch.empty(2, heads, dim, dtype=torch.bfloat16, device="cuda")
        skv.kv_append(layer, k[at], v[at], have, q=query, q_out=query, inv_freq=inv, lengths_out=then)
        skv.decode_attention(layer, query, then, out, workspace=work)
        have, then = then, have
        outs.append((query, out))
        step = torch.full((2, vh, d), 9.0, dtype=torch.bfloat16, device="cuda")
        skv.gated_delta(*(z[at] for z in x), new_state, step)
        delta_outs.append(step)
    assert status(torch) == 0
    assert have.tolist() == total

    # the delta rule over each whole conversation
    whole = torch.empty(sum(total), vh, d, dtype=torch.bfloat16, device="cuda")
    whole[pick] = prompt_out
    for i in range(more):
        for s, n in enumerate(prompts):
            whole[first[s] + n + i] = delta_outs[i][s]
    check_delta(torch, x, torch.zeros_like(state), new_state, whole, first, [0, 1])
    # attention over the rotated keys as the cache's type holds them
    for s, n in enumerate(prompts):
        rows = torch.stack([R.rotated(torch, k[first[s] + t].double(), t, inv, "half")[0] for t in range(total[s])])
        keys, values = rows.transpose(0, 1).repeat_interleave(12, 0), v[first[s]:first[s + 1]].double().transpose(0, 1).repeat_interleave(12, 0)
        for i in range(more):
            query, out = outs[i][0][s].double(), outs[i][1][s].double()
            seen = n + i + 1
            p = torch.softmax(torch.einsum("hd,hnd->hn", query, keys[:, :seen]) / 16, -1)
            want = torch.einsum("hn,hnd->hd", p, values[:, :seen])
            # keys and values rounded to float16: a score moves by at most 2^-11 sum |q k| / 16, twice in a weight
            slack = 2 * 2.0 ** -11 * torch.einsum("hd,hnd->hn", query.abs(), keys[:, :seen].abs()).amax(1) / 16
            spread = torch.einsum("hn,hnd->hd", p, values[:, :seen].abs())
            assert ((out - want).abs() <= spread * (slack[:, None] + 2 * 2.0 ** -11 + 2.0 ** -13) + want.abs() * 2.0 ** -8 * 1.01 + 2.0 ** -24).all()
            # the query that was read is the rotated one
            turned, mag = R.rotated(torch, q[first[s] + n + i].double(), n + i, inv, "half")
            assert ((query - turned).abs() <= 6 * 2.0 ** -24 * mag + turned.abs() * 2.0 ** -8 * 1.01 + 2.0 ** -100).all()


def test_a_decode_step_in_a_graph_goes_on(torch_cuda):
    """Append, attention and a delta step captured once; each replay goes one cell further, with the bits of plain calls."""
    torch = torch_cuda
    cells, steps = [30, 257, 4], 5
    layers = [make_layer(torch, 121, [n + steps for n in cells]) for _ in range(2)]
    inv = 1e4 ** (-torch.arange(32, device="cuda") / 32)
    inputs = [[normal(torch, 130 + 10 * i + j, 3, h, 256, dtype=torch.bfloat16) for j, h in enumerate((24, 2, 2))] for i in range(steps)]
    deltas = [delta_inputs(torch, 200 + i, 3, 2, 4, 128, torch.bfloat16) for i in range(steps)]
    results = []
    for captured, layer in enumerate(layers):
        q, k, v = (torch.empty_like(x) for x in inputs[0])
        d = [torch.empty_like(x) for x in deltas[0]]
        have, then = ints(torch, cells), ints(torch, [0] * 3)
        state = normal(torch, 140, 3, 4, 128, 128, scale=0.1)
        out, delta_out = torch.empty_like(q), torch.empty(3, 4, 128, dtype=torch.bfloat16, device="cuda")
        work = torch.empty(skv.decode_attention_workspace(layer, 3, 24), dtype=torch.uint8, device="cuda")

        def step():
            on = torch.cuda.current_stream()
            skv.kv_append(layer, k, v, have, q=q, q_out=q, inv_freq=inv, lengths_out=then, stream=on)
            skv.decode_attention(layer, q, then, out, workspace=work, stream=on)
            skv.gated_delta(*d, state, delta_out, stream=on)
            have.copy_(then)

        graph = None
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        outs = []
        for i in range(steps):
            for to, new in zip((q, k, v, *d), (*inputs[i], *deltas[i])):
                to.copy_(new)
            graph.replay() if captured else step()
            outs += [out.clone(), delta_out.clone(), q.clone()]
        assert have.tolist() == [n + steps for n in cells]
        results.append((outs, state, layer.tensors[0], layer.tensors[1]))
    assert status(torch) == 0
    assert all(torch.equal(a, b) for a, b in zip(results[0][0], results[1][0]))
    assert all(torch.equal(a, b) for a, b in zip(results[0][1:], results[1][1:]))
    # and the first step's attention is the 64-bit one's over what the cache held then
    layer, lengths = layers[0], [n + 1 for n in cells]
    want, _, far, _ = R.attention(torch, layer, results[0][0][2], lengths, 0.0625)
    assert ((results[0][0][0].double() - want).abs() <= far).all()

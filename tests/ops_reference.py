"""The operators of skv.py in 64 bits, cell by cell and token by token, and bounds on what a kernel may be off.

HALF is the largest relative error of one rounding to a type (half its step)."""
import math

HALF = {"torch.float16": 2.0 ** -11, "torch.bfloat16": 2.0 ** -8, "torch.float32": 2.0 ** -24}
TINY = {"torch.float16": 2.0 ** -25, "torch.bfloat16": 2.0 ** -134}     # half the smallest step


def half(dtype) -> float:
    return HALF[str(dtype)]


def tiny(dtype) -> float:
    return TINY[str(dtype)]


def rotated(torch, x, cell, inv_freq, style):
    """x [..., dim] in 64 bits, turned by cell * inv_freq; and what each value's two products sum to in magnitude."""
    y, size = x.clone(), x.abs()
    half_rot = inv_freq.shape[0]
    a = torch.arange(half_rot, device=x.device)
    first, second = (a, a + half_rot) if style == "half" else (2 * a, 2 * a + 1)
    angle = float(cell) * inv_freq.double()
    c, s = angle.cos(), angle.sin()
    u, w = x[..., first], x[..., second]
    y[..., first], y[..., second] = u * c - w * s, w * c + u * s
    size[..., first] = size[..., second] = u.abs() + w.abs()
    return y, size


def cells_of(torch, layer, seq: int, n: int):
    """K and V of cells 0..n-1 of a sequence in 64 bits, [kv_head][n][dim] (an entry outside the pool: NaN), and which
    cells are held."""
    k_pool, v_pool, k_scale, v_scale, tables = layer.tensors
    pages, kv, size, dim = k_pool.shape
    row = tables[seq].tolist()
    held = torch.tensor([0 <= row[t // size] < pages for t in range(n)], dtype=torch.bool, device=k_pool.device)
    page = torch.tensor([row[t // size] if 0 <= row[t // size] < pages else 0 for t in range(n)], dtype=torch.long, device=k_pool.device)
    slot = torch.arange(n, device=k_pool.device) % size
    out = []
    for pool, scale in ((k_pool, k_scale), (v_pool, v_scale)):
        x = pool[page, :, slot].double()
        if scale is not None:
            x = x * scale[page, :, slot].double().repeat_interleave(64, -1)
        out.append(x.transpose(0, 1))
    return out[0], out[1], held


def attention(torch, layer, q, lengths, scale):
    """(out, lse, bound on |out|, bound on |lse|) of one token per sequence.

    Bound.  A score is a sum of `dim` products in 32 bits: off by at most (dim + 4) 2^-24 sum |q k| scale =: e (products
    of 16-bit values are exact; the scale, its application and an int8 group's scale are four more roundings).  So a
    weight is off by a factor within e^(+-2e) (the score's and the maximum's), by 2^-11 where it is rounded to 16 bits for
    the product with V, and by 2^-20 for exp, the rescalings of a running maximum and the joining of parts; the sum
    of n weights is off by the same without the 2^-11 (32 bits, random order: 2^-24 times its adds, under 2^-16 at
    256 adds a thread).  A 16-bit weight may also be a subnormal: 2^-25 of the largest (they are scaled by 2^15)."""
    n_seqs, heads, dim = q.shape
    kv = layer.n_head_kv
    out = torch.zeros(n_seqs, heads, dim, dtype=torch.float64, device=q.device)
    lse = torch.full((n_seqs, heads), -math.inf, dtype=torch.float64, device=q.device)
    far, far_lse = torch.zeros_like(out), torch.zeros_like(lse)
    size = layer.args.page_size
    for s in range(n_seqs):
        n = min(max(int(lengths[s]), 0), layer.tensors[4].shape[1] * size)
        if n == 0:
            continue
        k, v, held = cells_of(torch, layer, s, n)
        k, v = k.repeat_interleave(heads // kv, 0)[:, held], v.repeat_interleave(heads // kv, 0)[:, held]
        if k.shape[1] == 0:
            continue
        x = q[s].double()
        score = torch.einsum("hd,hnd->hn", x, k) * scale
        e = (dim + 4) * 2.0 ** -24 * torch.einsum("hd,hnd->hn", x.abs(), k.abs()).amax(1) * abs(scale)
        top = score.amax(1, keepdim=True)
        some = torch.isfinite(top[:, 0]) | torch.isnan(top[:, 0]) | (top[:, 0] == math.inf)
        weight = torch.where(score == -math.inf, 0.0, torch.exp(score - torch.where(some[:, None], top, 0.0)))
        total = weight.sum(1, keepdim=True)
        p = weight / torch.where(total > 0, total, 1.0)
        out[s] = torch.einsum("hn,hnd->hd", p, v)
        lse[s] = torch.where(total[:, 0] > 0, top[:, 0] + total[:, 0].log(), -math.inf)
        spread = torch.einsum("hn,hnd->hd", p, v.abs())
        off = 4 * e + 2.0 ** -11 + 2.0 ** -15
        far[s] = spread * off[:, None] + 2.0 ** -25 * v.abs().sum(1) / torch.where(total > 0, total, 1.0)
        far[s] += out[s].abs() * half(q.dtype) * (1 + 2.0 ** -8) + tiny(q.dtype)
        far_lse[s] = 2 * e + 2.0 ** -15 + lse[s].abs() * 2.0 ** -22
    return out, lse, far, far_lse


def delta(torch, q, k, v, g, beta, state, starts, rows, scale):
    """(out, state, bound on |out|, bound on the 2-norm of a head's state) of the gated delta rule.

    Bound.  One token changes a head's S by a decay, a product with k and an update; in 32 bits each is off by a few
    2^-24 of the 2-norm of what it works on (a dot product of d terms by sqrt(d) 2^-24 in the 2-norm for roundings
    that do not conspire; 16 covers d = 128 with the other roundings).  The step is a contraction for |k| <= 1,
    beta <= 1, g <= 0, so the errors of T tokens add up to at most T * 16 * 2^-24 of the largest norm met.  Where a chunk
    is worked out at once the same holds with its triangular system in between: another factor of 2.  The output is a
    product of q with S, whose operands may be rounded to 11 bits (2 * 2^-11 of |q| |S column| and as much for the
    part from inside of the chunk, whose weights sum over at most 64 tokens), and its own rounding."""
    n, kh, d = q.shape
    vh = v.shape[1]
    out = torch.zeros(n, vh, d, dtype=torch.float64, device=q.device)
    far = torch.zeros_like(out)
    final = state.double().clone()
    off = torch.zeros(state.shape[0], vh, dtype=torch.float64, device=q.device)
    ratio = vh // kh
    for s, r in enumerate(rows):
        S = final[r]
        a, b = starts[s], starts[s + 1]
        most = S.flatten(1).norm(dim=1)
        for t in range(a, b):
            key, query = k[t].double().repeat_interleave(ratio, 0), q[t].double().repeat_interleave(ratio, 0)
            S = S * torch.exp(g[t].double())[:, None, None]
            wrong = beta[t].double()[:, None] * (v[t].double() - torch.einsum("hi,hij->hj", key, S))
            S = S + key[:, :, None] * wrong[:, None, :]
            most = torch.maximum(most, torch.maximum(S.flatten(1).norm(dim=1), wrong.norm(dim=1)))
            out[t] = scale * torch.einsum("hi,hij->hj", query, S)
            column = torch.einsum("hi,hij->hj", query.abs(), S.abs())
            off_t = (t - a + 1) * 32 * 2.0 ** -24 * most
            inner = min(t - a + 1, 64) ** 0.5 * query.norm(dim=1) * most
            far[t] = (scale * (off_t * query.norm(dim=1) + 4 * 2.0 ** -11 * inner)[:, None] + scale * 2 * 2.0 ** -11 * column
                      + out[t].abs() * half(q.dtype) * (1 + 2.0 ** -8) + tiny(q.dtype))
        final[r] = S
        off[r] = (b - a) * 32 * 2.0 ** -24 * most
    return out, final, far, off

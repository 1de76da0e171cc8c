"""The gated delta rule of skv.py in 64 bits, 64 tokens at a time, with a bound for each output from what it is summed of.

With G the sums of g from a chunk's first token on, and S the state before it:
    A_ij = beta_i e^(G_i - G_j) k_i . k_j (j < i),  T = (I + A)^-1,  P_ij = e^(G_i - G_j) q_i . k_j (j <= i)
    R = beta (V - e^G K S),  V' = T R,  O = scale (e^G Q S + P V'),  S <- e^(G_end) S + K^T (e^(G_end - G) V')

What a kernel may be off (u v: products of magnitudes; c a value column; `top` the largest magnitude in the 16 columns c is one of):
  * Each product stage is off by W = 2^-18 of the sum of its magnitudes: sums of up to 128 products in 32 bits that round or
    cut 16 times by 2^-23 (2^-19), operands of two 16-bit parts (2^-22 each), factors with a few 2^-22.  K K^T and Q K^T are such
    stages: where q_i . k_j nearly cancels, P_ij is off by W of |q_i| . |k_j| all the same.
  * An operand's parts end 2^-39 below its largest value (here 2^-38), T's at 2^-30 (2^-29), P's 2^-37 d below the largest values of
    its query and the chunk's keys, bfloat16 q and k 2^-24 below the largest.
  * Q S takes one part of S: 2^-11 of each product.  P V' of bfloat16 outputs takes one part of each: 2^-11 twice.
  * What was off in S before the chunk grows no more, as a step is a contraction (beta |k|^2 <= 2): E_c bounds |dS_c|, and moves
    an output by at most |q| E_c.  What is new in R and V' is followed through |T|, |P| and |K|.
  * The output is rounded once, from a value that is off already: half a step of |O| and of what it is off by.
Token by token (chunk 1) the same holds without the 16-bit parts.

`far` bounds every element.  `square` is the mean square of the 16-bit roundings as if each were evenly spread over its step
(a third of its greatest square) and independent of the others, `rest` bounds what else there is: over some thousand values the
root mean square of the errors is at most that of both together.  A state gets a second bound in the same way: the stages' errors as
W of the root of the sum of their products' squares, independent of each other, over all of a head's columns."""
import ops_reference as R

W = 2.0 ** -18
HALF16 = 2.0 ** -11
GROUP = 16


def _top(x):
    """[head][row][column]: the largest magnitude over all rows of 16 columns, for each column, [head][1][column]."""
    return x.abs().amax(1, keepdim=True).unflatten(2, (-1, GROUP)).amax(-1, keepdim=True).expand(-1, -1, -1, GROUP).flatten(2)


def chunks(torch, q, k, v, g, beta, state, first, last, chunk):
    """Each chunk of one sequence: its tokens, and the matrices above in 64 bits, [head][token or key][...]."""
    ratio = v.shape[1] // k.shape[1]
    S = state.double()
    for a in range(first, last, chunk):
        b = min(a + chunk, last)
        Q, K = (x[a:b].double().repeat_interleave(ratio, 1).transpose(0, 1) for x in (q, k))
        V = v[a:b].double().transpose(0, 1)
        G = g[a:b].double().clamp(min=-1e4).cumsum(0).transpose(0, 1)
        write = beta[a:b].double().transpose(0, 1)[..., None]
        lower = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).tril()
        decay = torch.where(lower, torch.exp(torch.where(lower, G[..., :, None] - G[..., None, :], 0.0)), 0.0)
        A = (write * decay * (K @ K.transpose(1, 2))).tril(-1)
        eye = torch.eye(b - a, dtype=torch.float64, device=q.device)
        T = torch.linalg.solve_triangular(eye + A, eye.expand_as(A), upper=False, unitriangular=True)
        P = decay * (Q @ K.transpose(1, 2))
        into, left, whole = G.exp()[..., None], (G[:, -1:] - G).exp()[..., None], G[:, -1].exp()[:, None, None]
        rest = write * (V - into * (K @ S))
        value = T @ rest
        after = whole * S + (K * left).transpose(1, 2) @ value
        yield dict(decay=decay, a=a, b=b, Q=Q, K=K, V=V, write=write, A=A, T=T, P=P, into=into, left=left, whole=whole, R=rest, value=value, S=S, after=after)
        S = after


def delta(torch, q, k, v, g, beta, state, starts, rows, scale, chunk=64):
    """(out, state, far, square, rest, E, spread): see above; E [row][head][column], spread [row][head] of the 2-norm of a head's
    state.  Rows of no sequence: out and bounds are zeros."""
    out = torch.zeros(v.shape, dtype=torch.float64, device=q.device)
    far, square, rest = (torch.zeros_like(out) for _ in range(3))
    final = state.double().clone()
    off = torch.zeros(state.shape[0], v.shape[1], v.shape[2], dtype=torch.float64, device=q.device)
    spread = torch.zeros(state.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
    kind, d = q.dtype, q.shape[2]
    half, narrow = R.half(kind), kind == torch.bfloat16
    one = HALF16 if chunk > 1 else 0.0                    # S in Q S
    two = HALF16 if chunk > 1 and narrow else 0.0         # P and V' each
    for s, r in enumerate(rows):
        E = torch.zeros(v.shape[1], 1, d, dtype=torch.float64, device=q.device)
        square_sum = torch.zeros_like(E)
        for c in chunks(torch, q, k, v, g, beta, state[r], starts[s], starts[s + 1], chunk):
            S, K, Q, P, T, into = c["S"].abs(), c["K"].abs(), c["Q"].abs(), c["P"].abs(), c["T"].abs(), c["into"]
            value, wrong, write = c["value"].abs(), c["R"].abs(), c["write"]
            d_mix, d_solve = (W * c["decay"] * (x @ K.transpose(1, 2)) for x in (Q, write * K))    # of P, of A
            columns = S.sum(1, keepdim=True)
            key_floor = 2.0 ** -24 * K.amax((1, 2), keepdim=True) * columns * narrow
            query_floor = 2.0 ** -24 * Q.amax(2, keepdim=True) * columns * narrow
            d_rest = write * into * (2 * W * (K @ S) + 2.0 ** -38 * _top(S) * K.sum(2, keepdim=True) + key_floor) + W * write * c["V"].abs()
            d_rest = d_rest + 2.0 ** -38 * _top(wrong)
            eye = torch.eye(T.shape[1], dtype=torch.float64, device=q.device)
            ones = torch.ones_like(eye).tril()
            d_value = T @ d_rest + (T @ (W * eye + d_solve) @ T + 2.0 ** -29 * (T @ ones @ T)) @ wrong
            qs, pv = Q @ S, P @ value
            small = W * into * qs + into * (2.0 ** -38 * _top(S) * Q.sum(2, keepdim=True) + query_floor) + W * pv + d_mix @ value
            small = small + 2.0 ** -38 * _top(value) * P.sum(2, keepdim=True)
            small = small + 2.0 ** -37 * d * Q.amax(2, keepdim=True) * K.amax((1, 2), keepdim=True) * value.sum(1, keepdim=True)
            small = scale * (small + Q.norm(dim=2, keepdim=True) * E + P @ d_value)
            got = scale * (into * (c["Q"] @ c["S"]) + c["P"] @ c["value"])
            t = slice(c["a"], c["b"])
            out[t], rest[t] = got.transpose(0, 1), small.transpose(0, 1)
            far[t] = (small + scale * (one * into * qs + 2 * two * pv)).transpose(0, 1)
            square[t] = (scale ** 2 / 3 * (one ** 2 * into ** 2 * (Q ** 2 @ S ** 2) + 2 * two ** 2 * (P ** 2 @ value ** 2))).transpose(0, 1)
            left = c["left"]
            E = E + (K.norm(dim=2, keepdim=True) * left * (d_value + W * value)).sum(1, keepdim=True) + W * S.norm(dim=1, keepdim=True)
            E = E + 2.0 ** -38 * _top(left * value) * K.norm(dim=2).sum(1)[:, None, None]
            final[r] = c["after"]
            floors = write * into * (2.0 ** -38 * _top(S) * K.sum(2, keepdim=True) + key_floor) + 2.0 ** -38 * _top(wrong)
            d_rest2 = (write * W) ** 2 * (into ** 2 * (K ** 2 @ S ** 2) + c["V"] ** 2) + floors ** 2
            d_value2 = T ** 2 @ d_rest2 + (T @ (W * eye + d_solve) @ T) ** 2 @ wrong ** 2 + ((2.0 ** -29 * (T @ ones @ T)) @ wrong) ** 2
            square_sum = square_sum + ((K.norm(dim=2, keepdim=True) * left) ** 2 * (d_value2 + (W * value) ** 2)).sum(1, keepdim=True)
            square_sum = square_sum + (W * S.norm(dim=1, keepdim=True)) ** 2 + (2.0 ** -38 * _top(left * value) * K.norm(dim=2).sum(1)[:, None, None]) ** 2
        off[r], spread[r] = E[:, 0], square_sum.sum((1, 2)).sqrt()
    tiny = R.tiny(kind)
    return (out, final, far * (1 + half) + out.abs() * half + tiny, square + (out * half) ** 2 / 3, rest + tiny, off, spread)


def wrong_outputs(torch, got, bounds, tokens=slice(None)):
    """What is wrong with outputs [token][head][column]: None, or which of the two bounds they break and by what factor."""
    out, _, far, square, rest, *_ = bounds
    error = (got.double() - out).abs()[tokens]
    worst = float((error / far[tokens].clamp(min=2.0 ** -1000)).nan_to_num(nan=1e30).max()) if error.numel() else 0.0
    if worst > 1:
        return f"an element by {worst:.3g}"
    if error[:, 0].numel() >= 2048:
        size = (error ** 2).mean((0, 2)).sqrt()
        most = square[tokens].mean((0, 2)).sqrt() + (rest[tokens] ** 2).mean((0, 2)).sqrt()
        if bool((size > most).any()):
            return f"the root mean square by {float((size / most).max()):.3g}"
    return None


def wrong_state(torch, state, bounds):
    """What is wrong with the state: None, or which bound it breaks and by what factor."""
    _, final, _, _, _, off, spread = bounds
    size = (state.double() - final).norm(dim=2)
    for what, most, limit in (("a column", size, off + final.norm(dim=2) * 2.0 ** -23),
                              ("a head", size.norm(dim=2), spread + final.flatten(2).norm(dim=2) * 2.0 ** -23)):
        if not bool((most <= limit).all()):
            return f"{what} by {float((most / limit.clamp(min=2.0 ** -1000)).nan_to_num(nan=1e30).max()):.3g}"
    return None

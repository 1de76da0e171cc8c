"""The operators on a paged K/V cache and on the linear-attention state, as cases that can be timed and compared.

Three operators, at the geometry the framework moves (24 query heads, 2 K/V heads of 256, pages of 4 cells; 32 value
heads and 16 key heads of 128 on the state rows) and at others:

  append     K and V of new tokens into a paged cache, with the rotary positions applied on the way (and to q)
  attention  one new token per sequence over its paged cache
  delta      the gated delta rule on the fp32 state rows, one token per sequence or whole prompts

`own` False computes them in elementary torch operations, True through the framework's entry points.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GROUP = 64      # values per scale of an int8 cache
CHUNK = 64      # tokens per step of the plain delta rule


def _skv():
    path = os.path.join(os.getcwd(), "strata-concurrent_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import skv
    return skv


# ------------------------------------------------------------------------------------------------ cases

def listed():
    """Lengths are the ones the framework's own benchmark moves (1K, 4K, 32K, 128K) or ragged around them."""
    cache = {"heads": 24, "kv_heads": 2, "dim": 256, "page": 4, "rot": 64, "style": "half"}
    state = {"k_heads": 16, "v_heads": 32, "dim": 128}
    return [
        # one token of one conversation: the smallest call of a decode loop
        {"name": "append 1 token", "op": "append", **cache, "tokens": "1", "before": 32767, "type": "bf16", "int8": False},
        # one token of each of 64 conversations at once
        {"name": "append 64 x 1", "op": "append", **cache, "tokens": ",".join(["1"] * 64), "before": 4093, "type": "bf16", "int8": False},
        # a 32K prompt entering the cache
        {"name": "append 32K prompt", "op": "append", **cache, "tokens": "32768", "before": 0, "type": "bf16", "int8": False},
        # ragged prompts, some of them continuing a conversation, into an int8 cache
        {"name": "append ragged int8", "op": "append", **cache, "tokens": "1,2051,4096,255,3,1025,0,517", "before": 129, "type": "f16", "int8": True},
        # one short conversation: latency
        {"name": "attention 1K", "op": "attention", **cache, "lengths": "1000", "type": "bf16", "int8": False},
        # one long conversation: the whole card on one sequence
        {"name": "attention 128K", "op": "attention", **cache, "lengths": "131072", "type": "bf16", "int8": False},
        # a served batch, lengths log-uniform, one slot empty and one just begun
        {"name": "attention ragged 32", "op": "attention", **cache, "type": "f16", "int8": False,
         "lengths": "0,1,17,16384,1003,1024,1291,1400,1733,2047,2300,2515,3001,3333,4096,4099,4500,5121,6000,6145,7000,"
                    "7777,8192,8195,9001,10007,11111,12288,13001,14002,15555,2222"},
        # eight 32K conversations in an int8 cache
        {"name": "attention int8 8 x 32K", "op": "attention", **cache, "lengths": ",".join(["32768"] * 8), "type": "bf16", "int8": True},
        # one token of one conversation through one linear-attention layer
        {"name": "delta 1 token", "op": "delta", **state, "tokens": "1", "type": "bf16"},
        # one token of each of 64 conversations
        {"name": "delta 64 x 1", "op": "delta", **state, "tokens": ",".join(["1"] * 64), "type": "bf16"},
        # a 32K prompt
        {"name": "delta 32K prompt", "op": "delta", **state, "tokens": "32768", "type": "bf16"},
        # a batch of ragged prompts
        {"name": "delta ragged", "op": "delta", **state, "tokens": "4096,1,2047,1025,63,3333,0,512,65,1500,2500,800", "type": "f16"},
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    op = rng.choice(["append", "attention", "delta", "delta"])
    kind = rng.choice(["bf16", "f16"])
    if op == "delta":
        k_heads, ratio = rng.choice([(16, 2), (16, 3), (8, 1), (16, 1), (4, 4)])
        base = {"op": op, "k_heads": k_heads, "v_heads": k_heads * ratio, "dim": rng.choice([128, 128, 64]), "type": kind}
        if rng.random() < 0.5:       # decode
            n = _log_uniform(rng, 1, 96)
            return {**base, "tokens": ",".join(["1"] * n)}
        n = _log_uniform(rng, 1, 12)
        return {**base, "tokens": ",".join(str(_log_uniform(rng, 1, 16384 // n)) for _ in range(n))}
    heads, kv, dim, rot = rng.choice([(24, 2, 256, 64), (24, 2, 256, 64), (32, 8, 128, 128), (16, 1, 256, 64), (40, 8, 128, 64), (8, 8, 64, 32)])
    base = {"op": op, "heads": heads, "kv_heads": kv, "dim": dim, "page": rng.choice([4, 4, 16, 64]), "rot": rot,
            "style": rng.choice(["half", "pairs"]), "type": kind, "int8": rng.random() < 0.4}
    if op == "append":
        n = _log_uniform(rng, 1, 64)
        each = 1 if rng.random() < 0.4 else _log_uniform(rng, 1, 16384 // n)
        return {**base, "tokens": ",".join(str(rng.randint(max(1, each // 2), each)) for _ in range(n)), "before": rng.randint(0, 3000)}
    n = _log_uniform(rng, 1, 48)
    return {**base, "lengths": ",".join(str(_log_uniform(rng, 1, min(32768, 131072 // n))) for _ in range(n))}


def _ints(text):
    return [int(x) for x in text.split(",")]


def work(case):
    el = 2
    if case["op"] == "append":
        n, row = sum(_ints(case["tokens"])), case["kv_heads"] * case["dim"]
        out = row + row // GROUP * 2 if case["int8"] else row * 2
        q = case["heads"] * case["dim"]
        return {"bytes": n * (2 * row * el + 2 * out + 2 * q * el) + 4 * n / case["page"],
                "flops": n * (3 * (case["heads"] + case["kv_heads"]) * case["rot"] + (4 * row if case["int8"] else 0))}
    if case["op"] == "attention":
        lens = _ints(case["lengths"])
        row = case["kv_heads"] * case["dim"]
        cell = row + row // GROUP * 2 if case["int8"] else row * 2
        q = case["heads"] * case["dim"]
        return {"bytes": sum(lens) * (2 * cell + 4 / case["page"]) + len(lens) * (2 * q * el + 4 * case["heads"]),
                "flops": 4.0 * sum(lens) * q}
    counts = _ints(case["tokens"])
    n, d = sum(counts), case["dim"]
    rows = sum(c > 0 for c in counts)
    return {"bytes": n * (2 * case["k_heads"] * d * el + 2 * case["v_heads"] * d * el + 8 * case["v_heads"]) + rows * 2 * 4 * case["v_heads"] * d * d,
            "flops": 7.0 * n * case["v_heads"] * d * d}


# ------------------------------------------------------------------------------------------------ inputs

def _normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _tables(gen, cells, page, spare):
    """A page table per sequence at random pages of one pool, and the pool's pages.  Rows are padded with page 0."""
    need = [(c + page - 1) // page for c in cells]
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    width = max(need) + 1
    table = torch.zeros(len(cells), width, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, total


def _starts(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": dict(case)}
    kind = DTYPES[case["type"]]
    if case["op"] == "delta":
        counts = _ints(case["tokens"])
        n, d, kh, vh = sum(counts), case["dim"], case["k_heads"], case["v_heads"]
        unit = lambda x: (x / x.float().norm(dim=-1, keepdim=True)).to(kind)  # noqa: E731
        st["q"], st["k"] = unit(_normal(gen, n, kh, d)), unit(_normal(gen, n, kh, d))
        st["v"] = _normal(gen, n, vh, d, dtype=kind)
        # a head forgets over some ten to some thousand tokens; the write strength is a sigmoid
        slow = torch.exp(torch.rand(vh, generator=gen, device="cuda") * 5 - 7)
        st["g"] = -slow * torch.nn.functional.softplus(_normal(gen, n, vh) + 1)
        st["beta"] = torch.sigmoid(_normal(gen, n, vh))
        st["state"] = _normal(gen, len(counts), vh, d, d, scale=0.02)
        st["starts"] = None if all(c == 1 for c in counts) else _starts(counts)
        st["longest"] = max(counts)
        st["out"] = torch.zeros(n, vh, d, dtype=kind, device="cuda")
        st["scale"] = d ** -0.5
        if own:     # the workspace a program keeps beside its state rows
            skv = _skv()
            st["workspace"] = torch.zeros(max(16, skv.gated_delta_workspace(n, len(counts), vh, d, st["longest"])), dtype=torch.uint8, device="cuda")
        return st
    heads, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "append":
        counts = _ints(case["tokens"])
        before = [case["before"] if i % 2 == 0 else case["before"] // 3 for i in range(len(counts))]
        cells = [b + c for b, c in zip(before, counts)]
        n = sum(counts)
        # the projection's output: q, k and v of a token side by side
        qkv = _normal(gen, n, (heads + 2 * kv) * d, dtype=kind)
        st["q"], st["k"], st["v"] = (x.unflatten(1, (-1, d)) for x in qkv.split([heads * d, kv * d, kv * d], dim=1))
        st["q_out"] = torch.empty(n, heads, d, dtype=kind, device="cuda")
        st["before"] = torch.tensor(before, dtype=torch.int32, device="cuda")
        st["starts"] = None if all(c == 1 for c in counts) else _starts(counts)
        st["after"] = torch.zeros(len(counts), dtype=torch.int32, device="cuda")
        half = case["rot"] // 2
        st["inv_freq"] = (1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)).float()
    else:
        cells = _ints(case["lengths"])
        st["q"] = _normal(gen, len(cells), heads, d, dtype=kind)
        st["lengths"] = torch.tensor(cells, dtype=torch.int32, device="cuda")
        st["out"] = torch.empty(len(cells), heads, d, dtype=kind, device="cuda")
        st["lse"] = torch.empty(len(cells), heads, dtype=torch.float32, device="cuda")
        st["scale"] = d ** -0.5
    st["table"], pages = _tables(gen, cells, page, 8)
    for x in ("k", "v"):
        if case["int8"]:
            st[x + "_pool"] = torch.randint(-127, 128, (pages, kv, page, d), generator=gen, device="cuda", dtype=torch.int8)
            st[x + "_scale"] = (torch.rand(pages, kv, page, d // GROUP, generator=gen, device="cuda") * 0.02 + 0.01).half()
        else:
            st[x + "_pool"] = _normal(gen, pages, kv, page, d, dtype=torch.float16)
            st[x + "_scale"] = None
    if own:     # the handle a program keeps for a layer of its cache, and the workspace of its stream
        skv = _skv()
        st["layer"] = skv.KvLayer(st["k_pool"], st["v_pool"], st["table"], k_scale=st["k_scale"], v_scale=st["v_scale"])
        if case["op"] == "attention":
            st["workspace"] = torch.zeros(skv.decode_attention_workspace(st["layer"], len(cells), heads), dtype=torch.uint8, device="cuda")
    return st


# ------------------------------------------------------------------------------------------------ the plain forms

def _dequant(codes, scale):
    return (codes.float().unflatten(-1, (-1, GROUP)) * scale.float().unsqueeze(-1)).flatten(-2)


def _cells(st, counts_before):
    """(sequence, cell) of every new token, packed."""
    starts = st["starts"]
    n = st["q"].shape[0]
    if starts is None:
        seq = torch.arange(n, device="cuda")
        return seq, counts_before.long()
    seq = torch.searchsorted(starts[1:].contiguous().long(), torch.arange(n, device="cuda"), right=True)
    return seq, counts_before.long()[seq] + torch.arange(n, device="cuda") - starts.long()[seq]


def _rotate(x, cell, inv_freq, rot, style):
    angle = cell.double()[:, None, None] * inv_freq.double()
    cos, sin = angle.cos().float(), angle.sin().float()
    x = x.float()
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if style == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
    p, q = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([p, q], -1) if style == "half" else torch.stack([p, q], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _quantize(x):
    x = x.unflatten(-1, (-1, GROUP))
    scale = (x.abs().amax(-1) / 127).half()
    step = scale.float().unsqueeze(-1)
    codes = torch.where(step > 0, (x / step).round().clamp(-127, 127), 0.0)
    return codes.to(torch.int8).flatten(-2), scale


def _plain_append(st):
    case = st["case"]
    seq, cell = _cells(st, st["before"])
    page = st["table"].long()[seq, cell // case["page"]]
    slot = cell % case["page"]
    turn = (cell, st["inv_freq"], case["rot"], case["style"])
    for x, rows in (("k", _rotate(st["k"], *turn)), ("v", st["v"].float())):
        if case["int8"]:
            st[x + "_pool"][page, :, slot], st[x + "_scale"][page, :, slot] = _quantize(rows)
        else:
            st[x + "_pool"][page, :, slot] = rows.half()
    st["q_out"].copy_(_rotate(st["q"], *turn))
    counts = 1 if st["starts"] is None else st["starts"][1:] - st["starts"][:-1]
    torch.add(st["before"], counts, out=st["after"])


def _plain_attention(st):
    case = st["case"]
    kv, d = case["kv_heads"], case["dim"]
    lengths = st["lengths"].long()
    longest = max(_ints(case["lengths"]))
    cell = torch.arange(longest, device="cuda")
    page, slot = st["table"].long()[:, cell // case["page"]], cell % case["page"]

    def rows(x):    # [sequence, kv head, cell, dim]
        if case["int8"]:
            got = _dequant(st[x + "_pool"][page, :, slot], st[x + "_scale"][page, :, slot])
        else:
            got = st[x + "_pool"][page, :, slot].float()
        return got.transpose(1, 2)

    q = st["q"].float().unflatten(1, (kv, -1)) * st["scale"]
    score = q @ rows("k").transpose(-1, -2)
    inside = (cell < lengths[:, None])[:, None, None]
    score = torch.where(inside, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.where(inside, torch.exp(score - top), 0.0)
    total = weight.sum(-1, keepdim=True)
    out = torch.where(total > 0, (weight @ rows("v")) / total, 0.0)
    st["out"].copy_(out.flatten(1, 2))
    st["lse"].copy_((top + total.log()).flatten(1))


def _padded(st):
    """q, k, v, g and beta of every sequence, [sequence, head, token, ...] in 32 bits, zeros behind its last token."""
    counts = torch.tensor(_ints(st["case"]["tokens"]), device="cuda")
    longest = -(-int(st["longest"]) // CHUNK) * CHUNK if st["longest"] > 1 else 1
    token = torch.arange(longest, device="cuda")
    first = torch.cumsum(counts, 0) - counts
    inside = token < counts[:, None]
    at = torch.where(inside, first[:, None] + token, 0)
    ratio = st["case"]["v_heads"] // st["case"]["k_heads"]

    def take(x):
        x = torch.where(inside.view(*inside.shape, *[1] * (x.dim() - 1)), x[at].float(), 0.0).transpose(1, 2)
        return x.repeat_interleave(ratio, 1) if x.dim() == 4 and x.shape[1] != st["case"]["v_heads"] else x

    return [take(st[x]) for x in ("q", "k", "v", "g", "beta")], inside, first[:, None] + token


def _plain_delta(st):
    """Chunk by chunk: within a chunk the corrected values solve a unit lower triangular system, whose inverse is the
    product of I + (-A)^(2^i); it is taken in 64 bits, as its terms cancel."""
    (q, k, v, g, beta), inside, at = _padded(st)
    step = min(CHUNK, q.shape[2])
    q, k, v, g, beta = (x.unflatten(2, (-1, step)) for x in (q * st["scale"], k, v, g, beta))
    total = g.double().cumsum(-1)
    lower = torch.ones(step, step, dtype=torch.bool, device="cuda").tril()
    decay = torch.where(lower, torch.exp(torch.where(lower, total[..., :, None] - total[..., None, :], 0.0)), 0.0)
    eye = torch.eye(step, dtype=torch.float64, device="cuda")
    power = -(beta[..., None].double() * (k.double() @ k.double().transpose(-1, -2)) * decay).tril(-1)
    inverse = eye + power
    for _ in range(max(0, step.bit_length() - 2)):
        power = power @ power
        inverse = inverse + inverse @ power
    inverse = inverse.float()
    mix = (q @ k.transpose(-1, -2)) * decay.float()
    into, rest, whole = total.exp().float(), (total[..., -1:] - total).exp().float(), total[..., -1].exp().float()
    state, outs = st["state"], []
    for c in range(q.shape[2]):
        held = into[:, :, c, :, None]
        value = inverse[:, :, c] @ (beta[:, :, c, :, None] * (v[:, :, c] - held * (k[:, :, c] @ state)))
        outs.append(held * (q[:, :, c] @ state) + mix[:, :, c] @ value)
        state = whole[:, :, c, None, None] * state + (k[:, :, c] * rest[:, :, c, :, None]).transpose(-1, -2) @ value
    st["state"].copy_(state)
    out = torch.cat(outs, 2).transpose(1, 2)
    st["out"][at[inside]] = out[inside].to(st["out"].dtype)


# ------------------------------------------------------------------------------------------------ one pass

def run(st):
    case = st["case"]
    if case["op"] == "append":
        if own:
            _skv().kv_append(st["layer"], st["k"], st["v"], st["before"], seq_starts=st["starts"], q=st["q"], q_out=st["q_out"],
                             inv_freq=st["inv_freq"], rope_style=case["style"], lengths_out=st["after"])
        else:
            _plain_append(st)
        pools = [st["k_pool"], st["v_pool"]]
        if case["int8"]:    # the values that the codes stand for
            pools = [_dequant(st[x + "_pool"], st[x + "_scale"]).half() for x in "kv"]
        return {"k": pools[0], "v": pools[1], "q": st["q_out"], "after": st["after"]}
    if case["op"] == "attention":
        if own:
            _skv().decode_attention(st["layer"], st["q"], st["lengths"], st["out"], scale=st["scale"], lse=st["lse"], workspace=st["workspace"])
        else:
            _plain_attention(st)
        return {"out": st["out"], "lse": st["lse"]}
    if own:
        _skv().gated_delta(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"], st["out"], seq_starts=st["starts"],
                           max_tokens=st["longest"], scale=st["scale"], workspace=st["workspace"])
    else:
        _plain_delta(st)
    return {"out": st["out"], "state": st["state"]}


# ------------------------------------------------------------------------------------------------ 64 bits

def _exact_append(case, st):
    counts, before = _ints(case["tokens"]), st["before"].tolist()
    page, rot = case["page"], case["rot"]
    pools = {}
    for x in "kv":
        pools[x] = st[x + "_pool"].double()
        if case["int8"]:
            pools[x] = pools[x] * st[x + "_scale"].double().repeat_interleave(GROUP, -1)
    first = [i if case["style"] == "half" else 2 * i for i in range(rot // 2)]
    second = [i + rot // 2 if case["style"] == "half" else 2 * i + 1 for i in range(rot // 2)]

    def turned(x, cell):
        z = torch.polar(torch.ones_like(cell, dtype=torch.float64)[:, None], torch.outer(cell.double(), st["inv_freq"].double()))[:, None]
        w = torch.complex(x[..., first], x[..., second]) * z
        y = x.clone()
        y[..., first], y[..., second] = w.real, w.imag
        return y

    q_out, at = torch.empty_like(st["q"], dtype=torch.float64), 0
    for s, n in enumerate(counts):
        cell = torch.arange(before[s], before[s] + n, device="cuda")
        rows = slice(at, at + n)
        at += n
        q_out[rows] = turned(st["q"][rows].double(), cell)
        for x in "kv":
            new = st[x][rows].double()
            new = turned(new, cell) if x == "k" else new
            if case["int8"]:
                grouped = new.reshape(n, case["kv_heads"], case["dim"] // GROUP, GROUP)
                step = (grouped.abs().amax(-1, keepdim=True) / 127).half().double()
                new = ((grouped / step).round().clamp(-127, 127) * step).reshape(new.shape)
            pools[x][st["table"][s].long()[cell // page], :, cell % page] = new
    after = torch.tensor([b + n for b, n in zip(before, counts)], dtype=torch.int32)
    return {"k": pools["k"], "v": pools["v"], "q": q_out, "after": after}


def _exact_attention(case, st):
    kv, d = case["kv_heads"], case["dim"]
    outs, lses = [], []
    for s, n in enumerate(_ints(case["lengths"])):
        if n == 0:
            outs.append(torch.zeros(case["heads"], d, dtype=torch.float64, device="cuda"))
            lses.append(torch.full((case["heads"],), -math.inf, dtype=torch.float64, device="cuda"))
            continue
        pages = st["table"][s, :-(-n // case["page"])].long()
        held = {}
        for x in "kv":
            rows = st[x + "_pool"][pages].double()
            if case["int8"]:
                rows = rows * st[x + "_scale"][pages].double().repeat_interleave(GROUP, -1)
            held[x] = rows.permute(1, 0, 2, 3).reshape(kv, -1, d)[:, :n].repeat_interleave(case["heads"] // kv, 0)
        score = torch.einsum("hd,hnd->hn", st["q"][s].double() * st["scale"], held["k"])
        lses.append(torch.logsumexp(score, -1))
        outs.append(torch.einsum("hn,hnd->hd", torch.softmax(score, -1), held["v"]))
    return {"out": torch.stack(outs), "lse": torch.stack(lses)}


def _exact_delta(case, st):
    """Token by token, all sequences that still have one at a time."""
    counts = _ints(case["tokens"])
    ratio = case["v_heads"] // case["k_heads"]
    starts = [sum(counts[:s]) for s in range(len(counts))]
    order = sorted(range(len(counts)), key=lambda s: -counts[s])    # the longest first: those left are a prefix
    state = st["state"].double()[order]
    q, k = (st[x].double().repeat_interleave(ratio, 1) for x in ("q", "k"))
    v, keep, beta = st["v"].double(), st["g"].double().exp(), st["beta"].double()
    q = q * st["scale"]
    out = torch.zeros_like(v)
    first = torch.tensor([starts[s] for s in order], device="cuda")
    left = len(order)
    for t in range(max(counts)):
        while counts[order[left - 1]] <= t:
            left -= 1
        at = first[:left] + t
        held = state[:left]
        held *= keep[at][..., None, None]
        key = k[at][..., None, :]
        wrong = (v[at][..., None, :] - key @ held) * beta[at][..., None, None]
        held += key.transpose(-1, -2) @ wrong
        out[at] = (q[at][..., None, :] @ held).squeeze(-2)
    final = torch.empty_like(state)
    final[order] = state
    return {"out": out, "state": final}


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "delta": _exact_delta}[case["op"]](case, st)

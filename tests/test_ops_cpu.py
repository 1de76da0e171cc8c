"""The operators' refusals and their binding, without a GPU: every bad call ends before anything reaches a device."""
import ctypes as C

import pytest

import skv

P = 0x10000     # a 256-byte aligned address that is never followed


def layer(**kw):
    base = dict(k_pool=P, v_pool=P, page_tables=P, table_stride=8, page_limit=64, n_tables=4, n_head_kv=2, head_dim=256,
                page_size=4, format=skv.KV_F16)
    return skv.KvLayerArgs(**{**base, **kw})


def append(**kw):
    base = dict(k=P, v=P, k_stride=512, v_stride=512, q=P, q_out=P, q_stride=6144, q_out_stride=6144, lengths=P, inv_freq=P,
                n_tokens=4, n_seqs=4, n_head=24, n_rot=64, rope_style=0, dtype=0, rope_scale=1.0)
    return skv.AppendArgs(**{**base, **kw})


def attention(**kw):
    base = dict(q=P, out=P, q_stride=6144, out_stride=6144, lengths=P, workspace=P, workspace_bytes=1 << 40, n_seqs=4,
                n_head=24, dtype=0, scale=0.0625)
    return skv.AttentionArgs(**{**base, **kw})


def delta(**kw):
    base = dict(q=P, k=P, v=P, out=P, q_stride=2048, k_stride=2048, v_stride=4096, out_stride=4096, g=P, beta=P, g_stride=32,
                beta_stride=32, state=P, state_stride=32 * 128 * 128, state_rows=4, workspace=P, workspace_bytes=1 << 40,
                n_tokens=4, n_seqs=4, n_k_heads=16, n_v_heads=32, head_dim=128, max_tokens=1, dtype=1, scale=0.1)
    return skv.GatedDeltaArgs(**{**base, **kw})


def refused(rc, text):
    assert rc == skv.EINVAL, (rc, skv.lib().skv_last_error())
    assert text in skv.lib().skv_last_error().decode()


BAD_LAYERS = [
    (dict(head_dim=96), "head_dim"), (dict(page_size=3), "page_size"), (dict(page_size=512), "page_size"), (dict(page_size=0), "page_size"),
    (dict(n_head_kv=0), "n_head_kv"), (dict(k_pool=None), "missing pool"), (dict(v_pool=None), "missing pool"),
    (dict(page_tables=None), "missing pool"), (dict(v_pool=P + 8), "16-byte"), (dict(format=2), "format"),
    (dict(format=skv.KV_INT8), "scales"), (dict(format=skv.KV_INT8, k_scale=P, v_scale=P + 4), "8-byte"),
    (dict(page_limit=0), "page_limit"), (dict(page_limit=1 << 31), "page_limit"), (dict(table_stride=0), "table_stride"),
    (dict(n_tables=3), "page tables"), (dict(page_tables=P + 2), "4-byte"),
]


@pytest.mark.parametrize("bad,text", BAD_LAYERS)
def test_a_layer_that_cannot_be_addressed_is_refused(bad, text):
    L = skv.lib()
    refused(L.skv_kv_append(C.byref(layer(**bad)), C.byref(append()), None), text)
    refused(L.skv_decode_attention(C.byref(layer(**bad)), C.byref(attention()), None), text)


@pytest.mark.parametrize("bad,text", [
    (dict(n_tokens=-1), "negative"), (dict(n_seqs=-1), "negative"), (dict(k=None), "missing"), (dict(v=None), "missing"),
    (dict(k=P + 2), "16-byte"), (dict(v_stride=516), "multiples of 8"), (dict(k_stride=256), "shorter"), (dict(lengths=None), "lengths"),
    (dict(n_tokens=5), "one row"), (dict(lengths_out=P), "lengths_out"), (dict(dtype=2), "dtype"), (dict(rope_style=2), "style"),
    (dict(n_rot=24), "n_rot"), (dict(n_rot=272), "n_rot"), (dict(n_rot=-16), "n_rot"), (dict(inv_freq=None), "inv_freq"),
    (dict(q=None), "together"), (dict(q_out=None), "together"), (dict(n_head=0), "n_head"), (dict(q_stride=4096), "shorter"),
    (dict(q_out=P + 4), "16-byte"), (dict(q_stride=8192), "in place"),
])
def test_append_refuses(bad, text):
    refused(skv.lib().skv_kv_append(C.byref(layer()), C.byref(append(**bad)), None), text)


@pytest.mark.parametrize("bad,text", [
    (dict(n_seqs=-1), "n_seqs"), (dict(n_head=0), "n_head"), (dict(n_head=25), "multiple"), (dict(dtype=7), "dtype"),
    (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(q=None), "missing"), (dict(out=None), "missing"),
    (dict(lengths=None), "missing"), (dict(q=P + 8), "16-byte"), (dict(out_stride=6148), "multiples of 8"),
    (dict(out_stride=2048), "shorter"), (dict(workspace=None), "workspace"), (dict(workspace=P + 16), "workspace"),
    (dict(workspace_bytes=0), "workspace"),
])
def test_attention_refuses(bad, text):
    refused(skv.lib().skv_decode_attention(C.byref(layer()), C.byref(attention(**bad)), None), text)


@pytest.mark.parametrize("bad,text", [
    (dict(n_tokens=-1), "negative"), (dict(head_dim=96), "head_dim"), (dict(n_k_heads=0), "multiple"), (dict(n_v_heads=24), "multiple"),
    (dict(dtype=2), "dtype"), (dict(scale=float("nan")), "finite"), (dict(n_tokens=3), "one token"), (dict(max_tokens=-1), "negative"),
    (dict(q=None), "missing"), (dict(state=None), "missing"), (dict(g=None), "missing"), (dict(v=P + 8), "16-byte"),
    (dict(state=P + 4), "16-byte"), (dict(out_stride=4100), "multiples"), (dict(state_stride=32 * 128 * 128 + 2), "multiples"),
    (dict(k_stride=1024), "shorter"), (dict(state_stride=128), "overlap"), (dict(state_rows=0), "none"), (dict(state_rows=3), "fewer"),
])
def test_delta_refuses(bad, text):
    refused(skv.lib().skv_gated_delta(C.byref(delta(**bad)), None), text)


@pytest.mark.parametrize("call,name", [(c, n) for c, names in (
    ("append", ("lengths", "lengths_out", "seq_starts", "inv_freq")), ("attention", ("lengths", "lse")),
    ("delta", ("g", "beta", "state_index", "seq_starts"))) for n in names])
@pytest.mark.parametrize("off", [1, 2])
def test_arrays_of_32_bits_off_their_alignment_are_refused(call, name, off):
    L, bad = skv.lib(), {name: P + 0x100 + off}
    if call == "append":
        refused(L.skv_kv_append(C.byref(layer()), C.byref(append(**bad)), None), "4-byte")
    elif call == "attention":
        refused(L.skv_decode_attention(C.byref(layer()), C.byref(attention(**bad)), None), "4-byte")
    else:
        refused(L.skv_gated_delta(C.byref(delta(**bad)), None), "4-byte")


def test_no_arguments_and_nothing_to_do():
    L = skv.lib()
    refused(L.skv_kv_append(None, C.byref(append()), None), "no layer")
    refused(L.skv_kv_append(C.byref(layer()), None, None), "no arguments")
    refused(L.skv_decode_attention(None, C.byref(attention()), None), "no layer")
    refused(L.skv_decode_attention(C.byref(layer()), None, None), "no arguments")
    refused(L.skv_gated_delta(None, None), "no arguments")
    assert L.skv_kv_append(C.byref(layer()), C.byref(append(n_seqs=0, n_tokens=0)), None) == skv.OK
    assert L.skv_decode_attention(C.byref(layer()), C.byref(attention(n_seqs=0)), None) == skv.OK
    assert L.skv_gated_delta(C.byref(delta(n_seqs=0, n_tokens=0)), None) == skv.OK
    assert L.skv_gated_delta(C.byref(delta(max_tokens=0)), None) == skv.OK


def test_workspace_sizes():
    L, out = skv.lib(), C.c_uint64(7)
    assert L.skv_decode_attention_workspace(C.byref(layer()), 4, 24, C.byref(out)) == skv.OK and out.value % 256 == 0
    refused(L.skv_decode_attention_workspace(C.byref(layer()), 4, 24, None), "null output")
    refused(L.skv_decode_attention_workspace(C.byref(layer()), 4, 0, C.byref(out)), "bad counts")
    assert L.skv_gated_delta_workspace(100, 3, 32, 128, 50, C.byref(out)) == skv.OK and out.value % 256 == 0
    refused(L.skv_gated_delta_workspace(100, 3, 32, 100, 50, C.byref(out)), "bad sizes")
    refused(L.skv_gated_delta_workspace(-1, 3, 32, 128, 50, C.byref(out)), "bad sizes")


@pytest.mark.parametrize("seqs,kv,heads,fits", [
    (1 << 16, 2, 24, True), (1 << 29, 2, 24, True), ((1 << 29) + 1, 2, 24, False), (1 << 28, 2, 34, True), ((1 << 28) + 1, 2, 34, False),
    (1 << 30, 1, 16, True), ((1 << 31) - 1, 1, 16, False), (1 << 30, 1, 17, False)])
def test_attention_and_its_workspace_take_the_same_number_of_sequences(seqs, kv, heads, fits):
    """Both refuse above 2^30 items (a sequence's K/V heads, in blocks of 16 query heads), and neither before: the
    call then gets as far as a refusal of its scale or of its workspace, the last ones on the host."""
    L, out, big = skv.lib(), C.c_uint64(), layer(n_tables=(1 << 31) - 1, n_head_kv=kv)
    rc = L.skv_decode_attention_workspace(C.byref(big), seqs, heads, C.byref(out))
    args = dict(n_seqs=seqs, n_head=heads, q_stride=heads * 256, out_stride=heads * 256, workspace_bytes=0)
    call = L.skv_decode_attention(C.byref(big), C.byref(attention(**args)), None)
    if fits:
        assert rc == skv.OK and out.value % 256 == 0
        refused(call, "workspace")
    else:
        assert (rc, call) == (skv.ERANGE, skv.ERANGE)
        assert "too many" in L.skv_last_error().decode()


@pytest.mark.parametrize("heads", [25, 4098])
def test_the_attention_workspace_refuses_the_heads_that_attention_refuses(heads):
    L, out = skv.lib(), C.c_uint64()
    refused(L.skv_decode_attention_workspace(C.byref(layer()), 4, heads, C.byref(out)), "multiple")
    refused(L.skv_decode_attention(C.byref(layer()), C.byref(attention(n_head=heads, q_stride=1 << 21, out_stride=1 << 21)), None), "multiple")


def test_the_binding_refuses_tensors_that_want_a_gradient():
    """There is no backward pass; where no gradient is recorded such a tensor is as good as any."""
    torch = pytest.importorskip("torch")
    x, vector = (torch.zeros(*shape, dtype=dt, requires_grad=True) for shape, dt in (((1, 2, 256), torch.float16), ((8,), torch.float32)))
    pool, table = torch.zeros(8, 2, 4, 256, dtype=torch.float16, requires_grad=True), torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(TypeError, match="q: requires a gradient"):
        skv._rows(x, "q", 0)
    with pytest.raises(TypeError, match="inv_freq: requires a gradient"):
        skv._vector(vector, "inv_freq", -1, "torch.float32", 0)
    with pytest.raises(TypeError, match="requires a gradient"):
        skv.KvLayer(pool, pool, table)
    with torch.no_grad():
        assert skv._vector(vector, "inv_freq", -1, "torch.float32", 0) == vector.data_ptr()
        with pytest.raises(ValueError, match="not on the GPU"):
            skv._rows(x, "q", 0)
        with pytest.raises(ValueError, match="on the GPU"):
            skv.KvLayer(pool, pool, table)


def test_the_binding_takes_what_has_a_tensors_methods():
    """Without a requires_grad of its own, too: it gets as far as the look at its device."""
    torch = pytest.importorskip("torch")

    class Like:
        def __init__(self, x):
            self.x = x

        def __getattr__(self, name):
            if name == "requires_grad":
                raise AttributeError(name)
            return getattr(self.x, name)

    with pytest.raises(ValueError, match="not on the GPU"):
        skv._rows(Like(torch.zeros(1, 2, 256, dtype=torch.float16)), "q", 0)
    assert skv._vector(Like(torch.zeros(4, dtype=torch.int32)), "lengths", -1, "torch.int32", 4)


def test_the_binding_refuses_tensors_that_do_not_fit():
    """CPU tensors, wrong types, shapes and layouts never reach the library."""
    torch = pytest.importorskip("torch")
    pool = torch.zeros(8, 2, 4, 256, dtype=torch.float16)
    table = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="on the GPU"):
        skv.KvLayer(pool, pool.clone(), table)
    with pytest.raises(TypeError, match="float16 or two int8"):
        skv.KvLayer(pool.float(), pool.float(), table)
    with pytest.raises(ValueError, match="scales"):
        skv.KvLayer(pool.to(torch.int8), pool.to(torch.int8), table)
    x = torch.zeros(1, 2, 256, dtype=torch.float16)
    with pytest.raises(ValueError, match="not on the GPU"):
        skv._rows(x, "q", 0)
    with pytest.raises(ValueError, match="not on the GPU"):
        skv._rows(x, "q", -1)          # a layer's or a first tensor's own place, when that is no GPU
    with pytest.raises(TypeError, match="float16"):
        skv._rows(x.float(), "q", 0)
    with pytest.raises(TypeError, match="all"):
        skv._rows(x, "q", 0, torch.bfloat16)
    with pytest.raises(ValueError, match="back to back"):
        skv._rows(x.transpose(1, 2), "q", 0)
    with pytest.raises(TypeError, match="int32"):
        skv._vector(torch.zeros(3), "lengths", 0, "torch.int32", 3)
    with pytest.raises(TypeError, match="workspace"):
        skv._room(torch.zeros(3), 0)
    with pytest.raises(ValueError, match="not on the GPU"):
        skv.gated_delta(x, x, x, torch.zeros(1, 2), torch.zeros(1, 2), torch.zeros(1, 2, 256, 256), x)

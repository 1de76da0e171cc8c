"""skv.py - Python bindings of libstrata_kv.so (the B200 KV handoff / park-resume C ABI, include/strata_kv.h).

This is the host mirror the tests and bench.py drive.  It is plumbing over the C ABI: every byte is moved and computed by
the sm_100a kernels in csrc/.  There is no Python or CPU fallback: if the library is missing the
import of any entry point raises.

Layout of a sequence's cache in a block pool (one pool per GPU):
    slot s (block_bytes = 2 * pages_per_block * page_bytes) = [K pages 0..63][V pages 0..63] of ONE layer's
    256-token block; a page is the reference's [kv_head][page_size=4][head_dim] fp16 run
    (include/strata/kernels/qsa.hpp:178).  Layer l's logical page p of K lives at pool page
    table_l[p // 64] * 128 + p % 64 and of V at table_l[p // 64] * 128 + 64 + p % 64, which is the reference's
    QsaState::page_table format (include/strata/core/layer.hpp:220) over k_pool = pool base,
    v_pool = pool base + 64 pages.
"""
from __future__ import annotations

import ctypes as C
import os
import struct
from dataclasses import dataclass

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libstrata_kv.so")

OK, EINVAL, ECUDA, ENOMEM, ETIMEOUT, EDEVICE, ERANGE = range(7)
STATUS_BAD_SRC_PAGE, STATUS_BAD_DST_PAGE, STATUS_WAIT_TIMEOUT, STATUS_BAD_STATE_ROW = 0x1, 0x2, 0x4, 0x8
COPY_AUTO, COPY_TMA, COPY_VEC = 0, 1, 2
PARK_DIRECT, PARK_STAGED = 1, 2
MAX_SEGMENTS = 64
NOALLOC_MAX_SEGMENTS = 512

DTYPE_F16, DTYPE_BF16 = 0, 1
KV_F16, KV_INT8 = 0, 1
ROPE_STYLES = {"half": 0, "pairs": 1}

PAGE_CELLS = 4
BLOCK_TOKENS = 256


class SkvError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"strata_kv error {code}: {message}")
        self.code = code


class Segment(C.Structure):
    _fields_ = [("src", C.c_void_p), ("dst", C.c_void_p), ("src_pages", C.c_void_p), ("dst_pages", C.c_void_p),
                ("bytes", C.c_uint64), ("page_bytes", C.c_uint32), ("reserved", C.c_uint32),
                ("src_page_limit", C.c_int64), ("dst_page_limit", C.c_int64)]


class SchedRun(C.Structure):
    """skv_sched_run: one transfer of a many-to-many hand-off batch (skv_schedule_phases)."""
    _fields_ = [("phase", C.c_int32), ("src", C.c_int32), ("lo", C.c_uint64), ("hi", C.c_uint64),
                ("wait", C.c_int32), ("signal_dst", C.c_int32), ("signal_idx", C.c_int32), ("reserved", C.c_int32)]


class KvLayerArgs(C.Structure):
    """skv_kv_layer."""
    _fields_ = [("k_pool", C.c_void_p), ("v_pool", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("page_tables", C.c_void_p), ("table_stride", C.c_int64), ("page_limit", C.c_int64),
                ("n_tables", C.c_int32), ("n_head_kv", C.c_int32), ("head_dim", C.c_int32), ("page_size", C.c_int32),
                ("format", C.c_int32), ("reserved", C.c_int32)]


class AppendArgs(C.Structure):
    """skv_append_args."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_stride", C.c_int64), ("v_stride", C.c_int64),
                ("q", C.c_void_p), ("q_out", C.c_void_p), ("q_stride", C.c_int64), ("q_out_stride", C.c_int64),
                ("seq_starts", C.c_void_p), ("lengths", C.c_void_p), ("lengths_out", C.c_void_p), ("inv_freq", C.c_void_p),
                ("n_tokens", C.c_int32), ("n_seqs", C.c_int32), ("n_head", C.c_int32), ("n_rot", C.c_int32),
                ("rope_style", C.c_int32), ("dtype", C.c_int32), ("rope_scale", C.c_float), ("reserved", C.c_int32)]


class AttentionArgs(C.Structure):
    """skv_attention_args."""
    _fields_ = [("q", C.c_void_p), ("out", C.c_void_p), ("q_stride", C.c_int64), ("out_stride", C.c_int64),
                ("lse", C.c_void_p), ("lengths", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64),
                ("n_seqs", C.c_int32), ("n_head", C.c_int32), ("dtype", C.c_int32), ("scale", C.c_float)]


class GatedDeltaArgs(C.Structure):
    """skv_gdn_args."""
    _fields_ = [("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("out", C.c_void_p),
                ("q_stride", C.c_int64), ("k_stride", C.c_int64), ("v_stride", C.c_int64), ("out_stride", C.c_int64),
                ("g", C.c_void_p), ("beta", C.c_void_p), ("g_stride", C.c_int64), ("beta_stride", C.c_int64),
                ("state", C.c_void_p), ("state_stride", C.c_int64), ("state_rows", C.c_int64),
                ("state_index", C.c_void_p), ("seq_starts", C.c_void_p), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_uint64), ("n_tokens", C.c_int32), ("n_seqs", C.c_int32),
                ("n_k_heads", C.c_int32), ("n_v_heads", C.c_int32), ("head_dim", C.c_int32), ("max_tokens", C.c_int32),
                ("dtype", C.c_int32), ("scale", C.c_float)]


_lib = None

_SIGNATURES = {
    "skv_last_error": ([], C.c_char_p),
    "skv_version": ([], C.c_int),
    "skv_pool_create": ([C.c_int, C.c_int64, C.c_uint64, C.POINTER(C.c_void_p)], C.c_int),
    "skv_pool_wrap": ([C.c_int, C.c_void_p, C.c_int64, C.c_uint64, C.POINTER(C.c_void_p)], C.c_int),
    "skv_pool_destroy": ([C.c_void_p], C.c_int),
    "skv_pool_base": ([C.c_void_p], C.c_void_p),
    "skv_pool_block_bytes": ([C.c_void_p], C.c_uint64),
    "skv_pool_blocks": ([C.c_void_p], C.c_int64),
    "skv_pool_device": ([C.c_void_p], C.c_int),
    "skv_alloc_blocks": ([C.c_void_p, C.c_int64, C.c_void_p], C.c_int),
    "skv_free_blocks": ([C.c_void_p, C.c_void_p, C.c_int64], C.c_int),
    "skv_pool_free_count": ([C.c_void_p], C.c_int64),
    "skv_pool_scramble": ([C.c_void_p, C.c_uint64], C.c_int),
    "skv_expand_block_table": ([C.c_void_p, C.c_int64, C.c_int64, C.c_int64, C.c_int64, C.c_void_p], C.c_int),
    "skv_copy": ([C.c_void_p, C.c_int, C.c_int, C.c_void_p], C.c_int),
    "skv_copy_noalloc": ([C.c_void_p, C.c_int, C.c_void_p, C.c_void_p], C.c_int),
    "skv_copy_gated": ([C.c_void_p, C.c_int, C.c_void_p, C.c_uint64, C.c_uint64, C.c_void_p, C.c_uint64, C.c_void_p],
                       C.c_int),
    "skv_copy_chained": ([C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_uint64, C.c_uint64, C.c_void_p], C.c_int),
    "skv_set_copy_tuning": ([C.c_int, C.c_uint32, C.c_int, C.c_int], C.c_int),
    "skv_get_copy_tuning": ([C.POINTER(C.c_int), C.POINTER(C.c_uint32), C.POINTER(C.c_int), C.POINTER(C.c_int)], C.c_int),
    "skv_query_status": ([C.c_int, C.c_void_p, C.POINTER(C.c_uint32)], C.c_int),
    "skv_clear_status": ([C.c_int, C.c_void_p], C.c_int),
    "skv_device_initialized": ([C.c_int], C.c_int),
    "skv_host_alloc": ([C.c_uint64, C.POINTER(C.c_void_p)], C.c_int),
    "skv_host_free": ([C.c_void_p], C.c_int),
    "skv_host_register": ([C.c_void_p, C.c_uint64], C.c_int),
    "skv_host_unregister": ([C.c_void_p], C.c_int),
    "skv_park": ([C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_uint64, C.c_void_p], C.c_int),
    "skv_resume": ([C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_uint64, C.c_void_p], C.c_int),
    "skv_enable_peer": ([C.c_int, C.c_int], C.c_int),
    "skv_ipc_export": ([C.c_void_p, C.c_void_p], C.c_int),
    "skv_ipc_import": ([C.c_int, C.c_void_p, C.POINTER(C.c_void_p)], C.c_int),
    "skv_ipc_close": ([C.c_void_p], C.c_int),
    "skv_signal": ([C.c_void_p, C.c_uint64, C.c_void_p], C.c_int),
    "skv_wait_flag": ([C.c_void_p, C.c_uint64, C.c_uint64, C.c_void_p], C.c_int),
    "skv_schedule_phases": ([C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_int, C.c_void_p, C.POINTER(C.c_uint64),
                             C.POINTER(C.c_int)], C.c_int),
    "skv_slice_segments": ([C.c_void_p, C.c_int, C.c_uint64, C.c_uint64, C.c_void_p, C.c_int, C.POINTER(C.c_int)],
                           C.c_int),
    "skv_kv_append": ([C.c_void_p, C.c_void_p, C.c_void_p], C.c_int),
    "skv_decode_attention": ([C.c_void_p, C.c_void_p, C.c_void_p], C.c_int),
    "skv_decode_attention_workspace": ([C.c_void_p, C.c_int, C.c_int, C.POINTER(C.c_uint64)], C.c_int),
    "skv_gated_delta": ([C.c_void_p, C.c_void_p], C.c_int),
    "skv_gated_delta_workspace": ([C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(C.c_uint64)], C.c_int),
}


def exported_names() -> list:
    return sorted(_SIGNATURES)


def lib() -> C.CDLL:
    """The loaded C ABI.  Raises (never falls back) when the CUDA library was not built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `python strata-concurrent_b200/build.py` "
                               "(there is no CPU fallback)")
        L = C.CDLL(LIB_PATH)
        for name, (args, res) in _SIGNATURES.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = res
        _lib = L
    return _lib


def check(rc: int) -> None:
    if rc:
        raise SkvError(rc, lib().skv_last_error().decode())


def _ptr(x) -> int | None:
    """A raw address from an int, a torch tensor, a numpy array or None."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    if isinstance(x, np.ndarray):
        return x.ctypes.data
    raise TypeError(f"cannot take the address of {type(x)}")


def _stream(stream) -> int | None:
    if stream is None:
        return None
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


# ------------------------------------------------------------------------------------------------ segments

def segment(src, dst, nbytes: int, *, src_pages=None, dst_pages=None, page_bytes: int = 0,
            src_page_limit: int = 0, dst_page_limit: int = 0) -> Segment:
    return Segment(_ptr(src), _ptr(dst), _ptr(src_pages), _ptr(dst_pages), int(nbytes), int(page_bytes), 0,
                   int(src_page_limit), int(dst_page_limit))


def _segment_unit(seg: Segment) -> int:
    """The granule a segment is cut on: a whole page when either side is paged, else 16 bytes."""
    unit = seg.page_bytes if (seg.src_pages or seg.dst_pages) else 16
    if unit <= 0 or seg.bytes % unit:
        raise ValueError("a segment splits on whole pages (paged) or 16-byte units (contiguous)")
    return unit


def slice_segment(seg: Segment, start: int, end: int) -> Segment:
    """Bytes [start, end) of one segment as a segment of its own; both ends must lie on the segment's granule
    (a whole page when a side is paged, 16 bytes otherwise)."""
    unit = _segment_unit(seg)
    if start % unit or end % unit or not 0 <= start < end <= seg.bytes:
        raise ValueError(f"slice [{start}, {end}) of a {seg.bytes}-byte segment is not on {unit}-byte granules")
    first_page = start // unit if (seg.src_pages or seg.dst_pages) else 0
    return Segment(
        seg.src if seg.src_pages else (seg.src or 0) + start,
        seg.dst if seg.dst_pages else (seg.dst or 0) + start,
        seg.src_pages + 4 * first_page if seg.src_pages else None,
        seg.dst_pages + 4 * first_page if seg.dst_pages else None,
        end - start, seg.page_bytes, 0, seg.src_page_limit, seg.dst_page_limit)


def split_segment(seg: Segment, max_bytes: int) -> list:
    """Cut one segment into pieces of at most `max_bytes` (whole pages for a paged side, 16-byte multiples for a
    contiguous one), in order: the pieces move exactly the bytes of the whole.  Used to pipeline a long copy
    chunk by chunk (a relay or a chained fan-out signals each piece as it lands)."""
    unit = _segment_unit(seg)
    per = max(1, max_bytes // unit) * unit
    return [slice_segment(seg, at, min(at + per, seg.bytes)) for at in range(0, seg.bytes, per)]


def slice_segments(segs: list, start: int, end: int) -> list:
    """Bytes [start, end) of a list of segments taken as one stream, in order.  A cut that falls inside a segment
    is rounded down to that segment's granule, so adjacent slices [a, b) and [b, c) always tile the stream
    exactly."""
    out, at = [], 0
    for seg in segs:
        lo, hi = max(start, at), min(end, at + seg.bytes)
        if lo < hi:
            unit = _segment_unit(seg)
            a = (lo - at) // unit * unit
            b = seg.bytes if hi == at + seg.bytes else (hi - at) // unit * unit
            if a < b:
                out.append(slice_segment(seg, a, b))
        at += seg.bytes
    return out


def copy(segs: list, engine: int = COPY_AUTO, stream=None) -> None:
    """ONE kernel launch moving every segment (gather, scatter, pool->pool, state rows, P2P, host)."""
    for i in range(0, max(len(segs), 1), MAX_SEGMENTS):
        chunk = segs[i:i + MAX_SEGMENTS]
        arr = (Segment * len(chunk))(*chunk)
        check(lib().skv_copy(arr, len(chunk), engine, _stream(stream)))


def copy_chained(segs: list, wait_flags=None, signal_flags=None, value: int = 1, timeout_ns: int = 0,
                 stream=None) -> None:
    """One TMA launch moving `segs` as a pipeline of chunks (segment c = chunk c): chunk c waits for
    wait_flags[c] >= value and, once landed, stores value to signal_flags[c] (flag arrays of 8-byte words)."""
    arr = (Segment * len(segs))(*segs)
    check(lib().skv_copy_chained(arr, len(segs), _ptr(wait_flags), _ptr(signal_flags), int(value), int(timeout_ns),
                                 _stream(stream)))


def copy_gated(segs: list, wait_flag=None, wait_value: int = 0, done_flag=None, done_value: int = 0,
               timeout_ns: int = 0, stream=None) -> None:
    """ONE TMA launch moving `segs` that first waits for *wait_flag >= wait_value and, once everything landed,
    releases done_value into *done_flag (either flag may be None)."""
    arr = (Segment * len(segs))(*segs)
    check(lib().skv_copy_gated(arr, len(segs), _ptr(wait_flag), int(wait_value), int(timeout_ns), _ptr(done_flag),
                               int(done_value), _stream(stream)))


def set_copy_tuning(tma_stages: int, tma_tile_bytes: int, tma_ctas_per_sm: int, vec_ctas_per_sm: int) -> None:
    check(lib().skv_set_copy_tuning(tma_stages, tma_tile_bytes, tma_ctas_per_sm, vec_ctas_per_sm))


def get_copy_tuning() -> tuple:
    a, b, c, d = C.c_int(), C.c_uint32(), C.c_int(), C.c_int()
    check(lib().skv_get_copy_tuning(C.byref(a), C.byref(b), C.byref(c), C.byref(d)))
    return a.value, b.value, c.value, d.value


def query_status(device: int, stream=None) -> int:
    out = C.c_uint32()
    check(lib().skv_query_status(device, _stream(stream), C.byref(out)))
    return out.value


def clear_status(device: int, stream=None) -> None:
    check(lib().skv_clear_status(device, _stream(stream)))


def park(segs: list, mode: int, staging=None, staging_bytes: int = 0, stream=None) -> None:
    arr = (Segment * len(segs))(*segs)
    check(lib().skv_park(arr, len(segs), mode, _ptr(staging), staging_bytes, _stream(stream)))


def resume(segs: list, mode: int, staging=None, staging_bytes: int = 0, stream=None) -> None:
    arr = (Segment * len(segs))(*segs)
    check(lib().skv_resume(arr, len(segs), mode, _ptr(staging), staging_bytes, _stream(stream)))


class SharedHostBuffer:
    """Pinned, device-mapped memory shared by the processes of one node: an anonymous shared-memory file (memfd)
    that the creator sizes and every user maps and registers with CUDA (skv_host_register).  `handle()` gives what
    another process needs to map the same pages: (pid, fd)."""

    def __init__(self, nbytes: int, handle: tuple | None = None):
        import mmap
        import os
        if handle is None:
            self.fd = os.memfd_create("skv-shared-host", 0)
            os.ftruncate(self.fd, nbytes)
        else:
            pid, fd = handle
            self.fd = os.open(f"/proc/{pid}/fd/{fd}", os.O_RDWR)
        self.nbytes = nbytes
        self.map = mmap.mmap(self.fd, nbytes, mmap.MAP_SHARED, mmap.PROT_READ | mmap.PROT_WRITE)
        self.ptr = C.addressof(C.c_char.from_buffer(self.map))
        check(lib().skv_host_register(self.ptr, nbytes))

    def handle(self) -> tuple:
        import os
        return (os.getpid(), self.fd)

    def close(self) -> None:
        import os
        if self.map is not None:
            check(lib().skv_host_unregister(self.ptr))
            self.ptr = 0
            self.map.close()
            os.close(self.fd)
            self.map = None


def ipc_export(dev_ptr: int) -> bytes:
    """The 64-byte CUDA IPC handle of a cudaMalloc'd allocation (its base address)."""
    h = (C.c_uint8 * 64)()
    check(lib().skv_ipc_export(dev_ptr, C.cast(h, C.c_void_p)))
    return bytes(h)


def ipc_import(device: int, handle: bytes) -> int:
    """Open a peer process's allocation on `device`; returns the mapped base address."""
    h = (C.c_uint8 * 64).from_buffer_copy(handle)
    out = C.c_void_p()
    check(lib().skv_ipc_import(device, C.cast(h, C.c_void_p), C.byref(out)))
    return out.value


def ipc_close(ptr: int) -> None:
    check(lib().skv_ipc_close(ptr))


def signal(flag: int, value: int, stream=None) -> None:
    check(lib().skv_signal(flag, value, _stream(stream)))


def wait_flag(flag: int, value: int, timeout_ns: int, stream=None) -> None:
    check(lib().skv_wait_flag(flag, value, timeout_ns, _stream(stream)))


class HostBuffer:
    """Pinned, device-mapped host memory (skv_host_alloc) with a numpy view."""

    def __init__(self, nbytes: int):
        p = C.c_void_p()
        check(lib().skv_host_alloc(nbytes, C.byref(p)))
        self.ptr = p.value or 0
        self.nbytes = nbytes
        self.array = (np.ctypeslib.as_array((C.c_uint8 * nbytes).from_address(self.ptr)) if nbytes
                      else np.zeros(0, dtype=np.uint8))

    def close(self) -> None:
        if self.ptr:
            check(lib().skv_host_free(self.ptr))
            self.ptr = 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ------------------------------------------------------------------------------------------------ the block pool

class Pool:
    """A KV block pool (skv_pool_*).  `memory` may be a caller-owned device tensor (wrapped, not freed here)."""

    def __init__(self, device: int, n_blocks: int, block_bytes: int, memory=None):
        h = C.c_void_p()
        if memory is None:
            check(lib().skv_pool_create(device, n_blocks, block_bytes, C.byref(h)))
        else:
            check(lib().skv_pool_wrap(device, _ptr(memory), n_blocks, block_bytes, C.byref(h)))
        self.handle = h.value
        self.memory = memory
        self.device = device
        self.n_blocks = n_blocks
        self.block_bytes = block_bytes

    @property
    def base(self) -> int:
        return lib().skv_pool_base(self.handle)

    def alloc(self, n: int) -> np.ndarray:
        out = np.empty(n, dtype=np.int32)
        check(lib().skv_alloc_blocks(self.handle, n, out.ctypes.data))
        return out

    def free(self, ids) -> None:
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        check(lib().skv_free_blocks(self.handle, ids.ctypes.data, len(ids)))

    def free_count(self) -> int:
        return int(lib().skv_pool_free_count(self.handle))

    def scramble(self, seed: int) -> None:
        check(lib().skv_pool_scramble(self.handle, seed))

    def close(self) -> None:
        if self.handle:
            check(lib().skv_pool_destroy(self.handle))
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def expand_block_table(blocks, pages_per_block: int, slot_pages: int, page_offset: int) -> np.ndarray:
    blocks = np.ascontiguousarray(blocks, dtype=np.int32)
    out = np.empty(len(blocks) * pages_per_block, dtype=np.int32)
    check(lib().skv_expand_block_table(blocks.ctypes.data, len(blocks), pages_per_block, slot_pages, page_offset,
                                       out.ctypes.data))
    return out


# ------------------------------------------------------------------------------------------------ handoff plans

@dataclass
class KvGeometry:
    """The shape facts of the moved cache (include/strata/core/layout.hpp:27-60 at the configs' values)."""
    n_layers: int = 48
    qsa_interval: int = 4
    n_head_kv: int = 2
    head_dim: int = 256
    ssm_state_size: int = 128
    ssm_v_heads: int = 32
    ssm_d_conv: int = 4
    ssm_conv_channels: int = 8192

    @property
    def n_qsa(self) -> int:
        return self.n_layers // self.qsa_interval

    @property
    def n_gdn(self) -> int:
        return self.n_layers - self.n_qsa

    @property
    def page_bytes(self) -> int:
        return self.n_head_kv * PAGE_CELLS * self.head_dim * 2

    @property
    def pages_per_block(self) -> int:
        return BLOCK_TOKENS // PAGE_CELLS

    @property
    def slot_pages(self) -> int:
        return 2 * self.pages_per_block

    @property
    def block_bytes(self) -> int:
        return self.slot_pages * self.page_bytes

    @property
    def gdn_bytes(self) -> int:
        s = self.ssm_state_size
        return self.n_gdn * (s * self.ssm_v_heads * s + self.ssm_conv_channels * (self.ssm_d_conv - 1)) * 4

    def pages(self, tokens: int) -> int:
        return (tokens + PAGE_CELLS - 1) // PAGE_CELLS

    def blocks(self, tokens: int) -> int:
        return (tokens + BLOCK_TOKENS - 1) // BLOCK_TOKENS

    def metric_bytes(self, tokens: int) -> int:
        return 2 * self.n_qsa * self.pages(tokens) * self.page_bytes + self.gdn_bytes + 4 * tokens


def layer_page_tables(g: KvGeometry, blocks) -> tuple:
    """(K table, V table) in pool pages for one layer's block list."""
    k = expand_block_table(blocks, g.pages_per_block, g.slot_pages, 0)
    v = expand_block_table(blocks, g.pages_per_block, g.slot_pages, g.pages_per_block)
    return k, v


class PooledSequence:
    """One sequence resident on a GPU: per-layer block tables into `pool` (device page tables in `tables`,
    an int32 device tensor [n_layers_moved, 2, pages_per_seq]), plus its GDN state rows and its token ids.
    `tables`, `gdn` and `ids` are caller-owned device buffers (any object with data_ptr(), or ints)."""

    def __init__(self, g: KvGeometry, pool: Pool, tokens: int, layers: int, blocks: np.ndarray, tables, gdn, ids):
        self.g, self.pool, self.tokens, self.layers = g, pool, tokens, layers
        self.blocks = blocks            # host copy of the block table, (layers, n_blocks) int32
        self.tables = tables
        self.gdn, self.ids = gdn, ids

    @staticmethod
    def host_tables(g: KvGeometry, blocks: np.ndarray) -> np.ndarray:
        layers, nb = blocks.shape
        out = np.empty((layers, 2, nb * g.pages_per_block), dtype=np.int32)
        for layer in range(layers):
            out[layer, 0], out[layer, 1] = layer_page_tables(g, blocks[layer])
        return out

    def table_ptr(self, layer: int, kv: int) -> int:
        per = self.g.blocks(self.tokens) * self.g.pages_per_block
        return _ptr(self.tables) + ((layer * 2 + kv) * per) * 4

    @property
    def pool_pages(self) -> int:
        return self.pool.n_blocks * self.g.slot_pages


def kv_segments_pool_to_pool(src: PooledSequence, dst: PooledSequence, dst_base=None) -> list:
    """K and V of every moved layer, source pool pages -> destination pool pages (one segment each).
    `dst_base` overrides the destination pool address (a peer mapping of the decode GPU's pool)."""
    g = src.g
    n = g.pages(src.tokens) * g.page_bytes
    base = dst.pool.base if dst_base is None else dst_base
    segs = []
    for layer in range(src.layers):
        for kv in (0, 1):
            segs.append(segment(src.pool.base, base, n, src_pages=src.table_ptr(layer, kv),
                                dst_pages=dst.table_ptr(layer, kv), page_bytes=g.page_bytes,
                                src_page_limit=src.pool_pages, dst_page_limit=dst.pool_pages))
    return segs


def state_segments(src: PooledSequence, dst_gdn, dst_ids) -> list:
    """The running state that travels with the cache: the GDN recurrent + conv rows and the token ids."""
    return [segment(src.gdn, dst_gdn, src.g.gdn_bytes), segment(src.ids, dst_ids, 16 * ((4 * src.tokens + 15) // 16))]


def image_offsets(g: KvGeometry, tokens: int, layers: int) -> dict:
    """The contiguous packed image (what a park writes): per layer K then V, then the GDN rows, then the ids,
    each 256-byte aligned."""
    n = g.pages(tokens) * g.page_bytes
    off, at = {}, 0
    for layer in range(layers):
        for kv in (0, 1):
            off[(layer, kv)] = at
            at += (n + 255) & ~255
    off["gdn"] = at
    at += (g.gdn_bytes + 255) & ~255
    off["ids"] = at
    at += (4 * tokens + 255) & ~255
    off["total"] = at
    return off


def pack_segments(src: PooledSequence, image) -> list:
    """Pool -> contiguous image (gather / pack, the B200 conversation_kv_save)."""
    g, t = src.g, src.tokens
    off = image_offsets(g, t, src.layers)
    base = _ptr(image)
    n = g.pages(t) * g.page_bytes
    segs = [segment(src.pool.base, base + off[(layer, kv)], n, src_pages=src.table_ptr(layer, kv),
                    page_bytes=g.page_bytes, src_page_limit=src.pool_pages)
            for layer in range(src.layers) for kv in (0, 1)]
    segs.append(segment(src.gdn, base + off["gdn"], g.gdn_bytes))
    segs.append(segment(src.ids, base + off["ids"], 16 * ((4 * t + 15) // 16)))
    return segs


def unpack_segments(image, dst: PooledSequence) -> list:
    """Contiguous image -> pool (scatter / unpack, the B200 conversation_kv_restore)."""
    g, t = dst.g, dst.tokens
    off = image_offsets(g, t, dst.layers)
    base = _ptr(image)
    n = g.pages(t) * g.page_bytes
    segs = [segment(base + off[(layer, kv)], dst.pool.base, n, dst_pages=dst.table_ptr(layer, kv),
                    page_bytes=g.page_bytes, dst_page_limit=dst.pool_pages)
            for layer in range(dst.layers) for kv in (0, 1)]
    segs.append(segment(base + off["gdn"], dst.gdn, g.gdn_bytes))
    segs.append(segment(base + off["ids"], dst.ids, 16 * ((4 * t + 15) // 16)))
    return segs


# ------------------------------------------------------------------------------------------------ operators
# On device tensors (torch's, or anything with its data_ptr, shape, stride, dtype and device).  They run on the current
# device and, like the copies, on `stream` (None: the legacy default stream).  They have no backward pass: a tensor that
# requires a gradient is refused while gradients are recorded (torch.no_grad, or detach(), says that none is wanted).

_CODES = {"torch.float16": DTYPE_F16, "torch.bfloat16": DTYPE_BF16}
_KNOWN = {}     # dtype object -> (its name, its code or None), so that a call formats no text

# The argument structures as the library reads them, packed: a third of the time of filling a ctypes structure.
_APPEND = struct.Struct("@PPqqPPqqPPPPiiiiiifi")
_ATTENTION = struct.Struct("@PPqqPPPQiiif")
_DELTA = struct.Struct("@PPPPqqqqPPqqPqqPPPQiiiiiiif")
assert (_APPEND.size, _ATTENTION.size, _DELTA.size) == tuple(C.sizeof(x) for x in (AppendArgs, AttentionArgs, GatedDeltaArgs))


def _dtype(x) -> tuple:
    got = _KNOWN.get(x.dtype)
    if got is None:
        name = str(x.dtype)
        got = _KNOWN[x.dtype] = (name, _CODES.get(name))
    return got


def _no_gradient(what: str) -> None:
    """Called for a tensor that requires a gradient."""
    import torch
    if torch.is_grad_enabled():
        raise TypeError(f"{what}: requires a gradient, and the operators have no backward pass (detach it, or use torch.no_grad)")


def _rows(x, what: str, device: int, kind=None) -> tuple:
    """(address, rows, heads, values, elements between rows) of a [row][head][value] tensor on GPU `device`, of dtype `kind`
    (None: a float16 or bfloat16 one), whose heads lie back to back."""
    if getattr(x, "requires_grad", False):
        _no_gradient(what)
    n, heads, dim = x.shape
    if x.is_contiguous():
        step = heads * dim
    else:
        step, between, one = x.stride()
        if (between != dim and heads > 1) or (one != 1 and dim > 1):
            raise ValueError(f"{what}: the heads of a row must lie back to back")
        if n <= 1:
            step = heads * dim
    if (x.dtype is not kind) if kind is not None else _dtype(x)[1] is None:
        raise TypeError(f"{what}: {x.dtype} (all of a call's activations are float16, or all bfloat16)")
    if x.get_device() != device or device < 0:
        raise ValueError(f"{what}: not on the GPU of the others")
    return x.data_ptr(), n, heads, dim, step


def _vector(x, what: str, device: int, name: str, at_least: int) -> int:
    """The address of a contiguous 1-d tensor of at least so many `name` values on GPU `device`."""
    if getattr(x, "requires_grad", False):
        _no_gradient(what)
    got = _KNOWN.get(x.dtype) or _dtype(x)
    if got[0] != name or x.dim() != 1 or x.get_device() != device or not x.is_contiguous():
        raise TypeError(f"{what}: a contiguous 1-d {name} tensor on the GPU of the others")
    if x.shape[0] < at_least:
        raise ValueError(f"{what}: {x.shape[0]} entries, {at_least} needed")
    return x.data_ptr()


def _room(x, device: int) -> tuple:
    """(address, bytes) of a workspace; of none, nothing."""
    if x is None:
        return 0, 0
    if x.get_device() != device or not x.is_contiguous():
        raise TypeError("workspace: a contiguous tensor on the GPU of the others")
    return x.data_ptr(), x.nbytes


class KvLayer:
    """One layer's paged K and V over a batch of sequences (skv_kv_layer): pools of [page][kv_head][cell][head_dim]
    values (float16, or int8 with float16 scales [page][kv_head][cell][head_dim / 64]) and int32 page tables
    [sequence][page], all on the GPU.  Keeps references to the tensors it was made of."""

    def __init__(self, k_pool, v_pool, page_tables, *, k_scale=None, v_scale=None):
        pages, n_head_kv, page_size, head_dim = k_pool.shape
        fmt = {"torch.float16": KV_F16, "torch.int8": KV_INT8}.get(_dtype(k_pool)[0])
        if fmt is None or k_pool.dtype != v_pool.dtype or k_pool.shape != v_pool.shape:
            raise TypeError("KvLayer: two float16 or two int8 pools of one shape")
        scales = [x for x in (k_scale, v_scale) if x is not None]
        if len(scales) != (2 if fmt == KV_INT8 else 0):
            raise ValueError("KvLayer: an int8 pool comes with its scales, a float16 pool with none")
        for x in scales:
            if _dtype(x)[0] != "torch.float16" or tuple(x.shape) != (pages, n_head_kv, page_size, head_dim // 64):
                raise TypeError("KvLayer: scales are float16, [page][kv_head][cell][head_dim / 64]")
        self.device = k_pool.get_device()
        for x in (k_pool, v_pool, *scales):
            if getattr(x, "requires_grad", False):
                _no_gradient("KvLayer")
            if not x.is_contiguous() or x.get_device() != self.device or self.device < 0:
                raise ValueError("KvLayer: pools and scales must be contiguous and on the GPU, all on one")
        self._init(k_pool, v_pool, k_scale, v_scale, page_tables, pages, n_head_kv, head_dim, page_size, fmt)

    def _init(self, k, v, k_scale, v_scale, tables, limit, n_head_kv, head_dim, page_size, fmt):
        if _dtype(tables)[0] != "torch.int32" or tables.dim() != 2 or tables.get_device() != self.device or (tables.shape[1] > 1 and tables.stride(1) != 1):
            raise TypeError("KvLayer: page tables are int32, [sequence][page], on the GPU, the pages of a row contiguous")
        n_tables, width = tables.shape
        step = tables.stride(0) if n_tables > 1 else width
        if step < width:
            raise ValueError("KvLayer: the rows of the page tables overlap")
        self.tensors = (k, v, k_scale, v_scale, tables)
        self.n_head_kv, self.head_dim, self.n_tables = n_head_kv, head_dim, n_tables
        self.args = KvLayerArgs(_ptr(k), _ptr(v), _ptr(k_scale), _ptr(v_scale), tables.data_ptr(), step, limit, n_tables,
                                n_head_kv, head_dim, page_size, fmt, 0)
        self.at = C.addressof(self.args)

    @classmethod
    def of_pool(cls, g: KvGeometry, pool: Pool, page_tables) -> "KvLayer":
        """A layer held in a block pool: `page_tables` are the K tables (layer_page_tables) of its sequences; the V page
        of a slot lies pages_per_block pages behind its K page.  A block pool's pages are float16; an int8 cache is made of
        tensors of its own (KvLayer)."""
        self = cls.__new__(cls)
        shift = g.pages_per_block
        self.device = pool.device
        self._init(pool.base, pool.base + shift * g.page_bytes, None, None, page_tables,
                   pool.n_blocks * g.slot_pages - shift, g.n_head_kv, g.head_dim, PAGE_CELLS, KV_F16)
        self.pool = pool
        return self


def kv_append(layer: KvLayer, k, v, lengths, *, seq_starts=None, q=None, q_out=None, inv_freq=None,
              rope_style: str = "half", rope_scale: float = 1.0, lengths_out=None, stream=None) -> None:
    """Write the K and V rows of new tokens ([token][kv_head][head_dim]) into cells lengths[s], lengths[s]+1, ... of
    their sequences, K rotated by its cell's number, and q rotated into q_out (skv_kv_append)."""
    dev = layer.device
    kp, n, kv, dim, ks = _rows(k, "k", dev)
    kind = k.dtype
    vp, vn, vkv, vdim, vs = _rows(v, "v", dev, kind)
    if vn != n or vkv != kv or vdim != dim or kv != layer.n_head_kv or dim != layer.head_dim:
        raise ValueError("kv_append: k and v are [token][kv_head][head_dim] of the layer")
    n_seqs = n if seq_starts is None else seq_starts.shape[0] - 1
    qp = qo = qs = qos = heads = rot = 0
    if (q is None) != (q_out is None):
        raise ValueError("kv_append: q and q_out come together")
    if q is not None:
        qp, qn, heads, qd, qs = _rows(q, "q", dev, kind)
        qo, on, oh, od, qos = _rows(q_out, "q_out", dev, kind)
        if qn != n or qd != dim or on != n or oh != heads or od != dim:
            raise ValueError("kv_append: q and q_out are [token][head][head_dim]")
    if inv_freq is not None:
        rot = 2 * inv_freq.shape[0]
    args = _APPEND.pack(kp, vp, ks, vs, qp, qo, qs, qos,
                        0 if seq_starts is None else _vector(seq_starts, "seq_starts", dev, "torch.int32", 1),
                        _vector(lengths, "lengths", dev, "torch.int32", n_seqs),
                        0 if lengths_out is None else _vector(lengths_out, "lengths_out", dev, "torch.int32", n_seqs),
                        0 if inv_freq is None else _vector(inv_freq, "inv_freq", dev, "torch.float32", 0),
                        n, n_seqs, heads, rot, ROPE_STYLES[rope_style], _dtype(k)[1], rope_scale, 0)
    check(lib().skv_kv_append(layer.at, args, _stream(stream)))


def decode_attention_workspace(layer: KvLayer, n_seqs: int, n_head: int) -> int:
    """Bytes of device memory that decode_attention needs beside its tensors."""
    out = C.c_uint64()
    check(lib().skv_decode_attention_workspace(layer.at, n_seqs, n_head, C.byref(out)))
    return out.value


def decode_attention(layer: KvLayer, q, lengths, out, *, workspace, scale: float | None = None, lse=None, stream=None) -> None:
    """out = softmax(scale * q K^T) V of one new token per sequence ([sequence][head][head_dim]) over the first
    lengths[s] cells of its cache (skv_decode_attention).  scale: head_dim ** -0.5 when None."""
    dev = layer.device
    qp, n, heads, dim, qs = _rows(q, "q", dev)
    op, on, oh, od, os_ = _rows(out, "out", dev, q.dtype)
    if on != n or oh != heads or od != dim or dim != layer.head_dim:
        raise ValueError("decode_attention: q and out are [sequence][head][head_dim] of the layer")
    lp = 0
    if lse is not None:
        if getattr(lse, "requires_grad", False):
            _no_gradient("lse")
        if _dtype(lse)[0] != "torch.float32" or lse.shape != (n, heads) or not lse.is_contiguous() or lse.get_device() != dev:
            raise TypeError("decode_attention: lse is a contiguous float32 [sequence][head] tensor on the GPU")
        lp = lse.data_ptr()
    args = _ATTENTION.pack(qp, op, qs, os_, lp, _vector(lengths, "lengths", dev, "torch.int32", n), *_room(workspace, dev),
                           n, heads, _dtype(q)[1], dim ** -0.5 if scale is None else scale)
    check(lib().skv_decode_attention(layer.at, args, _stream(stream)))


def gated_delta_workspace(n_tokens: int, n_seqs: int, n_v_heads: int, head_dim: int, max_tokens: int) -> int:
    """Bytes of device memory that gated_delta needs beside its tensors (0 where every sequence is short)."""
    out = C.c_uint64()
    check(lib().skv_gated_delta_workspace(n_tokens, n_seqs, n_v_heads, head_dim, max_tokens, C.byref(out)))
    return out.value


def gated_delta(q, k, v, g, beta, state, out, *, seq_starts=None, state_index=None, max_tokens: int | None = None,
                scale: float | None = None, workspace=None, stream=None) -> None:
    """The gated delta rule over packed sequences (skv_gated_delta): q, k [token][k_head][dim], v, out
    [token][v_head][dim], g, beta float32 [token][v_head], state float32 [row][v_head][dim key][dim value], updated in
    place.  max_tokens bounds the tokens of one sequence (all of them when None; a close bound
    splits the work better: eight sequences of 2,048 tokens take 486 us with it, 736 without).  scale: dim ** -0.5 when None."""
    dev = q.get_device()
    qp, n, kh, dim, qs = _rows(q, "q", dev)
    kind = q.dtype
    kp, kn, kkh, kd, ks = _rows(k, "k", dev, kind)
    vp, vn, vh, vd, vs = _rows(v, "v", dev, kind)
    op, on, oh, od, os_ = _rows(out, "out", dev, kind)
    if kn != n or kkh != kh or kd != dim or vn != n or vd != dim or on != n or oh != vh or od != dim:
        raise ValueError("gated_delta: q and k are [token][k_head][dim], v and out [token][v_head][dim]")
    steps = []
    if getattr(state, "requires_grad", False):
        _no_gradient("state")
    for x, what in ((g, "g"), (beta, "beta")):
        if getattr(x, "requires_grad", False):
            _no_gradient(what)
        if _dtype(x)[0] != "torch.float32" or x.shape != (n, vh) or x.get_device() != dev:
            raise TypeError(f"gated_delta: {what} is a float32 [token][v_head] tensor on the GPU")
        if x.is_contiguous():
            steps.append(vh)
        else:
            step, one = x.stride()
            if one != 1 and vh > 1:
                raise ValueError(f"gated_delta: the heads of {what} must lie back to back")
            steps.append(step if n > 1 else vh)
    rows = state.shape[0]
    if _dtype(state)[0] != "torch.float32" or state.shape[1:] != (vh, dim, dim) or state.get_device() != dev:
        raise TypeError("gated_delta: state is float32 [row][v_head][dim][dim] on the GPU")
    if state.is_contiguous():
        row = vh * dim * dim
    else:
        if not state[0].is_contiguous():
            raise ValueError("gated_delta: each row of the state must be contiguous")
        row = state.stride(0) if rows > 1 else vh * dim * dim
    n_seqs = n if seq_starts is None else seq_starts.shape[0] - 1
    if max_tokens is None:
        max_tokens = 1 if seq_starts is None else n
    args = _DELTA.pack(qp, kp, vp, op, qs, ks, vs, os_, g.data_ptr(), beta.data_ptr(), steps[0], steps[1], state.data_ptr(), row, rows,
                       0 if state_index is None else _vector(state_index, "state_index", dev, "torch.int32", n_seqs),
                       0 if seq_starts is None else _vector(seq_starts, "seq_starts", dev, "torch.int32", 1),
                       *_room(workspace, dev), n, n_seqs,
                       kh, vh, dim, max_tokens, _dtype(q)[1], dim ** -0.5 if scale is None else scale)
    check(lib().skv_gated_delta(args, _stream(stream)))

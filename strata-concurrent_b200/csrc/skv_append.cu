// skv_append.cu - skv_kv_append: K and V of new tokens into their cells of a paged cache, rotated on the way, and q
// beside them.
//
// Pure streaming: every value is read once and written once, so the bytes bound it, where the instructions beside them stay
// few.  A CTA takes kTokens tokens and a share of their rows (a row is one head of q, K or V of one token).  It computes the
// cosines and sines of its tokens once (the angle cell * inv_freq in 64 bits, reduced by whole turns, then a 32-bit sincos of
// at most pi) and every row uses them from shared memory.  Of K and V, head_dim / 8 lanes hold a row, 16 bytes each; the
// half-style pair of a lane's values lies in another lane of the same row: one shuffle.  Of q, by far the most rows, what is
// not turned is copied as it lies (or left, in place), and what is turned goes 16 values a thread, both of a pair, in full
// warps: 32K tokens 155 us, 166 with q's rows treated like K's, at 80 % of all issue slots.
//
// Measured (24 + 4 heads of 256, 64 turned, in a graph): 32K tokens into an fp16 cache 155 us, 6.1 TB/s; into an int8 cache
// 155 us, 5.9 TB/s.  A ragged batch of 7,948 tokens into an int8 cache 45 us, 4.9 TB/s: its 994 CTAs are 1.7 times what runs at
// once, and cutting them finer repeats the angles.  One token 3 us: a launch.
#include "skv_ops.h"

#include <string>

namespace skv {

int check_layer(const skv_kv_layer* l, int n_seqs, const char* what) {
    const auto no = [what](const char* why) { return fail(SKV_EINVAL, std::string(what) + ": " + why); };
    if (!l) return no("no layer");
    if (l->format != SKV_KV_F16 && l->format != SKV_KV_INT8) return no("unknown cache format");
    if (l->head_dim != 64 && l->head_dim != 128 && l->head_dim != 256) return no("head_dim must be 64, 128 or 256");
    if (l->page_size < 1 || l->page_size > 256 || (l->page_size & (l->page_size - 1)))
        return no("page_size must be a power of two up to 256");
    if (l->n_head_kv < 1 || l->n_head_kv > 1024) return no("n_head_kv must be in [1, 1024]");
    if (l->page_limit < 1 || l->page_limit > INT32_MAX || l->table_stride < 1 || l->table_stride > INT32_MAX)
        return no("page_limit and table_stride must be in [1, 2^31)");
    if (n_seqs > l->n_tables) return no("more sequences than page tables");
    if (!l->k_pool || !l->v_pool || !l->page_tables) return no("missing pool or page table");
    if (!ops_aligned16(l->k_pool) || !ops_aligned16(l->v_pool)) return no("pools must be 16-byte aligned");
    if (l->format == SKV_KV_INT8) {
        if (!l->k_scale || !l->v_scale) return no("an int8 layer needs its scales");
        if ((reinterpret_cast<uintptr_t>(l->k_scale) | reinterpret_cast<uintptr_t>(l->v_scale)) & 7u)
            return no("scales must be 8-byte aligned");
    }
    if (!ops_aligned4(l->page_tables)) return no("page tables must be 4-byte aligned");
    return SKV_OK;
}

int check_layer_memory(const skv_kv_layer& l, int device, const char* what) {
    const bool scales = l.format == SKV_KV_INT8;
    for (const void* p : {l.k_pool, l.v_pool, scales ? l.k_scale : nullptr, scales ? l.v_scale : nullptr})
        if (p && !ops_own_memory(p, device)) return fail(SKV_EINVAL, std::string(what) + ": the pool is not memory of the current device");
    return SKV_OK;
}

LayerDev to_device(const skv_kv_layer& l) {
    LayerDev d{};
    d.k = static_cast<uint8_t*>(l.k_pool);
    d.v = static_cast<uint8_t*>(l.v_pool);
    d.k_scale = static_cast<__half*>(l.k_scale);
    d.v_scale = static_cast<__half*>(l.v_scale);
    d.tables = l.page_tables;
    d.table_stride = l.table_stride;
    d.page_limit = l.page_limit;
    d.n_head_kv = l.n_head_kv;
    while ((1 << d.page_shift) < l.page_size) ++d.page_shift;
    return d;
}

namespace {

constexpr int kTokens = 8;      // tokens per CTA
constexpr int kThreads = 256;
// 16-byte pieces a thread has on their way at once: of K and V, beside those it works on; of q's copies; and of q's turned
// pieces, two each.  32K tokens of 24 + 4 heads of 256, fp16 and int8 caches, and a ragged int8 batch: 8 copies and 2 turns
// 155, 155 and 45 us; 4 and 2 158, 162 and 46; 2 and 1 164, 169 and 51; 4 and 4 172, 222 and 67 (registers cost CTAs).  One of K
// and V ahead in place of two: 159, 157 and 45.  4 or 16 tokens per CTA: 162 and 163, 166 and 171, 48 and 49.
constexpr int kAhead = 2;
constexpr int kCopies = 8, kTurns = 2;
constexpr int kMaxPairs = 128;  // n_rot / 2 of the widest head

struct AppendDev {
    LayerDev layer;
    skv_append_args a;
    uint32_t* status;
    int share;        // rows (over all of the CTA's tokens) per CTA in y
    float per_kv, per_q, per_turn;   // 1 / rows of K and V a token, 1 / rows of q a token, 1 / groups of eight pairs a row
};

/// r / d of small numbers (below 2^20 here), by = 1 / d: exact, as r + 1/2 is half a part away from the next quotient.
__device__ __forceinline__ int quotient_of(int r, float by) { return (int) (((float) r + 0.5f) * by); }
__device__ __forceinline__ void turn_pair(float& x, float& y, float2 c) {
    const float u = x;
    x = u * c.x - y * c.y;
    y = y * c.x + u * c.y;
}

/// The sequence of packed row `row`, the last s with starts[s] <= row, found by a whole warp, 32 places at a time; -1
/// outside of [starts[0], starts[n]).
__device__ __forceinline__ int sequence_of(const int32_t* starts, int n, int row) {
    const int lane = threadIdx.x & 31;
    int lo = -1, hi = n;   // starts[lo] <= row (or lo = -1), row < starts[hi] (or hi = n, checked below)
    while (hi - lo > 1) {
        const int step = (hi - lo - 1 + 31) / 32, at = lo + (lane + 1) * step;
        const int below = __popc(__ballot_sync(0xffffffffu, at < hi && __ldg(starts + min(at, n)) <= row));
        hi = min(hi, lo + (below + 1) * step);
        lo += below * step;
    }
    return lo < 0 || row >= __ldg(starts + n) ? -1 : lo;
}

/// One group of eight lanes quantizes its 64 values: the scale, and this lane's eight codes packed.
__device__ __forceinline__ uint2 quantize(const float (&x)[8], __half& scale) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));   // fmaxf passes a NaN over
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    scale = __float2half_rn(fminf(top / 127.0f, 65504.0f));
    const float step = __half2float(scale), by = step > 0.0f ? 1.0f / step : 0.0f, half = 0.5f * step;
    // The quotient by a reciprocal, rounded as it is added to 1.5 * 2^23, whose low byte is then the code.  What it leaves over
    // is exact (a code and a scale have 18 bits together) and, where it is less than half a step, proves the code.
    constexpr float kWhole = 12582912.0f;
    uint32_t w[2] = {0, 0}, code[8];
    bool sure = top <= 127.25f * step;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = fmaf(x[i], by, kWhole);
        code[i] = __float_as_uint(c);
        sure = sure && fabsf(fmaf(kWhole - c, step, x[i])) < half;   // not for a NaN, nor where the step is zero
    }
    if (sure) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = __byte_perm(__byte_perm(code[4 * i], code[4 * i + 1], 0x0040), __byte_perm(code[4 * i + 2], code[4 * i + 3], 0x0040), 0x5410);
        return make_uint2(w[0], w[1]);
    }
    if (step == 0.0f) return make_uint2(0, 0);   // a group too small for a scale
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // ties, codes off by one, and values far past the scale
        float c = rintf(fminf(fmaxf(x[i] * by, -127.0f), 127.0f));   // a NaN becomes -127 here ...
        const float left = fmaf(-c, step, x[i]);
        if (left > half && c < 127.0f) c += 1.0f;
        else if (left < -half && c > -127.0f) c -= 1.0f;
        else if (fabsf(left) == half && ((int) c & 1)) c += left > 0.0f ? 1.0f : -1.0f;
        c = x[i] == x[i] ? fminf(fmaxf(c, -127.0f), 127.0f) : 0.0f;   // ... and 0 here
        w[i >> 2] |= ((uint32_t) (int) c & 0xffu) << ((i & 3) * 8);
    }
    return make_uint2(w[0], w[1]);
}

template <typename T, int kDim, bool kInt8>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendDev p) {
    constexpr int kLanes = kDim / 8;
    __shared__ float2 turn[kTokens][kMaxPairs];
    __shared__ bool s_held[kTokens];      // by a sequence
    __shared__ int64_t s_cell[kTokens], s_row[kTokens];
    const skv_append_args& a = p.a;
    const int tid = threadIdx.x, first = blockIdx.x * kTokens;
    const int pairs = a.n_rot >> 1;
    const int kv = p.layer.n_head_kv, kv_rows = 2 * kv * kTokens;
    const int lane = tid % kLanes, at = lane * 8;
    const int lo = blockIdx.y * p.share, hi = min(lo + p.share, kv_rows + (a.q ? a.n_head * kTokens : 0));
    const int kv_hi = min(hi, kv_rows);
    constexpr int kTrip = kThreads / kLanes;
    uint4 ahead[kAhead];
    // the CTA's rows: K's heads and V's of its first token, of the next one ...; then q's in the same way.  Only rows of the
    // call's arrays are touched, whether or not a sequence has them: what no sequence has is not used.
    const auto fetch = [&](int base) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int r = base + i * kTrip + tid / kLanes;
            const int t = quotient_of(r, p.per_kv), row = r - t * 2 * kv;
            ahead[i] = make_uint4(0, 0, 0, 0);
            if (r < kv_hi && first + t < a.n_tokens) {
                const int64_t token = first + t;
                const T* src = row < kv ? static_cast<const T*>(a.k) + token * a.k_stride + row * kDim
                                        : static_cast<const T*>(a.v) + token * a.v_stride + (row - kv) * kDim;
                ahead[i] = *reinterpret_cast<const uint4*>(src + at);
            }
        }
    };
    wait_for_previous();
    fetch(lo);   // on their way while the angles are worked out

    if (blockIdx.y == 0 && a.lengths_out && blockIdx.x < 65536) {   // as many CTAs as keep the steps within 32 bits
        for (uint32_t s = blockIdx.x * kThreads + tid; s < (uint32_t) a.n_seqs; s += min(gridDim.x, 65536u) * kThreads) {
            const int n = a.seq_starts ? max(0, __ldg(a.seq_starts + s + 1) - __ldg(a.seq_starts + s)) : 1;
            a.lengths_out[s] = (int) min((uint32_t) max(0, __ldg(a.lengths + s)) + (uint32_t) n, 0x7fffffffu);
        }
    }
    // a warp per token: its sequence, its cell, and the cell's row in the pools
    for (int i = tid >> 5; i < kTokens; i += kThreads / 32) {
        const int t = first + i;
        int s = -1;
        int64_t cell = 0, row = -1;
        if (t < a.n_tokens) {
            s = a.seq_starts ? sequence_of(a.seq_starts, a.n_seqs, t) : t;
            if (s >= 0) {
                const int held = __ldg(a.lengths + s);
                // behind a negative length there are no cells: q is turned as at cell 0
                if (held >= 0) {
                    cell = (int64_t) held + (a.seq_starts ? t - __ldg(a.seq_starts + s) : 0);
                    row = cell_row(p.layer, s, cell, 0);
                }
                if (row < 0 && (tid & 31) == 0) atomicOr(p.status, SKV_STATUS_BAD_DST_PAGE);
            }
        }
        if ((tid & 31) == 0) {
            s_held[i] = s >= 0;
            s_cell[i] = cell;
            s_row[i] = row;
        }
    }
    __syncthreads();
    for (int i = tid; i < kTokens * pairs; i += kThreads) {
        const int t = i / pairs, j = i - t * pairs;
        if (!s_held[t]) continue;
        const double angle = (double) s_cell[t] * (double) __ldg(a.inv_freq + j);
        const double turns = rint(angle * 0.15915494309189533577);   // 1 / (2 pi)
        // 2 pi in two parts: turns * the first is exact enough for 2^31 cells of one radian each
        const double rest = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586232, angle));
        float sn, cs;
        sincosf((float) rest, &sn, &cs);
        turn[t][j] = make_float2(cs * a.rope_scale, sn * a.rope_scale);
    }
    __syncthreads();

    // ---- K and V.  Every lane of a row makes the same trips, and a warp's lanes meet at the shuffles: rows past the end are idle
    for (int base = lo; base < kv_hi; base += kAhead * kTrip) {
        uint4 now[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) now[i] = ahead[i];
        if (base + kAhead * kTrip < kv_hi) fetch(base + kAhead * kTrip);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int r = base + i * kTrip + tid / kLanes;
            if (base + i * kTrip >= kv_hi) break;   // the same for the whole CTA
            const int t = min(quotient_of(r, p.per_kv), kTokens - 1), row = r - t * 2 * kv;
            const bool on = r < kv_hi && s_held[t], is_k = row < kv;
            const uint4 raw = now[i];
            float x[8];
            unpack8<T>(raw, x);
            if (pairs) {
                if (a.rope_style == SKV_ROPE_HALF) {
                    const int hop = pairs / 8;   // lanes between the two values of a pair
                    const bool low = at < pairs;
                    const int other = (tid & 31) + (low ? hop : -hop);
                    uint4 o;
                    o.x = __shfl_sync(0xffffffffu, raw.x, other & 31);
                    o.y = __shfl_sync(0xffffffffu, raw.y, other & 31);
                    o.z = __shfl_sync(0xffffffffu, raw.z, other & 31);
                    o.w = __shfl_sync(0xffffffffu, raw.w, other & 31);
                    if (on && is_k && at < a.n_rot) {
                        float y[8];
                        unpack8<T>(o, y);
                        const int j = low ? at : at - pairs;
#pragma unroll
                        for (int m = 0; m < 8; ++m) {
                            const float2 c = turn[t][j + m];
                            x[m] = low ? x[m] * c.x - y[m] * c.y : x[m] * c.x + y[m] * c.y;
                        }
                    }
                } else if (on && is_k && at < a.n_rot) {
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        const float2 c = turn[t][at / 2 + m];
                        const float u = x[2 * m], w = x[2 * m + 1];
                        x[2 * m] = u * c.x - w * c.y;
                        x[2 * m + 1] = w * c.x + u * c.y;
                    }
                }
            }
            const int64_t to = on && s_row[t] >= 0 ? s_row[t] + ((int64_t) (is_k ? row : row - kv) << p.layer.page_shift) : -1;
            if (kInt8) {
                __half scale;
                const uint2 codes = quantize(x, scale);
                if (to >= 0) {
                    uint8_t* pool = is_k ? p.layer.k : p.layer.v;
                    *reinterpret_cast<uint2*>(pool + to * kDim + at) = codes;
                    if ((lane & 7) == 0) (is_k ? p.layer.k_scale : p.layer.v_scale)[to * (kDim / kInt8Group) + lane / 8] = scale;
                }
            } else if (to >= 0) {
                // rounded to the cache's fp16, once; a bf16 value past its range becomes infinite
                *reinterpret_cast<uint4*>((is_k ? p.layer.k : p.layer.v) + (to * kDim + at) * 2) = pack8<__half>(x);
            }
        }
    }
    if (hi <= kv_rows) return;

    // ---- q.  What is not turned is copied as it lies, unless it lies there already
    const int q_lo = max(lo - kv_rows, 0), q_hi = hi - kv_rows;
    const T* const q = static_cast<const T*>(a.q);
    T* const q_out = static_cast<T*>(a.q_out);
    if (a.n_rot < kDim && q != q_out) {
        for (int base = q_lo + tid / kLanes; base < q_hi; base += kCopies * kTrip) {
            uint4 w[kCopies];
            int64_t to[kCopies];
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const int r = base + i * kTrip, t = quotient_of(r, p.per_q);
                to[i] = -1;
                if (r < q_hi && at >= a.n_rot && s_held[t]) {
                    const int64_t token = first + t, in = (r - t * a.n_head) * kDim + at;
                    to[i] = token * a.q_out_stride + in;
                    w[i] = *reinterpret_cast<const uint4*>(q + token * a.q_stride + in);
                }
            }
#pragma unroll
            for (int i = 0; i < kCopies; ++i)
                if (to[i] >= 0) *reinterpret_cast<uint4*>(q_out + to[i]) = w[i];
        }
    }
    // ... and eight pairs a thread are turned, in whole warps whatever part of a row that is: 16 bytes at one place and 16 at
    // another, half a rotation or 16 bytes away
    if (pairs) {
        const bool halves = a.rope_style == SKV_ROPE_HALF;
        const int per = a.n_rot >> 4, apart = halves ? pairs : 8;
        const int end = q_hi * per;
        for (int base = q_lo * per + tid; base < end; base += kTurns * kThreads) {
            uint4 v[kTurns], w[kTurns];
            int64_t to[kTurns];
            const float2* by[kTurns];
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                const int e = base + i * kThreads, r = quotient_of(e, p.per_turn), j = e - r * per, t = quotient_of(r, p.per_q);
                to[i] = -1;
                if (e < end && s_held[t]) {
                    const int64_t token = first + t, in = (r - t * a.n_head) * kDim + j * (halves ? 8 : 16);
                    to[i] = token * a.q_out_stride + in;
                    by[i] = &turn[t][j * 8];
                    v[i] = *reinterpret_cast<const uint4*>(q + token * a.q_stride + in);
                    w[i] = *reinterpret_cast<const uint4*>(q + token * a.q_stride + in + apart);
                }
            }
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                if (to[i] < 0) continue;
                float x[8], y[8];
                unpack8<T>(v[i], x);
                unpack8<T>(w[i], y);
                if (halves) {
#pragma unroll
                    for (int m = 0; m < 8; ++m) turn_pair(x[m], y[m], by[i][m]);
                } else {
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        turn_pair(x[2 * m], x[2 * m + 1], by[i][m]);
                        turn_pair(y[2 * m], y[2 * m + 1], by[i][m + 4]);
                    }
                }
                *reinterpret_cast<uint4*>(q_out + to[i]) = pack8<T>(x);
                *reinterpret_cast<uint4*>(q_out + to[i] + apart) = pack8<T>(y);
            }
        }
    }
}

template <typename T, int kDim>
cudaError_t launch(const AppendDev& p, dim3 grid, bool int8, cudaStream_t stream) {
    return int8 ? launch_early(append_kernel<T, kDim, true>, grid, kThreads, 0, stream, p)
                : launch_early(append_kernel<T, kDim, false>, grid, kThreads, 0, stream, p);
}
template <typename T>
cudaError_t launch(const AppendDev& p, int dim, dim3 grid, bool int8, cudaStream_t stream) {
    return dim == 64 ? launch<T, 64>(p, grid, int8, stream) : dim == 128 ? launch<T, 128>(p, grid, int8, stream) : launch<T, 256>(p, grid, int8, stream);
}

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" int skv_kv_append(const skv_kv_layer* layer, const skv_append_args* args, void* stream) {
    const auto no = [](const char* why) { return fail(SKV_EINVAL, std::string("skv_kv_append: ") + why); };
    if (!args) return no("no arguments");
    const skv_append_args& a = *args;
    if (a.n_tokens < 0 || a.n_seqs < 0) return no("negative counts");
    if (const int rc = check_layer(layer, a.n_seqs, "skv_kv_append")) return rc;
    if (a.n_seqs == 0) return SKV_OK;
    if (!a.lengths) return no("no lengths");
    if (!a.seq_starts && a.n_tokens != a.n_seqs) return no("without seq_starts every sequence has one row");
    if (!ops_aligned4(a.lengths, a.lengths_out, a.seq_starts, a.inv_freq)) return no("lengths, starts and inv_freq must be 4-byte aligned");
    if (a.lengths_out == a.lengths) return no("lengths_out must not be lengths");
    if (a.dtype != SKV_DTYPE_F16 && a.dtype != SKV_DTYPE_BF16) return no("unknown dtype");
    if (a.rope_style != SKV_ROPE_HALF && a.rope_style != SKV_ROPE_PAIRS) return no("unknown rope style");
    if (a.n_rot < 0 || a.n_rot > layer->head_dim || a.n_rot % 16) return no("n_rot must be a multiple of 16, at most head_dim");
    if (a.n_rot && !a.inv_freq) return no("a rotation needs inv_freq");
    if (a.n_tokens) {
        if (!a.k || !a.v) return no("missing k or v");
        if (!ops_aligned16(a.k) || !ops_aligned16(a.v) || a.k_stride % 8 || a.v_stride % 8)
            return no("k and v must be 16-byte aligned, their strides multiples of 8");
        const int64_t row = (int64_t) layer->n_head_kv * layer->head_dim;
        if (a.n_tokens > 1 && (a.k_stride < row || a.v_stride < row)) return no("a stride is shorter than its row");
    }
    if ((a.q == nullptr) != (a.q_out == nullptr)) return no("q and q_out come together");
    if (a.q) {
        if (a.n_head < 1 || a.n_head > 4096) return no("n_head must be in [1, 4096]");
        if (!ops_aligned16(a.q) || !ops_aligned16(a.q_out) || a.q_stride % 8 || a.q_out_stride % 8)
            return no("q and q_out must be 16-byte aligned, their strides multiples of 8");
        if (a.n_tokens > 1 && (a.q_stride < (int64_t) a.n_head * layer->head_dim || a.q_out_stride < (int64_t) a.n_head * layer->head_dim))
            return no("a stride is shorter than its row");
        if (a.q == a.q_out && a.q_stride != a.q_out_stride) return no("q in place needs one stride");
    }
    DeviceCtx* ctx = current_ctx();
    if (!ctx) return SKV_ECUDA;
    if (const int rc = check_layer_memory(*layer, ctx->device, "skv_kv_append")) return rc;
    AppendDev p{};
    p.layer = to_device(*layer);
    p.a = a;
    p.status = ctx->status;
    // Few tokens: spread each CTA's rows over more CTAs, down to one trip each, until the GPU has two per SM.
    const int blocks = a.n_tokens ? (a.n_tokens - 1) / kTokens + 1 : 1;
    const int rows = ((a.q ? a.n_head : 0) + 2 * layer->n_head_kv) * kTokens, trip = kThreads * 8 / layer->head_dim;
    int split = (2 * ctx->sms + blocks - 1) / blocks;
    const int trips = (rows + trip - 1) / trip;
    if (split > trips) split = trips;
    p.share = (trips + split - 1) / split * trip;
    p.per_kv = 1.0f / (float) (2 * layer->n_head_kv);
    p.per_q = a.q ? 1.0f / (float) a.n_head : 1.0f;
    p.per_turn = a.n_rot ? 16.0f / (float) a.n_rot : 1.0f;
    const dim3 grid((unsigned) blocks, (unsigned) ((rows + p.share - 1) / p.share));
    const auto s = static_cast<cudaStream_t>(stream);
    const bool int8 = layer->format == SKV_KV_INT8;
    const cudaError_t e = a.dtype == SKV_DTYPE_F16 ? launch<__half>(p, layer->head_dim, grid, int8, s)
                                                   : launch<__nv_bfloat16>(p, layer->head_dim, grid, int8, s);
    return e == cudaSuccess ? SKV_OK : cuda_fail(e, "skv_kv_append");
}

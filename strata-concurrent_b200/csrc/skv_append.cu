// skv_append.cu - skv_kv_append: K and V of new tokens into their cells of a paged cache, rotated on the way, and q
// beside them.
//
// Pure streaming: every value is read once and written once, so the bytes bound it.  A CTA takes kTokens tokens and
// a share of their rows (a row is one head of q, K or V of one token).  It computes the cosines and sines of its tokens
// once (the angle cell * inv_freq in 64 bits, reduced by whole turns, then a 32-bit sincos of at most pi) and every row
// uses them from shared memory; head_dim / 8 lanes hold a row, 16 bytes each, so a warp's loads and stores are whole
// lines.  The half-style pair of a lane's values lies in another lane of the same row: one shuffle.
//
// Measured (24 + 4 heads of 256, 64 turned, in a graph): 32K tokens into an fp16 cache 166 us, 5.7 TB/s; into an int8 cache
// 190 us, 4.7 TB/s, where finding the codes costs issue slots.  A ragged batch of 7,948 tokens into an int8 cache 52 us: its
// 994 CTAs are 1.3 times what runs at once, and cutting them finer repeats the angles (47 to 57 us more or less at two, eight
// and 48 CTAs per SM).  One token 2.8 us: a launch.
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
    if (reinterpret_cast<uintptr_t>(l->page_tables) & 3u) return no("page tables must be 4-byte aligned");
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
// Rows a thread has on their way at once, beside those it works on.  With 8 tokens per CTA, 32K tokens of 24 + 4 heads of
// 256 take 167 us at 2 and at 4, 188 at 7 (registers cost CTAs); 8K tokens 57 at 2, 66 at 4.  4 or 16 tokens per CTA: 170, 167
// and, for 64 single tokens, 3.1 and 4.2 against 3.3.
constexpr int kAhead = 2;
constexpr int kMaxPairs = 128;  // n_rot / 2 of the widest head

struct AppendDev {
    LayerDev layer;
    skv_append_args a;
    uint32_t* status;
    int share;        // rows (over all of the CTA's tokens) per CTA in y
    float per_row;    // 1 / rows of a token
};

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
    const int kv = p.layer.n_head_kv, rows = (a.q ? a.n_head : 0) + 2 * kv;
    const int lane = tid % kLanes, at = lane * 8;
    const int lo = blockIdx.y * p.share, hi = min(lo + p.share, rows * kTokens);
    constexpr int kTrip = kThreads / kLanes;
    uint4 ahead[kAhead];
    // row r of the CTA's tokens: K's heads, V's, q's of the first token, then the next one's.  Only rows of the call's
    // arrays are touched, whether or not a sequence has them: what no sequence has is not used.
    const auto fetch = [&](int base) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int r = base + i * kTrip + tid / kLanes;
            const int t = (int) (((float) r + 0.5f) * p.per_row), row = r - t * rows;   // exact: r < 2^17
            ahead[i] = make_uint4(0, 0, 0, 0);
            if (r < hi && first + t < a.n_tokens) {
                const int64_t token = first + t;
                const T* src = row < kv ? static_cast<const T*>(a.k) + token * a.k_stride + row * kDim
                             : row < 2 * kv ? static_cast<const T*>(a.v) + token * a.v_stride + (row - kv) * kDim
                                            : static_cast<const T*>(a.q) + token * a.q_stride + (row - 2 * kv) * kDim;
                ahead[i] = *reinterpret_cast<const uint4*>(src + at);
            }
        }
    };
    wait_for_previous();
    fetch(lo);   // on their way while the angles are worked out

    if (blockIdx.y == 0 && a.lengths_out) {
        for (int s = blockIdx.x * kThreads + tid; s < a.n_seqs; s += gridDim.x * kThreads) {
            const int n = a.seq_starts ? max(0, __ldg(a.seq_starts + s + 1) - __ldg(a.seq_starts + s)) : 1;
            a.lengths_out[s] = max(0, __ldg(a.lengths + s)) + n;
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

    // every lane of a row makes the same trips, and a warp's lanes meet at the shuffles: rows past the end are idle
    for (int base = lo; base < hi; base += kAhead * kTrip) {
        uint4 now[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) now[i] = ahead[i];
        if (base + kAhead * kTrip < hi) fetch(base + kAhead * kTrip);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int r = base + i * kTrip + tid / kLanes;
        if (base + i * kTrip >= hi) break;   // the same for the whole CTA
        const int t = min((int) (((float) r + 0.5f) * p.per_row), kTokens - 1), row = r - t * rows;
        const bool on = r < hi && s_held[t];
        const int64_t token = first + t;
        const bool is_k = row < kv, is_v = !is_k && row < 2 * kv;
        const int head = is_k ? row : is_v ? row - kv : row - 2 * kv;
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
                if (on && !is_v && at < a.n_rot) {
                    float y[8];
                    unpack8<T>(o, y);
                    const int j = low ? at : at - pairs;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 c = turn[t][j + i];
                        x[i] = low ? x[i] * c.x - y[i] * c.y : x[i] * c.x + y[i] * c.y;
                    }
                }
            } else if (on && !is_v && at < a.n_rot) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 c = turn[t][at / 2 + i];
                    const float u = x[2 * i], w = x[2 * i + 1];
                    x[2 * i] = u * c.x - w * c.y;
                    x[2 * i + 1] = w * c.x + u * c.y;
                }
            }
        }
        int64_t to = -1;
        if (on && (is_k || is_v) && s_row[t] >= 0) to = s_row[t] + ((int64_t) head << p.layer.page_shift);
        if (kInt8) {
            __half scale;
            uint2 codes;
            if (__any_sync(0xffffffffu, to >= 0)) codes = quantize(x, scale);   // not for a warp of query rows
            if (to >= 0) {
                uint8_t* pool = is_k ? p.layer.k : p.layer.v;
                *reinterpret_cast<uint2*>(pool + to * kDim + at) = codes;
                if ((lane & 7) == 0) (is_k ? p.layer.k_scale : p.layer.v_scale)[to * (kDim / kInt8Group) + lane / 8] = scale;
            }
        } else if (to >= 0) {
            // rounded to the cache's fp16, once; a bf16 value past its range becomes infinite
            *reinterpret_cast<uint4*>((is_k ? p.layer.k : p.layer.v) + (to * kDim + at) * 2) = pack8<__half>(x);
        }
        if (on && !is_k && !is_v)
            *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + token * a.q_out_stride + head * kDim + at) = pack8<T>(x);
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
    if (!ops_own_memory(layer->k_pool, ctx->device)) return no("the pool is not memory of the current device");
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
    p.per_row = 1.0f / (float) (rows / kTokens > 0 ? rows / kTokens : 1);
    const dim3 grid((unsigned) blocks, (unsigned) ((rows + p.share - 1) / p.share));
    const auto s = static_cast<cudaStream_t>(stream);
    const bool int8 = layer->format == SKV_KV_INT8;
    const cudaError_t e = a.dtype == SKV_DTYPE_F16 ? launch<__half>(p, layer->head_dim, grid, int8, s)
                                                   : launch<__nv_bfloat16>(p, layer->head_dim, grid, int8, s);
    return e == cudaSuccess ? SKV_OK : cuda_fail(e, "skv_kv_append");
}

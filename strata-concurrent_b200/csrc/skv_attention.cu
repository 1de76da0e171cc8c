// skv_attention.cu - skv_decode_attention: one new token per sequence over its paged cache.
//
//   s_t = scale * q . k_t;   m = max s_t;   out = sum e^(s_t - m) v_t / sum e^(s_t - m);   lse = m + ln sum
//
// One CTA per (query head, sequence): each warp walks every eighth cell with a running maximum and sum, holding
// head_dim / 32 values of q and of the output per lane, and the warps' parts are joined through shared memory.
#include "skv_ops.h"

#include <cmath>
#include <string>

namespace skv {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct AttnDev {
    LayerDev layer;
    skv_attention_args a;
    uint32_t* status;
    int group;
};

template <typename T, int kDim, bool kInt8>
__global__ void __launch_bounds__(kThreads) attention_kernel(const __grid_constant__ AttnDev p) {
    constexpr int kPer = kDim / 32;
    const skv_attention_args& a = p.a;
    const int head = blockIdx.x, seq = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t table_cells = p.layer.table_stride << p.layer.page_shift;
    const int asked = __ldg(a.lengths + seq);
    const int64_t n = asked < 0 ? 0 : asked > table_cells ? table_cells : asked;
    if ((asked < 0 || asked > table_cells) && threadIdx.x == 0) atomicOr(p.status, SKV_STATUS_BAD_SRC_PAGE);
    float q[kPer], o[kPer], m = -INFINITY, sum = 0.0f;
    const T* qr = static_cast<const T*>(a.q) + seq * a.q_stride + head * kDim + lane * kPer;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        q[i] = (float) qr[i] * a.scale;
        o[i] = 0.0f;
    }
    for (int64_t t = warp; t < n; t += kWarps) {
        const int64_t row = cell_row(p.layer, seq, t, head / p.group);
        if (row < 0) {
            if (lane == 0) atomicOr(p.status, SKV_STATUS_BAD_SRC_PAGE);
            continue;
        }
        float k[kPer], v[kPer];
        if (kInt8) {
            const int g = lane * kPer / kInt8Group;
            const float ks = __half2float(p.layer.k_scale[row * (kDim / kInt8Group) + g]);
            const float vs = __half2float(p.layer.v_scale[row * (kDim / kInt8Group) + g]);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                k[i] = ks * (float) reinterpret_cast<const int8_t*>(p.layer.k)[row * kDim + lane * kPer + i];
                v[i] = vs * (float) reinterpret_cast<const int8_t*>(p.layer.v)[row * kDim + lane * kPer + i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                k[i] = __half2float(reinterpret_cast<const __half*>(p.layer.k)[row * kDim + lane * kPer + i]);
                v[i] = __half2float(reinterpret_cast<const __half*>(p.layer.v)[row * kDim + lane * kPer + i]);
            }
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) s = fmaf(q[i], k[i], s);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (s == -INFINITY) continue;   // a weight of zero, and no maximum to take a difference from
        const float top = fmaxf(m, s), keep = expf(m - top), w = expf(s - top);
        sum = sum * keep + w;
#pragma unroll
        for (int i = 0; i < kPer; ++i) o[i] = o[i] * keep + w * v[i];
        m = top;
    }
    __shared__ float s_m[kWarps], s_sum[kWarps], s_o[kWarps][kDim];
    if (lane == 0) {
        s_m[warp] = m;
        s_sum[warp] = sum;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) s_o[warp][lane * kPer + i] = o[i];
    __syncthreads();
    float top = -INFINITY, total = 0.0f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
    for (int w = 0; w < kWarps; ++w) total += s_sum[w] != 0.0f ? s_sum[w] * expf(s_m[w] - top) : 0.0f;
    if (threadIdx.x < kDim) {
        float x = 0.0f;
        for (int w = 0; w < kWarps; ++w)
            if (s_sum[w] != 0.0f) x += s_o[w][threadIdx.x] * expf(s_m[w] - top);
        static_cast<T*>(a.out)[seq * a.out_stride + head * kDim + threadIdx.x] = Pair<T>::one(total != 0.0f ? x / total : 0.0f);
    }
    if (a.lse && threadIdx.x == 0) a.lse[(int64_t) seq * a.n_head + head] = total != 0.0f ? top + logf(total) : -INFINITY;
}

template <typename T, int kDim>
void launch(const AttnDev& p, bool int8, cudaStream_t stream) {
    const dim3 grid((unsigned) p.a.n_head, (unsigned) p.a.n_seqs);
    if (int8) attention_kernel<T, kDim, true><<<grid, kThreads, 0, stream>>>(p);
    else attention_kernel<T, kDim, false><<<grid, kThreads, 0, stream>>>(p);
}
template <typename T>
void launch(const AttnDev& p, int dim, bool int8, cudaStream_t stream) {
    if (dim == 64) launch<T, 64>(p, int8, stream);
    else if (dim == 128) launch<T, 128>(p, int8, stream);
    else launch<T, 256>(p, int8, stream);
}

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" {

int skv_decode_attention_workspace(const skv_kv_layer* layer, int n_seqs, int n_head, uint64_t* out_bytes) {
    if (!out_bytes) return fail(SKV_EINVAL, "skv_decode_attention_workspace: null output");
    *out_bytes = 0;
    if (n_seqs < 0 || n_head < 1) return fail(SKV_EINVAL, "skv_decode_attention_workspace: bad counts");
    if (const int rc = check_layer(layer, n_seqs, "skv_decode_attention_workspace")) return rc;
    *out_bytes = 256;
    return SKV_OK;
}

int skv_decode_attention(const skv_kv_layer* layer, const skv_attention_args* args, void* stream) {
    const auto no = [](const char* why) { return fail(SKV_EINVAL, std::string("skv_decode_attention: ") + why); };
    if (!args) return no("no arguments");
    const skv_attention_args& a = *args;
    if (a.n_seqs < 0 || a.n_seqs > 65535) return no("n_seqs must be in [0, 65535]");
    if (const int rc = check_layer(layer, a.n_seqs, "skv_decode_attention")) return rc;
    if (a.n_head < 1 || a.n_head > 4096 || a.n_head % layer->n_head_kv) return no("n_head must be a multiple of n_head_kv, at most 4096");
    if (a.dtype != SKV_DTYPE_F16 && a.dtype != SKV_DTYPE_BF16) return no("unknown dtype");
    if (!(a.scale > -INFINITY && a.scale < INFINITY)) return no("the scale must be finite");
    if (a.n_seqs == 0) return SKV_OK;
    if (!a.q || !a.out || !a.lengths) return no("missing q, out or lengths");
    if (!ops_aligned16(a.q) || !ops_aligned16(a.out) || a.q_stride % 8 || a.out_stride % 8)
        return no("q and out must be 16-byte aligned, their strides multiples of 8");
    const int64_t row = (int64_t) a.n_head * layer->head_dim;
    if (a.n_seqs > 1 && (a.q_stride < row || a.out_stride < row)) return no("a stride is shorter than its row");
    uint64_t need = 0;
    if (const int rc = skv_decode_attention_workspace(layer, a.n_seqs, a.n_head, &need)) return rc;
    if (!a.workspace || (reinterpret_cast<uintptr_t>(a.workspace) & 255u) || a.workspace_bytes < need)
        return no("the workspace must be 256-byte aligned and as large as skv_decode_attention_workspace says");
    DeviceCtx* ctx = current_ctx();
    if (!ctx) return SKV_ECUDA;
    if (!ops_own_memory(layer->k_pool, ctx->device)) return no("the pool is not memory of the current device");
    AttnDev p{};
    p.layer = to_device(*layer);
    p.a = a;
    p.status = ctx->status;
    p.group = a.n_head / layer->n_head_kv;
    const auto s = static_cast<cudaStream_t>(stream);
    if (a.dtype == SKV_DTYPE_F16) launch<__half>(p, layer->head_dim, layer->format == SKV_KV_INT8, s);
    else launch<__nv_bfloat16>(p, layer->head_dim, layer->format == SKV_KV_INT8, s);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SKV_OK : cuda_fail(e, "skv_decode_attention");
}

}  // extern "C"

// skv_delta.cu - skv_gated_delta: the gated delta rule on the fp32 state rows of linear-attention layers.
//
//   S <- e^g S;   d = beta (v - k^T S);   S <- S + k d^T;   out = scale * S^T q
//
// token_kernel runs it token by token.  The value columns of S never meet, so a CTA takes one head's slice of
// kSlice of them (128 threads, 8 rows x 4 columns each at head_dim 128, in registers from its first token to its last).
// One pass over the slice gives both k^T S and q^T S; the new output is q^T S + (q . k) d, so a token costs one
// reduction over the rows: two shuffles and one exchange between the four warps.  A single token is bound by the
// bytes of S, read and written once; 32 columns are 128 bytes of a row, whole lines.
#include "skv_ops.h"

#include <cmath>
#include <string>

namespace skv {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kSlice = 32;                       // value columns per CTA
constexpr int kGroups = kThreads / (kSlice / 4); // row groups: 16

struct DeltaDev {
    skv_gdn_args a;
    uint32_t* status;
    int ratio;   // value heads per key head
};

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads) token_kernel(const __grid_constant__ DeltaDev p) {
    constexpr int kRows = kDim / kGroups;        // rows of S per thread, kGroups apart
    constexpr int kSlices = kDim / kSlice;
    const skv_gdn_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slice = blockIdx.x % kSlices;
    const int64_t item = blockIdx.x / kSlices;
    const int head = (int) (item % a.n_v_heads), seq = (int) (item / a.n_v_heads);
    const int col = slice * kSlice + (tid & 7) * 4, row0 = tid >> 3;

    int begin = seq, end = seq + 1;
    if (a.seq_starts) {
        begin = min(max(__ldg(a.seq_starts + seq), 0), a.n_tokens);
        end = min(max(__ldg(a.seq_starts + seq + 1), begin), a.n_tokens);
        end = min(end, begin + a.max_tokens);
    }
    if (begin == end) return;
    const int64_t r = a.state_index ? __ldg(a.state_index + seq) : seq;
    if (r < 0 || r >= a.state_rows) {
        if (tid == 0) atomicOr(p.status, SKV_STATUS_BAD_STATE_ROW);
        return;
    }
    float* state = a.state + r * a.state_stride + (int64_t) head * kDim * kDim;
    float4 s[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) s[i] = *reinterpret_cast<const float4*>(state + (row0 + i * kGroups) * kDim + col);

    __shared__ float s_q[2][kDim], s_k[2][kDim];
    __shared__ float4 s_part[2][kWarps][8][2];
    __shared__ float s_qk[2][kWarps];
    const T* qh = static_cast<const T*>(a.q) + (head / p.ratio) * kDim;
    const T* kh = static_cast<const T*>(a.k) + (head / p.ratio) * kDim;
    for (int t = begin; t < end; ++t) {
        const int b = t & 1;   // two buffers: the next token's writes meet no reader of this one's
        if (tid < kDim) {
            s_q[b][tid] = (float) qh[(int64_t) t * a.q_stride + tid];
            s_k[b][tid] = (float) kh[(int64_t) t * a.k_stride + tid];
        }
        const float keep = expf(__ldg(a.g + (int64_t) t * a.g_stride + head));
        const float beta = __ldg(a.beta + (int64_t) t * a.beta_stride + head);
        const T* vr = static_cast<const T*>(a.v) + (int64_t) t * a.v_stride + head * kDim + col;
        const float2 v01 = Pair<T>::up(reinterpret_cast<const uint32_t*>(vr)[0]), v23 = Pair<T>::up(reinterpret_cast<const uint32_t*>(vr)[1]);
        __syncthreads();
        float4 ks = make_float4(0, 0, 0, 0), qs = ks;
        float qk = 0.0f;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const float k = s_k[b][row0 + i * kGroups], q = s_q[b][row0 + i * kGroups];
            s[i].x *= keep; s[i].y *= keep; s[i].z *= keep; s[i].w *= keep;
            ks.x = fmaf(k, s[i].x, ks.x); ks.y = fmaf(k, s[i].y, ks.y); ks.z = fmaf(k, s[i].z, ks.z); ks.w = fmaf(k, s[i].w, ks.w);
            qs.x = fmaf(q, s[i].x, qs.x); qs.y = fmaf(q, s[i].y, qs.y); qs.z = fmaf(q, s[i].z, qs.z); qs.w = fmaf(q, s[i].w, qs.w);
            qk = fmaf(k, q, qk);
        }
#pragma unroll
        for (int m = 8; m < 32; m <<= 1) {
            ks.x += __shfl_xor_sync(0xffffffffu, ks.x, m); ks.y += __shfl_xor_sync(0xffffffffu, ks.y, m);
            ks.z += __shfl_xor_sync(0xffffffffu, ks.z, m); ks.w += __shfl_xor_sync(0xffffffffu, ks.w, m);
            qs.x += __shfl_xor_sync(0xffffffffu, qs.x, m); qs.y += __shfl_xor_sync(0xffffffffu, qs.y, m);
            qs.z += __shfl_xor_sync(0xffffffffu, qs.z, m); qs.w += __shfl_xor_sync(0xffffffffu, qs.w, m);
            qk += __shfl_xor_sync(0xffffffffu, qk, m);
        }
        if (lane < 8) {
            s_part[b][warp][lane][0] = ks;
            s_part[b][warp][lane][1] = qs;
            if (lane == 0) s_qk[b][warp] = qk;
        }
        __syncthreads();
        ks = qs = make_float4(0, 0, 0, 0);
        qk = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float4 x = s_part[b][w][tid & 7][0], y = s_part[b][w][tid & 7][1];
            ks.x += x.x; ks.y += x.y; ks.z += x.z; ks.w += x.w;
            qs.x += y.x; qs.y += y.y; qs.z += y.z; qs.w += y.w;
            qk += s_qk[b][w];
        }
        const float4 d = make_float4(beta * (v01.x - ks.x), beta * (v01.y - ks.y), beta * (v23.x - ks.z), beta * (v23.y - ks.w));
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const float k = s_k[b][row0 + i * kGroups];
            s[i].x = fmaf(k, d.x, s[i].x); s[i].y = fmaf(k, d.y, s[i].y); s[i].z = fmaf(k, d.z, s[i].z); s[i].w = fmaf(k, d.w, s[i].w);
        }
        if (tid < 8) {
            uint2 o;
            o.x = Pair<T>::down(a.scale * fmaf(qk, d.x, qs.x), a.scale * fmaf(qk, d.y, qs.y));
            o.y = Pair<T>::down(a.scale * fmaf(qk, d.z, qs.z), a.scale * fmaf(qk, d.w, qs.w));
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (int64_t) t * a.out_stride + head * kDim + col) = o;
        }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) *reinterpret_cast<float4*>(state + (row0 + i * kGroups) * kDim + col) = s[i];
}

template <typename T>
void launch_tokens(const DeltaDev& p, cudaStream_t stream) {
    const unsigned grid = (unsigned) ((int64_t) p.a.n_seqs * p.a.n_v_heads * (p.a.head_dim / kSlice));
    if (p.a.head_dim == 64) token_kernel<T, 64><<<grid, kThreads, 0, stream>>>(p);
    else token_kernel<T, 128><<<grid, kThreads, 0, stream>>>(p);
}

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" {

int skv_gated_delta_workspace(int n_tokens, int n_seqs, int n_v_heads, int head_dim, int max_tokens, uint64_t* out_bytes) {
    if (!out_bytes) return fail(SKV_EINVAL, "skv_gated_delta_workspace: null output");
    *out_bytes = 0;
    if (n_tokens < 0 || n_seqs < 0 || n_v_heads < 1 || max_tokens < 0 || (head_dim != 64 && head_dim != 128))
        return fail(SKV_EINVAL, "skv_gated_delta_workspace: bad sizes");
    return SKV_OK;
}

int skv_gated_delta(const skv_gdn_args* args, void* stream) {
    const auto no = [](const char* why) { return fail(SKV_EINVAL, std::string("skv_gated_delta: ") + why); };
    if (!args) return no("no arguments");
    const skv_gdn_args& a = *args;
    if (a.n_tokens < 0 || a.n_seqs < 0 || a.max_tokens < 0) return no("negative counts");
    if (a.head_dim != 64 && a.head_dim != 128) return no("head_dim must be 64 or 128");
    if (a.n_k_heads < 1 || a.n_v_heads < 1 || a.n_v_heads > 4096 || a.n_v_heads % a.n_k_heads)
        return no("n_v_heads must be a multiple of n_k_heads, at most 4096");
    if (a.dtype != SKV_DTYPE_F16 && a.dtype != SKV_DTYPE_BF16) return no("unknown dtype");
    if (!(a.scale > -INFINITY && a.scale < INFINITY)) return no("the scale must be finite");
    if (!a.seq_starts && a.n_tokens != a.n_seqs) return no("without seq_starts every sequence has one token");
    if ((int64_t) a.n_seqs * a.n_v_heads > INT32_MAX / 4) return fail(SKV_ERANGE, "skv_gated_delta: too many sequences and heads");
    if (a.n_seqs == 0 || a.n_tokens == 0 || a.max_tokens == 0) return SKV_OK;
    if (!a.q || !a.k || !a.v || !a.out || !a.g || !a.beta || !a.state) return no("missing buffer");
    if (!ops_aligned16(a.q) || !ops_aligned16(a.k) || !ops_aligned16(a.v) || !ops_aligned16(a.out) || !ops_aligned16(a.state))
        return no("q, k, v, out and state must be 16-byte aligned");
    if (a.q_stride % 8 || a.k_stride % 8 || a.v_stride % 8 || a.out_stride % 8 || a.state_stride % 4)
        return no("strides must be multiples of 8 elements (4 floats for the state)");
    const int64_t kw = (int64_t) a.n_k_heads * a.head_dim, vw = (int64_t) a.n_v_heads * a.head_dim;
    if (a.n_tokens > 1 && (a.q_stride < kw || a.k_stride < kw || a.v_stride < vw || a.out_stride < vw))
        return no("a stride is shorter than its row");
    if (a.state_rows < 1 || (a.state_rows > 1 && a.state_stride < vw * a.head_dim)) return no("the state rows overlap or are none");
    if (!a.state_index && a.state_rows < a.n_seqs) return no("fewer state rows than sequences");
    uint64_t need = 0;
    if (const int rc = skv_gated_delta_workspace(a.n_tokens, a.n_seqs, a.n_v_heads, a.head_dim, a.max_tokens, &need)) return rc;
    if (need && (!a.workspace || (reinterpret_cast<uintptr_t>(a.workspace) & 255u) || a.workspace_bytes < need))
        return no("the workspace must be 256-byte aligned and as large as skv_gated_delta_workspace says");
    DeviceCtx* ctx = current_ctx();
    if (!ctx) return SKV_ECUDA;
    if (!ops_own_memory(a.state, ctx->device)) return no("the state is not memory of the current device");
    DeltaDev p{};
    p.a = a;
    p.status = ctx->status;
    p.ratio = a.n_v_heads / a.n_k_heads;
    const auto s = static_cast<cudaStream_t>(stream);
    if (a.dtype == SKV_DTYPE_F16) launch_tokens<__half>(p, s);
    else launch_tokens<__nv_bfloat16>(p, s);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SKV_OK : cuda_fail(e, "skv_gated_delta");
}

}  // extern "C"

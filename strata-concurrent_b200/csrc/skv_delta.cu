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
#include <type_traits>

namespace skv {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kSlice = 32;                       // value columns per CTA
constexpr int kGroups = kThreads / (kSlice / 4); // row groups: 16
constexpr int kChunksFrom = 32;                  // tokens of the longest sequence

struct DeltaDev {
    skv_gdn_args a;
    uint32_t* status;
    int ratio;   // value heads per key head
};

/// The tokens [begin, end) of a sequence; false when it has none.
__device__ __forceinline__ bool tokens_of(const skv_gdn_args& a, int seq, int& begin, int& end) {
    begin = seq;
    end = seq + 1;
    if (a.seq_starts) {
        begin = min(max(__ldg(a.seq_starts + seq), 0), a.n_tokens);
        end = min(max(__ldg(a.seq_starts + seq + 1), begin), a.n_tokens);
        if (end - begin > a.max_tokens) end = begin + a.max_tokens;
    }
    return begin < end;
}
/// A sequence's state of one head; null (and the status bit) when its row lies outside of the state.
__device__ __forceinline__ float* state_of(const DeltaDev& p, int seq, int head, int dim) {
    const int64_t r = p.a.state_index ? __ldg(p.a.state_index + seq) : seq;
    if (r < 0 || r >= p.a.state_rows) {
        if (threadIdx.x == 0) atomicOr(p.status, SKV_STATUS_BAD_STATE_ROW);
        return nullptr;
    }
    return p.a.state + r * p.a.state_stride + (int64_t) head * dim * dim;
}

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

    int begin, end;
    if (!tokens_of(a, seq, begin, end)) return;
    float* const state = state_of(p, seq, head, kDim);
    if (!state) return;
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

// ---------------------------------------------------------------- chunks of 64 tokens
//
// With G_i the sum of g over a chunk's tokens up to i, and S the state before it:
//     (I + A) V' = beta (V - e^G K S),   A_ij = beta_i e^(G_i - G_j) k_i . k_j  (j < i)
//     O  = scale (e^G Q S + P V'),       P_ij = e^(G_i - G_j) q_i . k_j         (j <= i)
//     S <- e^(G_63) S + K^T (e^(G_63 - G) V')
// A CTA takes one head's slice of 16 kConsumers value columns through all of its sequence's chunks.  Four producer warps
// stay one chunk ahead: they stage K, Q and V, and work out P and T = (I + A)^-1, which need no state.  Each consumer warp
// holds the transposed state of 16 columns in its accumulators and runs the recurrence alone: what a product leaves in
// accumulators is the left operand of the next (S^T K^T, then V'^T = R^T T^T, then S^T += V'^T K), so nothing of
// the chain passes through memory.  The chain bounds a single long sequence, so the slices are narrow when few CTAs
// would run (2 consumers: 128 CTAs for 32 heads), wider when there are more than fill the GPU (4).
//
// Precision.  Every product is fp16 with 32-bit sums.  A 32-bit operand (S, R, V', T) enters as the sum of two fp16 values
// after scaling by a power of two that puts the largest near 2^14: 22 bits, and 2^-39 of the largest at least; the state
// therefore keeps 32-bit quality.  Only what goes to the 16-bit output alone (Q S, P V') takes the first of the two.  K and Q
// are exact: fp16 as they are, bfloat16 scaled by a power of two (K by one per chunk, Q by one per row), up to values
// 2^-24 of the largest.  The sums G are taken in 64 bits, so that a decay of e^-200 in a chunk (deeper ones are as good
// as that) leaves the others' differences exact.

constexpr int kChunk = 64;
constexpr int kProducers = 4;
constexpr int kProducerThreads = kProducers * 32;
constexpr int kScratch = 68;          // floats between rows of the 32-bit scratch matrices
constexpr float kInverseScale = 1024.0f;   // T's entries are at most about 1: their fp16 parts keep clear of subnormals

__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, bool on) {   // off: zeros, nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <int kThreadsOf>
__device__ __forceinline__ void meet(int id) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kThreadsOf) : "memory");
}
template <int kThreadsOf>
__device__ __forceinline__ void pass(int id) {
    asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kThreadsOf) : "memory");
}
__device__ __forceinline__ float power_of_two(int e) {   // e clamped to the normal numbers
    return __int_as_float((min(max(e, -126), 127) + 127) << 23);
}
__device__ __forceinline__ int exponent_of(float x) {    // floor(log2 |x|); -127 for zero and subnormals
    return ((__float_as_int(x) >> 23) & 0xff) - 127;
}
/// The power that puts values of at most `top` near 2^14 when they are divided by it.  Within the range in which its
/// reciprocal and products of two such powers with fp16 values are normal numbers: values below 2^-106 may lose bits.
__device__ __forceinline__ int power_for(float top) { return max(exponent_of(top) - 14, -120); }
/// The largest magnitude in the warp (an infinity or a NaN counts as the largest).
__device__ __forceinline__ float warp_largest(float x) {
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x) & 0x7fffffffu));
}
/// The 16-byte chunk `chunk` of row `row`, swizzled so that eight rows' equal chunks lie in eight bank groups.
template <int kChunks>
__device__ __forceinline__ uint32_t chunk_at(int row, int chunk) {
    return (uint32_t) (row * kChunks + (kChunks >= 8 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3))) * 16u;
}
/// x and y as the sum of two pairs of fp16 values.
__device__ __forceinline__ void split(float x, float y, uint32_t& high, uint32_t& low) {
    high = Pair<__half>::down(x, y);
    const float2 h = Pair<__half>::up(high);
    low = Pair<__half>::down(x - h.x, y - h.y);
}

/// Per token of a chunk, for the consumers.
struct Factors {
    float value[kChunk];    // 2^F beta
    float key[kChunk];      // 2^2F beta e^G
    float query[kChunk];    // e^G
    float out[kChunk];      // scale 2^(the query row's power)
    float update[kChunk];   // e^(G_63 - G)
    float whole;            // e^(G_63)
};

template <int kDim, int kConsumers>
struct ChunkRoom {
    static constexpr int kTileBytes = kChunk * kDim * 2, kValueBytes = kChunk * kConsumers * 32, kSquareBytes = kChunk * kChunk * 2;
    struct Buffer {
        alignas(128) uint8_t k[kTileBytes], q[kTileBytes], v[kValueBytes], t_high[kSquareBytes], t_low[kSquareBytes], mix[kSquareBytes];
        Factors f;
    };
    Buffer buffer[2];
    float a[kChunk * kScratch], t[kChunk * kScratch], x[kChunk / 2 * kScratch];
    double sums[kChunk];
    float beta[kChunk];
    float largest[kProducers];
};

template <typename T, int kDim, int kConsumers>
__device__ __forceinline__ void produce(const DeltaDev& p, ChunkRoom<kDim, kConsumers>& room, int begin, int end, int head, int slice) {
    constexpr int kAll = kProducerThreads + kConsumers * 32, kChunks = kDim / 8, kMine = kChunk * kChunks / kProducerThreads;
    constexpr int kValueChunks = kConsumers * 2;
    const skv_gdn_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const T* qh = static_cast<const T*>(a.q) + (head / p.ratio) * kDim;
    const T* kh = static_cast<const T*>(a.k) + (head / p.ratio) * kDim;
    const T* vh = static_cast<const T*>(a.v) + head * kDim + slice * kConsumers * 16;
    uint4 next_k[kMine], next_q[kMine];
    float next_g = 0.0f, next_beta = 0.0f;
    const auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int at = i * kProducerThreads + tid, r = at / kChunks, chunk = at % kChunks;
            const bool on = t0 + r < end;
            const int64_t t = on ? t0 + r : begin;
            next_k[i] = on ? __ldg(reinterpret_cast<const uint4*>(kh + t * a.k_stride + chunk * 8)) : make_uint4(0, 0, 0, 0);
            next_q[i] = on ? __ldg(reinterpret_cast<const uint4*>(qh + t * a.q_stride + chunk * 8)) : make_uint4(0, 0, 0, 0);
        }
        if (tid < kChunk) {
            const bool on = t0 + tid < end;
            next_g = on ? __ldg(a.g + (int64_t) (t0 + tid) * a.g_stride + head) : 0.0f;
            next_beta = on ? __ldg(a.beta + (int64_t) (t0 + tid) * a.beta_stride + head) : 0.0f;
        }
    };
    fetch(begin);
    int b = 0;
    for (int t0 = begin, n = 0; t0 < end; t0 += kChunk, ++n, b ^= 1) {
        auto& buf = room.buffer[b];
        if (n >= 2) meet<kAll>(3 + b);   // the consumers are done with this buffer
        // ---- V of the slice as it is; K and Q as fp16
        for (int at = tid; at < kChunk * kValueChunks; at += kProducerThreads) {
            const int r = at / kValueChunks, chunk = at % kValueChunks;
            const bool on = t0 + r < end;
            copy_async16(smem_at(buf.v) + chunk_at<kValueChunks>(r, chunk), vh + (int64_t) (on ? t0 + r : begin) * a.v_stride + chunk * 8, on);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        int key_power = 0;
        if constexpr (!std::is_same<T, __half>::value) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                float x[8];
                unpack8<T>(next_k[i], x);
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]));
            }
            top = warp_largest(top);
            if (lane == 0) room.largest[warp] = top;
            meet<kProducerThreads>(5);
            top = fmaxf(fmaxf(room.largest[0], room.largest[1]), fmaxf(room.largest[2], room.largest[3]));
            key_power = top > 0.0f && top < INFINITY ? min(max(exponent_of(top), -60), 60) : 0;
        }
        const float key_down = power_of_two(-key_power);
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int at = i * kProducerThreads + tid, r = at / kChunks, chunk = at % kChunks;
            uint4 k = next_k[i], q = next_q[i];
            int power = 0;
            if constexpr (!std::is_same<T, __half>::value) {
                float x[8], top = 0.0f;
                unpack8<T>(k, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= key_down;
                k = pack8<__half>(x);
                unpack8<T>(q, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]));
#pragma unroll
                for (int m = 1; m < kChunks; m <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
                power = top > 0.0f && top < INFINITY ? min(max(exponent_of(top), -126), 126) : 0;
                const float down = power_of_two(-power);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= down;
                q = pack8<__half>(x);
            }
            *reinterpret_cast<uint4*>(buf.k + chunk_at<kChunks>(r, chunk)) = k;
            *reinterpret_cast<uint4*>(buf.q + chunk_at<kChunks>(r, chunk)) = q;
            if (chunk == 0) buf.f.out[r] = a.scale * power_of_two(power);
        }
        // ---- the decays: warp 0, two tokens a lane, sums in 64 bits
        if (tid < kChunk) {
            room.sums[tid] = next_g < -200.0f ? -200.0 : (double) next_g;
            room.beta[tid] = next_beta;
        }
        meet<kProducerThreads>(5);
        if (warp == 0) {
            const double x = room.sums[2 * lane], y = room.sums[2 * lane + 1];
            double up = x + y;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const double o = __shfl_up_sync(0xffffffffu, up, d);
                if (lane >= d) up += o;
            }
            const double all = __shfl_sync(0xffffffffu, up, 31);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int t = 2 * lane + h;
                const double sum = h ? up : up - y;
                const float into = expf((float) sum), beta = room.beta[t], fit = power_of_two(key_power);
                room.sums[t] = sum;
                buf.f.value[t] = fit * beta;
                buf.f.key[t] = fit * fit * beta * into;
                buf.f.query[t] = into;
                buf.f.update[t] = expf((float) (all - sum));
                if (t == 0) buf.f.whole = expf((float) all);
            }
        }
        if (t0 + kChunk < end) fetch(t0 + kChunk);
        meet<kProducerThreads>(5);
        // ---- K K^T and Q K^T of 16 tokens per warp, up to the diagonal; A (32 bits) and P (fp16)
        {
            float kk[8][4], qk[8][4];
#pragma unroll
            for (int t = 0; t < 8; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) kk[t][j] = qk[t][j] = 0.0f;
            const uint32_t k_at = smem_at(buf.k), q_at = smem_at(buf.q);
#pragma unroll
            for (int i = 0; i < kDim / 16; ++i) {
                uint32_t x[4], y[4];
                load_matrices(x, k_at + chunk_at<kChunks>(warp * 16 + (lane & 15), 2 * i + (lane >> 4)));
                load_matrices(y, q_at + chunk_at<kChunks>(warp * 16 + (lane & 15), 2 * i + (lane >> 4)));
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if (t <= warp) {
                        uint32_t m[4];
                        load_matrices(m, k_at + chunk_at<kChunks>(t * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * i + ((lane >> 3) & 1)));
                        multiply(kk[2 * t], x, m[0], m[1]);
                        multiply(kk[2 * t + 1], x, m[2], m[3]);
                        multiply(qk[2 * t], y, m[0], m[1]);
                        multiply(qk[2 * t + 1], y, m[2], m[3]);
                    }
                }
            }
            const float fit = power_of_two(key_power), fit2 = fit * fit;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = warp * 16 + g + h * 8;
                const double sum = room.sums[row];
                const float by = fit2 * room.beta[row];
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    if (t < 2 * warp + 2) {
                        const int col = t * 8 + 2 * c;
                        const float d0 = col <= row ? expf((float) (sum - room.sums[col])) : 0.0f;
                        const float d1 = col + 1 <= row ? expf((float) (sum - room.sums[col + 1])) : 0.0f;
                        // a decay of zero wipes out even an infinite product
                        *reinterpret_cast<float2*>(&room.a[row * kScratch + col]) =
                            make_float2(col < row ? by * d0 * kk[t][2 * h] : 0.0f, col + 1 < row ? by * d1 * kk[t][2 * h + 1] : 0.0f);
                        *reinterpret_cast<uint32_t*>(buf.mix + chunk_at<8>(row, t) + c * 4) =
                            Pair<__half>::down(col <= row ? d0 * qk[t][2 * h] : 0.0f, col + 1 <= row ? d1 * qk[t][2 * h + 1] : 0.0f);
                    }
                }
            }
        }
        meet<kProducerThreads>(5);
        // ---- T = (I + A)^-1: the diagonal blocks of 16 by substitution, a column per thread
        if (tid < kChunk) {
            const int base = tid & ~15, col = tid & 15;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float r[16];
#pragma unroll
                for (int j = 0; j < (i + 3) / 4; ++j)
                    *reinterpret_cast<float4*>(&r[4 * j]) = *reinterpret_cast<const float4*>(&room.a[(base + i) * kScratch + base + 4 * j]);
                float s0 = i == col ? 1.0f : 0.0f, s1 = 0.0f;
#pragma unroll
                for (int j = 0; j < i; ++j) {
                    if (j & 1) s1 = fmaf(-r[j], x[j], s1);
                    else s0 = fmaf(-r[j], x[j], s0);
                }
                x[i] = s0 + s1;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) room.t[(base + i) * kScratch + base + col] = x[i];
        }
        meet<kProducerThreads>(5);
        // below them, T21 = -T22 (A21 T11): blocks of 16 in each half, then the block of 32
        {
            const int half_at = (tid >> 6) * 32, r = (tid & 63) >> 2, col = (tid & 3) * 4;
            float4 s = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const float w = room.a[(half_at + 16 + r) * kScratch + half_at + k];
                const float4 y = *reinterpret_cast<const float4*>(&room.t[(half_at + k) * kScratch + half_at + col]);
                s.x = fmaf(w, y.x, s.x); s.y = fmaf(w, y.y, s.y); s.z = fmaf(w, y.z, s.z); s.w = fmaf(w, y.w, s.w);
            }
            *reinterpret_cast<float4*>(&room.x[r * kScratch + (tid >> 6) * 16 + col]) = s;
            meet<kProducerThreads>(5);
            s = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const float w = -room.t[(half_at + 16 + r) * kScratch + half_at + 16 + k];
                const float4 y = *reinterpret_cast<const float4*>(&room.x[k * kScratch + (tid >> 6) * 16 + col]);
                s.x = fmaf(w, y.x, s.x); s.y = fmaf(w, y.y, s.y); s.z = fmaf(w, y.z, s.z); s.w = fmaf(w, y.w, s.w);
            }
            *reinterpret_cast<float4*>(&room.t[(half_at + 16 + r) * kScratch + half_at + col]) = s;
            // above the diagonal blocks of each half the sums below read zeros
            *reinterpret_cast<float4*>(&room.t[(half_at + r) * kScratch + half_at + 16 + col]) = make_float4(0, 0, 0, 0);
            meet<kProducerThreads>(5);
        }
        {
            const int r = tid >> 2, col = (tid & 3) * 8;
            float4 s = make_float4(0, 0, 0, 0), u = s;
#pragma unroll 8
            for (int k = 0; k < 32; ++k) {
                const float w = room.a[(32 + r) * kScratch + k];
                const float4 y = *reinterpret_cast<const float4*>(&room.t[k * kScratch + col]);
                const float4 z = *reinterpret_cast<const float4*>(&room.t[k * kScratch + col + 4]);
                s.x = fmaf(w, y.x, s.x); s.y = fmaf(w, y.y, s.y); s.z = fmaf(w, y.z, s.z); s.w = fmaf(w, y.w, s.w);
                u.x = fmaf(w, z.x, u.x); u.y = fmaf(w, z.y, u.y); u.z = fmaf(w, z.z, u.z); u.w = fmaf(w, z.w, u.w);
            }
            *reinterpret_cast<float4*>(&room.x[r * kScratch + col]) = s;
            *reinterpret_cast<float4*>(&room.x[r * kScratch + col + 4]) = u;
            meet<kProducerThreads>(5);
            s = u = make_float4(0, 0, 0, 0);
#pragma unroll 8
            for (int k = 0; k < 32; ++k) {
                const float w = -room.t[(32 + r) * kScratch + 32 + k];
                const float4 y = *reinterpret_cast<const float4*>(&room.x[k * kScratch + col]);
                const float4 z = *reinterpret_cast<const float4*>(&room.x[k * kScratch + col + 4]);
                s.x = fmaf(w, y.x, s.x); s.y = fmaf(w, y.y, s.y); s.z = fmaf(w, y.z, s.z); s.w = fmaf(w, y.w, s.w);
                u.x = fmaf(w, z.x, u.x); u.y = fmaf(w, z.y, u.y); u.z = fmaf(w, z.z, u.z); u.w = fmaf(w, z.w, u.w);
            }
            *reinterpret_cast<float4*>(&room.t[(32 + r) * kScratch + col]) = s;
            *reinterpret_cast<float4*>(&room.t[(32 + r) * kScratch + col + 4]) = u;
            meet<kProducerThreads>(5);
        }
        // ---- T in two fp16 parts; the blocks above the diagonal blocks are not read
#pragma unroll
        for (int i = 0; i < kChunk * 8 / kProducerThreads; ++i) {
            const int at = i * kProducerThreads + tid, r = at >> 3, chunk = at & 7;
            if (chunk / 2 <= r / 16) {
                uint32_t high[4], low[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 x = *reinterpret_cast<const float2*>(&room.t[r * kScratch + chunk * 8 + 2 * j]);
                    split(x.x * kInverseScale, x.y * kInverseScale, high[j], low[j]);
                }
                *reinterpret_cast<uint4*>(buf.t_high + chunk_at<8>(r, chunk)) = make_uint4(high[0], high[1], high[2], high[3]);
                *reinterpret_cast<uint4*>(buf.t_low + chunk_at<8>(r, chunk)) = make_uint4(low[0], low[1], low[2], low[3]);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        pass<kAll>(1 + b);   // the buffer is full
    }
}

template <typename T, int kDim, int kConsumers>
__device__ __forceinline__ void consume(const DeltaDev& p, ChunkRoom<kDim, kConsumers>& room, int begin, int end, int head, int slice, float* state) {
    constexpr int kAll = kProducerThreads + kConsumers * 32, kChunks = kDim / 8, kValueChunks = kConsumers * 2;
    const skv_gdn_args& a = p.a;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - kProducers, g = lane >> 2, c = lane & 3;
    const int col0 = (slice * kConsumers + warp) * 16;   // the warp's value columns
    // S^T: rows (value columns) g, g + 8; columns (keys) 8 i + 2c, 2c + 1
    float s[kDim / 8][4];
#pragma unroll
    for (int i = 0; i < kDim / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = state[(i * 8 + 2 * c + (j & 1)) * kDim + col0 + g + (j >> 1) * 8];
    T* out = static_cast<T*>(a.out) + head * kDim + col0 + 2 * c;
    int b = 0;
    for (int t0 = begin; t0 < end; t0 += kChunk, b ^= 1) {
        const auto& buf = room.buffer[b];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < kDim / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(s[i][j]));
        const int s_power = power_for(warp_largest(top));
        const float s_down = power_of_two(-s_power), s_up = power_of_two(s_power);
        meet<kAll>(1 + b);       // the buffer is full
        // ---- S^T K^T and S^T Q^T
        float ks[8][4], o[8][4];
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) ks[t][j] = o[t][j] = 0.0f;
        const uint32_t k_at = smem_at(buf.k), q_at = smem_at(buf.q);
#pragma unroll
        for (int i = 0; i < kDim / 16; ++i) {
            uint32_t high[4], low[4];
            split(s[2 * i][0] * s_down, s[2 * i][1] * s_down, high[0], low[0]);
            split(s[2 * i][2] * s_down, s[2 * i][3] * s_down, high[1], low[1]);
            split(s[2 * i + 1][0] * s_down, s[2 * i + 1][1] * s_down, high[2], low[2]);
            split(s[2 * i + 1][2] * s_down, s[2 * i + 1][3] * s_down, high[3], low[3]);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                uint32_t m[4];
                const uint32_t at = chunk_at<kChunks>(t * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * i + ((lane >> 3) & 1));
                load_matrices(m, k_at + at);
                multiply(ks[2 * t], high, m[0], m[1]);
                multiply(ks[2 * t + 1], high, m[2], m[3]);
                multiply(ks[2 * t], low, m[0], m[1]);
                multiply(ks[2 * t + 1], low, m[2], m[3]);
                load_matrices(m, q_at + at);
                multiply(o[2 * t], high, m[0], m[1]);
                multiply(o[2 * t + 1], high, m[2], m[3]);
            }
        }
        // ---- R = beta (V - e^G K S), in place of K S
        top = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            uint32_t m[4];
            load_matrices_t(m, smem_at(buf.v) + chunk_at<kValueChunks>(t * 16 + (lane & 7) + ((lane >> 4) << 3), warp * 2 + ((lane >> 3) & 1)));
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int at = (2 * t + u) * 8 + 2 * c;
                const float2 fv = *reinterpret_cast<const float2*>(&buf.f.value[at]);
                float2 fk = *reinterpret_cast<const float2*>(&buf.f.key[at]);
                fk.x *= s_up;
                fk.y *= s_up;
                const float2 v0 = Pair<T>::up(m[2 * u]), v1 = Pair<T>::up(m[2 * u + 1]);
                float (&r)[4] = ks[2 * t + u];
                r[0] = fv.x * v0.x - fk.x * r[0];
                r[1] = fv.y * v0.y - fk.y * r[1];
                r[2] = fv.x * v1.x - fk.x * r[2];
                r[3] = fv.y * v1.y - fk.y * r[3];
#pragma unroll
                for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(r[j]));
            }
        }
        const int r_power = power_for(warp_largest(top));
        const float r_down = power_of_two(-r_power);
        // ---- V' = T R
        float v[8][4];
        {
            uint32_t high[4][4], low[4][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    split(ks[2 * t + (j >> 1)][2 * (j & 1)] * r_down, ks[2 * t + (j >> 1)][2 * (j & 1) + 1] * r_down, high[t][j], low[t][j]);
            }
#pragma unroll
            for (int t = 0; t < 8; ++t) v[t][0] = v[t][1] = v[t][2] = v[t][3] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int t = i; t < 4; ++t) {
                    uint32_t m[4];
                    const uint32_t at = chunk_at<8>(t * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * i + ((lane >> 3) & 1));
                    load_matrices(m, smem_at(buf.t_high) + at);
                    multiply(v[2 * t], high[i], m[0], m[1]);
                    multiply(v[2 * t + 1], high[i], m[2], m[3]);
                    multiply(v[2 * t], low[i], m[0], m[1]);
                    multiply(v[2 * t + 1], low[i], m[2], m[3]);
                    load_matrices(m, smem_at(buf.t_low) + at);
                    multiply(v[2 * t], high[i], m[0], m[1]);
                    multiply(v[2 * t + 1], high[i], m[2], m[3]);
                }
            }
        }
        const int v_unit = r_power - 10;   // V' = 2^v_unit v
        // ---- S <- e^(G_63) S + K^T (e^(G_63 - G) V')
        uint32_t first[4][4];              // V' as it enters the output
        int o_power;
        {
            top = 0.0f;
            float most = 0.0f;
            float w[8][4];
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const float2 f = *reinterpret_cast<const float2*>(&buf.f.update[t * 8 + 2 * c]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[t][j] = v[t][j] * (j & 1 ? f.y : f.x);
                    top = fmaxf(top, fabsf(w[t][j]));
                    most = fmaxf(most, fabsf(v[t][j]));
                }
            }
            // one power for S and the update: the update's, or 2^-60 of what S would need where the update is smaller yet
            int w_power = exponent_of(warp_largest(top)) - 14 + v_unit;
            w_power = min(max(w_power, max(s_power - 60, -120)), 120);
            o_power = min(max(exponent_of(warp_largest(most)) - 14 + v_unit, max(s_power - 60, -120)), 120);
            const float w_down = power_of_two(v_unit - w_power), v_down = power_of_two(v_unit - o_power);
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    first[t][j] = Pair<__half>::down(v[2 * t + (j >> 1)][2 * (j & 1)] * v_down, v[2 * t + (j >> 1)][2 * (j & 1) + 1] * v_down);
            const float keep = buf.f.whole * power_of_two(-w_power), up = power_of_two(w_power);
#pragma unroll
            for (int i = 0; i < kDim / 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][j] *= keep;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                uint32_t high[4], low[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    split(w[2 * t + (j >> 1)][2 * (j & 1)] * w_down, w[2 * t + (j >> 1)][2 * (j & 1) + 1] * w_down, high[j], low[j]);
#pragma unroll
                for (int i = 0; i < kDim / 16; ++i) {
                    uint32_t m[4];
                    load_matrices_t(m, k_at + chunk_at<kChunks>(t * 16 + (lane & 15), 2 * i + (lane >> 4)));
                    multiply(s[2 * i], high, m[0], m[1]);
                    multiply(s[2 * i + 1], high, m[2], m[3]);
                    multiply(s[2 * i], low, m[0], m[1]);
                    multiply(s[2 * i + 1], low, m[2], m[3]);
                }
            }
#pragma unroll
            for (int i = 0; i < kDim / 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][j] *= up;
        }
        // ---- O = scale (e^G Q S + P V')
        const float o_fit = power_of_two(s_power - o_power), o_up = power_of_two(o_power);
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const float2 f = *reinterpret_cast<const float2*>(&buf.f.query[t * 8 + 2 * c]);
            o[t][0] *= f.x * o_fit;
            o[t][1] *= f.y * o_fit;
            o[t][2] *= f.x * o_fit;
            o[t][3] *= f.y * o_fit;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int t = i; t < 4; ++t) {
                uint32_t m[4];
                load_matrices(m, smem_at(buf.mix) + chunk_at<8>(t * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * i + ((lane >> 3) & 1)));
                multiply(o[2 * t], first[i], m[0], m[1]);
                multiply(o[2 * t + 1], first[i], m[2], m[3]);
            }
        }
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            float2 f = *reinterpret_cast<const float2*>(&buf.f.out[t * 8 + 2 * c]);
            f.x *= o_up;
            f.y *= o_up;
            const uint32_t lo = transpose8(Pair<T>::down(o[t][0] * f.x, o[t][1] * f.y));
            const uint32_t hi = transpose8(Pair<T>::down(o[t][2] * f.x, o[t][3] * f.y));
            const int token = t0 + t * 8 + g;
            if (token < end) {
                *reinterpret_cast<uint32_t*>(out + (int64_t) token * a.out_stride) = lo;
                *reinterpret_cast<uint32_t*>(out + (int64_t) token * a.out_stride + 8) = hi;
            }
        }
        if (t0 + 2 * kChunk < end) pass<kAll>(3 + b);   // the buffer may be filled again
    }
#pragma unroll
    for (int i = 0; i < kDim / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) state[(i * 8 + 2 * c + (j & 1)) * kDim + col0 + g + (j >> 1) * 8] = s[i][j];
}

template <typename T, int kDim, int kConsumers>
__global__ void __launch_bounds__(kProducerThreads + kConsumers * 32, 1) chunk_kernel(const __grid_constant__ DeltaDev p) {
    extern __shared__ __align__(128) uint8_t smem[];
    auto& room = *reinterpret_cast<ChunkRoom<kDim, kConsumers>*>(smem);
    constexpr int kSlices = kDim / (kConsumers * 16);
    const skv_gdn_args& a = p.a;
    const int slice = blockIdx.x % kSlices;
    const int64_t item = blockIdx.x / kSlices;
    const int head = (int) (item % a.n_v_heads), seq = (int) (item / a.n_v_heads);
    int begin, end;
    if (!tokens_of(a, seq, begin, end)) return;
    float* const state = state_of(p, seq, head, kDim);
    if (!state) return;
    if (threadIdx.x < kProducerThreads) produce<T, kDim, kConsumers>(p, room, begin, end, head, slice);
    else consume<T, kDim, kConsumers>(p, room, begin, end, head, slice, state);
}

template <typename T>
cudaError_t launch_tokens(const DeltaDev& p, cudaStream_t stream) {
    const unsigned grid = (unsigned) ((int64_t) p.a.n_seqs * p.a.n_v_heads * (p.a.head_dim / kSlice));
    if (p.a.head_dim == 64) token_kernel<T, 64><<<grid, kThreads, 0, stream>>>(p);
    else token_kernel<T, 128><<<grid, kThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

template <typename T, int kDim, int kConsumers>
cudaError_t launch_chunks(const DeltaDev& p, cudaStream_t stream) {
    constexpr int kSmem = sizeof(ChunkRoom<kDim, kConsumers>);
    static_assert(kSmem <= 227 * 1024, "the buffers fit an SM");
    const cudaError_t e = cudaFuncSetAttribute(chunk_kernel<T, kDim, kConsumers>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    const unsigned grid = (unsigned) ((int64_t) p.a.n_seqs * p.a.n_v_heads * (kDim / (kConsumers * 16)));
    chunk_kernel<T, kDim, kConsumers><<<grid, kProducerThreads + kConsumers * 32, kSmem, stream>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch(const DeltaDev& p, int sms, cudaStream_t stream) {
    if (p.a.max_tokens < kChunksFrom) return launch_tokens<T>(p, stream);
    const bool few = (int64_t) p.a.n_seqs * p.a.n_v_heads * (p.a.head_dim / 32) <= sms;
    if (p.a.head_dim == 64) return few ? launch_chunks<T, 64, 2>(p, stream) : launch_chunks<T, 64, 4>(p, stream);
    return few ? launch_chunks<T, 128, 2>(p, stream) : launch_chunks<T, 128, 4>(p, stream);
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
    const cudaError_t e = a.dtype == SKV_DTYPE_F16 ? launch<__half>(p, ctx->sms, s) : launch<__nv_bfloat16>(p, ctx->sms, s);
    return e == cudaSuccess ? SKV_OK : cuda_fail(e, "skv_gated_delta");
}

}  // extern "C"

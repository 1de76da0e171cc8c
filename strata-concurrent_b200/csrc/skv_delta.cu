// skv_delta.cu - skv_gated_delta: the gated delta rule on the fp32 state rows of linear-attention layers.
//
//   S <- e^g S;   d = beta (v - k^T S);   S <- S + k d^T;   out = scale * S^T q
//
// token_kernel runs it token by token.  The value columns of S never meet, so a CTA takes one head's slice of
// kSlice of them (128 threads, 8 rows x 4 columns each at head_dim 128, in registers from its first token to its last).
// One pass over the slice gives both k^T S and q^T S; the new output is q^T S + (q . k) d, so a token costs one
// reduction over the rows: two shuffles and one exchange between the four warps.  A single token is bound by the
// bytes of S, read and written once; 32 columns are 128 bytes of a row, whole lines.  64 sequences of 32 heads of 128, a
// token each: 44 us in a graph, 6.1 TB/s; one sequence 2.2 us.
#include "skv_ops.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstddef>
#include <string>
#include <type_traits>

namespace skv {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kSlice = 32;                       // value columns per CTA
constexpr int kGroups = kThreads / (kSlice / 4); // row groups: 16
// Chunks from so many tokens of the longest sequence on.  32 heads of 128, one sequence: 12.2 us for 16 tokens by tokens,
// 14.7 in a chunk (17.4 and 14.9 for 24); 8 sequences 39 and 32 (22 and 31 for 8 tokens), 32 sequences 121 and 92.
constexpr int kChunksFrom = 16;

struct Record;

struct DeltaDev {
    skv_gdn_args a;
    uint32_t* status;
    Record* records;   // [slot][value head], when the call runs in chunks
    int ratio;         // value heads per key head
    int ranked;        // longest sequences first
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
    wait_for_previous();

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
// What needs no state, P and T = (I + A)^-1 with the decays, is worked out first, for all chunks at once: prepare_kernel
// writes a record per chunk and head into the workspace.  Then chunk_kernel takes one head's slice of 16 kGroupsOf value
// columns through all chunks of its sequence.  Four loader warps stay a chunk ahead.  State warps hold the transposed state of
// 16 columns each in accumulators, alone or as a pair with a half of the keys each (kSplit).  Output warps turn the states
// and V' that those leave in shared memory into O.  What a product leaves in accumulators is the left operand of the next
// (S^T K^T, then V'^T = R^T T^T, then S^T += V'^T K), so the chain from chunk to chunk passes through memory once, where a
// pair's sums over the keys meet, or not at all.  That chain's latency, not the flops, bounds a long sequence: hence the pairs
// and slices of 32 columns where few CTAs would run, 4 state warps with a scheduler each; a whole head per CTA, whose
// 8 state warps share the copies and records, where there are more than fill the GPU.
//
// Measured, 32 heads of 128 on 16 key heads: one bfloat16 sequence of 32K tokens 1,623 us, 230 of them prepare_kernel (the
// chain takes 2.7 us a chunk; the bytes alone would take 125); 12 ragged fp16 sequences of 15,943 tokens in all 529 us (521
// before rows of P had powers of their own).
//
// Precision.  Every product is fp16 with 32-bit sums.  A 32-bit operand (S, R, V', T, A) enters as the sum of two fp16
// values after scaling by a power of two that puts the largest near 2^14: 22 bits, and 2^-39 of the largest at least (T:
// 2^-30 of 1); the state therefore keeps 32-bit quality.  The largest is that of a warp's 16 value columns, of S over its keys, of
// R and V' over the chunk's tokens: a power per column would keep a small column's bits beside large ones, but put four
// shuffles in place of one reduction into each of four searches on the chain.  What goes to the output alone (Q S, P V') takes the first of the two where that
// is bfloat16, eight times coarser; for fp16 outputs P and V' take both.  K and Q are exact: fp16 as they are, bfloat16
// scaled by a power of two (K by one per chunk, Q by one per row), up to values 2^-24 of the largest.  A row of P is scaled by
// a power of two that follows from the largest values of its query and of the chunk's keys: it neither overflows nor loses
// more than what lies 2^-39 below what its products could reach.  The sums G are taken
// in 64 bits and kept as two 32-bit parts, so that a decay of e^-200 in a chunk (deeper ones are as good as that) leaves the
// others' differences exact.

constexpr int kChunk = 64;
constexpr int kLoaders = 4;
constexpr int kLoaderThreads = kLoaders * 32;
constexpr int kScratch = 68;          // floats between rows of the 32-bit scratch matrices
// T's entries are about 1 at most for keys of about unit length: 2^5 of them leaves their two fp16 parts 30 bits below 1,
// and room for entries of 2,000 where keys differ in length.
constexpr int kInversePower = 5;
constexpr float kInverseScale = 1 << kInversePower;

__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, bool on) {   // off: zeros, nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
/// The same without ordering against other memory accesses but the barriers below: for code that meets by those alone and
/// reads what others wrote before them, so that its loads can run ahead.
__device__ __forceinline__ void peek_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void peek_matrices_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
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
/// The largest magnitude of an accumulator array, in four chains.
template <int kTiles>
__device__ __forceinline__ float largest_of(const float (&x)[kTiles][4]) {
    float top[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) top[j] = fmaxf(top[j], fabsf(x[i][j]));
    return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}
/// x and y as the sum of two pairs of fp16 values.
__device__ __forceinline__ void split(float x, float y, uint32_t& high, uint32_t& low) {
    high = Pair<__half>::down(x, y);
    const float2 h = Pair<__half>::up(high);
    low = Pair<__half>::down(x - h.x, y - h.y);
}

/// The eight rows of 16 tokens that a lane of the left and one of the right half of ldmatrix name: of a right operand
/// [token][key], and of its transpose.
__device__ __forceinline__ int right_row() { return (threadIdx.x & 7) + ((threadIdx.x >> 4) & 1) * 8; }
__device__ __forceinline__ int right_half() { return (threadIdx.x >> 3) & 1; }

/// Per token of a chunk.
struct Factors {
    float value[kChunk];    // 2^F beta
    float key[kChunk];      // 2^2F beta e^G
    float query[kChunk];    // e^G 2^-(the power of P's row)
    float out[kChunk];      // scale 2^(the query row's power and that of P's row)
    float update[kChunk];   // e^(G_63 - G)
    float down[kChunk];     // 2^-(the query row's power)
    float whole;            // e^(G_63)
    float key_down;         // 2^-F, F the power of the chunk's keys
    float pad[2];
};
/// What prepare_kernel leaves of a chunk and head: the ten blocks of 16 x 16 on and below the diagonal of T (in two fp16
/// parts, times kInverseScale) and of P, and the factors.
constexpr int kBlockBytes = 512, kTriangleBytes = 10 * kBlockBytes;
struct Record {
    uint8_t t_high[kTriangleBytes], t_low[kTriangleBytes], mix[kTriangleBytes];
    Factors f;
    uint8_t mix_low[kTriangleBytes];   // P's second part, for fp16 outputs alone
};
static_assert(sizeof(Record) % 16 == 0 && offsetof(Record, mix_low) % 16 == 0, "copied 16 bytes at a time");
__host__ __device__ constexpr int block_of(int i, int j) { return i * (i + 1) / 2 + j; }
/// The 16-byte half `chunk` of row `row` of a block, swizzled so that eight rows' equal halves lie in eight bank groups.
__device__ __forceinline__ uint32_t half_row_at(int row, int chunk) { return (uint32_t) (row * 2 + (chunk ^ ((row >> 2) & 1))) * 16u; }

/// The record slot of a sequence's first chunk: a sequence of n tokens from `begin` on takes ceil(n / 64) slots, at most
/// floor((begin + n) / 64) - floor(begin / 64) + 1, so sequence s starts at floor(begin / 64) + s.
__device__ __forceinline__ int64_t first_slot(int begin, int seq) { return begin / kChunk + seq; }

int64_t record_slots(int n_tokens, int n_seqs) { return (int64_t) n_tokens / kChunk + n_seqs; }
bool chunked(bool packed, int max_tokens) { return packed && max_tokens >= kChunksFrom; }

/// fp16 parts of the left operand (16 x 16) at `at` in a 32-bit scratch matrix.
__device__ __forceinline__ void left_parts(const float* at, float scale, uint32_t (&high)[4], uint32_t (&low)[4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 x = *reinterpret_cast<const float2*>(at + (g + (j & 1) * 8) * kScratch + 2 * c + (j >> 1) * 8);
        split(x.x * scale, x.y * scale, high[j], low[j]);
    }
}
/// ... and of the right operand (16 x 8).
__device__ __forceinline__ void right_parts(const float* at, float scale, uint32_t (&high)[2], uint32_t (&low)[2]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float* x = at + (2 * c + j * 8) * kScratch + g;
        split(x[0] * scale, x[kScratch] * scale, high[j], low[j]);
    }
}
__device__ __forceinline__ void multiply_parts(float (&c)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], const uint32_t (&bh)[2], const uint32_t (&bl)[2]) {
    multiply(c, ah, bl[0], bl[1]);
    multiply(c, al, bh[0], bh[1]);
    multiply(c, ah, bh[0], bh[1]);
}
__device__ __forceinline__ void store_product(float* at, float by, const float (&x)[4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    *reinterpret_cast<float2*>(at + g * kScratch + 2 * c) = make_float2(by * x[0], by * x[1]);
    *reinterpret_cast<float2*>(at + (g + 8) * kScratch + 2 * c) = make_float2(by * x[2], by * x[3]);
}

template <int kDim>
struct PrepareRoom {
    union {
        struct { uint8_t k[kChunk * kDim * 2], q[kChunk * kDim * 2]; } in;
        struct { float a[kChunk * kScratch], t[kChunk * kScratch]; } work;   // X lies in A's rows 0 - 31, columns 32 - 63, which hold nothing
    };
    alignas(16) uint8_t mix[kTriangleBytes];
    uint8_t mix_low[kTriangleBytes];
    float2 sums[kChunk];      // G log2 e in two parts
    float rest[kChunk];       // e^(G_r - G), r the last token of the same 16
    double carry[2];          // the first 32 tokens' sum, and all
    float beta[kChunk];
    int power[kChunk];        // of the query rows
    int mix_power[kChunk];    // of P's rows, beyond that of the query's
    float largest[4];
};

/// Blocks (kRow, kFrom), (kRow, kFrom + 1) .. of K K^T and Q K^T, two tiles of eight tokens each from tile kAt on.
template <int kDim, int kRow, int kFrom, int kBlocks, int kAt>
__device__ __forceinline__ void products(uint32_t k_at, uint32_t q_at, float (&kk)[6][4], float (&qk)[6][4]) {
    constexpr int kChunks = kDim / 8;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int t = 0; t < 2 * kBlocks; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) kk[kAt + t][j] = qk[kAt + t][j] = 0.0f;
#pragma unroll
    for (int i = 0; i < kDim / 16; ++i) {
        uint32_t x[4], y[4];
        load_matrices(x, k_at + chunk_at<kChunks>(kRow * 16 + (lane & 15), 2 * i + (lane >> 4)));
        load_matrices(y, q_at + chunk_at<kChunks>(kRow * 16 + (lane & 15), 2 * i + (lane >> 4)));
#pragma unroll
        for (int t = 0; t < kBlocks; ++t) {
            uint32_t m[4];
            load_matrices(m, k_at + chunk_at<kChunks>((kFrom + t) * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * i + ((lane >> 3) & 1)));
            multiply(kk[kAt + 2 * t], x, m[0], m[1]);
            multiply(kk[kAt + 2 * t + 1], x, m[2], m[3]);
            multiply(qk[kAt + 2 * t], y, m[0], m[1]);
            multiply(qk[kAt + 2 * t + 1], y, m[2], m[3]);
        }
    }
}
/// A (32 bits) and P (fp16) of those blocks.  Below the diagonal block a decay e^(G_i - G_j) is the product of e^(G_i - G_r)
/// and e^(G_r - G_j), r the last token of j's block: both at most 1, the second one per token.
template <int kDim, int kRow, int kFrom, int kBlocks, int kAt, bool kFine>
__device__ __forceinline__ void decayed(PrepareRoom<kDim>& room, float fit2, const float (&kk)[6][4], const float (&qk)[6][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int in = g + h * 8, row = kRow * 16 + in;
        const float2 sum = room.sums[row];
        const float by = fit2 * room.beta[row], down = power_of_two(-room.mix_power[row]);
#pragma unroll
        for (int u = 0; u < kBlocks; ++u) {
            const bool below = kFrom + u < kRow;
            const float2 ref = room.sums[(kFrom + u) * 16 + 15];
            const float part = below ? exp2f((sum.x - ref.x) + (sum.y - ref.y)) : 0.0f;
#pragma unroll
            for (int t = 2 * u; t < 2 * u + 2; ++t) {
                const int col = kFrom * 16 + t * 8 + 2 * c;
                float d0, d1;
                if (below) {
                    const float2 rest = *reinterpret_cast<const float2*>(&room.rest[col]);
                    d0 = part * rest.x;
                    d1 = part * rest.y;
                } else {
                    // above the diagonal a decay of zero wipes out even an infinite product
                    const float4 other = *reinterpret_cast<const float4*>(&room.sums[col]);   // of col and col + 1
                    d0 = exp2f((sum.x - other.x) + (sum.y - other.y));
                    d1 = exp2f((sum.x - other.z) + (sum.y - other.w));
                }
                const bool q0 = below || col <= row, q1 = below || col + 1 <= row, k0 = below || col < row, k1 = below || col + 1 < row;
                *reinterpret_cast<float2*>(&room.work.a[row * kScratch + col]) =
                    make_float2(k0 ? by * d0 * kk[kAt + t][2 * h] : 0.0f, k1 ? by * d1 * kk[kAt + t][2 * h + 1] : 0.0f);
                uint32_t high, low;
                split(q0 ? d0 * (down * qk[kAt + t][2 * h]) : 0.0f, q1 ? d1 * (down * qk[kAt + t][2 * h + 1]) : 0.0f, high, low);
                const uint32_t to = block_of(kRow, kFrom + u) * kBlockBytes + half_row_at(in, t & 1) + c * 4;
                *reinterpret_cast<uint32_t*>(room.mix + to) = high;
                if constexpr (kFine) *reinterpret_cast<uint32_t*>(room.mix_low + to) = low;
            }
        }
    }
}

/// One chunk of one key head, for all of its value heads: K, Q and their products serve them all.  Four warps; four CTAs
/// an SM hide the short phases' latencies.
template <typename T, int kDim>
__global__ void __launch_bounds__(kLoaderThreads, 4) prepare_kernel(const __grid_constant__ DeltaDev p) {
    extern __shared__ __align__(128) uint8_t smem[];
    auto& room = *reinterpret_cast<PrepareRoom<kDim>*>(smem);
    constexpr int kChunks = kDim / 8, kMine = kChunk * kChunks / kLoaderThreads;
    constexpr bool kFine = std::is_same<T, __half>::value;
    const skv_gdn_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int key_head = (int) (blockIdx.x % a.n_k_heads);
    const int64_t slot = blockIdx.x / a.n_k_heads;
    wait_for_previous();
    // the last sequence whose slots begin at or before this one
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        const int at = min(max(__ldg(a.seq_starts + mid), 0), a.n_tokens);
        if (first_slot(at, mid) <= slot) lo = mid;
        else hi = mid;
    }
    int begin, end;
    if (!tokens_of(a, lo, begin, end)) return;
    const int64_t chunk_of = slot - first_slot(begin, lo);
    if (chunk_of < 0 || chunk_of * kChunk >= end - begin) return;
    const int t0 = begin + (int) chunk_of * kChunk;

    // ---- K and Q as fp16
    const T* qh = static_cast<const T*>(a.q) + key_head * kDim;
    const T* kh = static_cast<const T*>(a.k) + key_head * kDim;
    uint4 k[kMine], q[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int at = i * kLoaderThreads + tid, r = at / kChunks, chunk = at % kChunks;
        const bool on = t0 + r < end;
        k[i] = on ? __ldg(reinterpret_cast<const uint4*>(kh + (int64_t) (t0 + r) * a.k_stride + chunk * 8)) : make_uint4(0, 0, 0, 0);
        q[i] = on ? __ldg(reinterpret_cast<const uint4*>(qh + (int64_t) (t0 + r) * a.q_stride + chunk * 8)) : make_uint4(0, 0, 0, 0);
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        float x[8];
        unpack8<T>(k[i], x);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]));
    }
    top = warp_largest(top);
    if (lane == 0) room.largest[warp] = top;
    __syncthreads();
    top = fmaxf(fmaxf(room.largest[0], room.largest[1]), fmaxf(room.largest[2], room.largest[3]));
    const int key_exponent = top > 0.0f && top < INFINITY ? exponent_of(top) : 0;
    const int key_power = std::is_same<T, __half>::value ? 0 : min(max(key_exponent, -60), 60);
    // A product of a query row and a key, as the tensor cores have them, is below kDim 2^(their largest values' exponents + 2);
    // divided by this and by 2^(the query's exponent) it is below 2^14, whatever their sizes, and small ones keep their bits.
    constexpr int kLogDim = kDim == 64 ? 6 : 7;
    const int mix_base = max(key_exponent - key_power, -24) + kLogDim + 2 - 14;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int at = i * kLoaderThreads + tid, r = at / kChunks, chunk = at % kChunks;
        int power = 0;
        float x[8], most = 0.0f;
        unpack8<T>(q[i], x);
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[j]));
#pragma unroll
        for (int m = 1; m < kChunks; m <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m));
        const int query_exponent = most > 0.0f && most < INFINITY ? exponent_of(most) : 0;
        if constexpr (!std::is_same<T, __half>::value) {
            power = min(max(query_exponent, -126), 126);
            const float down = power_of_two(-power);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] *= down;
            q[i] = pack8<__half>(x);
            unpack8<T>(k[i], x);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] *= power_of_two(-key_power);
            k[i] = pack8<__half>(x);
        }
        *reinterpret_cast<uint4*>(room.in.k + chunk_at<kChunks>(r, chunk)) = k[i];
        *reinterpret_cast<uint4*>(room.in.q + chunk_at<kChunks>(r, chunk)) = q[i];
        if (chunk == 0) {
            room.power[r] = power;
            room.mix_power[r] = mix_base + query_exponent - power;
        }
    }
    __syncthreads();
    // ---- K K^T and Q K^T on and below the diagonal: ten blocks of 16 x 16, at most three a warp
    const uint32_t k_at = smem_at(room.in.k), q_at = smem_at(room.in.q);
    float kk[6][4], qk[6][4];
    if (warp == 0) products<kDim, 3, 0, 2, 0>(k_at, q_at, kk, qk);
    else if (warp == 1) products<kDim, 3, 2, 2, 0>(k_at, q_at, kk, qk);
    else if (warp == 2) products<kDim, 2, 0, 3, 0>(k_at, q_at, kk, qk);
    else {
        products<kDim, 1, 0, 2, 0>(k_at, q_at, kk, qk);
        products<kDim, 0, 0, 1, 4>(k_at, q_at, kk, qk);
    }
    __syncthreads();   // the scratch matrices lie where K and Q are

    const float fit = power_of_two(key_power), fit2 = fit * fit;
    auto& work = room.work;
    for (int head = key_head * p.ratio; head < (key_head + 1) * p.ratio; ++head) {
        Record& record = p.records[slot * a.n_v_heads + head];
        // ---- the decays: a token per lane of two warps, sums in 64 bits
        float g = 0.0f, beta = 0.0f;
        double sum = 0.0;
        if (warp < 2) {
            if (t0 + tid < end) {
                g = __ldg(a.g + (int64_t) (t0 + tid) * a.g_stride + head);
                beta = __ldg(a.beta + (int64_t) (t0 + tid) * a.beta_stride + head);
            }
            sum = g < -200.0f ? -200.0 : (double) g;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const double o = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += o;
            }
            if (tid == 31) room.carry[0] = sum;
        }
        __syncthreads();
        if (warp < 2) {
            if (warp == 1) sum += room.carry[0];
            if (tid == 63) room.carry[1] = sum;
            const double turns = sum * 1.4426950408889634074;   // log2 e
            const float high = (float) turns;
            room.sums[tid] = make_float2(high, (float) (turns - (double) high));
            room.rest[tid] = exp2f((float) (__shfl_sync(0xffffffffu, turns, lane | 15) - turns));
            room.beta[tid] = beta;
        }
        __syncthreads();
        if (warp < 2) {
            const double all = room.carry[1];
            const float into = expf((float) sum);
            record.f.value[tid] = fit * beta;
            record.f.key[tid] = fit2 * beta * into;
            record.f.query[tid] = into * power_of_two(-room.mix_power[tid]);
            record.f.update[tid] = expf((float) (all - sum));
            record.f.out[tid] = a.scale * power_of_two(room.power[tid]) * power_of_two(room.mix_power[tid]);
            record.f.down[tid] = power_of_two(-room.power[tid]);
            if (tid == 0) {
                record.f.whole = expf((float) all);
                record.f.key_down = power_of_two(-key_power);
            }
            if (warp == 0) decayed<kDim, 3, 0, 2, 0, kFine>(room, fit2, kk, qk);
            else decayed<kDim, 3, 2, 2, 0, kFine>(room, fit2, kk, qk);
        } else if (warp == 2) {
            decayed<kDim, 2, 0, 3, 0, kFine>(room, fit2, kk, qk);
        } else {
            decayed<kDim, 1, 0, 2, 0, kFine>(room, fit2, kk, qk);
            decayed<kDim, 0, 0, 1, 4, kFine>(room, fit2, kk, qk);
        }
        __syncthreads();
        // ---- T = (I + A)^-1: the diagonal blocks of 16 by substitution, a column per thread
        if (tid < kChunk) {
            const int base = tid & ~15, col = tid & 15;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float r[16];
#pragma unroll
                for (int j = 0; j < (i + 3) / 4; ++j)
                    *reinterpret_cast<float4*>(&r[4 * j]) = *reinterpret_cast<const float4*>(&work.a[(base + i) * kScratch + base + 4 * j]);
                float s0 = i == col ? 1.0f : 0.0f, s1 = 0.0f;
#pragma unroll
                for (int j = 0; j < i; ++j) {
                    if (j & 1) s1 = fmaf(-r[j], x[j], s1);
                    else s0 = fmaf(-r[j], x[j], s0);
                }
                x[i] = s0 + s1;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) work.t[(base + i) * kScratch + base + col] = x[i];
        } else {
            // above the diagonal blocks of each half the products below read zeros
            for (int i = tid - kChunk; i < 2 * 16 * 16; i += kChunk)
                work.t[(i / 256 * 32 + i % 256 / 16) * kScratch + i / 256 * 32 + 16 + i % 16] = 0.0f;
        }
        __syncthreads();
        // below them T21 = -T22 (A21 T11): the blocks of 16 of each half, then the block of 32, eight columns a warp
        constexpr float kUnit = kInverseScale, kDown = 1.0f / (kUnit * kUnit);
        uint32_t ah[4], al[4], bh[2], bl[2];
        {
            const int at = (warp >> 1) * 32, col = (warp & 1) * 8;
            float c[4] = {0, 0, 0, 0}, d[4] = {0, 0, 0, 0};
            left_parts(&work.a[(at + 16) * kScratch + at], kUnit, ah, al);
            right_parts(&work.t[at * kScratch + at + col], kUnit, bh, bl);
            multiply_parts(c, ah, al, bh, bl);
            store_product(&work.a[(warp >> 1) * 16 * kScratch + 32 + col], kDown, c);
            __syncwarp();
            left_parts(&work.t[(at + 16) * kScratch + at + 16], -kUnit, ah, al);
            right_parts(&work.a[(warp >> 1) * 16 * kScratch + 32 + col], kUnit, bh, bl);
            multiply_parts(d, ah, al, bh, bl);
            store_product(&work.t[(at + 16) * kScratch + at + col], kDown, d);
        }
        __syncthreads();
        {
            const int col = warp * 8;
            float c[2][4] = {}, d[2][4] = {};
#pragma unroll
            for (int k16 = 0; k16 < 2; ++k16) {
                right_parts(&work.t[k16 * 16 * kScratch + col], kUnit, bh, bl);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    left_parts(&work.a[(32 + m * 16) * kScratch + k16 * 16], kUnit, ah, al);
                    multiply_parts(c[m], ah, al, bh, bl);
                }
            }
#pragma unroll
            for (int m = 0; m < 2; ++m) store_product(&work.a[m * 16 * kScratch + 32 + col], kDown, c[m]);
            __syncwarp();
#pragma unroll
            for (int k16 = 0; k16 < 2; ++k16) {
                right_parts(&work.a[k16 * 16 * kScratch + 32 + col], kUnit, bh, bl);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    left_parts(&work.t[(32 + m * 16) * kScratch + 32 + k16 * 16], -kUnit, ah, al);
                    multiply_parts(d[m], ah, al, bh, bl);
                }
            }
#pragma unroll
            for (int m = 0; m < 2; ++m) store_product(&work.t[(32 + m * 16) * kScratch + col], kDown, d[m]);
        }
        __syncthreads();
        // ---- T in two fp16 parts, and P
        for (int at = tid; at < kTriangleBytes / 16; at += kLoaderThreads) {
            const int block = at / 32, r = at % 32 / 2, chunk = at % 2;
            const int i = block < 1 ? 0 : block < 3 ? 1 : block < 6 ? 2 : 3, j = block - block_of(i, 0);
            const float4* x = reinterpret_cast<const float4*>(&work.t[(i * 16 + r) * kScratch + j * 16 + chunk * 8]);
            const float4 u = x[0], v = x[1];
            uint32_t high[4], low[4];
            split(u.x * kUnit, u.y * kUnit, high[0], low[0]);
            split(u.z * kUnit, u.w * kUnit, high[1], low[1]);
            split(v.x * kUnit, v.y * kUnit, high[2], low[2]);
            split(v.z * kUnit, v.w * kUnit, high[3], low[3]);
            const uint32_t to = block * kBlockBytes + half_row_at(r, chunk);
            *reinterpret_cast<uint4*>(record.t_high + to) = make_uint4(high[0], high[1], high[2], high[3]);
            *reinterpret_cast<uint4*>(record.t_low + to) = make_uint4(low[0], low[1], low[2], low[3]);
            *reinterpret_cast<uint4*>(record.mix + at * 16) = *reinterpret_cast<const uint4*>(room.mix + at * 16);
            if constexpr (kFine) *reinterpret_cast<uint4*>(record.mix_low + at * 16) = *reinterpret_cast<const uint4*>(room.mix_low + at * 16);
        }
        __syncthreads();   // the next head writes A and P again
    }
}

/// A chunk CTA: kGroupsOf groups of 16 value columns, the keys of a group split over kSplit state warps, and the outputs of
/// kTogether groups in one output warp.  kFine: P and V' enter the output in both of their parts (an fp16 output would
/// otherwise be off by 1.7 times its own rounding, with them by at most 1.4; for a bfloat16 one the first parts are eight
/// times finer than that).
template <int kDim, int kGroupsOf, int kSplit, int kTogether, bool kFine>
struct ChunkRoom {
    static constexpr int kStates = kGroupsOf * kSplit, kOutputs = kGroupsOf / kTogether;
    static constexpr int kThreadsOf = (kLoaders + kStates + kOutputs) * 32;   // loaders, state warps, output warps
    static constexpr int kMeeting = (kSplit * kTogether + 1) * 32;              // the state warps of an output warp, and it
    static constexpr int kSlices = kDim / (kGroupsOf * 16);
    struct Buffer {
        alignas(128) uint8_t k[kChunk * kDim * 2], q[kChunk * kDim * 2], v[kChunk * kGroupsOf * 32];
        Record record;
    };
    Buffer buffer[2];
    float4 sums[kSplit == 1 ? 1 : kStates][kSplit == 1 ? 1 : 8][kSplit == 1 ? 1 : 32];   // K S over half of the keys, which a state warp hands its partner
    uint4 states[kGroupsOf][kDim / 16][32];       // S as the output takes it: fp16 left operands, 16 keys each
    static constexpr int kCopies = kFine && kSplit == 1 ? 1 : 2;   // of V', by chunks: two where they fit
    uint4 values[kCopies][kGroupsOf][4][32];      // V' as the output takes it, 16 tokens each
    uint4 values_low[kFine ? kCopies : 1][kFine ? kGroupsOf : 1][kFine ? 4 : 1][kFine ? 32 : 1];   // and its second part
    static constexpr bool kRest = kFine;
    int state_power[kGroupsOf][kSplit], value_power[kCopies][kGroupsOf];
};
// Barriers.  A buffer is full (loaders arrive, the others wait) and empty again (the other way round); the two of a pair
// hand over their sums; S is ready for its output warp (which waits), and V' is (all meet: so states are never more
// than one chunk ahead of their output, whose reads of S are over by then).  Where there is one copy of V', the output has
// read it (state warps wait before they write the next).
enum : int { kFull = 0, kEmpty = 2, kPair = 4, kValueFree = 4, kStateReady = 8, kValueReady = 12 };

template <typename T, int kDim, typename Room>
__device__ __forceinline__ void load_chunks(const DeltaDev& p, Room& room, int begin, int end, int seq, int head, int slice) {
    constexpr int kAll = Room::kThreadsOf, kChunks = kDim / 8, kMine = kChunk * kChunks / kLoaderThreads;
    constexpr int kValueChunks = sizeof(Room::Buffer::v) / (kChunk * 16);
    const skv_gdn_args& a = p.a;
    const int tid = threadIdx.x;
    const T* qh = static_cast<const T*>(a.q) + (head / p.ratio) * kDim;
    const T* kh = static_cast<const T*>(a.k) + (head / p.ratio) * kDim;
    const T* vh = static_cast<const T*>(a.v) + head * kDim + slice * kValueChunks * 8;
    const Record* record = p.records + first_slot(begin, seq) * a.n_v_heads + head;
    int b = 0;
    for (int t0 = begin, n = 0; t0 < end; t0 += kChunk, ++n, b ^= 1, record += a.n_v_heads) {
        auto& buf = room.buffer[b];
        if (n >= 2) meet<kAll>(kEmpty + b);
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int at = i * kLoaderThreads + tid, r = at / kChunks, chunk = at % kChunks;
            const uint32_t to = chunk_at<kChunks>(r, chunk);
            const bool on = t0 + r < end;
            const int64_t t = on ? t0 + r : begin;
            copy_async16(smem_at(buf.k) + to, kh + t * a.k_stride + chunk * 8, on);
            copy_async16(smem_at(buf.q) + to, qh + t * a.q_stride + chunk * 8, on);
        }
        for (int at = tid; at < kChunk * kValueChunks; at += kLoaderThreads) {
            const int r = at / kValueChunks, chunk = at % kValueChunks;
            const bool on = t0 + r < end;
            copy_async16(smem_at(buf.v) + chunk_at<kValueChunks>(r, chunk), vh + (int64_t) (on ? t0 + r : begin) * a.v_stride + chunk * 8, on);
        }
        for (int at = tid; at < (int) ((Room::kRest ? sizeof(Record) : offsetof(Record, mix_low)) / 16); at += kLoaderThreads)
            copy_async16(smem_at(&buf.record) + at * 16, reinterpret_cast<const uint8_t*>(record) + at * 16, true);
        asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
        if constexpr (!std::is_same<T, __half>::value) {
            // bfloat16 becomes fp16 where it lies, each thread what it copied
            const float key_down = __ldg(&record->f.key_down);
#pragma unroll 4
            for (int i = 0; i < kMine; ++i) {
                const int at = i * kLoaderThreads + tid, r = at / kChunks, chunk = at % kChunks;
                const uint32_t to = chunk_at<kChunks>(r, chunk);
                const float down = __ldg(&record->f.down[r]);
                float x[8];
                unpack8<T>(*reinterpret_cast<const uint4*>(buf.k + to), x);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= key_down;
                *reinterpret_cast<uint4*>(buf.k + to) = pack8<__half>(x);
                unpack8<T>(*reinterpret_cast<const uint4*>(buf.q + to), x);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= down;
                *reinterpret_cast<uint4*>(buf.q + to) = pack8<__half>(x);
            }
        }
        pass<kAll>(kFull + b);
    }
}

/// The chain of states of 16 value columns, over all keys or (a pair of warps) a half of them each.
template <typename T, int kDim, int kSplit, int kTogether, typename Room>
__device__ __forceinline__ void advance(Room& room, int begin, int end, int slice, float* state) {
    constexpr int kAll = Room::kThreadsOf, kMeeting = Room::kMeeting, kChunks = kDim / 8;
    constexpr int kValueChunks = sizeof(Room::Buffer::v) / (kChunk * 16);
    constexpr int kKeys = kDim / kSplit;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - kLoaders, g = lane >> 2, c = lane & 3;
    const int part = kSplit == 1 ? 0 : warp & 1, group = kSplit == 1 ? warp : warp >> 1, key0 = part * kKeys;
    const int output = group / kTogether;
    const int col0 = slice * kValueChunks * 8 + group * 16;   // the group's value columns
    // S^T: rows (value columns) g, g + 8; columns (keys from key0 on) 8 i + 2c, 2c + 1
    float s[kKeys / 8][4];
#pragma unroll
    for (int i = 0; i < kKeys / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = state[(key0 + i * 8 + 2 * c + (j & 1)) * kDim + col0 + g + (j >> 1) * 8];
    int b = 0, unit = 0;         // S = 2^unit s
    for (int t0 = begin; t0 < end; t0 += kChunk, b ^= 1) {
        const auto& buf = room.buffer[b];
        const int s_power = max(exponent_of(warp_largest(largest_of(s))) - 14 + unit, -120);
        const float s_down = power_of_two(unit - s_power), s_up = power_of_two(s_power);
        meet<kAll>(kFull + b);   // and both warps of a pair have read what they handed over
        // ---- S^T K^T over the warp's keys
        const uint32_t k_at = smem_at(buf.k);
        float ks[8][4];
#pragma unroll
        for (int t = 0; t < 8; ++t) ks[t][0] = ks[t][1] = ks[t][2] = ks[t][3] = 0.0f;
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i) {
            uint32_t high[4], low[4], m[4][4];   // products that add to the same sums are kept apart
#pragma unroll
            for (int t = 0; t < 4; ++t) peek_matrices(m[t], k_at + chunk_at<kChunks>(t * 16 + right_row(), key0 / 8 + 2 * i + right_half()));
#pragma unroll
            for (int j = 0; j < 4; ++j)
                split(s[2 * i + (j >> 1)][2 * (j & 1)] * s_down, s[2 * i + (j >> 1)][2 * (j & 1) + 1] * s_down, high[j], low[j]);
            room.states[group][key0 / 16 + i][lane] = make_uint4(high[0], high[1], high[2], high[3]);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                multiply(ks[2 * t], high, m[t][0], m[t][1]);
                multiply(ks[2 * t + 1], high, m[t][2], m[t][3]);
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                multiply(ks[2 * t], low, m[t][0], m[t][1]);
                multiply(ks[2 * t + 1], low, m[t][2], m[t][3]);
            }
        }
        if (lane == 0) room.state_power[group][part] = s_power;
        pass<kMeeting>(kStateReady + output);
        if constexpr (kSplit == 2) {
            // ---- the other half of the keys
#pragma unroll
            for (int t = 0; t < 8; ++t) room.sums[warp][t][lane] = make_float4(ks[t][0] * s_up, ks[t][1] * s_up, ks[t][2] * s_up, ks[t][3] * s_up);
            meet<64>(kPair + group);
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const float4 x = room.sums[warp ^ 1][t][lane];
                ks[t][0] = fmaf(ks[t][0], s_up, x.x);
                ks[t][1] = fmaf(ks[t][1], s_up, x.y);
                ks[t][2] = fmaf(ks[t][2], s_up, x.z);
                ks[t][3] = fmaf(ks[t][3], s_up, x.w);
            }
        }
        // ---- R = beta (V - e^G K S), in place of K S
        const float k_unit = kSplit == 1 ? s_up : 1.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            uint32_t m[4];
            peek_matrices_t(m, smem_at(buf.v) + chunk_at<kValueChunks>(t * 16 + right_row(), group * 2 + right_half()));
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int at = (2 * t + u) * 8 + 2 * c;
                const float2 fv = *reinterpret_cast<const float2*>(&buf.record.f.value[at]);
                float2 fk = *reinterpret_cast<const float2*>(&buf.record.f.key[at]);
                fk.x *= k_unit;
                fk.y *= k_unit;
                const float2 v0 = Pair<T>::up(m[2 * u]), v1 = Pair<T>::up(m[2 * u + 1]);
                float (&r)[4] = ks[2 * t + u];
                r[0] = fv.x * v0.x - fk.x * r[0];
                r[1] = fv.y * v0.y - fk.y * r[1];
                r[2] = fv.x * v1.x - fk.x * r[2];
                r[3] = fv.y * v1.y - fk.y * r[3];
            }
        }
        const int r_power = power_for(warp_largest(largest_of(ks)));
        const float r_down = power_of_two(-r_power);
        // ---- V' = T R
        float v[8][4];
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t][0] = v[t][1] = v[t][2] = v[t][3] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t high[4], low[4], m[4][4];
#pragma unroll
            for (int t = i; t < 4; ++t) peek_matrices(m[t], smem_at(buf.record.t_high) + block_of(t, i) * kBlockBytes + half_row_at(right_row(), right_half()));
#pragma unroll
            for (int j = 0; j < 4; ++j)
                split(ks[2 * i + (j >> 1)][2 * (j & 1)] * r_down, ks[2 * i + (j >> 1)][2 * (j & 1) + 1] * r_down, high[j], low[j]);
#pragma unroll
            for (int t = i; t < 4; ++t) {
                multiply(v[2 * t], high, m[t][0], m[t][1]);
                multiply(v[2 * t + 1], high, m[t][2], m[t][3]);
            }
#pragma unroll
            for (int t = i; t < 4; ++t) {
                multiply(v[2 * t], low, m[t][0], m[t][1]);
                multiply(v[2 * t + 1], low, m[t][2], m[t][3]);
            }
#pragma unroll
            for (int t = i; t < 4; ++t) {
                peek_matrices(m[t], smem_at(buf.record.t_low) + block_of(t, i) * kBlockBytes + half_row_at(right_row(), right_half()));
                multiply(v[2 * t], high, m[t][0], m[t][1]);
                multiply(v[2 * t + 1], high, m[t][2], m[t][3]);
            }
        }
        const int v_unit = r_power - kInversePower;   // V' = 2^v_unit v
        // ---- V' for the output, from one warp of a pair
        const int copy = Room::kCopies == 1 ? 0 : b;
        if constexpr (Room::kCopies == 1) {
            static_assert(kSplit == 1, "the pairs' barriers are free");
            if (t0 > begin) meet<kMeeting>(kValueFree + output);
        }
        if (part == 0) {
            const int most = kSplit == 1 ? s_power : max(s_power, room.state_power[group][kSplit - 1]);
            const int o_power = min(max(exponent_of(warp_largest(largest_of(v))) - 14 + v_unit, max(most - 60, -120)), 120);
            const float v_down = power_of_two(v_unit - o_power);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                uint32_t high[4], low[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    split(v[2 * t + (j >> 1)][2 * (j & 1)] * v_down, v[2 * t + (j >> 1)][2 * (j & 1) + 1] * v_down, high[j], low[j]);
                room.values[copy][group][t][lane] = make_uint4(high[0], high[1], high[2], high[3]);
                if constexpr (Room::kRest) room.values_low[copy][group][t][lane] = make_uint4(low[0], low[1], low[2], low[3]);
            }
            if (lane == 0) room.value_power[copy][group] = o_power;
        }
        meet<kMeeting>(kValueReady + output);
        // ---- S <- e^(G_63) S + K^T (e^(G_63 - G) V')
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const float2 f = *reinterpret_cast<const float2*>(&buf.record.f.update[t * 8 + 2 * c]);
            v[t][0] *= f.x;
            v[t][1] *= f.y;
            v[t][2] *= f.x;
            v[t][3] *= f.y;
        }
        // one power for S and the update: the update's, or 2^-60 of what S would need where the update is smaller yet
        int w_power = exponent_of(warp_largest(largest_of(v))) - 14 + v_unit;
        w_power = min(max(w_power, max(s_power - 60, -120)), 120);
        const float w_down = power_of_two(v_unit - w_power), keep = buf.record.f.whole * power_of_two(unit - w_power);
#pragma unroll
        for (int i = 0; i < kKeys / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] *= keep;
        unit = w_power;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            uint32_t high[4], low[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                split(v[2 * t + (j >> 1)][2 * (j & 1)] * w_down, v[2 * t + (j >> 1)][2 * (j & 1) + 1] * w_down, high[j], low[j]);
#pragma unroll
            for (int h = 0; h < kKeys / 64 + (kKeys < 64); ++h) {   // 64 keys at a time
                constexpr int kDeep = kKeys < 64 ? kKeys / 16 : 4;
                uint32_t m[kDeep][4];
#pragma unroll
                for (int i = 0; i < kDeep; ++i)
                    peek_matrices_t(m[i], k_at + chunk_at<kChunks>(t * 16 + (lane & 15), key0 / 8 + 2 * (h * 4 + i) + (lane >> 4)));
#pragma unroll
                for (int i = 0; i < kDeep; ++i) {
                    multiply(s[2 * (h * 4 + i)], high, m[i][0], m[i][1]);
                    multiply(s[2 * (h * 4 + i) + 1], high, m[i][2], m[i][3]);
                }
#pragma unroll
                for (int i = 0; i < kDeep; ++i) {
                    multiply(s[2 * (h * 4 + i)], low, m[i][0], m[i][1]);
                    multiply(s[2 * (h * 4 + i) + 1], low, m[i][2], m[i][3]);
                }
            }
        }
        if (t0 + 2 * kChunk < end) pass<kAll>(kEmpty + b);
    }
#pragma unroll
    for (int i = 0; i < kKeys / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            state[(key0 + i * 8 + 2 * c + (j & 1)) * kDim + col0 + g + (j >> 1) * 8] = s[i][j] * power_of_two(unit);
}

/// O = scale (e^G Q S + P V') of kTogether groups' columns.
template <typename T, int kDim, int kSplit, int kTogether, typename Room>
__device__ __forceinline__ void put_out(const DeltaDev& p, Room& room, int begin, int end, int head, int slice) {
    constexpr int kAll = Room::kThreadsOf, kMeeting = Room::kMeeting, kChunks = kDim / 8, kDeep = kDim / kSplit / 16;
    constexpr int kValueChunks = sizeof(Room::Buffer::v) / (kChunk * 16);
    const skv_gdn_args& a = p.a;
    const int lane = threadIdx.x & 31, output = (threadIdx.x >> 5) - kLoaders - Room::kStates, g = lane >> 2, c = lane & 3;
    T* const out = static_cast<T*>(a.out) + head * kDim + slice * kValueChunks * 8 + output * kTogether * 16 + 2 * c;
    int b = 0;
    for (int t0 = begin; t0 < end; t0 += kChunk, b ^= 1) {
        const auto& buf = room.buffer[b];
        float o[kTogether][8][4];
#pragma unroll
        for (int y = 0; y < kTogether; ++y)
#pragma unroll
            for (int t = 0; t < 8; ++t) o[y][t][0] = o[y][t][1] = o[y][t][2] = o[y][t][3] = 0.0f;
        meet<kAll>(kFull + b);
        meet<kMeeting>(kStateReady + output);
        // of a pair, the part with the smaller power first: its sums are scaled down to the other's
        int s_power[kTogether], first = 0;
#pragma unroll
        for (int y = 0; y < kTogether; ++y) s_power[y] = room.state_power[output * kTogether + y][0];
        const int other = kSplit == 1 ? s_power[0] : room.state_power[output * kTogether][kSplit - 1];
        static_assert(kSplit == 1 || kTogether == 1, "one order of the parts");
        if constexpr (kSplit == 2) first = other < s_power[0];
        const uint32_t q_at = smem_at(buf.q);
#pragma unroll
        for (int h = 0; h < kSplit; ++h) {
            if (h == 1) {
                const float down = power_of_two(-abs(other - s_power[0]));
#pragma unroll
                for (int t = 0; t < 8; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[0][t][j] *= down;
            }
#pragma unroll
            for (int u = 0; u < kDeep; ++u) {
                const int i = (first ^ h) * kDeep + u;
                uint32_t high[kTogether][4];
#pragma unroll
                for (int y = 0; y < kTogether; ++y) {
                    const uint4 x = room.states[output * kTogether + y][i][lane];
                    high[y][0] = x.x; high[y][1] = x.y; high[y][2] = x.z; high[y][3] = x.w;
                }
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    uint32_t m[4];
                    peek_matrices(m, q_at + chunk_at<kChunks>(t * 16 + right_row(), 2 * i + right_half()));
#pragma unroll
                    for (int y = 0; y < kTogether; ++y) {
                        multiply(o[y][2 * t], high[y], m[0], m[1]);
                        multiply(o[y][2 * t + 1], high[y], m[2], m[3]);
                    }
                }
            }
        }
        if constexpr (kSplit == 2) s_power[0] = max(s_power[0], other);
        meet<kMeeting>(kValueReady + output);
        const int copy = Room::kCopies == 1 ? 0 : b;
        float up[kTogether];
#pragma unroll
        for (int y = 0; y < kTogether; ++y) {
            const int o_power = room.value_power[copy][output * kTogether + y];
            const float fit = power_of_two(s_power[y] - o_power);
            up[y] = power_of_two(o_power);
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const float2 f = *reinterpret_cast<const float2*>(&buf.record.f.query[t * 8 + 2 * c]);
                o[y][t][0] *= f.x * fit;
                o[y][t][1] *= f.y * fit;
                o[y][t][2] *= f.x * fit;
                o[y][t][3] *= f.y * fit;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t high[kTogether][4], low[kTogether][4];
#pragma unroll
            for (int y = 0; y < kTogether; ++y) {
                const uint4 x = room.values[copy][output * kTogether + y][i][lane];
                high[y][0] = x.x; high[y][1] = x.y; high[y][2] = x.z; high[y][3] = x.w;
                if constexpr (Room::kRest) {
                    const uint4 z = room.values_low[copy][output * kTogether + y][i][lane];
                    low[y][0] = z.x; low[y][1] = z.y; low[y][2] = z.z; low[y][3] = z.w;
                }
            }
#pragma unroll
            for (int t = i; t < 4; ++t) {
                uint32_t m[4];
                const uint32_t at = block_of(t, i) * kBlockBytes + half_row_at(right_row(), right_half());
                peek_matrices(m, smem_at(buf.record.mix) + at);
#pragma unroll
                for (int y = 0; y < kTogether; ++y) {
                    multiply(o[y][2 * t], high[y], m[0], m[1]);
                    multiply(o[y][2 * t + 1], high[y], m[2], m[3]);
                }
                if constexpr (Room::kRest) {
                    uint32_t n[4];
                    peek_matrices(n, smem_at(buf.record.mix_low) + at);
#pragma unroll
                    for (int y = 0; y < kTogether; ++y) {
                        multiply(o[y][2 * t], low[y], m[0], m[1]);
                        multiply(o[y][2 * t + 1], low[y], m[2], m[3]);
                        multiply(o[y][2 * t], high[y], n[0], n[1]);
                        multiply(o[y][2 * t + 1], high[y], n[2], n[3]);
                    }
                }
            }
        }
        if constexpr (Room::kCopies == 1) {
            if (t0 + kChunk < end) pass<kMeeting>(kValueFree + output);
        }
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const float2 f = *reinterpret_cast<const float2*>(&buf.record.f.out[t * 8 + 2 * c]);
            const int token = t0 + t * 8 + g;
#pragma unroll
            for (int y = 0; y < kTogether; ++y) {
                const uint32_t lo = transpose8(Pair<T>::down(o[y][t][0] * up[y] * f.x, o[y][t][1] * up[y] * f.y));
                const uint32_t hi = transpose8(Pair<T>::down(o[y][t][2] * up[y] * f.x, o[y][t][3] * up[y] * f.y));
                if (token < end) {
                    *reinterpret_cast<uint32_t*>(out + (int64_t) token * a.out_stride + y * 16) = lo;
                    *reinterpret_cast<uint32_t*>(out + (int64_t) token * a.out_stride + y * 16 + 8) = hi;
                }
            }
        }
        if (t0 + 2 * kChunk < end) pass<kAll>(kEmpty + b);
    }
}

/// Registers per thread of the roles where the CTA has 512 threads: they add up to what it was launched with.
constexpr int kLoaderRegisters = 48, kStateRegisters = 176, kOutputRegisters = 112;
static_assert(kLoaderRegisters * 128 + kStateRegisters * 256 + kOutputRegisters * 128 == 128 * 512, "the shares of 512 threads launched with 128 each");

/// Up to so many sequences are taken longest first, so that no long one begins when the others end: 12 ragged prompts of
/// 15,943 tokens 522 us (570 in their order; 529 now), four of 1K and then one of 4K 344 (476); fp16, 32 heads of 128.
constexpr int kRanked = 128;   // chunks times this stay below 2^32

template <typename T, int kDim, int kGroupsOf, int kSplit, int kTogether>
__global__ void __launch_bounds__(ChunkRoom<kDim, kGroupsOf, kSplit, kTogether, std::is_same<T, __half>::value>::kThreadsOf, 1) chunk_kernel(const __grid_constant__ DeltaDev p) {
    using Room = ChunkRoom<kDim, kGroupsOf, kSplit, kTogether, std::is_same<T, __half>::value>;
    extern __shared__ __align__(128) uint8_t smem[];
    auto& room = *reinterpret_cast<Room*>(smem);
    constexpr bool kShares = Room::kThreadsOf == 512;
    const skv_gdn_args& a = p.a;
    const int slice = blockIdx.x % Room::kSlices;
    const int64_t item = blockIdx.x / Room::kSlices;
    const int head = (int) (item % a.n_v_heads);
    int seq = (int) (item / a.n_v_heads);
    wait_for_previous();
    int begin, end;
    if (p.ranked) {
        // a key per sequence: its chunks, then its place; the rank of a sequence is the number of greater keys, two threads each
        __shared__ alignas(16) uint32_t s_keys[kRanked];
        __shared__ int s_seq;
        const int tid = threadIdx.x;
        if (tid < kRanked)
            s_keys[tid] = tid >= a.n_seqs ? 0u : (tokens_of(a, tid, begin, end) ? (uint32_t) (end - begin + kChunk - 1) / kChunk * kRanked : 0u) + kRanked - 1 - tid;
        __syncthreads();
        if (tid < 2 * kRanked) {
            const uint32_t mine = s_keys[tid >> 1];
            int rank = 0;
            for (int i = (tid & 1) * 4; i < a.n_seqs; i += 8) {
                const uint4 x = *reinterpret_cast<const uint4*>(s_keys + i);
                rank += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
            }
            rank += __shfl_xor_sync(0xffffffffu, rank, 1);
            if ((tid >> 1) < a.n_seqs && rank == seq) s_seq = tid >> 1;
        }
        __syncthreads();
        seq = s_seq;
    }
    if (!tokens_of(a, seq, begin, end)) return;
    float* const state = state_of(p, seq, head, kDim);
    if (!state) return;
    const int warp = threadIdx.x >> 5;
    if (warp < kLoaders) {
        if constexpr (kShares) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoaderRegisters));
        load_chunks<T, kDim>(p, room, begin, end, seq, head, slice);
    } else if (warp < kLoaders + Room::kStates) {
        if constexpr (kShares) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kStateRegisters));
        advance<T, kDim, kSplit, kTogether>(room, begin, end, slice, state);
    } else {
        if constexpr (kShares) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOutputRegisters));
        put_out<T, kDim, kSplit, kTogether>(p, room, begin, end, head, slice);
    }
}

template <typename T>
cudaError_t launch_tokens(const DeltaDev& p, cudaStream_t stream) {
    const unsigned grid = (unsigned) ((int64_t) p.a.n_seqs * p.a.n_v_heads * (p.a.head_dim / kSlice));
    return p.a.head_dim == 64 ? launch_early(token_kernel<T, 64>, dim3(grid), kThreads, 0, stream, p)
                              : launch_early(token_kernel<T, 128>, dim3(grid), kThreads, 0, stream, p);
}

template <typename T, int kDim, int kGroupsOf, int kSplit, int kTogether>
cudaError_t launch_chunks(const DeltaDev& p, int sms, cudaStream_t stream) {
    using Room = ChunkRoom<kDim, kGroupsOf, kSplit, kTogether, std::is_same<T, __half>::value>;
    constexpr auto kKernel = chunk_kernel<T, kDim, kGroupsOf, kSplit, kTogether>;
    constexpr int kSmem = sizeof(Room), kPrepare = sizeof(PrepareRoom<kDim>);
    static_assert(kSmem + 4 * kRanked + 64 <= 227 * 1024, "the buffers fit an SM");
    static_assert(Room::kThreadsOf >= 2 * kRanked, "two threads per ranked sequence");
    if constexpr (Room::kThreadsOf == 512) {
        // the roles' shares add up only if the CTA was launched with the registers they were made for
        static std::atomic<int> registers{0};   // the answer is kept, a failure to get one is not
        if (registers == 0) {
            cudaFuncAttributes f{};
            const cudaError_t e = cudaFuncGetAttributes(&f, kKernel);
            if (e != cudaSuccess) return e;
            registers = f.numRegs;
        }
        if (registers != 128) return cudaErrorInvalidConfiguration;
    }
    cudaError_t e = cudaFuncSetAttribute(prepare_kernel<T, kDim>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPrepare);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    // finding the rank costs a CTA about 0.5 us, a long sequence that begins late some 6 us a chunk: 100 sequences of 64 tokens
    // 314 us in their order, 328 by rank
    DeltaDev to = p;
    const int64_t ctas = (int64_t) p.a.n_seqs * p.a.n_v_heads * Room::kSlices;
    to.ranked = p.a.n_seqs > 1 && p.a.n_seqs <= kRanked && (int64_t) (std::min(p.a.max_tokens, p.a.n_tokens) / kChunk + 1) * 4 * sms > ctas;
    e = launch_early(prepare_kernel<T, kDim>, dim3((unsigned) (record_slots(p.a.n_tokens, p.a.n_seqs) * p.a.n_k_heads)), kLoaderThreads, kPrepare, stream, p);
    if (e != cudaSuccess) return e;
    return launch_early(kKernel, dim3((unsigned) ctas), Room::kThreadsOf, kSmem, stream, to);
}

/// How long a launch of so many CTAs per sequence and head takes, one CTA per SM, in tokens of one CTA: the longest sequence
/// when all run at once; else what the longest ones take in their rounds or, if that is more, all tokens over the SMs and half
/// of another sequence for the uneven end.
int64_t span_of(const skv_gdn_args& a, int sms, int slices) {
    const int64_t ctas = (int64_t) a.n_v_heads * slices, longest = std::min(a.max_tokens, a.n_tokens);
    if (ctas * a.n_seqs <= sms) return longest;
    const int64_t other = a.n_seqs > 1 ? std::min((a.n_tokens - longest) / (a.n_seqs - 1), longest) : 0;
    return std::max((ctas + sms - 1) / sms * longest, a.n_tokens * ctas / sms + other / 2);
}

template <typename T>
cudaError_t launch(const DeltaDev& p, int sms, cudaStream_t stream) {
    if (!chunked(p.a.seq_starts != nullptr, p.a.max_tokens)) return launch_tokens<T>(p, stream);
    // A chunk takes CTAs of 32 columns with the keys in halves, CTAs of 64, and CTAs of all 128 about 2, 3 and 4 units of time
    // (at head_dim 64, 32 and 64 columns: 3 and 4); the wider, the fewer CTAs.  In us, bfloat16, 2,048 tokens a sequence,
    // 128 wide: one sequence of 32 heads 116, 157, 204; of 48 heads 206, 165, 208; two of 32 216, 175, 218; of 48 314, 316,
    // 234; eight of 32 736, 658, 486.  One of 8K and 15 of 100 tokens, 32 heads: 482, 622, 797; 64 heads: 919, 747, 845.
    const int64_t narrow = span_of(p.a, sms, p.a.head_dim / 32);
    if (p.a.head_dim == 64)
        return narrow * 3 <= span_of(p.a, sms, 1) * 4 ? launch_chunks<T, 64, 2, 2, 1>(p, sms, stream) : launch_chunks<T, 64, 4, 1, 2>(p, sms, stream);
    const int64_t middle = span_of(p.a, sms, 2) * 3, wide = span_of(p.a, sms, 1) * 4;
    if (narrow * 2 <= std::min(middle, wide)) return launch_chunks<T, 128, 2, 2, 1>(p, sms, stream);
    return middle <= wide ? launch_chunks<T, 128, 4, 2, 1>(p, sms, stream) : launch_chunks<T, 128, 8, 1, 2>(p, sms, stream);
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
    if (chunked(true, max_tokens)) *out_bytes = ((uint64_t) record_slots(n_tokens, n_seqs) * n_v_heads * sizeof(Record) + 255) / 256 * 256;
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
    if (!ops_aligned4(a.g, a.beta, a.state_index, a.seq_starts)) return no("g, beta, state_index and seq_starts must be 4-byte aligned");
    if (a.q_stride % 8 || a.k_stride % 8 || a.v_stride % 8 || a.out_stride % 8 || a.state_stride % 4)
        return no("strides must be multiples of 8 elements (4 floats for the state)");
    const int64_t kw = (int64_t) a.n_k_heads * a.head_dim, vw = (int64_t) a.n_v_heads * a.head_dim;
    if (a.n_tokens > 1 && (a.q_stride < kw || a.k_stride < kw || a.v_stride < vw || a.out_stride < vw))
        return no("a stride is shorter than its row");
    if (a.state_rows < 1 || (a.state_rows > 1 && a.state_stride < vw * a.head_dim)) return no("the state rows overlap or are none");
    if (!a.state_index && a.state_rows < a.n_seqs) return no("fewer state rows than sequences");
    uint64_t need = 0;
    if (const int rc = skv_gated_delta_workspace(a.n_tokens, a.n_seqs, a.n_v_heads, a.head_dim, a.seq_starts ? a.max_tokens : 1, &need)) return rc;
    if (need / sizeof(Record) > INT32_MAX) return fail(SKV_ERANGE, "skv_gated_delta: too many tokens and heads");
    if (need && (!a.workspace || (reinterpret_cast<uintptr_t>(a.workspace) & 255u) || a.workspace_bytes < need))
        return no("the workspace must be 256-byte aligned and as large as skv_gated_delta_workspace says");
    DeviceCtx* ctx = current_ctx();
    if (!ctx) return SKV_ECUDA;
    if (!ops_own_memory(a.state, ctx->device)) return no("the state is not memory of the current device");
    DeltaDev p{};
    p.a = a;
    p.status = ctx->status;
    p.records = static_cast<Record*>(a.workspace);
    p.ratio = a.n_v_heads / a.n_k_heads;
    const auto s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = a.dtype == SKV_DTYPE_F16 ? launch<__half>(p, ctx->sms, s) : launch<__nv_bfloat16>(p, ctx->sms, s);
    return e == cudaSuccess ? SKV_OK : cuda_fail(e, "skv_gated_delta");
}

}  // extern "C"

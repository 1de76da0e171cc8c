// skv_attention.cu - skv_decode_attention: one new token per sequence over its paged cache.
//
//   s_t = scale * q . k_t;   m = max s_t;   out = sum e^(s_t - m) v_t / sum e^(s_t - m);   lse = m + ln sum
//
// The cache is read once, so its bytes bound the operator, and everything else has to fit beside the stream: the products
// go through the tensor cores (the up to 16 query heads that share a K/V head are the 16 rows of an m16n8k16 product, as
// 12 of them on CUDA cores would take 12 flops per byte, more than the cores have at this bandwidth).
//
// Split.  The work is the tiles of all (sequence, K/V head) items laid end to end; each CTA takes an equal, contiguous share
// of them, worked out from the lengths on the device, so one long sequence and many ragged ones load the GPU alike.  An
// item that lies inside one share is finished there; an item cut by a share's border leaves parts (its unnormalised
// output, maximum and sum) that join_kernel adds up in a fixed order.
//
// A tile is 32 KiB of K and as much of V (64 cells of 256 fp16 values; 64 int8 cells are half of that).  A CTA of four warps
// holds one tile of K and two of V, and two to four CTAs share an SM: 192 KiB of copies on their way per SM, and one CTA's
// products run under another's barriers (one CTA of eight warps and three tiles: 128K cells 76 us, 32 ragged sequences 101,
// against 63 and 75).  Each warp copies its own quarter of the cells (16-byte cp.async, chunks swizzled by the row so that
// ldmatrix meets no bank twice) and scores it; the warps exchange row maxima and weights through shared memory and each
// multiplies all weights with its own quarter of V's columns.  So no warp holds an output that another has to add, and a
// tile costs two barriers.
//
// Measured (24 heads on 2 K/V heads of 256, both kernels, in a graph): 131,072 fp16 cells 54 us, 5.0 TB/s; 32 ragged
// sequences of 378 MB in all 73 us, 5.2 TB/s: the cache's bytes bound these, with 3 to 7 us of it the join.  8 x 32K int8 cells
// 76.8 us, 3.6 TB/s: the latency of converting every code to fp16 in front of its product, with three warps a scheduler.  1,000
// cells 11.5 us: two kernels' latencies.
//
// Precision.  fp16 queries and cache values meet in exact products, summed in 32 bits.  A bfloat16 query row is scaled by a
// power of two to below 2 and becomes fp16 without loss, up to values 2^-24 of its largest.  Weights are rounded to fp16
// for the product with V (2^-11 each; they are scaled by 2^15, so a weight is a normal number down to 2^-29 of the
// largest), their sum is taken before that rounding.  int8 codes are exact in fp16; K's scales are applied to the 32-bit
// sums of their 64 values, V's to the weights before they are rounded, under a running power of two per group.
#include "skv_ops.h"

#include <cmath>
#include <string>
#include <type_traits>

namespace skv {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;        // query heads per item: the rows of one matrix product
constexpr int kMaxSms = 160;
constexpr int kJoinThreads = 128;

struct AttnDev {
    LayerDev layer;
    skv_attention_args a;
    uint32_t* status;
    int group;      // query heads per K/V head
    int blocks;     // items per (sequence, K/V head): group / 16, rounded up
    float* part_o;  // [share][2][16][dim]
    float2* part_ml;// [share][2][16]: maximum (of base-2 exponents) and sum
    int2* cut;      // [share]: the item whose first part is this share's second (-1: none), and its parts
};

template <int kDim, bool kInt8>
struct Geo {
    static constexpr int kRowBytes = kDim * (kInt8 ? 1 : 2);
    // cells per tile: a plane (K or V of a tile) of 32 KiB, at most a lane per cell of a warp; 16 KiB where four sets of
    // weights lie beside it
    static constexpr int kTile = kInt8 && kDim == 256 ? 64 : 32768 / kRowBytes < 128 ? 32768 / kRowBytes : 128;
    static constexpr int kCells = kTile / kWarps;                                     // per warp
    static constexpr int kChunks = kRowBytes / 16;
    static constexpr int kGroups = kInt8 ? kDim / kInt8Group : 1;
    static constexpr int kScaleBytes = kInt8 ? (kGroups * 2 < 4 ? 4 : kGroups * 2) : 0;
    static constexpr int kPlane = kTile * kRowBytes;
    static constexpr int kSlotBytes = kPlane + kTile * kScaleBytes;
    static constexpr int kWeightStride = kTile + 8;   // halves: rows 16 bytes apart modulo 128, ldmatrix meets no bank twice
    static constexpr int kWeightBytes = kGroups * kRows * kWeightStride * 2;
    static constexpr int kQueryStride = kDim + 8;     // halves
    static constexpr int kQueryBytes = kInt8 ? kRows * kQueryStride * 2 : 0;
    static constexpr int kSmem = 3 * kSlotBytes + kWeightBytes + kQueryBytes;   // K, and V twice
    static constexpr int kPerSm = kPlane > 24000 ? 2 : kPlane > 12000 ? 3 : 4;   // CTAs: as many as shared memory holds
    static constexpr int kCols = kDim / kWarps;       // of the output, per warp
    static constexpr int kOutTiles = kCols / 8;
};

// ---------------------------------------------------------------- small pieces

__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
/// The first kRead of kBytes bytes, and zeros behind them; off: zeros, nothing is read.
template <int kBytes, int kRead = kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool on) {
    if constexpr (kBytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? kRead : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kBytes), "r"(on ? kRead : 0) : "memory");
}
/// Where a copy of 4 or 8 bytes that holds the scales of `row` begins (a multiple of its size), in bytes, and how many of them
/// are read: at head_dim 64 a row has one scale of two bytes; an even row's is the first half of its word, whose second
/// half may lie behind the last row.
constexpr __host__ __device__ int64_t scales_at(int64_t row, int groups) { return (row * groups * 2) & ~(int64_t) 3; }
constexpr __host__ __device__ int scales_read(int64_t row, int groups) { return groups > 1 ? groups * 2 : row & 1 ? 4 : 2; }
constexpr bool scales_lie_within(int64_t rows, int groups) {
    for (int64_t row = 0; row < rows; ++row) {
        const int64_t at = scales_at(row, groups), end = at + scales_read(row, groups);
        if (at % (groups > 1 ? groups * 2 : 4) || end > rows * groups * 2 || row * groups * 2 < at || (row + 1) * groups * 2 > end) return false;
    }
    return true;
}
static_assert(scales_lie_within(1, 1) && scales_lie_within(2, 1) && scales_lie_within(7, 1) && scales_lie_within(5, 2) && scales_lie_within(5, 4),
              "a row's scales are read, and nothing behind the last row's");
__device__ __forceinline__ void commit_async() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void wait_async() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}
/// Ordered by the waits and barriers around them (all volatile), not against the thread's own stores: what they read
/// was copied or written before one of those, so they can run ahead between them.
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void load_matrices_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
/// The CTA's barrier, a warp's meeting.
__device__ __forceinline__ void meet() { asm volatile("bar.sync 0;" ::: "memory"); }
__device__ __forceinline__ void meet_warp() { asm volatile("bar.warp.sync 0xffffffff;" ::: "memory"); }
/// c += a b, 16 x 8 x 16 in fp16 with 32-bit sums.
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
/// Two of four signed codes as fp16, exactly: the byte u = code + 128 under the exponent of 1024 is 1024 + u.
template <uint32_t kPick>
__device__ __forceinline__ uint32_t codes_to_half(uint32_t biased) {
    const uint32_t w = __byte_perm(biased, 0x64646464u, kPick);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0x6480)));   // 1152
    return *reinterpret_cast<const uint32_t*>(&h);
}
/// The scales of a cell's groups; head_dim 64 has one, in the lower or the upper (`odd`) half of its word.
template <int kGroups>
__device__ __forceinline__ void load_scales(const uint8_t* at, bool odd, float (&x)[kGroups]) {
    if constexpr (kGroups == 1) x[0] = __half2float(reinterpret_cast<const __half*>(at)[odd]);
    else {
        uint32_t w[kGroups / 2];
        if constexpr (kGroups == 4) {
            const uint2 y = *reinterpret_cast<const uint2*>(at);
            w[0] = y.x;
            w[1] = y.y;
        } else w[0] = *reinterpret_cast<const uint32_t*>(at);
#pragma unroll
        for (int i = 0; i < kGroups / 2; ++i) {
            const float2 f = Pair<__half>::up(w[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}
__device__ __forceinline__ float power_of_two(int e) {   // e clamped to the normal numbers
    return __int_as_float((min(max(e, -126), 127) + 127) << 23);
}
/// The 16-byte chunk `chunk` of row `row` of a tile, swizzled so that eight rows' equal chunks lie in eight bank groups.
template <int kChunks>
__device__ __forceinline__ uint32_t chunk_at(int row, int chunk) {
    return (uint32_t) (row * kChunks + (kChunks >= 8 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3))) * 16u;
}

/// The cells of a sequence that are attended.
__device__ __forceinline__ int64_t cells_of(const AttnDev& p, int seq) {
    const int64_t table = p.layer.table_stride << p.layer.page_shift;
    const int n = __ldg(p.a.lengths + seq);
    return n < 0 ? 0 : n > table ? table : n;
}

/// `before` plus the sum of v over this thread and those before it; `before` grows by the CTA's sum.  Every thread calls it.
__device__ __forceinline__ int64_t cta_scan(int64_t v, int64_t& before, int64_t* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += o;
    }
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    v += before;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) v += scratch[w];
        before += scratch[w];
    }
    __syncthreads();
    return v;
}

/// a / b of non-negative numbers, in 32 bits where they fit.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return ((a | b) >> 31) == 0 ? (int64_t) ((uint32_t) a / (uint32_t) b) : a / b;
}

/// A place in the sequence of all tiles.
struct Cursor {
    int seq, item;        // item: the K/V head and block of heads within the sequence
    int tile, tiles;      // of the sequence
    int64_t cells;
};
__device__ __forceinline__ int kv_of(const Cursor& c, const AttnDev& p) { return c.item / p.blocks; }
template <int kTile>
__device__ __forceinline__ void step(Cursor& c, const AttnDev& p, int items) {
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.item < items) return;
    c.item = 0;
    do {
        if (++c.seq >= p.a.n_seqs) return;   // the last share's end
        c.cells = cells_of(p, c.seq);
    } while (c.cells == 0);
    c.tiles = (int) ((c.cells + kTile - 1) / kTile);
}

// ---------------------------------------------------------------- the kernel

template <typename T, int kDim, bool kInt8>
__global__ void __launch_bounds__(kThreads, Geo<kDim, kInt8>::kPerSm) attention_kernel(const __grid_constant__ AttnDev p) {
    using G = Geo<kDim, kInt8>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_top[kWarps][kRows], s_sum[kWarps][kRows];
    __shared__ alignas(16) int s_power[kWarps][4];   // int8: per V scale group
    __shared__ int64_t s_scan[kWarps];
    __shared__ int64_t s_first[2];   // the first sequence of the share, and the tiles before it
    __shared__ int64_t s_share[3];   // for the end: the share's first tile, all tiles, all shares
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int items = p.layer.n_head_kv * p.blocks, n_seqs = p.a.n_seqs;
    const skv_attention_args& a = p.a;

    wait_for_previous();
    // ---- the share: `count` tiles from `from` on, of all.  The tiles of sequences 0 .. s, a thread per sequence, in trips
    const auto tiles_of = [&](int s) { return s < n_seqs ? (cells_of(p, s) + G::kTile - 1) / G::kTile * items : 0; };
    int64_t total = 0, end = 0, n = 0;   // of the trip's sequence: the tiles up to its end, and its own
    for (int base = 0; base < n_seqs; base += kThreads) {
        n = tiles_of(base + tid);
        end = cta_scan(n, total, s_scan);
    }
    const int64_t shares = total < (int64_t) gridDim.x ? total : (int64_t) gridDim.x;
    // sequences without cells
    for (int s = blockIdx.x; s < n_seqs; s += gridDim.x) {
        const int asked = __ldg(a.lengths + s);
        if (tid == 0 && (asked < 0 || asked > (p.layer.table_stride << p.layer.page_shift))) atomicOr(p.status, SKV_STATUS_BAD_SRC_PAGE);
        if (asked > 0) continue;
        for (int i = tid; i < a.n_head * kDim / 8; i += kThreads)
            *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + s * a.out_stride + i * 8) = make_uint4(0, 0, 0, 0);
        if (a.lse)
            for (int i = tid; i < a.n_head; i += kThreads) a.lse[(int64_t) s * a.n_head + i] = -INFINITY;
    }
    if ((int64_t) blockIdx.x >= shares) {
        if (tid == 0) p.cut[blockIdx.x] = make_int2(-1, 0);
        return;
    }
    const int64_t from = quotient(total * blockIdx.x, shares), count = quotient(total * (blockIdx.x + 1), shares) - from;
    if (n_seqs <= kThreads) {   // the one trip is still at hand
        if (n && from >= end - n && from < end) {
            s_first[0] = tid;
            s_first[1] = end - n;
        }
        meet();
    } else {
        int64_t before = 0;
        for (int base = 0; base < n_seqs && before <= from; base += kThreads) {
            n = tiles_of(base + tid);
            end = cta_scan(n, before, s_scan);
            if (n && from >= end - n && from < end) {
                s_first[0] = base + tid;
                s_first[1] = end - n;
            }
            meet();
        }
    }
    if (tid == 0) {
        s_share[0] = from;
        s_share[1] = total;
        s_share[2] = shares;
    }
    Cursor load;
    load.seq = (int) s_first[0];
    load.cells = cells_of(p, load.seq);
    load.tiles = (int) ((load.cells + G::kTile - 1) / G::kTile);
    load.item = (int) quotient(from - s_first[1], load.tiles);
    load.tile = (int) (from - s_first[1] - (int64_t) load.item * load.tiles);
    Cursor here = load;

    // ---- loading.  Lane i of a warp knows the warp's cell i; its table entry is read a tile before its copies are issued.
    // A warp alone reads the K it copied, so the next tile's K follows as soon as it has its scores; V has two slots, and
    // the next tile's follows once all warps have met after using the one before.
    static_assert(G::kCells <= 32 && G::kCells % 8 == 0, "a lane per cell, whole 8-row matrices");
    int entry = 0, within = -1;      // the next tile's table entry, and its cell's row within the page (-1: no cell)
    auto find = [&]() {
        const int64_t cell = (int64_t) load.tile * G::kTile + warp * G::kCells + lane;
        within = -1;
        if (lane < G::kCells && cell < load.cells) {
            within = (kv_of(load, p) << p.layer.page_shift) + (int) (cell & ((1 << p.layer.page_shift) - 1));
            entry = __ldg(p.layer.tables + (int64_t) load.seq * p.layer.table_stride + (cell >> p.layer.page_shift));
        }
    };
    int64_t found = 0, row = -1;     // tiles found so far; the row of the tile whose K was issued last
    uint32_t held = 0, odd = 0;      // of that tile: the cells that are there, the rows that are odd
    auto copy_plane = [&](int slot, const uint8_t* pool, const __half* scales) {
        constexpr int kPer = 32 / G::kChunks;   // rows per trip of the warp
        const uint32_t base = smem_at(smem) + slot * G::kSlotBytes, to = base + warp * G::kCells * G::kRowBytes;
        const int64_t byte = row < 0 ? -1 : row * G::kRowBytes;
#pragma unroll
        for (int i = 0; i < G::kCells / kPer; ++i) {
            const int r = i * kPer + lane / G::kChunks, chunk = lane % G::kChunks;
            const int64_t from_byte = __shfl_sync(0xffffffffu, byte, r);
            copy_async<16>(to + chunk_at<G::kChunks>(r, chunk), pool + (from_byte < 0 ? 0 : from_byte) + chunk * 16, from_byte >= 0);
        }
        if constexpr (kInt8) {
            if (lane < G::kCells) {
                const uint32_t dst = base + G::kPlane + (warp * G::kCells + lane) * G::kScaleBytes;
                const uint8_t* src = reinterpret_cast<const uint8_t*>(scales) + (row < 0 ? 0 : scales_at(row, G::kGroups));
                if (G::kGroups == 1 && !(row & 1)) copy_async<G::kScaleBytes, scales_read(0, G::kGroups)>(dst, src, row >= 0);
                else copy_async<G::kScaleBytes, scales_read(1, G::kGroups)>(dst, src, row >= 0);
            }
        }
    };
    // the next tile's rows and K, and the entries of the tile after it
    auto issue_k = [&]() {
        held = 0;
        if (found < count) {
            const bool there = within >= 0 && entry >= 0 && entry < p.layer.page_limit;
            if (within >= 0 && !there) atomicOr(p.status, SKV_STATUS_BAD_SRC_PAGE);
            row = there ? (((int64_t) entry * p.layer.n_head_kv) << p.layer.page_shift) + within : -1;
            held = __ballot_sync(0xffffffffu, there);
            odd = __ballot_sync(0xffffffffu, row & 1);
            copy_plane(0, p.layer.k, p.layer.k_scale);
            ++found;
            if (found < count) {
                step<G::kTile>(load, p, items);
                find();
            }
        }
        commit_async();   // a group per call, empty ones too: the count of groups stands for the count of planes
    };
    auto issue_v = [&](int slot, bool on) {
        if (on) copy_plane(slot, p.layer.v, p.layer.v_scale);
        commit_async();
    };
    find();
    issue_k();
    issue_v(1, true);

    // ---- the item's query, 16 heads x kDim, the left operand of all its products: of an fp16 cache in registers; of an int8
    // one, whose conversions need those, in shared memory
    uint32_t q[kInt8 ? 1 : kDim / 16][4];
    float factor[2];   // of rows g and g + 8: scale, log2 e, and the power of two the row was divided by
    uint8_t* const queries = smem + 3 * G::kSlotBytes + G::kWeightBytes;
    __shared__ float s_factor[kRows];
    // the power of two that a row is divided by; in range for every finite row, 1 for one with an infinity
    const auto power_of_row = [](float top) {
        return top > 0.0f && top < INFINITY ? min(max(((__float_as_int(top) >> 23) & 0xff) - 127, -126), 126) : 0;
    };
    auto load_query = [&]() {
        const int kv = kv_of(here, p), first = (here.item - kv * p.blocks) * kRows;
        if constexpr (kInt8) {
            // eight lanes a row; of each 16 values 4c, 4c+1 go to places 2c, 2c+1 and 4c+2, 4c+3 to 2c+8, 2c+9, so that
            // the operand's columns meet K's as a register of four codes holds them
            const int row = tid >> 3, r = first + row;
            const bool on = r < p.group;
            const T* src = static_cast<const T*>(a.q) + (int64_t) here.seq * a.q_stride + (int64_t) (kv * p.group + (on ? r : 0)) * kDim;
            float top = 0.0f;
            constexpr int kPieces = kDim / 64;    // of 8 values, per lane
            uint4 w[kPieces];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                w[i] = on ? *reinterpret_cast<const uint4*>(src + ((tid & 7) * kPieces + i) * 8) : make_uint4(0, 0, 0, 0);
                if constexpr (!std::is_same<T, __half>::value) {
                    float x[8];
                    unpack8<T>(w[i], x);
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]));
                }
            }
            int e = 0;
            if constexpr (!std::is_same<T, __half>::value) {
#pragma unroll
                for (int m = 1; m < 8; m <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
                e = power_of_row(top);
                const float down = power_of_two(-e);
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    float x[8];
                    unpack8<T>(w[i], x);
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] *= down;
                    w[i] = pack8<__half>(x);
                }
            }
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                // half of a block of 16: its pairs 0 and 2 go to the first eight places, 1 and 3 to the last eight
                const int piece = (tid & 7) * kPieces + i;
                uint2* to = reinterpret_cast<uint2*>(queries + (row * G::kQueryStride + piece / 2 * 16 + (piece & 1) * 4) * 2);
                to[0] = make_uint2(w[i].x, w[i].z);
                to[2] = make_uint2(w[i].y, w[i].w);
            }
            if ((tid & 7) == 0) s_factor[row] = a.scale * 1.4426950408889634f * power_of_two(e);
            meet();
            factor[0] = s_factor[g];
            factor[1] = s_factor[g + 8];
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = first + g + h * 8;
                const bool on = r < p.group;
                const T* src = static_cast<const T*>(a.q) + (int64_t) here.seq * a.q_stride + (int64_t) (kv * p.group + (on ? r : 0)) * kDim;
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < kDim / 16; ++i) {
                    // values 2c, 2c+1 and 2c+8, 2c+9 of each 16, as ldmatrix hands out K's rows
                    const uint32_t* w = reinterpret_cast<const uint32_t*>(src + i * 16);
                    q[i][h] = on ? w[c] : 0u;
                    q[i][h + 2] = on ? w[c + 4] : 0u;
                    if constexpr (!std::is_same<T, __half>::value) {
                        const float2 x = Pair<T>::up(q[i][h]), y = Pair<T>::up(q[i][h + 2]);
                        top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
                    }
                }
                int e = 0;
                if constexpr (!std::is_same<T, __half>::value) {
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    e = power_of_row(top);
                    const float down = power_of_two(-e);
#pragma unroll
                    for (int i = 0; i < kDim / 16; ++i) {
                        const float2 x = Pair<T>::up(q[i][h]), y = Pair<T>::up(q[i][h + 2]);
                        q[i][h] = Pair<__half>::down(x.x * down, x.y * down);
                        q[i][h + 2] = Pair<__half>::down(y.x * down, y.y * down);
                    }
                }
                factor[h] = a.scale * 1.4426950408889634f * power_of_two(e);
            }
        }
    };
    load_query();

    float out[G::kOutTiles][4], top[2], sum[2];
    int powers[G::kGroups];   // int8: the running power of two above V's scales, per group
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < G::kOutTiles; ++i) out[i][0] = out[i][1] = out[i][2] = out[i][3] = 0.0f;
        top[0] = top[1] = -INFINITY;
        sum[0] = sum[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < G::kGroups; ++i) powers[i] = -24;
    };
    clear();
    uint8_t* const weights = smem + 3 * G::kSlotBytes;
    int first_tile = here.tile;   // of the item, in this share

    int v_slot = 1;
    for (n = 0; n < count; ++n, v_slot = 3 - v_slot) {
        const uint8_t* const v_base = smem + v_slot * G::kSlotBytes;
        const uint32_t held_now = held, odd_now = odd;
        wait_async<1>();          // K of this tile
        meet_warp();

        // ---- scores of the warp's cells: rows g, g + 8; cells 8 t + 2c, 2c + 1
        constexpr int kTiles = G::kCells / 8;
        float score[kTiles][4];
        const uint32_t k_at = smem_at(smem) + warp * G::kCells * G::kRowBytes;
        if constexpr (!kInt8) {
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                float x[4] = {0, 0, 0, 0}, y[4] = {0, 0, 0, 0};   // two chains of sums
#pragma unroll
                for (int i = 0; i < kDim / 32; ++i) {
                    uint32_t b[4];
                    load_matrices(b, k_at + chunk_at<G::kChunks>(t * 8 + (lane & 7), i * 4 + (lane >> 3)));
                    multiply(x, q[2 * i], b[0], b[1]);
                    multiply(y, q[2 * i + 1], b[2], b[3]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) score[t][j] = x[j] + y[j];
            }
        } else {
            const uint32_t q_at = smem_at(queries) + ((lane & 15) * G::kQueryStride + (lane >> 4) * 8) * 2;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) score[t][0] = score[t][1] = score[t][2] = score[t][3] = 0.0f;
#pragma unroll
            for (int i = 0; i < G::kGroups; ++i) {
                uint32_t w[4][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) load_matrices(w[j], q_at + (i * 4 + j) * 32);
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    uint32_t b[4];
                    load_matrices(b, k_at + chunk_at<G::kChunks>(t * 8 + (lane & 7), i * 4 + (lane >> 3)));
                    float x[4] = {0, 0, 0, 0}, y[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 4; ++j) b[j] ^= 0x80808080u;
                    multiply(x, w[0], codes_to_half<0x4140>(b[0]), codes_to_half<0x4342>(b[0]));
                    multiply(y, w[1], codes_to_half<0x4140>(b[1]), codes_to_half<0x4342>(b[1]));
                    multiply(x, w[2], codes_to_half<0x4140>(b[2]), codes_to_half<0x4342>(b[2]));
                    multiply(y, w[3], codes_to_half<0x4140>(b[3]), codes_to_half<0x4342>(b[3]));
                    const int cell = t * 8 + 2 * c;
                    const uint8_t* s_at = smem + G::kPlane + (warp * G::kCells + cell) * G::kScaleBytes;
                    const int h0 = kDim == 64 ? (odd_now >> cell) & 1 : i, h1 = kDim == 64 ? (odd_now >> (cell + 1)) & 1 : i;
                    const float s0 = __half2float(reinterpret_cast<const __half*>(s_at)[h0]);
                    const float s1 = __half2float(reinterpret_cast<const __half*>(s_at + G::kScaleBytes)[h1]);
                    score[t][0] = fmaf(x[0] + y[0], s0, score[t][0]);
                    score[t][1] = fmaf(x[1] + y[1], s1, score[t][1]);
                    score[t][2] = fmaf(x[2] + y[2], s0, score[t][2]);
                    score[t][3] = fmaf(x[3] + y[3], s1, score[t][3]);
                }
            }
        }
        meet_warp();
        issue_k();
        float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool on = (held_now >> (t * 8 + 2 * c + (j & 1))) & 1u;
                score[t][j] = on ? score[t][j] * factor[j >> 1] : -INFINITY;
                most[j >> 1] = fmaxf(most[j >> 1], score[t][j]);   // fmaxf passes a NaN over; its weight is NaN all the same
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 1));
            most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 2));
            if (c == 0) s_top[warp][g + h * 8] = most[h];
        }
        if constexpr (kInt8) {
            // the largest V scale of the warp's cells per group, as the power of two above it
            wait_async<1>();              // V of this tile
            meet_warp();
            float scale[G::kGroups];
            load_scales(v_base + G::kPlane + (warp * G::kCells + (lane < G::kCells ? lane : 0)) * G::kScaleBytes, (odd_now >> lane) & 1, scale);
            int e[4] = {-24, -24, -24, -24};
#pragma unroll
            for (int i = 0; i < G::kGroups; ++i) {
                const float s = fabsf(scale[i]);
                const int x = s > 0.0f && lane < G::kCells ? min(((__float_as_int(s) >> 23) & 0xff) - 126, 17) : -24;
                e[i] = __reduce_max_sync(0xffffffffu, x);
            }
            if (lane == 0) *reinterpret_cast<int4*>(s_power[warp]) = make_int4(e[0], e[1], e[2], e[3]);
        }
        meet();   // row maxima; and every warp is done with V of the tile before, whose slot is filled again
        issue_v(3 - v_slot, n + 1 < count);

        float keep[2], now[2], shrink = 1.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float x = top[h];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) x = fmaxf(x, s_top[w][g + h * 8]);
            now[h] = x == -INFINITY ? 0.0f : x;   // nothing but minus infinity so far: any reference will do
            keep[h] = exp2f(top[h] - now[h]);
            top[h] = x;
            sum[h] *= keep[h];
        }
        if constexpr (kInt8) {
            // within an item a power only grows: what was summed under a smaller one is scaled down
            const int mine = warp * G::kCols / kInt8Group;
            int most[4] = {-24, -24, -24, -24};
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const int4 x = *reinterpret_cast<const int4*>(s_power[w]);
                most[0] = max(most[0], x.x);
                most[1] = max(most[1], x.y);
                most[2] = max(most[2], x.z);
                most[3] = max(most[3], x.w);
            }
#pragma unroll
            for (int i = 0; i < G::kGroups; ++i) {
                const int x = max(powers[i], most[i]);
                if (i == mine) shrink = power_of_two(powers[i] - x);
                powers[i] = x;
            }
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int cell = warp * G::kCells + t * 8 + 2 * c;
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = exp2f(score[t][j] - now[j >> 1]);
                sum[j >> 1] += w[j];
                w[j] *= 32768.0f;
            }
            if constexpr (!kInt8) {
                uint32_t* at = reinterpret_cast<uint32_t*>(weights + (g * G::kWeightStride + cell) * 2);
                at[0] = Pair<__half>::down(w[0], w[1]);
                at[8 * G::kWeightStride / 2] = Pair<__half>::down(w[2], w[3]);
            } else {
                const uint8_t* s_at = v_base + G::kPlane + cell * G::kScaleBytes;
                const int in = t * 8 + 2 * c;
                float v0[G::kGroups], v1[G::kGroups];
                load_scales(s_at, (odd_now >> in) & 1, v0);
                load_scales(s_at + G::kScaleBytes, (odd_now >> (in + 1)) & 1, v1);
#pragma unroll
                for (int i = 0; i < G::kGroups; ++i) {
                    const float down = power_of_two(-powers[i]), s0 = down * v0[i], s1 = down * v1[i];
                    uint32_t* at = reinterpret_cast<uint32_t*>(weights + ((i * kRows + g) * G::kWeightStride + cell) * 2);
                    at[0] = Pair<__half>::down(w[0] * s0, w[1] * s1);
                    at[8 * G::kWeightStride / 2] = Pair<__half>::down(w[2] * s0, w[3] * s1);
                }
            }
        }
        wait_async<2>();   // V of this tile
        meet();   // weights, and everybody's part of V

        // ---- output: all cells x the warp's columns
#pragma unroll
        for (int i = 0; i < G::kOutTiles; ++i) {
            out[i][0] *= keep[0] * shrink;
            out[i][1] *= keep[0] * shrink;
            out[i][2] *= keep[1] * shrink;
            out[i][3] *= keep[1] * shrink;
        }
        const int group = kInt8 ? warp * G::kCols / kInt8Group : 0;
        const uint32_t w_at = smem_at(weights) + ((group * kRows + (lane & 15)) * G::kWeightStride + (lane >> 4) * 8) * 2;
        const uint32_t v_at = smem_at(v_base);
#pragma unroll
        for (int k = 0; k < G::kTile / 32; ++k) {   // 32 cells: two products deep
            uint32_t w0[4], w1[4];
            load_matrices(w0, w_at + k * 64);
            load_matrices(w1, w_at + k * 64 + 32);
            if constexpr (kInt8) {
#pragma unroll
                for (int j = 0; j < G::kCols / 16; ++j) {
                    uint32_t b[4];
                    load_matrices_t(b, v_at + chunk_at<G::kChunks>(k * 32 + lane, warp * G::kCols / 16 + j));
#pragma unroll
                    for (int i = 0; i < 4; ++i) b[i] ^= 0x80808080u;
                    // even columns, odd columns
                    multiply(out[2 * j], w0, codes_to_half<0x4240>(b[0]), codes_to_half<0x4240>(b[1]));
                    multiply(out[2 * j + 1], w0, codes_to_half<0x4341>(b[0]), codes_to_half<0x4341>(b[1]));
                    multiply(out[2 * j], w1, codes_to_half<0x4240>(b[2]), codes_to_half<0x4240>(b[3]));
                    multiply(out[2 * j + 1], w1, codes_to_half<0x4341>(b[2]), codes_to_half<0x4341>(b[3]));
                }
            } else {
#pragma unroll
                for (int j = 0; j < G::kOutTiles / 2; ++j) {
                    uint32_t b[4];
                    const int chunk = warp * G::kOutTiles + j * 2 + (lane >> 4);
                    load_matrices_t(b, v_at + chunk_at<G::kChunks>(k * 32 + (lane & 15), chunk));
                    multiply(out[2 * j], w0, b[0], b[1]);
                    multiply(out[2 * j + 1], w0, b[2], b[3]);
                    load_matrices_t(b, v_at + chunk_at<G::kChunks>(k * 32 + 16 + (lane & 15), chunk));
                    multiply(out[2 * j], w1, b[0], b[1]);
                    multiply(out[2 * j + 1], w1, b[2], b[3]);
                }
            }
        }

        // ---- the item's end, or the share's
        if (here.tile + 1 == here.tiles || n + 1 == count) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
                sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
                if (c == 0) s_sum[warp][g + h * 8] = sum[h];
            }
            meet();
            const bool whole = first_tile == 0 && here.tile + 1 == here.tiles;
            const int slot = first_tile == 0 ? 1 : 0;
            const int kv = kv_of(here, p), first = (here.item - kv * p.blocks) * kRows;
            float fit = 1.0f / 32768.0f;
            if constexpr (kInt8) {
#pragma unroll
                for (int i = 0; i < G::kGroups; ++i)
                    if (i == group) fit *= power_of_two(powers[i]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = first + g + h * 8;
                float l = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) l += s_sum[w][g + h * 8];
                if (r < p.group) {
                    const int64_t head = (int64_t) kv * p.group + r;
                    const float by = whole ? (l != 0.0f ? fit / l : 0.0f) : fit;
                    T* to = static_cast<T*>(a.out) + (int64_t) here.seq * a.out_stride + head * kDim;
                    float* part = p.part_o + (((int64_t) blockIdx.x * 2 + slot) * kRows + g + h * 8) * kDim;
#pragma unroll
                    for (int i = 0; i < G::kOutTiles; ++i) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            int d;
                            if constexpr (!kInt8) d = warp * G::kCols + i * 8 + 2 * c + j;
                            else d = warp * G::kCols + (i >> 1) * 16 + 4 * c + 2 * j + (i & 1);
                            // an empty row (nothing held, or minus infinity throughout) is zeros
                            const float x = whole && l == 0.0f ? 0.0f : out[i][h * 2 + j] * by;
                            if (whole) to[d] = Pair<T>::one(x);
                            else part[d] = x;
                        }
                    }
                    if (warp == 0 && c == 0) {
                        if (!whole) p.part_ml[((int64_t) blockIdx.x * 2 + slot) * kRows + g + h * 8] = make_float2(top[h], l);
                        else if (a.lse)
                            a.lse[(int64_t) here.seq * a.n_head + head] = l != 0.0f ? (top[h] + log2f(l)) * 0.6931471805599453f : -INFINITY;
                    }
                }
            }
            if (tid == 0 && n + 1 == count) {
                const int64_t last = s_share[0] + n + (here.tiles - 1 - here.tile);   // the item's last tile, and the share that has it
                const int64_t holder = quotient((last + 1) * s_share[2] - 1, s_share[1]);
                p.cut[blockIdx.x] = !whole && slot == 1 ? make_int2(here.seq * items + here.item, (int) (holder - blockIdx.x) + 1) : make_int2(-1, 0);
            }
            if (n + 1 < count) {
                step<G::kTile>(here, p, items);
                first_tile = 0;
                clear();
                load_query();
            }
        } else {
            ++here.tile;
        }
    }
    wait_async<0>();
}

/// Joins the parts of the items that a share began and others went on with: each part counts by 2^(its maximum - the
/// largest), in the order of the shares.  A task is one head of one cut item, or, where there are fewer of them than CTAs
/// (one long sequence leaves 148 parts of each of 24 heads on 2 CTAs per SM), a piece of its columns.
template <typename T, int kDim>
__global__ void __launch_bounds__(kJoinThreads, 8) join_kernel(const __grid_constant__ AttnDev p, int shares) {
    constexpr int kTrips = (kMaxSms * 4 + kJoinThreads - 1) / kJoinThreads, kJoinWarps = kJoinThreads / 32, kBatch = 6;
    __shared__ int s_count[kTrips * kJoinWarps];
    __shared__ int4 s_cut[kMaxSms * 4];   // the share that began it, the item, its parts
    __shared__ float s_weight[kMaxSms * 4];
    __shared__ float s_top[kJoinWarps], s_sum[kJoinWarps];
    __shared__ float4 s_out[kJoinThreads];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rows = min(p.group, kRows), items = p.layer.n_head_kv * p.blocks;
    wait_for_previous();
    // the cut items, in order
    int2 cut[kTrips];
    uint32_t mask[kTrips];
#pragma unroll
    for (int t = 0; t < kTrips; ++t) {
        const int i = t * kJoinThreads + tid;
        cut[t] = i < shares ? __ldcg(p.cut + i) : make_int2(-1, 0);
    }
#pragma unroll
    for (int t = 0; t < kTrips; ++t) {
        mask[t] = __ballot_sync(0xffffffffu, cut[t].x >= 0);
        if (lane == 0) s_count[t * kJoinWarps + warp] = __popc(mask[t]);
    }
    __syncthreads();
    int cuts = 0;
#pragma unroll
    for (int t = 0; t < kTrips; ++t)
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) {
            if (w == warp && cut[t].x >= 0)
                s_cut[cuts + __popc(mask[t] & ((1u << lane) - 1u))] = make_int4(t * kJoinThreads + tid, cut[t].x, cut[t].y, 0);
            cuts += s_count[t * kJoinWarps + w];
        }
    __syncthreads();
    int pieces = 1;
    while (pieces < kDim / 32 && cuts * rows * pieces * 2 <= (int) gridDim.x) pieces *= 2;
    const int lanes = kDim / 4 / pieces, sets = kJoinThreads / lanes;   // four columns a lane
    const int at = tid % lanes, set = tid / lanes;
    for (int task = blockIdx.x; task < cuts * rows * pieces; task += gridDim.x) {
        const int4 of = s_cut[task / (rows * pieces)];
        const int row = task / pieces % rows, piece = task % pieces, n = of.z;
        const int seq = of.y / items, item = of.y % items;
        const int kv = item / p.blocks, r = (item % p.blocks) * kRows + row;
        if (r >= p.group) continue;   // the same for the whole CTA
        const int column = (piece * lanes + at) * 4;
        // part i of the head: the share's second place for the first, the first place of the shares after it
        const auto place = [&](int i) { return (((int64_t) of.x + i) * 2 + (i == 0 ? 1 : 0)) * kRows + row; };
        const auto load = [&](int i) {
            return i < n ? __ldcg(reinterpret_cast<const float4*>(p.part_o + place(i) * kDim + column)) : make_float4(0, 0, 0, 0);
        };
        float4 ahead[kBatch];   // on their way while the weights are worked out
#pragma unroll
        for (int j = 0; j < kBatch; ++j) ahead[j] = load(set + j * sets);
        float top = -INFINITY;
        for (int i = tid; i < n; i += kJoinThreads) top = fmaxf(top, __ldcg(p.part_ml + place(i)).x);
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (lane == 0) s_top[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, s_top[w]);
        float sum = 0.0f;
        for (int i = tid; i < n; i += kJoinThreads) {
            const float2 ml = __ldcg(p.part_ml + place(i));
            const float weight = exp2f(ml.x - (top == -INFINITY ? 0.0f : top));
            s_weight[i] = weight;
            sum = fmaf(weight, ml.y, sum);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) sum += s_sum[w];
        float4 o = make_float4(0, 0, 0, 0);
        for (int i = set; i < n; i += kBatch * sets) {
            float4 x[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) x[j] = ahead[j];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) ahead[j] = load(i + (kBatch + j) * sets);
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const float w = i + j * sets < n ? s_weight[i + j * sets] : 0.0f;
                o.x = fmaf(w, x[j].x, o.x); o.y = fmaf(w, x[j].y, o.y); o.z = fmaf(w, x[j].z, o.z); o.w = fmaf(w, x[j].w, o.w);
            }
        }
        s_out[tid] = o;
        __syncthreads();
        const int64_t head = (int64_t) kv * p.group + r;
        if (set == 0) {
            for (int i = 1; i < min(sets, n); ++i) {
                const float4 x = s_out[i * lanes + at];
                o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
            }
            const float by = 1.0f / sum;
            if (sum == 0.0f) o = make_float4(0, 0, 0, 0);
            else o = make_float4(o.x * by, o.y * by, o.z * by, o.w * by);
            *reinterpret_cast<uint2*>(static_cast<T*>(p.a.out) + (int64_t) seq * p.a.out_stride + head * kDim + column) =
                make_uint2(Pair<T>::down(o.x, o.y), Pair<T>::down(o.z, o.w));
        }
        if (tid == 0 && piece == 0 && p.a.lse)
            p.a.lse[(int64_t) seq * p.a.n_head + head] = sum != 0.0f ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
        __syncthreads();   // the next task writes s_top, s_weight and s_out again
    }
}

template <typename T, int kDim, bool kInt8>
cudaError_t launch(const AttnDev& p, int sms, cudaStream_t stream) {
    constexpr int kSmem = Geo<kDim, kInt8>::kSmem, kPerSm = Geo<kDim, kInt8>::kPerSm;
    static_assert((kSmem + 3 * 1024) * kPerSm <= (int) kSmemPerSm && kPerSm <= 4, "the CTAs fit an SM");
    const int ctas = sms * kPerSm;
    cudaError_t e = cudaFuncSetAttribute(attention_kernel<T, kDim, kInt8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    // (Letting the join in any earlier, while shares still run, costs 2 us a call.)
    e = launch_early(attention_kernel<T, kDim, kInt8>, dim3((unsigned) ctas), kThreads, kSmem, stream, p);
    if (e != cudaSuccess) return e;
    return launch_early(join_kernel<T, kDim>, dim3((unsigned) sms * 8), kJoinThreads, 0, stream, p, ctas);
}
template <typename T>
cudaError_t launch(const AttnDev& p, int dim, bool int8, int sms, cudaStream_t stream) {
    if (dim == 64) return int8 ? launch<T, 64, true>(p, sms, stream) : launch<T, 64, false>(p, sms, stream);
    if (dim == 128) return int8 ? launch<T, 128, true>(p, sms, stream) : launch<T, 128, false>(p, sms, stream);
    return int8 ? launch<T, 256, true>(p, sms, stream) : launch<T, 256, false>(p, sms, stream);
}

/// A call's items and sequences are counted in 32 bits, in steps of up to a grid's CTAs.
bool too_many_items(const skv_kv_layer& l, int n_seqs, int n_head) {
    const int blocks = (n_head / l.n_head_kv + kRows - 1) / kRows;
    return (int64_t) n_seqs * l.n_head_kv * blocks > (1 << 30);
}

/// The workspace: parts, their maxima and sums, the shares' cuts.
struct Room {
    size_t ml, cut, bytes;
    explicit Room(const skv_kv_layer& l) {
        const bool int8 = l.format == SKV_KV_INT8;
        const size_t shares = (size_t) kMaxSms * (l.head_dim == 64 ? per_sm<64>(int8) : l.head_dim == 128 ? per_sm<128>(int8) : per_sm<256>(int8));
        ml = shares * 2 * kRows * l.head_dim * sizeof(float);
        cut = ml + shares * 2 * kRows * sizeof(float2);
        bytes = (cut + shares * sizeof(int2) + 255) / 256 * 256;
    }
    template <int kDim>
    static int per_sm(bool int8) { return int8 ? Geo<kDim, true>::kPerSm : Geo<kDim, false>::kPerSm; }
};

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" {
int skv_decode_attention_workspace(const skv_kv_layer* layer, int n_seqs, int n_head, uint64_t* out_bytes) {
    if (!out_bytes) return fail(SKV_EINVAL, "skv_decode_attention_workspace: null output");
    *out_bytes = 0;
    if (n_seqs < 0 || n_head < 1) return fail(SKV_EINVAL, "skv_decode_attention_workspace: bad counts");
    if (const int rc = check_layer(layer, n_seqs, "skv_decode_attention_workspace")) return rc;
    if (n_head > 4096 || n_head % layer->n_head_kv)
        return fail(SKV_EINVAL, "skv_decode_attention_workspace: n_head must be a multiple of n_head_kv, at most 4096");
    if (too_many_items(*layer, n_seqs, n_head)) return fail(SKV_ERANGE, "skv_decode_attention_workspace: too many sequences and heads");
    *out_bytes = Room(*layer).bytes;
    return SKV_OK;
}

int skv_decode_attention(const skv_kv_layer* layer, const skv_attention_args* args, void* stream) {
    const auto no = [](const char* why) { return fail(SKV_EINVAL, std::string("skv_decode_attention: ") + why); };
    if (!args) return no("no arguments");
    const skv_attention_args& a = *args;
    if (a.n_seqs < 0) return no("n_seqs is negative");
    if (const int rc = check_layer(layer, a.n_seqs, "skv_decode_attention")) return rc;
    if (a.n_head < 1 || a.n_head > 4096 || a.n_head % layer->n_head_kv) return no("n_head must be a multiple of n_head_kv, at most 4096");
    if (a.dtype != SKV_DTYPE_F16 && a.dtype != SKV_DTYPE_BF16) return no("unknown dtype");
    if (!(a.scale > -INFINITY && a.scale < INFINITY)) return no("the scale must be finite");
    if (a.n_seqs == 0) return SKV_OK;
    if (!a.q || !a.out || !a.lengths) return no("missing q, out or lengths");
    if (!ops_aligned4(a.lengths, a.lse)) return no("lengths and lse must be 4-byte aligned");
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
    if (const int rc = check_layer_memory(*layer, ctx->device, "skv_decode_attention")) return rc;
    const Room room(*layer);
    AttnDev p{};
    p.layer = to_device(*layer);
    p.a = a;
    p.status = ctx->status;
    p.group = a.n_head / layer->n_head_kv;
    p.blocks = (p.group + kRows - 1) / kRows;
    p.part_o = static_cast<float*>(a.workspace);
    p.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(a.workspace) + room.ml);
    p.cut = reinterpret_cast<int2*>(static_cast<uint8_t*>(a.workspace) + room.cut);
    const int sms = ctx->sms < kMaxSms ? ctx->sms : kMaxSms;
    const auto s = static_cast<cudaStream_t>(stream);
    const bool int8 = layer->format == SKV_KV_INT8;
    const cudaError_t e = a.dtype == SKV_DTYPE_F16 ? launch<__half>(p, layer->head_dim, int8, sms, s)
                                                   : launch<__nv_bfloat16>(p, layer->head_dim, int8, sms, s);
    return e == cudaSuccess ? SKV_OK : cuda_fail(e, "skv_decode_attention");
}

}  // extern "C"

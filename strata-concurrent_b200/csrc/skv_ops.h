// skv_ops.h - what the operators on a cache and a state row share: argument checks on the host, small device helpers.
#pragma once

#include "skv_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace skv {

/// Values per scale of an int8 cell (KV_Q8_GROUP of the parked format).
constexpr int kInt8Group = 64;

/// Every one of the arrays of 32-bit values lies on a multiple of their size (none counts as well).
template <typename... P>
bool ops_aligned4(const P*... p) {
    return ((reinterpret_cast<uintptr_t>(p) | ...) & 3u) == 0;
}
inline bool ops_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

/// True when `p` is memory of `device` itself: a host address or another GPU's memory is refused before a launch.
inline bool ops_own_memory(const void* p, int device) {
    cudaPointerAttributes a{};
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
        (void) cudaGetLastError();
        return false;
    }
    return (a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged) && a.device == device;
}

/// Refuses a layer that the kernels cannot address; SKV_OK otherwise.
int check_layer(const skv_kv_layer* layer, int n_seqs, const char* what);
/// Refuses a layer whose pools or scales are not memory of `device`; SKV_OK otherwise.
int check_layer_memory(const skv_kv_layer& layer, int device, const char* what);

/// A layer as the kernels take it.
struct LayerDev {
    uint8_t* k;
    uint8_t* v;
    __half* k_scale;
    __half* v_scale;
    const int32_t* tables;
    int64_t table_stride;
    int64_t page_limit;
    int32_t n_head_kv;
    int32_t page_shift;   // page_size = 1 << page_shift
};

LayerDev to_device(const skv_kv_layer& layer);

// ---------------------------------------------------------------- device helpers

#ifdef __CUDACC__

template <typename T>
struct Pair;   // two values in one register
template <>
struct Pair<__half> {
    static __device__ __forceinline__ float2 up(uint32_t r) { return __half22float2(*reinterpret_cast<const __half2*>(&r)); }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ __half one(float a) { return __float2half_rn(a); }
};
template <>
struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ float2 up(uint32_t r) {
        return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ __nv_bfloat16 one(float a) { return __float2bfloat16_rn(a); }
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& r, float (&x)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = Pair<T>::up(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return make_uint4(Pair<T>::down(x[0], x[1]), Pair<T>::down(x[2], x[3]), Pair<T>::down(x[4], x[5]),
                      Pair<T>::down(x[6], x[7]));
}

/// A kernel launched with launch_early begins with this: whatever ran before on the stream has then ended.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

/// A launch that may be set up while the kernel before it on the stream ends; the kernel waits for that one itself.  One
/// step of the delta rule in a graph of them takes 2.2 us so, 2.7 without; attention over 1,000 cells, two kernels, 11.4 and 14.4.
template <typename... Parameters, typename... Arguments>
cudaError_t launch_early(void (*kernel)(Parameters...), dim3 grid, int threads, size_t smem, cudaStream_t stream, const Arguments&... arguments) {
    cudaLaunchConfig_t config{};
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    config.stream = stream;
    config.gridDim = grid;
    config.blockDim = dim3((unsigned) threads);
    config.dynamicSmemBytes = smem;
    return cudaLaunchKernelEx(&config, kernel, arguments...);
}

/// The row (page * n_head_kv + head) * page_size + slot of a cell: values at row * head_dim, scales at row * head_dim / 64.
/// Negative when the cell lies past the table or its entry outside the pool.
__device__ __forceinline__ int64_t cell_row(const LayerDev& l, int seq, int64_t cell, int head) {
    const int64_t p = cell >> l.page_shift;
    if (cell < 0 || p >= l.table_stride) return -1;
    const int64_t page = __ldg(l.tables + (int64_t) seq * l.table_stride + p);
    if (page < 0 || page >= l.page_limit) return -1;
    return ((page * l.n_head_kv + head) << l.page_shift) + (cell & ((1 << l.page_shift) - 1));
}

#endif

}  // namespace skv

// model.cuh -- what the operators of include/lcpp_b200_model.h share: row
// element types, 16-byte vectors of them, argument checks and the guard that
// keeps C++ exceptions inside the library.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/lcpp_b200_model.h"
#include "common.cuh"

namespace lcpp {
namespace model {

// LCPP_KERNEL_BLOCK_TABLE / _ROUTER / _DISPATCH (include/lcpp_b200_diag.h)
constexpr int kTimerBlockTable = 9, kTimerRouter = 10, kTimerDispatch = 11;

inline int row_dtype_bytes(lcpp_dtype dt)
{
    switch (dt) {
    case LCPP_F32: return 4;
    case LCPP_F16: case LCPP_BF16: return 2;
    default: return 0;
    }
}

inline bool misaligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

// Both ranges non-empty and at least one byte in common.
inline bool overlap(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && a_bytes && b_bytes && x < y + b_bytes && y < x + a_bytes;
}

// An array that a call reads or writes.
struct Array {
    const void* p;
    uint64_t bytes;
    bool written;
};

// Some two of them, one written, share a byte: blocks read an input while
// another one writes the outputs, and two outputs hold different things.
template <size_t N>
bool clash(const Array (&arrays)[N])
{
    for (size_t i = 0; i < N; ++i)
        for (size_t j = 0; j < i; ++j)
            if ((arrays[i].written || arrays[j].written) &&
                overlap(arrays[i].p, arrays[i].bytes, arrays[j].p, arrays[j].bytes))
                return true;
    return false;
}

// Bytes from the first to the last element of `rows` strided rows.
inline uint64_t span_bytes(uint64_t rows, uint64_t stride, uint64_t columns, int element)
{
    return rows ? ((rows - 1) * stride + columns) * uint64_t(element) : 0;
}

// An array has a byte in common with the elements of strided rows; it may lie
// in what is left between them.
inline bool overlap_rows(const void* base, uint64_t rows, uint64_t stride, uint64_t columns, int element, const void* a,
                         uint64_t bytes)
{
    if (!columns || !overlap(base, span_bytes(rows, stride, columns, element), a, bytes)) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(base), y = reinterpret_cast<uintptr_t>(a);
    if (rows == 1 || y < x) return true;
    const uint64_t pitch = stride * uint64_t(element), at = (y - x) % pitch;
    return at < columns * uint64_t(element) || bytes > pitch - at;
}

// 16-byte loads and stores need every row to start on a 16-byte boundary.
inline bool rows_16b(const void* p, uint64_t stride, int element)
{
    return !misaligned(p, 16) && stride * uint64_t(element) % 16 == 0;
}

// Runs a C entry point's body; an exception (the attribute caches allocate)
// becomes a status.
template <typename F>
lcpp_status guarded(const char* name, F&& body) noexcept
{
    try {
        diag::Range range(name);
        return body();
    } catch (...) {
        return LCPP_ERR_INTERNAL;
    }
}

// Launches `kernel` without waiting for the launch before it on the stream to
// end: the kernel itself waits (wait_for_previous) before it touches what that
// one writes.  The launch before must be the same call's.
template <typename... P>
lcpp_status launch_early(void (*kernel)(P...), unsigned grid, int block, size_t smem, cudaStream_t s, P... args)
{
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(block);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    config.attrs = &early;
    config.numAttrs = 1;
    LCPP_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, args...));
    return LCPP_OK;
}
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

inline lcpp_status launched() { return cudaGetLastError() == cudaSuccess ? LCPP_OK : LCPP_ERR_CUDA; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of elements as floats and back.
template <typename T>
struct Vec {
    static constexpr int kN = 16 / int(sizeof(T));
    static __device__ __forceinline__ void unpack(const uint4& raw, float (&out)[kN])
    {
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int i = 0; i < kN; ++i) out[i] = to_float(e[i]);
    }
    static __device__ __forceinline__ uint4 pack(const float (&in)[kN])
    {
        uint4 raw;
        T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int i = 0; i < kN; ++i) e[i] = from_float<T>(in[i]);
        return raw;
    }
};

template <typename F>
lcpp_status with_row_type(lcpp_dtype dt, F&& fn)
{
    switch (dt) {
    case LCPP_F32: return fn(float{});
    case LCPP_F16: return fn(__half{});
    case LCPP_BF16: return fn(__nv_bfloat16{});
    default: return LCPP_ERR_UNSUPPORTED_DTYPE;
    }
}

}  // namespace model
}  // namespace lcpp

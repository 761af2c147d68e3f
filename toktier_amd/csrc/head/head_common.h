// Shared parts of the answering end's kernels: argument checks, launches,
// 16-byte pieces and wave reductions.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include "../../../include/toktier_head.h"

namespace tkh {

// ---- host side

// Records the message of tk_head_last_error and returns the status.
int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// The same for an error of the HIP runtime, which is left with none.
int fail_hip(const char* what, hipError_t e);

// Makes `device` current for a call and restores the caller's device after;
// refuses a device that is not a gfx950.
class DeviceScope {
public:
    explicit DeviceScope(int device);
    ~DeviceScope();
    int status() const { return status_; }

private:
    int prev_ = -1, status_ = TKH_OK;
};

template <typename... Params, typename... Args>
int launch(const char* name, void (*kernel)(Params...), dim3 grid, dim3 block, size_t lds,
           void* stream, Args... args) {
    static_assert(sizeof...(Params) == sizeof...(Args), "kernel arguments");
    return [&](Params... p) {
        void* ptrs[] = {(void*)&p...};
        hipError_t e = hipLaunchKernel((const void*)kernel, grid, block, ptrs, lds,
                                       (hipStream_t)stream);
        return e == hipSuccess ? TKH_OK : fail_hip(name, e);
    }(static_cast<Params>(args)...);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether workgroups of so many threads fit one launch: fewer than 2^32
// threads along an axis.
inline bool fits_launch(int64_t groups, int64_t threads) { return groups <= 0xffffffffll / threads; }

// ---- device side

constexpr int kBlock = 128;  // values that share a scale

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

template <typename T> struct Num;
template <> struct Num<float> {
    static __device__ float get(float v) { return v; }
    static __device__ float put(float v) { return v; }
};
template <> struct Num<__hip_bfloat16> {
    // the upper half of a float; rounded to nearest even, NaN kept
    static __device__ float get(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ uint16_t put(float v) {
        __bf16 b = (__bf16)v;
        return __builtin_bit_cast(uint16_t, b);
    }
};
template <> struct Num<__half> {
    static __device__ float get(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ uint16_t put(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// How a type lies in memory: 16-bit floats are handled by their bits.
template <typename T> struct Raw { typedef uint16_t type; };
template <> struct Raw<float> { typedef float type; };

// N consecutive values from an address aligned to one value. gfx950 reads
// and writes wide words at any such address, so this is one instruction for
// up to 16 bytes whatever the row's alignment.
template <typename R, int N> struct __attribute__((packed, aligned(sizeof(R)))) Pack {
    R v[N];
};

template <typename R, int N>
__device__ __forceinline__ void load_pack(R (&dst)[N], const R* src) {
    const Pack<R, N> p = *reinterpret_cast<const Pack<R, N>*>(src);
#pragma unroll
    for (int i = 0; i < N; ++i) dst[i] = p.v[i];
}

template <typename R, int N>
__device__ __forceinline__ void store_pack(R* dst, const R (&src)[N]) {
    Pack<R, N> p;
#pragma unroll
    for (int i = 0; i < N; ++i) p.v[i] = src[i];
    *reinterpret_cast<Pack<R, N>*>(dst) = p;
}

}  // namespace tkh

#pragma once
// What the paged cache's kernels share: the cache as a kernel sees it, element
// conversions, and each token's visible keys (HIP sources only).
#include <hip/hip_runtime.h>

#include <cstdint>

#include "gfd_capi.h"

namespace gfd {
namespace kv {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Element types: how a 32-bit word holds them.
struct Bf16 {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {  // nearest even
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
    }
    static __device__ __forceinline__ f32x2 unpack(uint32_t w) {
        return f32x2{__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)};
    }
};
struct Fp16 {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), f16x2));
    }
    static __device__ __forceinline__ f32x2 unpack(uint32_t w) {
        return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
    }
};
struct E4m3 {
    static constexpr int kBytes = 1;
};

// n / d for 0 <= n < 2^31 by a multiplication: floor(n * mul / 2^(32 + shift))
// with mul = ceil(2^(32 + shift) / d), shift = ceil(log2 d) - 1 (d = 1: n
// itself).  mul is below 2^32, and its excess over 2^(32 + shift) / d is less
// than 1, so the quotient's is less than n / 2^(32 + shift) <= 1 / d: exact.
struct Divider {
    uint32_t d, mul, shift;
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return d == 1 ? n : __umulhi(n, mul) >> shift; }
};
inline Divider make_divider(uint32_t d) {
    Divider r{d, 0, 0};
    if (d > 1) {
        uint32_t bits = 0;
        while ((1ull << bits) < d) bits++;
        r.shift = bits - 1;
        r.mul = (uint32_t)(((1ull << (32 + r.shift)) + d - 1) / d);
    }
    return r;
}

// The cache with strides in bytes.
struct Cache {
    uint8_t* k;
    uint8_t* v;
    int64_t page_stride, slot_stride, head_stride;
    int num_pages;
    Divider page;
    float k_scale, v_scale;  // 1 unless the type is E4M3
};

// A launch has fewer threads along a grid than this.
constexpr int64_t kGridThreads = 1ll << 32;
// Launches, and returns this launch's own status: the last error of the thread may be an earlier call's.
template <typename... P>
int start(void (*kernel)(P...), dim3 grid, int threads, hipStream_t st, const P&... args) {
    void* pointers[] = {const_cast<P*>(&args)...};
    const hipError_t e = hipLaunchKernel((const void*)kernel, grid, dim3((unsigned)threads), pointers, 0, st);
    if (e != hipSuccess) (void)hipGetLastError();  // it is returned, and is no later call's
    return (int)e;
}
// The text behind gfd_last_error() for a refused call, or one whose launch failed with rc; returns the call's result.
int refused(const char* name, const char* why);
int launched(const char* name, int rc);

// An argument that a kernel for the cache relies on, or NULL if all hold.
const char* check_cache(const gfd_kv_cache* c);
Cache make_cache(const gfd_kv_cache& c);

}  // namespace kv
}  // namespace gfd

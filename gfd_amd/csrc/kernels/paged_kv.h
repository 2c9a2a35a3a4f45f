#pragma once
// What the paged cache's kernels share: the cache as a kernel sees it, element
// conversions, and each token's visible keys (HIP sources only).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

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
    static constexpr int kBits = 16;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {  // nearest even
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
    }
    static __device__ __forceinline__ f32x2 unpack(uint32_t w) {
        return f32x2{__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)};
    }
};
struct Fp16 {
    static constexpr int kBits = 16;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), f16x2));
    }
    static __device__ __forceinline__ f32x2 unpack(uint32_t w) {
        return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
    }
};
struct E4m3 {
    static constexpr int kBits = 8;
};
// 4-bit floats, kGroup4 of them with a power of two, whose exponent is a byte (255: NaN).
struct E2m1 {
    static constexpr int kBits = 4;
};
constexpr int kGroup4 = 32;
constexpr int kScaleNan = 255;
// The scales that an append writes: 6 times the largest is finite in the rows' type (8 times it would not be), half of
// the least is the least that the type tells from zero (bf16: its least of full precision).
template <typename T>
struct ScaleRange;
template <>
struct ScaleRange<Bf16> {
    static constexpr int kLeast = 1, kMost = 252;
};
template <>
struct ScaleRange<Fp16> {
    static constexpr int kLeast = 104, kMost = 140;
};
// A scale as the conversions take it.  One beyond what an append writes would leave some numbers of its group infinite and
// others not: it is read as NaN, so that a group's numbers are finite all together or not at all.
template <typename T>
__device__ __forceinline__ float scale_of(uint32_t byte) {
    return __uint_as_float((byte > (uint32_t)ScaleRange<T>::kMost ? (uint32_t)kScaleNan : byte) << 23);
}
// The same for four scales in a word: bytes above kMost become kScaleNan.
template <typename T>
__device__ __forceinline__ uint32_t read_scales(uint32_t w) {
    constexpr uint32_t kRest = 0x7Fu - (ScaleRange<T>::kMost & 0x7Fu);  // added to 7 bits, sets the eighth above kMost
    static_assert(ScaleRange<T>::kMost >= 128, "the eighth bit is set too");
    const uint32_t hot = ((w & 0x7F7F7F7Fu) + kRest * 0x01010101u) & w & 0x80808080u;
    return w | ((hot << 1) - (hot >> 7));
}
// Two numbers, byte `byte` of w, as a pair of T: the first in the low half of the byte and of the pair.
template <typename T>
__device__ __forceinline__ uint32_t widen4(uint32_t w, int byte, float scale) {
    static_assert(std::is_same<T, Bf16>::value || std::is_same<T, Fp16>::value, "rows are bf16 or fp16");
    if constexpr (std::is_same<T, Bf16>::value) {
        const auto at = [&](auto b) {
            return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, decltype(b)::value));
        };
        return byte == 0   ? at(std::integral_constant<int, 0>())
               : byte == 1 ? at(std::integral_constant<int, 1>())
               : byte == 2 ? at(std::integral_constant<int, 2>())
                           : at(std::integral_constant<int, 3>());
    } else {
        const auto at = [&](auto b) {
            return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, decltype(b)::value));
        };
        return byte == 0   ? at(std::integral_constant<int, 0>())
               : byte == 1 ? at(std::integral_constant<int, 1>())
               : byte == 2 ? at(std::integral_constant<int, 2>())
                           : at(std::integral_constant<int, 3>());
    }
}
template <typename T>
__device__ __forceinline__ u32x4 widen4(uint32_t w, float scale) {  // all eight
    return u32x4{widen4<T>(w, 0, scale), widen4<T>(w, 1, scale), widen4<T>(w, 2, scale), widen4<T>(w, 3, scale)};
}

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
// Of 4-bit numbers, with their scales, whose offset within a page is a 16th of the numbers'.  Apart, as small calls of other types
// take longer with larger arguments (a prefix of 1024 keys for 8 requests: 14.0 us, with them 14.2).
struct Cache4 : Cache {
    uint8_t* k_scales;
    uint8_t* v_scales;
    int64_t scale_page_stride;
    int heads_inner;  // a slot's heads are neighbours
};
template <typename S>
using CacheOf = typename std::conditional<S::kBits == 4, Cache4, Cache>::type;

// Byte offsets of a row (slot and head of a page): of its numbers, and of 4-bit ones' scales.
struct Place4 {
    int64_t row, scales;
};
template <typename S>
using Place = typename std::conditional<S::kBits == 4, Place4, int64_t>::type;
template <typename S>
__device__ __forceinline__ Place<S> place_of(const CacheOf<S>& c, int page, uint32_t slot, int64_t head) {
    const int64_t in = slot * c.slot_stride + head;
    if constexpr (S::kBits == 4) return Place4{page * c.page_stride + in, page * c.scale_page_stride + (in >> 4)};
    else return page * c.page_stride + in;
}
__device__ __forceinline__ int64_t numbers_at(int64_t p) { return p; }
__device__ __forceinline__ int64_t numbers_at(const Place4& p) { return p.row; }

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
const char* check_cache(const gfd_kv4_cache* c);
Cache make_cache(const gfd_kv_cache& c);
Cache4 make_cache(const gfd_kv4_cache& c);

}  // namespace kv
}  // namespace gfd

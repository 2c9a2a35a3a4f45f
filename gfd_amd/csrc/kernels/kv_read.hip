// Tokens' keys and values back out of the paged cache, as rows (gfx950): a
// copy of 16-bit numbers, 8- and 4-bit ones widened and scaled on the way.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gfd_capi.h"
#include "paged_attention.h"

namespace gfd {
namespace kv {
namespace {

constexpr int kBlock = 256;

struct ReadRows {
    uint16_t* k;
    uint16_t* v;
    int64_t k_stride, v_stride;
    const int64_t* slots;
    int num_tokens, heads, dim;
    int* error;
};

// 8 values of a row of type S, from value a on, as rows have them.
template <typename T, typename S>
__device__ __forceinline__ u32x4 eight(const uint8_t* base, const uint8_t* scales, const Place<S>& place, int a, float scale) {
    const uint8_t* p = base + numbers_at(place) + a * S::kBits / 8;
    if constexpr (S::kBits == 16) {
        return *(const u32x4*)p;
    } else if constexpr (S::kBits == 8) {
        const u32x2 w = *(const u32x2*)p;
        u32x4 y;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const auto x = (i & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i / 2], true)
                                   : __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i / 2], false);
            y[i] = T::pack(x[0] * scale, x[1] * scale);
        }
        return y;
    } else {
        return widen4<T>(*(const uint32_t*)p, scale_of<T>(scales[place.scales + a / kGroup4]));
    }
}

constexpr int kUnits = 2;  // a thread's, at once

// A thread takes the same 8 dims of a key and of its value, kUnits times; neighbours are neighbours in the rows.  Bound by
// the bytes: 16384 tokens of 8 heads of 128 in 4 bits, 85 MB in 17.5 us behind the append that wrote them.  Calls back to
// back over three caches by turns, pages in any order: 16 bits 134 MB in 28.6 us (4.7 TB/s), 8 bits 101 MB in 23.9, 4 bits 21.1; 1000
// tokens 3.9, 4.2, 4.0, a launch.
template <typename T, typename S>
__global__ __launch_bounds__(kBlock) void kv_read_kernel(ReadRows r, CacheOf<S> c, Divider per_token) {
    const int shift = r.dim == 64 ? 3 : r.dim == 128 ? 4 : 5;  // units of 8 values a head
    const uint8_t *k_scales = nullptr, *v_scales = nullptr;
    if constexpr (S::kBits == 4) k_scales = c.k_scales, v_scales = c.v_scales;
    const int64_t units = (int64_t)r.num_tokens * per_token.d, step = (int64_t)gridDim.x * kBlock * kUnits;
    for (int64_t first = (int64_t)blockIdx.x * kBlock * kUnits; first < units; first += step) {
        u32x4 k[kUnits], v[kUnits];
        int64_t t[kUnits];
        int to[kUnits];
        // The workgroup's first token, and the units from its start on: within 32 bits.
        const int64_t t0 = first / per_token.d;
        const int rest = (int)(first - t0 * per_token.d) + (int)threadIdx.x;
#pragma unroll
        for (int i = 0; i < kUnits; i++) {
            const uint32_t n = (uint32_t)(rest + i * kBlock), u = per_token.div(n);
            t[i] = t0 + u;
            const int unit = (int)(n - u * per_token.d), head = unit >> shift, a = 8 * (unit & ((1 << shift) - 1));
            to[i] = head * r.dim + a;
            const int64_t slot = t[i] < r.num_tokens ? r.slots[t[i]] : -1;
            if (slot >= (int64_t)c.num_pages * c.page.d && r.error && unit == 0) atomicOr(r.error, GFD_KV_ERR_PAGE);
            if (slot < 0 || slot >= (int64_t)c.num_pages * c.page.d) {
                t[i] = -1;
                continue;
            }
            const int64_t page = slot / c.page.d;
            const auto place = place_of<S>(c, (int)page, (uint32_t)(slot - page * c.page.d), head * c.head_stride);
            if (r.k) k[i] = eight<T, S>(c.k, k_scales, place, a, c.k_scale);
            if (r.v) v[i] = eight<T, S>(c.v, v_scales, place, a, c.v_scale);
        }
#pragma unroll
        for (int i = 0; i < kUnits; i++) {
            if (t[i] < 0) continue;
            if (r.k) *(u32x4*)(r.k + t[i] * r.k_stride + to[i]) = k[i];
            if (r.v) *(u32x4*)(r.v + t[i] * r.v_stride + to[i]) = v[i];
        }
    }
}

template <typename T, typename S>
int launch(const ReadRows& r, const CacheOf<S>& c, hipStream_t st) {
    const int per_token = r.heads * (r.dim / 8);
    const int64_t groups = ((int64_t)r.num_tokens * per_token + kBlock * kUnits - 1) / (kBlock * kUnits);
    return start(kv_read_kernel<T, S>, dim3((unsigned)std::min<int64_t>(groups, 1 << 20)), kBlock, st, r, c,
                 make_divider((uint32_t)per_token));
}

const char* check(const gfd_kv_read_rows* rows) {
    if (!rows) return "no rows";
    const gfd_kv_read_rows& w = *rows;
    if (w.dtype != GFD_BF16 && w.dtype != GFD_FP16) return "rows are neither GFD_BF16 nor GFD_FP16";
    if (w.num_tokens < 0) return "negative num_tokens";
    if ((w.k_stride | w.v_stride) % 8 != 0 || ((uintptr_t)w.k | (uintptr_t)w.v) % 16 != 0)
        return "rows' pointers or strides are not multiples of 16 bytes";
    if (w.num_tokens && !w.slots) return "slots is missing";
    return nullptr;
}

template <typename C>
ReadRows make(const gfd_kv_read_rows& w, const C& c, int* error) {
    return ReadRows{(uint16_t*)w.k, (uint16_t*)w.v, w.k_stride, w.v_stride, w.slots, w.num_tokens, c.num_heads,
                    c.head_dim, error};
}

}  // namespace
}  // namespace kv
}  // namespace gfd

extern "C" int gfd_kv_read(const gfd_kv_cache* cache, const gfd_kv_read_rows* rows, int* error_flag, void* stream) {
    using namespace gfd::kv;
    constexpr char kName[] = "gfd_kv_read";
    if (const char* why = check_cache(cache)) return refused(kName, why);
    if (const char* why = check(rows)) return refused(kName, why);
    if (cache->dtype != GFD_E4M3 && cache->dtype != rows->dtype)
        return refused(kName, "the cache's type is neither the rows' nor GFD_E4M3");
    if (rows->num_tokens == 0 || (!rows->k && !rows->v)) return 0;
    const ReadRows r = make(*rows, *cache, error_flag);
    const auto c = make_cache(*cache);
    const hipStream_t st = (hipStream_t)stream;
    if (cache->dtype == GFD_E4M3)
        return launched(kName, rows->dtype == GFD_BF16 ? launch<Bf16, E4m3>(r, c, st) : launch<Fp16, E4m3>(r, c, st));
    return launched(kName, launch<Bf16, Bf16>(r, c, st));  // bits, of either type
}

extern "C" int gfd_kv4_read(const gfd_kv4_cache* cache, const gfd_kv_read_rows* rows, int* error_flag, void* stream) {
    using namespace gfd::kv;
    constexpr char kName[] = "gfd_kv4_read";
    if (const char* why = check_cache(cache)) return refused(kName, why);
    if (const char* why = check(rows)) return refused(kName, why);
    if (rows->num_tokens == 0 || (!rows->k && !rows->v)) return 0;
    const ReadRows r = make(*rows, *cache, error_flag);
    const auto c = make_cache(*cache);
    const hipStream_t st = (hipStream_t)stream;
    return launched(kName, rows->dtype == GFD_BF16 ? launch<Bf16, E2m1>(r, c, st) : launch<Fp16, E2m1>(r, c, st));
}

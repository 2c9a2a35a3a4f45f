// Appending a step's keys and values to the paged cache, with the position
// rotation of queries and keys on the way (gfx950).
//
// Pair (a, b) of a head at position p: angle = p * inv_freq, a' = a cos - b
// sin, b' = b cos + a sin.  The angle's whole turns are taken off in 64 bits
// (p * inv_freq / 2 pi is off by 2^-53 of itself there; in 32 bits a position of
// 2^20 would be off by 0.06), the rotation is computed in 32 bits and rounded once to the
// stored type.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>

#include "capi_error.h"
#include "gfd_capi.h"
#include "paged_kv.h"

namespace gfd {
namespace kv {

const char* check_cache(const gfd_kv_cache* c) {
    if (!c || !c->k || !c->v) return "no cache";
    if (c->dtype != GFD_BF16 && c->dtype != GFD_FP16 && c->dtype != GFD_E4M3) return "unknown cache type";
    if (c->num_pages < 1 || c->page_size < 1 || c->page_size > 65536 || c->num_heads < 1 || c->num_heads > 65535)
        return "cache sizes out of range";
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return "head_dim is not 64, 128 or 256";
    const int64_t per16 = c->dtype == GFD_E4M3 ? 16 : 8;
    if (((uintptr_t)c->k | (uintptr_t)c->v) % 16 != 0 || c->page_stride % per16 != 0 || c->slot_stride % per16 != 0 ||
        c->head_stride % per16 != 0)
        return "cache pointers or strides are not multiples of 16 bytes";
    if (c->page_stride < 0 || c->slot_stride < 0 || c->head_stride < 0) return "negative cache stride";
    if (c->dtype == GFD_E4M3 && !(c->k_scale > 0 && c->v_scale > 0 && c->k_scale <= 3.4e38f && c->v_scale <= 3.4e38f))
        return "k_scale and v_scale of an 8-bit cache are positive and finite";
    return nullptr;
}

Cache make_cache(const gfd_kv_cache& c) {
    const int64_t size = c.dtype == GFD_E4M3 ? 1 : 2;
    const bool scaled = c.dtype == GFD_E4M3;
    return Cache{(uint8_t*)c.k, (uint8_t*)c.v, c.page_stride * size, c.slot_stride * size, c.head_stride * size,
                 c.num_pages, make_divider((uint32_t)c.page_size), scaled ? c.k_scale : 1.f, scaled ? c.v_scale : 1.f};
}

namespace {

struct Rows {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const int* positions;
    const int64_t* slots;
    const float* inv_freq;
    int num_tokens, q_heads, kv_heads, dim, rotary;
    float k_div, v_div;  // stored = x / div
    int* error;
};

constexpr int kBlock = 256;

template <typename T>
__device__ __forceinline__ float load_one(const uint16_t* p) {
    return T::unpack(*p)[0];
}

// Two values to the stored type, in the low bits of the result.
template <typename T>
struct Store {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ void one(uint8_t* p, float x) { *(uint16_t*)p = (uint16_t)T::pack(x, 0.f); }
};
template <>
struct Store<E4m3> {
    static constexpr int kBytes = 1;
    static __device__ __forceinline__ void one(uint8_t* p, float x) {
        const float y = x != x ? x : fminf(fmaxf(x, -448.f), 448.f);
        *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, 0.f, 0, false);
    }
};

// One workgroup per token; a thread per element of its heads' halves.
template <typename T, typename S, bool kPairs>
__global__ __launch_bounds__(kBlock) void kv_append_kernel(Rows r, Cache c) {
    __shared__ f32x2 turn[128];
    const int t = (int)blockIdx.x, half = r.rotary / 2;
    for (int i = (int)threadIdx.x; i < half; i += kBlock) {
        const double turns = (double)r.positions[t] * ((double)r.inv_freq[i] * 0.15915494309189533577);
        float s, co;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &co);
        turn[i] = f32x2{co, s};
    }
    __syncthreads();
    const int64_t slot = r.slots[t];
    const bool inside = slot < (int64_t)c.num_pages * c.page.d;
    if (!inside && threadIdx.x == 0 && r.error) atomicOr(r.error, GFD_KV_ERR_PAGE);
    const int64_t page = slot / c.page.d, at = page * c.page_stride + (slot - page * c.page.d) * c.slot_stride;
    const int units = r.dim / 2;
    const int first = r.q ? 0 : r.q_heads;
    for (int u = first * units + (int)threadIdx.x; u < (r.q_heads + 2 * r.kv_heads) * units; u += kBlock) {
        const int h = u / units, i = u - h * units;
        const bool is_q = h < r.q_heads, is_v = h >= r.q_heads + r.kv_heads;
        const int head = is_q ? h : is_v ? h - r.q_heads - r.kv_heads : h - r.q_heads;
        const bool turned = i < half;
        // Past the rotated dims the pairs are neighbours.
        const int ia = turned && !kPairs ? i : 2 * i, ib = turned && !kPairs ? i + half : 2 * i + 1;
        const uint16_t* src = is_q ? r.q + t * r.q_stride : is_v ? r.v + t * r.v_stride : r.k + t * r.k_stride;
        const int va = is_v ? 2 * i : ia, vb = is_v ? 2 * i + 1 : ib;
        float a = load_one<T>(src + (int64_t)head * r.dim + va), b = load_one<T>(src + (int64_t)head * r.dim + vb);
        if (turned && !is_v) {
            const f32x2 w = turn[i];
            const float x = a * w[0] - b * w[1], y = b * w[0] + a * w[1];
            a = x;
            b = y;
        }
        if (is_q) {
            uint16_t* d = r.q_out + t * r.q_out_stride + (int64_t)head * r.dim;
            Store<T>::one((uint8_t*)(d + va), a);
            Store<T>::one((uint8_t*)(d + vb), b);
        } else if (slot >= 0 && inside) {
            uint8_t* d = (is_v ? c.v : c.k) + at + head * c.head_stride;
            const float div = is_v ? r.v_div : r.k_div;
            Store<S>::one(d + va * Store<S>::kBytes, Store<S>::kBytes == 1 ? a / div : a);
            Store<S>::one(d + vb * Store<S>::kBytes, Store<S>::kBytes == 1 ? b / div : b);
        }
    }
}

int refuse(const char* why) {
    static thread_local char text[160];
    snprintf(text, sizeof(text), "gfd_kv_append: %s", why);
    gfd_internal_set_error(text);
    return (int)hipErrorInvalidValue;
}

template <typename T, typename S>
int launch(const Rows& r, const Cache& c, bool pairs, hipStream_t st) {
    if (pairs)
        hipLaunchKernelGGL((kv_append_kernel<T, S, true>), dim3(r.num_tokens), dim3(kBlock), 0, st, r, c);
    else
        hipLaunchKernelGGL((kv_append_kernel<T, S, false>), dim3(r.num_tokens), dim3(kBlock), 0, st, r, c);
    return (int)hipGetLastError();
}

}  // namespace
}  // namespace kv
}  // namespace gfd

extern "C" int gfd_kv_append(const gfd_kv_cache* cache, const gfd_kv_rows* rows, int* error_flag, void* stream) {
    using namespace gfd::kv;
    if (const char* why = check_cache(cache)) return refuse(why);
    if (!rows) return refuse("no rows");
    const gfd_kv_rows& w = *rows;
    if (w.dtype != GFD_BF16 && w.dtype != GFD_FP16) return refuse("rows are neither GFD_BF16 nor GFD_FP16");
    if (cache->dtype != GFD_E4M3 && cache->dtype != w.dtype) return refuse("the cache's type is neither the rows' nor GFD_E4M3");
    if (w.num_tokens < 0) return refuse("negative num_tokens");
    if (w.rotary_dim < 0 || w.rotary_dim > cache->head_dim || w.rotary_dim % 2 != 0)
        return refuse("rotary_dim is odd or outside 0..head_dim");
    if ((w.q != nullptr) != (w.q_out != nullptr)) return refuse("q and q_out go together");
    if (w.q && (w.num_q_heads < 1 || w.num_q_heads > 65535)) return refuse("num_q_heads out of range");
    if (((w.q ? w.q_stride | w.q_out_stride : 0) | w.k_stride | w.v_stride) % 8 != 0 ||
        ((uintptr_t)w.q | (uintptr_t)w.q_out | (uintptr_t)w.k | (uintptr_t)w.v) % 16 != 0)
        return refuse("rows' pointers or strides are not multiples of 16 bytes");
    if (w.num_tokens == 0) return 0;
    if (!w.k || !w.v || !w.slots || (w.rotary_dim && (!w.positions || !w.inv_freq)))
        return refuse("k, v, slots, positions or inv_freq is missing");
    const Rows r{(const uint16_t*)w.q, (const uint16_t*)w.k, (const uint16_t*)w.v, (uint16_t*)w.q_out, w.q_stride,
                 w.k_stride, w.v_stride, w.q_out_stride, w.positions, w.slots, w.inv_freq, w.num_tokens,
                 w.q ? w.num_q_heads : 0, cache->num_heads, cache->head_dim, w.rotary_dim, cache->k_scale,
                 cache->v_scale, error_flag};
    const Cache c = make_cache(*cache);
    const hipStream_t st = (hipStream_t)stream;
    const bool pairs = w.interleaved != 0;
    if (cache->dtype == GFD_E4M3)
        return w.dtype == GFD_BF16 ? launch<Bf16, E4m3>(r, c, pairs, st) : launch<Fp16, E4m3>(r, c, pairs, st);
    return w.dtype == GFD_BF16 ? launch<Bf16, Bf16>(r, c, pairs, st) : launch<Fp16, Fp16>(r, c, pairs, st);
}

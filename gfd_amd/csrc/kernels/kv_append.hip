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

int refused(const char* name, const char* why) {
    static thread_local char text[192];
    snprintf(text, sizeof(text), "%s: %s", name, why);
    gfd_internal_set_error(text);
    return (int)hipErrorInvalidValue;
}

int launched(const char* name, int rc) {
    if (rc) {
        static thread_local char text[192];
        snprintf(text, sizeof(text), "%s: the launch failed: %s", name, hipGetErrorString((hipError_t)rc));
        gfd_internal_set_error(text);
    }
    return rc;
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

constexpr int kBlock = 256, kTokens = 4;

// Eight values to the stored type.
template <typename T>
struct Store {
    static __device__ __forceinline__ void eight(uint8_t* p, const float (&x)[8], float) {
        *(u32x4*)p = u32x4{T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7])};
    }
    static constexpr int kBytes = 2;
};
template <>
struct Store<E4m3> {
    static constexpr int kBytes = 1;
    static __device__ __forceinline__ float cut(float x) {
        return x != x ? x : __builtin_amdgcn_fmed3f(x, -448.f, 448.f);
    }
    static __device__ __forceinline__ void eight(uint8_t* p, const float (&x)[8], float div) {
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            int y = __builtin_amdgcn_cvt_pk_fp8_f32(cut(x[4 * i] / div), cut(x[4 * i + 1] / div), 0, false);
            w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(cut(x[4 * i + 2] / div), cut(x[4 * i + 3] / div), y, true);
        }
        *(u32x2*)p = u32x2{w[0], w[1]};
    }
};

template <typename T>
__device__ __forceinline__ void unpack8(u32x4 w, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const f32x2 y = T::unpack(w[i]);
        x[2 * i] = y[0];
        x[2 * i + 1] = y[1];
    }
}

// How the rotated pairs lie: side by side, a half apart in whole chunks of 8, or a half apart.
enum { kSide, kChunksApart, kApart };

// A workgroup takes kTokensHere tokens: their turns go to LDS, then each thread takes 16 values of a
// head at a time, two chunks of 16 bytes.  A pair's two chunks are taken together; where
// a half is no whole number of chunks, a head's lanes (of one wave) pass their chunks through LDS instead.
// The first values are under way while the turns are computed.  Bound by the rows' and
// the cache's bytes, which it moves at the rate of a large copy: 16384 tokens of 32 + 8 heads of 128 into an 8-bit cache,
// 369 MB in 73 us; 4097 tokens of 64 rotated dims, 101 MB in 21.5 us.  Eight tokens take a launch.
template <typename T, typename S, int kPairs, int kTokensHere>
__global__ __launch_bounds__(kBlock) void kv_append_kernel(Rows r, Cache c) {
    __shared__ f32x2 turns[kTokensHere][128];
    __shared__ int64_t places[kTokensHere];
    __shared__ u32x4 chunks[kPairs == kApart ? kBlock * 2 : 1];
    const int tid = (int)threadIdx.x, t0 = (int)blockIdx.x * kTokensHere, half = r.rotary / 2;
    const int shift = r.dim == 64 ? 2 : r.dim == 128 ? 3 : 4;  // a head's units of 16 values
    const int first = (r.q ? 0 : r.q_heads) << shift, per_token = ((r.q_heads + 2 * r.kv_heads) << shift) - first;
    const int tokens = min(kTokensHere, r.num_tokens - t0), units = tokens * per_token;

    struct Unit {
        int t, head, kind, a, b;  // kind 0 q, 1 k, 2 v; first values of the chunks
        u32x4 x, y;
    };
    const auto load = [&](int n) {
        Unit u;
        u.t = 0;
        if constexpr (kTokensHere > 1) {
            while (n >= per_token) n -= per_token, u.t++;
        }
        n += first;
        const int h = n >> shift, i = n & ((1 << shift) - 1);
        u.kind = h < r.q_heads ? 0 : h < r.q_heads + r.kv_heads ? 1 : 2;
        u.head = u.kind == 0 ? h : u.kind == 1 ? h - r.q_heads : h - r.q_heads - r.kv_heads;
        u.a = 16 * i;
        u.b = u.a + 8;
        if (kPairs == kChunksApart && u.kind != 2 && 8 * i < half) {
            u.a = 8 * i;
            u.b = u.a + half;
        }
        const int64_t t = t0 + u.t;
        const uint16_t* p = (u.kind == 0   ? r.q + t * r.q_stride
                             : u.kind == 1 ? r.k + t * r.k_stride
                                           : r.v + t * r.v_stride) + (int64_t)u.head * r.dim;
        u.x = *(const u32x4*)(p + u.a);
        u.y = *(const u32x4*)(p + u.b);
        return u;
    };
    Unit u;
    if (tid < units) u = load(tid);

    for (int n = tid; n < tokens * half; n += kBlock) {
        const int t = n / half, i = n - t * half;
        const double whole = (double)r.positions[t0 + t] * ((double)r.inv_freq[i] * 0.15915494309189533577);
        float s, co;
        sincospif((float)(2.0 * (whole - rint(whole))), &s, &co);
        turns[t][i] = f32x2{co, s};
    }
    if (tid < tokens) {
        const int64_t slot = r.slots[t0 + tid];
        int64_t at = -1;
        if (slot >= 0) {
            if (slot < (int64_t)c.num_pages * c.page.d) {
                const int64_t page = slot / c.page.d;
                at = page * c.page_stride + (slot - page * c.page.d) * c.slot_stride;
            } else if (r.error) {
                atomicOr(r.error, GFD_KV_ERR_PAGE);
            }
        }
        places[tid] = at;
    }
    __syncthreads();

    for (int n = tid; n < units;) {
        float x[8], y[8];
        unpack8<T>(u.x, x);
        unpack8<T>(u.y, y);
        const f32x2* turn = turns[u.t];
        if (kPairs == kSide) {
            if (u.kind != 2 && u.a < 2 * half) {
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    float& p = i < 8 ? x[i] : y[i - 8];
                    float& q = i < 8 ? x[i + 1] : y[i - 7];
                    const int at = (u.a + i) / 2;
                    if (at >= half) continue;
                    const f32x2 w = turn[at];
                    const float p0 = p;
                    p = p0 * w[0] - q * w[1];
                    q = q * w[0] + p0 * w[1];
                }
            }
        } else if (kPairs == kChunksApart) {
            if (u.kind != 2 && u.a < half) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const f32x2 w = turn[u.a + i];
                    const float p0 = x[i], q0 = y[i];
                    x[i] = p0 * w[0] - q0 * w[1];
                    y[i] = q0 * w[0] + p0 * w[1];
                }
            }
        } else {
            const uint16_t* row = (const uint16_t*)(chunks + (tid >> shift << shift) * 2);
            chunks[2 * tid] = u.x;
            chunks[2 * tid + 1] = u.y;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            if (u.kind != 2) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    float& p = i < 8 ? x[i] : y[i - 8];
                    const int at = u.a + i;
                    if (at >= 2 * half) continue;
                    const f32x2 w = turn[at < half ? at : at - half];
                    const float q = T::unpack(row[at < half ? at + half : at - half])[0];
                    p = at < half ? p * w[0] - q * w[1] : p * w[0] + q * w[1];
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        const Unit now = u;
        n += kBlock;
        // In place, a head's queries are all loaded before any is stored: a thread holds both chunks of its
        // pairs, and the next units are other heads'.
        if (n < units) u = load(n);
        if (now.kind == 0) {
            uint16_t* d = r.q_out + (t0 + now.t) * r.q_out_stride + (int64_t)now.head * r.dim;
            Store<T>::eight((uint8_t*)(d + now.a), x, 1.f);
            Store<T>::eight((uint8_t*)(d + now.b), y, 1.f);
        } else if (places[now.t] >= 0) {
            uint8_t* d = (now.kind == 2 ? c.v : c.k) + places[now.t] + now.head * c.head_stride;
            const float div = now.kind == 2 ? r.v_div : r.k_div;
            Store<S>::eight(d + now.a * Store<S>::kBytes, x, div);
            Store<S>::eight(d + now.b * Store<S>::kBytes, y, div);
        }
    }
}

constexpr char kName[] = "gfd_kv_append";
int refuse(const char* why) { return refused(kName, why); }

template <typename T, typename S, int kTokensHere>
int launch(const Rows& r, const Cache& c, bool pairs, hipStream_t st) {
    const dim3 grid((unsigned)((r.num_tokens + kTokensHere - 1) / kTokensHere));
    const auto go = [&](auto kernel) { return start(kernel, grid, kBlock, st, r, c); };
    if (pairs) return go(kv_append_kernel<T, S, kSide, kTokensHere>);
    if (r.rotary % 16 == 0) return go(kv_append_kernel<T, S, kChunksApart, kTokensHere>);
    return go(kv_append_kernel<T, S, kApart, kTokensHere>);
}

// Tokens share a workgroup's start-up where that still fills the card.
template <typename T, typename S>
int launch(const Rows& r, const Cache& c, bool pairs, hipStream_t st) {
    return r.num_tokens >= 2048 * kTokens ? launch<T, S, kTokens>(r, c, pairs, st) : launch<T, S, 1>(r, c, pairs, st);
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
    if (((int64_t)w.num_tokens + kTokens - 1) / kTokens * kBlock >= kGridThreads)
        return refuse("more work than one launch takes");
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
        return launched(kName, w.dtype == GFD_BF16 ? launch<Bf16, E4m3>(r, c, pairs, st)
                                                   : launch<Fp16, E4m3>(r, c, pairs, st));
    return launched(kName, w.dtype == GFD_BF16 ? launch<Bf16, Bf16>(r, c, pairs, st)
                                               : launch<Fp16, Fp16>(r, c, pairs, st));
}

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
#include "kv_rows.h"

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

const char* check_cache(const gfd_kv4_cache* c) {
    if (!c || !c->k || !c->v || !c->k_scales || !c->v_scales) return "no cache";
    if (c->num_pages < 1 || c->page_size < 1 || c->page_size > 65536 || c->num_heads < 1 || c->num_heads > 65535)
        return "cache sizes out of range";
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return "head_dim is not 64, 128 or 256";
    if (((uintptr_t)c->k | (uintptr_t)c->v) % 16 != 0 || (c->page_stride | c->slot_stride | c->head_stride) % 16 != 0)
        return "cache pointers or strides are not multiples of 16 bytes";
    const int64_t most = 0x7FFFFFFF;
    for (const int64_t stride : {c->page_stride, c->slot_stride, c->head_stride, c->scale_page_stride}) {
        if (stride < 0) return "negative cache stride";
        if (stride > most) return "cache stride over 2^31 - 1";
    }
    if ((c->page_size - 1) * c->slot_stride + (c->num_heads - 1) * c->head_stride + c->head_dim / 2 > most + 1)
        return "a page's rows do not end within 2^31 bytes";
    return nullptr;
}

Cache4 make_cache(const gfd_kv4_cache& c) {
    Cache4 x;
    (Cache&)x = Cache{(uint8_t*)c.k, (uint8_t*)c.v, c.page_stride, c.slot_stride, c.head_stride, c.num_pages,
                      make_divider((uint32_t)c.page_size), 1.f, 1.f};
    x.k_scales = (uint8_t*)c.k_scales;
    x.v_scales = (uint8_t*)c.v_scales;
    x.scale_page_stride = c.scale_page_stride;
    x.heads_inner = c.head_stride <= c.slot_stride;
    return x;
}

Cache make_cache(const gfd_kv_cache& c) {
    const int64_t size = c.dtype == GFD_E4M3 ? 1 : 2;
    const bool scaled = c.dtype == GFD_E4M3;
    return Cache{(uint8_t*)c.k, (uint8_t*)c.v, c.page_stride * size, c.slot_stride * size, c.head_stride * size,
                 c.num_pages, make_divider((uint32_t)c.page_size), scaled ? c.k_scale : 1.f, scaled ? c.v_scale : 1.f};
}

const char* check_rows(const gfd_kv_rows* rows, int head_dim, const gfd_rotary_axes* axes) {
    if (!rows) return "no rows";
    const gfd_kv_rows& w = *rows;
    if (w.dtype != GFD_BF16 && w.dtype != GFD_FP16) return "rows are neither GFD_BF16 nor GFD_FP16";
    if (w.num_tokens < 0) return "negative num_tokens";
    if (((int64_t)w.num_tokens + kAppendTokens - 1) / kAppendTokens * kAppendBlock >= kGridThreads)
        return "more work than one launch takes";
    if (w.rotary_dim < 0 || w.rotary_dim > head_dim || w.rotary_dim % 2 != 0)
        return "rotary_dim is odd or outside 0..head_dim";
    if ((w.q != nullptr) != (w.q_out != nullptr)) return "q and q_out go together";
    if (w.q && (w.num_q_heads < 1 || w.num_q_heads > 65535)) return "num_q_heads out of range";
    if (((w.q ? w.q_stride | w.q_out_stride : 0) | w.k_stride | w.v_stride) % 8 != 0 ||
        ((uintptr_t)w.q | (uintptr_t)w.q_out | (uintptr_t)w.k | (uintptr_t)w.v) % 16 != 0)
        return "rows' pointers or strides are not multiples of 16 bytes";
    if (axes && (axes->num_axes < 1 || axes->num_axes > 256)) return "num_axes is outside 1..256";
    if (w.num_tokens == 0) return nullptr;
    if (!w.k || !w.v || !w.slots || (w.rotary_dim && (!(axes ? axes->positions : w.positions) || !w.inv_freq)))
        return "k, v, slots, positions or inv_freq is missing";
    if (axes && w.rotary_dim && !axes->axis) return "axis is missing";
    return nullptr;
}

Rows make_rows(const gfd_kv_rows& w, int num_heads, int head_dim, const gfd_rotary_axes* axes, float k_div, float v_div,
               int* error) {
    Rows r{(const uint16_t*)w.q, (const uint16_t*)w.k, (const uint16_t*)w.v, (uint16_t*)w.q_out, w.q_stride, w.k_stride,
           w.v_stride, w.q_out_stride, w.positions, w.slots, w.inv_freq, w.num_tokens, w.q ? w.num_q_heads : 0,
           num_heads, head_dim, w.rotary_dim, k_div, v_div, error, nullptr, nullptr, 0, 0, 0, 0};
    if (axes) {
        r.axes_positions = axes->positions;
        r.axis = axes->axis;
        r.axis_stride = axes->axis_stride;
        r.token_stride = axes->token_stride;
        r.num_axes = axes->num_axes;
        r.float_positions = axes->float_positions;
    }
    return r;
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

constexpr int kBlock = kAppendBlock, kTokens = kAppendTokens;

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

// A workgroup takes kTokensHere tokens: their turns go to LDS, then each thread takes 16 values of a
// head at a time, two chunks of 16 bytes.  A pair's two chunks are taken together; where
// a half is no whole number of chunks, a head's lanes (of one wave) pass their chunks through LDS instead.
// The first values are under way while the turns are computed.  Bound by the rows' and
// the cache's bytes, which it moves at the rate of a large copy: 16384 tokens of 32 + 8 heads of 128 into an 8-bit cache,
// 369 MB in 73 us; 4097 tokens of 64 rotated dims, 101 MB in 21.5 us.  Eight tokens take a launch.
// Positions of several axes have kernels of their own (kAxes): where one kernel asks which kind it has, the 4097 tokens
// take 24.5 us, of 36 rotated dims 6001 take 38.4 for 33.5.  The rows' loads differ too, each the faster one or even: with the other
// one 4097 tokens of one axis take 23.1 us for 22.0 (side by side), 16384 of three 81.9 for 81.0.
template <typename T, typename S, int kPairs, int kTokensHere, bool kAxes>
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
        if constexpr (kAxes) {
            u.x = eight_of(r, u.kind, t, u.head * r.dim + u.a);
            u.y = eight_of(r, u.kind, t, u.head * r.dim + u.b);
        } else {
            const uint16_t* p = (u.kind == 0   ? r.q + t * r.q_stride
                                 : u.kind == 1 ? r.k + t * r.k_stride
                                               : r.v + t * r.v_stride) + (int64_t)u.head * r.dim;
            u.x = *(const u32x4*)(p + u.a);
            u.y = *(const u32x4*)(p + u.b);
        }
        return u;
    };
    Unit u;
    if (tid < units) u = load(tid);

    for (int n = tid; n < tokens * half; n += kBlock) {
        const int t = n / half, i = n - t * half;
        const double position = kAxes ? position_of(r, t0 + t, i) : (double)r.positions[t0 + t];
        const double whole = position * ((double)r.inv_freq[i] * 0.15915494309189533577);
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

template <typename T, typename S, int kTokensHere, bool kAxes>
int launch(const Rows& r, const Cache& c, bool pairs, hipStream_t st) {
    const dim3 grid((unsigned)((r.num_tokens + kTokensHere - 1) / kTokensHere));
    const auto go = [&](auto kernel) { return start(kernel, grid, kBlock, st, r, c); };
    if (pairs) return go(kv_append_kernel<T, S, kSide, kTokensHere, kAxes>);
    if (r.rotary % 16 == 0) return go(kv_append_kernel<T, S, kChunksApart, kTokensHere, kAxes>);
    return go(kv_append_kernel<T, S, kApart, kTokensHere, kAxes>);
}

// Tokens share a workgroup's start-up where that still fills the card.
template <typename T, typename S>
int launch(const Rows& r, const Cache& c, bool pairs, hipStream_t st) {
    const bool many = r.num_tokens >= 2048 * kTokens;
    if (r.axis) return many ? launch<T, S, kTokens, true>(r, c, pairs, st) : launch<T, S, 1, true>(r, c, pairs, st);
    return many ? launch<T, S, kTokens, false>(r, c, pairs, st) : launch<T, S, 1, false>(r, c, pairs, st);
}

int append(const char* name, const gfd_kv_cache* cache, const gfd_kv_rows* rows, const gfd_rotary_axes* axes,
           int* error_flag, void* stream) {
    if (const char* why = check_cache(cache)) return refused(name, why);
    if (const char* why = check_rows(rows, cache->head_dim, axes)) return refused(name, why);
    const gfd_kv_rows& w = *rows;
    if (cache->dtype != GFD_E4M3 && cache->dtype != w.dtype)
        return refused(name, "the cache's type is neither the rows' nor GFD_E4M3");
    if (w.num_tokens == 0) return 0;
    const Rows r = make_rows(w, cache->num_heads, cache->head_dim, axes, cache->k_scale, cache->v_scale, error_flag);
    const Cache c = make_cache(*cache);
    const hipStream_t st = (hipStream_t)stream;
    const bool pairs = w.interleaved != 0;
    if (cache->dtype == GFD_E4M3)
        return launched(name, w.dtype == GFD_BF16 ? launch<Bf16, E4m3>(r, c, pairs, st)
                                                  : launch<Fp16, E4m3>(r, c, pairs, st));
    return launched(name, w.dtype == GFD_BF16 ? launch<Bf16, Bf16>(r, c, pairs, st)
                                              : launch<Fp16, Fp16>(r, c, pairs, st));
}

}  // namespace
}  // namespace kv
}  // namespace gfd

extern "C" int gfd_kv_append(const gfd_kv_cache* cache, const gfd_kv_rows* rows, int* error_flag, void* stream) {
    return gfd::kv::append("gfd_kv_append", cache, rows, nullptr, error_flag, stream);
}

extern "C" int gfd_kv_append_axes(const gfd_kv_cache* cache, const gfd_kv_rows* rows, const gfd_rotary_axes* axes,
                                  int* error_flag, void* stream) {
    return gfd::kv::append("gfd_kv_append_axes", cache, rows, axes, error_flag, stream);
}

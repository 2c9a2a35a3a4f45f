// Appending a step's keys and values to a cache of 4-bit numbers, with the
// position rotation of queries and keys on the way (gfx950).
//
// A group of 32 neighbouring dims x has the scale 2^e, the least power of two of
// which the largest magnitude is at most seven, and the numbers round(x / 2^e)
// among 0, 0.5, 1, 1.5, 2, 3, 4, 6.  With m 2^n the largest magnitude, 1 <= m < 2, that is
// e = n - 2 up to m = 1.75 and n - 1 above: an addition to the float's bits carries into
// its exponent from there on.  What lies between six and seven steps is rounded to six, no further than
// from the middle between four and six; a limit of six would double the step of
// every group whose largest is between, one of eight would leave errors of two steps.
//
// A number is decided by the 32-bit result of the rotation, so that is computed as the formula says: sine and
// cosine to the nearest float (angles in 64 bits, their turns taken off with twice as many), two products and their
// sum each rounded once.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "gfd_capi.h"
#include "kv_rows.h"

namespace gfd {
namespace kv {
namespace {

constexpr int kBlock = kAppendBlock, kTokens = kAppendTokens;

// cos and sin of position * freq.  1 / (2 pi) is kTurn + kTurnRest; the product of a position under 2^29 and a
// float has at most 53 bits.
__device__ __forceinline__ f32x2 turn_of(double position, float freq) {
    constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnRest = -0x1.6b01ec5417056p-57;
    const double angle = position * (double)freq, whole = angle * kTurn;
    const double rest = __builtin_fma(angle, kTurn, -whole) + angle * kTurnRest;
    double s, c;
    sincospi(2.0 * ((whole - __builtin_rint(whole)) + rest), &s, &c);
    return f32x2{(float)c, (float)s};
}

// a cos - b sin of a pair's first value, b cos + a sin of its second: x cos + other (-sin or sin).
__device__ __forceinline__ float rotated(float x, float other, f32x2 turn, bool first) {
#pragma clang fp contract(off)
    return x * turn[0] + other * __uint_as_float(__float_as_uint(turn[1]) ^ (first ? 0x80000000u : 0u));
}

// The largest of four neighbouring lanes.
__device__ __forceinline__ float largest(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // NaN stays
__device__ __forceinline__ float across4_max(float x) {
    x = largest(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xB1, 0xF, 0xF, true)));  // lanes 1 0 3 2
    return largest(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4E, 0xF, 0xF, true)));  // lanes 2 3 0 1
}

// Bound by the rows' bytes: 16384 tokens of 32 + 8 heads of 128, 354 MB in 80 us, 4.4 TB/s.
// A thread takes 8 values of a head at a time, so four neighbours have a group, and a head's threads are of one wave: they
// pass their chunks through LDS for the other halves of their pairs.
template <typename T, int kPairs, int kTokensHere>
__global__ __launch_bounds__(kBlock) void kv4_append_kernel(Rows r, Cache4 c) {
    __shared__ f32x2 turns[kTokensHere][128];
    __shared__ Place4 places[kTokensHere];  // row -1: none
    __shared__ u32x4 chunks[kPairs == kSide ? 1 : kBlock];
    const int tid = (int)threadIdx.x, t0 = (int)blockIdx.x * kTokensHere, half = r.rotary / 2;
    const int shift = r.dim == 64 ? 3 : r.dim == 128 ? 4 : 5;  // a head's units of 8 values
    const int first = (r.q ? 0 : r.q_heads) << shift, per_token = ((r.q_heads + 2 * r.kv_heads) << shift) - first;
    const int tokens = min(kTokensHere, r.num_tokens - t0), units = tokens * per_token;

    struct Unit {
        int t, head, kind, a;  // kind 0 q, 1 k, 2 v; first value
        u32x4 x;
    };
    const auto load = [&](int n) {
        Unit u;
        u.t = 0;
        if constexpr (kTokensHere > 1) {
            while (n >= per_token) n -= per_token, u.t++;
        }
        n += first;
        const int h = n >> shift;
        u.a = 8 * (n & ((1 << shift) - 1));
        u.kind = h < r.q_heads ? 0 : h < r.q_heads + r.kv_heads ? 1 : 2;
        u.head = u.kind == 0 ? h : u.kind == 1 ? h - r.q_heads : h - r.q_heads - r.kv_heads;
        const int64_t t = t0 + u.t;
        u.x = eight_of(r, u.kind, t, u.head * r.dim + u.a);
        return u;
    };
    // Two units are under way; past the last one it is read again, so that every wait is for the oldest load only.
    Unit even = load(min(tid, units - 1)), odd = load(min(tid + kBlock, units - 1));

    for (int n = tid; n < tokens * half; n += kBlock) {
        const int t = n / half, i = n - t * half;
        turns[t][i] = turn_of(position_of(r, t0 + t, i), r.inv_freq[i]);
    }
    if (tid < tokens) {
        const int64_t slot = r.slots[t0 + tid];
        Place4 at{-1, 0};
        if (slot >= 0) {
            if (slot < (int64_t)c.num_pages * c.page.d) {
                const int64_t page = slot / c.page.d;
                at = place_of<E2m1>(c, (int)page, (uint32_t)(slot - page * c.page.d), 0);
            } else if (r.error) {
                atomicOr(r.error, GFD_KV_ERR_PAGE);
            }
        }
        places[tid] = at;
    }
    __syncthreads();

    const auto step = [&](Unit& u, int n) {
        float x[8];
        unpack8<T>(u.x, x);
        const f32x2* turn = turns[u.t];
        if (kPairs == kSide) {
            if (u.kind != 2 && u.a < 2 * half) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const int at = (u.a + i) / 2;
                    if (at >= half) continue;
                    const float x0 = x[i];
                    x[i] = rotated(x0, x[i + 1], turn[at], true);
                    x[i + 1] = rotated(x[i + 1], x0, turn[at], false);
                }
            }
        } else {
            u32x4* const head = chunks + (tid >> shift << shift);
            chunks[tid] = u.x;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            if (u.kind != 2 && u.a < 2 * half) {
                if constexpr (kPairs == kChunksApart) {
                    const bool front = u.a < half;
                    float other[8];
                    unpack8<T>(head[(front ? u.a + half : u.a - half) / 8], other);
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = rotated(x[i], other[i], turn[(front ? u.a : u.a - half) + i], front);
                } else {
                    const uint16_t* row = (const uint16_t*)head;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int at = u.a + i;
                        if (at >= 2 * half) continue;
                        const bool front = at < half;
                        const float other = T::unpack(row[front ? at + half : at - half])[0];
                        x[i] = rotated(x[i], other, turn[front ? at : at - half], front);
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        const Unit now = u;
        // In place, a head's queries are all loaded before any is stored: its chunks were read through LDS, and the next
        // units are other heads'.
        u = load(min(n + 2 * kBlock, units - 1));
        if (now.kind == 0) {
            *(u32x4*)(r.q_out + (t0 + now.t) * r.q_out_stride + (int64_t)now.head * r.dim + now.a) =
                u32x4{T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7])};
            return;
        }
        float most = fabsf(x[0]);
#pragma unroll
        for (int i = 1; i < 8; i++) most = largest(most, fabsf(x[i]));
        const uint32_t top = __float_as_uint(across4_max(most));
        const bool finite = top < 0x7F800000u;
        const int exponent = (int)((top + 0x1FFFFFu) >> 23) - 2;
        const int byte = min(max(exponent, ScaleRange<T>::kLeast), ScaleRange<T>::kMost);
        const float by = __uint_as_float((uint32_t)(254 - byte) << 23);
        const auto number = [&](int i) { return __builtin_amdgcn_fmed3f(x[i] * by, -6.f, 6.f); };  // any if not finite
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, number(0), number(1), 1.f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, number(2), number(3), 1.f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, number(4), number(5), 1.f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, number(6), number(7), 1.f, 3);
        const Place4 place = places[now.t];
        if (place.row < 0) return;
        const int64_t head = now.head * c.head_stride;
        *(uint32_t*)((now.kind == 2 ? c.v : c.k) + place.row + head + now.a / 2) = w;
        if (now.a % kGroup4 == 0)
            (now.kind == 2 ? c.v_scales : c.k_scales)[place.scales + (head >> 4) + now.a / kGroup4] =
                (uint8_t)(finite ? byte : kScaleNan);
    };
    for (int n = tid; n < units; n += 2 * kBlock) {
        step(even, n);
        if (n + kBlock >= units) break;
        step(odd, n + kBlock);
    }
}

template <typename T, int kTokensHere>
int launch(const Rows& r, const Cache4& c, bool pairs, hipStream_t st) {
    const dim3 grid((unsigned)((r.num_tokens + kTokensHere - 1) / kTokensHere));
    const auto go = [&](auto kernel) { return start(kernel, grid, kBlock, st, r, c); };
    if (pairs) return go(kv4_append_kernel<T, kSide, kTokensHere>);
    if (r.rotary % 16 == 0) return go(kv4_append_kernel<T, kChunksApart, kTokensHere>);
    return go(kv4_append_kernel<T, kApart, kTokensHere>);
}

// Tokens share a workgroup's start-up where that still fills the card.
template <typename T>
int launch(const Rows& r, const Cache4& c, bool pairs, hipStream_t st) {
    return r.num_tokens >= 2048 * kTokens ? launch<T, kTokens>(r, c, pairs, st) : launch<T, 1>(r, c, pairs, st);
}

}  // namespace
}  // namespace kv
}  // namespace gfd

extern "C" int gfd_kv4_append(const gfd_kv4_cache* cache, const gfd_kv_rows* rows, const gfd_rotary_axes* axes,
                              int* error_flag, void* stream) {
    using namespace gfd::kv;
    constexpr char kName[] = "gfd_kv4_append";
    if (const char* why = check_cache(cache)) return refused(kName, why);
    if (const char* why = check_rows(rows, cache->head_dim, axes)) return refused(kName, why);
    if (rows->num_tokens == 0) return 0;
    const Rows r = make_rows(*rows, cache->num_heads, cache->head_dim, axes, 1.f, 1.f, error_flag);
    const Cache4 c = make_cache(*cache);
    const bool pairs = rows->interleaved != 0;
    return launched(kName, rows->dtype == GFD_BF16 ? launch<Bf16>(r, c, pairs, (hipStream_t)stream)
                                                   : launch<Fp16>(r, c, pairs, (hipStream_t)stream));
}

#pragma once
// Attention of few rows: single tokens, drafted tokens, small shared prefixes.
//
// Up to 16 or 32 rows share a head's keys and values, so each byte is used for
// at most 32 rows and the cache's bytes bound the time.  What counts is loads in
// flight: the waves of a workgroup take tiles of 32 keys by turns and without
// waiting for one another, the next tile's keys under way during a tile's
// softmax and its values during the next scores.  A long axis is split over workgroups.
//
// A tile: scores^T[32 keys][16 rows] by 16x16x32 products, keys as the left operand
// (lane: key l % 16, 8 dims of a 32, by l / 16), for which they pass through the
// wave's own LDS: whole rows come from memory faster than the operand's 64-byte
// pieces (64 ragged contexts of up to 8192 keys: 182 us for 191).  The result's lane holds row
// l % 16 and the keys 4 (l / 16) + r of both halves.  As the right operand of out^T += V^T P
// the lane has to hold 8 keys of a 32, and which 8 is free as long as the values
// agree: so it keeps its own, and loads the values of those 8 keys, D / 16
// adjacent dims each (a row of D by 16 lanes).  Left operand i takes dim i of every
// lane: two neighbouring keys' halves joined by a byte permutation, no LDS.
//
// Nothing is read twice, and loads say so (nontemporal: 64 x 8192 keys 361 us for 390).  Spills would
// undo it, a reload waits for every load: two waves a SIMD without spills take 165 us
// where three with eight of them take 187.
//
// 64 x 8192 keys of 8 heads of 128 in bf16: 2.1 GB in 361 us, 5.9 TB/s (a large read: 6.2).
// 64 ragged contexts of up to 8192: 160 us, 5.2 TB/s.  33 windows of 4096 keys of 256 dims in 8 bits,
// capped: 60 us, 4.9 TB/s.  700 keys of one token: 7.6 us and 3.9 to join, a chain of loads
// (lengths, pages, keys) and a launch each.  Many short contexts take a wave each: 128 of 128 keys in 16 us, 4.2 TB/s.
#include <algorithm>
#include <type_traits>

#include "paged_attention.h"

namespace gfd {
namespace kv {

constexpr int kRowsTile = 32;

template <int N>
struct Words {
    uint32_t w[N];
};

template <int N>  // words
__device__ __forceinline__ Words<N> load_words(const uint8_t* p) {
    Words<N> r;
    if constexpr (N == 1) {
        r.w[0] = __builtin_nontemporal_load((const uint32_t*)p);
    } else if constexpr (N == 2) {
        const u32x2 x = __builtin_nontemporal_load((const u32x2*)p);
        r.w[0] = x[0];
        r.w[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u32x4 x = __builtin_nontemporal_load((const u32x4*)(p + 4 * i));
#pragma unroll
            for (int j = 0; j < 4; j++) r.w[i + j] = x[j];
        }
    }
    return r;
}

template <typename T, typename S, int D, int R>
struct RowsKernel {
    static constexpr int kSize = S::kBytes;
    static constexpr int kDims = D / 16;                   // a lane's dims of a value row
    static constexpr int kSteps = D / 32;                  // products per 16 keys
    static constexpr int kKeyChunks = D * kSize / 16;      // of 16 bytes a key
    static constexpr int kKeyLoads = kRowsTile * kKeyChunks / 64;
    static constexpr int kValWords = kDims * kSize / 4;
    static constexpr int kAcc = kDims * 4;                 // a lane's outputs per 16 rows
    // 32 rows of 128 dims and more: with the rows' operand in registers too, a lane would need more than it has.
    static constexpr bool kLdsRows = (R == 2 && D >= 128) || D == 256;

    struct Tile {
        u32x4 k[kKeyLoads];
        Words<kValWords> v[8];
    };

    // Dims of product step s and quarter g start here: a chunk of 16 bytes is one step's, or two steps'.
    static __device__ __forceinline__ int step_dim(int s, int g) {
        return kSize == 2 ? 32 * s + 8 * g : 64 * (s / 2) + 16 * g + 8 * (s % 2);
    }
    // Where a key's chunk lies in the wave's LDS: neighbours are spread over the banks.
    static __device__ __forceinline__ int key_at(int key, int chunk) {
        constexpr int kPerTurn = kKeyChunks >= 16 ? 1 : 16 / kKeyChunks;  // keys that span the banks
        return key * kKeyChunks + (chunk ^ ((key / kPerTurn) & (kKeyChunks >= 16 ? 15 : kKeyChunks - 1)));
    }

    // A load takes whole keys, as many as 1024 bytes hold: the cache's bytes are not used again, and
    // whole rows at a time come faster than the operand's own 64-byte pieces of 16 keys.
    static __device__ __forceinline__ void load_keys(Tile& t, const Cache& c, const int64_t* off, int lane) {
#pragma unroll
        for (int i = 0; i < kKeyLoads; i++) {
            const int n = i * 64 + lane;
            const int64_t o = off[n / kKeyChunks];
            t.k[i] = __builtin_nontemporal_load((const u32x4*)(c.k + (o < 0 ? 0 : o) + n % kKeyChunks * 16));
        }
    }
    static __device__ __forceinline__ void store_keys(const Tile& t, u32x4* lds, int lane) {
#pragma unroll
        for (int i = 0; i < kKeyLoads; i++) {
            const int n = i * 64 + lane;
            lds[key_at(n / kKeyChunks, n % kKeyChunks)] = t.k[i];
        }
    }
    static __device__ __forceinline__ int load_values(Tile& t, const Cache& c, const int64_t* off, int lane) {
        int valid = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int64_t o = off[16 * (j >> 2) + 4 * (lane >> 4) + (j & 3)];
            valid |= (o >= 0) << j;
            t.v[j] = load_words<kValWords>(c.v + (o < 0 ? 0 : o) + (lane & 15) * kDims * kSize);
        }
        return valid;
    }

    // Keys' operands of step s (two steps for 8-bit keys) for 16 keys from first on.
    static constexpr int kStepsPerChunk = kSize == 2 ? 1 : 2;
    static __device__ __forceinline__ void key_frags(const u32x4* lds, int first, int s, int lane,
                                                     u32x4 (&f)[kStepsPerChunk]) {
        const u32x4 x = lds[key_at(first + (lane & 15), s / kStepsPerChunk * 4 + (lane >> 4))];
        if constexpr (kSize == 2) {
            f[0] = x;
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++)
                f[i] = u32x4{Mma<T>::widen_lo(x[2 * i]), Mma<T>::widen_hi(x[2 * i]), Mma<T>::widen_lo(x[2 * i + 1]),
                             Mma<T>::widen_hi(x[2 * i + 1])};
        }
    }
    // Word i of a value row in 16-bit pairs.
    static __device__ __forceinline__ uint32_t value_pair(const Words<kValWords>& v, int i) {
        if constexpr (kSize == 2) return v.w[i];
        else return (i & 1) ? Mma<T>::widen_hi(v.w[i / 2]) : Mma<T>::widen_lo(v.w[i / 2]);
    }
    // A word as it lies in the cache, infinities and NaN made zero.
    static __device__ __forceinline__ uint32_t only_finite_word(uint32_t w) {
        if constexpr (kSize == 2) return only_finite<T>(w);
        const uint32_t nan = ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;  // e4m3: all ones but the sign
        return w & ~((nan >> 7) * 0xFFu);
    }
    static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b, int odd) {
        return __builtin_amdgcn_perm(b, a, odd ? 0x07060302u : 0x05040100u);
    }
};

template <typename T, typename S, int D, int R, int kWaves>
struct RowsLds {
    using K = RowsKernel<T, S, D, R>;
    i32x4 rows[16 * R];
    int64_t offsets[kWaves == 1 ? kRowsShort : kRowsPiece];
    union {
        int samples[kSamples + 1];
        float merge[kWaves == 1 ? 1 : kWaves / 2][kWaves == 1 ? 1 : R * K::kAcc + 2 * R][64];
        u32x4 keys[kWaves][kRowsTile * K::kKeyChunks];
    };
    u32x4 queries[K::kLdsRows ? R * K::kSteps : 1][64];
    int any_bad;
};

// kWaves 1: ranges of at most kRowsShort keys.  kPieces: ranges of more than kRowsPiece keys.
template <typename T, typename S, int D, int R, int kWaves, bool kPieces>
__device__ __forceinline__ void attend_rows(const Call& a, const Cache& c, const Stage& prefix, const Stage& own, int item,
                                            RowsLds<T, S, D, R, kWaves>& lds) {
    using K = RowsKernel<T, S, D, R>;
    constexpr int kRows = 16 * R, kThreads = 64 * kWaves;
    // Heads vary fastest: their keys lie side by side.  Ranges vary slowest: the last ones are often empty.
    const int prefix_items = prefix.blocks * prefix.splits * a.kv_heads;
    const Stage st = item < prefix_items ? prefix : own;
    if (item >= prefix_items) item -= prefix_items;
    const int kv_head = item % a.kv_heads, block = item / a.kv_heads % st.blocks,
              split = item / a.kv_heads / st.blocks;
    const int tid = (int)threadIdx.x, lane = tid & 63, col = lane & 15, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    // Most ranges of short sequences: nothing, and no need to look further.
    if (!st.prefix && split > 0 && (int64_t)split * st.chunk >= min(a.kv_len[block], a.max_kv_len) - a.prefix_len) return;
    Block k;
    if (!find_rows<kRows>(a, st, block, &k)) return;
    if (st.prefix) {
        sample_starts(a, lds.samples, kThreads);
        __syncthreads();
    }
    Range g{0x7FFFFFFF, 0, 0, 0x7FFFFFFF};
    if (wave == 0 && lane < kRows) {
        const Row r = row_of(a, st, k, lds.samples, lane);
        lds.rows[lane] = i32x4{r.t, r.pos, r.lo, r.hi};
    }
    if (tid == 0) lds.any_bad = 0;
    __syncthreads();
    const auto read_row = [&](int i) {
        const i32x4 x = lds.rows[16 * i + col];
        return Row{x[0], x[1], x[2], x[3]};
    };
    Row row[R];
    for (int i = 0; i < R; i++) range_add(g, row[i] = read_row(i));
    // With pieces it is read again where it is used: registers are short.
    const auto row_at = [&](int i) { return kPieces ? read_row(i) : row[i]; };
    g.lo = lanes_min(g.lo);
    g.hi = -lanes_min(-g.hi);
    g.all_lo = -lanes_min(-g.all_lo);
    g.all_hi = lanes_min(g.all_hi);
    if (g.hi == 0) g.lo = 0;

    const int splits = st.prefix ? st.splits : max(1, (g.hi - g.lo + st.chunk - 1) / st.chunk);
    if (split >= splits) return;
    if (!st.prefix && split == 0 && tid == 0 && a.block_splits) a.block_splits[block * a.kv_heads + kv_head] = splits;
    const int base = (st.prefix ? 0 : g.lo) + split * st.chunk;
    const int c0 = max(base, g.lo), c1 = min(base + st.chunk, g.hi);
    const int64_t head = kv_head * c.head_stride;
    const int tiles = c1 > c0 ? (c1 - c0 + kRowsTile - 1) / kRowsTile : 0;
    // kPieces: a range is walked in pieces, whose keys' offsets are in LDS.
    constexpr int kPieceTiles = (kWaves == 1 ? kRowsShort : kRowsPiece) / kRowsTile;
    static_assert(kPieceTiles % kWaves == 0, "all waves end a piece together");
    const auto look_up = [&](int piece) {
        const int n0 = c0 + piece * kPieceTiles * kRowsTile;
        const int most = (kPieces ? min(tiles - piece * kPieceTiles, kPieceTiles) : tiles) * kRowsTile;
        for (int n = tid; n < most; n += kThreads) {
            const int64_t o = n0 + n < c1 ? key_offset(c, k.table, n0 + n, head, a.error) : -1;
            if (o < 0 && n0 + n < c1) lds.any_bad = 1;
            lds.offsets[n] = o;
        }
    };
    look_up(0);

    // The rows' operand, zero where there is no row.
    u32x4 q[K::kLdsRows ? 1 : R][K::kSteps];
    const float factor = a.factor, shift = a.shift - Mma<T>::kRaise;  // of a weight and of a maximum
    float slope[R];  // in the scores' units
    for (int i = 0; i < R; i++) {
        const int h = head_of(a, k, 16 * i + col, kv_head);
        const uint16_t* p = a.q + row_at(i).t * a.q_stride + (int64_t)h * D;
        for (int s = 0; s < K::kSteps; s++) {
            if (K::kLdsRows && wave != (i * K::kSteps + s) % kWaves) continue;
            const u32x4 x = row_at(i).t >= 0 ? *(const u32x4*)(p + K::step_dim(s, quarter)) : u32x4{0, 0, 0, 0};
            if constexpr (K::kLdsRows) lds.queries[i * K::kSteps + s][lane] = x;
            else q[i][s] = x;
        }
        slope[i] = a.slopes && row_at(i).t >= 0 ? a.slopes[h] * (kLog2e / factor) : 0.f;
    }

    __syncthreads();
    bool bad = lds.any_bad != 0;
    float m[R], sum[R];
    f32x4 o[R][K::kDims];
    for (int i = 0; i < R; i++) {
        m[i] = -INFINITY;
        sum[i] = 0.f;
        for (int d = 0; d < K::kDims; d++) o[i][d] = f32x4{0, 0, 0, 0};
    }
    typename K::Tile t;
    u32x4* const my_keys = lds.keys[wave];
    int valid = 0;
    bool any_odd = false;
    if (wave < tiles) {
        K::load_keys(t, c, lds.offsets + wave * kRowsTile, lane);
        valid = K::load_values(t, c, lds.offsets + wave * kRowsTile, lane);
    }
    for (int tile = wave; tile < tiles; tile += kWaves) {
        const int n0 = c0 + tile * kRowsTile;
        const bool more = tile + kWaves < tiles;
        // A piece's last tiles, one a wave, with another piece behind it: all waves are here.
        const bool turn = kPieces && tile % kPieceTiles >= kPieceTiles - kWaves &&
                          tile / kPieceTiles * kPieceTiles + kPieceTiles < tiles;
        const int64_t* next = lds.offsets + (kPieces ? (tile + kWaves) % kPieceTiles : tile + kWaves) * kRowsTile;
        if constexpr (K::kLdsRows) asm volatile("" ::: "memory");  // read again for each tile
        K::store_keys(t, my_keys, lane);
        // Other lanes of the wave read them: its LDS accesses are in order, the compiler has to keep them so.
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (turn) {
            __syncthreads();
            look_up(tile / kPieceTiles + 1);
            __syncthreads();
            bad = lds.any_bad != 0;
        }
        if (more) K::load_keys(t, c, next, lane);
        f32x4 x[R][2];
#pragma unroll
        for (int i = 0; i < R; i++) x[i][0] = x[i][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < K::kSteps; s += K::kStepsPerChunk) {
            u32x4 k0[K::kStepsPerChunk], k1[K::kStepsPerChunk];
            K::key_frags(my_keys, 0, s, lane, k0);
            K::key_frags(my_keys, 16, s, lane, k1);
#pragma unroll
            for (int j = 0; j < K::kStepsPerChunk; j++)
#pragma unroll
                for (int i = 0; i < R; i++) {
                    u32x4 qf;
                    if constexpr (K::kLdsRows) qf = lds.queries[i * K::kSteps + s + j][lane];
                    else qf = q[i][s + j];
                    x[i][0] = Mma<T>::m16(k0[j], qf, x[i][0]);
                    x[i][1] = Mma<T>::m16(k1[j], qf, x[i][1]);
                }
        }
        const bool whole = !bad && g.all_lo <= n0 && n0 + kRowsTile <= min(g.all_hi, c1);
        u32x4 p[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            if (a.cap_in >= 0.f) {
                const auto most = [&] {
                    float y = fabsf(x[i][0][0]);
#pragma unroll
                    for (int j = 1; j < 8; j++) y = max_f32(y, fabsf(x[i][j >> 2][j & 3]));
                    return y;
                };
                cap_scores(a, most, [&](auto form) {
#pragma unroll
                    for (int j = 0; j < 8; j++) x[i][j >> 2][j & 3] = form(x[i][j >> 2][j & 3]);
                });
            }
            if (a.slopes) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int n = n0 + 16 * (j >> 2) + 4 * quarter + (j & 3);
                    x[i][j >> 2][j & 3] =
                        __builtin_fmaf(-slope[i], fabsf((float)(row_at(i).pos - n)), x[i][j >> 2][j & 3]);
                }
            }
            if (!whole) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int n = n0 + 16 * (j >> 2) + 4 * quarter + (j & 3);
                    const bool on = n >= row_at(i).lo && n < row_at(i).hi && ((valid >> j) & 1);
                    if (!on) x[i][j >> 2][j & 3] = -INFINITY;
                }
            }
            float top = x[i][0][0];
#pragma unroll
            for (int j = 1; j < 8; j++) top = max_f32(top, x[i][j >> 2][j & 3]);
            top = across16_max(top);
            if (__any(!(top <= m[i]))) {
                const float next_m = max_f32(m[i], top);
                const float keep = m[i] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[i] - next_m) * factor);
                m[i] = next_m;
                sum[i] *= keep;
#pragma unroll
                for (int d = 0; d < K::kDims; d++) o[i][d] *= keep;
            }
            const float base_m = (m[i] == -INFINITY ? 0.f : m[i] * factor) - Mma<T>::kRaise;
            float e[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][j >> 2][j & 3], factor, -base_m));
                sum[i] += e[j];
            }
            // A weight is rounded to the values' 16-bit type, as the matrix product takes it.
#pragma unroll
            for (int j = 0; j < 4; j++) p[i][j] = T::pack(e[2 * j], e[2 * j + 1]);
        }
        if (!whole) {
            // Values of keys outside the range count as zeros.  Of keys that some rows see and
            // others do not, infinities and NaN reach only the rows that do: a weight of zero
            // would not stop them.  They are zeros in the product and are added below.
            uint32_t odd = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
#pragma unroll
                for (int i = 0; i < K::kValWords; i++) t.v[j].w[i] = (valid >> j) & 1 ? t.v[j].w[i] : 0u;
#pragma unroll
                for (int i = 0; i < K::kDims / 2; i++) odd |= not_finite<T>(K::value_pair(t.v[j], i));
            }
            if (__any(odd != 0)) {
                any_odd = true;
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int i = 0; i < K::kValWords; i++) t.v[j].w[i] = K::only_finite_word(t.v[j].w[i]);
            }
        }
#pragma unroll
        for (int d = 0; d < K::kDims; d++) {
            u32x4 vf;
#pragma unroll
            for (int j = 0; j < 4; j++)
                vf[j] = K::join(K::value_pair(t.v[2 * j], d / 2), K::value_pair(t.v[2 * j + 1], d / 2), d & 1);
#pragma unroll
            for (int i = 0; i < R; i++) o[i][d] = Mma<T>::m16(vf, p[i], o[i][d]);
        }
        if (more) valid = K::load_values(t, c, next, lane);
    }

    // The infinities and NaN that were left out, key by key.  Where the product had some in, they add nothing new.
    if (any_odd) {
#pragma unroll 1
        for (int n0 = c0 + wave * kRowsTile; n0 < c1; n0 += kWaves * kRowsTile)
#pragma unroll 1
            for (int n = n0; n < min(n0 + kRowsTile, c1); n++) {
                const int64_t at = key_offset(c, k.table, n, head, nullptr);
                const uint8_t* from = c.v + (at < 0 ? 0 : at) + 4 * quarter * K::kDims * K::kSize;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const auto v = load_words<K::kValWords>(from + r * K::kDims * K::kSize);
#pragma unroll
                    for (int d = 0; d < K::kDims; d++) {
                        const uint32_t pair = K::value_pair(v, d / 2);
                        const float x = T::unpack(pair & ~only_finite<T>(pair))[d & 1];
#pragma unroll
                        for (int i = 0; i < R; i++)
                            o[i][d][r] += at >= 0 && n >= row_at(i).lo && n < row_at(i).hi ? x : 0.f;
                    }
                }
            }
    }

    // The waves' results joined pairwise, in the lanes' own layout, where the keys were.
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R; i++) sum[i] = across16_sum(sum[i]);
    for (int half = kWaves / 2; half; half /= 2) {
        if (wave >= half && wave < 2 * half) {
            float(*to)[64] = lds.merge[wave - half];
#pragma unroll
            for (int i = 0; i < R; i++) {
                to[2 * i][lane] = m[i];
                to[2 * i + 1][lane] = sum[i];
#pragma unroll
                for (int d = 0; d < K::kAcc; d++) to[2 * R + i * K::kAcc + d][lane] = o[i][d >> 2][d & 3];
            }
        }
        __syncthreads();
        if (wave < half) {
            float(*from)[64] = lds.merge[wave];
#pragma unroll
            for (int i = 0; i < R; i++) {
                const float m2 = from[2 * i][lane], top = max_f32(m[i], m2);
                const float keep = m[i] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[i] - top) * factor);
                const float take = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m2 - top) * factor);
                m[i] = top;
                sum[i] = sum[i] * keep + from[2 * i + 1][lane] * take;
#pragma unroll
                for (int d = 0; d < K::kAcc; d++)
                    o[i][d >> 2][d & 3] = o[i][d >> 2][d & 3] * keep + from[2 * R + i * K::kAcc + d][lane] * take;
            }
        }
        __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int i = 0; i < R; i++) {
        if (row_at(i).t < 0) continue;
        const int h = head_of(a, k, 16 * i + col, kv_head);
        if (st.direct && splits == 1) {
            const float w = sum[i] == 0.f ? 0.f : c.v_scale / sum[i];
            uint16_t* out = a.out + row_at(i).t * a.out_stride + (int64_t)h * D + 4 * quarter * K::kDims;
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int d = 0; d < K::kDims; d += 4) {
                    const u32x2 y{T::pack(o[i][d][r] * w, o[i][d + 1][r] * w),
                                  T::pack(o[i][d + 2][r] * w, o[i][d + 3][r] * w)};
                    *(u32x2*)(out + r * K::kDims + d) = sum[i] == 0.f ? u32x2{0, 0} : y;
                }
            if (a.lse && quarter == 0)
                a.lse[(int64_t)row_at(i).t * a.q_heads + h] =
                    sum[i] == 0.f ? -INFINITY : (m[i] * factor + shift + __builtin_amdgcn_logf(sum[i])) * kLn2;
        } else {
            const int64_t at = slot_of(a, st.first_slot + split, row_at(i).t, h);
            if (quarter == 0) a.part_ml[at] = f32x2{m[i] * factor + shift, sum[i]};
            float* out = a.part_o + at * D + 4 * quarter * K::kDims;
            if (sum[i] == 0.f) continue;  // its weight is zero and it is not read
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int d = 0; d < K::kDims; d += 4)
                    *(f32x4*)(out + r * K::kDims + d) =
                        f32x4{o[i][d][r], o[i][d + 1][r], o[i][d + 2][r], o[i][d + 3][r]};
        }
    }
}

template <typename T, typename S, int D, int R, int kWaves, bool kPieces>
__global__ __launch_bounds__(64 * kWaves, D == 256 && (R == 2 || S::kBytes == 2) ? 1 : 2) void attend_rows_kernel(
    Call a, Cache c, Stage prefix, Stage own) {
    __shared__ RowsLds<T, S, D, R, kWaves> lds;
    attend_rows<T, S, D, R, kWaves, kPieces>(a, c, prefix, own, (int)blockIdx.x, lds);
}

template <typename T, typename S>
int launch_rows(const Call& a, const Cache& c, const Stage& prefix, const Stage& own, int dim, bool wide, int waves,
                hipStream_t st) {
    const dim3 grid((unsigned)((prefix.blocks * prefix.splits + own.blocks * own.splits) * a.kv_heads));
    const auto go = [&](auto kernel) { return start(kernel, grid, 64 * waves, st, a, c, prefix, own); };
    const auto pick = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (waves == 1) return wide ? go(attend_rows_kernel<T, S, D, 2, 1, false>) : go(attend_rows_kernel<T, S, D, 1, 1, false>);
        if (std::max(prefix.chunk, own.chunk) > kRowsPiece)
            return wide ? go(attend_rows_kernel<T, S, D, 2, 4, true>) : go(attend_rows_kernel<T, S, D, 1, 4, true>);
        return wide ? go(attend_rows_kernel<T, S, D, 2, 4, false>) : go(attend_rows_kernel<T, S, D, 1, 4, false>);
    };
    if (dim == 64) return pick(std::integral_constant<int, 64>());
    if (dim == 128) return pick(std::integral_constant<int, 128>());
    return pick(std::integral_constant<int, 256>());
}

}  // namespace kv
}  // namespace gfd

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
// capped: 60 us, 4.9 TB/s.  4-bit keys of 128 dims: 64 x 8192 of them in 120 us, 4.7 TB/s, 64 ragged contexts of up to 16384 in
// 97, where the loads alone take 105 of the 120 and the conversions, products and exponents alone 102.  Several tokens of 4
// heads a key, 64 ragged contexts of up to 8192 in 4 bits: 1 token 58 us, 2 60, 4 (16 rows) 65, 5 (20 rows) 99, 8 104: of 17 to 32
// rows a lane holds twice the results, and two waves fit a SIMD in place of four.
// 700 keys of one token: 7.6 us and 3.9 to join, a chain of loads (lengths, pages, keys) and a launch each.  Many
// short contexts take a wave each: 128 of 128 keys in 16 us, 4.2 TB/s.
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

template <int kBytes>
__device__ __forceinline__ Words<(kBytes + 3) / 4> load_words(const uint8_t* p) {
    Words<(kBytes + 3) / 4> r;
    if constexpr (kBytes == 2) {
        r.w[0] = __builtin_nontemporal_load((const uint16_t*)p);
    } else if constexpr (kBytes == 4) {
        r.w[0] = __builtin_nontemporal_load((const uint32_t*)p);
    } else if constexpr (kBytes == 8) {
        const u32x2 x = __builtin_nontemporal_load((const u32x2*)p);
        r.w[0] = x[0];
        r.w[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < kBytes / 4; i += 4) {
            const u32x4 x = __builtin_nontemporal_load((const u32x4*)(p + 4 * i));
#pragma unroll
            for (int j = 0; j < 4; j++) r.w[i + j] = x[j];
        }
    }
    return r;
}

// What 16-bit, 8-bit and 4-bit caches share.
template <typename T, typename S, int D, int R, int kStepsPerChunk>
struct RowsShape {
    static constexpr int kDims = D / 16;                   // a lane's dims of a value row
    static constexpr int kSteps = D / 32;                  // products per 16 keys
    static constexpr int kAcc = kDims * 4;                 // a lane's outputs per 16 rows
    // 32 rows of 128 dims and more: with the rows' operand in registers too, a lane would need more than it has.  4 bits: so
    // that four waves fit a SIMD (64 x 8192 keys 121 us, with three 127).
    static constexpr bool kLdsRows = (R == 2 && D >= 128) || D == 256 || (S::kBits == 4 && D == 128);

    // Dims of product step s and quarter g start here: what a lane reads of a key at once, 16 bytes (8 of 64 4-bit dims),
    // is 1 step's, 2 or 4 steps'.
    static __device__ __forceinline__ int step_dim(int s, int g) {
        return 32 * (s / kStepsPerChunk * kStepsPerChunk) + 8 * kStepsPerChunk * g + 8 * (s % kStepsPerChunk);
    }
    // Where a key's chunk lies in the wave's LDS: neighbours are spread over the banks.
    template <int kKeyChunks>
    static __device__ __forceinline__ int key_at(int key, int chunk) {
        constexpr int kPerTurn = kKeyChunks >= 16 ? 1 : 16 / kKeyChunks;  // keys that span the banks
        return key * kKeyChunks + (chunk ^ ((key / kPerTurn) & (kKeyChunks >= 16 ? 15 : kKeyChunks - 1)));
    }
    static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b, int odd) {
        return __builtin_amdgcn_perm(b, a, odd ? 0x07060302u : 0x05040100u);
    }
};

template <typename T, typename S, int D, int R>
struct RowsKernel : RowsShape<T, S, D, R, S::kBits == 16 ? 1 : 2> {
    using Shape = RowsShape<T, S, D, R, S::kBits == 16 ? 1 : 2>;
    using Shape::kDims;
    static constexpr int kBits = S::kBits;
    static constexpr int kKeyChunks = D * kBits / 128;     // of 16 bytes a key
    static constexpr int kKeyLoads = kRowsTile * kKeyChunks / 64;
    static constexpr int kValBytes = kDims * kBits / 8;
    static constexpr int kValWords = kValBytes / 4;
    static constexpr int kStepsPerChunk = kBits == 16 ? 1 : 2;

    using Value = Words<kValWords>;  // a lane's dims of one key's values
    using Values = Value[8];
    struct Tile {
        u32x4 k[kKeyLoads];
        Values v;
        int valid;  // bit j: value j is there
    };
    using Lds = u32x4[kRowsTile * kKeyChunks];  // of a wave

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
    static __device__ __forceinline__ void store(const Tile& t, Lds& lds, int lane) {
#pragma unroll
        for (int i = 0; i < kKeyLoads; i++) {
            const int n = i * 64 + lane;
            lds[Shape::template key_at<kKeyChunks>(n / kKeyChunks, n % kKeyChunks)] = t.k[i];
        }
    }
    static __device__ __forceinline__ void load_values(Tile& t, const Cache& c, const int64_t* off, int lane) {
        t.valid = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int64_t o = off[16 * (j >> 2) + 4 * (lane >> 4) + (j & 3)];
            t.valid |= (o >= 0) << j;
            t.v[j] = value(c, o < 0 ? 0 : o, lane & 15);
        }
    }
    // The dims of a row that lane n of its 16 has.
    static __device__ __forceinline__ Value value(const Cache& c, int64_t place, int n) {
        return load_words<kValBytes>(c.v + place + n * kValBytes);
    }

    // Keys' operands of step s (two steps for 8-bit keys) for 16 keys from first on.
    static __device__ __forceinline__ void key_frags(const Lds& lds, int first, int s, int lane,
                                                     u32x4 (&f)[kStepsPerChunk]) {
        const u32x4 x = lds[Shape::template key_at<kKeyChunks>(first + (lane & 15), s / kStepsPerChunk * 4 + (lane >> 4))];
        if constexpr (kBits == 16) {
            f[0] = x;
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++)
                f[i] = u32x4{Mma<T>::widen_lo(x[2 * i]), Mma<T>::widen_hi(x[2 * i]), Mma<T>::widen_lo(x[2 * i + 1]),
                             Mma<T>::widen_hi(x[2 * i + 1])};
        }
    }
    // Word i of a value row in 16-bit pairs.
    static __device__ __forceinline__ uint32_t value_pair(const Value& v, int i) {
        if constexpr (kBits == 16) return v.w[i];
        else return (i & 1) ? Mma<T>::widen_hi(v.w[i / 2]) : Mma<T>::widen_lo(v.w[i / 2]);
    }
    // Values as they lie in the cache, all of them made zero, or the infinities and NaN.
    static __device__ __forceinline__ void keep(Value& v, bool there) {
#pragma unroll
        for (int i = 0; i < kValWords; i++) v.w[i] = there ? v.w[i] : 0u;
    }
    static __device__ __forceinline__ void keep_finite(Value& v) {
#pragma unroll
        for (int i = 0; i < kValWords; i++) {
            if constexpr (kBits == 16) {
                v.w[i] = only_finite<T>(v.w[i]);
            } else {
                const uint32_t nan = ((v.w[i] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;  // e4m3: all ones but the sign
                v.w[i] &= ~((nan >> 7) * 0xFFu);
            }
        }
    }
};

// 4-bit numbers.  A tile of 128 dims is 2 KiB of keys and as much of values, and 256 bytes of scales: loads of a lane's own
// pieces would be many for few bytes, so whole rows of keys, of values and the scales (a key's by a lane, a value's by
// another) pass through the wave's LDS.  They are all under way during the tile before (two tiles under way were no
// faster: what bounds is half the bytes, half the instructions that widen them).
template <typename T, int D, int R>
struct RowsKernel<T, E2m1, D, R> : RowsShape<T, E2m1, D, R, D == 64 ? 2 : 4> {
    using Shape = RowsShape<T, E2m1, D, R, D == 64 ? 2 : 4>;
    using Shape::kDims;
    static constexpr int kBits = 4;
    static constexpr int kKeyChunks = D / 32;  // of 16 bytes a row, and its scales
    static constexpr int kKeyLoads = kRowsTile * kKeyChunks / 64;
    static constexpr int kValBytes = kDims / 2;
    static constexpr int kValWords = (kValBytes + 3) / 4;
    static constexpr int kStepsPerChunk = D == 64 ? 2 : 4;

    struct Value {  // a lane's dims of one key's values, all of one group
        uint32_t w[kValWords];
        float scale;
    };
    using Values = Value[8];
    struct Tile {
        u32x4 k[kKeyLoads], v[kKeyLoads];
        uint32_t scales[(kKeyChunks + 3) / 4];
        int valid;  // bit j: value j is there
    };
    struct Lds {
        u32x4 keys[kRowsTile * kKeyChunks], values[kRowsTile * kKeyChunks];
        uint8_t scales[2][kKeyChunks][kRowsTile];  // of keys and of values
    };

    // there: a bit for each key.
    static __device__ __forceinline__ void load(Tile& t, const Cache4& c, const Place4* off, uint32_t there, int lane) {
        const uint32_t w = there >> 4 * (lane >> 4);
        t.valid = (w & 15) | (w >> 12 & 0xF0);
        int64_t o[kKeyLoads];
#pragma unroll
        for (int i = 0; i < kKeyLoads; i++) {
            const int n = i * 64 + lane;
            o[i] = off[n / kKeyChunks].row + n % kKeyChunks * 16;
        }
        if (c.heads_inner) {  // a line has neighbouring heads' rows too: it is to stay until they are read
            asm volatile("");  // the two kinds of loads are not to become one
#pragma unroll
            for (int i = 0; i < kKeyLoads; i++) {
                t.k[i] = *(const u32x4*)(c.k + o[i]);
                t.v[i] = *(const u32x4*)(c.v + o[i]);
            }
            asm volatile("");
        } else {
#pragma unroll
            for (int i = 0; i < kKeyLoads; i++) {
                t.k[i] = __builtin_nontemporal_load((const u32x4*)(c.k + o[i]));
                t.v[i] = __builtin_nontemporal_load((const u32x4*)(c.v + o[i]));
            }
        }
        load_scales(t.scales, (lane < 32 ? c.k_scales : c.v_scales) + off[lane & 31].scales);
    }
    // They lie at any address.
    static __device__ __forceinline__ void load_scales(uint32_t (&s)[(kKeyChunks + 3) / 4], const uint8_t* p) {
        if constexpr (D == 64) {
            uint16_t x;
            __builtin_memcpy(&x, p, 2);
            s[0] = x;
        } else {
            __builtin_memcpy(s, p, kKeyChunks);
        }
    }
    // A value row's place: the four that a lane's quarters read at once lie side by side, and so do the four that
    // are stored at once.
    static __device__ __forceinline__ int value_at(int key) {
        const int quarter = (key >> 2) & 3, r = key & 3;
        return ((key & 16) + 4 * r + ((quarter + r) & 3)) * kKeyChunks;
    }
    static __device__ __forceinline__ void store(const Tile& t, Lds& lds, int lane) {
#pragma unroll
        for (int i = 0; i < kKeyLoads; i++) {
            const int n = i * 64 + lane;
            lds.keys[Shape::template key_at<kKeyChunks>(n / kKeyChunks, n % kKeyChunks)] = t.k[i];
            lds.values[value_at(n / kKeyChunks) + n % kKeyChunks] = t.v[i];
        }
#pragma unroll
        for (int g = 0; g < kKeyChunks; g += 4) {
            const uint32_t w = read_scales<T>(t.scales[g / 4]);
#pragma unroll
            for (int b = 0; b < (D == 64 ? 2 : 4); b++) lds.scales[lane >> 5][g + b][lane & 31] = (uint8_t)(w >> 8 * b);
        }
    }

    static __device__ __forceinline__ void key_frags(const Lds& lds, int first, int s, int lane,
                                                     u32x4 (&f)[kStepsPerChunk]) {
        const int key = first + (lane & 15), chunk = D == 64 ? lane >> 5 : s / 4 * 4 + (lane >> 4);
        const float scale = __uint_as_float((uint32_t)lds.scales[0][chunk][key] << 23);
        const u32x4* const x = lds.keys + Shape::template key_at<kKeyChunks>(key, chunk);
        uint32_t w[kStepsPerChunk];
        if constexpr (D == 64) {
            const u32x2 y = ((const u32x2*)x)[(lane >> 4) & 1];
            w[0] = y[0], w[1] = y[1];
        } else {
            const u32x4 y = *x;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = y[i];
        }
#pragma unroll
        for (int i = 0; i < kStepsPerChunk; i++) f[i] = widen4<T>(w[i], scale);
    }
    static __device__ __forceinline__ void values(const Lds& lds, int lane, Values& v) {
        const int quarter = lane >> 4, n = lane & 15;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t scales = *(const uint32_t*)&lds.scales[1][n * kDims / kGroup4][16 * h + 4 * quarter];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                Value& x = v[4 * h + r];
                const uint8_t* p = (const uint8_t*)(lds.values + value_at(16 * h + 4 * quarter + r)) + n * kValBytes;
                if constexpr (kValBytes == 2) {
                    x.w[0] = *(const uint16_t*)p;
                } else if constexpr (kValBytes == 4) {
                    x.w[0] = *(const uint32_t*)p;
                } else {
                    const u32x2 y = *(const u32x2*)p;
                    x.w[0] = y[0], x.w[1] = y[1];
                }
                x.scale = __uint_as_float((r == 3 ? scales >> 1 : scales << (23 - 8 * r)) & 0x7F800000u);
            }
        }
    }
    static __device__ __forceinline__ Value value(const Cache4& c, const Place4& place, int n) {
        Value x;
        const auto w = load_words<kValBytes>(c.v + place.row + n * kValBytes);
#pragma unroll
        for (int i = 0; i < kValWords; i++) x.w[i] = w.w[i];
        x.scale = scale_of<T>(c.v_scales[place.scales + n * kDims / kGroup4]);
        return x;
    }
    static __device__ __forceinline__ uint32_t value_pair(const Value& v, int i) {
        return widen4<T>(v.w[i / 4], i % 4, v.scale);
    }
    static __device__ __forceinline__ void keep(Value& v, bool there) {
#pragma unroll
        for (int i = 0; i < kValWords; i++) v.w[i] = there ? v.w[i] : 0u;
        v.scale = there ? v.scale : 1.f;
    }
    static __device__ __forceinline__ void keep_finite(Value& v) { keep(v, __float_as_uint(v.scale) != (uint32_t)kScaleNan << 23); }
};

template <typename T, typename S, int D, int R, int kWaves>
struct RowsLds {
    using K = RowsKernel<T, S, D, R>;
    i32x4 rows[16 * R];
    // Of the range's keys, or a piece's.  4 bits: 0 where none is, and a bit each that says so; else -1.
    static constexpr int kKeys = kWaves == 1 ? kRowsShort : kRowsPiece;
    // The last tile is none.
    Place<S> offsets[kKeys + (S::kBits == 4 ? kRowsTile : 0)];
    uint32_t there[S::kBits == 4 ? kKeys / kRowsTile + 1 : 1];
    union {
        int samples[kSamples + 1];
        float merge[kWaves == 1 ? 1 : kWaves / 2][kWaves == 1 ? 1 : R * K::kAcc + 2 * R][64];
        typename K::Lds tiles[kWaves];
    };
    u32x4 queries[K::kLdsRows ? R * K::kSteps : 1][64];
    int any_bad;
};

// kWaves 1: ranges of at most kRowsShort keys.  kPieces: ranges of more than kRowsPiece keys.
template <typename T, typename S, int D, int R, int kWaves, bool kPieces>
__device__ __forceinline__ void attend_rows(const Call& a, const CacheOf<S>& c, const Stage& prefix, const Stage& own, int item,
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
    if constexpr (K::kBits == 4) {
        if (tid < kRowsTile) lds.offsets[lds.kKeys + tid] = Place4{0, 0};
        if (tid == 0) lds.there[lds.kKeys / kRowsTile] = 0;
    }
    __syncthreads();
    const auto read_row = [&](int i) {
        const i32x4 x = lds.rows[16 * i + col];
        return Row{x[0], x[1], x[2], x[3]};
    };
    Row row[R];
    for (int i = 0; i < R; i++) range_add(g, row[i] = read_row(i));
    // With pieces, and 4 bits, it is read again where it is used: registers are short.
    const auto row_at = [&](int i) { return kPieces || K::kBits == 4 ? read_row(i) : row[i]; };
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
            Place<S> o;
            const bool in = n0 + n < c1, there = in && key_place<S>(c, k.table, n0 + n, head, a.error, &o);
            if (in && !there) lds.any_bad = 1;
            if constexpr (K::kBits == 4) {
                const uint64_t bits = __ballot(there);
                if (!there) o = Place4{0, 0};
                if (n % kRowsTile == 0) lds.there[n / kRowsTile] = (uint32_t)(bits >> (lane & 32));
            } else {
                if (!there) o = -1;
            }
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
    typename K::Lds& my_tile = lds.tiles[wave];
    bool any_odd = false;
    if constexpr (K::kBits == 4) {
        const int at = wave < tiles ? wave : lds.kKeys / kRowsTile;
        K::load(t, c, lds.offsets + at * kRowsTile, lds.there[at], lane);
    } else if (wave < tiles) {
        K::load_keys(t, c, lds.offsets + wave * kRowsTile, lane);
        K::load_values(t, c, lds.offsets + wave * kRowsTile, lane);
    }
    for (int tile = wave; tile < tiles; tile += kWaves) {
        const int n0 = c0 + tile * kRowsTile;
        const bool more = tile + kWaves < tiles;
        // A piece's last tiles, one a wave, with another piece behind it: all waves are here.
        const bool turn = kPieces && tile % kPieceTiles >= kPieceTiles - kWaves &&
                          tile / kPieceTiles * kPieceTiles + kPieceTiles < tiles;
        const int next = kPieces ? (tile + kWaves) % kPieceTiles : tile + kWaves;
        if constexpr (K::kLdsRows) asm volatile("" ::: "memory");  // read again for each tile
        K::store(t, my_tile, lane);
        const int valid = t.valid;
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
        if constexpr (K::kBits == 4) {
            // Whether or not there is such a tile, so that each wait is for the oldest loads only.
            const int at = more ? next : lds.kKeys / kRowsTile;
            K::load(t, c, lds.offsets + at * kRowsTile, lds.there[at], lane);
        } else {
            if (more) K::load_keys(t, c, lds.offsets + next * kRowsTile, lane);
        }
        f32x4 x[R][2];
#pragma unroll
        for (int i = 0; i < R; i++) x[i][0] = x[i][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < K::kSteps; s += K::kStepsPerChunk) {
            const auto query = [&](int i, int j) {
                if constexpr (K::kLdsRows) return lds.queries[i * K::kSteps + s + j][lane];
                else return q[i][s + j];
            };
            if constexpr (K::kBits == 4 && D != 256) {
                // 16 keys after the others: those of 32, widened, would take the registers of a wave.
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    u32x4 kf[K::kStepsPerChunk];
                    K::key_frags(my_tile, 16 * h, s, lane, kf);
#pragma unroll
                    for (int j = 0; j < K::kStepsPerChunk; j++)
#pragma unroll
                        for (int i = 0; i < R; i++) x[i][h] = Mma<T>::m16(kf[j], query(i, j), x[i][h]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                u32x4 k0[K::kStepsPerChunk], k1[K::kStepsPerChunk];
                K::key_frags(my_tile, 0, s, lane, k0);
                K::key_frags(my_tile, 16, s, lane, k1);
#pragma unroll
                for (int j = 0; j < K::kStepsPerChunk; j++)
#pragma unroll
                    for (int i = 0; i < R; i++) {
                        const u32x4 qf = query(i, j);
                        x[i][0] = Mma<T>::m16(k0[j], qf, x[i][0]);
                        x[i][1] = Mma<T>::m16(k1[j], qf, x[i][1]);
                    }
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
        typename K::Values read;
        auto& v = [&]() -> typename K::Values& {
            if constexpr (K::kBits == 4) {
                K::values(my_tile, lane, read);
                return read;
            } else {
                return t.v;
            }
        }();
        if (!whole) {
            // Values of keys outside the range count as zeros.  Of keys that some rows see and
            // others do not, infinities and NaN reach only the rows that do: a weight of zero
            // would not stop them.  They are zeros in the product and are added below.
            uint32_t odd = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                K::keep(v[j], (valid >> j) & 1);
#pragma unroll
                for (int i = 0; i < K::kDims / 2; i++) odd |= not_finite<T>(K::value_pair(v[j], i));
            }
            if (__any(odd != 0)) {
                any_odd = true;
#pragma unroll
                for (int j = 0; j < 8; j++) K::keep_finite(v[j]);
            }
        }
#pragma unroll
        for (int d = 0; d < K::kDims; d++) {
            u32x4 vf;
#pragma unroll
            for (int j = 0; j < 4; j++)
                vf[j] = K::join(K::value_pair(v[2 * j], d / 2), K::value_pair(v[2 * j + 1], d / 2), d & 1);
#pragma unroll
            for (int i = 0; i < R; i++) o[i][d] = Mma<T>::m16(vf, p[i], o[i][d]);
        }
        if constexpr (K::kBits != 4) {
            if (more) K::load_values(t, c, lds.offsets + next * kRowsTile, lane);
        }
    }

    // The infinities and NaN that were left out, key by key.  Where the product had some in, they add nothing new.
    if (any_odd) {
#pragma unroll 1
        for (int n0 = c0 + wave * kRowsTile; n0 < c1; n0 += kWaves * kRowsTile)
#pragma unroll 1
            for (int n = n0; n < min(n0 + kRowsTile, c1); n++) {
                Place<S> at{};
                const bool there = key_place<S>(c, k.table, n, head, nullptr, &at);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const auto v = K::value(c, at, 4 * quarter + r);
#pragma unroll
                    for (int d = 0; d < K::kDims; d++) {
                        const uint32_t pair = K::value_pair(v, d / 2);
                        const float x = T::unpack(pair & ~only_finite<T>(pair))[d & 1];
#pragma unroll
                        for (int i = 0; i < R; i++)
                            o[i][d][r] += there && n >= row_at(i).lo && n < row_at(i).hi ? x : 0.f;
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

// Waves that a SIMD is to hold.
template <typename S, int D, int R, bool kPieces>
constexpr int rows_waves() {
    if (S::kBits == 4 && D != 256 && R == 1) return kPieces ? 3 : 4;  // with pieces a few registers more
    return D == 256 && (R == 2 || S::kBits == 16) ? 1 : 2;
}

// Which of the items workgroup id takes, and how many workgroups so many items of all heads need.  Workgroups go to the 8
// XCDs by turns.  A row of 4-bit numbers is half a line of an L2, or less, and its scales a small part of one: the heads of
// a range stay on one XCD, which then fetches a line once (64 x 8192 keys,
// heads inside slots: 209 us, so 166; what of it is read with loads that keep lines 143).  Ranges of one sequence are spread over
// the XCDs, or the longest ones would be one XCD's (64 ragged contexts of up to 16384: 131 us, so 105).
template <typename S>
__device__ __forceinline__ int rows_item(int id, int heads) {
    if constexpr (S::kBits != 4) return id;
    const int turn = id >> 3, eight = turn / heads;
    return (eight * 8 + ((id + eight + (eight >> 3)) & 7)) * heads + turn % heads;
}
template <typename S>
int64_t rows_groups(int64_t ranges, int heads) {
    return S::kBits == 4 ? (ranges + 7) / 8 * 8 * heads : ranges * heads;
}

template <typename T, typename S, int D, int R, int kWaves, bool kPieces>
__global__ __launch_bounds__(64 * kWaves, (rows_waves<S, D, R, kPieces>())) void attend_rows_kernel(
    Call a, CacheOf<S> c, Stage prefix, Stage own) {
    __shared__ RowsLds<T, S, D, R, kWaves> lds;
    const int item = rows_item<S>((int)blockIdx.x, a.kv_heads);
    if (S::kBits == 4 && item >= (prefix.blocks * prefix.splits + own.blocks * own.splits) * a.kv_heads) return;
    attend_rows<T, S, D, R, kWaves, kPieces>(a, c, prefix, own, item, lds);
}

template <typename T, typename S>
int launch_rows(const Call& a, const CacheOf<S>& c, const Stage& prefix, const Stage& own, int dim, bool wide, int waves,
                hipStream_t st) {
    const dim3 grid((unsigned)rows_groups<S>((int64_t)prefix.blocks * prefix.splits + (int64_t)own.blocks * own.splits, a.kv_heads));
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

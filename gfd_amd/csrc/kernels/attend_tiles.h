#pragma once
// Attention of many rows: prompts, chunks of prompts, a batch over its shared prefix.
//
// Each key is used by hundreds of rows, so the matrix products bound the time.  A
// workgroup of W waves takes 32 W rows, 32 a wave, and walks the keys in tiles
// that all of its waves read from LDS.  A tile's keys and values lie there
// as 16-bit numbers (8- and 4-bit ones are widened on the way in, once for the
// workgroup), twice: the next tiles are loaded to registers while this one is
// computed, and written behind it, so that a tile costs one barrier.
//
// A tile: scores^T[32 keys][32 rows] by 32x32x16 products, keys as the left operand.
// The result's lane holds row l % 32 and the keys 8 (r / 4) + 4 (l / 32) + r % 4;
// eight of these, rounded, are the right operand of out^T[32 dims][32 rows] += V^T P
// as they lie.  V^T comes from LDS by transposing reads, 4 keys of one dim a lane.
// Chunks of 16 bytes are swapped by row, so that neither read finds two rows in a bank
// (with a swap by 8 rows, 43% of the LDS's cycles were conflicts).
//
// 4096 tokens over 16384 keys, 32 heads of 128 in bf16: 925 us, 1040 TFLOP/s, where a library product of
// 8192^3 reaches 1186 (the card's power holds both: 1.9 GHz with the matrix pipes at 46%,
// and 1.6 to 1.9 GHz at 70%).  8192 packed tokens with capped scores: 210 us, 485 TFLOP/s; a cap costs
// two more transcendental instructions a score, and the longest document's blocks end last: with 1.5 waves a SIMD on
// average neither pipe is full (20% and 31%), a wave waits 36% of its time for results.
// 7 ragged prompts of 64 dims with a bias: 57 us, the 30 tiles of the longest one by 4 waves, one a SIMD, which waits
// 47% of its time: a tile's scores, maximum, exponents and values follow one another, and nothing else is there.
// 4-bit keys, 2048 tokens over 8192, 32 heads of 128: 262 us, 920 TFLOP/s, pipes at 37% at 2.1 GHz with 1.7 waves a SIMD;
// capped 319, biased 293, 6 packed documents 90, each token with a window of 1024 keys 51; of 64 dims 179, capped 265, biased 217;
// 1024 tokens of 16 heads of 256 dims 256, capped, biased and in 6 documents 245.
// Tried and slower: half of the waves a product behind the others (1130 us for 1096), tiles of 32 keys with
// three under way (2048 tokens 85 us for 74), two groups of 4 waves to a block (packed tokens 263 us for 223).
// Of 4 bits, the scores of a tile before the weights of the one ahead of it: 2048 over 8192 takes 5% more.
#include <type_traits>

#include "paged_attention.h"

namespace gfd {
namespace kv {

template <typename T, typename S, int D, int W>
struct TilesKernel {
    static constexpr int kThreads = 64 * W, kRows = 32 * W;
    static constexpr int kTile = D == 256 ? 32 : 64;  // keys; two tiles of keys and values are 64 KiB (D 64: 32)
    static constexpr int kHalves = kTile / 32;
    static constexpr int kSteps = D / 16, kDims = D / 32;
    static constexpr int kChunks = D / 8;  // of 8 elements a row
    static constexpr int kUnits = kTile * kChunks / kThreads;
    static_assert(kUnits >= 1, "a thread moves a chunk at least");
    static constexpr int kUnitWords = S::kBits / 4;

    struct Staged {
        uint32_t k[kUnits][kUnitWords], v[kUnits][kUnitWords];
        uint32_t k_scale[S::kBits == 4 ? kUnits : 1], v_scale[S::kBits == 4 ? kUnits : 1];  // 4 bits: of the chunks' groups
    };
    // A thread moves the same chunk of every kStride-th row.
    static constexpr int kStride = kThreads / kChunks;
    static_assert(kThreads % kChunks == 0, "a thread's chunks are all the same");

    // Where a row's chunk lies, so that rows that are read together meet in no bank (64 of 4 bytes).  Keys: one chunk
    // of 16 rows at once.  Values: two neighbouring chunks of 4 rows.  A row of 128 bytes (D 64) is half the banks.
    static __device__ __forceinline__ int swap_k(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
    static __device__ __forceinline__ int swap_v(int row) { return D == 64 ? ((row >> 1) & 1) * 4 : (row & 3) * 4; }

    // kc and vc: the thread's chunk of the cache's first row.
    static __device__ __forceinline__ void load(Staged& g, const CacheOf<S>& c, const uint8_t* kc, const uint8_t* vc,
                                                const Place<S>* off, int tid) {
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            const Place<S> place = off[tid / kChunks + u * kStride];
            const int64_t o = numbers_at(place);
            if constexpr (S::kBits == 4) {
                const int64_t at = place.scales + tid % kChunks * 8 / kGroup4;
                g.k[u][0] = *(const uint32_t*)(kc + o);
                g.v[u][0] = *(const uint32_t*)(vc + o);
                g.k_scale[u] = c.k_scales[at];
                g.v_scale[u] = c.v_scales[at];
            } else if constexpr (S::kBits == 16) {
                const u32x4 k = *(const u32x4*)(kc + o), v = *(const u32x4*)(vc + o);
#pragma unroll
                for (int i = 0; i < 4; i++) g.k[u][i] = k[i], g.v[u][i] = v[i];
            } else {
                const u32x2 k = *(const u32x2*)(kc + o), v = *(const u32x2*)(vc + o);
#pragma unroll
                for (int i = 0; i < 2; i++) g.k[u][i] = k[i], g.v[u][i] = v[i];
            }
        }
    }
    static __device__ __forceinline__ u32x4 widened(const uint32_t (&w)[kUnitWords], uint32_t scale) {
        if constexpr (S::kBits == 4) return widen4<T>(w[0], scale_of<T>(scale));
        else if constexpr (S::kBits == 16) return u32x4{w[0], w[1], w[2], w[3]};
        else return u32x4{Mma<T>::widen_lo(w[0]), Mma<T>::widen_hi(w[0]), Mma<T>::widen_lo(w[1]), Mma<T>::widen_hi(w[1])};
    }
    // Values of keys that are not there (there: not NULL if there may be such) become zeros; keys may be anything,
    // their scores are not used.  Nonzero where look is set and a value is infinite or NaN.
    static __device__ __forceinline__ uint32_t store(const Staged& g, uint16_t* kb, uint16_t* vb, int tid,
                                                     const int* there, bool look) {
        const int chunk = tid % kChunks;
        u32x4 v[kUnits];
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            const int row = tid / kChunks + u * kStride;
            v[u] = widened(g.v[u], g.v_scale[S::kBits == 4 ? u : 0]);
            *(u32x4*)(kb + row * D + (chunk ^ swap_k(row)) * 8) = widened(g.k[u], g.k_scale[S::kBits == 4 ? u : 0]);
        }
        if (there) {
#pragma unroll
            for (int u = 0; u < kUnits; u++) v[u] = there[tid / kChunks + u * kStride] ? v[u] : u32x4{0, 0, 0, 0};
        }
        uint32_t odd = 0;
        if (look) {
#pragma unroll
            for (int u = 0; u < kUnits; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) odd |= not_finite<T>(v[u][i]);
        }
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            const int row = tid / kChunks + u * kStride;
            *(u32x4*)(vb + row * D + (chunk ^ swap_v(row)) * 8) = v[u];
        }
        return odd;
    }

    static __device__ __forceinline__ u32x2 transposed(const uint16_t* p) {
        return __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
    }
};

// What happens to a score on its way to the exponent.
enum { kPlain, kCapped, kBiased };

template <typename T, typename S, int D, int W>
struct TilesLds {
    using K = TilesKernel<T, S, D, W>;
    union {
        u32x4 keys[2][K::kTile * D / 8];
        int samples[kSamples + 1];
    };
    u32x4 values[2][K::kTile * D / 8];
    i32x4 rows[K::kRows];
    Place<S> offsets[4][K::kTile];  // where keys lie, 0 where none is
    int there[4][K::kTile];
    int bad[8], odd[8], ranges[4][W];
};

template <typename T, typename S, int D, int W, int kScores>
__device__ __forceinline__ void attend_tiles(const Call& a, const CacheOf<S>& c, const Stage& prefix, const Stage& own, int id,
                                             TilesLds<T, S, D, W>& lds) {
    using K = TilesKernel<T, S, D, W>;
    constexpr int kTile = K::kTile, kRows = K::kRows;
    // Tiles under way: two where the registers hold them (4096 tokens over 16384 keys, 8 waves: 948 us, with one 1056).
    // 4 waves that move 128 dims of 16 bits hold one.
    constexpr int kAhead = W == 8 || D == 64 || S::kBits < 16 || (D == 256 && kScores != kBiased) ? 2 : 1;
    auto &keys_lds = lds.keys, &values_lds = lds.values;
    auto &rows = lds.rows;
    auto &offsets = lds.offsets;
    auto &there = lds.there;
    auto &bad = lds.bad, &odd = lds.odd;
    auto &ranges = lds.ranges;
    int* const samples = lds.samples;

    const int tid = (int)threadIdx.x, lane = tid & 63, col = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Workgroups go to the 8 XCDs by turns.  Blocks that share keys are kept on one XCD, whose
    // L2 then holds them, wherever the heads divide that way.
    int kv_head, item;
    {
        const int xcd = id & 7, turn = id >> 3;
        const int items = prefix.blocks * prefix.splits + own.blocks * own.splits;
        if (a.kv_heads % 8 == 0) {
            kv_head = xcd + 8 * (turn / items);
            item = turn % items;
        } else if (8 % a.kv_heads == 0) {
            kv_head = xcd % a.kv_heads;
            item = turn * (8 / a.kv_heads) + xcd / a.kv_heads;
        } else {
            kv_head = id % a.kv_heads;
            item = id / a.kv_heads;
        }
        if (item >= items || kv_head >= a.kv_heads) return;
    }
    const int prefix_items = prefix.blocks * prefix.splits;
    const Stage st = item < prefix_items ? prefix : own;
    if (item >= prefix_items) item -= prefix_items;
    const int block = item % st.blocks, split = item / st.blocks;

    Block k;
    if (!find_rows<kRows>(a, st, block, &k)) return;
    if (st.prefix) {
        sample_starts(a, samples, K::kThreads);
        __syncthreads();
    }
    if (tid < kRows) {
        const Row r = row_of(a, st, k, samples, tid);
        rows[tid] = i32x4{r.t, r.pos, r.lo, r.hi};
    }
    if (tid < 8) bad[tid] = odd[tid] = 0;
    __syncthreads();
    const int r0 = 32 * wave + col;
    // Read again where it is used: registers are short.
    const auto my_row = [&] {
        const i32x4 x = rows[r0];
        return Row{x[0], x[1], x[2], x[3]};
    };
    Range w{0x7FFFFFFF, 0, 0, 0x7FFFFFFF};
    range_add(w, my_row());
    w.lo = lanes_min(w.lo);
    w.hi = -lanes_min(-w.hi);
    w.all_lo = -lanes_min(-w.all_lo);
    w.all_hi = lanes_min(w.all_hi);
    if (lane == 0) ranges[0][wave] = w.lo, ranges[1][wave] = w.hi, ranges[2][wave] = w.all_lo, ranges[3][wave] = w.all_hi;
    __syncthreads();
    Range g{0x7FFFFFFF, 0, 0, 0x7FFFFFFF};
    for (int i = 0; i < W; i++) {
        g.lo = min(g.lo, ranges[0][i]);
        g.hi = max(g.hi, ranges[1][i]);
        g.all_lo = max(g.all_lo, ranges[2][i]);
        g.all_hi = min(g.all_hi, ranges[3][i]);
    }
    g.lo = __builtin_amdgcn_readfirstlane(g.hi == 0 ? 0 : g.lo);
    g.hi = __builtin_amdgcn_readfirstlane(g.hi);
    g.all_lo = __builtin_amdgcn_readfirstlane(g.all_lo);
    g.all_hi = __builtin_amdgcn_readfirstlane(g.all_hi);

    const int splits = st.prefix ? st.splits : max(1, (g.hi - g.lo + st.chunk - 1) / st.chunk);
    if (split >= splits) return;
    if (!st.prefix && split == 0 && tid == 0 && a.block_splits) a.block_splits[block * a.kv_heads + kv_head] = splits;
    const int base = (st.prefix ? 0 : g.lo) + split * st.chunk;
    const int c0 = max(base, g.lo), c1 = min(base + st.chunk, g.hi);
    const int64_t head = kv_head * c.head_stride;
    const int tiles = c1 > c0 ? (c1 - c0 + kTile - 1) / kTile : 0;

    // The rows' operand, zero where there is no row.
    u32x4 q[K::kSteps];
    int pos;
    float slope = 0.f;
    {
        const Row row = my_row();
        const int h = head_of(a, k, r0, kv_head);
        pos = row.pos;
        if (kScores == kBiased && row.t >= 0) slope = a.slopes[h];
        const uint16_t* p = a.q + row.t * a.q_stride + (int64_t)h * D + 8 * hi;
#pragma unroll
        for (int s = 0; s < K::kSteps; s++) q[s] = row.t >= 0 ? *(const u32x4*)(p + 16 * s) : u32x4{0, 0, 0, 0};
    }
    // A bias in the scores' units: the sums of the product start from it, or it is added to what a cap leaves.
    const float factor = a.factor;
    slope *= kLog2e / factor;
    const int least_pos = kScores == kBiased ? lanes_min(my_row().t >= 0 ? pos : 0x7FFFFFFF) : 0;
    const int last_pos = kScores == kBiased ? -lanes_min(my_row().t >= 0 ? -pos : 0x7FFFFFFF) : 0;
    // A maximum that has grown by less than 2^kSlack is left as it is: weights and sums stay within
    // what 16 and 32 bits hold, and the output is rescaled in a few tiles only.
    constexpr float kRaise = Mma<T>::kRaise > 0.f ? Mma<T>::kRaise - Mma<T>::kSlack : 0.f;
    const float slack = Mma<T>::kSlack / factor;

    float m = -INFINITY, sum = 0.f;
    f32x16 o[K::kDims];
#pragma unroll
    for (int i = 0; i < K::kDims; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[i][r] = 0.f;

    typename K::Staged staged[kAhead];
    const auto whole = [&](const Range& x, int n0) { return x.all_lo <= n0 && n0 + kTile <= min(x.all_hi, c1); };
    for (int n = tid; n < 3 * kTile; n += K::kThreads) {
        const bool in = c0 + n < c1;
        Place<S> at{};
        const bool found = in && key_place<S>(c, k.table, c0 + n, head, a.error, &at);
        if (in && !found) bad[n / kTile] = 1;
        offsets[n / kTile][n % kTile] = at;
        there[n / kTile][n % kTile] = found;
    }
    const uint8_t* const kc = c.k + tid % K::kChunks * S::kBits;
    const uint8_t* const vc = c.v + tid % K::kChunks * S::kBits;
    const auto place = [&](const typename K::Staged& x, int t) {  // tile t to LDS
        const int n0 = c0 + t * kTile;
        const bool full = n0 + kTile <= c1 && !bad[t & 7];
        if (K::store(x, (uint16_t*)keys_lds[t & 1], (uint16_t*)values_lds[t & 1], tid, full ? nullptr : there[t & 3],
                     !whole(g, n0)))
            odd[t & 7] = 1;
    };
    __syncthreads();
    if (tiles > 0) {
        K::load(staged[0], c, kc, vc, offsets[0], tid);
        if constexpr (kAhead == 2) K::load(staged[1], c, kc, vc, offsets[1], tid);
        place(staged[0], 0);
    }
    __syncthreads();

    const int swap_k = K::swap_k(col);
    const int key_at = col * D;
    const int lane16 = lane & 15, v_row = 4 * hi + (lane16 >> 2);
    int value_at[K::kDims];
#pragma unroll
    for (int i = 0; i < K::kDims; i++)
        value_at[i] = v_row * D + ((4 * i + 2 * ((lane >> 4) & 1) + ((lane16 & 3) >> 1)) ^ K::swap_v(v_row)) * 8 +
                      (lane16 & 1) * 4;

    // A tile: later ones' loads start, in the order of their use and whether or not there are such tiles (offsets
    // past the end are 0, which reads the cache's start), so that each wait is for the oldest loads only.
    const auto step = [&](int t, typename K::Staged& next, typename K::Staged& later) {
        const int n0 = c0 + t * kTile;
        const bool more = t + 1 < tiles;
        // The pages of the tile after those, by the first wave's lanes.
        const int n_look = n0 + 3 * kTile + (lane & (kTile - 1));
        const auto page_of = [&](int n) { return c.page.div((uint32_t)min(n, c1 - 1)); };
        int id_look = 0;
        if (wave == 0) id_look = k.table[page_of(n_look)];
        K::load(later, c, kc, vc, offsets[(t + kAhead) & 3], tid);

        if (odd[t & 7]) {
            // Of keys that some rows see and others do not, infinities and NaN reach only the rows
            // that do: a weight of zero would not stop them.  They are added to those rows one by one
            // and are zeros in the product.
            uint16_t* vb = (uint16_t*)values_lds[t & 1];
            const Row row = my_row();
#pragma unroll 1
            for (int n = 0; n < kTile; n++) {
                if (n0 + n < row.lo || n0 + n >= min(row.hi, c1)) continue;
#pragma unroll
                for (int d = 0; d < K::kDims; d++)
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const int chunk = (4 * d + (r >> 2)) ^ K::swap_v(n);
                        const u32x2 v = *(const u32x2*)(vb + n * D + chunk * 8 + 4 * hi);
                        if (!(not_finite<T>(v[0]) | not_finite<T>(v[1]))) continue;
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            o[d][r + j] += T::unpack(v[j >> 1] & ~only_finite<T>(v[j >> 1]))[j & 1];
                    }
            }
            __syncthreads();
            for (int n = tid; n < kTile * D / 2; n += K::kThreads)
                ((uint32_t*)vb)[n] = only_finite<T>(((uint32_t*)vb)[n]);
            __syncthreads();
        }
        if (n0 < w.hi && n0 + kTile > w.lo) {
            const uint16_t* kb = (const uint16_t*)keys_lds[t & 1] + key_at;
            const uint16_t* vb = (const uint16_t*)values_lds[t & 1];
            f32x16 x[K::kHalves];
            const auto add_bias = [&](auto first) {
                // Where all keys lie behind all rows, or before them, it grows by a slope from key to key.
                const float far = (float)(n0 + 4 * hi - pos);
                const bool behind = n0 + kTile - 1 <= least_pos;
                if (behind || n0 >= last_pos) {
                    const float by = behind ? slope : -slope, from = by * far;
#pragma unroll
                    for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                        for (int r = 0; r < 16; r++) {
                            const float b = __builtin_fmaf(by, (float)(32 * i + 8 * (r >> 2) + (r & 3)), from);
                            x[i][r] = decltype(first)::value ? b : x[i][r] + b;
                        }
                } else {
#pragma unroll
                    for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                        for (int r = 0; r < 16; r++) {
                            const float b = -slope * fabsf(far + (float)(32 * i + 8 * (r >> 2) + (r & 3)));
                            x[i][r] = decltype(first)::value ? b : x[i][r] + b;
                        }
                }
            };
            if (kScores == kBiased && a.cap_in < 0.f) {
                add_bias(std::true_type());
            } else {
#pragma unroll
                for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                    for (int r = 0; r < 16; r++) x[i][r] = 0.f;
            }
#pragma unroll
            for (int s = 0; s < K::kSteps; s++)
#pragma unroll
                for (int i = 0; i < K::kHalves; i++)
                    x[i] = Mma<T>::m32(*(const u32x4*)(kb + 32 * i * D + (((2 * s + hi) ^ swap_k) * 8)), q[s], x[i]);
            // Keys are read two products ahead.
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int s = 0; s < K::kSteps * K::kHalves - 4; s++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
            if (kScores == kCapped || (kScores == kBiased && a.cap_in >= 0.f)) {
                const auto most = [&] {
                    float y = fabsf(x[0][0]);
#pragma unroll
                    for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                        for (int r = 0; r < 16; r++) y = max_f32(y, fabsf(x[i][r]));
                    return y;
                };
                cap_scores(a, most, [&](auto form) {
#pragma unroll
                    for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                        for (int r = 0; r < 16; r++) x[i][r] = form(x[i][r]);
                });
                if (kScores == kBiased) add_bias(std::false_type());
            }
            const bool gap = bad[t & 7];
            if (gap || !whole(w, n0)) {
                // A lane's keys are these constants and n0 + 4 hi.
                const Row row = my_row();
                const int from = row.lo - n0 - 4 * hi, to = min(row.hi, c1) - n0 - 4 * hi;
#pragma unroll
                for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int n = 32 * i + 8 * (r >> 2) + (r & 3);
                        x[i][r] = n >= from && n < to ? x[i][r] : -INFINITY;
                    }
                if (gap) {
                    const uint64_t in = __ballot(there[t & 3][lane & (kTile - 1)]) >> (4 * hi);
#pragma unroll
                    for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                        for (int r = 0; r < 16; r++)
                            x[i][r] = (in >> (32 * i + 8 * (r >> 2) + (r & 3))) & 1 ? x[i][r] : -INFINITY;
                }
            }
            float top = x[0][0];
#pragma unroll
            for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) top = max_f32(top, x[i][r]);
            top = across32_max(top);
            if (__any(!(top <= m + slack))) {
                const float next = max_f32(m, top);
                const float keep = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - next) * factor);
                m = next;
                sum *= keep;
#pragma unroll
                for (int i = 0; i < K::kDims; i++) o[i] *= keep;
            }
            const float base_m = (m == -INFINITY ? 0.f : m * factor) - kRaise;
            // A weight is rounded to the values' 16-bit type, as the matrix product takes it.
            u32x4 p[K::kHalves][2];
#pragma unroll
            for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][r], factor, -base_m));
                    const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][r + 1], factor, -base_m));
                    sum += e0;
                    sum += e1;
                    p[i][r >> 3][(r >> 1) & 3] = T::pack(e0, e1);
                }
#pragma unroll
            for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                for (int s = 0; s < 2; s++)
#pragma unroll
                    for (int d = 0; d < K::kDims; d++) {
                        const uint16_t* at = vb + value_at[d] + (32 * i + 16 * s) * D;
                        const u32x2 v0 = K::transposed(at), v1 = K::transposed(at + 8 * D);
                        o[d] = Mma<T>::m32(u32x4{v0[0], v0[1], v1[0], v1[1]}, p[i][s], o[d]);
                    }
        }

        if (more) place(next, t + 1);
        if (wave == 0) {
            Place<S> at{};
            bool found = false;
            if (n_look < c1) {
                if (id_look < 0 || id_look >= c.num_pages) {
                    bad[(t + 3) & 7] = 1;
                    if (a.error) atomicOr(a.error, GFD_KV_ERR_PAGE);
                } else {
                    at = place_of<S>(c, id_look, (uint32_t)n_look - page_of(n_look) * c.page.d, head);
                    found = true;
                }
            }
            if (lane < kTile) {
                offsets[(t + 3) & 3][lane] = at;
                there[(t + 3) & 3][lane] = found;
            }
        }
        if (tid == 0) bad[(t + 5) & 7] = odd[(t + 5) & 7] = 0;
        __syncthreads();
    };
    // The rows' operand is there before the first tile: left to the loop, its wait would stand in front of every
    // tile's first product and cover the next tiles' loads too.
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    if constexpr (kAhead == 1) {
        for (int t = 0; t < tiles; t++) step(t, staged[0], staged[0]);
    } else {
        for (int t = 0; t < tiles; t += 2) {
            step(t, staged[1], staged[0]);
            if (t + 1 < tiles) step(t + 1, staged[0], staged[1]);
        }
    }

    sum = across32_sum(sum);
    const Row row = my_row();
    const int h = head_of(a, k, r0, kv_head);
    if (row.t < 0) return;
    if (st.direct && splits == 1) {
        const float scale = sum == 0.f ? 0.f : c.v_scale / sum;
        uint16_t* out = a.out + row.t * a.out_stride + (int64_t)h * D + 4 * hi;
#pragma unroll
        for (int d = 0; d < K::kDims; d++)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const u32x2 y{T::pack(o[d][r] * scale, o[d][r + 1] * scale),
                              T::pack(o[d][r + 2] * scale, o[d][r + 3] * scale)};
                *(u32x2*)(out + 32 * d + 2 * r) = sum == 0.f ? u32x2{0, 0} : y;
            }
        if (a.lse && hi == 0)
            a.lse[(int64_t)row.t * a.q_heads + h] =
                sum == 0.f ? -INFINITY : (m * factor + (a.shift - kRaise) + __builtin_amdgcn_logf(sum)) * kLn2;
    } else {
        const int64_t at = slot_of(a, st.first_slot + split, row.t, h);
        if (hi == 0) a.part_ml[at] = f32x2{m * factor + (a.shift - kRaise), sum};
        if (sum == 0.f) return;  // its weight is zero and it is not read
        float* out = a.part_o + at * D + 4 * hi;
#pragma unroll
        for (int d = 0; d < K::kDims; d++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *(f32x4*)(out + 32 * d + 2 * r) = f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
    }
}

template <typename T, typename S, int D, int W, int kScores>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : 2) void attend_tiles_kernel(Call a, CacheOf<S> c, Stage prefix, Stage own) {
    __shared__ TilesLds<T, S, D, W> lds;
    attend_tiles<T, S, D, W, kScores>(a, c, prefix, own, (int)blockIdx.x, lds);
}

// Workgroups that a launch has for these stages: XCDs' shares are rounded up to whole turns.
inline int64_t tiles_groups(const Call& a, const Stage& prefix, const Stage& own) {
    const int64_t items = (int64_t)prefix.blocks * prefix.splits + (int64_t)own.blocks * own.splits;
    const int64_t turns = a.kv_heads % 8 == 0   ? items * (a.kv_heads / 8)
                          : 8 % a.kv_heads == 0 ? (items + 8 / a.kv_heads - 1) / (8 / a.kv_heads)
                                                : (items * a.kv_heads + 7) / 8;
    return turns * 8;
}

// f(scores) with the kind of scores that the call has, as a constant.
template <typename F>
int with_scores(const Call& a, F f) {
    if (a.slopes) return f(std::integral_constant<int, kBiased>());
    if (a.cap_in >= 0.f) return f(std::integral_constant<int, kCapped>());
    return f(std::integral_constant<int, kPlain>());
}

template <typename T, typename S>
int launch_tiles(const Call& a, const CacheOf<S>& c, const Stage& prefix, const Stage& own, int dim, int waves,
                 hipStream_t st) {
    const dim3 grid((unsigned)tiles_groups(a, prefix, own));
    const auto go = [&](auto kernel, int w) {
        return start(kernel, grid, 64 * w, st, a, c, prefix, own);
    };
    const auto pick = [&](auto d) {
        constexpr int D = decltype(d)::value;
        return with_scores(a, [&](auto scores) {
            constexpr int kScores = decltype(scores)::value;
            if constexpr (D != 256) {
                if (waves == 8) return go(attend_tiles_kernel<T, S, D, 8, kScores>, 8);
            }
            return go(attend_tiles_kernel<T, S, D, 4, kScores>, 4);
        });
    };
    if (dim == 64) return pick(std::integral_constant<int, 64>());
    if (dim == 128) return pick(std::integral_constant<int, 128>());
    return pick(std::integral_constant<int, 256>());
}

}  // namespace kv
}  // namespace gfd

#pragma once
// Attention of many rows: prompts, chunks of prompts, a batch over its shared prefix.
//
// Each key is used by hundreds of rows, so the matrix products bound the time.  A
// workgroup of W waves takes 32 W rows, 32 a wave, and walks the keys in tiles
// that all of its waves read from LDS.  A tile's keys and values lie there
// as 16-bit numbers (8-bit ones are widened on the way in, once for the
// workgroup), twice: the next tiles are loaded to registers while this one is
// computed, and written behind it, so that a tile costs one barrier.
//
// A tile: scores^T[32 keys][32 rows] by 32x32x16 products, keys as the left operand.
// The result's lane holds row l % 32 and the keys 8 (r / 4) + 4 (l / 32) + r % 4;
// eight of these, rounded, are the right operand of out^T[32 dims][32 rows] += V^T P
// as they lie.  V^T comes from LDS by transposing reads, 4 keys of one dim a lane.
// Chunks of 16 bytes are swapped by row, so that neither read finds two rows in a bank.
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
    static constexpr int kUnitWords = 2 * S::kBytes;

    struct Staged {
        uint32_t k[kUnits][kUnitWords], v[kUnits][kUnitWords];
        bool on[kUnits];
    };

    // Where a row's chunk lies, so that rows that are read together meet in no bank (64 of 4 bytes).  Keys: one chunk
    // of 16 rows at once.  Values: two neighbouring chunks of 4 rows.  A row of 128 bytes (D 64) is half the banks.
    static __device__ __forceinline__ int swap_k(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
    static __device__ __forceinline__ int swap_v(int row) { return D == 64 ? ((row >> 1) & 1) * 4 : (row & 3) * 4; }

    static __device__ __forceinline__ void load(Staged& g, const Cache& c, const int64_t* off, int tid) {
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            const int n = tid + u * kThreads, row = n / kChunks, chunk = n % kChunks;
            const int64_t o = off[row];
            g.on[u] = o >= 0;
            const int64_t at = (o < 0 ? 0 : o) + chunk * 8 * S::kBytes;
            if constexpr (S::kBytes == 2) {
                const u32x4 k = *(const u32x4*)(c.k + at), v = *(const u32x4*)(c.v + at);
#pragma unroll
                for (int i = 0; i < 4; i++) g.k[u][i] = k[i], g.v[u][i] = v[i];
            } else {
                const u32x2 k = *(const u32x2*)(c.k + at), v = *(const u32x2*)(c.v + at);
#pragma unroll
                for (int i = 0; i < 2; i++) g.k[u][i] = k[i], g.v[u][i] = v[i];
            }
        }
    }
    static __device__ __forceinline__ u32x4 widened(const uint32_t (&w)[kUnitWords], bool on) {
        u32x4 r;
        if constexpr (S::kBytes == 2) r = u32x4{w[0], w[1], w[2], w[3]};
        else r = u32x4{Mma<T>::widen_lo(w[0]), Mma<T>::widen_hi(w[0]), Mma<T>::widen_lo(w[1]), Mma<T>::widen_hi(w[1])};
        return on ? r : u32x4{0, 0, 0, 0};
    }
    // Nonzero where look is set and a value is infinite or NaN.
    static __device__ __forceinline__ uint32_t store(const Staged& g, uint16_t* kb, uint16_t* vb, int tid, bool look) {
        uint32_t odd = 0;
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            const int n = tid + u * kThreads, row = n / kChunks, chunk = n % kChunks;
            const u32x4 v = widened(g.v[u], g.on[u]);
            *(u32x4*)(kb + row * D + (chunk ^ swap_k(row)) * 8) = widened(g.k[u], g.on[u]);
            *(u32x4*)(vb + row * D + (chunk ^ swap_v(row)) * 8) = v;
            if (look) {
#pragma unroll
                for (int i = 0; i < 4; i++) odd |= not_finite<T>(v[i]);
            }
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

template <typename T, typename S, int D, int W, int kScores>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : 2) void attend_tiles_kernel(Call a, Cache c, Stage prefix, Stage own) {
    using K = TilesKernel<T, S, D, W>;
    constexpr int kTile = K::kTile, kRows = K::kRows;
    // Tiles under way.  A tile's 64 keys take less time than a load from memory (1.9 us) where a CU has
    // one workgroup or the dims are few, so two, where the registers hold them: not where 4 waves move 128
    // dims of 16 bits, or do more with the scores.
    constexpr int kAhead = W == 8 || D == 64 || (S::kBytes == 1 && (D == 256 || kScores == kPlain)) ||
                                   (D == 256 && kScores != kBiased) ? 2 : 1;
    __shared__ u32x4 keys_lds[2][kTile * D / 8];
    __shared__ u32x4 values_lds[2][kTile * D / 8];
    __shared__ i32x4 rows[kRows];
    __shared__ int64_t offsets[4][kTile];
    __shared__ int bad[8], odd[8], ranges[4][W];
    int* const samples = (int*)keys_lds;
    static_assert(sizeof(keys_lds) >= (kSamples + 1) * sizeof(int), "samples fit the keys");

    const int tid = (int)threadIdx.x, lane = tid & 63, col = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Workgroups go to the 8 XCDs by turns.  Blocks that share keys are kept on one XCD, whose
    // L2 then holds them, wherever the heads divide that way.
    int kv_head, item;
    {
        const int id = (int)blockIdx.x, xcd = id & 7, turn = id >> 3;
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
        if (kScores == kBiased && a.slopes && row.t >= 0) slope = a.slopes[h] * kLog2e;
        const uint16_t* p = a.q + row.t * a.q_stride + (int64_t)h * D + 8 * hi;
#pragma unroll
        for (int s = 0; s < K::kSteps; s++) q[s] = row.t >= 0 ? *(const u32x4*)(p + 16 * s) : u32x4{0, 0, 0, 0};
    }
    // Exponents have base 2.  Plain scores stay the product's sums: the factor is positive, so the
    // maximum is the same, and one multiply-add under the exponent applies it.  Capped ones,
    // cap tanh y = cap - 2 cap / (e^2y + 1), stay -1 / (e^2y + 1): off by a few 2^-24 as the sums are.
    const float raw = a.scale * c.k_scale, cap = a.softcap * kLog2e;
    const float into_cap = a.softcap > 0.f ? raw / a.softcap * (2.f * kLog2e) : 0.f;
    const float factor = kScores == kPlain ? raw * kLog2e : kScores == kCapped ? 2.f * cap : 1.f;
    const float shift = kScores == kPlain ? 0.f : cap;
    const int least_pos = kScores == kBiased ? lanes_min(my_row().t >= 0 ? pos : 0x7FFFFFFF) : 0;
    // A maximum that has grown by less than 2^8 is left as it is: weights and sums stay far from
    // what 16 and 32 bits hold, and the output is rescaled in a few tiles only.
    const float slack = 8.f / factor;

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
        const int64_t at = in ? key_offset(c, k.table, c0 + n, head, a.error) : -1;
        if (in && at < 0) bad[n / kTile] = 1;
        offsets[n / kTile][n % kTile] = at;
    }
    __syncthreads();
    if (tiles > 0) {
        K::load(staged[0], c, offsets[0], tid);
        if constexpr (kAhead == 2) K::load(staged[1], c, offsets[1], tid);
        if (K::store(staged[0], (uint16_t*)keys_lds[0], (uint16_t*)values_lds[0], tid, !whole(g, c0))) odd[0] = 1;
    }
    __syncthreads();

    const int swap_k = K::swap_k(col);
    const int key_at = col * D;
    const int lane16 = lane & 15, v_row = 4 * hi + (lane16 >> 2);
    int value_at[K::kDims];
#pragma unroll
    for (int i = 0; i < K::kDims; i++)
        value_at[i] = v_row * D + ((4 * i + 2 * ((lane >> 4) & 1) + ((lane16 & 3) >> 1)) ^ K::swap_v(v_row)) * 8 + (lane16 & 1) * 4;

    // A tile: later ones' loads start, in the order of their use and whether or not there are such tiles (offsets
    // past the end are -1, which reads the cache's start), so that each wait is for the oldest loads only.
    const auto step = [&](int t, typename K::Staged& next, typename K::Staged& later) {
        const int n0 = c0 + t * kTile;
        const bool more = t + 1 < tiles;
        const auto page_of = [&](int n) { return c.page.div((uint32_t)min(n, c1 - 1)); };
        const int id3 = k.table[page_of(n0 + 3 * kTile + (tid & (kTile - 1)))];
        K::load(later, c, offsets[(t + kAhead) & 3], tid);

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
#pragma unroll
            for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) x[i][r] = 0.f;
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
            if constexpr (kScores != kPlain) {
                const auto capped = [&](float y) {
                    return __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(y * into_cap));
                };
                if (kScores == kCapped || a.softcap > 0.f) {
#pragma unroll
                    for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                        for (int r = 0; r < 16; r++) x[i][r] = capped(x[i][r]);
                }
                if constexpr (kScores == kBiased) {
                    const float by = a.softcap > 0.f ? 2.f * cap : raw * kLog2e;
                    // Where all keys lie behind all rows, a row's bias grows by its slope from key to key.
                    const int far = n0 + 4 * hi - pos;
                    if (n0 + kTile - 1 <= least_pos) {
                        const float bias = slope * (float)far;
#pragma unroll
                        for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                            for (int r = 0; r < 16; r++)
                                x[i][r] = __builtin_fmaf(
                                    x[i][r], by, __builtin_fmaf(slope, (float)(32 * i + 8 * (r >> 2) + (r & 3)), bias));
                    } else {
#pragma unroll
                        for (int i = 0; i < K::kHalves; i++)
#pragma unroll
                            for (int r = 0; r < 16; r++)
                                x[i][r] = __builtin_fmaf(
                                    -slope, fabsf((float)(far + 32 * i + 8 * (r >> 2) + (r & 3))), x[i][r] * by);
                    }
                }
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
                    const uint64_t in = __ballot(offsets[t & 3][lane & (kTile - 1)] >= 0) >> (4 * hi);
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
            const float base_m = m == -INFINITY ? 0.f : m * factor;
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

        if (more && K::store(next, (uint16_t*)keys_lds[(t + 1) & 1], (uint16_t*)values_lds[(t + 1) & 1], tid,
                             !whole(g, n0 + kTile)))
            odd[(t + 1) & 7] = 1;
        if (tid < kTile) {
            int64_t at = -1;
            const int n3 = n0 + 3 * kTile + tid;
            if (n3 < c1) {
                if (id3 < 0 || id3 >= c.num_pages) {
                    bad[(t + 3) & 7] = 1;
                    if (a.error) atomicOr(a.error, GFD_KV_ERR_PAGE);
                } else {
                    at = id3 * c.page_stride + (int64_t)((uint32_t)n3 - page_of(n3) * c.page.d) * c.slot_stride + head;
                }
            }
            offsets[(t + 3) & 3][tid] = at;
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
                sum == 0.f ? -INFINITY : (m * factor + shift + __builtin_amdgcn_logf(sum)) * kLn2;
    } else {
        const int64_t at = slot_of(a, st.first_slot + split, row.t, h);
        if (hi == 0) a.part_ml[at] = f32x2{m == -INFINITY ? m : m * factor + shift, sum};
        if (sum == 0.f) return;  // its weight is zero and it is not read
        float* out = a.part_o + at * D + 4 * hi;
#pragma unroll
        for (int d = 0; d < K::kDims; d++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *(f32x4*)(out + 32 * d + 2 * r) = f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
    }
}

template <typename T, typename S>
int launch_tiles(const Call& a, const Cache& c, const Stage& prefix, const Stage& own, int dim, int waves,
                 hipStream_t st) {
    const int64_t items = (int64_t)prefix.blocks * prefix.splits + (int64_t)own.blocks * own.splits;
    // See the kernel: XCDs' shares are rounded up to whole turns.
    const int64_t turns = a.kv_heads % 8 == 0   ? items * (a.kv_heads / 8)
                          : 8 % a.kv_heads == 0 ? (items + 8 / a.kv_heads - 1) / (8 / a.kv_heads)
                                                : (items * a.kv_heads + 7) / 8;
    const dim3 grid((unsigned)(turns * 8));
    const auto go = [&](auto kernel, int w) {
        hipLaunchKernelGGL(kernel, grid, dim3(64 * w), 0, st, a, c, prefix, own);
    };
    const auto pick = [&](auto d) {
        constexpr int D = decltype(d)::value;
        const auto with = [&](auto scores) {
            constexpr int kScores = decltype(scores)::value;
            if constexpr (D != 256) {
                if (waves == 8) return go(attend_tiles_kernel<T, S, D, 8, kScores>, 8);
            }
            go(attend_tiles_kernel<T, S, D, 4, kScores>, 4);
        };
        if (a.slopes) with(std::integral_constant<int, kBiased>());
        else if (a.softcap > 0.f) with(std::integral_constant<int, kCapped>());
        else with(std::integral_constant<int, kPlain>());
    };
    if (dim == 64) pick(std::integral_constant<int, 64>());
    if (dim == 128) pick(std::integral_constant<int, 128>());
    if (dim == 256) pick(std::integral_constant<int, 256>());
    return (int)hipGetLastError();
}

}  // namespace kv
}  // namespace gfd

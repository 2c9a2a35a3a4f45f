// Attention over the paged cache (gfx950): the calls' checks, what they launch,
// and the kernel that joins partial results.
//
// Per query row (token, head) with score s_j over its visible keys j:
// out = sum exp(s_j - m) v_j / sum exp(s_j - m), lse = m + log of that sum,
// with the running maximum m and sums in 32 bits.  A range of keys leaves
// (m, sum, unnormalised out); ranges are joined by M = max m, each weighted by exp(m - M).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gfd_capi.h"
#include "paged_attention.h"

namespace gfd {
namespace kv {
namespace {

constexpr int kJoinBlock = 256;

// A workgroup joins kPart rows of an own-keys block, a wave per row: a lane
// weighs one range of 64, then holds D / 64 dims.  Reads what the ranges left once; a
// launch and a chain of four loads for small batches (3.4 us), 4 to 9 us for 2048 rows of up to 18 ranges.
template <typename T, int D, int kRows, int kPart>
__global__ __launch_bounds__(kJoinBlock) void join_kernel(Call a, Cache c, Stage own) {
    constexpr int kDims = D / 64, kWaves = kJoinBlock / 64;
    typedef float Dims __attribute__((ext_vector_type(kDims)));
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int kv_head = (int)blockIdx.x % a.kv_heads, block = (int)blockIdx.x / a.kv_heads;
    const int splits = a.block_splits[blockIdx.x], slots = own.first_slot + splits;  // unset without rows
    if (own.direct && splits == 1) return;
    Block k;
    if (!find_rows<kRows>(a, own, block, &k)) return;

    const int first = (int)blockIdx.y * kPart;
    for (int r = first + wave; r < min(first + kPart, k.rows); r += kWaves) {
        const int t = k.seq.first + (int)a.group.div((uint32_t)(k.first_row + r));
        const int h = head_of(a, k, r, kv_head);
        float top = -INFINITY;
        for (int s0 = 0; s0 < slots; s0 += 64) {
            if (s0 + lane < slots) top = max_f32(top, a.part_ml[slot_of(a, s0 + lane, t, h)][0]);
        }
        top = across16_max(top);
        for (int off = 8; off; off >>= 1) top = max_f32(top, __shfl_xor(top, off));
        float total = 0.f;
        Dims o = 0.f;
        for (int s0 = 0; s0 < slots; s0 += 64) {
            float w = 0.f, l = 0.f;
            if (s0 + lane < slots) {
                const f32x2 ml = a.part_ml[slot_of(a, s0 + lane, t, h)];
                l = ml[1];
                w = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[0] - top);
            }
            total += l == 0.f ? 0.f : w * l;
            const float* from = a.part_o + slot_of(a, s0, t, h) * D + lane * kDims;
            const int64_t step = (int64_t)a.num_tokens * a.q_heads * D;
            const int n = min(64, slots - s0);
            for (int s = 0; s < n; s += 8) {  // lanes past the last range weigh nothing
                Dims x[8];
                float ws[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    ws[j] = __shfl(w, s + j);
                    x[j] = 0.f;
                    if (__shfl(l, s + j) != 0.f) x[j] = *(const Dims*)(from + (s + j) * step);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) o += ws[j] * x[j];
            }
        }
        total = across16_sum(total);
        for (int off = 8; off; off >>= 1) total += __shfl_xor(total, off);
        const float scale = total == 0.f ? 0.f : c.v_scale / total;
        uint16_t* out = a.out + t * a.out_stride + (int64_t)h * D + lane * kDims;
        if constexpr (kDims == 1) {
            out[0] = (uint16_t)T::pack(o[0] * scale, 0.f);
        } else {
            for (int d = 0; d < kDims; d += 2) *(uint32_t*)(out + d) = T::pack(o[d] * scale, o[d + 1] * scale);
        }
        if (a.lse && lane == 0)
            a.lse[(int64_t)t * a.q_heads + h] =
                total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * kLn2;
    }
}

// How a call is cut into row blocks and key ranges.
struct Plan {
    int prefix_waves, own_waves;  // of a block of 32 rows a wave; 0: few rows (attend_rows.h)
    int few_waves;                // of a workgroup of few rows
    int rows;                     // of an own-keys block
    Stage prefix, own;
    int slots;      // partial results per row
    int64_t threads;  // of the largest launch, at most
    int64_t bytes;  // of workspace
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Workgroups of four waves that fit a CU: two, but one of 256 dims, whose outputs take the registers of two waves a
// SIMD (not so for up to 16 rows of an 8-bit cache).
constexpr int kCus = 256;
int fit_cu(int dim, bool few, int rows, int dtype) {
    return dim != 256 || (few && rows == 16 && dtype == GFD_E4M3) ? 2 : 1;
}
// Few rows: a round is what fits the card at once.  Sequences of very different
// lengths spread best over kRounds rounds of them (64 of up to 8192 keys: ranges of 1024 163 us, of 512 173),
// but a range of a few hundred keys is half start-up (8 of 8192: ranges of 256 64 us, of 512 57), and
// below one round the shortest range, a tile per wave, counts.  256 dims: one sequence of 8000 keys 24.6 us, with
// rounds of two workgroups a CU 33.7; two times 5 tokens 36.4, 48.6; 8 sequences of 3000 54, 49.
// Past kMostRounds ranges grow instead, walked in pieces: a full card gains nothing from more of them, and what they
// leave to be joined would grow with the context (512 of 131072 keys: 1.1 GB in ranges of one piece, 17 MB so).
// 64 of up to 32768: 616 us, in ranges of one piece 634; 512 of up to 4096, whole 515, 520.
constexpr int kRounds = 4, kMostRounds = 16, kMinChunk = 128, kGoodChunk = 512;
// From so many workgroups on (two a CU), short contexts get a wave each: of four waves most would
// find no tile or one, and what takes the time is a workgroup's start (91 times 12 heads of 256 dims and 27 keys:
// 46 us, with one wave 17; 70 times 8 heads of 128 dims and 128 keys: 15.2, 12.7).
constexpr int kOneWave = 512;
// Many rows: what ranges leave has to be joined, so blocks are split only where they leave half of the CUs empty,
// and not below 4 tiles.  Then as many workgroups as fit a CU (4 times 60 tokens over 4000 keys: 31 us, with one 35; 1000
// tokens over 2000 keys, a block each: 65 us whole, 75 in two ranges), but beside few rows that take the other half
// of the CUs one (64 requests on 32768 shared keys: 91 us, with two 103).  256 dims: 100 tokens over 4196 keys 54 us,
// with two workgroups a CU 69; 512 over 2048 84, 98; a prefix of 32768 for 64 requests 160, with two 183.
constexpr int kTilesMinChunk = 256;

void split(Stage* st, int64_t items, int64_t keys, bool few, int fit) {
    if (few) {
        const int64_t round = (int64_t)fit * kCus;
        const auto chunk_for = [&](int64_t groups) {
            return ceil_div(ceil_div(keys * items, groups), kMinChunk) * kMinChunk;
        };
        const int64_t least = std::max<int64_t>(kMinChunk, std::min<int64_t>(kGoodChunk, chunk_for(round)));
        const int64_t spread = std::min<int64_t>(kRowsPiece, std::max(least, chunk_for(round * kRounds)));
        const int64_t whole = std::max<int64_t>(1, ceil_div(keys, kMinChunk)) * kMinChunk;
        st->chunk = (int)std::min(whole, std::max(spread, chunk_for(round * kMostRounds)));
    } else {
        const int64_t fill = st->prefix ? kCus : fit * kCus;
        const int64_t parts = items * 2 > kCus ? 1 : fill / std::max<int64_t>(items, 1);
        st->chunk = (int)std::max<int64_t>(kTilesMinChunk, ceil_div(ceil_div(keys, parts), 64) * 64);
    }
    st->splits = (int)std::max<int64_t>(1, ceil_div(keys, st->chunk));
}

// Waves of a block of many rows: 8, for half the reads of the cache, where that still gives every CU two blocks
// (4096 tokens over 16384 keys: 950 us, with 4 waves 1077; 2048 tokens of 32 heads, one block each: 87 us, with 4 73).
int tile_waves(int64_t rows, int64_t heads, int dim) { return dim != 256 && rows * heads >= 2 * 256 * 256 ? 8 : 4; }

Plan make_plan(const gfd_kv_cache& cache, const gfd_attention& w, int prefix_len) {
    Plan p{};
    const int64_t group = w.num_q_heads / cache.num_heads, heads = cache.num_heads;
    const int64_t seq_rows = std::min<int64_t>(w.max_q_len, w.num_tokens) * group;
    const int64_t all_rows = w.num_tokens * group;
    // Keys that a block can see: with a window, those of its tokens' windows (a prefix mask adds later keys).
    int64_t keys = std::max(w.max_kv_len - prefix_len, 0);
    if (w.window && !w.prefix_end) keys = std::min<int64_t>(keys, (int64_t)w.window + w.max_q_len);
    if (seq_rows <= 32) {
        p.rows = seq_rows <= 16 ? 16 : 32;
        if (prefix_len && all_rows <= 32) p.rows = all_rows <= 16 ? 16 : 32;  // one launch takes both stages
        p.own.blocks = w.batch;
        p.own.whole = 1;
    } else {
        p.own_waves = tile_waves(all_rows, heads, cache.head_dim);
        p.rows = 32 * p.own_waves;
        p.own.blocks = (int)std::min<int64_t>(w.batch * ceil_div(seq_rows, p.rows), all_rows / p.rows + w.batch);
    }
    const auto fit = [&](bool few) { return fit_cu(cache.head_dim, few, p.rows, cache.dtype); };
    split(&p.own, p.own.blocks * heads, keys, !p.own_waves, fit(!p.own_waves));
    p.few_waves = 4;
    if (!p.own_waves && !prefix_len && keys <= kRowsShort && p.own.blocks * heads >= kOneWave) {
        p.few_waves = 1;
        p.own.chunk = kRowsShort;
        p.own.splits = 1;
    }
    p.own.direct = !prefix_len;
    if (prefix_len) {
        p.prefix.prefix = 1;
        p.prefix_waves = all_rows <= 32 ? 0 : p.own_waves ? p.own_waves : 4;
        p.prefix.blocks = (int)ceil_div(all_rows, p.prefix_waves ? 32 * p.prefix_waves : p.rows);
        split(&p.prefix, p.prefix.blocks * heads, prefix_len, !p.prefix_waves, fit(!p.prefix_waves));
        p.own.first_slot = p.prefix.splits;
    }
    p.slots = p.own.first_slot + p.own.splits;
    // Turns of 8 workgroups are filled up.  The join, where there is one, has as many threads at most.
    const int64_t items = ((int64_t)p.prefix.blocks * p.prefix.splits + (int64_t)p.own.blocks * p.own.splits) * heads;
    p.threads = (items + 16) * 64 * (p.own_waves ? p.own_waves : p.few_waves);
    if (p.slots > 1)
        p.bytes = (int64_t)p.slots * w.num_tokens * w.num_q_heads * (cache.head_dim + 2) * 4 + p.own.blocks * heads * 4;
    return p;
}

template <typename T, int D, int kRows, int kPart>
int launch_join(const Call& a, const Cache& c, const Stage& own, hipStream_t st) {
    return start(join_kernel<T, D, kRows, kPart>, dim3((unsigned)(own.blocks * a.kv_heads), kRows / kPart), kJoinBlock, st,
                 a, c, own);
}
template <typename T, int D>
int launch_join(const Call& a, const Cache& c, const Plan& p, hipStream_t st) {
    // A wave a row takes the least time where few rows leave the card empty (100 tokens over 4196 keys: 33 us in all,
    // with four rows a wave 38); with many it does not matter.
    const bool few = (int64_t)p.own.blocks * p.rows * a.kv_heads <= 16384;
    if (p.rows == 16) return launch_join<T, D, 16, 4>(a, c, p.own, st);
    if (p.rows == 32) return launch_join<T, D, 32, 4>(a, c, p.own, st);
    if (p.rows == 128) return few ? launch_join<T, D, 128, 4>(a, c, p.own, st) : launch_join<T, D, 128, 16>(a, c, p.own, st);
    return few ? launch_join<T, D, 256, 4>(a, c, p.own, st) : launch_join<T, D, 256, 16>(a, c, p.own, st);
}

template <typename T, typename S>
int launch(const Call& a, const Cache& c, const Plan& p, int dim, hipStream_t st) {
    int rc;
    if (p.own_waves) {  // both stages have blocks of the same rows
        rc = launch_tiles<T, S>(a, c, p.prefix, p.own, dim, p.own_waves, st);
    } else if (p.prefix_waves && p.own.chunk > kRowsPiece) {  // a batch that fills the card without the prefix
        const Stage none{0, 0, 0, 0, 1, 0, 0};
        rc = launch_tiles<T, S>(a, c, p.prefix, none, dim, p.prefix_waves, st);
        if (!rc) rc = launch_rows<T, S>(a, c, none, p.own, dim, p.rows == 32, p.few_waves, st);
    } else if (p.prefix_waves) {
        rc = launch_both<T, S>(a, c, p.prefix, p.own, dim, p.rows == 32, st);
    } else {
        rc = launch_rows<T, S>(a, c, p.prefix, p.own, dim, p.rows == 32, p.few_waves, st);
    }
    if (rc || p.slots == 1) return rc;
    return dim == 64 ? launch_join<T, 64>(a, c, p, st) : dim == 128 ? launch_join<T, 128>(a, c, p, st)
                                                                   : launch_join<T, 256>(a, c, p, st);
}

const char* check_call(const gfd_kv_cache* cache, const gfd_attention* call, int prefix_len) {
    if (const char* why = check_cache(cache)) return why;
    if (!call) return "no call";
    const gfd_attention& w = *call;
    if (w.dtype != GFD_BF16 && w.dtype != GFD_FP16) return "q is neither GFD_BF16 nor GFD_FP16";
    if (cache->dtype != GFD_E4M3 && cache->dtype != w.dtype) return "the cache's type is neither q's nor GFD_E4M3";
    if (w.num_q_heads < 1 || w.num_q_heads > 65535 || w.num_q_heads % cache->num_heads != 0)
        return "num_q_heads is no multiple of the cache's heads";
    if (w.batch < 0 || w.num_tokens < 0 || w.max_q_len < 0 || w.max_kv_len < 0 || w.max_kv_len > (1 << 30) ||
        w.batch > (1 << 24) || w.num_tokens > (1 << 24))
        return "batch, num_tokens, max_q_len or max_kv_len out of range";
    if (prefix_len < 0 || prefix_len > (1 << 30)) return "prefix_len out of range";
    if (!(w.softcap >= 0.f) || w.softcap > 3.4e38f) return "softcap is negative or not finite";
    if (!(w.scale > 0.f) || w.scale > 3.4e38f) return "scale is not positive and finite";
    // Scores are kept in units of the product with the stored keys: the factor between must not leave 32 bits.
    const double raw = (double)w.scale * (cache->dtype == GFD_E4M3 ? cache->k_scale : 1.f);
    if (raw < 0x1p-100 || raw > 0x1p100) return "scale times k_scale is outside 2^-100 to 2^100";
    if (w.window < 0) return "negative window";
    if ((w.q_stride | w.out_stride) % 8 != 0 || ((uintptr_t)w.q | (uintptr_t)w.out) % 16 != 0)
        return "rows' pointers or strides are not multiples of 16 bytes";
    const int64_t pages = ((int64_t)std::max(w.max_kv_len - prefix_len, 0) + cache->page_size - 1) / cache->page_size;
    if (w.table_stride < pages) return "block_table's rows are shorter than max_kv_len needs";
    // The first two keep the plan's products within 64 bits: a workgroup has a wave at least.
    if ((int64_t)w.num_tokens * w.num_q_heads > (1 << 30) || (int64_t)w.batch * cache->num_heads >= kGridThreads / 64 ||
        make_plan(*cache, w, prefix_len).threads >= kGridThreads)
        return "more work than one launch takes";
    return nullptr;
}

int attention(const char* name, const gfd_kv_cache* cache, const gfd_attention* call, const int* prefix_table,
              int prefix_len, void* workspace, size_t workspace_bytes, int* error_flag, void* stream) {
    if (const char* why = check_call(cache, call, prefix_len)) return refused(name, why);
    const gfd_attention& w = *call;
    if (w.batch == 0 || w.num_tokens == 0 || w.max_q_len == 0) return 0;
    if (!w.q || !w.out || !w.q_start || !w.kv_len) return refused(name, "q, out, q_start or kv_len is missing");
    if (!w.block_table && w.max_kv_len > prefix_len) return refused(name, "block_table is missing");
    if (!prefix_table && prefix_len > 0) return refused(name, "prefix_table is missing");
    const Plan p = make_plan(*cache, w, prefix_len);
    if (p.bytes && (!workspace || workspace_bytes < (size_t)p.bytes || (uintptr_t)workspace % 16 != 0))
        return refused(name, "workspace is missing, not 16-byte aligned or smaller than gfd_attention_workspace_bytes says");
    const int64_t rows = (int64_t)w.num_tokens * w.num_q_heads;
    float* const part_o = p.bytes ? (float*)workspace : nullptr;
    float* const part_ml = p.bytes ? part_o + p.slots * rows * cache->head_dim : nullptr;
    float* const splits = p.bytes ? part_ml + p.slots * rows * 2 : nullptr;
    const Cache c = make_cache(*cache);
    const float raw = w.scale * c.k_scale;
    // Of a cap past what 32 bits hold of it, the quotients' ends: scores far below it stay as they are, others are +-cap_out.
    const auto held = [](double x) { return (float)std::min(x, 3.4028234e38); };
    const float cap_in = w.softcap > 0.f ? held((double)raw / w.softcap) : -1.f;
    const float cap_out = w.softcap > 0.f ? held((double)w.softcap / raw) : 0.f;
    const bool cap_small = w.softcap >= kCapLeast && w.softcap <= kCapSmall;
    const float factor = (cap_small ? 2.f * w.softcap : raw) * kLog2e, shift = cap_small ? w.softcap * kLog2e : 0.f;
    const Call a{(const uint16_t*)w.q, (uint16_t*)w.out, w.lse, w.q_stride, w.out_stride, w.q_start, w.kv_len,
                 w.block_table, w.table_stride, prefix_table, prefix_len, w.doc_start, w.prefix_end, w.slopes, factor, shift,
                 cap_in, cap_out, cap_small, w.window, w.batch, w.num_tokens, w.max_q_len, w.max_kv_len,
                 w.num_q_heads, cache->num_heads, make_divider((uint32_t)(w.num_q_heads / cache->num_heads)), error_flag,
                 (f32x2*)part_ml, part_o, (int*)splits};
    const hipStream_t st = (hipStream_t)stream;
    if (cache->dtype == GFD_E4M3)
        return launched(name, w.dtype == GFD_BF16 ? launch<Bf16, E4m3>(a, c, p, cache->head_dim, st)
                                                  : launch<Fp16, E4m3>(a, c, p, cache->head_dim, st));
    return launched(name, w.dtype == GFD_BF16 ? launch<Bf16, Bf16>(a, c, p, cache->head_dim, st)
                                              : launch<Fp16, Fp16>(a, c, p, cache->head_dim, st));
}

}  // namespace
}  // namespace kv
}  // namespace gfd

extern "C" int64_t gfd_attention_workspace_bytes(const gfd_kv_cache* cache, const gfd_attention* call, int prefix_len) {
    using namespace gfd::kv;
    if (const char* why = check_call(cache, call, prefix_len)) {
        refused("gfd_attention_workspace_bytes", why);
        return -1;
    }
    return make_plan(*cache, *call, prefix_len).bytes;
}

extern "C" int gfd_paged_attention(const gfd_kv_cache* cache, const gfd_attention* call, void* workspace,
                                   size_t workspace_bytes, int* error_flag, void* stream) {
    return gfd::kv::attention("gfd_paged_attention", cache, call, nullptr, 0, workspace, workspace_bytes, error_flag,
                              stream);
}

extern "C" int gfd_shared_prefix_attention(const gfd_kv_cache* cache, const gfd_attention* call,
                                           const int* prefix_table, int prefix_len, void* workspace,
                                           size_t workspace_bytes, int* error_flag, void* stream) {
    return gfd::kv::attention("gfd_shared_prefix_attention", cache, call, prefix_table, prefix_len, workspace,
                              workspace_bytes, error_flag, stream);
}

#pragma once
// What the kernels of attention over the paged cache share: a call as a kernel
// sees it, the rows and key ranges that a workgroup takes, and partial results
// (HIP sources only).
//
// A query row is a (token, head) pair; the rows of one head of the cache are
// packed token by token, group heads a token, so that keys and values are read
// once for the whole group.  Scores are computed transposed, keys x rows: in the
// matrix instructions' result layout a lane then holds the scores of one row,
// which are, rounded, the very operand that the product with the values takes.
// Maxima, sums and rescaling are a lane's own, but for one exchange a tile.
#include "paged_kv.h"

namespace gfd {
namespace kv {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

struct Call {
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    int64_t q_stride, out_stride;
    const int* q_start;
    const int* kv_len;
    const int* table;
    int64_t table_stride;
    const int* prefix_table;
    int prefix_len;
    const int* doc_start;
    const int* prefix_end;
    const float* slopes;
    // Scores are kept as x, the product of q and the stored key or what a cap makes of it; their exponent of base 2 is
    // x factor + shift.  The factor is positive, so maxima are the same, and one multiply-add under the exponent applies it.
    float factor, shift;
    float cap_in, cap_out;  // of a product x: x cap_in = s / softcap, cap_out softcap's own; cap_in < 0: no cap
    int cap_small;
    int window, batch, num_tokens, max_q_len, max_kv_len, q_heads, kv_heads;
    Divider group;
    int* error;
    // Partial results, [slot][token][head]: maximum and sum, and the unnormalised output.
    f32x2* part_ml;
    float* part_o;
    int* block_splits;  // ranges that an own-keys block has, [block][head of the cache]
};

// One kind of work of a launch: row blocks times key ranges times the cache's heads.
struct Stage {
    int prefix;      // 1: the shared prefix's keys, rows of all tokens; 0: what follows, sequence by sequence
    int blocks;      // row blocks; one per sequence if whole
    int whole;       // a sequence's rows fit a block
    int splits;      // key ranges per block, at most
    int chunk;       // keys per range
    int first_slot;  // of its partial results
    int direct;      // a block with one range writes the result itself
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// A row as its lane needs it; keys count from the stage's first.  t < 0: no row.
struct Row {
    int t, pos, lo, hi;
};

// Tokens of sequence b that the call covers.
struct Sequence {
    int first, q_len, rows_q, kv_len;  // rows_q: at most max_q_len; kv_len as given: positions count from it
    bool cut;
};

__device__ __forceinline__ Sequence sequence(const Call& a, int start, int end, int kv_len) {
    Sequence s;
    s.first = min(max(start, 0), a.num_tokens);
    s.q_len = min(max(end, s.first), a.num_tokens) - s.first;
    s.rows_q = min(s.q_len, a.max_q_len);
    s.kv_len = max(kv_len, 0);
    s.cut = s.q_len > a.max_q_len || kv_len > a.max_kv_len;
    return s;
}
__device__ __forceinline__ Sequence sequence(const Call& a, int b) {
    return sequence(a, a.q_start[b], a.q_start[b + 1], a.kv_len[b]);
}

__device__ __forceinline__ Row make_row(const Call& a, const Sequence& s, int i, bool prefix) {
    Row r;
    r.t = s.first + i;
    r.pos = s.kv_len - s.q_len + i;
    r.lo = a.doc_start ? max(a.doc_start[r.t], 0) : 0;
    if (a.window > 0 && r.pos >= a.window) r.lo = max(r.lo, r.pos - a.window + 1);
    r.hi = min(min(s.kv_len, a.max_kv_len), a.prefix_end ? max(r.pos + 1, a.prefix_end[r.t]) : r.pos + 1);
    if (prefix) {
        r.hi = min(r.hi, a.prefix_len);
    } else {
        r.pos -= a.prefix_len;
        r.lo = max(r.lo - a.prefix_len, 0);
        r.hi -= a.prefix_len;
    }
    if (r.hi <= r.lo) r.lo = r.hi = 0;
    return r;
}

// The rows of a workgroup.
struct Block {
    int b, first_row, rows;  // rows of sequence b (own keys) or of all tokens (prefix)
    Sequence seq;            // own keys
    const int* table;
};

// Where index lies among the blocks of kRows rows that the sequences have, the
// last block of a sequence first: it sees the most keys.  A wave's lanes each
// count a sequence's blocks.
template <int kRows>
__device__ __forceinline__ bool find_block(const Call& a, int index, Block* k) {
    const int lane = (int)threadIdx.x & 63;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int b = min(b0 + lane, a.batch - 1), start = a.q_start[b], end = a.q_start[b + 1], kv_len = a.kv_len[b];
        const int n = b0 + lane < a.batch
                          ? (int)(((int64_t)sequence(a, start, end, kv_len).rows_q * a.group.d + kRows - 1) / kRows)
                          : 0;
        int sum = n;
        for (int off = 1; off < 64; off <<= 1) {
            const int up = __shfl_up(sum, off);
            if (lane >= off) sum += up;
        }
        const int total = __shfl(sum, 63);
        if (index < total) {
            const int at = __ffsll((long long)__ballot(index < sum)) - 1;
            const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
            k->b = b0 + at;
            k->first_row = (of(sum) - 1 - index) * kRows;
            k->seq = sequence(a, of(start), of(end), of(kv_len));
            return true;
        }
        index -= total;
    }
    return false;
}

// The last sequence b with q_start[b] <= t, by every step-th entry in LDS.
constexpr int kSamples = 512;
__device__ __forceinline__ void sample_starts(const Call& a, int* samples, int threads) {
    const int step = (a.batch + kSamples - 1) / kSamples;
    for (int i = (int)threadIdx.x; i <= kSamples; i += threads) samples[i] = a.q_start[min(i * step, a.batch)];
}
__device__ __forceinline__ int sequence_of(const Call& a, const int* samples, int t) {
    const int step = (a.batch + kSamples - 1) / kSamples;
    if (t < samples[0] || t >= samples[kSamples]) return -1;
    int lo = 0, hi = kSamples;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (samples[mid] <= t) lo = mid; else hi = mid;
    }
    lo *= step;
    hi = min(lo + step, a.batch);
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.q_start[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

// What rows [0, rows) of a block see: [lo, hi) by any, [all_lo, all_hi) by every one.
struct Range {
    int lo, hi, all_lo, all_hi;
};

__device__ __forceinline__ void range_add(Range& g, const Row& r) {
    if (r.t < 0) return;
    if (r.hi > r.lo) {
        g.lo = min(g.lo, r.lo);
        g.hi = max(g.hi, r.hi);
    }
    g.all_lo = max(g.all_lo, r.lo);
    g.all_hi = min(g.all_hi, r.hi);
}

__device__ __forceinline__ int lanes_min(int x) {
    for (int off = 32; off; off >>= 1) x = min(x, __shfl_xor(x, off));
    return __builtin_amdgcn_readfirstlane(x);
}

// The rows of block block_index; false: none.
template <int kRows>
__device__ __forceinline__ bool find_rows(const Call& a, const Stage& st, int block_index, Block* k) {
    k->b = 0;
    if (st.prefix) {
        k->first_row = block_index * kRows;
        k->rows = (int)min((int64_t)kRows, (int64_t)a.num_tokens * a.group.d - k->first_row);
        k->table = a.prefix_table;
        return true;
    }
    if (st.whole) {
        k->b = block_index;
        k->first_row = 0;
        k->seq = sequence(a, k->b);
    } else if (!find_block<kRows>(a, block_index, k)) {
        return false;
    }
    k->table = a.table + (int64_t)k->b * a.table_stride;
    k->rows = (int)min((int64_t)kRows, (int64_t)k->seq.rows_q * a.group.d - k->first_row);
    return k->rows > 0;
}

// Row r of a block.
__device__ __forceinline__ Row row_of(const Call& a, const Stage& st, const Block& k, const int* samples, int r) {
    Row x{-1, 0, 0, 0};
    if (r >= k.rows) return x;
    const int i = (int)a.group.div((uint32_t)(k.first_row + r));
    if (!st.prefix) {
        if (k.seq.cut && a.error) atomicOr(a.error, GFD_KV_ERR_LENGTH);
        return make_row(a, k.seq, i, false);
    }
    const int b = sequence_of(a, samples, i);
    if (b < 0) return x;
    const Sequence s = sequence(a, b);
    if (i - s.first >= s.rows_q || i < s.first) return x;
    return make_row(a, s, i - s.first, true);
}

__device__ __forceinline__ int head_of(const Call& a, const Block& k, int r, int kv_head) {
    const uint32_t n = (uint32_t)(k.first_row + r);
    return kv_head * (int)a.group.d + (int)(n - a.group.div(n) * a.group.d);
}

// Byte offset of a key, -1 where its page is none of the cache's.
__device__ __forceinline__ int64_t key_offset(const Cache& c, const int* table, int n, int64_t head, int* error) {
    const uint32_t page = c.page.div((uint32_t)n);
    const int id = table[page];
    if (id < 0 || id >= c.num_pages) {
        if (error) atomicOr(error, GFD_KV_ERR_PAGE);
        return -1;
    }
    return id * c.page_stride + (int64_t)((uint32_t)n - page * c.page.d) * c.slot_stride + head;
}

__device__ __forceinline__ int64_t slot_of(const Call& a, int slot, int t, int h) {
    return ((int64_t)slot * a.num_tokens + t) * a.q_heads + h;
}

__device__ __forceinline__ float max_f32(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// The maximum, or the sum, over the lanes that share a row.
__device__ __forceinline__ float across32_max(float x) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max_f32(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float across32_sum(float x) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
__device__ __forceinline__ float across16_max(float x) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return across32_max(max_f32(__uint_as_float(p[0]), __uint_as_float(p[1])));
}
__device__ __forceinline__ float across16_sum(float x) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return across32_sum(__uint_as_float(p[0]) + __uint_as_float(p[1]));
}

// softcap tanh(s / softcap) in units of the products' sums x, y = x cap_in.  Three forms:
// far, for caps of kCapLeast to kCapSmall: cap - 2 cap / (e^2y + 1), kept as -1 / (e^2y + 1), off by 4 2^-24 of the cap: 2^-16
//   of a score's unit at most, little against the weights' rounding (2^-12, 2^-9);
// near, where |y| <= kCapNear for all of a tile's scores: x (1 + z P(z)), z = y^2, off by 2 2^-24 of itself however large
//   the cap (P: a least-maximum fit of tanh(y) / y there, off by 0.6 2^-24);
// any: both, and a choice.
// 8192 packed tokens, whose scores have a spread of 1.5: without a cap 174 us, far 211, near 214, any 290.
constexpr float kCapNear = 0.75f, kCapSmall = 64.f, kCapLeast = 0x1p-20f;
__device__ __forceinline__ float capped_near(float x, float cap_in) {
    const float y = x * cap_in, z = y * y;
    float p = -4.769478459e-03f;
    p = __builtin_fmaf(p, z, 1.966489665e-02f);
    p = __builtin_fmaf(p, z, -5.339024961e-02f);
    p = __builtin_fmaf(p, z, 1.332652122e-01f);
    p = __builtin_fmaf(p, z, -3.333306909e-01f);
    return __builtin_fmaf(x * z, p, x);
}
__device__ __forceinline__ float capped_far(float x, float cap_in) {
    return __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(x * (cap_in * (2.f * kLog2e))));
}
__device__ __forceinline__ float capped_any(float x, float cap_in, float cap_out) {
    const float near = capped_near(x, cap_in), far = __builtin_fmaf(capped_far(x, cap_in), 2.f * cap_out, cap_out);
    return fabsf(x * cap_in) <= kCapNear ? near : far;
}
// all(f): every score becomes f(score); most(): the largest magnitude among a lane's, NaN if one is.
template <typename M, typename F>
__device__ __forceinline__ void cap_scores(const Call& a, M most, F all) {
    // The forms are not to share what they have in common: a tile's worth of it would be held.
    const auto apart = [](float x) {
        asm("" : "+v"(x));
        return x;
    };
    if (a.cap_small) all([&](float x) { return capped_far(x, a.cap_in); });
    else if (__any(!(most() * a.cap_in <= kCapNear))) all([&](float x) { return capped_any(apart(x), a.cap_in, a.cap_out); });
    else all([&](float x) { return capped_near(apart(x), a.cap_in); });
}

// Matrix instructions by element type, and tests on packed pairs.
template <typename T>
struct Mma;
template <>
struct Mma<Bf16> {
    // A weight is 2^kRaise e^(s - m), m the running maximum, which a score may pass by 2^kSlack (in kernels that
    // let it): 16 bits of this type hold weights of any size to the same relative step.
    static constexpr float kRaise = 0.f, kSlack = 8.f;
    static constexpr uint32_t kNear = 0x00800080u;  // added to a magnitude: bit 15 is set from infinity on
    static __device__ __forceinline__ f32x4 m16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 m32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
    // Two 8-bit floats (bits 0..15 of w, or 16..31): exact.
    static __device__ __forceinline__ uint32_t widen_lo(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    }
    static __device__ __forceinline__ uint32_t widen_hi(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
    }
};
template <>
struct Mma<Fp16> {
    // This type holds 2^-14 to 2^16 in full, below in steps of 2^-24.  Weights use its upper end, so that those of
    // many keys far below a maximum are not lost: down to 2^-29 of the largest they are rounded relatively, and what a
    // key loses below that is 2^-40 of the largest (2^-28 and 2^-39 where scores may pass the maximum by 2^1).
    // The small slack costs a few rescalings more: 7 ragged prompts of 64 dims 61 us, with 2^8 and no offset 59.5.
    static constexpr float kRaise = 15.f, kSlack = 1.f;
    static constexpr uint32_t kNear = 0x04000400u;
    static __device__ __forceinline__ f32x4 m16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
    static __device__ __forceinline__ f32x16 m32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
    static __device__ __forceinline__ uint32_t widen_lo(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    }
    static __device__ __forceinline__ uint32_t widen_hi(uint32_t w) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    }
};

// Bits 15 and 31 say which of a pair's values are infinite or NaN.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    return ((w & 0x7FFF7FFFu) + Mma<T>::kNear) & 0x80008000u;
}
// A pair with infinities and NaN made zero.
template <typename T>
__device__ __forceinline__ uint32_t only_finite(uint32_t w) {
    const uint32_t bad = not_finite<T>(w) >> 15;
    return w & ~(bad * 0xFFFFu);
}

// Few rows (attend_rows.h): a workgroup has the offsets of so many keys at a time.
constexpr int kRowsPiece = 1024;
constexpr int kRowsShort = 128;  // with one wave
template <typename T, typename S>
int launch_rows(const Call& a, const Cache& c, const Stage& prefix, const Stage& own, int dim, bool wide, int waves,
                hipStream_t st);
// Many rows (attend_tiles.h).
template <typename T, typename S>
int launch_tiles(const Call& a, const Cache& c, const Stage& prefix, const Stage& own, int dim, int waves,
                 hipStream_t st);

// A prefix of many rows and few rows that follow (attend_both.h).
template <typename T, typename S>
int launch_both(const Call& a, const Cache& c, const Stage& prefix, const Stage& own, int dim, bool wide,
                hipStream_t st);

}  // namespace kv
}  // namespace gfd

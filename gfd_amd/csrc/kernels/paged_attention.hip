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
#include <cstdio>

#include "attend_rows.h"
#include "capi_error.h"
#include "gfd_capi.h"
#include "paged_attention.h"

namespace gfd {
namespace kv {
namespace {

constexpr int kJoinBlock = 256, kJoinRows = 16;

// A workgroup joins kJoinRows rows of an own-keys block, a wave per row: a lane
// weighs one range of 64, then holds D / 64 dims.  Reads what the ranges
// left once; bound by the launch's latency for small batches.
template <typename T, int D, int kRows>
__global__ __launch_bounds__(kJoinBlock) void join_kernel(Call a, Cache c, Stage prefix, Stage own) {
    constexpr int kDims = D / 64, kWaves = kJoinBlock / 64;
    typedef float Dims __attribute__((ext_vector_type(kDims)));
    __shared__ int lo[kWaves], hi[kWaves];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int kv_head = (int)blockIdx.x % a.kv_heads;
    Block k;
    if (!find_rows<kRows>(a, own, (int)blockIdx.x / a.kv_heads, &k)) return;
    Range g{0x7FFFFFFF, 0, 0, 0};
    if (tid < kRows) range_add(g, row_of(a, own, k, nullptr, tid));
    g.lo = lanes_min(g.lo);
    g.hi = -lanes_min(-g.hi);
    if (lane == 0) lo[wave] = g.lo, hi[wave] = g.hi;
    __syncthreads();
    for (int i = 0; i < kWaves; i++) g.lo = min(g.lo, lo[i]), g.hi = max(g.hi, hi[i]);
    if (g.hi == 0) g.lo = 0;
    const int splits = max(1, (g.hi - g.lo + own.chunk - 1) / own.chunk), slots = own.first_slot + splits;
    if (own.direct && splits == 1) return;

    const int first = (int)blockIdx.y * kJoinRows;
    for (int r = first + wave; r < min(first + kJoinRows, k.rows); r += kWaves) {
        const int t = row_of(a, own, k, nullptr, r).t, h = head_of(a, k, r, kv_head);
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
            for (int s = 0; s < n; s += 4) {  // lanes past the last range weigh nothing
                Dims x[4];
                float ws[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    ws[j] = __shfl(w, s + j);
                    x[j] = 0.f;
                    if (__shfl(l, s + j) != 0.f) x[j] = *(const Dims*)(from + (s + j) * step);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) o += ws[j] * x[j];
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

// The sequence that token t belongs to: the last b with q_start[b] <= t; -1 if none.
__device__ __forceinline__ int simple_sequence_of(const Call& a, int t) {
    int lo = 0, hi = a.batch;  // q_start[lo] <= t < q_start[hi]
    if (t < a.q_start[0] || t >= a.q_start[a.batch]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.q_start[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

struct Seen {
    int pos, lo, hi;
};

__device__ __forceinline__ Seen visible(const Call& a, int t, int i, int q_len, int kv_len) {
    Seen s;
    s.pos = kv_len - q_len + i;
    s.lo = a.doc_start ? max(a.doc_start[t], 0) : 0;
    if (a.window > 0) s.lo = max(s.lo, s.pos - a.window + 1);
    s.hi = min(kv_len, a.prefix_end ? max(s.pos + 1, a.prefix_end[t]) : s.pos + 1);
    return s;
}

template <typename T>
__device__ __forceinline__ float load_one(const uint8_t* p, int i) { return T::unpack(((const uint16_t*)p)[i])[0]; }
template <>
__device__ __forceinline__ float load_one<E4m3>(const uint8_t* p, int i) {
    return __builtin_amdgcn_cvt_f32_fp8((int)p[i], 0);
}

// One wave per row: a lane scores one key of 64, then holds dim lane + 64 k of the sum.
template <typename T, typename S, int D>
__global__ __launch_bounds__(64) void attend_kernel(Call a, Cache c) {
    const int t = (int)blockIdx.x, h = (int)blockIdx.y, lane = (int)threadIdx.x;
    const int b = simple_sequence_of(a, t);
    if (b < 0) return;
    const int first = max(a.q_start[b], 0), q_len = a.q_start[b + 1] - first;
    int kv_len = a.kv_len[b];
    if (kv_len > a.max_kv_len || q_len > a.max_q_len) {
        if (lane == 0 && a.error) atomicOr(a.error, GFD_KV_ERR_LENGTH);
        kv_len = min(kv_len, a.max_kv_len);
    }
    if (t - first >= a.max_q_len) return;
    const Seen s = visible(a, t, t - first, q_len, kv_len);
    const int kv_head = h / a.group.d;
    __shared__ float q[D];
    for (int d = lane; d < D; d += 64) q[d] = load_one<T>((const uint8_t*)(a.q + t * a.q_stride + (int64_t)h * D), d);
    __syncthreads();
    float m = -INFINITY, sum = 0.f, o[D / 64] = {};
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    for (int j0 = s.lo; j0 < s.hi; j0 += 64) {
        const int j = j0 + lane;
        float x = -INFINITY;
        int64_t at = -1;
        if (j < s.hi) {
            const bool shared = j < a.prefix_len;
            const uint32_t n = (uint32_t)(shared ? j : j - a.prefix_len), page = c.page.div(n);
            const int id = shared ? a.prefix_table[page] : a.table[b * a.table_stride + page];
            if (id < 0 || id >= c.num_pages) {
                if (a.error) atomicOr(a.error, GFD_KV_ERR_PAGE);
            } else {
                at = id * c.page_stride + (int64_t)(n - page * c.page.d) * c.slot_stride + kv_head * c.head_stride;
                float dot = 0.f;
                for (int d = 0; d < D; d++) dot += q[d] * load_one<S>(c.k + at, d);
                x = dot * (a.scale * c.k_scale);
                if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
                if (a.slopes) x -= slope * fabsf((float)(s.pos - j));
            }
        }
        float top = x;
        for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
        // fmaxf leaves NaN out; a NaN score reaches the sum through its own exp.
        const float next = fmaxf(m, top), base = next == -INFINITY ? 0.f : next;
        const float p = at >= 0 ? expf(x - base) : 0.f, keep = expf(m - base);
        float part = p;
        for (int off = 32; off; off >>= 1) part += __shfl_xor(part, off);
        sum = sum * keep + part;
        m = next;
        for (int k = 0; k < D / 64; k++) o[k] *= keep;
        for (int n = 0; n < 64; n++) {
            const int64_t from = __shfl(at, n);
            const float w = __shfl(p, n);
            if (from < 0) continue;
            for (int k = 0; k < D / 64; k++) o[k] += w * load_one<S>(c.v + from, lane + 64 * k);
        }
    }
    uint16_t* out = a.out + t * a.out_stride + (int64_t)h * D;
    for (int k = 0; k < D / 64; k++)
        out[lane + 64 * k] = (uint16_t)T::pack(sum == 0.f ? 0.f : o[k] * (c.v_scale / sum), 0.f);
    if (a.lse && lane == 0) a.lse[(int64_t)t * a.q_heads + h] = sum == 0.f ? -INFINITY : m + logf(sum);
}

int refuse(const char* name, const char* why) {
    static thread_local char text[192];
    snprintf(text, sizeof(text), "%s: %s", name, why);
    gfd_internal_set_error(text);
    return (int)hipErrorInvalidValue;
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
    if (w.window < 0) return "negative window";
    if ((w.q_stride | w.out_stride) % 8 != 0 || ((uintptr_t)w.q | (uintptr_t)w.out) % 16 != 0)
        return "rows' pointers or strides are not multiples of 16 bytes";
    const int64_t pages = ((int64_t)std::max(w.max_kv_len - prefix_len, 0) + cache->page_size - 1) / cache->page_size;
    if (w.table_stride < pages) return "block_table's rows are shorter than max_kv_len needs";
    return nullptr;
}

// How a call is cut into row blocks and key ranges.
struct Plan {
    bool simple;      // more rows than 32 share keys: the kernel of one wave per row
    int rows;         // of an own-keys block
    Stage prefix, own;
    int slots;        // partial results per row
    int64_t bytes;    // of workspace
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Workgroups that fill the card: below kFill a block's keys are split, into ranges of
// at least kMinChunk keys (a tile per wave).  Ranges also end at kRowsMaxChunk, so that
// sequences of very different lengths are evenly spread.
constexpr int kFill = 2048, kMinChunk = 128;

void split(Stage* st, int64_t items, int64_t keys) {
    const int64_t want = ceil_div(keys * items, kFill);
    st->chunk = (int)std::min<int64_t>(kRowsMaxChunk, std::max<int64_t>(kMinChunk, ceil_div(want, kMinChunk) * kMinChunk));
    st->splits = (int)std::max<int64_t>(1, ceil_div(keys, st->chunk));
}

Plan make_plan(const gfd_kv_cache& cache, const gfd_attention& w, int prefix_len) {
    Plan p{};
    const int64_t group = w.num_q_heads / cache.num_heads, heads = cache.num_heads;
    const int64_t seq_rows = std::min<int64_t>(w.max_q_len, w.num_tokens) * group;
    const int64_t all_rows = w.num_tokens * group;
    p.simple = seq_rows > 32 || (prefix_len && all_rows > 32);
    p.rows = seq_rows <= 16 && (!prefix_len || all_rows <= 16) ? 16 : 32;
    // Keys that a block can see: with a window, those of its tokens' windows (a prefix mask only adds later keys).
    int64_t keys = std::max(w.max_kv_len - prefix_len, 0);
    if (w.window && !w.prefix_end) keys = std::min<int64_t>(keys, (int64_t)w.window + w.max_q_len);
    p.own.blocks = w.batch;
    p.own.whole = 1;
    split(&p.own, p.own.blocks * heads, keys);
    if (prefix_len) {
        p.prefix.prefix = 1;
        p.prefix.blocks = (int)ceil_div(all_rows, p.rows);
        split(&p.prefix, p.prefix.blocks * heads, prefix_len);
        p.own.first_slot = p.prefix.splits;
    } else {
        p.own.direct = 1;
    }
    p.slots = p.own.first_slot + p.own.splits;
    if (p.slots > 1 && !p.simple) p.bytes = (int64_t)p.slots * w.num_tokens * w.num_q_heads * (cache.head_dim + 2) * 4;
    return p;
}

template <typename T, int D>
int launch_join(const Call& a, const Cache& c, const Plan& p, hipStream_t st) {
    const dim3 grid((unsigned)(p.own.blocks * a.kv_heads), (unsigned)ceil_div(p.rows, kJoinRows));
    if (p.rows == 16)
        hipLaunchKernelGGL((join_kernel<T, D, 16>), grid, dim3(kJoinBlock), 0, st, a, c, p.prefix, p.own);
    else
        hipLaunchKernelGGL((join_kernel<T, D, 32>), grid, dim3(kJoinBlock), 0, st, a, c, p.prefix, p.own);
    return (int)hipGetLastError();
}

template <typename T, typename S>
int launch(const Call& a, const Cache& c, const Plan& p, int dim, hipStream_t st) {
    const dim3 grid((unsigned)a.num_tokens, (unsigned)a.q_heads);
    if (p.simple) {
    if (dim == 64) hipLaunchKernelGGL((attend_kernel<T, S, 64>), grid, dim3(64), 0, st, a, c);
    if (dim == 128) hipLaunchKernelGGL((attend_kernel<T, S, 128>), grid, dim3(64), 0, st, a, c);
    if (dim == 256) hipLaunchKernelGGL((attend_kernel<T, S, 256>), grid, dim3(64), 0, st, a, c);
    return (int)hipGetLastError();
    }
    if (const int rc = launch_rows<T, S>(a, c, p.prefix, p.own, dim, p.rows == 32, st)) return rc;
    if (p.slots == 1) return 0;
    return dim == 64 ? launch_join<T, 64>(a, c, p, st) : dim == 128 ? launch_join<T, 128>(a, c, p, st)
                                                                   : launch_join<T, 256>(a, c, p, st);
}

int attention(const char* name, const gfd_kv_cache* cache, const gfd_attention* call, const int* prefix_table,
              int prefix_len, void* workspace, size_t workspace_bytes, int* error_flag, void* stream) {
    if (const char* why = check_call(cache, call, prefix_len)) return refuse(name, why);
    const gfd_attention& w = *call;
    if (w.batch == 0 || w.num_tokens == 0 || w.max_q_len == 0) return 0;
    if (!w.q || !w.out || !w.q_start || !w.kv_len) return refuse(name, "q, out, q_start or kv_len is missing");
    if (!w.block_table && w.max_kv_len > prefix_len) return refuse(name, "block_table is missing");
    if (!prefix_table && prefix_len > 0) return refuse(name, "prefix_table is missing");
    const Plan p = make_plan(*cache, w, prefix_len);
    if (p.bytes && (!workspace || workspace_bytes < (size_t)p.bytes || (uintptr_t)workspace % 16 != 0))
        return refuse(name, "workspace is missing, not 16-byte aligned or smaller than gfd_attention_workspace_bytes says");
    const int64_t rows = (int64_t)w.num_tokens * w.num_q_heads;
    float* const part_o = (float*)workspace;
    const Call a{(const uint16_t*)w.q, (uint16_t*)w.out, w.lse, w.q_stride, w.out_stride, w.q_start, w.kv_len,
                 w.block_table, w.table_stride, prefix_table, prefix_len, w.doc_start, w.prefix_end, w.slopes, w.scale,
                 w.softcap, w.window, w.batch, w.num_tokens, w.max_q_len, w.max_kv_len, w.num_q_heads,
                 cache->num_heads, make_divider((uint32_t)(w.num_q_heads / cache->num_heads)), error_flag,
                 (f32x2*)(part_o + p.slots * rows * cache->head_dim), part_o};
    const Cache c = make_cache(*cache);
    const hipStream_t st = (hipStream_t)stream;
    if (cache->dtype == GFD_E4M3)
        return w.dtype == GFD_BF16 ? launch<Bf16, E4m3>(a, c, p, cache->head_dim, st)
                                   : launch<Fp16, E4m3>(a, c, p, cache->head_dim, st);
    return w.dtype == GFD_BF16 ? launch<Bf16, Bf16>(a, c, p, cache->head_dim, st)
                               : launch<Fp16, Fp16>(a, c, p, cache->head_dim, st);
}

}  // namespace
}  // namespace kv
}  // namespace gfd

extern "C" int64_t gfd_attention_workspace_bytes(const gfd_kv_cache* cache, const gfd_attention* call, int prefix_len) {
    using namespace gfd::kv;
    if (const char* why = check_call(cache, call, prefix_len)) {
        refuse("gfd_attention_workspace_bytes", why);
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

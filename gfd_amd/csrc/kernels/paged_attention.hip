// Attention over the paged cache (gfx950).
//
// Per query row (token, head) with score s_j over its visible keys j:
// out = sum exp(s_j - m) v_j / sum exp(s_j - m), lse = m + log of that sum,
// with the running maximum m and sums in 32 bits.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>

#include "capi_error.h"
#include "gfd_capi.h"
#include "paged_kv.h"

namespace gfd {
namespace kv {
namespace {

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
    float scale, softcap;
    int window, batch, num_tokens, max_q_len, max_kv_len, q_heads, kv_heads, group;
    int* error;
};

// The sequence that token t belongs to: the last b with q_start[b] <= t; -1 if none.
__device__ __forceinline__ int sequence_of(const Call& a, int t) {
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
    const int b = sequence_of(a, t);
    if (b < 0) return;
    const int first = max(a.q_start[b], 0), q_len = a.q_start[b + 1] - first;
    int kv_len = a.kv_len[b];
    if (kv_len > a.max_kv_len || q_len > a.max_q_len) {
        if (lane == 0 && a.error) atomicOr(a.error, GFD_KV_ERR_LENGTH);
        kv_len = min(kv_len, a.max_kv_len);
    }
    if (t - first >= a.max_q_len) return;
    const Seen s = visible(a, t, t - first, q_len, kv_len);
    const int kv_head = h / a.group;
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
    const int64_t pages = ((int64_t)max(w.max_kv_len - prefix_len, 0) + cache->page_size - 1) / cache->page_size;
    if (w.table_stride < pages) return "block_table's rows are shorter than max_kv_len needs";
    return nullptr;
}

template <typename T, typename S>
int launch(const Call& a, const Cache& c, int dim, hipStream_t st) {
    const dim3 grid((unsigned)a.num_tokens, (unsigned)a.q_heads);
    if (dim == 64) hipLaunchKernelGGL((attend_kernel<T, S, 64>), grid, dim3(64), 0, st, a, c);
    if (dim == 128) hipLaunchKernelGGL((attend_kernel<T, S, 128>), grid, dim3(64), 0, st, a, c);
    if (dim == 256) hipLaunchKernelGGL((attend_kernel<T, S, 256>), grid, dim3(64), 0, st, a, c);
    return (int)hipGetLastError();
}

int attention(const char* name, const gfd_kv_cache* cache, const gfd_attention* call, const int* prefix_table,
              int prefix_len, void* workspace, size_t workspace_bytes, int* error_flag, void* stream) {
    if (const char* why = check_call(cache, call, prefix_len)) return refuse(name, why);
    const gfd_attention& w = *call;
    if (w.batch == 0 || w.num_tokens == 0 || w.max_q_len == 0) return 0;
    if (!w.q || !w.out || !w.q_start || !w.kv_len) return refuse(name, "q, out, q_start or kv_len is missing");
    if (!w.block_table && w.max_kv_len > prefix_len) return refuse(name, "block_table is missing");
    if (!prefix_table && prefix_len > 0) return refuse(name, "prefix_table is missing");
    const Call a{(const uint16_t*)w.q, (uint16_t*)w.out, w.lse, w.q_stride, w.out_stride, w.q_start, w.kv_len,
                 w.block_table, w.table_stride, prefix_table, prefix_len, w.doc_start, w.prefix_end, w.slopes, w.scale,
                 w.softcap, w.window, w.batch, w.num_tokens, w.max_q_len, w.max_kv_len, w.num_q_heads,
                 cache->num_heads, w.num_q_heads / cache->num_heads, error_flag};
    const Cache c = make_cache(*cache);
    const hipStream_t st = (hipStream_t)stream;
    if (cache->dtype == GFD_E4M3)
        return w.dtype == GFD_BF16 ? launch<Bf16, E4m3>(a, c, cache->head_dim, st)
                                   : launch<Fp16, E4m3>(a, c, cache->head_dim, st);
    return w.dtype == GFD_BF16 ? launch<Bf16, Bf16>(a, c, cache->head_dim, st)
                               : launch<Fp16, Fp16>(a, c, cache->head_dim, st);
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
    return 0;
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

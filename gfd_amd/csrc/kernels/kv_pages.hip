// The paged cache's pages (gfx950): copied, shared by sequences that go on from
// others, let go of, and brought together.
//
// refs[p] counts the table entries that name page p.  Which pages a call takes is
// a rank among the free (or used) pages in their order, so a call's result is a function of its
// inputs: a first launch counts each chunk of pages, a second one adds the counts up and
// gives every page its rank.  Nothing waits for another workgroup and no atomic's order is
// used; refs only change by sums and by stores to pages that nothing else names.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gfd_capi.h"
#include "paged_kv.h"

namespace gfd {
namespace kv {
namespace {

constexpr int kBlock = 256, kWaves = kBlock / 64;
// Pages a workgroup ranks: kFew a thread in small pools, where one chain of loads after the other counts (256 sequences
// forked in a pool of 12000 pages: 4.5 us, with 4 a thread 11), kMany in large ones, as every workgroup adds up all counts.
constexpr int kFew = 1, kMany = 16, kSmallPool = 1 << 16;
constexpr int kSamples = 1024;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

__device__ __forceinline__ void report(int* error, int bit) {
    if (error) atomicOr(error, bit);
}

// The sum of what the threads before this one have; *total of all.  part: [kWaves].
template <typename N>
__device__ __forceinline__ N before(N x, N* part, N* total) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    N sum = x;
    for (int off = 1; off < 64; off <<= 1) {
        const N up = __shfl_up(sum, off);
        if (lane >= off) sum += up;
    }
    __syncthreads();  // part may still be read
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    N base = 0, all = 0;
    for (int i = 0; i < kWaves; i++) {
        if (i < wave) base += part[i];
        all += part[i];
    }
    *total = all;
    return base + sum - x;
}

struct Pool {
    const int* refs;
    int num_pages, chunks;
    Divider page;
};

// A thread's pages of a chunk; what lies past the last page is `past`.
template <int kPer>
struct Refs {
    int page, x[kPer];
    __device__ __forceinline__ Refs(const Pool& pool, int chunk, int past) {
        page = (chunk * kBlock + (int)threadIdx.x) * kPer;
#pragma unroll
        for (int i = 0; i < kPer; i++) x[i] = page + i < pool.num_pages ? pool.refs[page + i] : past;
    }
    __device__ __forceinline__ int free_pages() const {
        int n = 0;
#pragma unroll
        for (int i = 0; i < kPer; i++) n += x[i] == 0;
        return n;
    }
};

// What the chunks before this one count together; *total of all.
__device__ __forceinline__ int chunks_before(const int* counts, int chunks, int chunk, int* part, int* total) {
    int mine = 0, all = 0;
    for (int i = (int)threadIdx.x; i < chunks; i += kBlock) {
        const int n = counts[i];
        all += n;
        mine += i < chunk ? n : 0;
    }
    int sum;
    before(mine, part, &sum);
    const int base = sum;
    before(all, part, total);
    return base;
}

__device__ __forceinline__ int pages_of(const Divider& page, int tokens) {
    return (int)page.div((uint32_t)tokens + page.d - 1);
}

// ------------------------------------------------------------------ fork

struct Fork {
    Pool pool;
    int* refs;
    const int* table;
    int* child_table;
    int64_t table_stride, child_stride;
    int rows, child_rows;
    const int* parent;
    const int* child;
    const int* len;
    const int* capacity;
    gfd_kv_page_copy* copies;
    int num;
    int* error;
    int* counts;  // free pages, [chunk]
    int* first;   // needed pages before item i, [num + 1]
};

// Item i: entries [0, shared) are the parent's, [from, end) new pages; part: tokens on a page that is copied.
struct Item {
    int parent, child, shared, from, end, part;
};

constexpr int kMostTokens = 1 << 30;

__device__ __forceinline__ Item item_of(const Fork& f, int i, int* error) {
    Item x{f.parent[i], f.child[i], 0, 0, 0, 0};
    if (x.child < 0) return x;
    const int len = f.len[i], room = f.capacity ? max(f.capacity[i], len) : len;
    const bool fits = x.child < f.child_rows && x.parent >= -1 && x.parent < f.rows && len >= 0 && room <= kMostTokens;
    const int held = fits ? pages_of(f.pool.page, len) : 0, end = fits ? pages_of(f.pool.page, room) : 0;
    if (!fits || end > f.child_stride || (x.parent >= 0 && held > f.table_stride)) {
        report(error, GFD_KV_ERR_ROW);
        x.child = -1;
        return x;
    }
    x.from = held;
    x.end = end;
    if (x.parent >= 0) {
        x.shared = (int)f.pool.page.div((uint32_t)len);
        x.part = len - x.shared * (int)f.pool.page.d;
        x.from = x.shared;
    }
    return x;
}

// A workgroup counts a chunk's free pages; the last one the pages that the items before each need, kBlock items at a time.
// That is what a fork of many items takes: 256 of them 3 us, 3000 12, 65536 0.22 ms, 2^20 5.5 ms (fork_kernel 1.8 ms).
template <int kPer>
__global__ __launch_bounds__(kBlock) void fork_count_kernel(Fork f) {
    __shared__ int part[kWaves];
    __shared__ long long part64[kWaves];
    if ((int)blockIdx.x < f.pool.chunks) {
        const Refs<kPer> r(f.pool, (int)blockIdx.x, 1);
        int total;
        before(r.free_pages(), part, &total);
        if (threadIdx.x == 0) f.counts[blockIdx.x] = total;
        return;
    }
    // Ranks past every page are all the same: sums are held at kMostTokens.
    long long base = 0, total;
    for (int i0 = 0; i0 < f.num; i0 += kBlock) {
        const int i = i0 + (int)threadIdx.x;
        int need = 0;
        if (i < f.num) {
            const Item x = item_of(f, i, f.error);
            need = x.child < 0 ? 0 : x.end - x.from;
        }
        const long long at = base + before((long long)need, part64, &total);
        if (i < f.num) f.first[i] = (int)min(at, (long long)kMostTokens);
        base += total;
    }
    if (threadIdx.x == 0) f.first[f.num] = (int)min(base, (long long)kMostTokens);
}

// Gives a chunk's free pages to the items whose needs have their ranks.
template <int kPer>
__device__ __forceinline__ void give_pages(const Fork& f, int chunk, int* part, int* samples) {
    const Refs<kPer> r(f.pool, chunk, 1);
    const int needed = f.first[f.num], step = (f.num + kSamples - 1) / kSamples;
    int free_pages, total;
    const int base = chunks_before(f.counts, f.pool.chunks, chunk, part, &free_pages);
    if (base >= needed) return;
    for (int i = (int)threadIdx.x; i <= kSamples && i * step < f.num + step; i += kBlock) samples[i] = f.first[min(i * step, f.num)];
    int rank = base + before(r.free_pages(), part, &total);  // its barriers stand behind the samples too
#pragma unroll
    for (int n = 0; n < kPer; n++) {
        if (r.x[n] != 0) continue;
        if (rank >= needed) return;
        // The item with first[i] <= rank < first[i + 1].
        int lo = 0, hi = (f.num + step - 1) / step;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (samples[mid] <= rank) lo = mid; else hi = mid;
        }
        int before_item = samples[lo];
        lo *= step;
        hi = min(lo + step, f.num);
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2, at = f.first[mid];
            if (at <= rank) lo = mid, before_item = at; else hi = mid;
        }
        const Item it = item_of(f, lo, nullptr);
        const int j = it.from + (rank - before_item), page = r.page + n;
        f.child_table[it.child * f.child_stride + j] = page;
        f.refs[page] = 1;
        if (it.part && j == it.from) {
            const int src = f.table[it.parent * f.table_stride + j];
            const bool there = src >= 0 && src < f.pool.num_pages;
            if (!there) report(f.error, GFD_KV_ERR_PAGE);
            f.copies[lo] = there ? gfd_kv_page_copy{src, page, it.part, 0} : gfd_kv_page_copy{-1, -1, 0, 0};
        }
        rank++;
    }
}

// An item's shared entries, and what no free page was left for.
__device__ __forceinline__ void share_pages(const Fork& f, int i, int turn, int turns, int* part) {
    const Item x = item_of(f, i, nullptr);
    const bool first_turn = turn == 0 && threadIdx.x == 0;
    if (x.child < 0) {
        if (first_turn) f.copies[i] = gfd_kv_page_copy{-1, -1, 0, 0};
        return;
    }
    const int first = f.first[i];
    int free_pages;
    chunks_before(f.counts, f.pool.chunks, 0, part, &free_pages);
    int* const to = f.child_table + x.child * f.child_stride;
    for (int j = turn * kBlock + (int)threadIdx.x; j < x.shared; j += turns * kBlock) {
        int id = f.table[x.parent * f.table_stride + j];
        if (id >= 0 && id < f.pool.num_pages) {
            atomicAdd(f.refs + id, 1);
        } else {
            report(f.error, GFD_KV_ERR_PAGE);
            id = -1;
        }
        to[j] = id;
    }
    if (first_turn && (x.part == 0 || first >= free_pages)) f.copies[i] = gfd_kv_page_copy{-1, -1, 0, 0};
    const int lost = x.from + max(free_pages - first, 0);
    if (lost >= x.end) return;
    if (first_turn) report(f.error, GFD_KV_ERR_FULL);
    for (int j = lost + turn * kBlock + (int)threadIdx.x; j < x.end; j += turns * kBlock) to[j] = -1;
}

// A few launches' latency for a few sequences; the tables' bytes for many.
template <int kPer>
__global__ __launch_bounds__(kBlock) void fork_kernel(Fork f, int turns) {
    __shared__ int part[kWaves], samples[kSamples + 1];
    const int id = (int)blockIdx.x - f.pool.chunks;
    if (id < 0) give_pages<kPer>(f, (int)blockIdx.x, part, samples);
    else share_pages(f, id / turns, id % turns, turns, part);
}

// ------------------------------------------------------------------ free

struct Free {
    int* refs;
    Divider page;
    int num_pages;
    const int* table;
    int64_t table_stride;
    int rows;
    const int* row;
    const int* len;
    int* error;
};

__global__ __launch_bounds__(kBlock) void free_kernel(Free f, int turns) {
    const int i = (int)blockIdx.x / turns, turn = (int)blockIdx.x % turns;
    const int row = f.row[i], len = f.len[i];
    if (row < 0) return;
    const int pages = len >= 0 && len <= kMostTokens ? pages_of(f.page, len) : -1;
    if (row >= f.rows || pages < 0 || pages > f.table_stride) {
        if (turn == 0 && threadIdx.x == 0) report(f.error, GFD_KV_ERR_ROW);
        return;
    }
    for (int j = turn * kBlock + (int)threadIdx.x; j < pages; j += turns * kBlock) {
        const int id = f.table[row * f.table_stride + j];
        if (id < 0) continue;
        if (id >= f.num_pages) {
            report(f.error, GFD_KV_ERR_PAGE);
        } else if (atomicSub(f.refs + id, 1) <= 0) {
            atomicAdd(f.refs + id, 1);  // whoever else takes one too many puts it back as well
            report(f.error, GFD_KV_ERR_REFS);
        }
    }
}

// --------------------------------------------------------------- compact

struct Compact {
    Pool pool;
    int* new_refs;
    const int* table;
    int* new_table;
    int64_t table_stride, new_stride;
    const int* len;
    int rows;
    int* page_map;
    gfd_kv_page_copy* copies;
    int* num_copies;
    int* error;
    int* counts;     // used pages, [chunk]
    int* where;      // [num_pages]: the page's new place, -1 for a free one, -2 - i for the one that copy i moves
    int* src;        // [num_pages / 2]: of copy i
    int* src_refs;
    int* dst;
};

template <int kPer>
__global__ __launch_bounds__(kBlock) void compact_count_kernel(Compact f) {
    __shared__ int part[kWaves];
    int total;
    const Refs<kPer> r(f.pool, (int)blockIdx.x, 0);
    before(kPer - r.free_pages(), part, &total);
    if (threadIdx.x == 0) f.counts[blockIdx.x] = total;
}

// Every page's rank among the used ones.  With n used pages, of which m lie before page n, the used page of rank k from
// page n on is copy k - m's source, and the free page p before n, with k used ones before it, copy p - k's destination.
// In place new_refs only gets what is there already: other workgroups still count.
template <int kPer>
__global__ __launch_bounds__(kBlock) void compact_rank_kernel(Compact f) {
    __shared__ int part[kWaves];
    int used, total, in_front, all;
    const int chunk = (int)blockIdx.x;
    const Refs<kPer> r(f.pool, chunk, 0);
    const int base = chunks_before(f.counts, f.pool.chunks, chunk, part, &used);
    const int edge = used / (kPer * kBlock);
    const Refs<kPer> at_edge(f.pool, edge, 0);
    int mine = 0;
#pragma unroll
    for (int n = 0; n < kPer; n++) mine += at_edge.page + n < used && at_edge.x[n] != 0;
    before(mine, part, &in_front);
    in_front += chunks_before(f.counts, f.pool.chunks, edge, part, &all);
    if (chunk == 0 && threadIdx.x == 0) *f.num_copies = used - in_front;
    int rank = base + before(kPer - r.free_pages(), part, &total);
#pragma unroll
    for (int n = 0; n < kPer; n++) {
        const int p = r.page + n;
        if (p >= f.pool.num_pages) return;
        int to = -1;
        if (r.x[n] != 0) {
            to = p;
            if (p >= used) {
                const int i = rank - in_front;
                f.src[i] = p;
                f.src_refs[i] = r.x[n];
                to = -2 - i;
            }
            rank++;
        } else if (p < used) {
            f.dst[p - rank] = p;
        }
        f.where[p] = to;
        if (to == p || (r.x[n] == 0 && p >= used)) f.new_refs[p] = r.x[n];
        if (f.page_map && to >= -1) f.page_map[p] = to;
    }
}

__global__ __launch_bounds__(kBlock) void compact_kernel(Compact f, int copy_groups, int turns) {
    if ((int)blockIdx.x < copy_groups) {
        const int i = (int)blockIdx.x * kBlock + (int)threadIdx.x;
        if (i >= *f.num_copies) return;
        const int src = f.src[i], dst = f.dst[i];
        f.copies[i] = gfd_kv_page_copy{src, dst, (int)f.pool.page.d, 0};
        f.new_refs[dst] = f.src_refs[i];
        f.new_refs[src] = 0;
        if (f.page_map) f.page_map[src] = dst;
        return;
    }
    const int id = (int)blockIdx.x - copy_groups, row = id / turns, turn = id % turns;
    const int len = f.len[row], pages = len >= 0 && len <= kMostTokens ? pages_of(f.pool.page, len) : -1;
    if (pages < 0 || pages > f.table_stride || pages > f.new_stride) {
        if (turn == 0 && threadIdx.x == 0) report(f.error, GFD_KV_ERR_ROW);
        return;
    }
    for (int j = turn * kBlock + (int)threadIdx.x; j < pages; j += turns * kBlock) {
        const int id = f.table[row * f.table_stride + j];
        int to = -1;
        if (id >= 0 && id < f.pool.num_pages) {
            to = f.where[id];
            if (to < -1) to = f.dst[-2 - to];
        }
        if (to < 0 && id != -1) report(f.error, GFD_KV_ERR_PAGE);
        f.new_table[row * f.new_stride + j] = to;
    }
}

// ------------------------------------------------------------------ copy

template <typename S>
struct Copy {
    CacheOf<S> dst, src;
    const gfd_kv_page_copy* copies;
    const int* count;
    int max_copies, heads, row_chunks, parts, heads_inner;  // chunks of 16 bytes a row: 2^row_chunks
    Divider inner;  // of a page's rows: heads, or slots
    int* error;
};

constexpr int kUnits = 4;  // rows' chunks a thread copies at once, of keys and of values

// A workgroup copies kBlock kUnits chunks of 16 bytes of a page's keys and the same of its values, in the order of the
// destination; with a chunk of 4-bit numbers goes its scale.  Bound by the bytes.
template <typename S>
__global__ __launch_bounds__(kBlock) void copy_pages_kernel(Copy<S> f, int64_t groups) {
    const int count = f.count ? min(max(*f.count, 0), f.max_copies) : f.max_copies;
    const int rows = f.heads * (int)f.dst.page.d;
    for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
        const int i = (int)(g / f.parts), unit = (int)(g - (int64_t)i * f.parts) * kBlock * kUnits + (int)threadIdx.x;
        if (i >= count) return;
        const gfd_kv_page_copy p = f.copies[i];
        if (p.src < 0 || p.dst < 0) continue;
        if (p.src >= f.src.num_pages || p.dst >= f.dst.num_pages || p.slots < 0 || p.slots > (int)f.dst.page.d) {
            if (threadIdx.x == 0) report(f.error, p.slots < 0 || p.slots > (int)f.dst.page.d ? GFD_KV_ERR_LENGTH : GFD_KV_ERR_PAGE);
            continue;
        }
        u32x4 k[kUnits], v[kUnits];
        uint8_t ks[kUnits], vs[kUnits];
        Place<S> to[kUnits];
        bool there[kUnits];
#pragma unroll
        for (int n = 0; n < kUnits; n++) {
            const int at = unit + n * kBlock, row = at >> f.row_chunks, chunk = at & ((1 << f.row_chunks) - 1);
            const int outer = (int)f.inner.div((uint32_t)row), inner = row - outer * (int)f.inner.d;
            const int slot = f.heads_inner ? outer : inner, head = f.heads_inner ? inner : outer;
            there[n] = row < rows && slot < p.slots;
            if (!there[n]) continue;
            to[n] = place_of<S>(f.dst, p.dst, (uint32_t)slot, head * f.dst.head_stride + 16 * chunk);
            const auto from = place_of<S>(f.src, p.src, (uint32_t)slot, head * f.src.head_stride + 16 * chunk);
            k[n] = *(const u32x4*)(f.src.k + numbers_at(from));
            v[n] = *(const u32x4*)(f.src.v + numbers_at(from));
            if constexpr (S::kBits == 4) {
                ks[n] = f.src.k_scales[from.scales];
                vs[n] = f.src.v_scales[from.scales];
            }
        }
#pragma unroll
        for (int n = 0; n < kUnits; n++) {
            if (!there[n]) continue;
            *(u32x4*)(f.dst.k + numbers_at(to[n])) = k[n];
            *(u32x4*)(f.dst.v + numbers_at(to[n])) = v[n];
            if constexpr (S::kBits == 4) {
                f.dst.k_scales[to[n].scales] = ks[n];
                f.dst.v_scales[to[n].scales] = vs[n];
            }
        }
    }
}

template <typename S, typename C>
int copy_pages(const char* name, const C* dst, const C* src, const gfd_kv_page_copy* copies, int max_copies,
               const int* count, int* error, void* stream) {
    if (const char* why = check_cache(dst)) return refused(name, why);
    if (const char* why = check_cache(src)) return refused(name, why);
    if (dst->page_size != src->page_size || dst->num_heads != src->num_heads || dst->head_dim != src->head_dim)
        return refused(name, "the caches' pages differ in size");
    if (max_copies < 0) return refused(name, "negative max_copies");
    if (max_copies == 0) return 0;
    if (!copies || (uintptr_t)copies % 16 != 0) return refused(name, "copies is missing or not 16-byte aligned");
    Copy<S> f{make_cache(*dst), make_cache(*src), copies, count, max_copies, dst->num_heads, 0, 0, 0, {}, error};
    while (16 * 8 << f.row_chunks < dst->head_dim * S::kBits) f.row_chunks++;
    const int64_t units = ((int64_t)dst->num_heads * dst->page_size) << f.row_chunks;
    if (units >= 1ll << 31) return refused(name, "a page has more than 2^31 chunks of 16 bytes");
    f.parts = (int)ceil_div(units, kBlock * kUnits);
    f.heads_inner = dst->head_stride <= dst->slot_stride;
    f.inner = make_divider((uint32_t)(f.heads_inner ? dst->num_heads : dst->page_size));
    const int64_t groups = (int64_t)max_copies * f.parts;
    // As many workgroups as the card holds a few times over: of a list's places few may be used.
    const unsigned grid = (unsigned)std::min<int64_t>(groups, 16384);
    return launched(name, start(copy_pages_kernel<S>, dim3(grid), kBlock, (hipStream_t)stream, f, groups));
}

// ------------------------------------------------------------- the calls

const char* check_pool(const gfd_kv_pool* pool) {
    if (!pool || !pool->refs) return "no pool";
    if (pool->num_pages < 1 || pool->num_pages > 1 << 24) return "num_pages is outside 1..2^24";
    if (pool->page_size < 1 || pool->page_size > 65536) return "page_size is outside 1..65536";
    return nullptr;
}

int chunks_of(const gfd_kv_pool& p) {
    return (int)ceil_div(p.num_pages, kBlock * (p.num_pages <= kSmallPool ? kFew : kMany));
}
Pool make_pool(const gfd_kv_pool& p) {
    return Pool{p.refs, p.num_pages, chunks_of(p), make_divider((uint32_t)p.page_size)};
}
// f(pages a thread ranks), as a constant.
template <typename F>
int with_pages(const gfd_kv_pool& p, F f) {
    return p.num_pages <= kSmallPool ? f(std::integral_constant<int, kFew>()) : f(std::integral_constant<int, kMany>());
}

constexpr int kMostItems = 1 << 20;

// Counts of chunks, then a fork's sums of needs or what a compaction knows of the pages.
int64_t workspace_bytes(const gfd_kv_pool& p, int num) {
    const int64_t pages = p.num_pages;
    return 4 * (chunks_of(p) + std::max<int64_t>(num + 1, pages + 3 * (pages / 2)));
}

const char* check_workspace(const gfd_kv_pool& p, int num, const void* workspace, size_t bytes) {
    if (!workspace || (uintptr_t)workspace % 16 != 0 || bytes < (size_t)workspace_bytes(p, num))
        return "workspace is missing, not 16-byte aligned or smaller than gfd_kv_pool_workspace_bytes says";
    return nullptr;
}

// Workgroups a row: tables have up to stride entries a row, and few rows are to fill the card too.
int turns_of(int64_t stride, int num) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(stride, 4 * kBlock), 4096 / std::max(num, 1)));
}

const char* check_stride(int64_t stride, int rows) {
    if (rows < 0 || stride < 0 || stride > 1ll << 31) return "a table's rows or stride are out of range";
    return nullptr;
}

}  // namespace
}  // namespace kv
}  // namespace gfd

extern "C" int gfd_kv_copy_pages(const gfd_kv_cache* dst, const gfd_kv_cache* src, const gfd_kv_page_copy* copies,
                                 int max_copies, const int* count, int* error_flag, void* stream) {
    using namespace gfd::kv;
    constexpr char kName[] = "gfd_kv_copy_pages";
    if (const char* why = check_cache(dst)) return refused(kName, why);
    if (const char* why = check_cache(src)) return refused(kName, why);
    if (dst->dtype != src->dtype) return refused(kName, "the caches' types differ");
    if (dst->dtype == GFD_E4M3 && (dst->k_scale != src->k_scale || dst->v_scale != src->v_scale))
        return refused(kName, "the caches' scales differ");
    if (dst->dtype == GFD_E4M3) return copy_pages<E4m3>(kName, dst, src, copies, max_copies, count, error_flag, stream);
    return copy_pages<Bf16>(kName, dst, src, copies, max_copies, count, error_flag, stream);  // bits, of either type
}

extern "C" int gfd_kv4_copy_pages(const gfd_kv4_cache* dst, const gfd_kv4_cache* src, const gfd_kv_page_copy* copies,
                                  int max_copies, const int* count, int* error_flag, void* stream) {
    return gfd::kv::copy_pages<gfd::kv::E2m1>("gfd_kv4_copy_pages", dst, src, copies, max_copies, count, error_flag,
                                              stream);
}

extern "C" int64_t gfd_kv_pool_workspace_bytes(const gfd_kv_pool* pool, int num) {
    using namespace gfd::kv;
    constexpr char kName[] = "gfd_kv_pool_workspace_bytes";
    if (const char* why = check_pool(pool)) {
        refused(kName, why);
        return -1;
    }
    if (num < 0 || num > kMostItems) {
        refused(kName, "num is outside 0..2^20");
        return -1;
    }
    return workspace_bytes(*pool, num);
}

extern "C" int gfd_kv_fork(const gfd_kv_pool* pool, const gfd_kv_fork_call* call, void* workspace,
                           size_t workspace_size, int* error_flag, void* stream) {
    using namespace gfd::kv;
    constexpr char kName[] = "gfd_kv_fork";
    if (const char* why = check_pool(pool)) return refused(kName, why);
    if (!call) return refused(kName, "no call");
    const gfd_kv_fork_call& w = *call;
    if (w.num < 0 || w.num > kMostItems) return refused(kName, "num is outside 0..2^20");
    if (const char* why = check_stride(w.table_stride, w.rows)) return refused(kName, why);
    if (const char* why = check_stride(w.child_stride, w.child_rows)) return refused(kName, why);
    if (w.num == 0) return 0;
    if (!w.parent || !w.child || !w.len || !w.child_table || (w.rows && !w.table))
        return refused(kName, "parent, child, len or a table is missing");
    if (w.rows && w.table == w.child_table && w.table_stride != w.child_stride)
        return refused(kName, "table and child_table are one, with two strides");
    if (!w.copies || (uintptr_t)w.copies % 16 != 0) return refused(kName, "copies is missing or not 16-byte aligned");
    if (const char* why = check_workspace(*pool, w.num, workspace, workspace_size)) return refused(kName, why);
    const Pool p = make_pool(*pool);
    Fork f{p, pool->refs, w.table, w.child_table, w.table_stride, w.child_stride, w.rows, w.child_rows, w.parent,
           w.child, w.len, w.capacity, w.copies, w.num, error_flag, (int*)workspace, (int*)workspace + p.chunks};
    const hipStream_t st = (hipStream_t)stream;
    const int turns = turns_of(w.child_stride, w.num);
    return launched(kName, with_pages(*pool, [&](auto per) {
        constexpr int kPer = decltype(per)::value;
        const int rc = start(fork_count_kernel<kPer>, dim3((unsigned)p.chunks + 1), kBlock, st, f);
        return rc ? rc : start(fork_kernel<kPer>, dim3((unsigned)(p.chunks + w.num * turns)), kBlock, st, f, turns);
    }));
}

extern "C" int gfd_kv_free(const gfd_kv_pool* pool, const int* table, int64_t table_stride, int rows, const int* row,
                           const int* len, int num, int* error_flag, void* stream) {
    using namespace gfd::kv;
    constexpr char kName[] = "gfd_kv_free";
    if (const char* why = check_pool(pool)) return refused(kName, why);
    if (num < 0 || num > kMostItems) return refused(kName, "num is outside 0..2^20");
    if (const char* why = check_stride(table_stride, rows)) return refused(kName, why);
    if (num == 0) return 0;
    if (!row || !len || (rows && !table)) return refused(kName, "table, row or len is missing");
    const Pool p = make_pool(*pool);
    const Free f{pool->refs, p.page, p.num_pages, table, table_stride, rows, row, len, error_flag};
    const int turns = turns_of(table_stride, num);
    return launched(kName, start(free_kernel, dim3((unsigned)(num * turns)), kBlock, (hipStream_t)stream, f, turns));
}

extern "C" int gfd_kv_compact(const gfd_kv_pool* pool, const gfd_kv_compact_call* call, void* workspace,
                              size_t workspace_size, int* error_flag, void* stream) {
    using namespace gfd::kv;
    constexpr char kName[] = "gfd_kv_compact";
    if (const char* why = check_pool(pool)) return refused(kName, why);
    if (!call) return refused(kName, "no call");
    const gfd_kv_compact_call& w = *call;
    if (const char* why = check_stride(w.table_stride, w.rows)) return refused(kName, why);
    if (const char* why = check_stride(w.new_stride, w.rows)) return refused(kName, why);
    if (w.rows > kMostItems) return refused(kName, "more than 2^20 rows");
    if (!w.new_refs || !w.num_copies || (w.rows && (!w.table || !w.new_table || !w.len)))
        return refused(kName, "new_refs, num_copies, a table or len is missing");
    if (w.rows && w.table == w.new_table && w.table_stride != w.new_stride)
        return refused(kName, "table and new_table are one, with two strides");
    if ((!w.copies && pool->num_pages > 1) || (uintptr_t)w.copies % 16 != 0)
        return refused(kName, "copies is missing or not 16-byte aligned");
    if (const char* why = check_workspace(*pool, 0, workspace, workspace_size)) return refused(kName, why);
    const Pool p = make_pool(*pool);
    const int half = p.num_pages / 2;
    int* const counts = (int*)workspace;
    int* const where = counts + p.chunks;
    int* const src = where + p.num_pages;
    const Compact f{p, w.new_refs, w.table, w.new_table, w.table_stride, w.new_stride, w.len, w.rows, w.page_map,
                    w.copies, w.num_copies, error_flag, counts, where, src, src + half, src + 2 * half};
    const hipStream_t st = (hipStream_t)stream;
    const int copy_groups = (int)ceil_div(half, kBlock), turns = turns_of(w.table_stride, w.rows);
    int rc = with_pages(*pool, [&](auto per) {
        constexpr int kPer = decltype(per)::value;
        const int first = start(compact_count_kernel<kPer>, dim3((unsigned)p.chunks), kBlock, st, f);
        return first ? first : start(compact_rank_kernel<kPer>, dim3((unsigned)p.chunks), kBlock, st, f);
    });
    const int groups = copy_groups + w.rows * turns;
    if (!rc && groups) rc = start(compact_kernel, dim3((unsigned)groups), kBlock, st, f, copy_groups, turns);
    return launched(kName, rc);
}

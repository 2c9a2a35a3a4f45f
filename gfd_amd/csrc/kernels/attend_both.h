#pragma once
// A shared prefix of many rows and what follows it with few, in one launch: the
// prefix is bound by the matrix products and leaves half of each CU, which the rest, bound by the cache's bytes,
// fills as it comes (64 requests on 32768 shared keys: 91 us, in two launches 106; 17 times 4
// drafted tokens on 5001 shared 8-bit keys: 30 us, 40).  The prefix goes first: its workgroups are the long ones, and
// taking the two kinds by turns left one of them a CU (128 us).  Of 256 dims one workgroup fits a CU, and the rest
// follows the prefix on the CUs that end first: it is as good as two launches (64 requests on 32768: 160 us, 156; 200 on
// 16384: 345, 368; 17 times 4 tokens on 5001 in 8 bits: 61, 61).
#include "attend_rows.h"
#include "attend_tiles.h"

namespace gfd {
namespace kv {

template <typename T, typename S, int D, int R, int kScores>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attend_both_kernel(Call a, Cache c, Stage prefix,
                                                                                  Stage own, int prefix_turns) {
    __shared__ union Lds {
        RowsLds<T, S, D, R, 4> rows;
        TilesLds<T, S, D, 4> tiles;
    } lds;
    static_assert(TilesKernel<T, S, D, 4>::kThreads == 256, "both bodies have the same workgroups");
    // Turns of 8 workgroups, one for each XCD; the long ones first.
    const int xcd = (int)blockIdx.x & 7, turn = (int)blockIdx.x >> 3;
    const Stage none{0, 0, 0, 0, 1, 0, 0};
    if (turn >= prefix_turns) {
        const int item = (turn - prefix_turns) * 8 + xcd;
        if (item < own.blocks * own.splits * a.kv_heads) attend_rows<T, S, D, R, 4, false>(a, c, none, own, item, lds.rows);
    } else {
        attend_tiles<T, S, D, 4, kScores>(a, c, prefix, none, turn * 8 + xcd, lds.tiles);
    }
}

template <typename T, typename S>
int launch_both(const Call& a, const Cache& c, const Stage& prefix, const Stage& own, int dim, bool wide,
                hipStream_t st) {
    const Stage none{0, 0, 0, 0, 1, 0, 0};
    const int prefix_turns = (int)(tiles_groups(a, prefix, none) / 8),
              own_turns = (int)(((int64_t)own.blocks * own.splits * a.kv_heads + 7) / 8);
    const auto go = [&](auto kernel) {
        return start(kernel, dim3((unsigned)(8 * (prefix_turns + own_turns))), 256, st, a, c, prefix, own, prefix_turns);
    };
    const auto pick = [&](auto d) {
        constexpr int D = decltype(d)::value;
        return with_scores(a, [&](auto scores) {
            constexpr int kScores = decltype(scores)::value;
            return wide ? go(attend_both_kernel<T, S, D, 2, kScores>) : go(attend_both_kernel<T, S, D, 1, kScores>);
        });
    };
    if (dim == 64) return pick(std::integral_constant<int, 64>());
    if (dim == 128) return pick(std::integral_constant<int, 128>());
    return pick(std::integral_constant<int, 256>());
}

}  // namespace kv
}  // namespace gfd

#pragma once
// What appending to the paged cache shares between cache types: a step's rows
// as a kernel sees them, their positions, and the calls' checks (HIP sources only).
#include <cmath>

#include "paged_kv.h"

namespace gfd {
namespace kv {

struct Rows {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const int* positions;
    const int64_t* slots;
    const float* inv_freq;
    int num_tokens, q_heads, kv_heads, dim, rotary;
    float k_div, v_div;  // stored = x / div
    int* error;
    // Positions of several axes.  axis NULL: one, positions.
    const void* axes_positions;
    const uint8_t* axis;
    int64_t axis_stride, token_stride;
    int num_axes, float_positions;
};

constexpr int kAppendBlock = 256, kAppendTokens = 4;

// The position by which pair i of token t turns.
__device__ __forceinline__ double position_of(const Rows& r, int64_t t, int i) {
    if (!r.axis) return (double)r.positions[t];
    const int axis = r.axis[i];
    if (axis >= r.num_axes) {
        if (r.error) atomicOr(r.error, GFD_KV_ERR_AXIS);
        return 0.0;
    }
    const int64_t at = axis * r.axis_stride + t * r.token_stride;
    return r.float_positions ? (double)((const float*)r.axes_positions)[at] : (double)((const int*)r.axes_positions)[at];
}

// Eight values of row t of a kind (0 q, 1 k, 2 v), from value a on.  All of the choice's terms are values: written as a choice
// between members it becomes a load of the call's arguments in front of each load of a row, and a wait for all
// that is under way.
template <typename N>
__device__ __forceinline__ N pick(int kind, N q, N k, N v) {
    return kind == 0 ? q : kind == 1 ? k : v;
}
__device__ __forceinline__ u32x4 eight_of(const Rows& r, int kind, int64_t t, int a) {
    return *(const u32x4*)(pick(kind, r.q, r.k, r.v) + t * pick(kind, r.q_stride, r.k_stride, r.v_stride) + a);
}

template <typename T>
__device__ __forceinline__ void unpack8(u32x4 w, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const f32x2 y = T::unpack(w[i]);
        x[2 * i] = y[0];
        x[2 * i + 1] = y[1];
    }
}

// How the rotated pairs lie: side by side, a half apart in whole chunks of 8, or a half apart.
enum { kSide, kChunksApart, kApart };

// What a kernel relies on, or NULL if all of it holds.
const char* check_rows(const gfd_kv_rows* rows, int head_dim, const gfd_rotary_axes* axes);
Rows make_rows(const gfd_kv_rows& w, int num_heads, int head_dim, const gfd_rotary_axes* axes, float k_div, float v_div,
               int* error);

}  // namespace kv
}  // namespace gfd

// Rotary positions.
//
//   pair (a, b) of a head, angle t = pos[axis of the pair][row] * freq[pair]:  (a cos t - b sin t, b cos t + a sin t)
//
// Bound by memory: every value is read once and written once. The angles belong to a row and are shared by its heads, so a thread
// keeps V pairs of one row in registers and goes through the heads with them: the reduction of the argument in 64 bits costs what a
// few heads' rotation does. V pairs are one or two vectors of up to 16 bytes on each side.
#pragma once

#include "sequence.cuh"

namespace cck {
namespace seq {

// the axis that pair p turns with
__device__ __forceinline__ int axis_of(const cck_rotation& r, int p) {
    int a = 0, edge = r.section[0];
    while (a < r.axes - 1 && p >= edge) {
        edge += r.section[++a];
    }
    return a;
}
// Turns of pair p at position pos, reduced to [-1/2, 1/2] in 64 bits: of a position of a million and a frequency of 1 an f32 product
// would leave 0.03 radians open. What is left fits f32 to 2^-25 of a turn.
__device__ __forceinline__ float2 cos_sin(int pos, float freq) {
    const double turns = double(pos) * double(freq) * 0.15915494309189533577;
    const float t = float(turns - rint(turns));
    float2 cs;
    sincospif(2.f * t, &cs.y, &cs.x);
    return cs;
}
__device__ __forceinline__ float2 rotate(float a, float b, float2 cs) {
    return make_float2(fmaf(a, cs.x, -b * cs.y), fmaf(b, cs.x, a * cs.y));
}

// Rows of `x` rotated into `y` by the threads t of a block of nt, which is the g-th of a set. A row has `items` items a head: pairs
// [V p, V p + V) for p < rot_items, then 2V copied dimensions each. hs threads share a row's heads.
struct RotaryShape {
    int rows, dim, heads, rot_items, items, hs, sign;
    int64_t xr, xh, yr, yh;
    const void* x;
    void* y;
};
template <class T, int V>
__device__ __forceinline__ void rotary_block(const cck_rotation& R, const RotaryShape& s, int g, int t, int nt) {
    using Vt = Vec<T, V>;
    const int slots = nt / s.items, item = t % s.items;
    const int64_t slot = int64_t(g) * slots + t / s.items;
    const int64_t row = slot / s.hs;
    const int h0 = int(slot % s.hs);
    if (t >= slots * s.items || row >= s.rows) {
        return;
    }
    const bool turn = item < s.rot_items;
    const int p0 = item * V;
    // where the item's two vectors lie inside a head
    const int i0 = turn ? (R.adjacent ? 2 * p0 : p0) : R.dims + (item - s.rot_items) * 2 * V;
    const int i1 = turn && !R.adjacent ? p0 + R.dims / 2 : i0 + V;
    const bool both = turn || i1 < s.dim;
    const T* x = static_cast<const T*>(s.x) + row * s.xr;
    T* y = static_cast<T*>(s.y) + row * s.yr;
    constexpr int kAhead = 4; // heads whose loads are on their way together
    float2 cs[V];
    for (int h = h0; h < s.heads; h += kAhead * s.hs) {
        Vt a[kAhead], b[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (const int hh = h + u * s.hs; hh < s.heads) {
                a[u] = *reinterpret_cast<const Vt*>(x + hh * s.xh + i0);
                b[u] = both ? *reinterpret_cast<const Vt*>(x + hh * s.xh + i1) : a[u];
            }
        }
        if (h == h0 && turn) { // behind the first loads
#pragma unroll
            for (int v = 0; v < V; v++) {
                const int p = p0 + v;
                cs[v] = cos_sin(R.pos[axis_of(R, p) * R.pos_stride + row], R.freq[p]);
                cs[v].y = s.sign < 0 ? -cs[v].y : cs[v].y;
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (const int hh = h + u * s.hs; hh < s.heads) {
                if (turn) {
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        T &pa = R.adjacent ? (2 * v < V ? a[u].v[(2 * v) % V] : b[u].v[(2 * v) % V]) : a[u].v[v];
                        T &pb = R.adjacent ? (2 * v + 1 < V ? a[u].v[(2 * v + 1) % V] : b[u].v[(2 * v + 1) % V]) : b[u].v[v];
                        const float2 z = rotate(to_f32(pa), to_f32(pb), cs[v]);
                        pa = from_f32<T>(z.x), pb = from_f32<T>(z.y);
                    }
                }
                *reinterpret_cast<Vt*>(y + hh * s.yh + i0) = a[u];
                if (both) {
                    *reinterpret_cast<Vt*>(y + hh * s.yh + i1) = b[u];
                }
            }
        }
    }
}

template <class T, int V>
__global__ void __launch_bounds__(512) rotary_kernel(const cck_rotation R, const RotaryShape s) {
    rotary_block<T, V>(R, s, blockIdx.x, threadIdx.x, blockDim.x);
}

} // namespace seq
} // namespace cck

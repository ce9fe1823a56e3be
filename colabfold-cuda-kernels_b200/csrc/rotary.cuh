// Rotary positions.
//
//   pair (a, b) of a head, angle t = pos[axis of the pair][row] * freq[pair]:  (a cos t - b sin t, b cos t + a sin t)
//
// Bound by memory: every value is read once and written once. The angles belong to a row and are shared by its heads: a warp takes a row,
// or a part of a row's heads where rows are few, computes the row's cosines and sines once, into its own shared memory, while the first
// vectors are on their way; a lane then keeps V pairs and goes through heads with them. V pairs are one or two vectors of up to 16 bytes on
// each side. Warps wait for nobody and go from row to row: blocks that shared a table of several rows spent 3.5 us each, mostly waiting,
// and 8192 rows of 40 heads took 55 us; now 40, 4.2 TB/s.
#pragma once

#include "sequence.cuh"

namespace cck {
namespace seq {

// the axis that pair p turns with
__device__ __forceinline__ int axis_of(const cck_rotation& r, int p) {
    int edge = r.section[0];
    if (r.axes == 1 || p < edge) {
        return 0;
    }
    edge += r.section[1];
    if (r.axes == 2 || p < edge) {
        return 1;
    }
    return r.axes == 3 || p < edge + r.section[2] ? 2 : 3;
}
// A frequency as turns per position modulo one, in units of 2^-64: position times this, modulo 2^64, is the angle, reduced without an error but this
// rounding, 2^-65 of a turn times the position. 1 / 2 pi is in two doubles: in one, an angle of 2^20 radians would be off by 2^-32, and codes of rotated
// keys with it. An f32 product would leave 0.03 radians open at a position of a million.
struct Turns {
    uint64_t per;
    bool finite;
};
__device__ __forceinline__ Turns turns_of(float freq) {
    constexpr double kHigh = 0.15915494309189535, kLow = -9.839338337591243e-18;
    const double x = double(freq) * kHigh, rest = fma(double(freq), kHigh, -x) + double(freq) * kLow;
    const long long per = __double2ll_rn((x - rint(x)) * 18446744073709551616.0), more = __double2ll_rn((rest - rint(rest)) * 18446744073709551616.0);
    return {uint64_t(per) + uint64_t(more), freq - freq == 0.f};
}
// The nearest quarter turn is taken off in integers; what is left, at most pi / 4, goes through the Taylor series of sine and cosine about
// zero to the ninth and tenth power (the terms after them are below 2e-9 of the result). It is held in two floats, x + e, down to 2^-58 of a turn,
// so that a small angle keeps its digits, and the last additions carry what they round off: both come out within a few units of the last place of
// themselves, however small the sine is, as far as the angle itself is known (2^-62 of the position). With 2^-32 of a turn it took the same
// time, and a sine of 1e-4 was off by 1e-5 of itself.
__device__ __forceinline__ float2 cos_sin(int pos, Turns t) {
    const uint64_t angle = t.per * uint64_t(int64_t(pos)); // of a turn, in 2^-64
    const uint32_t top = uint32_t(angle >> 32);
    const int32_t quarter = int32_t(top + 0x20000000u) >> 30;          // -2 .. 1
    const int32_t rest = int32_t(top - (uint32_t(quarter) << 30));     // at most 2^29 either way
    const int32_t coarse = (rest + 32) & ~63;                          // 24 bits; the other 38, in 2^-58 of a turn, are 32 with a sign
    const int32_t fine = int32_t(__funnelshift_r(uint32_t(angle), uint32_t(rest - coarse), 6));
    constexpr double kUnit = 6.283185307179586477 / 4294967296.0;
    constexpr float kHigh = float(kUnit), kLow = float(kUnit - double(kHigh)), kFine = float(kUnit / 67108864.0);
    const float high = __int2float_rn(coarse), low = __int2float_rn(fine); // the first is exact
    const float x = high * kHigh, e = fmaf(high, kHigh, -x) + fmaf(high, kLow, low * kFine);
    const float y = x * x, z = fmaf(x, x, -y);
    float s = fmaf(y, 1.f / 362880.f, -1.f / 5040.f), c = fmaf(y, -1.f / 3628800.f, 1.f / 40320.f);
    s = fmaf(y, s, 1.f / 120.f), c = fmaf(y, c, -1.f / 720.f);
    s = fmaf(y, s, -1.f / 6.f), c = fmaf(y, c, 1.f / 24.f);
    const float h = fmaf(y, -0.5f, 1.f); // cos = 1 - y / 2 + ..: what h lost, the small terms, z and e
    c = h + fmaf(-x, e, fmaf(z, -0.5f, fmaf(y * y, c, fmaf(y, -0.5f, 1.f - h))));
    s = x + fmaf(x * y, s, e * h);
    // a quarter turn on: (c, s) -> (-s, c)
    const bool odd = quarter & 1;
    const float u = odd ? s : c, v = odd ? c : s;
    const uint32_t flip_c = uint32_t(quarter + 1) & 2u, flip_s = uint32_t(quarter) & 2u;
    const float2 cs = make_float2(__uint_as_float(__float_as_uint(u) ^ flip_c << 30), __uint_as_float(__float_as_uint(v) ^ flip_s << 30));
    return t.finite ? cs : make_float2(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff));
}
// the same in 64 bits, to the eighteenth power: the terms after them are below 2^-58 of the result
__device__ __forceinline__ double2 cos_sin_exactly(int pos, Turns t) {
    const uint64_t angle = t.per * uint64_t(int64_t(pos));
    const int quarter = int(int64_t(angle + (1ull << 61)) >> 62);
    const double x = double(int64_t(angle - (uint64_t(int64_t(quarter)) << 62))) * (6.283185307179586477 / 18446744073709551616.0), y = x * x;
    double s = 1.0, c = 1.0;
#pragma unroll
    for (int n = 18; n > 0; n -= 2) { // cosine 1 - y / (1 2) (1 - y / (3 4) (1 - ...)), sine over x 1 - y / (2 3) (1 - ...)
        s = n == 18 ? 1.0 : fma(y * (-1.0 / double(n * (n + 1))), s, 1.0), c = fma(y * (-1.0 / double(n * (n - 1))), c, 1.0);
    }
    s *= x;
    const double u = quarter & 1 ? s : c, v = quarter & 1 ? c : s;
    return make_double2(quarter == 1 || quarter == -2 ? -u : u, quarter < 0 ? -v : v);
}
__device__ __forceinline__ float2 rotate(float a, float b, float2 cs) {
    return make_float2(fmaf(a, cs.x, -b * cs.y), fmaf(b, cs.x, a * cs.y));
}

// Cosines and sines of `rows` rows from row0 on, all pairs: table[row][pair]. The block's threads t of nt, which are more than the pairs: one stays with a
// pair, whose frequency it converts once
__device__ __forceinline__ void fill_table(const cck_rotation& R, float2* table, int64_t row0, int rows, int t, int nt) {
    const int pairs = R.dims / 2, step = nt / pairs, p = t % pairs; // step: rows at once
    if (t >= step * pairs) {
        return;
    }
    const Turns f = turns_of(R.freq[p]);
    const int* pos = R.pos + axis_of(R, p) * R.pos_stride + row0;
#pragma unroll 4
    for (int r = t / pairs; r < rows; r += step) {
        table[r * pairs + p] = cos_sin(pos[r], f);
    }
}

// x rotated into y, a unit (one of `splits` parts of a row's heads) after the other: those of warp `unit`, + step, ... A head of a row has `items`
// items: pairs [V p, V p + V) for p < rot_items, then 2V copied dimensions each. table: the warp's own, dims / 2 entries.
struct RotaryShape {
    int dim, heads, rot_items, items, splits, part_heads, sign;
    int64_t units;
    int64_t xr, xh, yr, yh;
    const void* x;
    void* y;
};
template <class T, int V, bool kAdjacent>
__device__ __forceinline__ void rotary_warp(const cck_rotation& R, const RotaryShape& s, float2* table, int64_t unit, int64_t step, int64_t units) {
    using Vt = Words<V * sizeof(T)>;
    const int lane = threadIdx.x & 31, pairs = R.dims / 2;
    // the frequencies of this lane's first pairs, and their axes, stay
    constexpr int kKept = 2;
    Turns kept[kKept];
    const int* pos[kKept];
#pragma unroll
    for (int k = 0; k < kKept; k++) {
        if (const int p = lane + 32 * k; p < pairs) {
            kept[k] = turns_of(R.freq[p]), pos[k] = R.pos + axis_of(R, p) * R.pos_stride;
        }
    }
    const int stride = s.items < 32 ? 32 / s.items : 1, first = s.items < 32 ? lane / s.items : 0; // heads at once; this lane's
    const int64_t xs = stride * s.xh, ys = stride * s.yh;
#pragma unroll 1
    for (; unit < units; unit += step) {
        const int64_t row = s.splits == 1 ? unit : unit / s.splits;
        const int h_begin = s.splits == 1 ? 0 : int(unit - row * s.splits) * s.part_heads;
        const int heads = first < stride ? max(0, ceil_div(min(s.part_heads, s.heads - h_begin) - first, stride)) : 0; // of this lane
#pragma unroll 1
        for (int item0 = 0; item0 < s.items; item0 += 32) {
            const int item = s.items < 32 ? lane - first * s.items : item0 + lane;
            const bool turn = item < s.rot_items;
            const int p0 = item * V;
            // where the item's two vectors lie inside a head
            const int i0 = turn ? (kAdjacent ? 2 * p0 : p0) : R.dims + (item - s.rot_items) * 2 * V;
            const int i1 = turn && !kAdjacent ? p0 + pairs : i0 + V;
            const bool both = turn || i1 < s.dim;
            const T* x = static_cast<const T*>(s.x) + row * s.xr + (h_begin + first) * s.xh + i0;
            T* y = static_cast<T*>(s.y) + row * s.yr + (h_begin + first) * s.yh + i0;
            const int over = i1 - i0, mine = item < s.items ? heads : 0;
            constexpr int kAhead = 2; // heads whose loads are on their way together
            Vt a[kAhead], b[kAhead];
            auto load = [&](int left) {
#pragma unroll
                for (int u = 0; u < kAhead; u++, x += xs) {
                    if (u < left) {
                        a[u] = *reinterpret_cast<const Vt*>(x);
                        b[u] = both ? *reinterpret_cast<const Vt*>(x + over) : a[u];
                    }
                }
            };
            load(mine);
            if (item0 == 0) {
                __syncwarp(); // the last row's table has been read
#pragma unroll
                for (int k = 0; k < kKept; k++) {
                    if (lane + 32 * k < pairs) {
                        table[lane + 32 * k] = cos_sin(pos[k][row], kept[k]);
                    }
                }
#pragma unroll 1
                for (int p = lane + 32 * kKept; p < pairs; p += 32) {
                    table[p] = cos_sin(R.pos[axis_of(R, p) * R.pos_stride + row], turns_of(R.freq[p]));
                }
                __syncwarp();
            }
            float2 cs[V];
            if (turn) {
#pragma unroll
                for (int v = 0; v < V; v++) {
                    cs[v] = table[p0 + v];
                    cs[v].y = s.sign < 0 ? -cs[v].y : cs[v].y;
                }
            }
#pragma unroll 1
            for (int left = mine; left > 0; left -= kAhead) {
#pragma unroll
                for (int u = 0; u < kAhead; u++, y += ys) {
                    if (u >= left) {
                        break;
                    }
                    if (turn) {
                        float p[V], q[V];
                        to_floats<T, V>(a[u], p), to_floats<T, V>(b[u], q);
#pragma unroll
                        for (int v = 0; v < V; v++) {
                            // pair v: of the two vectors, or neighbours in their 2 V values
                            float &pa = !kAdjacent || 2 * v < V ? p[kAdjacent ? 2 * v % V : v] : q[2 * v % V];
                            float &pb = kAdjacent && 2 * v + 1 < V ? p[(2 * v + 1) % V] : q[kAdjacent ? (2 * v + 1) % V : v];
                            const float2 z = rotate(pa, pb, cs[v]);
                            pa = z.x, pb = z.y;
                        }
                        a[u] = from_floats<T, V>(p), b[u] = from_floats<T, V>(q);
                    }
                    *reinterpret_cast<Vt*>(y) = a[u];
                    if (both) {
                        *reinterpret_cast<Vt*>(y + over) = b[u];
                    }
                }
                load(left - kAhead);
            }
        }
    }
}

constexpr int kRotaryThreads = 256;
template <class T, int V, bool kAdjacent>
__global__ void __launch_bounds__(kRotaryThreads, 4) rotary_kernel(const __grid_constant__ cck_rotation R, const __grid_constant__ RotaryShape s) {
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = threadIdx.x >> 5, warps = kRotaryThreads / 32;
    rotary_warp<T, V, kAdjacent>(R, s, reinterpret_cast<float2*>(smem) + warp * (R.dims / 2), int64_t(blockIdx.x) * warps + warp, int64_t(gridDim.x) * warps, s.units);
}

} // namespace seq
} // namespace cck

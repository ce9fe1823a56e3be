// Attention over the paged 8-bit cache for few rows: decode steps, guessed tokens.
//
//   x(r, t) = softmax_scale log2(e) k_scale(t) (q_r . k_t) + log2 v_scale(t)          (k_t, v_t: codes)
//   m = max_t x,  p = 2^(x - m),  out = sum_t p v_t / sum_t p / v_scale(t)
//
// The values' scale rides in the exponent: p stays in [0, 1] whatever the scales of the pages are, goes to the tensor cores as f16
// and what it loses there (below 2^-24) is small against the largest term of the sum. One pass with running maximum and sum.
//
// Bound by memory: 2 * dim bytes a key and head, read once. Every warp runs on its own: it takes granules of 32 keys, which lie in one
// piece in a page, through a ring of bulk copies into its own shared memory, and multiplies with mma.m16n8k16 in f16 (codes are f16
// exactly). 16 query rows (the heads that share the keys, times the new tokens) fill a tile; a tcgen05 tile of 128 rows would be
// empty but for those. The cache's layout is such that both products read their operand as it lies, four codes a word, with the
// k index permuted alike on both sides:
//   q.k: lane (n = lane / 4, c = lane % 4) holds dims 16 k + 4 c .. + 3 of key n
//   p.v: lane (n, c) holds keys 16 s + 4 c .. + 3 of dim n; so score tile 2 s + j has keys 16 s + 4 (n / 2) + 2 j + n % 2 in its columns
#pragma once

#include <climits>

#include "sequence.cuh"

namespace cck {
namespace seq {

constexpr int kGranule = 32; // keys of one step of a warp

struct AttentionArgs {
    cck_cache cache;
    cck_batch batch;
    const void* q;
    void* out;
    int64_t qr, qh, or_, oh; // strides
    float* lse;
    float scale_log2; // softmax_scale * log2(e)
    int q_heads, group, causal, window;
    int row_tiles, splits, chunk; // splits: chunks of `chunk` keys (a multiple of kGranule) that the launch gives a sequence at most
    float *part_o, *part_ml;      // [splits][rows * q_heads][dim], [..][2]; null without splits
};

// keys [lo, hi) that row i (a place in its sequence) sees
__device__ __forceinline__ int2 seen_by(const AttentionArgs& A, int place, int len) {
    const int hi = A.causal ? min(len, place + 1) : len;
    const int lo = A.window > 0 ? max(0, place - A.window + 1) : 0;
    return make_int2(lo, max(hi, lo));
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}

constexpr int kDecodeWarps = 4;
template <int D>
struct DecodeShape {
    static constexpr int kStage = 2 * kGranule * D;                     // keys, then values
    static constexpr int kStages = 96 * 1024 / (kDecodeWarps * kStage); // two blocks of threads an SM
    static constexpr int kRing = kDecodeWarps * kStages * kStage;
    static constexpr int kSmem = kRing + kDecodeWarps * kStages * 8 + 16;
};

// four dims of a row's result: nothing seen (sum 0) gives 0, -inf
template <class T>
__device__ __forceinline__ void store_out(const AttentionArgs& A, int row, int q_head, int d, float4 y, float top, float sum) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const Vec<T, 4> v{{from_f32<T>(y.x * inv), from_f32<T>(y.y * inv), from_f32<T>(y.z * inv), from_f32<T>(y.w * inv)}};
    *reinterpret_cast<Vec<T, 4>*>(static_cast<T*>(A.out) + row * A.or_ + q_head * A.oh + d) = v;
    if (A.lse && d == 0) {
        A.lse[int64_t(row) * A.q_heads + q_head] = sum == 0.f ? -INFINITY : 0.69314718055994531f * (top + log2f(sum));
    }
}

// Keys that a tile of rows [r0, r1) (rows times heads of a group) sees: as a whole [lo, hi), all of its rows [all_lo, all_hi)
struct TileKeys {
    int lo, hi, all_lo, all_hi;
    int g0, g1; // granules of [lo, hi)
};
__device__ __forceinline__ TileKeys keys_of_tile(const AttentionArgs& A, const Sequence& s, int r0, int r1) {
    const int2 first = seen_by(A, s.place0 + r0 / A.group, s.len), last = seen_by(A, s.place0 + (r1 - 1) / A.group, s.len);
    TileKeys t;
    t.lo = first.x, t.hi = last.y, t.all_lo = last.x, t.all_hi = first.y;
    t.g0 = t.lo / kGranule, t.g1 = max(t.g0, ceil_div(t.hi, kGranule));
    return t;
}

// chunks that have keys; the last one takes what is left where a length is over max_len
__device__ __forceinline__ int chunks_of(const AttentionArgs& A, const TileKeys& t) {
    return min(A.splits, ceil_div(t.g1 - t.g0, A.chunk / kGranule));
}

// A page of the table for 16 or 32 keys, and its scales
struct Piece {
    int page;
    float a, e, iv; // scale of the scores; log2 and inverse of the values' scale
};
__device__ __forceinline__ Piece piece_at(const AttentionArgs& A, int b, int head, int key) {
    const cck_cache& C = A.cache;
    const int col = key / C.page_tokens;
    Piece r;
    r.page = 0, r.a = __int_as_float(0x7fffffff), r.e = 0.f, r.iv = 1.f; // not there: scores are NaN, page 0 is read in its place
    const int p = col < A.batch.table_pages ? A.batch.table[b * A.batch.table_stride + col] : -1;
    if (p >= 0 && p < C.pages) {
        const int64_t at = int64_t(p) * C.heads + head;
        const float vs = C.v_scale[at];
        r.page = p, r.a = C.k_scale[at] * A.scale_log2, r.e = log2f(vs), r.iv = 1.f / vs;
    }
    return r;
}

// codes of the 4 keys from `key` on that lie outside [lo, hi) become zero: an unused slot may hold NaN, and 0 * NaN is NaN
__device__ __forceinline__ uint32_t keep_keys(uint32_t w, int key, int lo, int hi) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (key + e < lo || key + e >= hi) {
            w &= ~(0xFFu << (8 * e));
        }
    }
    return w;
}

// MT: tiles of 16 rows a warp keeps
template <class T, int D, int MT>
__global__ void __launch_bounds__(kDecodeWarps * 32, 2) decode_kernel(const AttentionArgs A) {
    using S = DecodeShape<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n8 = lane >> 2, c4 = lane & 3;
    const int H = A.cache.heads, P = A.cache.page_tokens, G = A.group;
    int unit = blockIdx.x;
    const int split = unit % A.splits;
    unit /= A.splits;
    const int head = unit % H;
    unit /= H;
    const int tile = unit % A.row_tiles, b = unit / A.row_tiles;
    if (A.splits > 1) {
        let_next_start();
    }
    const Sequence s = sequence_of(A.batch, b);
    const int total = s.rows * G, r0 = tile * 16 * MT, r1 = min(r0 + 16 * MT, total);
    if (r0 >= total) {
        return;
    }
    const TileKeys keys = keys_of_tile(A, s, r0, r1);
    const int per = A.chunk / kGranule, ga = keys.g0 + split * per, gb = split == A.splits - 1 ? keys.g1 : min(keys.g1, ga + per);
    if (split > 0 && ga >= gb) {
        return;
    }
    const uint32_t ring = shared_u32(smem) + warp * S::kStages * S::kStage;
    const uint32_t bars = shared_u32(smem) + S::kRing + warp * S::kStages * 8;
    if (lane == 0) {
        for (int i = 0; i < S::kStages; i++) {
            bar_init(bars + 8 * i, 1);
        }
        bar_init_done();
    }
    __syncwarp();

    // this warp's granules: ga + warp, + kDecodeWarps, ...; a granule is one piece of a page, or two where pages hold 16 tokens.
    // A lane looks one piece up, so that 32 are known at a time: `now` for the granule worked on, `next` for copies ahead of it
    const int mine = gb > ga + warp ? ceil_div(gb - ga - warp, kDecodeWarps) : 0;
    const int pieces = P < kGranule ? 2 : 1, piece = kGranule / pieces;
    auto look_up = [&](int first) {
        const int j = first + lane, key = (ga + warp + j / pieces * kDecodeWarps) * kGranule + j % pieces * piece;
        return piece_at(A, b, head, j < mine * pieces && key < keys.hi && key + piece > keys.lo ? key : INT_MAX);
    };
    Piece now = look_up(0), next = look_up(32);
    int batch = 0; // `now` holds pieces 32 batch ..
    auto issue = [&](int i) { // granule i into its stage
        const uint32_t st = ring + i % S::kStages * S::kStage, bar = bars + i % S::kStages * 8;
        const int key = (ga + warp + i * kDecodeWarps) * kGranule;
        if (lane == 0) {
            bar_expect(bar, S::kStage);
        }
        for (int h = 0; h < pieces; h++) {
            const int j = i * pieces + h;
            const int page = __shfl_sync(0xffffffffu, j >> 5 == batch ? now.page : next.page, j & 31);
            const int64_t at = (int64_t(page) * H + head) * P * D + (key + h * piece) % P * D;
            if (lane == 0) {
                bulk_load(st + h * piece * D, static_cast<const char*>(A.cache.k) + at, piece * D, bar);
                bulk_load(st + (kGranule + h * piece) * D, static_cast<const char*>(A.cache.v) + at, piece * D, bar);
            }
        }
    };
    for (int i = 0; i < min(mine, S::kStages); i++) {
        issue(i);
    }

    // queries: this lane's two rows of each tile, f16 relative to a power of two at the row's largest
    uint32_t q[MT][D / 16][4];
    float qs[MT][2];
    int lo[MT][2], hi[MT][2];
#pragma unroll
    for (int t = 0; t < MT; t++) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const int r = r0 + t * 16 + half * 8 + n8;
            float x[D / 16][4], top = 0.f;
            lo[t][half] = hi[t][half] = 0;
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                Vec<T, 4> v{};
                if (r < r1) {
                    v = *reinterpret_cast<const Vec<T, 4>*>(static_cast<const T*>(A.q) + (s.row0 + r / G) * A.qr + (head * G + r % G) * A.qh + 16 * k + 4 * c4);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[k][e] = to_f32(v.v[e]), top = fmaxf(top, fabsf(x[k][e]));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            int ex = 0;
            if (top > 0.f && top <= 3.402823466e38f) {
                frexpf(top, &ex);
            }
            ex = max(ex, -100);
            const float down = ldexpf(1.f, -ex);
            qs[t][half] = ldexpf(1.f, ex);
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                q[t][k][half] = pack_f16(x[k][0] * down, x[k][1] * down);
                q[t][k][2 + half] = pack_f16(x[k][2] * down, x[k][3] * down);
            }
            if (r < r1) {
                const int2 see = seen_by(A, s.place0 + r / G, s.len);
                lo[t][half] = see.x, hi[t][half] = see.y;
            }
        }
    }

    float o[MT][D / 8][4] = {}, m[MT][2], l[MT][2] = {};
#pragma unroll
    for (int t = 0; t < MT; t++) {
        m[t][0] = m[t][1] = -INFINITY;
    }
    // where this lane's key of score tile 0 and its dim of value tile 0 lie in a stage
    const int tok = 4 * (n8 >> 1) + (n8 & 1);
    const uint32_t k_at = (tok >> 3) * 8 * D + (tok & 7) * 16 + 4 * c4, v_at = kGranule * D + n8 * 16 + 4 * c4;
    for (int i = 0; i < mine; i++) {
        if ((i * pieces) >> 5 != batch) {
            now = next, batch++;
            next = look_up(32 * (batch + 1));
        }
        float a[2], e[2], iv[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int from = (i * pieces + (pieces == 2 ? h : 0)) & 31;
            a[h] = __shfl_sync(0xffffffffu, now.a, from), e[h] = __shfl_sync(0xffffffffu, now.e, from), iv[h] = __shfl_sync(0xffffffffu, now.iv, from);
        }
        const uint32_t st = ring + i % S::kStages * S::kStage;
        const int key0 = (ga + warp + i * kDecodeWarps) * kGranule;
        if (!bar_wait(bars + i % S::kStages * 8, (i / S::kStages) & 1)) {
            l[0][0] = l[0][1] = l[MT - 1][0] = l[MT - 1][1] = __int_as_float(0x7fffffff); // never the case; rows come out as NaN
            break;
        }
        float x[MT][4][4] = {};
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                // tile j: keys 16 (j / 2) + 2 (j % 2) on from tile 0's; 2 (j % 2) stays inside a group of 8
                uint32_t b0, b1;
                unpack_e4m3(lds32(st + k_at + (j >> 1) * 16 * D + (j & 1) * 32 + k * 128), b0, b1);
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    mma_f16(x[t][j], q[t][k], b0, b1);
                }
            }
        }
        const bool whole = key0 >= keys.all_lo && key0 + kGranule <= keys.all_hi; // all rows see all keys
        uint32_t p[MT][4][2];
        bool grew = false;
        float corr[MT][2];
#pragma unroll
        for (int t = 0; t < MT; t++) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; j++) {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float& y = x[t][j][2 * half + c];
                        y = fmaf(y, a[j >> 1] * qs[t][half], e[j >> 1]);
                        if (!whole) {
                            const int key = key0 + 16 * (j >> 1) + 4 * c4 + 2 * (j & 1) + c;
                            y = key >= lo[t][half] && key < hi[t][half] ? y : -INFINITY;
                        }
                        top = fmaxf(top, y);
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float was = m[t][half], is = fmaxf(was, top), base = is == -INFINITY ? 0.f : is;
                corr[t][half] = exp2_fast(was - base);
                grew = grew || is > was;
                m[t][half] = is;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float p0 = exp2_fast(x[t][j][2 * half] - base), p1 = exp2_fast(x[t][j][2 * half + 1] - base);
                    sum = fmaf(p0 + p1, iv[j >> 1], sum);
                    p[t][j][half] = pack_f16(p0, p1);
                }
                l[t][half] = fmaf(l[t][half], corr[t][half], sum);
            }
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int t = 0; t < MT; t++) {
#pragma unroll
                for (int d = 0; d < D / 8; d++) {
                    o[t][d][0] *= corr[t][0], o[t][d][1] *= corr[t][0], o[t][d][2] *= corr[t][1], o[t][d][3] *= corr[t][1];
                }
            }
        }
        const bool ragged = key0 < keys.lo || key0 + kGranule > keys.hi || a[0] != a[0] || a[1] != a[1];
#pragma unroll
        for (int g = 0; g < 2; g++) {
#pragma unroll
            for (int d = 0; d < D / 8; d++) {
                uint32_t w = lds32(st + v_at + g * 16 * D + d * 128), b0, b1;
                if (ragged) {
                    w = a[g] == a[g] ? keep_keys(w, key0 + 16 * g + 4 * c4, keys.lo, keys.hi) : 0u;
                }
                unpack_e4m3(w, b0, b1);
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    const uint32_t pa[4] = {p[t][2 * g][0], p[t][2 * g][1], p[t][2 * g + 1][0], p[t][2 * g + 1][1]};
                    mma_f16(o[t][d], pa, b0, b1);
                }
            }
        }
        __syncwarp(); // the stage has been read
        if (i + S::kStages < mine) {
            issue(i + S::kStages);
        }
    }

    // the warps' shares together, through the ring
    constexpr int kPitch = D + 4, kRows = 16 * MT;
    static_assert(kDecodeWarps * kRows * (kPitch + 2) * 4 <= S::kRing, "the shares fit the ring");
    float* so = reinterpret_cast<float*>(smem);
    float* sm = so + kDecodeWarps * kRows * kPitch;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < MT; t++) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            float sum = l[t][half];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int row = warp * kRows + t * 16 + half * 8 + n8;
            if (c4 == 0) {
                sm[2 * row] = m[t][half], sm[2 * row + 1] = sum;
            }
#pragma unroll
            for (int d = 0; d < D / 8; d++) {
                *reinterpret_cast<float2*>(so + row * kPitch + 8 * d + 2 * c4) = make_float2(o[t][d][2 * half], o[t][d][2 * half + 1]);
            }
        }
    }
    __syncthreads();
    const bool alone = chunks_of(A, keys) <= 1; // what it has is the result
    constexpr int kLanes = D / 4;                // threads of a row, four dims each
    for (int i = threadIdx.x; i < (r1 - r0) * kLanes; i += kDecodeWarps * 32) {
        const int r = i / kLanes, d = i % kLanes * 4, row = r0 + r;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kDecodeWarps; w++) {
            top = fmaxf(top, sm[2 * (w * kRows + r)]);
        }
        const float base = top == -INFINITY ? 0.f : top;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kDecodeWarps; w++) {
            const float f = exp2_fast(sm[2 * (w * kRows + r)] - base);
            const float4 z = *reinterpret_cast<const float4*>(so + (w * kRows + r) * kPitch + d);
            sum = fmaf(sm[2 * (w * kRows + r) + 1], f, sum);
            y.x = fmaf(z.x, f, y.x), y.y = fmaf(z.y, f, y.y), y.z = fmaf(z.z, f, y.z), y.w = fmaf(z.w, f, y.w);
        }
        const int64_t at = int64_t(s.row0 + row / G) * A.q_heads + head * G + row % G;
        if (alone) {
            store_out<T>(A, s.row0 + row / G, head * G + row % G, d, y, top, sum);
        } else {
            const int64_t part = int64_t(split) * A.batch.rows * A.q_heads + at;
            *reinterpret_cast<float4*>(A.part_o + part * D + d) = y;
            if (d == 0) {
                *reinterpret_cast<float2*>(A.part_ml + 2 * part) = make_float2(top, sum);
            }
        }
    }
}

// The chunks of a row together. A warp takes a (row, query head); tile_rows is the first kernel's.
template <class T>
__global__ void __launch_bounds__(128) merge_kernel(const AttentionArgs A, int tile_rows) {
    wait_for_previous();
    const int lane = threadIdx.x & 31, D = A.cache.dim, G = A.group;
    const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int j = int(item % A.q_heads), b = int(item / A.q_heads / A.batch.max_new), i = int(item / A.q_heads % A.batch.max_new);
    if (b >= A.batch.sequences) {
        return;
    }
    const Sequence s = sequence_of(A.batch, b);
    if (i >= s.rows) {
        return;
    }
    const int r = i * G + j % G, r0 = r / tile_rows * tile_rows;
    const TileKeys keys = keys_of_tile(A, s, r0, min(r0 + tile_rows, s.rows * G));
    const int n = chunks_of(A, keys);
    if (n <= 1 || 4 * lane >= D) {
        return;
    }
    const int64_t at = int64_t(s.row0 + i) * A.q_heads + j, step = int64_t(A.batch.rows) * A.q_heads;
    float top = -INFINITY, sum = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < n; c++) {
        const float2 ml = *reinterpret_cast<const float2*>(A.part_ml + 2 * (at + c * step));
        const float4 z = *reinterpret_cast<const float4*>(A.part_o + (at + c * step) * D + 4 * lane);
        const float is = fmaxf(top, ml.x), base = is == -INFINITY ? 0.f : is;
        const float f = exp2_fast(top - base), g = exp2_fast(ml.x - base);
        top = is, sum = sum * f + ml.y * g;
        y.x = y.x * f + z.x * g, y.y = y.y * f + z.y * g, y.z = y.z * f + z.z * g, y.w = y.w * f + z.w * g;
    }
    store_out<T>(A, s.row0 + i, j, 4 * lane, y, top, sum);
}

} // namespace seq
} // namespace cck

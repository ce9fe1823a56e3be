// Attention over the paged 8-bit cache for few rows (up to 24 a head of the cache): decode steps, guessed tokens.
//
//   x(r, t) = softmax_scale log2(e) k_scale(t) (q_r . k_t) + log2 v_scale(t)          (k_t, v_t: codes)
//   m = max_t x,  p = 2^(x - m),  out = sum_t p v_t / sum_t p / v_scale(t)
//
// The values' scale rides in the exponent: p does not grow with the scales of the pages, goes to the tensor cores as f16 and what it
// loses there is small against the largest term of the sum. One pass with running maximum and sum.
//
// Bound by memory: 2 * dim bytes a key and head, read once. Every warp runs on its own: it takes granules of 32 or 64 keys, which lie in one
// piece in a page, through a ring of bulk copies into its own shared memory. Keys are the 16 rows of its tiles, the 8 columns are query
// rows (the heads that share the keys, times the new tokens): a tcgen05 tile of 128 rows would be empty but for those, and a warp
// that waits for nobody hides its copies better. What then counts is the number of instructions, whose fetch a warp pays for
// anew in every granule; so the codes go to the tensor cores as they lie:
//   K q^T   mma.m16n8k32 on e4m3. ldmatrix brings four 8 keys x 16 dims pieces at once. q, scaled to 256 at its row's largest, is split into
//           terms of 4 bits, each the e4m3 rounding of what the one before left: two hold a bf16, three an f16, down to the last one's
//           smallest step, 2^-17 of the row's largest. Sums are f32 (checked: nothing is cut off in the tensor core).
//   V^T p   mma.m16n8k16 on f16, to which the codes convert exactly. p needs the range: in terms of e4m3 a key of probability
//           2^-16 would vanish beside one of 1, and a long tail of such keys can outweigh it.
// Score rows i and i + 8 of tile u are keys 16 u + 4 (i / 2) + i % 2 and two on, such that transposing a score tile's two 8 x 8 halves
// gives p in the order in which a word of V holds four keys.
// The running maximum is only a reference: it moves when a score is 2^8 over the largest it was set by, so that shuffles and the
// rescaling of the sums are rare; p is at most 2^14, the largest at least 2^6, and what f16 loses (2^-25) lies below 2^-30 of that.
// 64 sequences of up to 8192 tokens, 32 heads on 8 of 128: 141 us, 5.7 TB/s, 0.87 of a copy's rate. One sequence of 700 in pages of 16: 14 us, a
// chain of a launch, a look at the table, a copy, six granules a warp, each fetching its instructions anew, and the way out.
#pragma once

#include <type_traits>

#include "sequence.cuh"

namespace cck {
namespace seq {

// Keys of one step of a warp: 8 KB of codes at 64 and 128 dims. A step has a fixed cost (its pages, its copies, the running maximum) of about
// what 32 keys cost at 128 dims.
constexpr int granule_of(int dim) {
    return dim <= 64 ? 64 : 32;
}

struct AttentionArgs {
    cck_cache cache;
    cck_batch batch;
    const void* q;
    void* out;
    int64_t qr, qh, or_, oh; // strides
    float* lse;
    float scale_log2; // softmax_scale * log2(e)
    int q_heads, group, causal, window;
    int reach; // tokens that a row of the table has pages for
    int granule_shift, page_shift; // keys of a step and tokens of a page are powers of two
    int unit_cost;
    int lose; // test door: the barriers of this block's first copies wait for an arrival that nobody makes; -1: none
    int tile_rows, row_tiles; // a sequence's rows times heads of a group, cut into tiles: `tiles` are those of all sequences, row_tiles each
    // shares of units that several blocks work on: sums [2 blocks][tile rows][dim], reference and sum [..][2]; null: a block takes a unit
    float *part_o, *part_ml;
    struct Split* splits;
};

// keys [lo, hi) that a row at `place` of its sequence sees. Those past the table's reach are not there and make the row NaN: the first of them does
__device__ __forceinline__ int2 seen_by(const AttentionArgs& A, int place, int len) {
    const int hi = A.causal ? min(len, place + 1) : len;
    const int lo = A.window > 0 && place >= A.window ? place - A.window + 1 : 0;
    return make_int2(lo, max(lo, min(hi, max(lo, A.reach) + 1)));
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
__device__ __forceinline__ void mma_e4m3(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// four pieces of 8 rows x 16 bytes; lane l gives the address of row l % 8 of piece l / 8
__device__ __forceinline__ void ldmatrix4(uint32_t (&w)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ float4 codes_to_f32(uint32_t w) {
    uint32_t lo, hi;
    unpack_e4m3(w, lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return make_float4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) { // an 8 x 8 matrix of f16 in the accumulators' layout
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

constexpr int kDecodeWarps = 4;
// p = 2^(x - base); base = largest x - kHeadroom when it is set, and is set anew when x - base is over kSlack (the difference: base + kSlack would
// round up to an x that f16 has no 2^(x - base) for, where scores are past 2^27). It begins at the lowest float, below all scores
constexpr float kHeadroom = 6.f, kSlack = 14.f, kNoBase = -3.402823466e38f;
// terms of 4 bits that hold a query
template <class T>
constexpr int kTermsOf = std::is_same_v<T, __half> ? 3 : 2;
// NT: tiles of 8 query rows. Blocks of threads an SM: what registers (32 NT of sums, 16 NT of queries at 128 dims) and shared memory hold
template <int D, int NT>
struct DecodeShape {
    static constexpr int kBlocks = NT == 1 ? 3 : 2;
    static constexpr int kKeys = granule_of(D), kStage = 2 * kKeys * D; // keys, then values
    static constexpr int kStages = (NT == 1 ? 64 : 96) * 1024 / (kDecodeWarps * kStage);
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
    t.g0 = t.lo >> A.granule_shift, t.g1 = max(t.g0, (t.hi + (1 << A.granule_shift) - 1) >> A.granule_shift);
    return t;
}

// ---- The work, cut into equal shares
//
// A unit is a (tile, head); its granules, and all units' one behind the other, are a line that the launch's blocks of threads cut
// into equal shares, whatever the lengths are. A block's share can begin inside a unit and end inside another: it leaves what it
// has of the first in slot 0 of its part of the workspace, of the last in slot 1, and merge_kernel puts the shares together.
struct Tile {
    Sequence s;
    int r0, rows; // rows r0 .. r0 + rows - 1 of the sequence's rows times heads of a group
};
__device__ __forceinline__ Tile tile_at(const AttentionArgs& A, int i) {
    Tile t;
    const int b = A.row_tiles == 1 ? i : i / A.row_tiles;
    t.s = sequence_of(A.batch, b);
    t.r0 = (i - b * A.row_tiles) * A.tile_rows, t.rows = max(0, min(A.tile_rows, t.s.rows * A.group - t.r0));
    return t;
}
// a unit's stretch of the line: its cost beside the granules (queries, the way out, an empty pipeline) in granules, then these
__device__ __forceinline__ int weight_of(const AttentionArgs& A, int i) {
    const Tile t = tile_at(A, i);
    if (t.rows == 0) {
        return 0;
    }
    const TileKeys k = keys_of_tile(A, t.s, t.r0, t.r0 + t.rows);
    return A.unit_cost + max(1, k.g1 - k.g0); // a tile that sees nothing still has rows to write
}
// Where a share begins: the tile, its start on the line of one head's granules, and the granules of a share (all have as many, the last
// ones fewer or none). A warp finds out together, 32 tiles at a time.
struct Line {
    int64_t size, left, start; // granules of all heads: of a share, left in this one, before the tile
    int tile;
};
__device__ __forceinline__ Line line_of(const AttentionArgs& A, int share, int shares) {
    const int n = A.batch.sequences * A.row_tiles, lane = threadIdx.x & 31, H = A.cache.heads;
    const int first = lane < n ? weight_of(A, lane) : 0;
    int64_t sum = first;
#pragma unroll 1
    for (int i = 32 + lane; i < n; i += 32) {
        sum += weight_of(A, i);
    }
#pragma unroll
    for (int o = 16; o; o /= 2) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    Line l;
    l.size = (sum * H + shares - 1) / shares, l.start = 0, l.tile = 0;
    const int64_t from = l.size * share;
    l.left = min(l.size, sum * H - from);
    if (l.left <= 0) {
        return l;
    }
    int64_t at = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int i = i0 + lane, g = i0 == 0 ? first : i < n ? weight_of(A, i) : 0;
        int upto = g;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            upto += lane >= o ? x : 0;
        }
        const int64_t start = (at + upto - g) * H;
        const unsigned hit = __ballot_sync(0xffffffffu, g > 0 && start <= from && from < start + int64_t(g) * H);
        if (hit) {
            const int who = __ffs(hit) - 1;
            l.tile = i0 + who, l.start = __shfl_sync(0xffffffffu, start, who);
            break;
        }
        at += __shfl_sync(0xffffffffu, upto, 31);
    }
    return l;
}
// A unit that begins in a share and goes on in the next: what merge_kernel needs of it, a word of four for each share. last: the last
// share that has a part of it; the share itself if there is no such unit.
struct Split {
    int tile, head, last, none;
};

// The keys of a granule that one page holds, and the page's scales
struct Piece {
    int64_t at; // their first code, in bytes from the cache's
    float ks, vs;
};
__device__ __forceinline__ Piece piece_at(const AttentionArgs& A, int b, int head, int key, bool wanted) {
    const cck_cache& C = A.cache;
    Piece r;
    r.at = 0, r.ks = __int_as_float(0x7fffffff), r.vs = 1.f; // not there: scores are NaN, page 0 is read in its place
    const int col = key >> A.page_shift;
    const int p = wanted && col < A.batch.table_pages ? A.batch.table[b * A.batch.table_stride + col] : -1;
    if (p >= 0 && p < C.pages) {
        const int64_t block = int64_t(p) * C.heads + head;
        r.at = ((block << A.page_shift) + (key & (C.page_tokens - 1))) * C.dim, r.ks = C.k_scale[block], r.vs = C.v_scale[block];
    }
    return r;
}
__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float inverse_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Codes of values outside [lo, hi) in a stage become zero: an unused slot may hold NaN, and 0 * NaN is NaN. Of pages that are not
// there (`absent`, a bit for each tile of 16 keys) all do.
template <int D, int kKeys>
__device__ __noinline__ void clear_values(uint32_t v, int lo, int hi, uint32_t absent) {
#pragma unroll 1
    for (int i = threadIdx.x & 31; i < kKeys * D / 4; i += 32) {
        const int key = i / (4 * D) * 16 + i % 4 * 4;
        uint32_t w;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(v + 4 * i));
        for (int e = 0; e < 4; e++) {
            if (key + e < lo || key + e >= hi || (absent >> (key / 16) & 1)) {
                w &= ~(0xFFu << (8 * e));
            }
        }
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(v + 4 * i), "r"(w) : "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the next copy into the stage comes after
    __syncwarp();
}

// A warp whose copy got lost: says so for the rest of the block's share and waits for its other copies, as long as they can take, so that none lands
// where somebody else has gone on
__device__ __noinline__ void give_up(int* lost, uint32_t bars, int slot, int phase, int others, int stages) {
    if ((threadIdx.x & 31) == 0) {
        *lost = 1;
    }
#pragma unroll 1
    for (int i = 0; i < others; i++) {
        if (++slot == stages) {
            slot = 0, phase ^= 1;
        }
        bar_wait(bars + slot * 8, phase, kDrainTries);
    }
    __syncwarp();
}

template <class T, int D, int NT>
__global__ void __launch_bounds__(kDecodeWarps * 32, DecodeShape<D, NT>::kBlocks) decode_kernel(const __grid_constant__ AttentionArgs A) {
    using S = DecodeShape<D, NT>;
    constexpr int kTerms = kTermsOf<T>;
    constexpr int kRows = 8 * NT, kTiles = S::kKeys / 16, kKeysShift = S::kKeys == 64 ? 6 : 5; // kTiles: of 16 keys
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int4 lost; // a word for each warp, written by itself and read by all between the barriers of a unit's end
    static_assert(kDecodeWarps == 4, "words of lost");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n8 = lane >> 2, c4 = lane & 3;
    const int H = A.cache.heads, G = A.group;
    const uint32_t ring = shared_u32(smem) + warp * S::kStages * S::kStage;
    const uint32_t bars = shared_u32(smem) + S::kRing + warp * S::kStages * 8;
    if (lane == 0) {
        for (int i = 0; i < S::kStages; i++) {
            bar_init(bars + 8 * i, warp == 0 && int(blockIdx.x) == A.lose ? 2 : 1);
        }
        bar_init_done();
        reinterpret_cast<int*>(&lost)[warp] = 0;
    }
    __syncwarp();
    bool gone = false; // a copy of this block got lost: the rest of its share is NaN, nothing is copied or waited for any more
    // what is left of this block's share, and where it is: tile, head, granules done of the unit
    int64_t left = 1, done = 0, size = 0, at = 0; // at: on the line
    int tile = blockIdx.x / H, head = blockIdx.x % H;
    Split split{0, 0, int(blockIdx.x), 0};
    if (A.part_o) {
        let_next_start();
        const Line line = line_of(A, blockIdx.x, gridDim.x);
        left = line.left, size = line.size, at = size * blockIdx.x, tile = line.tile;
        if (left > 0) {
            const int w = weight_of(A, tile);
            head = int((at - line.start) / w), done = at - line.start - int64_t(head) * w;
        }
    }
    int slot = 0, phase = 0;
#pragma unroll 1
    while (left > 0) {
        const Tile own = tile_at(A, tile);
        if (own.rows == 0) {
            if (!A.part_o) {
                return;
            }
            tile++, head = 0;
            continue;
        }
        const Sequence s = own.s;
        const int b = tile / A.row_tiles, r0 = own.r0, r1 = r0 + own.rows;
        const TileKeys keys = keys_of_tile(A, s, r0, r1);
        const int all = max(1, keys.g1 - keys.g0);
        // what of the unit's stretch of the line is the share's, without the cost at its head
        const int64_t to = A.part_o ? min(int64_t(all + A.unit_cost), done + left) : all + A.unit_cost, unit_at = at - done;
        const int ga = keys.g0 + max(0, int(done) - A.unit_cost), gb = keys.g0 + max(0, int(to) - A.unit_cost);
        left -= to - done, at = unit_at + to, done = 0;
        if (gb == ga) { // the cost alone: the next share begins with the unit
            break;
        }
        const bool alone = gb - ga == all; // a unit of this block only
        if (ga == keys.g0 && !alone) {
            split.tile = tile, split.head = head, split.last = int((unit_at + all + A.unit_cost - 1) / size);
        }
        const int part = 2 * blockIdx.x + (ga == keys.g0 ? 1 : 0);

        // this warp's granules: ga + warp, + kDecodeWarps, ...; a granule is one piece of a page, or several of small pages. A lane looks
        // one piece up, so that 32 are known at a time: `now` for the granule worked on, `next` for copies ahead of it
        const int mine = gone ? 0 : max(0, ceil_div(gb - ga - warp, kDecodeWarps));
        const int piece_shift = min(A.page_shift, kKeysShift), pieces_shift = kKeysShift - piece_shift, pieces = 1 << pieces_shift;
        auto look_up = [&](int first) {
            const int j = first + lane, key = (ga + warp + (j >> pieces_shift) * kDecodeWarps) * S::kKeys + ((j & (pieces - 1)) << piece_shift);
            return piece_at(A, b, head, key, j < mine << pieces_shift && key < keys.hi && key + (1 << piece_shift) > keys.lo);
        };
        Piece now = look_up(0), next = look_up(32);
        int batch = 0; // `now` holds pieces 32 batch ..
        auto issue = [&](int i, int slot) { // granule i into its stage
            const uint32_t st = ring + slot * S::kStage, bar = bars + slot * 8, bytes = D << piece_shift;
            if (lane == 0) {
                bar_expect(bar, S::kStage);
            }
#pragma unroll 1
            for (int h = 0; h < pieces; h++) {
                const int j = (i << pieces_shift) + h;
                const int64_t at = __shfl_sync(0xffffffffu, j >> 5 == batch ? now.at : next.at, j & 31);
                if (lane == 0) {
                    bulk_load(st + h * bytes, static_cast<const char*>(A.cache.k) + at, bytes, bar);
                    bulk_load(st + S::kKeys * D + h * bytes, static_cast<const char*>(A.cache.v) + at, bytes, bar);
                }
            }
        };
#pragma unroll 1
        for (int i = 0; i < min(mine, S::kStages); i++) {
            issue(i, (slot + i) % S::kStages);
        }

        // queries: lane n holds its dims of row 8 t + n, in terms; scores of rows 8 t + 2 c and the next come out in the lane
        uint32_t q[NT][D / 16][kTerms];
        float qs[NT][2];
        int lo[NT][2], hi[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int r = r0 + t * 8 + n8;
            Vec<T, 4> v[D / 16] = {};
            float top = 0.f;
            if (r < r1) {
                const T* from = static_cast<const T*>(A.q) + (s.row0 + r / G) * A.qr + (head * G + r % G) * A.qh + 4 * c4;
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    v[k] = *reinterpret_cast<const Vec<T, 4>*>(from + 16 * k);
                }
            }
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    top = fmaxf(top, fabsf(to_f32(v[k].v[e])));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^-ex brings the largest to [128, 256); an infinity makes the row NaN
            const int ex = min(max((__float_as_int(top) >> 23) - 134, -118), 118);
            const float down = top <= 3.402823466e38f ? exp2_int(-ex) : __int_as_float(0x7fffffff), up = exp2_int(ex);
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                float4 x = make_float4(to_f32(v[k].v[0]) * down, to_f32(v[k].v[1]) * down, to_f32(v[k].v[2]) * down, to_f32(v[k].v[3]) * down);
#pragma unroll
                for (int m = 0; m < kTerms; m++) {
                    q[t][k][m] = pack_e4m3(x.x, x.y, x.z, x.w);
                    const float4 y = codes_to_f32(q[t][k][m]);
                    x = make_float4(x.x - y.x, x.y - y.y, x.z - y.z, x.w - y.w);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int row = r0 + t * 8 + 2 * c4 + h;
                qs[t][h] = __shfl_sync(0xffffffffu, up, 4 * (2 * c4 + h));
                lo[t][h] = hi[t][h] = 0;
                if (row < r1) {
                    const int2 see = seen_by(A, s.place0 + row / G, s.len);
                    lo[t][h] = see.x, hi[t][h] = see.y;
                }
            }
        }

        float o[D / 16][NT][4] = {}, base[NT][2], l[NT][2] = {};
#pragma unroll
        for (int t = 0; t < NT; t++) {
            base[t][0] = base[t][1] = kNoBase;
        }
        const int tok = 4 * (n8 >> 1) + (n8 & 1); // the first key of the lane's score rows
        // the row of a stage that this lane names to ldmatrix: keys in the order of the score rows; dims
        const int mk = 4 * ((lane & 7) >> 1) + (lane & 1) + 2 * (lane >> 3 & 1);
        const uint32_t k_at = (mk >> 3) * 8 * D + (mk & 7) * 16 + (lane >> 4) * 128, v_at = S::kKeys * D + (lane >> 4) * 16 * D + (lane & 15) * 16;
#pragma unroll 1
        for (int i = 0; i < mine; i++) {
            if ((i << pieces_shift) >> 5 != batch) {
                now = next, batch++;
                next = look_up(32 * (batch + 1));
            }
            float a[kTiles], e[kTiles], iv[kTiles];
            uint32_t absent = 0;
            if (pieces == 1) {
                const float ks = __shfl_sync(0xffffffffu, now.ks, i & 31), vs = __shfl_sync(0xffffffffu, now.vs, i & 31);
                absent = ks == ks ? 0u : ~0u;
                a[0] = ks * A.scale_log2, e[0] = log2_fast(vs), iv[0] = inverse_fast(vs);
#pragma unroll
                for (int u = 1; u < kTiles; u++) {
                    a[u] = a[0], e[u] = e[0], iv[u] = iv[0];
                }
            } else {
#pragma unroll
                for (int u = 0; u < kTiles; u++) {
                    const int from = ((i << pieces_shift) + (u * 16 >> piece_shift)) & 31;
                    const float ks = __shfl_sync(0xffffffffu, now.ks, from), vs = __shfl_sync(0xffffffffu, now.vs, from);
                    absent |= ks == ks ? 0u : 1u << u;
                    a[u] = ks * A.scale_log2, e[u] = log2_fast(vs), iv[u] = inverse_fast(vs);
                }
            }
            const uint32_t st = ring + slot * S::kStage;
            const int key0 = (ga + warp + i * kDecodeWarps) * S::kKeys;
            if (!__all_sync(0xffffffffu, bar_wait(bars + slot * 8, phase))) {
                give_up(reinterpret_cast<int*>(&lost) + warp, bars, slot, phase, min(mine - i, S::kStages) - 1, S::kStages);
                break;
            }
            float x[kTiles][NT][4] = {};
#pragma unroll
            for (int k = 0; k < D / 32; k++) {
#pragma unroll
                for (int u = 0; u < kTiles; u++) {
                    uint32_t w[4];
                    ldmatrix4(w, st + k_at + u * 16 * D + k * 256);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
#pragma unroll
                        for (int m = 0; m < kTerms; m++) {
                            mma_e4m3(x[u][t], w, q[t][2 * k][m], q[t][2 * k + 1][m]);
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kTiles; u++) {
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const float f[2] = {a[u] * qs[t][0], a[u] * qs[t][1]};
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        x[u][t][v] = fmaf(x[u][t][v], f[v & 1], e[u]);
                    }
                }
            }
            // masked scores are -inf
            if (key0 < keys.all_lo || key0 + S::kKeys > keys.all_hi) {
#pragma unroll
                for (int u = 0; u < kTiles; u++) {
#pragma unroll
                    for (int t = 0; t < NT; t++) {
#pragma unroll
                        for (int v = 0; v < 4; v++) {
                            const int key = key0 + 16 * u + tok + (v & 2);
                            x[u][t][v] = key >= lo[t][v & 1] && key < hi[t][v & 1] ? x[u][t][v] : -INFINITY;
                        }
                    }
                }
            }
            uint32_t p[kTiles][NT][2];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int u = 0; u < kTiles; u++) {
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        top[v & 1] = fmaxf(top[v & 1], x[u][t][v]);
                    }
                }
                if (__any_sync(0xffffffffu, top[0] - base[t][0] > kSlack || top[1] - base[t][1] > kSlack)) {
                    float corr[2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const float was = base[t][h];
#pragma unroll
                        for (int w = 4; w <= 16; w *= 2) {
                            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], w));
                        }
                        base[t][h] = fmaxf(was, top[h] - kHeadroom);
                        corr[h] = exp2_fast(was - base[t][h]);
                        l[t][h] *= corr[h];
                    }
#pragma unroll
                    for (int d = 0; d < D / 16; d++) {
                        o[d][t][0] *= corr[0], o[d][t][1] *= corr[1], o[d][t][2] *= corr[0], o[d][t][3] *= corr[1];
                    }
                }
#pragma unroll
                for (int u = 0; u < kTiles; u++) {
                    const float p0 = exp2_fast(x[u][t][0] - base[t][0]), p1 = exp2_fast(x[u][t][1] - base[t][1]);
                    const float p2 = exp2_fast(x[u][t][2] - base[t][0]), p3 = exp2_fast(x[u][t][3] - base[t][1]);
                    l[t][0] = fmaf(p0 + p2, iv[u], l[t][0]), l[t][1] = fmaf(p1 + p3, iv[u], l[t][1]);
                    p[u][t][0] = transpose8(pack_f16(p0, p1)), p[u][t][1] = transpose8(pack_f16(p2, p3));
                }
            }
            if (key0 < keys.lo || key0 + S::kKeys > keys.hi || absent) {
                clear_values<D, S::kKeys>(st + S::kKeys * D, keys.lo - key0, keys.hi - key0, absent);
            }
#pragma unroll
            for (int u = 0; u < kTiles; u += 2) {
#pragma unroll
                for (int d = 0; d < D / 16; d++) {
                    uint32_t w[4], f[2][4]; // 16 dims of 32 keys; as f16, of 16 keys each
                    ldmatrix4(w, st + v_at + u * 16 * D + d * 256);
                    unpack_e4m3(w[0], f[0][0], f[0][2]), unpack_e4m3(w[1], f[0][1], f[0][3]);
                    unpack_e4m3(w[2], f[1][0], f[1][2]), unpack_e4m3(w[3], f[1][1], f[1][3]);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        mma_f16(o[d][t], f[0], p[u][t][0], p[u][t][1]);
                        mma_f16(o[d][t], f[1], p[u + 1][t][0], p[u + 1][t][1]);
                    }
                }
            }
            __syncwarp(); // the stage has been read
            if (i + S::kStages < mine) {
                issue(i + S::kStages, slot);
            }
            if (++slot == S::kStages) {
                slot = 0, phase ^= 1;
            }
        }

        // the warps' shares together, through the ring
        constexpr int kPitch = D + 4;
        static_assert(kDecodeWarps * kRows * (kPitch + 2) * 4 <= S::kRing, "the shares fit the ring");
        float* so = reinterpret_cast<float*>(smem);
        float* sm = so + kDecodeWarps * kRows * kPitch;
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float sum = l[t][h];
#pragma unroll
                for (int w = 4; w <= 16; w *= 2) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, w);
                }
                const int row = warp * kRows + t * 8 + 2 * c4 + h;
                if (n8 == 0) {
                    sm[2 * row] = base[t][h], sm[2 * row + 1] = sum;
                }
#pragma unroll
                for (int d = 0; d < D / 16; d++) {
                    so[row * kPitch + 16 * d + n8] = o[d][t][h], so[row * kPitch + 16 * d + 8 + n8] = o[d][t][2 + h];
                }
            }
        }
        __syncthreads();
        gone = lost.x | lost.y | lost.z | lost.w;
        constexpr int kLanes = D / 4; // threads of a row, four dims each
#pragma unroll 1
        for (int i = threadIdx.x; i < own.rows * kLanes; i += kDecodeWarps * 32) {
            const int r = i / kLanes, d = i % kLanes * 4;
            float top = kNoBase, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kDecodeWarps; w++) {
                top = fmaxf(top, sm[2 * (w * kRows + r)]);
            }
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kDecodeWarps; w++) {
                const float f = exp2_fast(sm[2 * (w * kRows + r)] - top);
                const float4 z = *reinterpret_cast<const float4*>(so + (w * kRows + r) * kPitch + d);
                sum = fmaf(sm[2 * (w * kRows + r) + 1], f, sum);
                y.x = fmaf(z.x, f, y.x), y.y = fmaf(z.y, f, y.y), y.z = fmaf(z.z, f, y.z), y.w = fmaf(z.w, f, y.w);
            }
            sum = gone ? __int_as_float(0x7fffffff) : sum; // which makes the row NaN, here or when its shares are joined
            if (alone) {
                store_out<T>(A, s.row0 + (r0 + r) / G, head * G + (r0 + r) % G, d, y, top, sum);
            } else {
                *reinterpret_cast<float4*>(A.part_o + (int64_t(part) * kRows + r) * D + d) = y;
                if (d == 0) {
                    *reinterpret_cast<float2*>(A.part_ml + 2 * (int64_t(part) * kRows + r)) = make_float2(top, sum);
                }
            }
        }
        if (!A.part_o) {
            return;
        }
        // The ring is free again for the next unit's copies, which write through the async proxy what was written and read here by ordinary
        // stores and loads: those are ordered before them by each thread's fence and the barrier
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        if (++head == H) {
            head = 0, tile++;
        }
    }
    if (A.part_o && threadIdx.x == 0) {
        A.splits[blockIdx.x] = split;
    }
}

// The shares of a unit together. Block x takes the x-th unit that begins in one share and goes on in the next. Its rows are dealt out to the
// blocks y and to the warps, or, where there are many shares, the shares of a row to the warps.
constexpr int kMergeWarps = 8, kMostShares = 1024;
template <class T>
__global__ void __launch_bounds__(kMergeWarps * 32) merge_kernel(const __grid_constant__ AttentionArgs A, int shares) {
    __shared__ float4 so[kMergeWarps][32];
    __shared__ float weights[kMostShares], tops[kMergeWarps], sums[kMergeWarps];
    __shared__ int before[kMergeWarps], found;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = A.cache.dim;
    wait_for_previous();
    // each thread counts the units that begin in its shares and go on
    const int each = ceil_div(shares, kMergeWarps * 32), s0 = threadIdx.x * each, s1 = min(shares, s0 + each);
    int count = 0;
    for (int c = s0; c < s1; c++) {
        count += A.splits[c].last != c;
    }
    int upto = count;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        upto += lane >= o ? x : 0;
    }
    if (lane == 31) {
        before[warp] = upto;
    }
    if (threadIdx.x == 0) {
        found = -1;
    }
    __syncthreads();
    int nth = int(blockIdx.x) - (upto - count);
    for (int w = 0; w < warp; w++) {
        nth -= before[w];
    }
    if (nth >= 0 && nth < count) {
        for (int c = s0; c < s1; c++) {
            if (A.splits[c].last != c && nth-- == 0) {
                found = c;
            }
        }
    }
    __syncthreads();
    const int c0 = found;
    if (c0 < 0) {
        return;
    }
    const Split split = A.splits[c0];
    const Tile own = tile_at(A, split.tile);
    const int n = split.last - c0 + 1;
    auto slot = [&](int c) { return (2 * int64_t(c0 + c) + (c == 0 ? 1 : 0)) * A.tile_rows; };
    if (n <= 2 * kMergeWarps) { // a row by a warp
#pragma unroll 1
        for (int r = blockIdx.y * kMergeWarps + warp; r < own.rows; r += gridDim.y * kMergeWarps) {
            float top = kNoBase, sum = 0.f;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int c = 0; c < n; c++) {
                const int64_t at = slot(c) + r;
                const float2 ml = *reinterpret_cast<const float2*>(A.part_ml + 2 * at);
                const float4 z = 4 * lane < D ? *reinterpret_cast<const float4*>(A.part_o + at * D + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
                const float is = fmaxf(top, ml.x), f = exp2_fast(top - is), w = exp2_fast(ml.x - is);
                top = is, sum = sum * f + ml.y * w;
                y.x = y.x * f + z.x * w, y.y = y.y * f + z.y * w, y.z = y.z * f + z.z * w, y.w = y.w * f + z.w * w;
            }
            if (4 * lane < D) {
                store_out<T>(A, own.s.row0 + (own.r0 + r) / A.group, split.head * A.group + (own.r0 + r) % A.group, 4 * lane, y, top, sum);
            }
        }
        return;
    }
    // a row by all warps: the weights of all shares first, so that their sums are loaded without waiting for one another
#pragma unroll 1
    for (int r = blockIdx.y; r < own.rows; r += gridDim.y) {
        float top = kNoBase, sum = 0.f;
        for (int c = threadIdx.x; c < n; c += kMergeWarps * 32) {
            top = fmaxf(top, A.part_ml[2 * (slot(c) + r)]);
        }
#pragma unroll
        for (int o = 16; o; o /= 2) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        __syncthreads(); // the last row's weights and shares have been read
        if (lane == 0) {
            tops[warp] = top;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kMergeWarps; w++) {
            top = fmaxf(top, tops[w]);
        }
        for (int c = threadIdx.x; c < n; c += kMergeWarps * 32) {
            const float2 ml = *reinterpret_cast<const float2*>(A.part_ml + 2 * (slot(c) + r));
            const float w = exp2_fast(ml.x - top);
            weights[c] = w, sum = fmaf(ml.y, w, sum);
        }
#pragma unroll
        for (int o = 16; o; o /= 2) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (lane == 0) {
            sums[warp] = sum;
        }
        __syncthreads();
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        if (4 * lane < D) {
#pragma unroll 8
            for (int c = warp; c < n; c += kMergeWarps) {
                const float4 z = *reinterpret_cast<const float4*>(A.part_o + (slot(c) + r) * D + 4 * lane);
                const float w = weights[c];
                y.x = fmaf(z.x, w, y.x), y.y = fmaf(z.y, w, y.y), y.z = fmaf(z.z, w, y.z), y.w = fmaf(z.w, w, y.w);
            }
        }
        so[warp][lane] = y;
        __syncthreads();
        if (warp == 0 && 4 * lane < D) {
            y = make_float4(0.f, 0.f, 0.f, 0.f), sum = 0.f;
#pragma unroll
            for (int w = 0; w < kMergeWarps; w++) {
                const float4 z = so[w][lane];
                y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w, sum += sums[w];
            }
            store_out<T>(A, own.s.row0 + (own.r0 + r) / A.group, split.head * A.group + (own.r0 + r) % A.group, 4 * lane, y, top, sum);
        }
    }
}

} // namespace seq
} // namespace cck

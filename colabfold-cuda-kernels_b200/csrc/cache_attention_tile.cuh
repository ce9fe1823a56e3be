// Attention over the paged 8-bit cache for many rows: prompts and pieces of them. The mathematics are cache_attention.cuh's.
//
// Bound by the tensor cores and by the exponentials, which take as long: for 256 rows and 128 keys of 128 dims 2048 cycles of
// tcgen05.mma and 2048 of the special function units. A block of threads keeps two tiles of 128 rows, so that one's products run
// beside the other's exponentials:
//   warps 0-3, 4-7   softmax of tile 0, 1: a thread owns a row, S comes from and p goes to tensor memory
//   warp 8           what to work on; loads: pages as they lie into the rings (one bulk copy a page: the cache's layout is the operand's)
//   warps 9 - 12     issue S of tile 0 and 1, p V of tile 0 and 1
//   warps 13-15      V to f16
// S = q K^T is kind::f8f6f4 on the codes, q in terms of 4 bits, two of a bf16 and three of an f16 (as in cache_attention.cuh, but into
// one accumulator: a term's last bit is 2^-17 of the row's largest): no work for K at all, in the time that f16 would take.
// O += p V is kind::f16 for the sake of p's range, p read from tensor memory. Tensor memory (512 columns): O 2 x 128, S 2 x 2 x 64. S is
// computed for 64 keys at a time into two buffers, p takes its place: a batch of eight tcgen05.mma needs some 530 cycles more than its
// products from the issue to the waiting thread, so that a tile whose S, softmax and p V follow one another takes 4800 cycles for 128 keys
// whatever the rates are. With a buffer ahead, the softmax is the chain: 4200 cycles for 128 keys, half of them the exponentials of two warps on
// one unit. (Every fourth pair of them by a polynomial instead took as long.) A unit's queries, first S and way out are 10000 cycles more.
// 4 pieces of up to 1024 tokens before contexts of up to 8192, 32 heads on 8 of 128, bf16: 333 us, 0.93 PFLOP/s, 0.56 of the bf16 rate
// measured for a library product (364 us and 0.51 among other calls, at lower clocks); prompts of 4096 with a window of 1024, 16 heads on 4 of 64, f16: 93 us, 0.18 of it: nine steps a unit.
#pragma once

#include <cstddef>

#include "cache_attention.cuh"

namespace cck {
namespace seq {

constexpr int kTileKeys = 128, kHalfKeys = 64, kTileRows = 128, kUnitRows = 2 * kTileRows, kTileThreads = 512;
constexpr int kConvertWarps = 3;
// Up to this, a score's last place is at most a half, and x - base is one fused operation. Where scores could be larger (q is at most 256, a code 448), x is
// rounded first, as base was: the fused difference would have digits that base has lost, and 2^(x - base) of the largest score itself could be past f16
constexpr float kFine = 4194304.f;

constexpr int kCtlBytes = 2048;
template <class T, int D>
struct TileShape {
    static constexpr int kTerms = kTermsOf<T>;
    static constexpr int kQ = kTileRows * D;          // bytes of a term of a tile
    static constexpr int kCodes = kTileKeys * D;      // bytes of the codes of K or V
    static constexpr int kKStages = kTerms == 3 ? 2 : 3, kVStages = kTerms == 3 && D == 128 ? 1 : 2, kHStages = 2; // K; V; V in f16
    static constexpr int kOffK = 2 * kTerms * kQ, kOffV = kOffK + kKStages * kCodes, kOffH = kOffV + kVStages * kCodes;
    static constexpr int kOffCtl = kOffH + kHStages * 2 * kCodes;
    static constexpr int kSmem = kOffCtl + kCtlBytes;
    static_assert(kSmem <= 227 * 1024, "shared memory");
};
// A tile's scales are read until its softmax is done. The loads of tile j wait for V of j - 3 to be converted, that for p V of j - 5: they are at
// most 5 tiles ahead. The scales are written before K's barrier is armed, which the products wait for, and these arrive at S's barrier.
constexpr int kScaleSlots = 8;
struct TileScale {
    float a, e, iv, unused; // 16 bytes, stored at once
};
// What a block works on, unit after unit: found out by the loading warp, read by all others
struct Segment {
    int head, r0, rows, row0, place0, len; // rows r0 .. of the sequence that begins at row0
    int lo, hi;                             // keys that the unit's rows see
    int ga, gb;                             // tiles of keys; none: the end
    int part;                               // slot of the workspace; -1: the unit is the block's alone
};
constexpr int kSegments = 3, kReaders = 8 + 4 + kConvertWarps; // warps that read a segment
struct TileCtl {
    uint64_t q_full[2], k_full[3], k_empty[3], v_full[2], v_empty[2], h_full[2], h_empty[2];
    uint64_t s_full[2][2], p_full[2][2], o_done[2][2]; // [tile][buffer of S]
    uint64_t seg_full[kSegments], seg_empty[kSegments];
    uint64_t drained[4]; // the products of a warp that gave up: S of tile 0 and 1, p V of tile 0 and 1
    Segment seg[kSegments];
    TileScale scale[kScaleSlots][kTileKeys / 16];
    uint32_t absent[kScaleSlots]; // a bit for each 16 keys whose page is not there, or that nobody sees
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(TileCtl) <= kCtlBytes, "control block");

// A wait that gives up after about a second, which nothing but a lost copy can cause; then every later one of the block returns at once: the
// roles run to the end of their segment on whatever is there, nothing is copied any more, and the block's whole share becomes NaN (give_up_share)
__device__ __forceinline__ void tile_wait(uint32_t b, uint32_t parity, volatile int* abort) {
#pragma unroll 1
    for (int i = 0; i < kWaitTries; i++) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(b), "r"(parity), "r"(4000)
            : "memory");
        if (ok) {
            return;
        }
        if (*abort) {
            return;
        }
    }
    *abort = 1;
}
__device__ __forceinline__ void tile_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
    tile_wait(shared_u32(bar), parity, abort);
}
__device__ __forceinline__ bool gave_up(TileCtl* ctl) { // a whole warp calls
    return __any_sync(0xffffffffu, *static_cast<volatile int*>(&ctl->abort));
}
// position in a ring
template <int N>
struct Ring {
    int i = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++i == N) {
            i = 0, phase ^= 1;
        }
    }
};

// ---- tensor memory and tcgen05
__device__ __forceinline__ void tm_ld32(uint32_t at, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t at, uint32_t* r) { // with the wait
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at)
        : "memory");
}
// waits for the thread's loads; the registers pass through so that no use of them moves before it
__device__ __forceinline__ void tm_ld_wait(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(at)
        : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]),
        "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at)
        : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void tm_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tm_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tm_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// Shared-memory descriptor of a K-major operand in core matrices of 8 rows x 16 bytes without a swizzle: `lead` bytes to the next 16
// bytes along k, `stride` to the next 8 rows. Start address >> 4 in bits [0,14), lead >> 4 in [16,30), stride >> 4 in [32,46), version 1
// in [46,48), no swizzle: 0 in [61,64). The high word is a constant; n bytes on are n >> 4 in the low one.
__device__ __forceinline__ uint32_t desc_low(uint32_t at, uint32_t lead) {
    return (at & 0x3FFFFu) >> 4 | (lead >> 4) << 16;
}
constexpr uint32_t desc_high(uint32_t stride) {
    return stride >> 4 | 1u << 14;
}
// f32 accumulator (bits [4,6) = 1), M >> 4 in [24,29), N >> 3 in [17,23), both operands K-major; the types' fields are 0: e4m3 of
// kind::f8f6f4, f16 of kind::f16
__device__ __forceinline__ uint32_t tile_idesc(int m, int n) {
    return 1u << 4 | uint32_t(n >> 3) << 17 | uint32_t(m >> 4) << 24;
}
__device__ __forceinline__ uint32_t elected() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e;
}
// The operands of tcgen05.mma live in uniform registers: everything here is a value that the compiler knows to be the same in all
// lanes (uniform()), and the whole warp issues, predicated on one lane
__device__ __forceinline__ uint32_t uniform(uint32_t v) {
    return __shfl_sync(0xffffffffu, v, 0);
}
__device__ __forceinline__ void mma_codes(uint32_t el, uint32_t d, uint32_t a, uint32_t a_high, uint32_t b, uint32_t b_high, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 e, %7, 0;\n\tmov.b64 x, {%1, %2};\n\tmov.b64 y, {%3, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], x, y, %5, p;\n\t}" ::"r"(d),
        "r"(a), "r"(a_high), "r"(b), "r"(b_high), "r"(idesc), "r"(acc), "r"(el)
        : "memory");
}
__device__ __forceinline__ void mma_halves(uint32_t el, uint32_t d, uint32_t a, uint32_t b, uint32_t b_high, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 e, %6, 0;\n\tmov.b64 y, {%2, %3};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(b_high), "r"(idesc), "r"(acc), "r"(el)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t el, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
        "r"(el)
        : "memory");
}

// pairs of f16 to codes and back
__device__ __forceinline__ uint32_t halves_to_codes(__half2 a, __half2 b) {
    uint32_t w;
    asm("{\n\t.reg .b16 x, y;\n\tcvt.rn.satfinite.e4m3x2.f16x2 x, %1;\n\tcvt.rn.satfinite.e4m3x2.f16x2 y, %2;\n\tmov.b32 %0, {x, y};\n\t}"
        : "=r"(w)
        : "r"(*reinterpret_cast<const uint32_t*>(&a)), "r"(*reinterpret_cast<const uint32_t*>(&b)));
    return w;
}
// the next segment; false at the end. A whole warp calls
__device__ __forceinline__ bool next_segment(TileCtl* ctl, Ring<kSegments>& r, Segment& g) {
    tile_wait(&ctl->seg_full[r.i], r.phase, &ctl->abort);
    g = ctl->seg[r.i];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
        bar_arrive(shared_u32(&ctl->seg_empty[r.i]));
    }
    r.next();
    return g.gb > g.ga && !gave_up(ctl);
}

template <class T, int D>
__device__ __forceinline__ void tile_softmax(const AttentionArgs& A, unsigned char* smem, TileCtl* ctl) {
    using S = TileShape<T, D>;
    const int t = threadIdx.x >> 7, row = threadIdx.x & 127;
    const uint32_t lanes = uint32_t(row & ~31) << 16, ts = ctl->tmem + lanes + t * 128, to = ctl->tmem + lanes + 256 + t * 128;
    // the scale's sign goes to the queries, so that the largest score of 16 keys is that of the largest product
    const float sign = A.scale_log2 < 0.f ? -1.f : 1.f;
    Ring<kSegments> segments;
    Segment g;
    uint32_t step = 0, own = 0; // tiles of keys so far: of the block, of this tile of rows
#pragma unroll 1
    while (next_segment(ctl, segments, g)) {
        const int n = g.gb - g.ga;
        if (t * kTileRows >= g.rows) { // the unit has no second tile
            step += n;
            continue;
        }
        const int rt = g.r0 + t * kTileRows, r = rt + row, r1 = g.r0 + g.rows;
        // The row in terms; one that is not there is zero. Scaled to 256 at its largest, a bf16 is an f16 too (down to 2^-32 of that), in which the
        // terms are split off, two at a time. (Rows dealt out to 16 lanes, with coalesced loads, took 20000 cycles of shuffles and waits.)
        float up = 0.f;
        {
            uint4 v[D / 8];
            const T* from = static_cast<const T*>(A.q) + (g.row0 + r / A.group) * A.qr + (g.head * A.group + r % A.group) * A.qh;
#pragma unroll
            for (int k = 0; k < D / 8; k++) {
                v[k] = r < r1 ? *reinterpret_cast<const uint4*>(from + 8 * k) : make_uint4(0, 0, 0, 0);
            }
            uint32_t most = 0;
#pragma unroll
            for (int k = 0; k < D / 8; k++) {
                most = largest_words(largest_words(most, v[k].x, v[k].y), v[k].z, v[k].w);
            }
            const float2 m = unpack2<T>(most);
            const float top = m.x > m.y || m.x != m.x ? m.x : m.y;
            const int ex = min(max((__float_as_int(top) >> 23) - 134, -118), 118);
            const float down = top <= 3.402823466e38f ? sign * exp2_int(-ex) : __int_as_float(0x7fffffff); // not finite: NaN as a whole
            up = sign * exp2_int(ex);
            unsigned char* to_q = smem + t * S::kTerms * S::kQ + (row >> 3) * 8 * D + (row & 7) * 16;
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                __half2 z[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint4& w = v[2 * k + e / 4];
                    const float2 x = unpack2<T>(e % 4 == 0 ? w.x : e % 4 == 1 ? w.y : e % 4 == 2 ? w.z : w.w);
                    z[e] = __floats2half2_rn(x.x * down, x.y * down);
                }
#pragma unroll
                for (int n = 0; n < S::kTerms; n++) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        w[e] = halves_to_codes(z[2 * e], z[2 * e + 1]);
                        uint32_t y[2];
                        unpack_e4m3(w[e], y[0], y[1]);
                        z[2 * e] = __hsub2(z[2 * e], *reinterpret_cast<const __half2*>(&y[0]));
                        z[2 * e + 1] = __hsub2(z[2 * e + 1], *reinterpret_cast<const __half2*>(&y[1]));
                    }
                    *reinterpret_cast<uint4*>(to_q + n * S::kQ + k * 128) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            bar_arrive(shared_u32(&ctl->q_full[t]));
        }
        int2 see = make_int2(0, 0);
        if (r < r1) {
            see = seen_by(A, g.place0 + r / A.group, g.len);
        }
        // keys that all rows of the tile see
        const int all_lo = seen_by(A, g.place0 + (min(rt + kTileRows, r1) - 1) / A.group, g.len).x, all_hi = seen_by(A, g.place0 + rt / A.group, g.len).y;
        float base = kNoBase, l = 0.f;
#pragma unroll 1
        for (int j = 0; j < 2 * n; j++) { // 64 keys at a time
            const int i = j >> 1, h = j & 1, key0 = (g.ga + i) * kTileKeys + h * kHalfKeys;
            const uint32_t td = ts + h * kHalfKeys;
            const TileScale* sc = ctl->scale[(step + i) % kScaleSlots] + 4 * h;
            tile_wait(&ctl->s_full[t][h], (own + i) & 1, &ctl->abort);
            tm_fence_after();
            uint32_t x[64];
            tm_ld32(td, x), tm_ld32(td + 32, x + 32);
            float f[4], e[4], top = -INFINITY;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                f[u] = sc[u].a * up, e[u] = sc[u].e;
            }
            const bool large = max3(f[0], f[1], fmaxf(f[2], f[3])) > kFine / (256.f * 448.f * D);
            tm_ld_wait(x), tm_ld_wait(x + 32);
            // masked scores are -inf; scaled first: a page that is not there has a NaN scale, which they must not take
            if (key0 < all_lo || key0 + kHalfKeys > all_hi || large) {
#pragma unroll
                for (int c = 0; c < 64; c++) {
                    const float y = fmaf(__uint_as_float(x[c]), f[c / 16], e[c / 16]);
                    x[c] = __float_as_uint(key0 + c >= see.x && key0 + c < see.y ? y : -INFINITY);
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    f[u] = 1.f, e[u] = 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float* y = reinterpret_cast<const float*>(x + 16 * u);
                const float m0 = max3(max3(y[0], y[1], y[2]), max3(y[3], y[4], y[5]), max3(y[6], y[7], y[8]));
                const float m1 = max3(max3(y[9], y[10], y[11]), max3(y[12], y[13], y[14]), y[15]);
                top = fmaxf(top, fmaf(fmaxf(m0, m1), f[u], e[u]));
            }
            if (__any_sync(0xffffffffu, top - base > kSlack)) {
                const float was = base;
                base = top - base > kSlack ? top - kHeadroom : base;
                const float corr = exp2_fast(was - base);
                l *= corr;
                if (j > 0) { // O is whole when the last p V is done; the next one waits for this p
                    tile_wait(&ctl->o_done[t][h ^ 1], (own + ((j - 1) >> 1)) & 1, &ctl->abort);
                    tm_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        uint32_t o[16];
                        tm_ld16(to + c, o);
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
                        }
                        tm_st16(to + c, o);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float eb = e[u] - base;
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                for (int k = 0; k < 8; k++) { // packed: half the instructions
                    const float2 y = __ffma2_rn(make_float2(__uint_as_float(x[16 * u + 2 * k]), __uint_as_float(x[16 * u + 2 * k + 1])), make_float2(f[u], f[u]), make_float2(eb, eb));
                    const float2 p = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                    sum = __fadd2_rn(sum, p);
                    x[8 * u + k] = pack_f16(p.x, p.y);
                }
                l = fmaf(sum.x + sum.y, sc[u].iv, l);
            }
            tm_st32(td, x);
            tm_st_wait();
            tm_fence_before();
            bar_arrive(shared_u32(&ctl->p_full[t][h]));
        }
        step += n;
        tile_wait(&ctl->o_done[t][0], (own + n - 1) & 1, &ctl->abort);
        tile_wait(&ctl->o_done[t][1], (own + n - 1) & 1, &ctl->abort);
        own += n;
        tm_fence_after();
        if (ctl->abort) {
            l = __int_as_float(0x7fffffff);
        }
        const int64_t part = int64_t(g.part) * kUnitRows + t * kTileRows + row;
        const int64_t out_row = g.row0 + r / A.group;
        const int out_head = g.head * A.group + r % A.group;
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tm_ld32(to + c, o);
            tm_ld_wait(o);
            if (r >= r1) {
            } else if (g.part < 0) {
                T* y = static_cast<T*>(A.out) + out_row * A.or_ + out_head * A.oh + c;
#pragma unroll
                for (int j = 0; j < 32; j += 8) {
                    Vec<T, 8> v;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        v.v[e] = from_f32<T>(__uint_as_float(o[j + e]) * inv);
                    }
                    *reinterpret_cast<Vec<T, 8>*>(y + j) = v;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    *reinterpret_cast<uint4*>(A.part_o + part * D + c + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                }
            }
        }
        if (r < r1) {
            if (g.part >= 0) {
                *reinterpret_cast<float2*>(A.part_ml + 2 * part) = make_float2(base, l);
            } else if (A.lse) {
                A.lse[out_row * A.q_heads + out_head] = l == 0.f ? -INFINITY : 0.69314718055994531f * (base + log2f(l));
            }
        }
        tm_fence_before();
    }
}

// A block's way through its share of the line, or its one unit: those of the last rows, which see the most keys, come first
struct Walk {
    int64_t left, done, size, at; // at: on the line
    int tile, head;
    Split split;
};
__device__ __forceinline__ Walk walk_from_start(const AttentionArgs& A) { // a whole warp calls
    const int H = A.cache.heads;
    Walk w{1, 0, 0, 0, int(A.batch.sequences * A.row_tiles - 1 - blockIdx.x / H), int(blockIdx.x % H), {0, 0, int(blockIdx.x), 0}};
    if (A.part_o) {
        const Line line = line_of(A, blockIdx.x, gridDim.x);
        w.left = line.left, w.size = line.size, w.at = line.size * blockIdx.x, w.tile = line.tile;
        if (w.left > 0) {
            const int g = weight_of(A, w.tile);
            w.head = int((w.at - line.start) / g), w.done = w.at - line.start - int64_t(w.head) * g;
        }
    }
    return w;
}
// the next unit, or part of one, and its sequence; false: there is none
__device__ __forceinline__ bool next_unit(const AttentionArgs& A, Walk& w, Segment& g, int& b) {
    g = Segment{}, b = 0;
    while (w.left > 0) {
        const Tile own = tile_at(A, w.tile);
        if (own.rows == 0) {
            w.left = A.part_o ? w.left : 0;
            w.tile++, w.head = 0;
            continue;
        }
        const TileKeys keys = keys_of_tile(A, own.s, own.r0, own.r0 + own.rows);
        const int all = max(1, keys.g1 - keys.g0);
        // what of the unit's stretch of the line is the share's, without the cost at its head
        const int64_t to = A.part_o ? min(int64_t(all + A.unit_cost), w.done + w.left) : all + A.unit_cost, unit_at = w.at - w.done;
        const int ga = max(0, int(w.done) - A.unit_cost), gb = max(0, int(to) - A.unit_cost);
        w.left = A.part_o ? w.left - (to - w.done) : 0, w.at = unit_at + to, w.done = 0;
        b = A.row_tiles == 1 ? w.tile : w.tile / A.row_tiles;
        g.head = w.head, g.r0 = own.r0, g.rows = own.rows, g.row0 = own.s.row0, g.place0 = own.s.place0, g.len = own.s.len, g.lo = keys.lo, g.hi = keys.hi;
        g.ga = keys.g0 + ga, g.gb = keys.g0 + gb;
        g.part = gb - ga == all ? -1 : 2 * int(blockIdx.x) + (ga == 0 ? 1 : 0);
        if (A.part_o && ga == 0 && gb > 0 && gb < all) {
            w.split.tile = w.tile, w.split.head = w.head, w.split.last = int((unit_at + all + A.unit_cost - 1) / w.size);
        }
        if (++w.head == A.cache.heads) {
            w.head = 0, w.tile++;
        }
        break;
    }
    return g.gb > g.ga;
}

// NaN for every row of the block's share, in the result or in its part of the workspace; all threads call, when all roles have ended
template <class T, int D>
__device__ __noinline__ void give_up_share(const AttentionArgs& A) {
    const float nan = __int_as_float(0x7fffffff);
    Walk w = walk_from_start(A);
    Segment g;
    int b;
#pragma unroll 1
    while (next_unit(A, w, g, b)) {
#pragma unroll 1
        for (int r = threadIdx.x; r < g.rows; r += kTileThreads) {
            const int64_t row = g.row0 + (g.r0 + r) / A.group;
            const int head = g.head * A.group + (g.r0 + r) % A.group;
            if (g.part >= 0) {
                *reinterpret_cast<float2*>(A.part_ml + 2 * (int64_t(g.part) * kUnitRows + r)) = make_float2(0.f, nan);
                continue;
            }
            T* y = static_cast<T*>(A.out) + row * A.or_ + head * A.oh;
#pragma unroll 1
            for (int d = 0; d < D; d++) {
                y[d] = from_f32<T>(nan);
            }
            if (A.lse) {
                A.lse[row * A.q_heads + head] = nan;
            }
        }
    }
    if (A.part_o && threadIdx.x == 0) {
        A.splits[blockIdx.x] = w.split;
    }
}

template <class T, int D>
__device__ __forceinline__ void tile_load(const AttentionArgs& A, unsigned char* smem, TileCtl* ctl) {
    using S = TileShape<T, D>;
    const int lane = threadIdx.x & 31;
    uint32_t step = 0;
    Ring<S::kKStages> kr;
    Ring<S::kVStages> vr;
    Ring<kSegments> segments;
    Walk walk = walk_from_start(A);
    bool stop = false;
#pragma unroll 1
    while (!stop) {
        Segment g;
        int b;
        const bool more = next_unit(A, walk, g, b);
        tile_wait(&ctl->seg_empty[segments.i], segments.phase ^ 1, &ctl->abort);
        if (lane == 0) {
            ctl->seg[segments.i] = g;
            bar_arrive(shared_u32(&ctl->seg_full[segments.i]));
        }
        segments.next();
        const int n = g.gb - g.ga;
        if (!more || gave_up(ctl)) {
            break;
        }
        // a lane looks 16 keys up, 8 lanes a tile, four tiles at a time
        auto look_up = [&](int first) {
            const int i = first + (lane >> 3), key = (g.ga + i) * kTileKeys + (lane & 7) * 16;
            return piece_at(A, b, g.head, key, i < n && key < g.hi && key + 16 > g.lo);
        };
        Piece now = look_up(0), next = look_up(4);
#pragma unroll 1
        for (int i = 0; i < n; i++) {
            if (i && (i & 3) == 0) {
                now = next, next = look_up(i + 4);
            }
            const int from = (i & 3) * 8;
            const uint32_t there = __ballot_sync(0xffffffffu, now.ks == now.ks) >> from & 0xFFu;
            // a copy for each page: the first of its 16-key pieces that is there; where a window begins inside a page, from there on
            const int mine = lane & 7, per = 1 << (A.page_shift - 4), group = mine & ~(per - 1);
            const uint32_t in_page = there >> group & ((1u << per) - 1);
            const bool leads = in_page && mine == group + __ffs(in_page) - 1 && lane >> 3 == (i & 3);
            const uint32_t bytes = uint32_t(__popc(in_page)) * 16 * D;
            tile_wait(&ctl->k_empty[kr.i], kr.phase ^ 1, &ctl->abort);
            if (gave_up(ctl)) { // no barrier is armed that may not be empty
                stop = true;
                break;
            }
            if (lane >> 3 == (i & 3)) {
                TileScale sc;
                sc.a = now.ks * A.scale_log2, sc.e = log2_fast(now.vs), sc.iv = inverse_fast(now.vs), sc.unused = 0.f;
                ctl->scale[(step + i) % kScaleSlots][mine] = sc;
            }
            if (lane == 0) {
                ctl->absent[(step + i) % kScaleSlots] = ~there & 0xFFu;
            }
            __syncwarp();
            const uint32_t kb = shared_u32(&ctl->k_full[kr.i]), vb = shared_u32(&ctl->v_full[vr.i]);
            if (lane == 0) {
                bar_expect(kb, __popc(there) * 16 * D);
            }
            __syncwarp();
            if (leads) {
                bulk_load(shared_u32(smem + S::kOffK + kr.i * S::kCodes + mine * 16 * D), static_cast<const char*>(A.cache.k) + now.at, bytes, kb);
            }
            kr.next();
            tile_wait(&ctl->v_empty[vr.i], vr.phase ^ 1, &ctl->abort);
            if (gave_up(ctl)) {
                stop = true;
                break;
            }
            if (lane == 0) {
                bar_expect(vb, __popc(there) * 16 * D);
            }
            __syncwarp();
            if (leads) {
                bulk_load(shared_u32(smem + S::kOffV + vr.i * S::kCodes + mine * 16 * D), static_cast<const char*>(A.cache.v) + now.at, bytes, vb);
            }
            vr.next();
        }
        step += n;
    }
    if (gave_up(ctl)) { // copies that are on their way land before the block ends; a stage that was never armed passes
#pragma unroll 1
        for (int i = 0; i < S::kKStages; i++) {
            bar_wait(shared_u32(&ctl->k_full[i]), i < kr.i ? kr.phase : kr.phase ^ 1, kDrainTries);
        }
#pragma unroll 1
        for (int i = 0; i < S::kVStages; i++) {
            bar_wait(shared_u32(&ctl->v_full[i]), i < vr.i ? vr.phase : vr.phase ^ 1, kDrainTries);
        }
        __syncwarp();
    }
    if (A.part_o && lane == 0) {
        A.splits[blockIdx.x] = walk.split;
    }
}

template <class T, int D>
__device__ __forceinline__ void tile_convert(unsigned char* smem, TileCtl* ctl) {
    using S = TileShape<T, D>;
    const int tid = threadIdx.x - (kTileThreads - 32 * kConvertWarps);
    Ring<kSegments> segments;
    Segment g;
    uint32_t step = 0;
    Ring<S::kVStages> vr;
    Ring<S::kHStages> hr;
#pragma unroll 1
    while (next_segment(ctl, segments, g)) {
        const int n = g.gb - g.ga;
#pragma unroll 1
        for (int i = 0; i < n; i++) {
            tile_wait(&ctl->v_full[vr.i], vr.phase, &ctl->abort);
            tile_wait(&ctl->h_empty[hr.i], hr.phase ^ 1, &ctl->abort);
            const uint32_t absent = ctl->absent[(step + i) % kScaleSlots];
            const int key0 = (g.ga + i) * kTileKeys;
            const bool edge = absent || key0 < g.lo || key0 + kTileKeys > g.hi;
            const uint4* from = reinterpret_cast<const uint4*>(smem + S::kOffV + vr.i * S::kCodes);
            uint4* to = reinterpret_cast<uint4*>(smem + S::kOffH + hr.i * 2 * S::kCodes);
#pragma unroll 4
            for (int c = tid; c < 8 * D; c += 32 * kConvertWarps) { // 16 keys of a dim
                uint4 w = from[c];
                const int k16 = c / D, d = c % D;
                if (edge) { // an unused slot may hold NaN, and 0 * NaN is NaN
                    const bool gone = absent >> k16 & 1;
                    auto keep = [&](uint32_t x, int key) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if (gone || key + e < g.lo || key + e >= g.hi) {
                                x &= ~(0xFFu << (8 * e));
                            }
                        }
                        return x;
                    };
                    const int key = key0 + 16 * k16;
                    w = make_uint4(keep(w.x, key), keep(w.y, key + 4), keep(w.z, key + 8), keep(w.w, key + 12));
                }
                uint4 lo, hi;
                unpack_e4m3(w.x, lo.x, lo.y), unpack_e4m3(w.y, lo.z, lo.w), unpack_e4m3(w.z, hi.x, hi.y), unpack_e4m3(w.w, hi.z, hi.w);
                to[2 * k16 * D + d] = lo, to[(2 * k16 + 1) * D + d] = hi;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if ((threadIdx.x & 31) == 0) {
                bar_arrive(shared_u32(&ctl->v_empty[vr.i]));
                bar_arrive(shared_u32(&ctl->h_full[hr.i]));
            }
            vr.next(), hr.next();
        }
        step += n;
    }
}

// a warp that issued products and gave up waits for them, so that tensor memory is free when it is given back
__device__ __forceinline__ void drain_products(TileCtl* ctl, uint32_t el, int which) {
    if (gave_up(ctl)) {
        mma_commit(el, shared_u32(&ctl->drained[which]));
        bar_wait(shared_u32(&ctl->drained[which]), 0, kDrainTries);
        __syncwarp();
    }
}
// The products, a warp for each kind and tile: S as soon as p V has read p from its buffer, p V as soon as p is there. What a warp runs
// between two batches is fetched anew each time, some 5 cycles an instruction: one warp that polled for whatever was ready held the tiles
// up to 5500 cycles a step, one warp for each tile to 4000.
template <class T, int D>
__device__ __forceinline__ void tile_scores(unsigned char* smem, TileCtl* ctl, uint32_t t) {
    using S = TileShape<T, D>;
    const uint32_t el = elected(), sm = uniform(shared_u32(smem)), bars = uniform(shared_u32(ctl)), is = tile_idesc(kTileRows, kHalfKeys);
    const uint32_t ts = uniform(ctl->tmem + t * 128), q = uniform(desc_low(sm + t * S::kTerms * S::kQ, 128)), k0 = desc_low(sm + S::kOffK, 128);
    const uint32_t s_full = bars + offsetof(TileCtl, s_full) + 16 * t, o_done = bars + offsetof(TileCtl, o_done) + 16 * t;
    volatile int* abort = &ctl->abort;
    Ring<S::kKStages> kr;
    Ring<kSegments> segments;
    Segment g;
    uint32_t turn = 0, units = 0; // parities: of the tile's steps before this one, of its units
#pragma unroll 1
    while (next_segment(ctl, segments, g)) {
        const int n = uniform(g.gb - g.ga);
        const bool mine = uniform(g.rows) > kTileRows * t; // else no second tile: its share of the stages is given back
        if (mine) {
            tile_wait(bars + offsetof(TileCtl, q_full) + 8 * t, units, abort);
            units ^= 1;
        }
#pragma unroll 1
        for (int i = 0; i < n; i++) {
            const uint32_t k = uniform(k0 + kr.i * (S::kCodes >> 4));
            tile_wait(bars + offsetof(TileCtl, k_full) + 8 * kr.i, kr.phase, abort);
            if (mine) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (i > 0) { // p of the step before, which lies where S goes, has been read
                        tile_wait(o_done + 8 * h, turn ^ 1, abort);
                    }
                    tm_fence_after();
#pragma unroll
                    for (int m = 0; m < S::kTerms; m++) {
#pragma unroll
                        for (int c = 0; c < D / 32; c++) {
                            mma_codes(el, ts + h * kHalfKeys, q + m * (S::kQ >> 4) + c * 16, desc_high(8 * D), k + h * (kHalfKeys * D >> 4) + c * 16, desc_high(8 * D), is, m + c > 0);
                        }
                    }
                    mma_commit(el, s_full + 8 * h);
                    if (el) { // the scales, which came with K, are the softmax's to read
                        bar_arrive(s_full + 8 * h);
                    }
                }
                turn ^= 1;
            }
            mma_commit(el, bars + offsetof(TileCtl, k_empty) + 8 * kr.i);
            kr.next();
        }
    }
    drain_products(ctl, el, t);
}
template <class T, int D>
__device__ __forceinline__ void tile_sums(unsigned char* smem, TileCtl* ctl, uint32_t t) {
    using S = TileShape<T, D>;
    const uint32_t el = elected(), sm = uniform(shared_u32(smem)), bars = uniform(shared_u32(ctl)), io = tile_idesc(kTileRows, D);
    const uint32_t ts = uniform(ctl->tmem + t * 128), to = uniform(ctl->tmem + 256 + t * 128), v0 = desc_low(sm + S::kOffH, 16 * D);
    const uint32_t p_full = bars + offsetof(TileCtl, p_full) + 16 * t, o_done = bars + offsetof(TileCtl, o_done) + 16 * t;
    volatile int* abort = &ctl->abort;
    Ring<S::kHStages> hr;
    Ring<kSegments> segments;
    Segment g;
    uint32_t turn = 0;
#pragma unroll 1
    while (next_segment(ctl, segments, g)) {
        const int n = uniform(g.gb - g.ga);
        const bool mine = uniform(g.rows) > kTileRows * t;
#pragma unroll 1
        for (int i = 0; i < n; i++) {
            const uint32_t v = uniform(v0 + hr.i * (2 * S::kCodes >> 4));
            tile_wait(bars + offsetof(TileCtl, h_full) + 8 * hr.i, hr.phase, abort);
            if (mine) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    tile_wait(p_full + 8 * h, turn, abort);
                    tm_fence_after();
#pragma unroll
                    for (int c = 0; c < kHalfKeys / 16; c++) {
                        mma_halves(el, to, ts + h * kHalfKeys + 8 * c, v + (h * kHalfKeys / 16 + c) * 2 * D, desc_high(128), io, h + c > 0 ? 1 : i);
                    }
                    mma_commit(el, o_done + 8 * h);
                }
                turn ^= 1;
            }
            mma_commit(el, bars + offsetof(TileCtl, h_empty) + 8 * hr.i);
            hr.next();
        }
    }
    drain_products(ctl, el, 2 + t);
}

template <class T, int D>
__global__ void __launch_bounds__(kTileThreads, 1) tile_kernel(const __grid_constant__ AttentionArgs A) {
    using S = TileShape<T, D>;
    extern __shared__ __align__(128) unsigned char smem[];
    TileCtl* ctl = reinterpret_cast<TileCtl*>(smem + S::kOffCtl);
    const int warp = threadIdx.x >> 5;
    if (A.part_o) {
        let_next_start();
    }
    if (threadIdx.x == 0) {
        auto init = [](uint64_t& b, int n) { bar_init(shared_u32(&b), n); };
        for (int t = 0; t < 2; t++) {
            init(ctl->q_full[t], kTileRows);
            for (int h = 0; h < 2; h++) {
                init(ctl->s_full[t][h], 2), init(ctl->p_full[t][h], kTileRows), init(ctl->o_done[t][h], 1);
            }
            init(ctl->v_full[t], 1), init(ctl->v_empty[t], kConvertWarps), init(ctl->h_full[t], kConvertWarps), init(ctl->h_empty[t], 2);
        }
        for (int i = 0; i < 3; i++) {
            init(ctl->k_full[i], int(blockIdx.x) == A.lose ? 2 : 1), init(ctl->k_empty[i], 2);
        }
        for (int i = 0; i < 4; i++) {
            init(ctl->drained[i], 1);
        }
        for (int i = 0; i < kSegments; i++) {
            init(ctl->seg_full[i], 1), init(ctl->seg_empty[i], kReaders);
        }
        bar_init_done();
        ctl->abort = 0;
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_u32(&ctl->tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tm_fence_before();
    }
    __syncthreads();
    tm_fence_after();
    if (warp < 8) {
        tile_softmax<T, D>(A, smem, ctl);
    } else if (warp == 8) {
        tile_load<T, D>(A, smem, ctl);
    } else if (warp < 11) {
        tile_scores<T, D>(smem, ctl, warp - 9);
    } else if (warp < 13) {
        tile_sums<T, D>(smem, ctl, warp - 11);
    } else {
        tile_convert<T, D>(smem, ctl);
    }
    tm_fence_before();
    __syncthreads();
    if (warp == 9) {
        tm_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(ctl->tmem), "r"(512) : "memory");
    }
    if (*static_cast<volatile int*>(&ctl->abort)) {
        give_up_share<T, D>(A);
    }
}

} // namespace seq
} // namespace cck

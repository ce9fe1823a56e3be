// New keys and values into the paged cache, the keys rotated on the way, queries rotated beside them.
//
//   top = max |x| over the new rows of a (page, head);  e = smallest exponent with top <= 448 * 2^e, at least the old one where older
//   tokens share the page;  code = e4m3(x * 2^-e), nearest even
//
// All of a page's new rows are needed before the first can be rounded. append_pages_kernel keeps them in registers, a group of threads for
// each (page, head) and as many heads at once as a block has groups; the angles of the page's rows are computed once, into shared memory,
// for all heads that a block goes through. It wants 16-bit values and rotated parts that are whole vectors. append_kernel takes everything
// else through shared memory, a block for each (page, head). Each row is read once, each code written once: bound by memory for
// prompts (eight of about 900 tokens, 32 + 8 + 8 heads of 128: 49 us, 3.2 TB/s), by latency for single tokens (64: 11 us with the launch) and for small pages,
// where a block is a chain of loads, angles, the largest value and the codes (2000 tokens of 3 x 20 heads of 64 in pages of 16: 17 us, 15.2 from a captured graph).
#pragma once

#include "rotary.cuh"

namespace cck {
namespace seq {

struct AppendArgs {
    cck_cache cache;
    cck_batch batch;
    cck_rotation rotation; // dims = 0: none
    const void *k, *v;
    int64_t kr, kh, vr, vh;
    int32_t* status;
    int blocks_per_seq; // (page, head) units: [sequences][blocks_per_seq][heads]
    int kv_blocks;      // of the grid; the others rotate queries
    RotaryShape q;
    // of append_pages_kernel: threads for a (page, head), blocks that share a page's heads
    int group_threads, head_splits;
    int apart; // blocks of query_kernel; 0: queries are rotated by the blocks from kv_blocks on
};

constexpr int kAppendThreads = 256;

// The page that unit `unit` of a launch is about, and its new rows; page < 0: nothing to do. `first`: the thread that reports
struct PageRows {
    int page, s0, s1, row0; // slots s0 .. s1 - 1 get the rows from row0 on
};
__device__ __forceinline__ PageRows page_rows(const AppendArgs& A, int unit, bool first) {
    const int P = A.cache.page_tokens, b = unit / A.blocks_per_seq, nth = unit % A.blocks_per_seq;
    const Sequence s = sequence_of(A.batch, b);
    const int from = max(s.place0, 0), to = s.place0 + s.rows, block = from / P + nth;
    const int lo = max(from, block * P), hi = min(to, block * P + P); // places of this page's new rows
    PageRows r{-1, lo - block * P, hi - block * P, s.row0 + lo - s.place0};
    if (lo < hi && block < A.batch.table_pages) {
        r.page = A.batch.table[b * A.batch.table_stride + block];
    }
    const bool none = r.page < 0 || r.page >= A.cache.pages;
    if (A.status && first && ((nth == 0 && s.cut) || (lo < hi && none))) {
        *A.status = 1;
    }
    r.page = none ? -1 : r.page;
    return r;
}
// the queries' units: rows behind the last sequence are left as they are
__device__ __forceinline__ int64_t query_units(const AppendArgs& A) {
    return int64_t(min(max(A.batch.first[A.batch.sequences], 0), A.batch.rows)) * A.q.splits;
}
// four codes times f (a power of two below 1), rounded again
__device__ __forceinline__ uint32_t lowered(uint32_t w, float f) {
    uint32_t lo, hi;
    unpack_e4m3(w, lo, hi);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo)), y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return pack_e4m3(x.x * f, x.y * f, y.x * f, y.y * f);
}
// The scales of a (page, head) after rows whose largest magnitudes are top_k and top_v: those that older tokens use only grow
struct PageScales {
    float k, v, inv_k, inv_v, lower_k, lower_v; // lower: what older codes are multiplied by
};
__device__ __forceinline__ PageScales page_scales(float top_k, float top_v, float old_k, float old_v, bool older) {
    PageScales s;
    s.k = exp2_int(scale_exponent(top_k)), s.v = exp2_int(scale_exponent(top_v));
    if (older) {
        s.k = old_k > s.k ? old_k : s.k, s.v = old_v > s.v ? old_v : s.v;
    }
    s.lower_k = older && old_k > 0.f ? old_k / s.k : 1.f, s.lower_v = older && old_v > 0.f ? old_v / s.v : 1.f;
    s.inv_k = 1.f / s.k, s.inv_v = 1.f / s.v;
    return s;
}

// shared memory of a unit of `rows` new rows: keys in f32, values as they came
__host__ __device__ constexpr int append_key_pitch(int dim) {
    return dim + 4;
}
__host__ __device__ constexpr int append_value_pitch(int dim, int size) {
    return dim + 16 / size;
}
inline size_t append_smem(int rows, int dim, int size) {
    return size_t(rows) * (append_key_pitch(dim) * 4 + append_value_pitch(dim, size) * size + 4) + 128;
}

// ---- Codes of rotated keys that lie next to a rounding's border
//
// A rotation in 32 bits is off by less than 2^-21 (|a'| + |b'|): cosine and sine by 2^-23, a product by 2^-24, for |a| + |b|, which is at most 1.42 times
// |a'| + |b'|, and the sum by 2^-24 of itself: 2.7 * 2^-23. Where both ends of that give the same code, it is the code of the rotation itself. Else, for
// one value in 2^15, the pair is rotated again in 64 bits and rounded once, so that the codes are those of the definition. Without it 31 codes of 12
// batches of 2000 rows of 20 heads of 64 were not. From a captured graph: 64 single tokens 6.4 us as before, eight prompts of about 900 tokens
// 47.4 -> 47.6, 2000 tokens in pages of 16 14.4 -> 15.2. Values at position 0 stay as they are and often lie on a border (of bf16's, one in 16): they
// are told apart by their sines, else a batch of such rows took 64 us instead of 46.
constexpr float kRotationOff = 1.f / 2097152.f;
// the code of a pair's first or second value after rotation, times inv
__device__ __forceinline__ uint32_t exact_code(const cck_rotation& R, int64_t row, int pair, float a, float b, bool second, float inv) {
    const double2 cs = cos_sin_exactly(R.pos[axis_of(R, pair) * R.pos_stride + row], turns_of(R.freq[pair]));
    const double x = (second ? fma(double(b), cs.x, double(a) * cs.y) : fma(double(a), cs.x, -double(b) * cs.y)) * double(inv);
    const float f = __double2float_rz(x); // to odd, so that the second rounding does not see a border that x is beside
    return pack_e4m3(double(f) == x || x != x ? f : __uint_as_float(__float_as_uint(f) | 1u), 0.f) & 0xFFu;
}
// the bytes in which two words of codes differ as values, a bit each: zero has two codes
__device__ __forceinline__ uint32_t differing(uint32_t v, uint32_t w) {
    return ((__vcmpne4(v, w) & __vcmpne4((v | w) & 0x7F7F7F7Fu, 0u) & 0x01010101u) * 0x10204080u) >> 28;
}

constexpr int kAppendSmem = 140 * 1024; // the most: 128 rows of 128 values in 32 bits

__device__ __forceinline__ bool is_finite(float x) {
    return fabsf(x) <= 3.402823466e38f;
}

template <class T, int VQ>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs A) {
    const cck_cache& C = A.cache;
    const int tid = threadIdx.x;
    extern __shared__ __align__(128) unsigned char smem[];
    if (int(blockIdx.x) >= A.kv_blocks) {
        const int warps = kAppendThreads / 32;
        const int64_t unit = int64_t(blockIdx.x - A.kv_blocks) * warps + (tid >> 5), step = int64_t(gridDim.x - A.kv_blocks) * warps;
        float2* table = reinterpret_cast<float2*>(smem) + (tid >> 5) * (A.rotation.dims / 2);
        if (A.rotation.adjacent) {
            rotary_warp<T, VQ, true>(A.rotation, A.q, table, unit, step, query_units(A));
        } else {
            rotary_warp<T, VQ, false>(A.rotation, A.q, table, unit, step, query_units(A));
        }
        return;
    }
    const int D = C.dim, P = C.page_tokens, head = blockIdx.x % C.heads;
    const PageRows pr = page_rows(A, blockIdx.x / C.heads, head == 0 && tid == 0);
    if (pr.page < 0) {
        return;
    }
    const int s0 = pr.s0, s1 = pr.s1, rows = s1 - s0, row0 = pr.row0;
    const int64_t at = int64_t(pr.page) * C.heads + head;

    const int kp = append_key_pitch(D), vp = append_value_pitch(D, sizeof(T));
    float* fk = reinterpret_cast<float*>(smem);
    T* fv = reinterpret_cast<T*>(fk + size_t(rows) * kp);
    int* bad = reinterpret_cast<int*>(fv + size_t(rows) * vp); // a row that holds NaN or an infinity
    float* red = reinterpret_cast<float*>(bad + rows + (rows & 1));
    const float old_k = C.k_scale[at], old_v = C.v_scale[at];
    for (int u = tid; u < rows; u += kAppendThreads) {
        bad[u] = 0;
    }
    __syncthreads();
    constexpr int V = 16 / sizeof(T);
    using Vt = Vec<T, V>;
    const int nv = D / V;
    for (int i = tid; i < rows * nv; i += kAppendThreads) {
        const int u = i / nv, d = i % nv * V;
        const Vt k = *reinterpret_cast<const Vt*>(static_cast<const T*>(A.k) + (row0 + u) * A.kr + head * A.kh + d);
        const Vt v = *reinterpret_cast<const Vt*>(static_cast<const T*>(A.v) + (row0 + u) * A.vr + head * A.vh + d);
        *reinterpret_cast<Vt*>(fv + u * vp + d) = v;
        bool fine = true;
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float x = to_f32(k.v[j]);
            fk[u * kp + d + j] = x;
            fine = fine && is_finite(x) && is_finite(to_f32(v.v[j]));
        }
        if (!fine) {
            bad[u] = 1;
        }
    }
    __syncthreads();
    float top_k = 0.f, top_v = 0.f;
    const int half = A.rotation.dims / 2;
    for (int i = tid; i < rows * half; i += kAppendThreads) {
        const int u = i / half, p = i % half;
        const float2 cs = cos_sin(A.rotation.pos[axis_of(A.rotation, p) * A.rotation.pos_stride + row0 + u], turns_of(A.rotation.freq[p]));
        float* a = fk + u * kp + (A.rotation.adjacent ? 2 * p : p);
        float* c = a + (A.rotation.adjacent ? 1 : half);
        const float2 z = rotate(*a, *c, cs);
        *a = z.x, *c = z.y;
    }
    __syncthreads();
    for (int i = tid; i < rows * D; i += kAppendThreads) {
        const int u = i / D, d = i % D;
        if (!bad[u]) {
            top_k = fmaxf(top_k, fabsf(fk[u * kp + d]));
            top_v = fmaxf(top_v, fabsf(to_f32(fv[u * vp + d])));
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        top_k = fmaxf(top_k, __shfl_xor_sync(0xffffffffu, top_k, o));
        top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, o));
    }
    if ((tid & 31) == 0) {
        red[tid >> 5] = top_k, red[8 + (tid >> 5)] = top_v;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; w++) {
        top_k = fmaxf(top_k, red[w]), top_v = fmaxf(top_v, red[8 + w]);
    }
    const PageScales sc = page_scales(top_k, top_v, old_k, old_v, s0 > 0);
    const float lower_k = sc.lower_k, lower_v = sc.lower_v, inv_k = sc.inv_k, inv_v = sc.inv_v;
    if (tid == 0) {
        C.k_scale[at] = sc.k, C.v_scale[at] = sc.v;
    }
    unsigned char* ck = static_cast<unsigned char*>(C.k) + at * P * D;
    unsigned char* cv = static_cast<unsigned char*>(C.v) + at * P * D;
    // keys: a token's 16 dimensions are 16 bytes
    const int strips = D / 16;
    if (lower_k < 1.f) {
        for (int i = tid; i < s0 * strips; i += kAppendThreads) {
            uint4* p = reinterpret_cast<uint4*>(ck + key_offset(D, i / strips, i % strips * 16));
            uint4 w = *p;
            w.x = lowered(w.x, lower_k), w.y = lowered(w.y, lower_k), w.z = lowered(w.z, lower_k), w.w = lowered(w.w, lower_k);
            *p = w;
        }
    }
    const float most_off = 2.f * top_k * (kRotationOff * inv_k); // of all values, for a first look
    for (int i = tid; i < rows * strips; i += kAppendThreads) {
        const int u = i / strips, d = i % strips * 16;
        const float off = d < A.rotation.dims ? most_off : 0.f;
        uint32_t w[4], beside = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float4 x = *reinterpret_cast<const float4*>(fk + u * kp + d + 4 * j);
            w[j] = bad[u] ? kNanCodes : pack_e4m3(x.x * inv_k, x.y * inv_k, x.z * inv_k, x.w * inv_k);
            beside |= differing(pack_e4m3(fmaf(x.x, inv_k, -off), fmaf(x.y, inv_k, -off), fmaf(x.z, inv_k, -off), fmaf(x.w, inv_k, -off)),
                                pack_e4m3(fmaf(x.x, inv_k, off), fmaf(x.y, inv_k, off), fmaf(x.z, inv_k, off), fmaf(x.w, inv_k, off)))
                      << (4 * j);
        }
        *reinterpret_cast<uint4*>(ck + key_offset(D, s0 + u, d)) = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll 1
        for (beside = bad[u] ? 0 : beside; beside; beside &= beside - 1) {
            const int e = d + __ffs(beside) - 1;
            if (e >= A.rotation.dims) {
                break;
            }
            const int pair = A.rotation.adjacent ? e >> 1 : e < half ? e : e - half, i0 = A.rotation.adjacent ? 2 * pair : pair, i1 = A.rotation.adjacent ? i0 + 1 : i0 + half;
            const float x = fk[u * kp + e], own = (fabsf(fk[u * kp + i0]) + fabsf(fk[u * kp + i1])) * (kRotationOff * inv_k);
            if (pack_e4m3(fmaf(x, inv_k, -own), 0.f) != pack_e4m3(fmaf(x, inv_k, own), 0.f) &&
                A.rotation.pos[axis_of(A.rotation, pair) * A.rotation.pos_stride + row0 + u]) {
                const T* k = static_cast<const T*>(A.k) + (row0 + u) * A.kr + head * A.kh;
                ck[key_offset(D, s0 + u, e)] = (unsigned char)exact_code(A.rotation, row0 + u, pair, to_f32(k[i0]), to_f32(k[i1]), e == i1, inv_k);
            }
        }
    }
    // values: a dimension's 16 tokens are 16 bytes
    const int g0 = lower_v < 1.f ? 0 : s0 / 16, g1 = ceil_div(s1, 16);
    for (int i = tid; i < (g1 - g0) * D; i += kAppendThreads) {
        const int g = g0 + i / D, d = i % D, t0 = g * 16;
        unsigned char* p = cv + value_offset(D, t0, d);
        if (t0 < s0 || t0 + 16 > s1) { // a group of older, new and unused slots
            for (int t = max(t0, lower_v < 1.f ? 0 : s0); t < min(s1, t0 + 16); t++) {
                if (t < s0) {
                    p[t - t0] = (unsigned char)lowered(p[t - t0], lower_v);
                } else {
                    const int u = t - s0;
                    p[t - t0] = bad[u] ? 0 : (unsigned char)pack_e4m3(to_f32(fv[u * vp + d]) * inv_v, 0.f);
                }
            }
            continue;
        }
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int u = t0 + 4 * j + e - s0;
                x[e] = bad[u] ? 0.f : to_f32(fv[u * vp + d]) * inv_v;
            }
            w[j] = pack_e4m3(x[0], x[1], x[2], x[3]);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Codes of a thread's two key items (as below) anew where `which` has a bit, 16 for each
template <class T, int D, bool kAdjacent>
__device__ __noinline__ void exact_codes(const AppendArgs& A, unsigned char* codes, int s0, int row0, int head, int gt, int GT, uint32_t which, float inv) {
#pragma unroll 1
    for (; which; which &= which - 1) {
        const int bit = __ffs(which) - 1, i = bit & 15, it = gt + (bit >> 4) * GT, c = it % (D / 16), slot = s0 + it / (D / 16);
        const int64_t row = row0 + it / (D / 16);
        const T* k = static_cast<const T*>(A.k) + row * A.kr + head * A.kh;
        const int pair = kAdjacent ? 8 * c + (i >> 1) : 8 * c + (i & 7);
        const bool second = kAdjacent ? i & 1 : i >> 3;
        const int i0 = kAdjacent ? 2 * pair : pair, i1 = kAdjacent ? i0 + 1 : i0 + A.rotation.dims / 2;
        codes[key_offset(D, slot, second ? i1 : i0)] = (unsigned char)exact_code(A.rotation, row, pair, to_f32(k[i0]), to_f32(k[i1]), second, inv);
    }
}

// The same in registers, for 16-bit values. Thread gt of a group's GT has key items gt + n GT (16 dims of a row: the two vectors that its pairs
// lie in) and value items (two dims of 16 tokens).
constexpr int kKeyItems = 2, kValueItems = 1, kPageThreads = 512; // of the widest group
template <class T, int D, bool kAdjacent>
__global__ void __launch_bounds__(kPageThreads, 1) append_pages_kernel(const __grid_constant__ AppendArgs A) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float2 red[2][kPageThreads / 32];
    __shared__ unsigned int bad[kPageThreads / 32][4]; // rows of a group that hold NaN or an infinity, a bit each
    const cck_cache& C = A.cache;
    const cck_rotation& R = A.rotation;
    const int tid = threadIdx.x, nt = blockDim.x;
    float2* table = reinterpret_cast<float2*>(smem);
    if (int(blockIdx.x) >= A.kv_blocks) {
        const int warps = nt / 32;
        rotary_warp<T, 8, kAdjacent>(R, A.q, table + (tid >> 5) * (R.dims / 2), int64_t(blockIdx.x - A.kv_blocks) * warps + (tid >> 5), int64_t(gridDim.x - A.kv_blocks) * warps,
                                    query_units(A));
        return;
    }
    if (A.apart) {
        let_next_start();
    }
    const int P = C.page_tokens, H = C.heads, part = blockIdx.x % A.head_splits;
    const PageRows pr = page_rows(A, blockIdx.x / A.head_splits, part == 0 && tid == 0);
    if (pr.page < 0) {
        return;
    }
    const int s0 = pr.s0, s1 = pr.s1, rows = s1 - s0;
    const int GT = A.group_threads, group = tid / GT, gt = tid % GT, at_once = nt / GT;
    const int h_begin = int(int64_t(part) * H / A.head_splits), h_end = int(int64_t(part + 1) * H / A.head_splits);
    constexpr int strips = D / 16;
    const int pairs = R.dims / 2, turned = R.dims / 16;
#pragma unroll 1
    for (int hb = h_begin, pass = 0; hb < h_end; hb += at_once, pass ^= 1) {
        const int head = hb + group;
        const bool active = head < h_end;
        const int64_t at = int64_t(pr.page) * H + (active ? head : 0);
        const float old_k = C.k_scale[at], old_v = C.v_scale[at];
        uint4 ka[kKeyItems], kb[kKeyItems];
        uint32_t va[kValueItems][16];
#pragma unroll
        for (int n = 0; n < kKeyItems; n++) {
            const int it = gt + n * GT, u = it / strips, c = it % strips;
            const int i0 = c < turned && !kAdjacent ? 8 * c : 16 * c, i1 = c < turned && !kAdjacent ? i0 + pairs : i0 + 8;
            ka[n] = kb[n] = make_uint4(0, 0, 0, 0);
            if (active && u < rows) {
                const T* k = static_cast<const T*>(A.k) + (pr.row0 + u) * A.kr + head * A.kh;
                ka[n] = *reinterpret_cast<const uint4*>(k + i0), kb[n] = *reinterpret_cast<const uint4*>(k + i1);
            }
        }
#pragma unroll
        for (int n = 0; n < kValueItems; n++) {
            const int it = gt + n * GT, t0 = (s0 / 16 + it / (D / 2)) * 16, d = it % (D / 2) * 2;
            const T* v = static_cast<const T*>(A.v) + (pr.row0 + t0 - s0) * A.vr + head * A.vh + d;
#pragma unroll
            for (int k = 0; k < 16; k++) {
                va[n][k] = 0;
                if (active && t0 + k >= s0 && t0 + k < s1) {
                    va[n][k] = *reinterpret_cast<const uint32_t*>(v + k * A.vr);
                }
            }
        }
        if (hb == h_begin) {
            if (pairs) {
                fill_table(R, table, pr.row0, rows, tid, nt); // behind the first loads
            }
            __syncthreads();
        }
        // keys rotated, in f32
        float x[kKeyItems][16], moved[kKeyItems] = {}; // moved: an item's largest sine; zero at position 0, where values stay as they are
        float top_k = 0.f, top_v = 0.f;
        // of the values as they came, two in a word, without their signs: the largest tells whether all are finite
        uint32_t most = 0, most_v = 0;
#pragma unroll
        for (int n = 0; n < kKeyItems; n++) {
            const int it = gt + n * GT, u = it / strips, c = it % strips;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 a = unpack2<T>(e == 0 ? ka[n].x : e == 1 ? ka[n].y : e == 2 ? ka[n].z : ka[n].w);
                const float2 b = unpack2<T>(e == 0 ? kb[n].x : e == 1 ? kb[n].y : e == 2 ? kb[n].z : kb[n].w);
                x[n][2 * e] = a.x, x[n][2 * e + 1] = a.y, x[n][8 + 2 * e] = b.x, x[n][9 + 2 * e] = b.y;
            }
            if (u < rows && c < turned) {
                const float4* cs = reinterpret_cast<const float4*>(table + u * pairs + 8 * c);
#pragma unroll
                for (int e = 0; e < 4; e++) { // two pairs
                    const float4 w = cs[e];
                    float &a0 = kAdjacent ? x[n][4 * e] : x[n][2 * e], &b0 = kAdjacent ? x[n][4 * e + 1] : x[n][8 + 2 * e];
                    float &a1 = kAdjacent ? x[n][4 * e + 2] : x[n][2 * e + 1], &b1 = kAdjacent ? x[n][4 * e + 3] : x[n][9 + 2 * e];
                    const float2 z0 = rotate(a0, b0, make_float2(w.x, w.y)), z1 = rotate(a1, b1, make_float2(w.z, w.w));
                    a0 = z0.x, b0 = z0.y, a1 = z1.x, b1 = z1.y;
                    moved[n] = fmaxf(moved[n], fmaxf(fabsf(w.y), fabsf(w.w)));
                }
            }
#pragma unroll
            for (int e = 0; e < 16; e++) {
                top_k = fmaxf(top_k, fabsf(x[n][e]));
            }
            most = largest_words(largest_words(most, ka[n].x, ka[n].y), ka[n].z, ka[n].w);
            most = largest_words(largest_words(most, kb[n].x, kb[n].y), kb[n].z, kb[n].w);
        }
#pragma unroll
        for (int n = 0; n < kValueItems; n++) {
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
                most_v = largest_words(most_v, va[n][k], va[n][k + 1]);
            }
        }
        {
            const float2 m = unpack2<T>(most_v);
            top_v = fmaxf(m.x, m.y);
        }
        const float2 all = unpack2<T>(largest_words(most, most_v, 0));
        const bool fine = is_finite(all.x) && is_finite(all.y);
        auto largest = [&]() { // of the group
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                top_k = fmaxf(top_k, __shfl_xor_sync(0xffffffffu, top_k, o)), top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, o));
            }
            if ((tid & 31) == 0) {
                red[pass][tid >> 5] = make_float2(top_k, top_v);
            }
        };
        auto gather = [&]() {
#pragma unroll 1
            for (int w = 0; w < GT / 32; w++) {
                const float2 m = red[pass][group * (GT / 32) + w];
                top_k = fmaxf(top_k, m.x), top_v = fmaxf(top_v, m.y);
            }
        };
        largest();
        const bool some_bad = __syncthreads_or(!fine);
        if (some_bad) { // seldom: tokens that become NaN in whole, and do not count for the scale
            if (tid < kPageThreads / 32 * 4) {
                bad[tid / 4][tid % 4] = 0;
            }
            __syncthreads();
#pragma unroll
            for (int n = 0; n < kKeyItems; n++) {
                const float2 m = unpack2<T>(largest_words(largest_words(largest_words(0, ka[n].x, ka[n].y), ka[n].z, ka[n].w), // as they came
                                                          largest_words(largest_words(0, kb[n].x, kb[n].y), kb[n].z, kb[n].w), 0));
                if (!is_finite(m.x) || !is_finite(m.y)) {
                    const int u = (gt + n * GT) / strips;
                    atomicOr(&bad[group][u / 32], 1u << (u % 32));
                }
            }
#pragma unroll
            for (int n = 0; n < kValueItems; n++) {
                const int t0 = (s0 / 16 + (gt + n * GT) / (D / 2)) * 16;
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const float2 a = unpack2<T>(va[n][k]);
                    if (!is_finite(a.x) || !is_finite(a.y)) {
                        const int u = t0 + k - s0;
                        atomicOr(&bad[group][u / 32], 1u << (u % 32));
                    }
                }
            }
            __syncthreads();
            top_k = top_v = 0.f;
#pragma unroll
            for (int n = 0; n < kKeyItems; n++) {
                const int u = (gt + n * GT) / strips;
                if (u < rows && !(bad[group][u / 32] >> (u % 32) & 1)) {
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        top_k = fmaxf(top_k, fabsf(x[n][e]));
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < kValueItems; n++) {
                const int t0 = (s0 / 16 + (gt + n * GT) / (D / 2)) * 16;
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const int u = t0 + k - s0;
                    if (u >= 0 && u < rows && (bad[group][u / 32] >> (u % 32) & 1)) {
                        va[n][k] = 0;
                    }
                    const float2 a = unpack2<T>(va[n][k]);
                    top_v = fmaxf(top_v, fmaxf(fabsf(a.x), fabsf(a.y)));
                }
            }
            largest();
            __syncthreads();
        }
        gather();
        if (!active) {
            continue;
        }
        const PageScales sc = page_scales(top_k, top_v, old_k, old_v, s0 > 0);
        if (gt == 0) {
            C.k_scale[at] = sc.k, C.v_scale[at] = sc.v;
        }
        unsigned char* ck = static_cast<unsigned char*>(C.k) + at * P * D;
        unsigned char* cv = static_cast<unsigned char*>(C.v) + at * P * D;
        static_assert(kKeyItems == 2, "bits of later");
        uint32_t later = 0; // values next to a border, 16 bits an item
#pragma unroll
        for (int n = 0; n < kKeyItems; n++) {
            const int it = gt + n * GT, u = it / strips, c = it % strips;
            if (u >= rows) {
                continue;
            }
            uint32_t w[4], beside = 0;
            const float off = moved[n] > 0.f ? kRotationOff * sc.inv_k : 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float lo[4], hi[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int i = 4 * e + j, other = kAdjacent ? i ^ 1 : i ^ 8;
                    const float m = (fabsf(x[n][i]) + fabsf(x[n][other])) * off;
                    lo[j] = fmaf(x[n][i], sc.inv_k, -m), hi[j] = fmaf(x[n][i], sc.inv_k, m);
                }
                w[e] = pack_e4m3(lo[0], lo[1], lo[2], lo[3]);
                beside |= differing(w[e], pack_e4m3(hi[0], hi[1], hi[2], hi[3])) << (4 * e);
            }
            beside = off > 0.f ? beside : 0; // other items have no pairs to rotate
            if (some_bad && (bad[group][u / 32] >> (u % 32) & 1)) {
                w[0] = w[1] = w[2] = w[3] = kNanCodes, beside = 0;
            }
            if (c < turned && !kAdjacent) {
                *reinterpret_cast<uint2*>(ck + key_offset(D, s0 + u, 8 * c)) = make_uint2(w[0], w[1]);
                *reinterpret_cast<uint2*>(ck + key_offset(D, s0 + u, 8 * c + pairs)) = make_uint2(w[2], w[3]);
            } else {
                *reinterpret_cast<uint4*>(ck + key_offset(D, s0 + u, 16 * c)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            later |= beside << (16 * n);
        }
#pragma unroll
        for (int n = 0; n < kValueItems; n++) {
            const int it = gt + n * GT, t0 = (s0 / 16 + it / (D / 2)) * 16, d = it % (D / 2) * 2;
            if (t0 >= s1) {
                continue;
            }
#pragma unroll
            for (int f = 0; f < 2; f++) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float y[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float2 a = unpack2<T>(va[n][4 * e + k]);
                        y[k] = (f ? a.y : a.x) * sc.inv_v;
                    }
                    w[e] = pack_e4m3(y[0], y[1], y[2], y[3]);
                }
                unsigned char* p = cv + value_offset(D, t0, d + f);
                if (t0 >= s0 && t0 + 16 <= s1) {
                    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
                } else { // older, new and unused slots
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        if (t0 + k >= s0 && t0 + k < s1) {
                            p[k] = (unsigned char)(w[k / 4] >> (8 * (k % 4)));
                        } else if (t0 + k < s0 && sc.lower_v < 1.f) {
                            p[k] = (unsigned char)lowered(p[k], sc.lower_v);
                        }
                    }
                }
            }
        }
        // older tokens of the page
        if (sc.lower_k < 1.f) {
#pragma unroll 1
            for (int i = gt; i < s0 * strips; i += GT) {
                uint4* p = reinterpret_cast<uint4*>(ck + key_offset(D, i / strips, i % strips * 16));
                uint4 w = *p;
                w.x = lowered(w.x, sc.lower_k), w.y = lowered(w.y, sc.lower_k), w.z = lowered(w.z, sc.lower_k), w.w = lowered(w.w, sc.lower_k);
                *p = w;
            }
        }
        if (sc.lower_v < 1.f) {
#pragma unroll 1
            for (int i = gt; i < s0 / 16 * D; i += GT) {
                uint4* p = reinterpret_cast<uint4*>(cv + i * 16);
                uint4 w = *p;
                w.x = lowered(w.x, sc.lower_v), w.y = lowered(w.y, sc.lower_v), w.z = lowered(w.z, sc.lower_v), w.w = lowered(w.w, sc.lower_v);
                *p = w;
            }
        }
        if (later) { // last, when nothing is held in registers over the call
            exact_codes<T, D, kAdjacent>(A, ck, s0, pr.row0, head, gt, GT, later, sc.inv_k);
        }
    }
}

// Many queries: beside append_pages_kernel instead of in its blocks, whose registers would leave them half of the warps. Reads and writes nothing
// that it does; the wait at the end is for what comes after both.
template <class T, bool kAdjacent>
__global__ void __launch_bounds__(kRotaryThreads, 4) query_kernel(const __grid_constant__ AppendArgs A) {
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = threadIdx.x >> 5, warps = kRotaryThreads / 32;
    rotary_warp<T, 8, kAdjacent>(A.rotation, A.q, reinterpret_cast<float2*>(smem) + warp * (A.rotation.dims / 2), int64_t(blockIdx.x) * warps + warp, int64_t(gridDim.x) * warps,
                                 query_units(A));
    wait_for_previous();
}

} // namespace seq
} // namespace cck

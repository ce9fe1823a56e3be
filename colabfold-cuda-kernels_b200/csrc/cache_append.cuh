// New keys and values into the paged cache, the keys rotated on the way, queries rotated beside them.
//
//   top = max |x| over the new rows of a (page, head);  e = smallest exponent with top <= 448 * 2^e, at least the old one where older
//   tokens share the page;  code = e4m3(x * 2^-e), nearest even
//
// A block of threads owns one (page, head): it needs all of the page's new rows before it can round the first, so that it holds them
// in shared memory, reads each row once and writes each code once. Bound by memory for prompts, by latency for single tokens.
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
};

constexpr int kAppendThreads = 256;

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

__device__ __forceinline__ bool is_finite(float x) {
    return fabsf(x) <= 3.402823466e38f;
}

template <class T, int VQ>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs A) {
    const cck_cache& C = A.cache;
    const int tid = threadIdx.x;
    if (int(blockIdx.x) >= A.kv_blocks) {
        rotary_block<T, VQ>(A.rotation, A.q, blockIdx.x - A.kv_blocks, tid, kAppendThreads);
        return;
    }
    const int D = C.dim, P = C.page_tokens;
    const int head = blockIdx.x % C.heads, unit = blockIdx.x / C.heads;
    const int b = unit / A.blocks_per_seq;
    const Sequence s = sequence_of(A.batch, b);
    const int from = max(s.place0, 0), to = s.place0 + s.rows;
    const int block = from / P + unit % A.blocks_per_seq;
    const bool first_unit = unit % A.blocks_per_seq == 0 && head == 0 && tid == 0;
    const int lo = max(from, block * P), hi = min(to, block * P + P); // places of this page's new rows
    int page = -1;
    if (lo < hi && block < A.batch.table_pages) {
        page = A.batch.table[b * A.batch.table_stride + block];
    }
    if (A.status && ((first_unit && s.cut) || (lo < hi && tid == 0 && (page < 0 || page >= C.pages)))) {
        *A.status = 1;
    }
    if (page < 0 || page >= C.pages) {
        return;
    }
    const int rows = hi - lo, s0 = lo - block * P, s1 = s0 + rows, row0 = s.row0 + lo - s.place0;
    const int64_t at = int64_t(page) * C.heads + head;

    extern __shared__ __align__(128) unsigned char smem[];
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
        const float2 cs = cos_sin(A.rotation.pos[axis_of(A.rotation, p) * A.rotation.pos_stride + row0 + u], A.rotation.freq[p]);
        float* a = fk + u * kp + (A.rotation.adjacent ? 2 * p : p);
        float* c = a + (A.rotation.adjacent ? 1 : half);
        const float2 z = rotate(*a, *c, cs);
        *a = z.x, *c = z.y;
    }
    __syncthreads();
    for (int i = tid; i < rows * D; i += kAppendThreads) {
        const int u = i / D, d = i % D;
        if (!bad[u]) {
            const float x = fabsf(fk[u * kp + d]);
            top_k = is_finite(x) ? fmaxf(top_k, x) : top_k;
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
    // the page's scales: one that older tokens use only grows
    const int ek = scale_exponent(top_k), ev = scale_exponent(top_v);
    float new_k = exp2_int(ek), new_v = exp2_int(ev);
    if (s0 > 0) {
        new_k = old_k > new_k ? old_k : new_k, new_v = old_v > new_v ? old_v : new_v;
    }
    const float lower_k = s0 > 0 && old_k > 0.f ? old_k / new_k : 1.f, lower_v = s0 > 0 && old_v > 0.f ? old_v / new_v : 1.f;
    const float inv_k = 1.f / new_k, inv_v = 1.f / new_v;
    if (tid == 0) {
        C.k_scale[at] = new_k, C.v_scale[at] = new_v;
    }
    unsigned char* ck = static_cast<unsigned char*>(C.k) + at * P * D;
    unsigned char* cv = static_cast<unsigned char*>(C.v) + at * P * D;
    auto lowered = [](uint32_t w, float f) {
        uint32_t lo2, hi2;
        unpack_e4m3(w, lo2, hi2);
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo2)), y = __half22float2(*reinterpret_cast<const __half2*>(&hi2));
        return pack_e4m3(x.x * f, x.y * f, y.x * f, y.y * f);
    };
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
    for (int i = tid; i < rows * strips; i += kAppendThreads) {
        const int u = i / strips, d = i % strips * 16;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float4 x = *reinterpret_cast<const float4*>(fk + u * kp + d + 4 * j);
            w[j] = bad[u] ? kNanCodes : pack_e4m3(x.x * inv_k, x.y * inv_k, x.z * inv_k, x.w * inv_k);
        }
        *reinterpret_cast<uint4*>(ck + key_offset(D, s0 + u, d)) = make_uint4(w[0], w[1], w[2], w[3]);
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

} // namespace seq
} // namespace cck

// What the sequence operators' kernels share: element types, the e4m3 codes and the cache's layout, a sequence's place in its batch,
// bulk copies with bounded waits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/cck_b200.h"

namespace cck {
namespace seq {

constexpr int kMinExp = -40, kMaxExp = 40; // exponents of a cache's scales
constexpr int kMostTokens = 1 << 30;       // of a sequence
constexpr int kMostHeads = 1 << 16;

__host__ __device__ constexpr int ceil_div(int a, int b) {
    return (a + b - 1) / b;
}

// ---- element types
template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(float x) {
    return x;
}
template <>
__device__ __forceinline__ float to_f32(__half x) {
    return __half2float(x);
}
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) {
    return __bfloat162float(x);
}
// rounds once, to nearest even: an output's own type
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32(float x) {
    return x;
}
template <>
__device__ __forceinline__ __half from_f32(float x) {
    return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float x) {
    return __float2bfloat16_rn(x);
}
template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};
// the same as words, which stay packed in registers
template <int kBytes>
struct alignas(kBytes) Words {
    uint32_t w[kBytes / 4];
};
template <>
struct alignas(2) Words<2> {
    uint16_t w[1];
};

// two 16-bit values of a word: kept packed, a register holds two of them
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float2 x);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float2 x) {
    const __half2 h = __float22half2_rn(x);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float2 x) {
    const __nv_bfloat162 h = __float22bfloat162_rn(x);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// N values of a vector to f32 and back
template <class T, int N>
__device__ __forceinline__ void to_floats(const Words<sizeof(T) * N>& v, float (&x)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            x[i] = __uint_as_float(v.w[i]);
        }
    } else if constexpr (N == 1) {
        x[0] = unpack2<T>(v.w[0]).x;
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const float2 y = unpack2<T>(v.w[i]);
            x[2 * i] = y.x, x[2 * i + 1] = y.y;
        }
    }
}
template <class T, int N>
__device__ __forceinline__ Words<sizeof(T) * N> from_floats(const float (&x)[N]) {
    Words<sizeof(T) * N> v;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            v.w[i] = __float_as_uint(x[i]);
        }
    } else if constexpr (N == 1) {
        v.w[0] = uint16_t(pack2<T>(make_float2(x[0], 0.f)));
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            v.w[i] = pack2<T>(make_float2(x[2 * i], x[2 * i + 1]));
        }
    }
    return v;
}

// Magnitudes of two 16-bit values a word: as signless integers they are in order, infinities and NaN above all others
__device__ __forceinline__ uint32_t largest_words(uint32_t m, uint32_t a, uint32_t b) {
    return __vimax3_s16x2(m, a & 0x7FFF7FFFu, b & 0x7FFF7FFFu);
}

// ---- e4m3
// two f32 to two codes (nearest even, saturating, NaN stays NaN): a in the low byte
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    return pack_e4m3(a, b) | pack_e4m3(c, d) << 16;
}
// four codes to two pairs of f16, exactly
__device__ __forceinline__ void unpack_e4m3(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
constexpr uint32_t kNanCodes = 0x7F7F7F7Fu;

// exponent of the smallest power of two s with top <= 448 s: 448 = 0.875 * 2^9
__device__ __forceinline__ int scale_exponent(float top) {
    if (!(top > 0.f)) {
        return kMinExp;
    }
    int x;
    const float m = frexpf(fminf(top, 3.402823466e38f), &x); // a rotation can bring finite values over the largest
    return min(max(x - 9 + (m > 0.875f ? 1 : 0), kMinExp), kMaxExp);
}
__device__ __forceinline__ float exp2_int(int e) { // |e| <= 126
    return __int_as_float((127 + e) << 23);
}

// ---- the cache's layout, in bytes inside one (page, head) block of page_tokens * dim
__host__ __device__ __forceinline__ int key_offset(int dim, int token, int d) {
    return (token >> 3) * 8 * dim + (d >> 4) * 128 + (token & 7) * 16 + (d & 15);
}
__host__ __device__ __forceinline__ int value_offset(int dim, int token, int d) {
    return (token >> 4) * 16 * dim + d * 16 + (token & 15);
}

// ---- a sequence of the batch, as its arrays say; whatever they hold, rows stay inside the tensors
struct Sequence {
    int row0, rows; // newest rows: row0 .. row0 + rows - 1
    int place0;     // of the first of them (negative: there are more rows than the length has places)
    int len;        // with them
    bool cut;       // something of it lies outside batch.rows, max_new or its length
};
__device__ __forceinline__ Sequence sequence_of(const cck_batch& b, int i) {
    Sequence s;
    const int first = b.first[i], all = b.first[i + 1] - first;
    s.row0 = first, s.len = min(max(b.len[i], 0), kMostTokens), s.place0 = s.len - all;
    s.rows = first < 0 || first > b.rows ? 0 : max(0, min(all, min(b.max_new, b.rows - first)));
    s.cut = s.rows != all || s.place0 < 0 || s.len != b.len[i];
    return s;
}

// ---- bulk copies and their mbarriers
__device__ __forceinline__ uint32_t shared_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void bar_init_done() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// contiguous bytes (a multiple of 16, both ends 16-byte aligned) to shared memory
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(__cvta_generic_to_global(src)), "r"(bytes), "r"(bar)
                 : "memory");
}
// Waits for the phase with this parity; gives up (false) after about a second, which nothing but a lost copy can cause, or after `tries` times 4 us.
constexpr int kWaitTries = 1 << 18, kDrainTries = 1 << 12; // kDrainTries: for copies that are on their way when another one got lost
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, int tries = kWaitTries) {
#pragma unroll 1
    for (int i = 0; i < tries; i++) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity), "r"(4000)
            : "memory");
        if (ok) {
            return true;
        }
    }
    return false;
}

// ---- dependent launches of one call: the second kernel may start while the first drains, and waits for its writes
__device__ __forceinline__ void let_next_start() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

} // namespace seq
} // namespace cck

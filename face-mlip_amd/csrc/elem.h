// Element types of the expert layer's operators (norm.hip, route.hip, grouped.h): rows in fp32, bf16,
// fp16 or e4m3 memory, arithmetic in fp32. A piece is eight neighbouring elements of a row, moved with
// 16-byte accesses whatever the row's alignment (gfx950 takes them at any element address), the
// last one of a row that is no multiple of eight element by element.
#pragma once
#include "common.h"

namespace face {

constexpr int kPiece = 8;

typedef v4u v4u_any __attribute__((aligned(1)));
typedef _Float16 f16;
typedef __bf16 bf16;

template <typename T>
__device__ __forceinline__ v4u ld16(const T* p) {
    return *reinterpret_cast<const v4u_any*>(p);
}
template <typename T>
__device__ __forceinline__ void st16(T* p, v4u v) {
    *reinterpret_cast<v4u_any*>(p) = v;
}

// Rounding to a 16-bit type is to nearest, ties to even; fp32 passes through.
template <typename T>
__device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f(float v) { return (T)v; }

// One value of two 16-bit halves each, as the row holds them.
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t u, float& a, float& b) {
    typedef T v2 __attribute__((ext_vector_type(2)));
    const v2 h = __builtin_bit_cast(v2, u);
    a = (float)h[0];
    b = (float)h[1];
}
template <>
__device__ __forceinline__ void unpack2<bf16>(uint32_t u, float& a, float& b) {
    a = __builtin_bit_cast(float, u << 16);
    b = __builtin_bit_cast(float, u & 0xffff0000u);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef T v2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){a, b}, v2));
}

// x sigmoid(x) and its slope s (1 + x (1 - s)). Beyond 87, where a float32 sigmoid (or one minus it) leaves the normal
// range, the factor is 0 and not its value at the cut, which x would make a result of (-3e38 times 1.6e-38); what is dropped
// is below 87 e^-87 = 2^-119. Two instructions; the factor itself beyond the cut, by another exponential, took 13 to 25 % more
// of a 16-bit product's time.
constexpr float kSiluCut = 87.f;
__device__ __forceinline__ float silu(float x) {
    float rest;
    const float s = gemm_sigmoid(x, rest, kSiluCut);
    return x * (x < -kSiluCut ? 0.f : s);
}
__device__ __forceinline__ float silu_slope(float x) {
    float rest;
    const float s = gemm_sigmoid(x, rest, kSiluCut);
    return (x < -kSiluCut ? 0.f : s) * fmaf(x, x > kSiluCut ? 0.f : rest, 1.f);
}

// x[0..7] = the elements [0, left) of the piece at p, zero beyond (left <= 0: none is read).
template <typename T>
__device__ __forceinline__ void load_piece(const T* p, int left, float x[kPiece]) {
    if (left >= kPiece) {
        if constexpr (sizeof(T) == 4) {
            const v4f a = __builtin_bit_cast(v4f, ld16(p)), b = __builtin_bit_cast(v4f, ld16(p + 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = a[e];
                x[4 + e] = b[e];
            }
        } else {
            const v4u a = ld16(p);
#pragma unroll
            for (int e = 0; e < 4; ++e) unpack2<T>(a[e], x[2 * e], x[2 * e + 1]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e) x[e] = e < left ? to_f(p[e]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, int left, const float x[kPiece]) {
    if (left >= kPiece) {
        if constexpr (sizeof(T) == 4) {
            st16(p, __builtin_bit_cast(v4u, (v4f){x[0], x[1], x[2], x[3]}));
            st16(p + 4, __builtin_bit_cast(v4u, (v4f){x[4], x[5], x[6], x[7]}));
        } else {
            v4u a;
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = pack2<T>(x[2 * e], x[2 * e + 1]);
            st16(p, a);
        }
    } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e)
            if (e < left) p[e] = from_f<T>(x[e]);
    }
}

// Calls f(T{}) for the element type that `dtype` names, FACE_ERR_ARG for another.
template <typename Fn>
static inline int with_dtype(int dtype, Fn f) {
    switch (dtype) {
        case FACE_F32: return f(float{});
        case FACE_BF16: return f(bf16{});
        case FACE_F16: return f(f16{});
        default: return FACE_ERR_ARG;
    }
}

// Rows of a row-wise kernel: `lanes` threads work on one row, each on up to kRowUnits pieces that it keeps
// from the first read to the last store, so that a row is read once: in registers, but for part of the rows of a
// workgroup of 1024 (norm.hip). Few lanes for short rows (four rows to a wave), that workgroup for the longest.
constexpr int kRowUnits = 8;
struct RowShape {
    int lanes, units;
};
static inline RowShape row_shape(int64_t width) {
    const int64_t p = (width + kPiece - 1) / kPiece;
    const int lanes = p <= 32 ? 16 : (p <= 64 * kRowUnits ? 64 : (p <= 256 * kRowUnits ? 256 : 1024));
    const int64_t u = (p + lanes - 1) / lanes;
    return {lanes, (int)(u <= 6 ? u : 8)};
}
constexpr int64_t kRowMax = (int64_t)1024 * kRowUnits * kPiece;

// Sum over the LANES threads of a row, the same in each of them. `part` is LDS of LANES / 64 floats (rows
// of more than a wave; every thread of the workgroup calls it then).
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* part) {
    if constexpr (LANES == 16) return row16_sum(v);
    v = group_sum(v, kWave);
    if constexpr (LANES > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
        for (int i = 0; i < LANES / 64; ++i) v += part[i];
    }
    return v;
}
// Largest of unsigned values, likewise.
template <int LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t v, float* part) {
    constexpr int W = LANES < 64 ? LANES : 64;
    for (int o = W >> 1; o > 0; o >>= 1) {
        const uint32_t w = (uint32_t)__shfl_xor((int)v, o, kWave);
        v = w > v ? w : v;
    }
    if constexpr (LANES > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = __builtin_bit_cast(float, v);
        __syncthreads();
        for (int i = 0; i < LANES / 64; ++i) {
            const uint32_t w = __builtin_bit_cast(uint32_t, part[i]);
            v = w > v ? w : v;
        }
    }
    return v;
}

// out (N, F) of `dtype` = sums of k neighbouring fp32 rows (N k, F), in order (route.hip).
int sum_slot_rows(const float* rows, int64_t N, int k, int F, int dtype, void* out, hipStream_t st);

}  // namespace face

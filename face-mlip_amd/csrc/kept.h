// Rows kept in 8 bits: e4m3 with a power of two for each 32 neighbouring columns of a row.
//
//   e = the least with max|x| <= 448 2^e over the block's finite values (2^e >= 2^-126),  q = e4m3(x 2^-e)
//
// The scale is a byte, e + 127, which is a float's exponent field: x 2^-e and q 2^e are exact, so what a value is
// kept as hangs on no order of operations, and the rounding to e4m3 (to nearest, ties to even, half a step 2^-4) is the only
// one. It may pass a type's largest value by half a step: what it stands for is cut to that. A NaN or an infinity is kept as NaN
// and leaves the others of its block as they are. A block's 32 columns lie in a quad
// of lanes, a piece each: its maximum is two cross-lane moves.
#pragma once
#include "elem.h"

namespace face {

constexpr int kKeptBlock = 32;
static __host__ __device__ __forceinline__ int64_t kept_blocks(int64_t F) { return (F + kKeptBlock - 1) / kKeptBlock; }

// The scale's byte of the quad's 32 values (zeros beyond the row's end). All lanes of a quad are active.
__device__ __forceinline__ uint32_t kept_scale(const float x[kPiece]) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < kPiece; ++e) {
        const uint32_t m = __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu;
        top = m < 0x7f800000u && m > top ? m : top;
    }
    const uint32_t a = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false);   // lane ^ 1
    top = a > top ? a : top;
    const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false);   // lane ^ 2
    top = b > top ? b : top;
    const int s = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u);     // 448 = 1.75 2^8
    return (uint32_t)(s < 1 ? 1 : s);
}

// Eight values times `inv` in e4m3. The instruction turns what rounds past 448 (infinities) into NaN.
template <bool NT = false>
__device__ __forceinline__ void store_e4m3(uint8_t* p, int left, const float x[kPiece], float inv) {
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[4] * inv, x[5] * inv, 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[6] * inv, x[7] * inv, hi, true);
    if (left >= kPiece) {
        typedef int v2i_any __attribute__((ext_vector_type(2), aligned(1)));
        if constexpr (NT) __builtin_nontemporal_store((v2i_any){lo, hi}, reinterpret_cast<v2i_any*>(p));
        else *reinterpret_cast<v2i_any*>(p) = (v2i_any){lo, hi};
    } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e)
            if (e < left) p[e] = (uint8_t)((uint32_t)(e < 4 ? lo : hi) >> (8 * (e & 3)));
    }
}

// Piece c / 8 of a row: its eight bytes at q + c, and its block's scale, written by the first lane of the quad.
template <bool NT = false>
__device__ __forceinline__ void store_kept(uint8_t* q, uint8_t* scale, int c, int F, const float x[kPiece]) {
    const uint32_t s = kept_scale(x);
    store_e4m3<NT>(q + c, F - c, x, __builtin_bit_cast(float, (254u - s) << 23));
    if ((c & (kKeptBlock - 1)) == 0 && c < F) scale[c / kKeptBlock] = (uint8_t)s;
}

// v within [-top, top]; a NaN stays one.
__device__ __forceinline__ float within(float v, float top) { return v > top ? top : (v < -top ? -top : v); }

// A kept piece on its way: its bytes and its scale.
struct KeptPiece {
    uint32_t lo, hi, scale;
};
template <bool NT = false>
__device__ __forceinline__ KeptPiece hold_kept(const uint8_t* q, const uint8_t* scale, int c, int F) {
    KeptPiece k = {0, 0, 0};
    if (c + kPiece <= F) {
        typedef uint32_t v2u_any __attribute__((ext_vector_type(2), aligned(1)));
        const v2u_any* p = reinterpret_cast<const v2u_any*>(q + c);
        const v2u_any v = NT ? __builtin_nontemporal_load(p) : *p;
        k.lo = v[0];
        k.hi = v[1];
    } else if (c < F) {
#pragma unroll
        for (int e = 0; e < kPiece; ++e)
            if (c + e < F) (e < 4 ? k.lo : k.hi) |= (uint32_t)q[c + e] << (8 * (e & 3));
    }
    if (c < F) k.scale = scale[c / kKeptBlock];
    return k;
}
// Its values at scale s; zeros beyond the row's end.
__device__ __forceinline__ void kept_values_at(const KeptPiece& k, float s, float x[kPiece]) {
    const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8((int)k.lo, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)k.lo, true);
    const v2f c = __builtin_amdgcn_cvt_pk_f32_fp8((int)k.hi, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)k.hi, true);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        x[e] = a[e] * s;
        x[2 + e] = b[e] * s;
        x[4 + e] = c[e] * s;
        x[6 + e] = d[e] * s;
    }
}
// Those of a row that a kernel kept, far from the largest float.
__device__ __forceinline__ void kept_values_near(const KeptPiece& k, float x[kPiece]) {
    kept_values_at(k, __builtin_bit_cast(float, k.scale << 23), x);
}
// Those of any row. Of the scales that store_kept does not write, 0 stands for 2^-127 and 255 for NaN.
__device__ __forceinline__ void kept_values(const KeptPiece& k, float x[kPiece]) {
    kept_values_at(k, __builtin_bit_cast(float, k.scale - 1 < 254u ? k.scale << 23 : (k.scale ? 0x7fc00000u : 0x00400000u)), x);
    if (k.scale >= 247u) {                       // 256 2^120: what the largest floats round to
#pragma unroll
        for (int e = 0; e < kPiece; ++e) x[e] = within(x[e], 0x1.fffffep127f);
    }
}

// Rows that a call reads or writes once pass the caches by where the call moves more than they hold (NT): 1 M rows of 256
// bytes written, then 1 M gathered, take 140 us with ordinary accesses, 87 us with these.
template <bool NT, typename T>
__device__ __forceinline__ v4u ld16s(const T* p) {
    if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const v4u_any*>(p));
    return ld16(p);
}
template <bool NT, typename T>
__device__ __forceinline__ void st16s(T* p, v4u v) {
    if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<v4u_any*>(p));
    else st16(p, v);
}
constexpr int64_t kStreamBytes = (int64_t)256 << 20;                 // the last level of cache
// Whether a call that moves n elements of T in pieces of eight does. bf16, both ways (us): norm of 64 MB rows (256 MB in all)
// 53 for 51 with ordinary accesses, of 96 MB 75 for 82, of 256 MB 185 for 197; a gate that keeps 128 MB rows 104 for 100, 192 MB
// 151 for 157. Not in fp32, whose piece is two accesses that each cover half of a stretch of memory: 24,000 x 1440, forward
// 124 us for 112, unpacked 42 for 31.
template <typename T>
static inline bool streams(int64_t n) { return sizeof(T) == 2 && n * (int64_t)sizeof(T) > kStreamBytes; }
// load_piece and store_piece of such rows.
template <bool NT, typename T>
__device__ __forceinline__ void load_row(const T* p, int left, float x[kPiece]) {
    if (NT && left >= kPiece) {
        if constexpr (sizeof(T) == 4) {
            const v4f a = __builtin_bit_cast(v4f, ld16s<NT>(p)), b = __builtin_bit_cast(v4f, ld16s<NT>(p + 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = a[e];
                x[4 + e] = b[e];
            }
        } else {
            const v4u a = ld16s<NT>(p);
#pragma unroll
            for (int e = 0; e < 4; ++e) unpack2<T>(a[e], x[2 * e], x[2 * e + 1]);
        }
    } else {
        load_piece(p, left, x);
    }
}
template <bool NT, typename T>
__device__ __forceinline__ void store_row(T* p, int left, const float x[kPiece]) {
    if (NT && left >= kPiece) {
        if constexpr (sizeof(T) == 4) {
            st16s<NT>(p, __builtin_bit_cast(v4u, (v4f){x[0], x[1], x[2], x[3]}));
            st16s<NT>(p + 4, __builtin_bit_cast(v4u, (v4f){x[4], x[5], x[6], x[7]}));
        } else {
            v4u a;
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = pack2<T>(x[2 * e], x[2 * e + 1]);
            st16s<NT>(p, a);
        }
    } else {
        store_piece(p, left, x);
    }
}

// A piece of a row in its memory's type, on its way: half the registers of its values where they are 16-bit.
template <typename T>
struct RawPiece {
    v4u a[sizeof(T) / 2];
};
template <bool NT = false, typename T>
__device__ __forceinline__ RawPiece<T> hold_raw(const T* p, int left) {
    RawPiece<T> r = {};
    if (left >= kPiece) {
        r.a[0] = ld16s<NT>(p);
        if constexpr (sizeof(T) == 4) r.a[1] = ld16s<NT>(p + 4);
    } else if (left > 0) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < kPiece; ++e)
                if (e < left) r.a[e >> 2][e & 3] = __builtin_bit_cast(uint32_t, p[e]);
        } else {
#pragma unroll
            for (int e = 0; e < kPiece; ++e)
                if (e < left) r.a[0][e >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, p[e]) << (16 * (e & 1));
        }
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void raw_values(const RawPiece<T>& r, float x[kPiece]) {
    if constexpr (sizeof(T) == 4) {
        const v4f a = __builtin_bit_cast(v4f, r.a[0]), b = __builtin_bit_cast(v4f, r.a[1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = a[e];
            x[4 + e] = b[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) unpack2<T>(r.a[0][e], x[2 * e], x[2 * e + 1]);
    }
}

// Sum over a wave in a fixed order, the same in every lane, without a trip through LDS.
__device__ __forceinline__ float wave_sum(float v) {
    v = row16_sum(v);
    const int i = __builtin_bit_cast(int, v);
    const float a = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 0));
    const float b = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 16));
    const float c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 32));
    const float d = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 48));
    return (a + b) + (c + d);
}
// Sums of two values over the LANES threads of a row (row_sum of elem.h for two). `part`: LDS, LANES / 32 floats.
template <int LANES>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* part) {
    if constexpr (LANES == 16) {
        a = row16_sum(a);
        b = row16_sum(b);
        return;
    }
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (LANES > 64) {
        constexpr int W = LANES / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            part[threadIdx.x >> 6] = a;
            part[W + (threadIdx.x >> 6)] = b;
        }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            a += part[i];
            b += part[W + i];
        }
    }
}

}  // namespace face

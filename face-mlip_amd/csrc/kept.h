// Rows kept in 8 bits: e4m3 with a power of two for each 32 neighbouring columns of a row.
//
//   e = the least with max|x| <= 448 2^e over the block's finite values (2^e >= 2^-126),  q = e4m3(x 2^-e)
//
// The scale is a byte, e + 127, which is a float's exponent field: x 2^-e and q 2^e are exact, so what a value is
// kept as hangs on no order of operations, and the rounding to e4m3 (to nearest, ties to even, half a step 2^-4) is the only
// one. It may pass a type's largest value by half a step: what it stands for is cut to that. A NaN or an infinity is kept as NaN
// and leaves the others of its block as they are. A block's 32 columns lie in 4 or
// 8 lanes side by side: its maximum is two or three cross-lane moves.
#pragma once
#include <type_traits>

#include "elem.h"

namespace face {

constexpr int kKeptBlock = 32;
static __host__ __device__ __forceinline__ int64_t kept_blocks(int64_t F) { return (F + kKeptBlock - 1) / kKeptBlock; }

// A lane has E values, 4 or 8, so that 32 / E lanes side by side have a block; all of them are active.
// The scale's byte of the lanes' 32 values (zeros beyond the row's end).
template <int E>
__device__ __forceinline__ uint32_t kept_scale(const float x[E]) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const uint32_t m = __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu;
        top = m < 0x7f800000u && m > top ? m : top;
    }
    auto step = [&](uint32_t v) { top = v > top ? v : top; };
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));              // lane ^ 1
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));              // lane ^ 2
    if constexpr (E == 4) step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x141, 0xF, 0xF, false));   // the other quad
    const int s = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u);                         // 448 = 1.75 2^8
    return (uint32_t)(s < 1 ? 1 : s);
}

// E values times `inv` in e4m3, to the bytes [c, c + E) of a row of F. The instruction turns what rounds past 448
// (infinities) into NaN.
template <int E, bool NT, bool CUT>
__device__ __forceinline__ void store_e4m3(uint8_t* row, int c, int F, const float x[E], float inv) {
    typedef uint32_t words __attribute__((ext_vector_type(E / 4)));
    typedef words words_any __attribute__((aligned(1)));
    typedef uint32_t u_any __attribute__((aligned(1)));
    typedef uint16_t s_any __attribute__((aligned(1)));
    uint32_t v[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
        v[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, lo, true);
    }
    const int left = F - c;
    uint8_t* p = row + c;
    if (left >= E) {
        words w;
#pragma unroll
        for (int i = 0; i < E / 4; ++i) w[i] = v[i];
        if constexpr (NT) __builtin_nontemporal_store(w, reinterpret_cast<words_any*>(p));
        else *reinterpret_cast<words_any*>(p) = w;
    } else if (CUT && left > 0) {
        uint32_t w = v[0];
        if constexpr (E == 8) {
            if (left & 4) *(u_any*)p = w;
            w = left & 4 ? v[1] : w;
        }
        if (left & 2) *(s_any*)(p + (left & 4)) = (uint16_t)w;
        if (left & 1) p[left & 6] = (uint8_t)(left & 2 ? w >> 16 : w);
    }
}

// The lane's columns from c on of a row: their bytes at q + c, and the block's scale, written by its first lane.
template <int E, bool NT, bool CUT>
__device__ __forceinline__ void store_kept(uint8_t* q, uint8_t* scale, int c, int F, const float x[E]) {
    const uint32_t s = kept_scale<E>(x);
    store_e4m3<E, NT, CUT>(q, c, F, x, __builtin_bit_cast(float, (254u - s) << 23));
    if ((c & (kKeptBlock - 1)) == 0 && c < F) scale[c / kKeptBlock] = (uint8_t)s;
}

// v within [-top, top]; a NaN stays one.
__device__ __forceinline__ float within(float v, float top) { return v > top ? top : (v < -top ? -top : v); }

// Kept values on their way: their bytes and their scale.
template <int E>
struct KeptPiece {
    uint32_t v[E / 4], scale;
    int s;                             // bits that they are to be shifted by: the row's last E bytes
};
template <int E, bool NT, bool CUT>
__device__ __forceinline__ KeptPiece<E> hold_kept(const uint8_t* q, const uint8_t* scale, int c, int F) {
    typedef uint32_t words __attribute__((ext_vector_type(E / 4)));
    typedef words words_any __attribute__((aligned(1)));
    KeptPiece<E> k = {};
    if (!CUT || F >= E) {
        if (c < F) {
            const int at = !CUT || c + E <= F ? c : F - E;
            const words_any* p = reinterpret_cast<const words_any*>(q + at);
            const words w = NT ? __builtin_nontemporal_load(p) : *p;
#pragma unroll
            for (int i = 0; i < E / 4; ++i) k.v[i] = w[i];
            k.s = 8 * (c - at);
        }
    } else if (c == 0) {
#pragma unroll
        for (int e = 0; e < E - 1; ++e)
            if (e < F) k.v[e / 4] |= (uint32_t)q[e] << (8 * (e & 3));
    }
    if (c < F) k.scale = scale[c / kKeptBlock];
    return k;
}
// The values at scale s; zeros beyond the row's end.
template <int E>
__device__ __forceinline__ void kept_values_at(const KeptPiece<E>& k, float s, float x[E]) {
    uint32_t w[2] = {k.v[0], E == 8 ? k.v[E / 4 - 1] : 0};
    if (k.s) {
        const uint64_t v = ((uint64_t)w[1] << 32 | w[0]) >> k.s;
        w[0] = (uint32_t)v;
        w[1] = (uint32_t)(v >> 32);
    }
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
        const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
        x[4 * i] = a[0] * s;
        x[4 * i + 1] = a[1] * s;
        x[4 * i + 2] = b[0] * s;
        x[4 * i + 3] = b[1] * s;
    }
}
// Those of a row that a kernel kept, far from the largest float.
template <int E>
__device__ __forceinline__ void kept_values_near(const KeptPiece<E>& k, float x[E]) {
    kept_values_at(k, __builtin_bit_cast(float, k.scale << 23), x);
}
// Those of any row. Of the scales that store_kept does not write, 0 stands for 2^-127 and 255 for NaN.
template <int E>
__device__ __forceinline__ void kept_values(const KeptPiece<E>& k, float x[E]) {
    kept_values_at(k, __builtin_bit_cast(float, k.scale - 1 < 254u ? k.scale << 23 : (k.scale ? 0x7fc00000u : 0x00400000u)), x);
    if (k.scale >= 247u) {                       // 256 2^120: what the largest floats round to
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = within(x[e], 0x1.fffffep127f);
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
// f(NT, CUT) as types, for a kernel that is launched in all four forms.
template <typename Fn>
static inline void with_forms(bool nt, bool cut, Fn f) {
    if (nt) cut ? f(std::true_type{}, std::true_type{}) : f(std::true_type{}, std::false_type{});
    else cut ? f(std::false_type{}, std::true_type{}) : f(std::false_type{}, std::false_type{});
}
constexpr int64_t kStreamBytes = (int64_t)256 << 20;                 // the last level of cache
// Whether a call that moves n elements of T does. bf16, both ways (us): norm of 64 MB rows (256 MB in all)
// 53 for 51 with ordinary accesses, of 96 MB 75 for 82, of 256 MB 185 for 197; a gate that keeps 128 MB rows 104 for 100, 192 MB
// 151 for 157. Only where neighbouring lanes' accesses lie side by side: with fp32 rows in pieces of eight, two accesses that
// each cover half of a stretch of memory, the norm of 24,000 x 1440 took 124 us for 112.
template <typename T>
static inline bool streams(int64_t n) { return n * (int64_t)sizeof(T) > kStreamBytes; }

// Sixteen bytes of a row, so that neighbouring lanes move neighbouring bytes whatever the type: columns [c, c + E) of F, zeros
// beyond. CUT: rows of any width; what ends before the sixteen bytes do is read as the row's last sixteen and shifted by `s` bits
// when its values are asked for, so that no load waits for another (element by element, 77,737 x 2876 fp16, norm kept in 8 bits,
// both directions, took 1269 us for 934). Only a row that is shorter than that goes by elements. Not CUT: whole multiples.
template <typename T>
struct Sixteen {
    static constexpr int E = 16 / (int)sizeof(T);
    v4u a;
    int s;
};
template <bool NT, bool CUT, typename T>
__device__ __forceinline__ Sixteen<T> hold16(const T* row, int c, int F) {
    constexpr int E = Sixteen<T>::E;
    Sixteen<T> r = {};
    if constexpr (!CUT) {
        if (c < F) r.a = ld16s<NT>(row + c);
    } else if (F >= E) {
        if (c < F) {
            const int at = c + E <= F ? c : F - E;
            r.a = ld16s<NT>(row + at);
            r.s = 8 * (int)sizeof(T) * (c - at);
        }
    } else if (c == 0) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < F) r.a[e] = __builtin_bit_cast(uint32_t, row[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 7; ++e)
                if (e < F) r.a[e >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, row[e]) << (16 * (e & 1));
        }
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void values16(const Sixteen<T>& r, float x[Sixteen<T>::E]) {
    v4u a = r.a;
    if (r.s) {                                   // 16 .. 112
        typedef uint64_t v2l __attribute__((ext_vector_type(2)));
        const v2l v = __builtin_bit_cast(v2l, a);
        const uint64_t lo = v[0], hi = v[1];
        a = __builtin_bit_cast(v4u, r.s >= 64 ? (v2l){hi >> (r.s - 64), 0} : (v2l){lo >> r.s | hi << (64 - r.s), hi >> r.s});
    }
    if constexpr (sizeof(T) == 4) {
        const v4f v = __builtin_bit_cast(v4f, a);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) unpack2<T>(a[e], x[2 * e], x[2 * e + 1]);
    }
}
template <bool NT, bool CUT, typename T>
__device__ __forceinline__ void load16(const T* row, int c, int F, float x[Sixteen<T>::E]) {
    values16<T>(hold16<NT, CUT>(row, c, F), x);
}
// To columns [c, c + E) of a row of F: what ends before in accesses of eight, four and two bytes.
template <bool NT, bool CUT, typename T>
__device__ __forceinline__ void store16(T* row, int c, int F, const float x[Sixteen<T>::E]) {
    typedef uint32_t v2u_any __attribute__((ext_vector_type(2), aligned(1)));
    typedef uint32_t u_any __attribute__((aligned(1)));
    typedef uint16_t s_any __attribute__((aligned(1)));
    const int left = F - c;
    v4u a;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 4) a[e] = __builtin_bit_cast(uint32_t, x[e]);
        else a[e] = pack2<T>(x[2 * e], x[2 * e + 1]);
    }
    if (left >= Sixteen<T>::E) {
        st16s<NT>(row + c, a);
    } else if (CUT && left > 0) {
        char* p = (char*)(row + c);
        const int n = left * (int)sizeof(T);
        if (n & 8) *(v2u_any*)p = (v2u_any){a[0], a[1]};
        const uint32_t w = n & 8 ? a[2] : a[0];
        if (n & 4) *(u_any*)(p + (n & 8)) = w;
        if constexpr (sizeof(T) == 2) {
            const uint32_t h = n & 8 ? a[3] : a[1];
            if (n & 2) *(s_any*)(p + (n & 12)) = (uint16_t)(n & 4 ? h : w);
        }
    }
}

// Workgroups in two dimensions: one of them holds fewer than 2^32 threads.
static inline dim3 row_grid(int64_t blocks) {
    constexpr int64_t kSide = 1 << 22;
    return blocks <= kSide ? dim3((unsigned)blocks) : dim3((unsigned)kSide, (unsigned)((blocks + kSide - 1) / kSide));
}
__device__ __forceinline__ int64_t row_block() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

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

// Root-mean-square norm of atom rows with the residual's addition, its backward, and rows in 8 bits:
//
//   s = x + r (rounded to the rows' type, as the residual stream holds it),  y = s w / sqrt(mean(s^2) + eps)
//   q = e4m3(y / scale),  scale = max(max|y| / 448, 2^-126) per row
//   ds = rstd (g - s rstd^2 mean(g s)) + ds_in,  g = dy w,  rstd = 1 / sqrt(mean(s^2) + eps)
//   dw = sum over rows of dy s rstd
//
// Everything between the first read of a row and its last store is fp32 in registers (up to 16384 columns); the statistics
// of the backward are formed again from s, which it has to read anyway, so that nothing but s is kept. Bound by
// bytes: a row is read once and each result written once. The sum is normalised as it was rounded: the
// backward reads that value, and the next layer's residual starts from it.
// A row lies in the registers of 16 lanes up to 256 columns, of a wave up to 4096, of four up to 16384. Longer ones are
// shared by 16 waves, which leaves 128 registers to a lane: the backward spills 13 to 648 of them to scratch, the forward 4 to
// 246 from 40,961 columns on.
// 24,000 x 1440 fp32 with the residual: forward 100 us, backward 121 + 5 us (4.9 TB/s of what they must move, as a large copy);
// 100,000 x 2304 bf16 to 8 bits 359 us (4.5 TB/s), in 16 bits forward 382 us (4.8 TB/s), backward 644 us (2.9 TB/s); 21 x 864
// 3.2 us, the launch. TB/s of long bf16 rows, forward / backward: 16,384 columns 4.6 / 1.7, 32,768 5.0 / 1.2, 65,536 3.0 / 0.5.
#include "elem.h"

namespace face {

constexpr float kE4m3Max = 448.f;
constexpr float kScaleMin = 0x1p-126f;          // smallest normal: the scale of a row of zeros

enum { kNorm = 0, kNormQ8 = 1, kQ8 = 2, kQ8Silu = 3 };

// Eight values in e4m3 (to nearest, ties to even; a NaN stays one). The instruction turns what rounds past 448
// into NaN; |y| / scale is at most 448 up to rounding, which rounds back to 448.
__device__ __forceinline__ void store_q8(uint8_t* p, int left, const float x[kPiece], float inv) {
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[4] * inv, x[5] * inv, 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[6] * inv, x[7] * inv, hi, true);
    if (left >= kPiece) {
        typedef int v2i_a1 __attribute__((ext_vector_type(2), aligned(1)));
        *reinterpret_cast<v2i_a1*>(p) = (v2i_a1){lo, hi};
    } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e)
            if (e < left) p[e] = (uint8_t)((uint32_t)(e < 4 ? lo : hi) >> (8 * (e & 3)));
    }
}

template <typename T, int LANES, int U, int MODE>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void rms_norm_fwd_kernel(
    const T* __restrict__ x, int64_t ld_x, const T* __restrict__ r, int64_t ld_r, int64_t N, int F,
    const T* __restrict__ w, float eps, T* __restrict__ y, T* __restrict__ s, uint8_t* __restrict__ q,
    float* __restrict__ scale) {
    constexpr int kThreads = LANES > 256 ? LANES : 256, kRows = kThreads / LANES;
    __shared__ float part[LANES / 64 + 1];
    const int lane = threadIdx.x % LANES;
    const int64_t n = (int64_t)blockIdx.x * kRows + threadIdx.x / LANES;
    if (n >= N) return;                          // a whole row's threads; rows of several waves have a workgroup each
    const T* xr = x + n * ld_x;
    const T* rr = r + n * ld_r;
    float v[U][kPiece];
    float ss = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = kPiece * (lane + LANES * u);
        load_piece(xr + c, F - c, v[u]);
    }
    if (r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = kPiece * (lane + LANES * u);
            float b[kPiece];
            load_piece(rr + c, F - c, b);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) v[u][e] = to_f(from_f<T>(v[u][e] + b[e]));
            store_piece(s + n * F + c, F - c, v[u]);
        }
    }
    float rs = 1.f;
    if constexpr (MODE <= kNormQ8) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < kPiece; ++e) ss = fmaf(v[u][e], v[u][e], ss);
        rs = 1.f / sqrtf(row_sum<LANES>(ss, part) / (float)F + eps);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = kPiece * (lane + LANES * u);
            float g[kPiece];
            load_piece(w + c, F - c, g);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) v[u][e] = v[u][e] * rs * g[e];
        }
    } else if constexpr (MODE == kQ8Silu) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < kPiece; ++e) v[u][e] = silu(v[u][e]);
    }
    if constexpr (MODE == kNorm) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = kPiece * (lane + LANES * u);
            store_piece(y + n * F + c, F - c, v[u]);
        }
    } else {
        // the magnitudes compare as integers, a NaN above everything: its row gets a NaN scale and no number
        uint32_t top = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                const uint32_t m = __builtin_bit_cast(uint32_t, v[u][e]) & 0x7fffffffu;
                top = m > top ? m : top;
            }
        const float amax = __builtin_bit_cast(float, row_max<LANES>(top, part));
        float sc = amax / kE4m3Max;
        if (sc < kScaleMin) sc = kScaleMin;
        const float inv = 1.f / sc;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = kPiece * (lane + LANES * u);
            store_q8(q + n * F + c, F - c, v[u], inv);
        }
        if (lane == 0) scale[n] = sc;
    }
}

// A workgroup takes rows blockIdx, blockIdx + grid, ... and keeps its columns' sums of dw in registers over
// all of them; its row of partial sums goes to `part_w` (grid, F), joined by column_sum_kernel in a fixed
// order: no atomics.
template <typename T, int LANES, int U>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void rms_norm_bwd_kernel(
    const T* __restrict__ s, int64_t ld_s, const T* __restrict__ dy, int64_t ld_dy, const T* __restrict__ ds_in,
    int64_t ld_ds, int64_t N, int F, const T* __restrict__ w, float eps, T* __restrict__ dx, float* __restrict__ part_w) {
    constexpr int kThreads = LANES > 256 ? LANES : 256, kRows = kThreads / LANES;
    __shared__ float part[LANES / 64 + 1];
    __shared__ float sums[kRows > 1 ? LANES * U * kPiece : 1];
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
    float acc[U][kPiece];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < kPiece; ++e) acc[u][e] = 0.f;
    for (int64_t n = (int64_t)blockIdx.x * kRows + slot; n < N; n += (int64_t)gridDim.x * kRows) {
        float v[U][kPiece], g[U][kPiece];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = kPiece * (lane + LANES * u);
            load_piece(s + n * ld_s + c, F - c, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = kPiece * (lane + LANES * u);
            if (dy)
                load_piece(dy + n * ld_dy + c, F - c, g[u]);
            else
#pragma unroll
                for (int e = 0; e < kPiece; ++e) g[u][e] = 0.f;
        }
        float ss = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < kPiece; ++e) ss = fmaf(v[u][e], v[u][e], ss);
        const float rs = 1.f / sqrtf(row_sum<LANES>(ss, part) / (float)F + eps);
        float gs = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = kPiece * (lane + LANES * u);
            float b[kPiece];
            load_piece(w + c, F - c, b);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                acc[u][e] = fmaf(g[u][e], v[u][e] * rs, acc[u][e]);
                g[u][e] *= b[e];
                gs = fmaf(g[u][e], v[u][e], gs);
            }
        }
        const float m = row_sum<LANES>(gs, part) / (float)F * rs * rs;
        if (dx) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = kPiece * (lane + LANES * u);
                float b[kPiece];
                if (ds_in)
                    load_piece(ds_in + n * ld_ds + c, F - c, b);
                else
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) b[e] = 0.f;
#pragma unroll
                for (int e = 0; e < kPiece; ++e) b[e] += rs * (g[u][e] - v[u][e] * m);
                store_piece(dx + n * F + c, F - c, b);
            }
        }
    }
    if (!part_w) return;
    if constexpr (kRows > 1) {
        for (int k = 0; k < kRows; ++k) {
            __syncthreads();
            if (slot == k) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) {
                        float& t = sums[(u * kPiece + e) * LANES + lane];
                        t = k ? t + acc[u][e] : acc[u][e];
                    }
            }
        }
        if (slot != kRows - 1) return;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < kPiece; ++e) acc[u][e] = sums[(u * kPiece + e) * LANES + lane];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = kPiece * (lane + LANES * u);
        store_piece(part_w + (int64_t)blockIdx.x * F + c, F - c, acc[u]);
    }
}

// out[c] = sum over `rows` of part (rows, F): 64 threads per column, each a sum of every 64th row, then a tree. 1024 rows of
// 1440: 16 steps of loads in flight together instead of 64 with 16 threads per column (21 us).
template <typename T>
__global__ __launch_bounds__(1024) void column_sum_kernel(const float* __restrict__ part, int rows, int F,
                                                          T* __restrict__ out) {
    __shared__ float sums[64][17];
    const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4;
    const int c = blockIdx.x * 16 + cx;
    float a = 0.f;
    if (c < F) {
#pragma unroll 8
        for (int r = ry; r < rows; r += 64) a += part[(int64_t)r * F + c];
    }
    sums[ry][cx] = a;
    __syncthreads();
    for (int o = 32; o > 0; o >>= 1) {
        if (ry < o) sums[ry][cx] += sums[ry + o][cx];
        __syncthreads();
    }
    if (ry == 0 && c < F) out[c] = from_f<T>(sums[0][cx]);
}

// Workgroups of the backward, each of which adds a row of partial sums. 1024 are four per CU, of which the registers let four
// run at once at 1 and 2 units of 64 lanes, three at 3 (141 registers in fp32), two at 4 and 5, one from 257 registers on: the others
// follow in a second round.
constexpr int64_t kNormBwdGroups = 1024;
static inline int64_t norm_bwd_grid(int64_t N, int F) {
    const RowShape sh = row_shape(F);
    const int64_t rows = sh.lanes > 256 ? 1 : 256 / sh.lanes, need = (N + rows - 1) / rows;
    return need < kNormBwdGroups ? need : kNormBwdGroups;
}

template <typename T, int MODE>
static int launch_norm_fwd(const T* x, int64_t ld_x, const T* r, int64_t ld_r, int64_t N, int F, const T* w, float eps,
                           T* y, T* s, uint8_t* q, float* scale, hipStream_t st) {
    const RowShape sh = row_shape(F);
    const int threads = sh.lanes > 256 ? sh.lanes : 256, rows = threads / sh.lanes;
    const int64_t blocks = (N + rows - 1) / rows;
    if (blocks > 0x7fffffff) return FACE_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)blocks), block(threads);
#define FACE_ROW(L_, U_)                                                                                                   \
    if (sh.lanes == L_ && sh.units == U_)                                                                                  \
        hipLaunchKernelGGL((rms_norm_fwd_kernel<T, L_, U_, MODE>), grid, block, 0, st, x, ld_x, r, ld_r, N, F, w, eps, y, \
                           s, q, scale);
#define FACE_ROWS                                                                                                 \
    FACE_ROW(16, 1) FACE_ROW(16, 2) FACE_ROW(64, 1) FACE_ROW(64, 2) FACE_ROW(64, 3) FACE_ROW(64, 4) FACE_ROW(64, 5) \
    FACE_ROW(64, 6) FACE_ROW(64, 8) FACE_ROW(256, 3) FACE_ROW(256, 4) FACE_ROW(256, 5) FACE_ROW(256, 6)             \
    FACE_ROW(256, 8) FACE_ROW(1024, 3) FACE_ROW(1024, 4) FACE_ROW(1024, 5) FACE_ROW(1024, 6) FACE_ROW(1024, 8)
    FACE_ROWS
#undef FACE_ROW
    FACE_LAUNCH_CHECK();
    return 0;
}

template <typename T>
static int launch_norm_bwd(const T* s, int64_t ld_s, const T* dy, int64_t ld_dy, const T* ds, int64_t ld_ds, int64_t N,
                           int F, const T* w, float eps, T* dx, T* dw, float* work, hipStream_t st) {
    const RowShape sh = row_shape(F);
    const int64_t blocks = norm_bwd_grid(N, F);
    float* part = dw ? work : nullptr;
    if (blocks) {
        const dim3 grid((unsigned)blocks), block(sh.lanes > 256 ? sh.lanes : 256);
#define FACE_ROW(L_, U_)                                                                                                 \
    if (sh.lanes == L_ && sh.units == U_)                                                                                \
        hipLaunchKernelGGL((rms_norm_bwd_kernel<T, L_, U_>), grid, block, 0, st, s, ld_s, dy, ld_dy, ds, ld_ds, N, F, w, \
                           eps, dx, part);
        FACE_ROWS
#undef FACE_ROW
        FACE_LAUNCH_CHECK();
    }
    if (dw) {
        hipLaunchKernelGGL(column_sum_kernel<T>, dim3((unsigned)((F + 15) / 16)), dim3(1024), 0, st, work, (int)blocks,
                           F, dw);
        FACE_LAUNCH_CHECK();
    }
    return 0;
}

// Rows of `width` elements `ld` apart that do not overlap.
static inline bool rows_ok(int64_t ld, int64_t width) { return ld >= width; }

}  // namespace face

using namespace face;

extern "C" int face_rms_norm_fwd(const void* x, int64_t ld_x, const void* r, int64_t ld_r, int64_t N, int32_t F,
                                 int32_t dtype, const void* w, float eps, void* y, void* s, void* q, float* scale,
                                 void* stream) {
    if (N < 0 || F <= 0 || !rows_ok(ld_x, F) || (r && !rows_ok(ld_r, F)) || !(eps >= 0.f)) return FACE_ERR_ARG;
    if (dtype != FACE_F32 && dtype != FACE_BF16 && dtype != FACE_F16) return FACE_ERR_ARG;
    if (F > kRowMax) return FACE_ERR_UNSUPPORTED;
    if (N == 0) return 0;
    if (!x || !w || (!y && !q) || (y && q) || (q && !scale) || (!r != !s)) return FACE_ERR_ARG;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (q)
            return launch_norm_fwd<T, kNormQ8>((const T*)x, ld_x, (const T*)r, ld_r, N, F, (const T*)w, eps, nullptr, (T*)s,
                                               (uint8_t*)q, scale, (hipStream_t)stream);
        return launch_norm_fwd<T, kNorm>((const T*)x, ld_x, (const T*)r, ld_r, N, F, (const T*)w, eps, (T*)y, (T*)s, nullptr,
                                         nullptr, (hipStream_t)stream);
    });
}

extern "C" int64_t face_rms_norm_bwd_work(int64_t N, int32_t F) {
    if (N <= 0 || F <= 0 || F > kRowMax) return 0;
    return norm_bwd_grid(N, F) * F * 4;
}

extern "C" int face_rms_norm_bwd(const void* s, int64_t ld_s, const void* dy, int64_t ld_dy, const void* ds,
                                 int64_t ld_ds, int64_t N, int32_t F, int32_t dtype, const void* w, float eps, void* dx,
                                 void* dw, void* work, int64_t work_bytes, void* stream) {
    if (N < 0 || F <= 0 || !rows_ok(ld_s, F) || (dy && !rows_ok(ld_dy, F)) || (ds && !rows_ok(ld_ds, F)) || !(eps >= 0.f))
        return FACE_ERR_ARG;
    if (dtype != FACE_F32 && dtype != FACE_BF16 && dtype != FACE_F16) return FACE_ERR_ARG;
    if (F > kRowMax) return FACE_ERR_UNSUPPORTED;
    if (!dx && !dw) return 0;
    if (N && (!s || !w)) return FACE_ERR_ARG;
    if (dw && N && (!work || work_bytes < face_rms_norm_bwd_work(N, F))) return FACE_ERR_ARG;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return launch_norm_bwd<T>((const T*)s, ld_s, (const T*)dy, ld_dy, (const T*)ds, ld_ds, N, F, (const T*)w, eps,
                                  (T*)dx, (T*)dw, (float*)work, (hipStream_t)stream);
    });
}

extern "C" int face_quantize_rows(const void* x, int64_t ld_x, int64_t N, int32_t F, int32_t dtype, int32_t x_op, void* q,
                                  float* scale, void* stream) {
    if (N < 0 || F <= 0 || !rows_ok(ld_x, F) || (x_op != 0 && x_op != 1)) return FACE_ERR_ARG;
    if (dtype != FACE_F32 && dtype != FACE_BF16 && dtype != FACE_F16) return FACE_ERR_ARG;
    if (F > kRowMax) return FACE_ERR_UNSUPPORTED;
    if (N == 0) return 0;
    if (!x || !q || !scale) return FACE_ERR_ARG;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        auto* f = x_op ? launch_norm_fwd<T, kQ8Silu> : launch_norm_fwd<T, kQ8>;
        return f((const T*)x, ld_x, nullptr, 0, N, F, nullptr, 0.f, nullptr, nullptr, (uint8_t*)q, scale,
                 (hipStream_t)stream);
    });
}

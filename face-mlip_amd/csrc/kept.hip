// Rows to 8 bits and back (kept.h), and the gated activation whose backward reads its inputs in 8 bits:
//
//   y = silu(a) b,  a = x[:F], b = x[F:]
//   da = dy b silu'(a),  db = dy silu(a);   kept: of a and b as 8 bits hold them, each half in blocks of its own
//
// A row is spread over a power of two of threads, sixteen bytes each at a time. Bound by bytes: 200,000 x 2 x 512 bf16, inputs
// kept, forward 132 us, backward 147 (0.82 GB each: 6.2 and 5.6 TB/s); 100,000 x 2304 bf16 to 8 bits 110 us, back 115 (0.7 GB).
#include "kept.h"

namespace face {

// Threads per row of E values each at a time (a power of two, whole blocks): about `turns` times each. The gate, with three
// to five rows on their way, takes one turn (165,864 x 97 fp32 kept, both directions, 100 us for 177 of four), the single row of
// a packing four (100,000 x 2304 bf16 there and back 224 us for 241 of one).
static inline int kept_lanes_log2(int64_t F, int E, int turns) {
    const int64_t p = kept_blocks(F) * (kKeptBlock / E);
    int lg = E == 4 ? 3 : 2;
    while (lg < 8 && ((int64_t)turns << lg) < p) ++lg;
    return lg;
}

struct RowAt {
    int64_t n;
    int lane, lanes;
};
__device__ __forceinline__ RowAt row_at(int lg) {
    return {row_block() * (256 >> lg) + (threadIdx.x >> lg), (int)threadIdx.x & ((1 << lg) - 1), 1 << lg};
}

template <typename T, bool NT, bool CUT>
__global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ x, int64_t ld, int64_t N, int F, int lg,
                                                   uint8_t* __restrict__ q, uint8_t* __restrict__ scale) {
    constexpr int E = Sixteen<T>::E;
    const RowAt r = row_at(lg);
    if (r.n >= N) return;
    const int end = kKeptBlock * (int)kept_blocks(F);                    // whole quads
    x += r.n * ld;
    q += r.n * F;
    scale += r.n * kept_blocks(F);
    for (int c = E * r.lane; c < end; c += E * r.lanes) {
        float v[E];
        load16<NT, CUT>(x, c, F, v);
        store_kept<E, NT, CUT>(q, scale, c, F, v);
    }
}

// The type's largest value.
template <typename T>
constexpr float kLargest = __is_same(T, f16) ? 65504.f : (__is_same(T, bf16) ? 0x1.fep127f : 0x1.fffffep127f);

template <typename T, bool NT, bool CUT>
__global__ __launch_bounds__(256) void unpack_kernel(const uint8_t* __restrict__ q, int64_t ld_q,
                                                     const uint8_t* __restrict__ scale, int64_t ld_s, int64_t N, int F, int lg,
                                                     T* __restrict__ x) {
    constexpr int E = Sixteen<T>::E;
    const RowAt r = row_at(lg);
    if (r.n >= N) return;
    q += r.n * ld_q;
    scale += r.n * ld_s;
    x += r.n * F;
    for (int c = E * r.lane; c < F; c += E * r.lanes) {
        float v[E];
        kept_values(hold_kept<E, NT, CUT>(q, scale, c, F), v);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = within(v[e], kLargest<T>);
        store16<NT, CUT>(x, c, F, v);
    }
}

// q (N, 2 F) and scale (N, 2, blocks of F), or null.
template <typename T, bool KEEP, bool NT, bool CUT>
__global__ __launch_bounds__(256) void gated_fwd_kernel(const T* __restrict__ x, int64_t ld, int64_t N, int F, int lg,
                                                        T* __restrict__ y, uint8_t* __restrict__ q, uint8_t* __restrict__ scale) {
    constexpr int E = Sixteen<T>::E;
    const RowAt r = row_at(lg);
    if (r.n >= N) return;
    const int blocks = (int)kept_blocks(F), end = KEEP ? kKeptBlock * blocks : F;
    x += r.n * ld;
    y += r.n * F;
    q += r.n * 2 * F;
    scale += r.n * 2 * blocks;
    for (int c = E * r.lane; c < end; c += E * r.lanes) {
        float a[E], b[E];
        load16<NT, CUT>(x, c, F, a);
        load16<NT, CUT>(x + F, c, F, b);
        if constexpr (KEEP) {
            store_kept<E, NT, CUT>(q, scale, c, F, a);
            store_kept<E, NT, CUT>(q + F, scale + blocks, c, F, b);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) a[e] = silu(a[e]) * b[e];
        store16<NT, CUT>(y, c, F, a);
    }
}

template <typename T, bool KEPT, bool NT, bool CUT>
__global__ __launch_bounds__(256) void gated_bwd_kernel(const T* __restrict__ x, int64_t ld, const uint8_t* __restrict__ q,
                                                        const uint8_t* __restrict__ scale, const T* __restrict__ dy,
                                                        int64_t ld_dy, int64_t N, int F, int lg, T* __restrict__ dx) {
    constexpr int E = Sixteen<T>::E;
    const RowAt r = row_at(lg);
    if (r.n >= N) return;
    const int blocks = (int)kept_blocks(F);
    x += r.n * ld;
    q += r.n * 2 * F;
    scale += r.n * 2 * blocks;
    dy += r.n * ld_dy;
    dx += r.n * 2 * F;
    for (int c = E * r.lane; c < F; c += E * r.lanes) {
        float a[E], b[E], d[E];
        load16<NT, CUT>(dy, c, F, d);
        if constexpr (KEPT) {
            kept_values(hold_kept<E, NT, CUT>(q, scale, c, F), a);
            kept_values(hold_kept<E, NT, CUT>(q + F, scale + blocks, c, F), b);
        } else {
            load16<NT, CUT>(x, c, F, a);
            load16<NT, CUT>(x + F, c, F, b);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float t = a[e];
            a[e] = d[e] * b[e] * silu_slope(t);
            b[e] = d[e] * silu(t);
        }
        store16<NT, CUT>(dx, c, F, a);
        store16<NT, CUT>(dx + F, c, F, b);
    }
}

constexpr int32_t kKeptMax = 1 << 28;            // longest row
static int kept_args(int64_t N, int32_t F, int32_t dtype) {
    if (N < 0 || F <= 0) return FACE_ERR_ARG;
    if (dtype != FACE_F32 && dtype != FACE_BF16 && dtype != FACE_F16) return FACE_ERR_ARG;
    if (F > kKeptMax || N > (int64_t)0x7fffffff) return FACE_ERR_UNSUPPORTED;
    return 0;
}
static dim3 kept_grid(int64_t N, int lg) { return row_grid((N + (256 >> lg) - 1) >> (8 - lg)); }

}  // namespace face

using namespace face;

extern "C" int face_pack_rows(const void* x, int64_t ld_x, int64_t N, int32_t F, int32_t dtype, void* q, void* scale,
                              void* stream) {
    if (int rc = kept_args(N, F, dtype)) return rc;
    if (ld_x < F) return FACE_ERR_ARG;
    if (N == 0) return 0;
    if (!x || !q || !scale) return FACE_ERR_ARG;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int lg = kept_lanes_log2(F, Sixteen<T>::E, 4);
        with_forms(streams<T>(N * F * 3 / 2), F % Sixteen<T>::E, [&](auto nt, auto cut) {
            hipLaunchKernelGGL((pack_kernel<T, nt.value, cut.value>), kept_grid(N, lg), dim3(256), 0, (hipStream_t)stream, (const T*)x, ld_x, N, F, lg,
                           (uint8_t*)q, (uint8_t*)scale);
        });
        FACE_LAUNCH_CHECK();
        return 0;
    });
}

extern "C" int face_unpack_rows(const void* q, int64_t ld_q, const void* scale, int64_t ld_s, int64_t N, int32_t F,
                                int32_t dtype, void* x, void* stream) {
    if (int rc = kept_args(N, F, dtype)) return rc;
    if (ld_q < F || ld_s < kept_blocks(F)) return FACE_ERR_ARG;
    if (N == 0) return 0;
    if (!x || !q || !scale) return FACE_ERR_ARG;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int lg = kept_lanes_log2(F, Sixteen<T>::E, 4);
        with_forms(streams<T>(N * F * 3 / 2), F % Sixteen<T>::E, [&](auto nt, auto cut) {
            hipLaunchKernelGGL((unpack_kernel<T, nt.value, cut.value>), kept_grid(N, lg), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)q, ld_q,
                           (const uint8_t*)scale, ld_s, N, F, lg, (T*)x);
        });
        FACE_LAUNCH_CHECK();
        return 0;
    });
}

extern "C" int face_gated_silu_fwd(const void* x, int64_t ld_x, int64_t N, int32_t F, int32_t dtype, void* y, void* q,
                                   void* scale, void* stream) {
    if (int rc = kept_args(N, F, dtype)) return rc;
    if (ld_x < 2 * (int64_t)F || !q != !scale) return FACE_ERR_ARG;
    if (N == 0) return 0;
    if (!x || !y) return FACE_ERR_ARG;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int lg = kept_lanes_log2(F, Sixteen<T>::E, 1);
        with_forms(streams<T>(N * F * (q ? 4 : 3)), F % Sixteen<T>::E, [&](auto nt, auto cut) {
            auto* kern = q ? gated_fwd_kernel<T, true, nt.value, cut.value> : gated_fwd_kernel<T, false, nt.value, cut.value>;
            hipLaunchKernelGGL(kern, kept_grid(N, lg), dim3(256), 0, (hipStream_t)stream, (const T*)x, ld_x, N, F, lg, (T*)y,
                           (uint8_t*)q, (uint8_t*)scale);
        });
        FACE_LAUNCH_CHECK();
        return 0;
    });
}

extern "C" int face_gated_silu_bwd(const void* x, int64_t ld_x, const void* q, const void* scale, const void* dy,
                                   int64_t ld_dy, int64_t N, int32_t F, int32_t dtype, void* dx, void* stream) {
    if (int rc = kept_args(N, F, dtype)) return rc;
    if ((x && ld_x < 2 * (int64_t)F) || ld_dy < F) return FACE_ERR_ARG;
    if (N == 0) return 0;
    if ((x ? q || scale : !q || !scale) || !dy || !dx) return FACE_ERR_ARG;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int lg = kept_lanes_log2(F, Sixteen<T>::E, 1);
        with_forms(streams<T>(N * F * (q ? 4 : 5)), F % Sixteen<T>::E, [&](auto nt, auto cut) {
            auto* kern = q ? gated_bwd_kernel<T, true, nt.value, cut.value> : gated_bwd_kernel<T, false, nt.value, cut.value>;
            hipLaunchKernelGGL(kern, kept_grid(N, lg), dim3(256), 0, (hipStream_t)stream, (const T*)x, ld_x, (const uint8_t*)q,
                           (const uint8_t*)scale, (const T*)dy, ld_dy, N, F, lg, (T*)dx);
        });
        FACE_LAUNCH_CHECK();
        return 0;
    });
}

// Rows laid out by expert and joined again, for the slots a = order[p] of a plan at the places p < ptr[G] (slot a is
// choice a % k of row a / k):
//
//   out     xs[p] = x[a / k], 0 behind ptr[G];   dx[i] = sum over the row's slots of dxs[place(a)]
//   back    y[i] = r[i] + sum_j w[i, j] xs[place(i k + j)];   dxs[p] = w[a] dy[a / k], dw[a] = dy[a / k] . xs[p]
//
// place is order's inverse, -1 for slots that have none: what leaves rows of x, or gathers into rows of y, goes by
// rows, reads or writes each of those once, and its other side by whole rows. With one choice per row there is nothing to share:
// xs is gathered by order, without the inverse, as in small calls. Bound by bytes: 100,000 x 2304 bf16 to two of eight experts: out
// 246 us (1.4 GB: 5.6 TB/s), its gradient 207, back 286 (1.8 GB), its gradients 412 (2.3 GB), the inverse 2 x 5.
#include "kept.h"

namespace face {

constexpr int64_t kPlacesOne = 8192;             // one workgroup inverts the order up to here

__device__ __forceinline__ int64_t places_of(const int32_t* ptr, int G, int64_t slots) {
    const int64_t m = ptr[G];
    return m < 0 ? 0 : (m < slots ? m : slots);
}

// The inverse in LDS, then written once.
__global__ __launch_bounds__(1024) void places_one_kernel(const int32_t* __restrict__ ptr, const int32_t* __restrict__ order,
                                                          int slots, int G, int32_t* __restrict__ place) {
    __shared__ int32_t at[kPlacesOne];
    const int m = (int)places_of(ptr, G, slots);
    for (int a = threadIdx.x; a < slots; a += 1024) at[a] = -1;
    __syncthreads();
    for (int p = threadIdx.x; p < m; p += 1024) {
        const int a = order[p];
        if (a >= 0 && a < slots) at[a] = p;
    }
    __syncthreads();
    for (int a = threadIdx.x; a < slots; a += 1024) place[a] = at[a];
}
__global__ __launch_bounds__(256) void places_none_kernel(int64_t slots, int32_t* __restrict__ place) {
    const int64_t a = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (a < slots) place[a] = -1;
}
__global__ __launch_bounds__(256) void places_kernel(const int32_t* __restrict__ ptr, const int32_t* __restrict__ order,
                                                     int64_t slots, int G, int32_t* __restrict__ place) {
    const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (p >= places_of(ptr, G, slots)) return;
    const int a = order[p];
    if (a >= 0 && a < slots) place[a] = (int32_t)p;
}

// Threads per row: one turn where 256 are enough (96,184 x 394 bf16 to three of 40 experts and back, both directions, 436 us
// for 566 of four turns).
static inline int sorted_lanes_log2(int64_t F, int size) {
    const int64_t p = (F * size + 15) / 16;
    int lg = 4;
    while (lg < 8 && ((int64_t)1 << lg) < p) ++lg;
    return lg;
}

// xs[p] = x[order[p] / k].
template <typename T, bool NT, bool CUT>
__global__ __launch_bounds__(256) void dispatch_gather_kernel(const T* __restrict__ x, int64_t ld,
                                                              const int32_t* __restrict__ ptr,
                                                              const int32_t* __restrict__ order, int64_t slots, int k, int G,
                                                              int F, int lg, T* __restrict__ xs) {
    constexpr int E = Sixteen<T>::E;
    const int64_t p = row_block() * (256 >> lg) + (threadIdx.x >> lg);
    if (p >= slots) return;
    const int a = p < places_of(ptr, G, slots) ? order[p] : -1;
    const bool some = a >= 0 && a < slots;
    const T* from = x + (int64_t)(some ? a / k : 0) * ld;
    for (int c = E * (threadIdx.x & ((1 << lg) - 1)); c < F; c += E << lg) {
        float v[E] = {};
        if (some) load16<NT, CUT>(from, c, F, v);
        store16<NT, CUT>(xs + p * F, c, F, v);
    }
}

// A row's threads write it to the places of its k slots, and zeros to those of the places i k .. i k + k - 1 that
// have no slot; four slots per turn, their places known before the row is.
template <typename T, bool NT, bool CUT>
__global__ __launch_bounds__(256) void dispatch_scatter_kernel(const T* __restrict__ x, int64_t ld,
                                                               const int32_t* __restrict__ ptr,
                                                               const int32_t* __restrict__ order,
                                                               const int32_t* __restrict__ place, int64_t slots, int k, int G,
                                                               int F, int lg, T* __restrict__ xs) {
    constexpr int E = Sixteen<T>::E;
    const int64_t n = row_block() * (256 >> lg) + (threadIdx.x >> lg);
    if (n * k >= slots) return;
    const int64_t m = places_of(ptr, G, slots);
    constexpr int J = 4;
    for (int j0 = 0; j0 < k; j0 += J) {
        int p[J];
        bool bare[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int64_t i = n * k + j0 + j;
            const bool in = j0 + j < k;
            p[j] = in ? place[i] : -1;
            const int a = in && i < m ? order[i] : -1;
            bare[j] = in && (a < 0 || a >= slots || place[a] != i);
        }
        for (int c = E * (threadIdx.x & ((1 << lg) - 1)); c < F; c += E << lg) {
            float v[E];
            const float none[E] = {};
            load16<NT, CUT>(x + n * ld, c, F, v);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if (p[j] >= 0) store16<NT, CUT>(xs + (int64_t)p[j] * F, c, F, v);
                if (bare[j]) store16<NT, CUT>(xs + (n * k + j0 + j) * F, c, F, none);
            }
        }
    }
}

// out[i] = r[i] + sum_j w[i, j] y[place(i k + j)], in order; w null: ones. Four slots per turn, their rows on the way
// together; the first four's places are known before any row is asked for.
template <typename T, bool NT, bool CUT>
__global__ __launch_bounds__(256) void return_fwd_kernel(const T* __restrict__ y, int64_t ld_y, const int32_t* __restrict__ place,
                                                         const float* __restrict__ w, const T* __restrict__ r, int64_t ld_r,
                                                         int64_t N, int k, int F, int lg, T* __restrict__ out) {
    constexpr int E = Sixteen<T>::E;
    const int64_t n = row_block() * (256 >> lg) + (threadIdx.x >> lg);
    if (n >= N) return;
    constexpr int J = 4;
    int p[J];
    float f[J];
    auto turn = [&](int j0) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int64_t i = n * k + j0 + j;
            p[j] = j0 + j < k ? place[i] : -1;
            f[j] = j0 + j < k && w ? w[i] : 1.f;
        }
    };
    turn(0);
    for (int c = E * (threadIdx.x & ((1 << lg) - 1)); c < F; c += E << lg) {
        float s[E] = {};
        if (r) load16<NT, CUT>(r + n * ld_r, c, F, s);
        for (int j0 = 0; j0 < k; j0 += J) {
            if (k > J) turn(j0);
            Sixteen<T> v[J];
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (p[j] >= 0) v[j] = hold16<NT, CUT>(y + (int64_t)p[j] * ld_y, c, F);
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (p[j] >= 0) {
                    float x[E];
                    values16<T>(v[j], x);
#pragma unroll
                    for (int e = 0; e < E; ++e) s[e] = fmaf(f[j], x[e], s[e]);
                }
        }
        store16<NT, CUT>(out + n * F, c, F, s);
    }
}

// dy[p] = w dout and dw = dout . y[p] at the places of the row's slots; zeros at places without a slot.
template <typename T, int LANES, bool NT, bool CUT>
__global__ __launch_bounds__(256) void return_bwd_kernel(const T* __restrict__ dout, int64_t ld_d, const T* __restrict__ y,
                                                         int64_t ld_y, const int32_t* __restrict__ ptr,
                                                         const int32_t* __restrict__ order,
                                                         const int32_t* __restrict__ place, const float* __restrict__ w,
                                                         int64_t N, int k, int G, int F, T* __restrict__ dy,
                                                         float* __restrict__ dw) {
    constexpr int E = Sixteen<T>::E;
    __shared__ float part[LANES / 64 + 1];
    const int lane = threadIdx.x % LANES;
    const int64_t n = row_block() * (256 / LANES) + threadIdx.x / LANES;
    if (n >= N) return;
    const int64_t slots = N * k, m = places_of(ptr, G, slots);
    constexpr int J = 4;
    for (int j0 = 0; j0 < k; j0 += J) {
        float s[J] = {}, f[J];
        int p[J];
        bool bare[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int64_t i = n * k + j0 + j;
            const bool in = j0 + j < k;
            f[j] = in && w ? w[i] : 1.f;
            p[j] = in ? place[i] : -1;
            const int a = in && i < m ? order[i] : -1;
            bare[j] = in && (a < 0 || a >= slots || place[a] != i);
        }
        for (int c = E * lane; c < F; c += E * LANES) {
            float d[E];
            load16<NT, CUT>(dout + n * ld_d, c, F, d);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                float v[E];
                if (dw && p[j] >= 0) {
                    load16<NT, CUT>(y + (int64_t)p[j] * ld_y, c, F, v);
#pragma unroll
                    for (int e = 0; e < E; ++e) s[j] = fmaf(d[e], v[e], s[j]);
                }
                if (!dy) continue;
                if (p[j] >= 0) {
#pragma unroll
                    for (int e = 0; e < E; ++e) v[e] = f[j] * d[e];
                    store16<NT, CUT>(dy + (int64_t)p[j] * F, c, F, v);
                }
                if (bare[j]) {
                    const float none[E] = {};
                    store16<NT, CUT>(dy + (n * k + j0 + j) * F, c, F, none);
                }
            }
        }
        if (dw) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const float t = row_sum<LANES>(s[j], part);
                if (lane == 0 && j0 + j < k) dw[n * k + j0 + j] = t;
            }
        }
    }
}

static int sorted_args(int64_t N, int32_t k, int32_t G, int32_t F, int32_t dtype) {
    if (N < 0 || k <= 0 || G <= 0 || F <= 0) return FACE_ERR_ARG;
    if (dtype != FACE_F32 && dtype != FACE_BF16 && dtype != FACE_F16) return FACE_ERR_ARG;
    if (F > (1 << 28) || N > (int64_t)0x7fffffff || N * k > (int64_t)0x7fffffff) return FACE_ERR_UNSUPPORTED;
    return 0;
}
static void launch_places(const int32_t* ptr, const int32_t* order, int64_t slots, int G, int32_t* place, hipStream_t st) {
    if (slots <= kPlacesOne) {
        hipLaunchKernelGGL(places_one_kernel, dim3(1), dim3(1024), 0, st, ptr, order, (int)slots, G, place);
        return;
    }
    const dim3 grid((unsigned)((slots + 255) / 256));
    hipLaunchKernelGGL(places_none_kernel, grid, dim3(256), 0, st, slots, place);
    hipLaunchKernelGGL(places_kernel, grid, dim3(256), 0, st, ptr, order, slots, G, place);
}
static dim3 sorted_grid(int64_t rows, int lg) { return row_grid((rows + (256 >> lg) - 1) >> (8 - lg)); }

}  // namespace face

using namespace face;

extern "C" int face_expert_dispatch(const void* x, int64_t ld_x, int32_t k, const int32_t* ptr, const int32_t* order,
                                    int32_t* place, int64_t N, int32_t G, int32_t F, int32_t dtype, void* xs, void* stream) {
    if (int rc = sorted_args(N, k, G, F, dtype)) return rc;
    if (ld_x < F) return FACE_ERR_ARG;
    if (N == 0) return 0;
    if (!x || !ptr || !order || !xs) return FACE_ERR_ARG;
    const int64_t slots = N * k;
    if (place) launch_places(ptr, order, slots, G, place, (hipStream_t)stream);
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        int lg = sorted_lanes_log2(F, sizeof(T));
        if (place && lg > 6) lg = 6;             // one row on its way, k written: 247 us for 270 of 256 threads (100,000 x 2304 bf16, k = 2)
        with_forms(streams<T>((slots + N) * F), F % Sixteen<T>::E, [&](auto nt, auto cut) {
            if (place)
                hipLaunchKernelGGL((dispatch_scatter_kernel<T, nt.value, cut.value>), sorted_grid(N, lg), dim3(256), 0,
                                   (hipStream_t)stream, (const T*)x, ld_x, ptr, order, place, slots, k, G, F, lg, (T*)xs);
            else
                hipLaunchKernelGGL((dispatch_gather_kernel<T, nt.value, cut.value>), sorted_grid(slots, lg), dim3(256), 0,
                                   (hipStream_t)stream, (const T*)x, ld_x, ptr, order, slots, k, G, F, lg, (T*)xs);
        });
        FACE_LAUNCH_CHECK();
        return 0;
    });
}

extern "C" int face_expert_return_fwd(const void* y, int64_t ld_y, const int32_t* ptr, const int32_t* order, int32_t* place,
                                      int32_t placed, const float* weight, const void* r, int64_t ld_r, int64_t N, int32_t k,
                                      int32_t G, int32_t F, int32_t dtype, void* out, void* stream) {
    if (int rc = sorted_args(N, k, G, F, dtype)) return rc;
    if (ld_y < F || (r && ld_r < F)) return FACE_ERR_ARG;
    if (N == 0) return 0;
    if (!y || !place || !out || (!placed && (!ptr || !order))) return FACE_ERR_ARG;
    if (!placed) launch_places(ptr, order, N * k, G, place, (hipStream_t)stream);
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int lg = sorted_lanes_log2(F, sizeof(T));
        with_forms(streams<T>((N * k + N * (r ? 2 : 1)) * F), F % Sixteen<T>::E, [&](auto nt, auto cut) {
            hipLaunchKernelGGL((return_fwd_kernel<T, nt.value, cut.value>), sorted_grid(N, lg), dim3(256), 0, (hipStream_t)stream,
                               (const T*)y, ld_y, place, weight, (const T*)r, ld_r, N, k, F, lg, (T*)out);
        });
        FACE_LAUNCH_CHECK();
        return 0;
    });
}

extern "C" int face_expert_return_bwd(const void* dout, int64_t ld_d, const void* y, int64_t ld_y, const int32_t* ptr,
                                      const int32_t* order, const int32_t* place, const float* weight, int64_t N, int32_t k,
                                      int32_t G, int32_t F, int32_t dtype, void* dy, float* dweight, void* stream) {
    if (int rc = sorted_args(N, k, G, F, dtype)) return rc;
    if (ld_d < F || (dweight && ld_y < F)) return FACE_ERR_ARG;
    if (N == 0 || (!dy && !dweight)) return 0;
    if (!dout || !ptr || !order || !place || (dweight && !y)) return FACE_ERR_ARG;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int L = F * sizeof(T) <= 256 ? 16 : (F * sizeof(T) <= 8192 ? 64 : 256), rows = 256 / L;
        const dim3 grid = row_grid((N + rows - 1) / rows);
        with_forms(streams<T>((2 * N * k + N) * F), F % Sixteen<T>::E, [&](auto nt, auto cut) {
            auto* kern = L == 16 ? return_bwd_kernel<T, 16, nt.value, cut.value>
                       : L == 64 ? return_bwd_kernel<T, 64, nt.value, cut.value> : return_bwd_kernel<T, 256, nt.value, cut.value>;
            hipLaunchKernelGGL(kern, grid, dim3(256), 0, (hipStream_t)stream, (const T*)dout, ld_d, (const T*)y, ld_y, ptr, order,
                               place, weight, N, k, G, F, (T*)dy, dweight);
        });
        FACE_LAUNCH_CHECK();
        return 0;
    });
}

// The gate of an expert layer, the grouping of its rows, and the join of the experts' results.
//
// Gate: p = softmax of a row's logits over the experts open to it (its row of `allowed`, and a logit above
// -inf); the k largest logits in descending order, ties to the lower expert; weight p, or p over the sum
// of the k. What a row cannot fill has expert -1 and weight 0.
//   renormalised: dl_e = w_j (g_j - sum_i w_i g_i) of a chosen expert, 0 of others
//   else:         dl_e = p_e ([e chosen] g_j - sum_i w_i g_i) of an open expert, 0 of others
// The zeros are written as such: a product would make NaN of them in a row whose sum is not finite.
// A group of 16 lanes holds a row in registers (64 lanes from 257 experts on) and finds each maximum with
// cross-lane moves on the VALU: 64 experts and k = 4 are 32 such steps and no trip through LDS. Bound by the
// row's latency where there are few, by these steps else: 100,000 rows x 64 experts, k = 4, masked 16 us (28 MB: 6 us
// of bytes), the gradient 18 us (55 MB: 11 us), without mask and renormalised 12 and 10 us.
#include "elem.h"

namespace face {

constexpr int kRouteMaxExperts = 1024, kRouteMaxK = 16;

// Order of the logits as unsigned values: a NaN above all, -0 as 0, and 0 for -inf, which cannot be chosen.
__device__ __forceinline__ uint32_t route_key(float l) {
    if (!(l == l)) return 0xffffffffu;
    const uint32_t u = __builtin_bit_cast(uint32_t, l + 0.f);
    const uint32_t k = (u >> 31) ? ~u : (u | 0x80000000u);
    return k > 0x007fffffu ? k : 0u;
}
__device__ __forceinline__ float route_value(uint32_t key) {
    return __builtin_bit_cast(float, key == 0xffffffffu ? 0x7fc00000u : (key >> 31) ? key & 0x7fffffffu : ~key);
}

// e^x of a logit below the largest: one instruction and a product, whose rounding is |x| steps of 2^-24, as the
// subtraction's is already. Below 2^-126 it may be 0.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    auto step = [&](uint32_t w) { v = w > v ? w : v; };
    if constexpr (LANES == 16) {
        step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
        step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
        step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
        step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
    } else {
        for (int o = 32; o > 0; o >>= 1) step((uint32_t)__shfl_xor((int)v, o, kWave));
    }
    return v;
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (LANES == 16) return row16_sum(v);
    return group_sum(v, kWave);
}

// The row's logits (lane holds experts lane + LANES v), -inf where it may not go.
template <typename T, int LANES, int V>
__device__ __forceinline__ void route_row(const T* __restrict__ l, const uint8_t* __restrict__ allowed,
                                          const int32_t* __restrict__ group, int n_groups, int64_t n, int E, int lane,
                                          float x[V]) {
    const float kNone = -__builtin_inff();
    // the logits are on their way before the row's mask is known
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = lane + LANES * v < E ? to_f(l[lane + LANES * v]) : kNone;
    if (!allowed) return;
    const int g = group ? group[n] : 0;
    const bool open = g >= 0 && g < n_groups;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = lane + LANES * v;
        if (e < E && !(open && allowed[(int64_t)g * E + e])) x[v] = kNone;
    }
}

template <typename T, int LANES, int V>
__global__ __launch_bounds__(256) void route_fwd_kernel(const T* __restrict__ logits, int64_t ld, int64_t N, int E, int k,
                                                        const uint8_t* __restrict__ allowed,
                                                        const int32_t* __restrict__ group, int n_groups, int renorm,
                                                        int32_t* __restrict__ expert, float* __restrict__ weight) {
    const int lane = threadIdx.x % LANES;
    const int64_t n = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (n >= N) return;
    float x[V];
    route_row<T, LANES, V>(logits + n * ld, allowed, group, n_groups, n, E, lane, x);
    uint32_t key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = route_key(x[v]);
    float top = 0.f, sum = 0.f, mine = 0.f;      // lane j keeps choice j
    int32_t got = -1;
    for (int j = 0; j < k; ++j) {
        uint32_t best = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) best = key[v] > best ? key[v] : best;
        best = lanes_max<LANES>(best);
        if (best == 0) break;                    // the same in all lanes of the row
        uint32_t at = 0;                         // ~expert, so that the lowest is the largest
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const uint32_t c = ~(uint32_t)(lane + LANES * v);
            at = key[v] == best && c > at ? c : at;
        }
        const int e = (int)~lanes_max<LANES>(at);
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (lane + LANES * v == e) key[v] = 0;
        const float l = route_value(best);
        if (j == 0) {
            top = l;
            if (!renorm) {
                float s = 0.f;
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (x[v] > -__builtin_inff() || x[v] != x[v]) s += exp_of(x[v] - top);
                sum = lanes_sum<LANES>(s);
            }
        }
        if (lane == j) {
            got = e;
            mine = exp_of(l - top);
        }
    }
    if (renorm) sum = lanes_sum<LANES>(mine);
    if (lane < k) {
        expert[n * k + lane] = got;
        weight[n * k + lane] = got >= 0 ? mine / sum : 0.f;
    }
}

template <typename T, int LANES, int V>
__global__ __launch_bounds__(256) void route_bwd_kernel(const T* __restrict__ logits, int64_t ld, int64_t N, int E, int k,
                                                        const uint8_t* __restrict__ allowed,
                                                        const int32_t* __restrict__ group, int n_groups, int renorm,
                                                        const int32_t* __restrict__ expert,
                                                        const float* __restrict__ weight, const float* __restrict__ dw,
                                                        T* __restrict__ dl) {
    const int lane = threadIdx.x % LANES;
    const int64_t n = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (n >= N) return;
    float d[V];
    uint32_t reached = 0;                        // bit v: the loss depends on the lane's expert v
    int my_e = -1;                               // lane j: choice j
    float my_w = 0.f, my_g = 0.f;
    if (lane < k) {
        my_e = expert[n * k + lane];
        my_w = weight[n * k + lane];
        my_g = dw[n * k + lane];
    }
    const float mean = lanes_sum<LANES>(my_e >= 0 ? my_w * my_g : 0.f);
    if (renorm) {
#pragma unroll
        for (int v = 0; v < V; ++v) d[v] = 0.f;
    } else {
        route_row<T, LANES, V>(logits + n * ld, allowed, group, n_groups, n, E, lane, d);
        // the largest open logit, a NaN first, as the forward shifts by
        uint32_t best = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const uint32_t key = route_key(d[v]);
            best = key > best ? key : best;
        }
        best = lanes_max<LANES>(best);
        const float top = route_value(best);
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const bool open = d[v] > -__builtin_inff() || d[v] != d[v];
            reached |= (uint32_t)open << v;
            d[v] = open ? exp_of(d[v] - top) : 0.f;
            s += d[v];
        }
        s = lanes_sum<LANES>(s);
        const float inv = best ? 1.f / s : 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) d[v] *= inv;                 // p
    }
    float up[V] = {};                            // g of the chosen, 0 of the others
    for (int j = 0; j < k; ++j) {
        const int e = __shfl(my_e, j, LANES);
        if (e < 0) break;
        const float g = __shfl(my_g, j, LANES), w = __shfl(my_w, j, LANES);
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (lane + LANES * v == e) {
                up[v] = g;
                if (renorm) {
                    d[v] = w;
                    reached |= 1u << v;
                }
            }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = lane + LANES * v;
        if (e < E) dl[n * E + e] = from_f<T>((reached >> v) & 1 ? d[v] * (up[v] - mean) : 0.f);
    }
}

// ---------------------------------------------------------------- grouping
// order = the slots sorted by expert, stably; ptr = where each expert's begin; slots of no expert in [0, G) last,
// from ptr[G] on. A counting sort over segments of the slots: counts per segment, their prefix sums expert by
// expert, then each segment places its slots. Within a wave the slots of one expert find their rank from the
// lanes that hold the same expert (one ballot per bit of its number), so equal experts keep their order.
constexpr int kPlanMaxGroups = 1024;
constexpr int kPlanThreads = 512, kPlanWaves = kPlanThreads / kWave;
constexpr int64_t kPlanOne = 4096;               // one workgroup does it all up to here

// Slots per workgroup: 1024 up to 1 M slots, then 1024 workgroups. 400,000 slots, 64 experts (us, all three launches): segments
// of 512 18.9, of 1024 15.7, of 2048 16.8, of 4096 22.1; 1,000 experts 39 / 31 / 30 / 35.
static inline int64_t plan_segment(int64_t A) {
    const int64_t s = (A + 1023) / 1024;
    return s > 1024 ? (s + 511) / 512 * 512 : 1024;
}

__device__ __forceinline__ int plan_group(const int32_t* expert, int64_t a, int64_t end, int G) {
    if (a >= end) return G + 1;                  // no slot
    const int e = expert[a];
    return e >= 0 && e < G ? e : G;
}
// Lanes of the wave whose g is the same.
__device__ __forceinline__ uint64_t same_lanes(int g, int bits) {
    uint64_t m = ~0ull;
    for (int b = 0; b < bits; ++b) {
        const uint64_t v = __ballot((g >> b) & 1);
        m &= (g >> b) & 1 ? v : ~v;
    }
    return m;
}

// Counts of each wave's part of the segment in cnt[wave][G + 1] (LDS).
__device__ __forceinline__ void plan_count(const int32_t* expert, int64_t a0, int64_t a1, int G, int bits, int* cnt) {
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    for (int i = threadIdx.x; i < kPlanWaves * (G + 1); i += kPlanThreads) cnt[i] = 0;
    __syncthreads();
    const int64_t per = (a1 - a0 + kPlanThreads - 1) / kPlanThreads * kWave;
    const int64_t b0 = a0 + wave * per, b1 = b0 + per < a1 ? b0 + per : a1;
    for (int64_t a = b0; a < b1; a += kWave) {
        const int g = plan_group(expert, a + lane, b1, G);
        const uint64_t m = same_lanes(g, bits);
        if (g <= G && (m & ((1ull << lane) - 1)) == 0) atomicAdd(&cnt[wave * (G + 1) + g], __popcll(m));
    }
    __syncthreads();
}
// Places the segment's slots; base[wave][g] is where the wave's first slot of expert g goes.
__device__ __forceinline__ void plan_place(const int32_t* expert, int64_t a0, int64_t a1, int G, int bits, int* base,
                                           int32_t* order) {
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int64_t per = (a1 - a0 + kPlanThreads - 1) / kPlanThreads * kWave;
    const int64_t b0 = a0 + wave * per, b1 = b0 + per < a1 ? b0 + per : a1;
    volatile int* mine = base + wave * (G + 1);
    for (int64_t a = b0; a < b1; a += kWave) {
        const int g = plan_group(expert, a + lane, b1, G);
        const uint64_t m = same_lanes(g, bits);
        const int rank = __popcll(m & ((1ull << lane) - 1));
        if (g <= G) {
            const int at = mine[g];
            order[at + rank] = (int32_t)(a + lane);
            __builtin_amdgcn_wave_barrier();     // every lane has read the place before the first one moves it on
            if (rank == 0) mine[g] = at + __popcll(m);
        }
        __builtin_amdgcn_wave_barrier();
    }
}
// cnt[wave][g] becomes the exclusive sum over the waves, plus begin[g].
__device__ __forceinline__ void plan_waves(int* cnt, const int* begin, int G) {
    for (int g = threadIdx.x; g <= G; g += kPlanThreads) {
        int at = begin[g];
        for (int w = 0; w < kPlanWaves; ++w) {
            const int c = cnt[w * (G + 1) + g];
            cnt[w * (G + 1) + g] = at;
            at += c;
        }
    }
    __syncthreads();
}
// begin[0..G] = exclusive sums of tot[0..G] (LDS, one workgroup).
__device__ __forceinline__ void plan_scan(const int* tot, int* begin, int G) {
    if (threadIdx.x < kWave) {
        const int lane = threadIdx.x;
        int run = 0;
        for (int g0 = 0; g0 <= G; g0 += kWave) {
            const int g = g0 + lane, c = g <= G ? tot[g] : 0;
            int s = c;
            for (int o = 1; o < kWave; o <<= 1) {
                const int t = __shfl_up(s, o, kWave);
                if (lane >= o) s += t;
            }
            if (g <= G) begin[g] = run + s - c;
            run += __shfl(s, kWave - 1, kWave);
        }
    }
    __syncthreads();
}

__global__ __launch_bounds__(kPlanThreads) void plan_one_kernel(const int32_t* __restrict__ expert, int64_t A, int G,
                                                                int bits, int32_t* __restrict__ ptr,
                                                                int32_t* __restrict__ order) {
    extern __shared__ int lds[];
    int *cnt = lds, *tot = cnt + kPlanWaves * (G + 1), *begin = tot + G + 1;
    plan_count(expert, 0, A, G, bits, cnt);
    for (int g = threadIdx.x; g <= G; g += kPlanThreads) {
        int s = 0;
        for (int w = 0; w < kPlanWaves; ++w) s += cnt[w * (G + 1) + g];
        tot[g] = s;
    }
    __syncthreads();
    plan_scan(tot, begin, G);
    for (int g = threadIdx.x; g <= G; g += kPlanThreads) ptr[g] = begin[g];
    plan_waves(cnt, begin, G);
    plan_place(expert, 0, A, G, bits, cnt, order);
}
__global__ __launch_bounds__(kPlanThreads) void plan_count_kernel(const int32_t* __restrict__ expert, int64_t A,
                                                                  int64_t seg, int G, int bits, int32_t* __restrict__ count) {
    extern __shared__ int cnt[];
    const int64_t a0 = blockIdx.x * seg, a1 = a0 + seg < A ? a0 + seg : A;
    plan_count(expert, a0, a1, G, bits, cnt);
    for (int g = threadIdx.x; g <= G; g += kPlanThreads) {
        int s = 0;
        for (int w = 0; w < kPlanWaves; ++w) s += cnt[w * (G + 1) + g];
        count[(int64_t)g * gridDim.x + blockIdx.x] = s;
    }
}
// count (G + 1, segs): every expert's row becomes its exclusive sums, tot its total. One wave per expert.
__global__ __launch_bounds__(256) void plan_rows_kernel(int32_t* __restrict__ count, int segs, int G,
                                                        int32_t* __restrict__ tot) {
    const int g = blockIdx.x * 4 + threadIdx.x / kWave, lane = threadIdx.x % kWave;
    if (g > G) return;
    int32_t* row = count + (int64_t)g * segs;
    int run = 0;
    for (int b0 = 0; b0 < segs; b0 += kWave) {
        const int b = b0 + lane, c = b < segs ? row[b] : 0;
        int s = c;
        for (int o = 1; o < kWave; o <<= 1) {
            const int t = __shfl_up(s, o, kWave);
            if (lane >= o) s += t;
        }
        if (b < segs) row[b] = run + s - c;
        run += __shfl(s, kWave - 1, kWave);
    }
    if (lane == 0) tot[g] = run;
}
__global__ __launch_bounds__(kPlanThreads) void plan_place_kernel(const int32_t* __restrict__ expert, int64_t A,
                                                                  int64_t seg, int G, int bits,
                                                                  const int32_t* __restrict__ count,
                                                                  const int32_t* __restrict__ tot,
                                                                  int32_t* __restrict__ ptr, int32_t* __restrict__ order) {
    extern __shared__ int lds[];
    int *cnt = lds, *all = cnt + kPlanWaves * (G + 1), *begin = all + G + 1;
    const int64_t a0 = blockIdx.x * seg, a1 = a0 + seg < A ? a0 + seg : A;
    for (int g = threadIdx.x; g <= G; g += kPlanThreads) all[g] = tot[g];
    plan_count(expert, a0, a1, G, bits, cnt);    // its barriers publish `all`
    plan_scan(all, begin, G);
    if (blockIdx.x == 0)
        for (int g = threadIdx.x; g <= G; g += kPlanThreads) ptr[g] = begin[g];
    __syncthreads();
    for (int g = threadIdx.x; g <= G; g += kPlanThreads) begin[g] += count[(int64_t)g * gridDim.x + blockIdx.x];
    __syncthreads();
    plan_waves(cnt, begin, G);
    plan_place(expert, a0, a1, G, bits, cnt, order);
}

// ---------------------------------------------------------------- join
// out[i] = r[i] + sum_j w[i, j] y[i k + j], one read of each row; a row's pieces are spread over LANES threads. Bound by
// bytes: 100,000 x 2 x 512 bf16 89 us forward (410 MB), 91 us backward (512 MB): 4.6 and 5.6 TB/s, part of it from the last
// level of cache.
// w null: factors of one. Y: the type of y's rows, T or float.
template <typename Y, typename T, int LANES>
__global__ __launch_bounds__(256) void combine_fwd_kernel(const Y* __restrict__ y, int64_t ld_y,
                                                          const float* __restrict__ w, const T* __restrict__ r,
                                                          int64_t ld_r, int64_t N, int k, int F, T* __restrict__ out) {
    const int64_t n = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (n >= N) return;
    for (int c = kPiece * (threadIdx.x % LANES); c < F; c += kPiece * LANES) {
        float a[kPiece] = {};
        if (r) load_piece(r + n * ld_r + c, F - c, a);
#pragma unroll 4
        for (int j = 0; j < k; ++j) {
            float v[kPiece];
            load_piece(y + (n * k + j) * ld_y + c, F - c, v);
            const float f = w ? w[n * k + j] : 1.f;
#pragma unroll
            for (int e = 0; e < kPiece; ++e) a[e] = fmaf(f, v[e], a[e]);
        }
        store_piece(out + n * F + c, F - c, a);
    }
}
// dy[i k + j] = w[i, j] dout[i], dw[i, j] = dout[i] . y[i k + j]; four slots per turn, so that a turn's rows are in
// flight together (dout is read again by the next turn, from the caches).
template <typename T, int LANES>
__global__ __launch_bounds__(256) void combine_bwd_kernel(const T* __restrict__ dout, int64_t ld_d,
                                                          const T* __restrict__ y, int64_t ld_y,
                                                          const float* __restrict__ w, int64_t N, int k, int F,
                                                          T* __restrict__ dy, float* __restrict__ dw) {
    __shared__ float part[LANES / 64 + 1];
    const int lane = threadIdx.x % LANES;
    const int64_t n = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (n >= N) return;
    constexpr int J = 4;
    for (int j0 = 0; j0 < k; j0 += J) {
        float s[J] = {}, f[J];
#pragma unroll
        for (int j = 0; j < J; ++j) f[j] = j0 + j < k ? w[n * k + j0 + j] : 0.f;
        for (int c = kPiece * lane; c < F; c += kPiece * LANES) {
            float d[kPiece];
            load_piece(dout + n * ld_d + c, F - c, d);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if (j0 + j >= k) break;
                const int64_t a = n * k + j0 + j;
                if (dw) {
                    float v[kPiece];
                    load_piece(y + a * ld_y + c, F - c, v);
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) s[j] = fmaf(d[e], v[e], s[j]);
                }
                if (dy) {
                    float v[kPiece];
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) v[e] = f[j] * d[e];
                    store_piece(dy + a * F + c, F - c, v);
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

// Threads per row of the join: about four pieces each.
static inline int join_lanes(int F) { return F <= 512 ? 16 : (F <= 4096 ? 64 : 256); }

template <typename Y, typename T>
static int launch_combine_fwd(const Y* y, int64_t ld_y, const float* w, const T* r, int64_t ld_r, int64_t N, int k, int F, T* out,
                              hipStream_t st) {
    const int L = join_lanes(F), rows = 256 / L;
    const dim3 grid((unsigned)((N + rows - 1) / rows));
    auto* kern = L == 16 ? combine_fwd_kernel<Y, T, 16> : (L == 64 ? combine_fwd_kernel<Y, T, 64> : combine_fwd_kernel<Y, T, 256>);
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, y, ld_y, w, r, ld_r, N, k, F, out);
    FACE_LAUNCH_CHECK();
    return 0;
}

int sum_slot_rows(const float* rows, int64_t N, int k, int F, int dtype, void* out, hipStream_t st) {
    if (F > (1 << 30) || N > (int64_t)0x7fffffff) return FACE_ERR_UNSUPPORTED;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return launch_combine_fwd<float, T>(rows, F, nullptr, nullptr, 0, N, k, F, (T*)out, st);
    });
}

}  // namespace face

using namespace face;

static int route_args(int64_t ld, int64_t N, int32_t E, int32_t k, int32_t dtype, const void* allowed, const void* group,
                      int32_t n_groups) {
    if (N < 0 || E <= 0 || k <= 0 || k > E || ld < E) return FACE_ERR_ARG;
    if (dtype != FACE_F32 && dtype != FACE_BF16 && dtype != FACE_F16) return FACE_ERR_ARG;
    if (N && (allowed ? n_groups <= 0 || (!group && n_groups != 1) : group != nullptr)) return FACE_ERR_ARG;
    if (E > kRouteMaxExperts || k > kRouteMaxK) return FACE_ERR_UNSUPPORTED;
    if (N > (int64_t)0x7fffffff * 4) return FACE_ERR_UNSUPPORTED;
    return 0;
}

// The variants: lanes per row and logits per lane.
#define FACE_ROUTE_SHAPES                                                                                        \
    if (E <= 16) { FACE_ROUTE(16, 1) } else if (E <= 32) { FACE_ROUTE(16, 2) } else if (E <= 64) { FACE_ROUTE(16, 4) } \
    else if (E <= 128) { FACE_ROUTE(16, 8) } else if (E <= 256) { FACE_ROUTE(16, 16) } else { FACE_ROUTE(64, 16) }

extern "C" int face_route_fwd(const void* logits, int64_t ld, int64_t N, int32_t E, int32_t k, int32_t dtype,
                              const uint8_t* allowed, const int32_t* group, int32_t n_groups, int32_t renorm,
                              int32_t* expert, float* weight, void* stream) {
    if (int rc = route_args(ld, N, E, k, dtype, allowed, group, n_groups)) return rc;
    if (N == 0) return 0;
    if (!logits || !expert || !weight) return FACE_ERR_ARG;
    const int64_t rows = E <= 256 ? 16 : 4;
    const dim3 grid((unsigned)((N + rows - 1) / rows));
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
#define FACE_ROUTE(L_, V_)                                                                                              \
    hipLaunchKernelGGL((route_fwd_kernel<T, L_, V_>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)logits, ld, N, \
                       E, k, allowed, group, n_groups, renorm, expert, weight);
        FACE_ROUTE_SHAPES
#undef FACE_ROUTE
        FACE_LAUNCH_CHECK();
        return 0;
    });
}

extern "C" int face_route_bwd(const void* logits, int64_t ld, int64_t N, int32_t E, int32_t k, int32_t dtype,
                              const uint8_t* allowed, const int32_t* group, int32_t n_groups, int32_t renorm,
                              const int32_t* expert, const float* weight, const float* dweight, void* dlogits,
                              void* stream) {
    if (int rc = route_args(ld, N, E, k, dtype, allowed, group, n_groups)) return rc;
    if (N == 0) return 0;
    if (!logits || !expert || !weight || !dweight || !dlogits) return FACE_ERR_ARG;
    const int64_t rows = E <= 256 ? 16 : 4;
    const dim3 grid((unsigned)((N + rows - 1) / rows));
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
#define FACE_ROUTE(L_, V_)                                                                                              \
    hipLaunchKernelGGL((route_bwd_kernel<T, L_, V_>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)logits, ld, N, \
                       E, k, allowed, group, n_groups, renorm, expert, weight, dweight, (T*)dlogits);
        FACE_ROUTE_SHAPES
#undef FACE_ROUTE
        FACE_LAUNCH_CHECK();
        return 0;
    });
}

extern "C" int64_t face_group_plan_work(int64_t slots, int32_t G) {
    if (slots <= kPlanOne || G <= 0 || G > kPlanMaxGroups) return 0;
    const int64_t seg = plan_segment(slots), segs = (slots + seg - 1) / seg;
    return 4 * (int64_t)(G + 1) * (segs + 1);
}

extern "C" int face_group_plan(const int32_t* expert, int64_t slots, int32_t G, int32_t* ptr, int32_t* order, void* work,
                               int64_t work_bytes, void* stream) {
    if (slots < 0 || G <= 0 || !ptr || (slots && (!expert || !order))) return FACE_ERR_ARG;
    if (G > kPlanMaxGroups || slots >= ((int64_t)1 << 31)) return FACE_ERR_UNSUPPORTED;
    if (work_bytes < face_group_plan_work(slots, G) || (!work && face_group_plan_work(slots, G))) return FACE_ERR_ARG;
    int bits = 1;
    while ((G + 1) >> bits) ++bits;
    const hipStream_t st = (hipStream_t)stream;
    const size_t lds = 4 * (size_t)(G + 1) * (kPlanWaves + 2);
    if (slots <= kPlanOne) {
        hipLaunchKernelGGL(plan_one_kernel, dim3(1), dim3(kPlanThreads), lds, st, expert, slots, G, bits, ptr, order);
        FACE_LAUNCH_CHECK();
        return 0;
    }
    const int64_t seg = plan_segment(slots);
    const int segs = (int)((slots + seg - 1) / seg);
    int32_t *tot = (int32_t*)work, *count = tot + G + 1;
    hipLaunchKernelGGL(plan_count_kernel, dim3(segs), dim3(kPlanThreads), lds, st, expert, slots, seg, G, bits, count);
    hipLaunchKernelGGL(plan_rows_kernel, dim3((G + 4) / 4), dim3(256), 0, st, count, segs, G, tot);
    hipLaunchKernelGGL(plan_place_kernel, dim3(segs), dim3(kPlanThreads), lds, st, expert, slots, seg, G, bits, count, tot,
                       ptr, order);
    FACE_LAUNCH_CHECK();
    return 0;
}

static int combine_args(int64_t N, int32_t k, int32_t F, int32_t dtype) {
    if (N < 0 || k <= 0 || F <= 0) return FACE_ERR_ARG;
    if (dtype != FACE_F32 && dtype != FACE_BF16 && dtype != FACE_F16) return FACE_ERR_ARG;
    if (F > (1 << 30) || N > (int64_t)0x7fffffff) return FACE_ERR_UNSUPPORTED;
    return 0;
}

extern "C" int face_expert_combine_fwd(const void* y, int64_t ld_y, const float* weight, const void* r, int64_t ld_r,
                                       int64_t N, int32_t k, int32_t F, int32_t dtype, void* out, void* stream) {
    if (int rc = combine_args(N, k, F, dtype)) return rc;
    if (ld_y < F || (r && ld_r < F)) return FACE_ERR_ARG;
    if (N == 0) return 0;
    if (!y || !out) return FACE_ERR_ARG;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return launch_combine_fwd<T, T>((const T*)y, ld_y, weight, (const T*)r, ld_r, N, k, F, (T*)out, (hipStream_t)stream);
    });
}

extern "C" int face_expert_combine_bwd(const void* dout, int64_t ld_d, const void* y, int64_t ld_y, const float* weight,
                                       int64_t N, int32_t k, int32_t F, int32_t dtype, void* dy, float* dweight,
                                       void* stream) {
    if (int rc = combine_args(N, k, F, dtype)) return rc;
    if (ld_d < F || (dweight && ld_y < F)) return FACE_ERR_ARG;
    if (N == 0 || (!dy && !dweight)) return 0;
    if (!dout || !weight || (dweight && !y)) return FACE_ERR_ARG;
    const int L = join_lanes(F), rows = 256 / L;
    const dim3 grid((unsigned)((N + rows - 1) / rows));
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        auto* kern = L == 16 ? combine_bwd_kernel<T, 16> : (L == 64 ? combine_bwd_kernel<T, 64> : combine_bwd_kernel<T, 256>);
        hipLaunchKernelGGL(kern, grid, dim3(256), 0, (hipStream_t)stream, (const T*)dout, ld_d, (const T*)y, ld_y, weight, N,
                           k, F, (T*)dy, dweight);
        FACE_LAUNCH_CHECK();
        return 0;
    });
}

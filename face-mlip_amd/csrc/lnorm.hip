// Layer norm of atom rows with the residual's addition, its backward with the gradients of weight and bias, rows
// in 8 bits for serving, and normalised rows kept in 8 bits for the backward:
//
//   s = x + r (rounded to the rows' type, as the residual stream holds it)
//   h = (s - mean s) rstd,  rstd = 1 / sqrt(mean((s - mean s)^2) + eps),  y = h w + b
//   ds = rstd (g - mean g - h mean(g h)) + ds_in,  g = dy w;   dw = sum over rows of dy h,  db = sum of dy
//
// Everything between the first read of a row and its last store is fp32 in registers up to 16384 columns: the mean
// first, then the squares around it, and with them the sum of the differences, which corrects the mean's own rounding.
// Longer rows are read three times by a workgroup of 1024. The backward takes mean and rstd (8 bytes a row) from the
// forward, so that its one reduction follows its only reads. Bound by bytes.
// A row lies in the registers of 16 lanes up to 256 columns, of a wave up to 2560, of four up to 10240, of eight up to 16384,
// in as few pieces a lane as hold it: only the last of them may end before the lane's, so the others are loaded and stored
// without a test. With a test at each (and rounded-up shapes) the backward of 100,000 x 2304 bf16 took 615 us for 354.
// 24,000 x 1440 fp32 with the residual: forward 99 us, backward 99 + 5 (5.6 TB/s of the 553 MB that each has to move);
// 100,000 x 2304 bf16 kept in 8 bits: forward 364 us (5.7 TB/s), backward 337 + 6 (4.8); 21 x 864 3.9 us, the launch. Reading
// the next row ahead of its turn spilled (497 us for 330 without).
#include "kept.h"

namespace face {

enum { kLn = 0, kLnQ8 = 1, kLnKept = 2 };

struct LnFwdArgs {
    const void *x, *r;
    int64_t ld_x, ld_r, N;
    int F;
    const void *w, *b;
    float eps;
    void *y, *s;
    uint8_t* q;                        // kLnQ8: the row in 8 bits; kLnKept: h kept
    float* scale;                      // kLnQ8: of each row
    uint8_t* block_scale;              // kLnKept
    float *mean, *rstd;                // may be null
};

// A lane's eight values of a row, on their way in the row's type.
template <typename T>
struct LnPiece {
    Sixteen<T> a[kPiece / Sixteen<T>::E];
    __device__ __forceinline__ void values(float x[kPiece]) const {
#pragma unroll
        for (int h = 0; h < kPiece / Sixteen<T>::E; ++h) values16<T>(a[h], x + Sixteen<T>::E * h);
    }
};
template <bool NT, typename T>
__device__ __forceinline__ LnPiece<T> hold_eight(const T* row, int c, int F) {
    LnPiece<T> r;
#pragma unroll
    for (int h = 0; h < kPiece / Sixteen<T>::E; ++h) r.a[h] = hold16<NT, true>(row, c + Sixteen<T>::E * h, F);
    return r;
}

// Which columns of a row a lane has as its piece u of U: eight neighbouring ones of 16-bit rows; of fp32 rows twice four, LANES
// chunks of four apart, so that the lanes of an access lie side by side. Only the last unit may be cut short.
template <typename T, int LANES, int U, bool CUT>
struct LnUnit {
    static constexpr int E = Sixteen<T>::E, H = kPiece / E;
    bool whole;                        // known when the loop over u is unrolled
    int c, F;                          // first column, columns of the row
    __device__ __forceinline__ LnUnit(int u, int lane, int F_) : whole(u + 1 < U), c(kPiece * LANES * u + E * lane), F(F_) {}
    __device__ __forceinline__ int at(int h) const { return c + E * LANES * h; }
    __device__ __forceinline__ bool inside(int e) const { return whole || at(e / E) + e % E < F; }
    template <bool NT>
    __device__ __forceinline__ LnPiece<T> hold(const T* row) const {
        LnPiece<T> r;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if (whole) r.a[h] = {ld16s<NT>(row + at(h)), 0};
            else r.a[h] = hold16<NT, CUT>(row, at(h), F);
        }
        return r;
    }
    template <bool NT>
    __device__ __forceinline__ void load(const T* row, float x[kPiece]) const {
        hold<NT>(row).values(x);
    }
    template <bool NT, typename Y>
    __device__ __forceinline__ void store(Y* row, const float x[kPiece]) const {
        const int end = whole ? c + kPiece * LANES : F;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            store16<NT, CUT>(row, at(h), end, x + E * h);
            if constexpr (sizeof(Y) != sizeof(T)) store16<NT, CUT>(row, at(h) + 4, end, x + 4);   // fp32 sums of 16-bit rows
        }
    }
    template <bool NT>
    __device__ __forceinline__ void store_8bit(uint8_t* q, const float x[kPiece], float inv) const {
#pragma unroll
        for (int h = 0; h < H; ++h) store_e4m3<E, NT, CUT>(q, at(h), whole ? c + kPiece * LANES : F, x + E * h, inv);
    }
    template <bool NT>
    __device__ __forceinline__ void keep(uint8_t* q, uint8_t* scale, const float x[kPiece]) const {
#pragma unroll
        for (int h = 0; h < H; ++h) store_kept<E, NT, CUT>(q, scale, at(h), whole ? c + kPiece * LANES : F, x + E * h);
    }
    template <bool NT>
    __device__ __forceinline__ void hold_kept_row(const uint8_t* q, const uint8_t* scale, KeptPiece<E> k[H]) const {
#pragma unroll
        for (int h = 0; h < H; ++h)
            k[h] = whole ? hold_kept<E, NT, false>(q, scale, at(h), at(h) + E) : hold_kept<E, NT, CUT>(q, scale, at(h), F);
    }
};

template <typename T, int LANES, int U, int MODE, bool NT, bool CUT>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void ln_fwd_kernel(LnFwdArgs a) {
    constexpr int kRows = LANES > 256 ? 1 : 256 / LANES;
    using Unit = LnUnit<T, LANES, U, CUT>;
    __shared__ float part[LANES / 32 + 1];
    const int lane = threadIdx.x % LANES, F = a.F;
    const int64_t n = row_block() * kRows + threadIdx.x / LANES;
    if (n >= a.N) return;                        // a whole row's threads; rows of several waves have a workgroup each
    const T *w = (const T*)a.w, *b = (const T*)a.b;
    float v[U][kPiece];
#pragma unroll
    for (int u = 0; u < U; ++u) Unit(u, lane, F).template load<NT>((const T*)a.x + n * a.ld_x, v[u]);
    if (a.r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const Unit at(u, lane, F);
            float t[kPiece];
            at.template load<NT>((const T*)a.r + n * a.ld_r, t);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) v[u][e] = to_f(from_f<T>(v[u][e] + t[e]));
            at.template store<NT>((T*)a.s + n * F, v[u]);
        }
    }
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < kPiece; ++e) sum += v[u][e];
    const float inv_f = 1.f / (float)F;
    float mean = row_sum<LANES>(sum, part) * inv_f;
    float d1 = 0.f, d2 = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const Unit at(u, lane, F);
#pragma unroll
        for (int e = 0; e < kPiece; ++e) {
            const float d = at.inside(e) ? v[u][e] - mean : 0.f;
            d1 += d;
            d2 = fmaf(d, d, d2);
        }
    }
    row_sum2<LANES>(d1, d2, part);
    d1 *= inv_f;
    mean += d1;
    const float var = fmaf(-d1, d1, d2 * inv_f);
    const float rs = 1.f / sqrtf(fmaxf(var, 0.f) + a.eps);
    if (lane == 0 && a.rstd) {
        a.rstd[n] = rs;
        if (a.mean) a.mean[n] = mean;
    }
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const Unit at(u, lane, F);
        float h[kPiece], g[kPiece], y[kPiece] = {};
        at.template load<false>(w, g);
        if (b) at.template load<false>(b, y);
#pragma unroll
        for (int e = 0; e < kPiece; ++e) {
            h[e] = at.inside(e) ? (v[u][e] - mean) * rs : 0.f;
            y[e] = fmaf(h[e], g[e], y[e]);
        }
        if constexpr (MODE == kLnKept) at.template keep<NT>(a.q + n * F, a.block_scale + n * kept_blocks(F), h);
        if constexpr (MODE == kLnQ8) {
            // the magnitudes compare as integers, a NaN above everything: its row gets a NaN scale and no number
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                v[u][e] = y[e];
                const uint32_t m = __builtin_bit_cast(uint32_t, y[e]) & 0x7fffffffu;
                top = m > top ? m : top;
            }
        } else {
            at.template store<NT>((T*)a.y + n * F, y);
        }
    }
    if constexpr (MODE == kLnQ8) {
        const float amax = __builtin_bit_cast(float, row_max<LANES>(top, part));
        float sc = amax / 448.f;
        if (sc < 0x1p-126f) sc = 0x1p-126f;
        const float inv = 1.f / sc;
#pragma unroll
        for (int u = 0; u < U; ++u) Unit(u, lane, F).template store_8bit<NT>(a.q + n * F, v[u], inv);
        if (lane == 0) a.scale[n] = sc;
    }
}

// Rows of any length, a workgroup each: read for the mean, for the squares and for the result (and for the largest
// magnitude of rows in 8 bits); a thread reads back only what it wrote itself.
template <typename T>
__device__ __forceinline__ void ln_piece(const float v[kPiece], float mean, float rs, const T* w, const T* b, int left,
                                         float h[kPiece], float y[kPiece]) {
    float g[kPiece], o[kPiece] = {};
    load_piece(w, left, g);
    if (b) load_piece(b, left, o);
#pragma unroll
    for (int e = 0; e < kPiece; ++e) {
        h[e] = e < left ? (v[e] - mean) * rs : 0.f;
        y[e] = fmaf(h[e], g[e], o[e]);
    }
}
template <typename T, int MODE>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(LnFwdArgs a) {
    constexpr int LANES = 1024;
    __shared__ float part[LANES / 32 + 1];
    const int lane = threadIdx.x, F = a.F;
    const int64_t n = row_block();
    if (n >= a.N) return;
    const T *w = (const T*)a.w, *b = (const T*)a.b;
    const T* x = (const T*)a.x + n * a.ld_x;
    const int end = (F + kKeptBlock - 1) / kKeptBlock * kKeptBlock;      // whole quads
    float sum = 0.f;
    if (a.r) {
        const T* r = (const T*)a.r + n * a.ld_r;
        T* s = (T*)a.s + n * F;
        for (int c = kPiece * lane; c < F; c += kPiece * LANES) {
            float v[kPiece], t[kPiece];
            load_piece(x + c, F - c, v);
            load_piece(r + c, F - c, t);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                v[e] = to_f(from_f<T>(v[e] + t[e]));
                sum += v[e];
            }
            store_piece(s + c, F - c, v);
        }
        x = s;
    } else {
        for (int c = kPiece * lane; c < F; c += kPiece * LANES) {
            float v[kPiece];
            load_piece(x + c, F - c, v);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) sum += v[e];
        }
    }
    const float inv_f = 1.f / (float)F;
    float mean = row_sum<LANES>(sum, part) * inv_f, d1 = 0.f, d2 = 0.f;
    for (int c = kPiece * lane; c < F; c += kPiece * LANES) {
        float v[kPiece];
        load_piece(x + c, F - c, v);
#pragma unroll
        for (int e = 0; e < kPiece; ++e) {
            const float d = c + e < F ? v[e] - mean : 0.f;
            d1 += d;
            d2 = fmaf(d, d, d2);
        }
    }
    row_sum2<LANES>(d1, d2, part);
    d1 *= inv_f;
    mean += d1;
    const float rs = 1.f / sqrtf(fmaxf(fmaf(-d1, d1, d2 * inv_f), 0.f) + a.eps);
    if (lane == 0 && a.rstd) {
        a.rstd[n] = rs;
        if (a.mean) a.mean[n] = mean;
    }
    uint32_t top = 0;
    for (int c = kPiece * lane; c < end; c += kPiece * LANES) {
        float v[kPiece], h[kPiece], y[kPiece];
        load_piece(x + c, F - c, v);
        ln_piece(v, mean, rs, w + c, b ? b + c : nullptr, F - c, h, y);
        if constexpr (MODE == kLnKept) store_kept<kPiece, false, true>(a.q + n * F, a.block_scale + n * kept_blocks(F), c, F, h);
        if constexpr (MODE == kLnQ8) {
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                const uint32_t m = __builtin_bit_cast(uint32_t, y[e]) & 0x7fffffffu;
                top = m > top ? m : top;
            }
        } else {
            store_piece((T*)a.y + n * F + c, F - c, y);
        }
    }
    if constexpr (MODE == kLnQ8) {
        const float amax = __builtin_bit_cast(float, row_max<LANES>(top, part));
        float sc = amax / 448.f;
        if (sc < 0x1p-126f) sc = 0x1p-126f;
        const float inv = 1.f / sc;
        for (int c = kPiece * lane; c < F; c += kPiece * LANES) {
            float v[kPiece], h[kPiece], y[kPiece];
            load_piece(x + c, F - c, v);
            ln_piece(v, mean, rs, w + c, b ? b + c : nullptr, F - c, h, y);
            store_e4m3<kPiece, false, true>(a.q + n * F, c, F, y, inv);
        }
        if (lane == 0) a.scale[n] = sc;
    }
}

struct LnBwdArgs {
    const void* s;                     // rows that were normalised, or null: h as it was kept
    int64_t ld_s;
    const uint8_t *q, *block_scale;
    const float *mean, *rstd;
    const void *dy, *ds;               // may be null: zeros
    int64_t ld_dy, ld_ds, N;
    int F;
    const void* w;
    void* dx;                          // may be null
    float* part;                       // (workgroups, 2 F): sums of dw, of db; may be null
};

// h of a piece, from the row as it was normalised or as it was kept.
template <typename T, bool KEPT, int E>
struct LnRow {
    LnPiece<T> a;
    __device__ __forceinline__ void values(float mean, float rs, float h[kPiece]) const {
        a.values(h);
#pragma unroll
        for (int e = 0; e < kPiece; ++e) h[e] = (h[e] - mean) * rs;
    }
};
template <typename T, int E>
struct LnRow<T, true, E> {
    KeptPiece<E> a[kPiece / E];
    __device__ __forceinline__ void values(float, float, float h[kPiece]) const {
#pragma unroll
        for (int i = 0; i < kPiece / E; ++i) kept_values_near(a[i], h + E * i);
    }
};

// A workgroup takes rows blockIdx, blockIdx + grid, ... and keeps its columns' sums of dw and db in registers over
// all of them; its row of partial sums is joined with the others' by ln_column_sum_kernel in a fixed order: no
// atomics. All of a row's reads are issued before the first is used. Beyond a row's end dy is 0, and h is finite where
// the row's is.
template <typename T, int LANES, int U, bool KEPT, bool NT, bool CUT>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void ln_bwd_kernel(LnBwdArgs a) {
    constexpr int kRows = LANES > 256 ? 1 : 256 / LANES;
    using Unit = LnUnit<T, LANES, U, CUT>;
    __shared__ float part[LANES / 32 + 1];
    __shared__ float sums[kRows > 1 ? 2 * LANES * U * kPiece : 1];
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES, F = a.F;
    const float inv_f = 1.f / (float)F;
    float aw[U][kPiece] = {}, ab[U][kPiece] = {};
    for (int64_t n = (int64_t)blockIdx.x * kRows + slot; n < a.N; n += (int64_t)gridDim.x * kRows) {
        LnRow<T, KEPT, Unit::E> row[U];
        LnPiece<T> dy[U], ds[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const Unit at(u, lane, F);
            if constexpr (KEPT) at.template hold_kept_row<NT>(a.q + n * F, a.block_scale + n * kept_blocks(F), row[u].a);
            else row[u].a = at.template hold<NT>((const T*)a.s + n * a.ld_s);
            dy[u] = a.dy ? at.template hold<NT>((const T*)a.dy + n * a.ld_dy) : LnPiece<T>{};
            ds[u] = a.ds && a.dx ? at.template hold<NT>((const T*)a.ds + n * a.ld_ds) : LnPiece<T>{};
        }
        const float mean = KEPT ? 0.f : a.mean[n], rs = a.rstd[n];
        float sg = 0.f, sh = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const Unit at(u, lane, F);
            float h[kPiece], d[kPiece], w[kPiece];
            row[u].values(mean, rs, h);
            dy[u].values(d);
            at.template load<false>((const T*)a.w, w);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                ab[u][e] += d[e];
                aw[u][e] = fmaf(d[e], h[e], aw[u][e]);
                const float g = d[e] * w[e];
                sg += g;
                sh = fmaf(g, h[e], sh);
            }
        }
        if (!a.dx) continue;
        row_sum2<LANES>(sg, sh, part);
        sg *= inv_f;
        sh *= inv_f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const Unit at(u, lane, F);
            float h[kPiece], d[kPiece], w[kPiece], o[kPiece];
            row[u].values(mean, rs, h);
            dy[u].values(d);
            ds[u].values(o);
            at.template load<false>((const T*)a.w, w);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) o[e] = fmaf(rs, fmaf(d[e], w[e], -sg) - h[e] * sh, o[e]);
            at.template store<NT>((T*)a.dx + n * F, o);
        }
    }
    if (!a.part) return;
    if constexpr (kRows > 1) {
        for (int k = 0; k < kRows; ++k) {
            __syncthreads();
            if (slot == k) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) {
                        float& t = sums[(u * kPiece + e) * LANES + lane];
                        float& o = sums[(U * kPiece + u * kPiece + e) * LANES + lane];
                        t = k ? t + aw[u][e] : aw[u][e];
                        o = k ? o + ab[u][e] : ab[u][e];
                    }
            }
        }
        if (slot != kRows - 1) return;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                aw[u][e] = sums[(u * kPiece + e) * LANES + lane];
                ab[u][e] = sums[(U * kPiece + u * kPiece + e) * LANES + lane];
            }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const Unit at(u, lane, F);
        float* p = a.part + (int64_t)blockIdx.x * 2 * F;
        at.template store<false>(p, aw[u]);
        at.template store<false>(p + F, ab[u]);
    }
}

// The same for rows of any length, a workgroup per row, each read twice; a thread adds to its own columns of the
// workgroup's partial sums in memory.
template <typename T, bool KEPT>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(LnBwdArgs a) {
    constexpr int LANES = 1024;
    __shared__ float part[LANES / 32 + 1];
    const int lane = threadIdx.x, F = a.F;
    const float inv_f = 1.f / (float)F;
    float* sums = a.part ? a.part + (int64_t)blockIdx.x * 2 * F : nullptr;
    bool first = true;
    for (int64_t n = blockIdx.x; n < a.N; n += gridDim.x) {
        const float mean = KEPT ? 0.f : a.mean[n], rs = a.rstd[n];
        float sg = 0.f, sh = 0.f;
        auto load = [&](int c, float h[kPiece], float d[kPiece], float w[kPiece]) {
            LnRow<T, KEPT, kPiece> row;
            if constexpr (KEPT) row.a[0] = hold_kept<kPiece, false, true>(a.q + n * F, a.block_scale + n * kept_blocks(F), c, F);
            else row.a = hold_eight<false>((const T*)a.s + n * a.ld_s, c, F);
            row.values(mean, rs, h);
            LnPiece<T> r = a.dy ? hold_eight<false>((const T*)a.dy + n * a.ld_dy, c, F) : LnPiece<T>{};
            r.values(d);
            load_piece((const T*)a.w + c, F - c, w);
        };
        for (int c = kPiece * lane; c < F; c += kPiece * LANES) {
            float h[kPiece], d[kPiece], w[kPiece];
            load(c, h, d, w);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                const float g = d[e] * w[e];
                sg += g;
                sh = fmaf(g, h[e], sh);
            }
            if (sums) {
                float p[kPiece] = {}, o[kPiece] = {};
                if (!first) {
                    load_piece(sums + c, F - c, p);
                    load_piece(sums + F + c, F - c, o);
                }
#pragma unroll
                for (int e = 0; e < kPiece; ++e) {
                    p[e] = fmaf(d[e], h[e], p[e]);
                    o[e] += d[e];
                }
                store_piece(sums + c, F - c, p);
                store_piece(sums + F + c, F - c, o);
            }
        }
        first = false;
        if (!a.dx) continue;
        row_sum2<LANES>(sg, sh, part);
        sg *= inv_f;
        sh *= inv_f;
        for (int c = kPiece * lane; c < F; c += kPiece * LANES) {
            float h[kPiece], d[kPiece], w[kPiece], o[kPiece] = {};
            load(c, h, d, w);
            if (a.ds) load_piece((const T*)a.ds + n * a.ld_ds + c, F - c, o);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) o[e] = fmaf(rs, fmaf(d[e], w[e], -sg) - h[e] * sh, o[e]);
            store_piece((T*)a.dx + n * F + c, F - c, o);
        }
    }
}

// dw[c], db[c] = sums over `rows` of part (rows, 2 F): 64 threads per column, each a sum of every 64th row, then a
// tree.
template <typename T>
__global__ __launch_bounds__(1024) void ln_column_sum_kernel(const float* __restrict__ part, int rows, int F,
                                                             T* __restrict__ dw, T* __restrict__ db) {
    __shared__ float sums[64][17];
    const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4;
    const int c = blockIdx.x * 16 + cx;
    float a = 0.f;
    if (c < 2 * F) {
#pragma unroll 8
        for (int r = ry; r < rows; r += 64) a += part[(int64_t)r * 2 * F + c];
    }
    sums[ry][cx] = a;
    __syncthreads();
    for (int o = 32; o > 0; o >>= 1) {
        if (ry < o) sums[ry][cx] += sums[ry + o][cx];
        __syncthreads();
    }
    if (ry == 0 && c < 2 * F) {
        T* out = c < F ? dw : db;
        if (out) out[c < F ? c : c - F] = from_f<T>(sums[0][cx]);
    }
}

constexpr int kLnHeld = 16384;                   // longest row that stays in registers
constexpr int kLnMax = 65536;

// The variants: lanes per row and pieces per lane, the fewest that hold the row. Large calls have a form for rows of whole sixteen
// bytes: the shifts of others cost registers (100,000 x 2304 bf16 kept in 8 bits, both directions, 819 us with them, 709 without).
#define FACE_LN_ROWS                                                                                                 \
    FACE_ROW(16, 1) FACE_ROW(16, 2) FACE_ROW(64, 1) FACE_ROW(64, 2) FACE_ROW(64, 3) FACE_ROW(64, 4) FACE_ROW(64, 5) \
    FACE_ROW(256, 2) FACE_ROW(256, 3) FACE_ROW(256, 4) FACE_ROW(256, 5) FACE_ROW(512, 3) FACE_ROW(512, 4)
static inline RowShape ln_shape(int F) {
    const int p = (F + kPiece - 1) / kPiece, lanes = p <= 32 ? 16 : (p <= 320 ? 64 : (p <= 1280 ? 256 : 512));
    return {lanes, (p + lanes - 1) / lanes};
}
static inline int64_t ln_rows(int F) { return F > 2560 ? 1 : 256 / ln_shape(F).lanes; }

// Workgroups of the backward: as many as the registers of its pieces let run at once on 256 CUs, so that all of them
// start together and end together (100,000 x 1440 bf16: 768 take 226 us, 512 238, 1024 259).
static inline int64_t ln_bwd_grid(int64_t N, int F, bool wide) {
    const RowShape sh = ln_shape(F);
    const int per = F > kLnHeld ? 2 : sh.lanes == 512 ? 1 : sh.units <= 2 ? (wide ? 3 : 4) : sh.units == 3 && !wide ? 3 : 2;
    const int64_t need = (N + ln_rows(F) - 1) / ln_rows(F);
    return need < 256 * per ? need : 256 * per;
}

template <typename T, int MODE>
static int launch_ln_fwd(const LnFwdArgs& a, hipStream_t st) {
    const RowShape sh = ln_shape(a.F);
    const int64_t rows = ln_rows(a.F), blocks = (a.N + rows - 1) / rows;
    if (blocks > 0x7fffffff) return FACE_ERR_UNSUPPORTED;
    const dim3 grid = row_grid(blocks);
    const bool nt = streams<T>(a.N * a.F * (a.r ? 4 : 2)), cut = a.F % Sixteen<T>::E;
    if (a.F > kLnHeld) {
        hipLaunchKernelGGL((ln_fwd_long_kernel<T, MODE>), grid, dim3(1024), 0, st, a);
    }
#define FACE_ROW(L_, U_)                                                                                                 \
    else if (sh.lanes == L_ && sh.units == U_)                                                                          \
        hipLaunchKernelGGL((!nt ? ln_fwd_kernel<T, L_, U_, MODE, false, true>                                           \
                            : cut ? ln_fwd_kernel<T, L_, U_, MODE, true, true> : ln_fwd_kernel<T, L_, U_, MODE, true, false>), \
                           grid, dim3(L_ > 256 ? L_ : 256), 0, st, a);
    FACE_LN_ROWS
#undef FACE_ROW
    FACE_LAUNCH_CHECK();
    return 0;
}

template <typename T, bool KEPT>
static int launch_ln_bwd(const LnBwdArgs& a, T* dw, T* db, hipStream_t st) {
    const RowShape sh = ln_shape(a.F);
    const int64_t blocks = ln_bwd_grid(a.N, a.F, sizeof(T) == 4);
    if (blocks) {
        const dim3 grid((unsigned)blocks);
        const bool nt = streams<T>(a.N * a.F * (a.ds ? 4 : 3)), cut = a.F % Sixteen<T>::E;
        if (a.F > kLnHeld) {
            hipLaunchKernelGGL((ln_bwd_long_kernel<T, KEPT>), grid, dim3(1024), 0, st, a);
        }
#define FACE_ROW(L_, U_)                                                                                                 \
    else if (sh.lanes == L_ && sh.units == U_)                                                                          \
        hipLaunchKernelGGL((!nt ? ln_bwd_kernel<T, L_, U_, KEPT, false, true>                                           \
                            : cut ? ln_bwd_kernel<T, L_, U_, KEPT, true, true> : ln_bwd_kernel<T, L_, U_, KEPT, true, false>), \
                           grid, dim3(L_ > 256 ? L_ : 256), 0, st, a);
        FACE_LN_ROWS
#undef FACE_ROW
        FACE_LAUNCH_CHECK();
    }
    if (dw || db) {
        hipLaunchKernelGGL(ln_column_sum_kernel<T>, dim3((unsigned)((2 * a.F + 15) / 16)), dim3(1024), 0, st, a.part,
                           (int)blocks, a.F, dw, db);
        FACE_LAUNCH_CHECK();
    }
    return 0;
}

static int ln_args(int64_t N, int32_t F, int32_t dtype) {
    if (N < 0 || F <= 0) return FACE_ERR_ARG;
    if (dtype != FACE_F32 && dtype != FACE_BF16 && dtype != FACE_F16) return FACE_ERR_ARG;
    if (F > kLnMax) return FACE_ERR_UNSUPPORTED;
    return 0;
}

}  // namespace face

using namespace face;

extern "C" int face_layer_norm_rows_fwd(const void* x, int64_t ld_x, const void* r, int64_t ld_r, int64_t N, int32_t F,
                                 int32_t dtype, const void* w, const void* b, float eps, void* y, void* s, void* q,
                                 float* scale, void* block_scale, float* mean, float* rstd, void* stream) {
    if (int rc = ln_args(N, F, dtype)) return rc;
    if (ld_x < F || (r && ld_r < F) || !(eps >= 0.f)) return FACE_ERR_ARG;
    if (N == 0) return 0;
    if (!x || !w || (!r != !s) || (scale && block_scale) || (!q != !(scale || block_scale))) return FACE_ERR_ARG;
    if (!y != (scale != nullptr) || (block_scale && !rstd) || (mean && !rstd)) return FACE_ERR_ARG;
    const LnFwdArgs a = {x, r, ld_x, ld_r, N, F, w, b, eps, y, s, (uint8_t*)q, scale, (uint8_t*)block_scale, mean, rstd};
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const hipStream_t st = (hipStream_t)stream;
        return scale ? launch_ln_fwd<T, kLnQ8>(a, st) : block_scale ? launch_ln_fwd<T, kLnKept>(a, st) : launch_ln_fwd<T, kLn>(a, st);
    });
}

extern "C" int64_t face_layer_norm_rows_bwd_work(int64_t N, int32_t F) {
    if (N <= 0 || F <= 0 || F > kLnMax) return 0;
    return ln_bwd_grid(N, F, false) * F * 8;
}

extern "C" int face_layer_norm_rows_bwd(const void* s, int64_t ld_s, const void* q, const void* block_scale, const float* mean,
                                 const float* rstd, const void* dy, int64_t ld_dy, const void* ds, int64_t ld_ds, int64_t N,
                                 int32_t F, int32_t dtype, const void* w, void* dx, void* dw, void* db, void* work,
                                 int64_t work_bytes, void* stream) {
    if (int rc = ln_args(N, F, dtype)) return rc;
    if ((s && ld_s < F) || (dy && ld_dy < F) || (ds && ld_ds < F)) return FACE_ERR_ARG;
    if (!dx && !dw && !db) return 0;
    if (N && (!w || !rstd || (s ? !mean || q : !q || !block_scale))) return FACE_ERR_ARG;
    const bool sums = dw || db;
    if (sums && N && (!work || work_bytes < face_layer_norm_rows_bwd_work(N, F))) return FACE_ERR_ARG;
    if (N == 0 && !sums) return 0;
    const LnBwdArgs a = {s, ld_s, (const uint8_t*)q, (const uint8_t*)block_scale, mean, rstd, dy, ds, ld_dy, ld_ds, N, F, w, dx,
                         sums ? (float*)work : nullptr};
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const hipStream_t st = (hipStream_t)stream;
        return s || !q ? launch_ln_bwd<T, false>(a, (T*)dw, (T*)db, st) : launch_ln_bwd<T, true>(a, (T*)dw, (T*)db, st);
    });
}

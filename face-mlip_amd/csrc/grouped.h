// Products of rows with the weights of their group (gfx950): the slots of a plan, sorted by group, against
// one weight matrix per group, ragged row counts that only the device knows.
//
//   forward        y[a] = op(x[a / xdiv]) W[g]^T + b[g]
//   input gradient d[a] = (dy[a] W[g]) * op'(z[a / zdiv])
//   weights        dW[g] = sum over the group's slots of dy[a]^T op(x[a / xdiv]),  db[g] = sum of dy[a]
//
// with a = order[i] the slot at place i of its group's range [ptr[g], ptr[g + 1]). Slots behind ptr[G] belong to
// no group; their rows of y and d are written as zeros.
//
// A workgroup owns a tile of rows of ONE group and of output columns; which, it finds from ptr by a
// wave-wide prefix sum of the groups' tile counts, so no launch waits for a count on the host. The grid holds the most
// tiles that so many slots and groups can make; what is left over ends at once. Both operands go through
// LDS in chunks along the sum, the next chunk's loads in registers during the present one's products:
//   * 16-bit rows as they are, on v_mfma_f32_32x32x16, or through silu, in two limbs of their type and twice the products; e4m3 rows on v_mfma_scale_f32_32x32x64_f8f6f4 at unit
//     scales (twice the bf16 rate; fp32 results: see e4m3_wide), their row and column scales applied to the sum;
//   * fp32 rows as three bf16 limbs, split once as they are staged, six products each (common.h);
//   * an operand whose sum runs along its rows is read 16 bytes a lane; one whose sum runs down its columns (the
//     weights of the input gradient, both operands of the weight gradient) is staged as it lies in memory and
//     transposed by ds_read_b64_tr_b16 on the way to the matrix cores.
// Where a launch has few tiles eight waves share one 32 x 32 tile and split every chunk's k among them, joined in LDS
// at the end in a fixed order: such calls wait for memory, and more workgroups have more loads in flight.
//
// Large calls are bound by the matrix cores and the power they may draw, up to four workgroups per CU covering each other's
// waits (a second buffer per workgroup leaves room for fewer: 128 x 128 of bf16 543 -> 562 us, of e4m3 268 -> 342 us).
// 200,000 slots of 100,000 x 2304 -> 512, eight groups: bf16 534 us (883 TFLOP/s; the library's product of one matrix 500),
// e4m3 287 us (1.6 PFLOP/s), bf16 input gradient 799 us (590 TFLOP/s, 1.84 GB of fp32 rows written), then 461 us for the sum of
// a row's slots; with a row per slot, in 16 bits, 625 us. 200,000 slots 512 -> 2304 in bf16 647 us, with SiLU on load 1570 (1230
// in one limb, of sqrt 2 of the error): it keeps the rows from going to LDS directly and is formed again for each of 18 column
// tiles.
// 24,000 x 1440 -> 320 in fp32, three groups: 142 us (155 TFLOP/s of the 190 that six bf16 products allow), input
// gradient 156 us. 21 rows x 192 -> 97 in fp32 6.1 us; two rows x 2048 -> 2048 in bf16 8.8 us, 16.8 MB of weights, by 128
// workgroups on 256 CUs.
#pragma once
#include "elem.h"
#include <type_traits>

namespace face {

// 8-bit rows. The e4m3 instructions align the products of a step to the largest and cut what is below 2^-13 of it
// (measured: errors up to 2^-10.4 of the largest product, one large among 63 small ones of a sign). The sum so far takes no
// part in it: sums of 2304 positive products are off by no more than their rounding to 16 bits. Results of 16 bits
// take them all the same: the operands' own rounding is 2^-4 of that product. Results in fp32 do not: e4m3_wide
// rows become bf16 as they are staged, exactly, and their sums are fp32 sums, at the bf16 rate.
struct e4m3 {
    uint8_t v;
};
struct e4m3_wide {
    uint8_t v;
};

struct GroupedArgs {
    const void* x;                 // rows of the left operand (x, or dy of the input gradient)
    int64_t ld_x;
    int32_t xdiv;                  // its row of slot a is a / xdiv
    int32_t x_op;                  // 1: silu as it loads
    const void* w;
    int64_t ld_w, w_group;         // strides between weight rows and groups
    const void* bias;              // (G, ld_b) or null
    int64_t ld_b;
    const float *xs, *ws;          // e4m3: scale of every row of x, and (G, n) of the weights' rows
    void* y;
    int64_t ld_y;
    const void* z;                 // op' of the input gradient: rows a / zdiv, or null
    int64_t ld_z;
    int32_t zdiv;
    int32_t n, k;                  // output columns, length of the sum
    const int32_t *ptr, *order;
    int64_t slots;
    int32_t groups;
    int32_t col_tiles;
    int64_t tiles;                 // row tiles the grid holds
};

struct GroupedWArgs {
    const void* x;                 // (.., k) with silu as it loads if x_op
    int64_t ld_x;
    int32_t xdiv, x_op;
    uint32_t div_mul, div_shift;   // a / xdiv = a div_mul >> div_shift for a < 2^31
    const void* dy;                // (slots, n)
    int64_t ld_dy;
    void* dw;                      // (G, n, k)
    void* db;                      // (G, n) or null
    float* part;                   // 2 shares partial results of n k [+ n] sums
    int32_t n, k;
    const int32_t *ptr, *order;
    int64_t slots;
    int32_t groups;
    int32_t col_tiles, row_tiles;
    int32_t shares;                // of the places in order, `share` each; 1: a workgroup per group instead
    int64_t share;
};

// ---------------------------------------------------------------- operands
template <typename T>
struct Operand {                                 // bf16, f16: one plane of 16-byte chunks of eight
    static constexpr int kPlanes = 1, kElems = 8;
};
template <>
struct Operand<float> {                          // three bf16 limbs of eight values
    static constexpr int kPlanes = 3, kElems = 8;
};
template <>
struct Operand<e4m3> {
    static constexpr int kPlanes = 1, kElems = 16;
};
template <typename T>
constexpr bool kIsQ8 = __is_same(T, e4m3) || __is_same(T, e4m3_wide);

// A 16-byte chunk's worth of a row (two 16-byte loads of fp32), in flight.
template <typename T>
struct Held {
    v4u a;
};
template <>
struct Held<float> {
    v4u a, b;
};
template <>
struct Held<e4m3_wide> {
    uint64_t a;
};

// The chunk at p, all of it.
template <typename T>
__device__ __forceinline__ Held<T> hold(const T* p) {
    Held<T> h;
    if constexpr (__is_same(T, e4m3_wide)) {
        typedef uint64_t any __attribute__((aligned(1)));
        h.a = *reinterpret_cast<const any*>(p);
    } else {
        h.a = ld16(p);
        if constexpr (sizeof(T) == 4) h.b = ld16(p + 4);
    }
    return h;
}
// The elements [0, left) of the chunk at p, zero beyond.
template <typename T>
__device__ __forceinline__ Held<T> hold(const T* p, int left) {
    Held<T> h = {};
    if (left >= Operand<T>::kElems) {
        h = hold(p);
    } else if (left > 0) {
        if constexpr (__is_same(T, e4m3_wide)) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) h.a |= (uint64_t)p[e].v << (8 * e);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t v = e < left ? __builtin_bit_cast(uint32_t, p[e]) : 0u;
                if (e < 4) h.a[e & 3] = v;
                else h.b[e & 3] = v;
            }
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) h.a[e >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, p[e]) << (16 * (e & 1));
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (e < left) h.a[e >> 2] |= (uint32_t)p[e].v << (8 * (e & 3));
        }
    }
    return h;
}

// silu of fp32 rows as they are held.
__device__ __forceinline__ void apply_silu(Held<float>& h) {
    v4f a = __builtin_bit_cast(v4f, h.a), b = __builtin_bit_cast(v4f, h.b);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        a[e] = silu(a[e]);
        b[e] = silu(b[e]);
    }
    h.a = __builtin_bit_cast(v4u, a);
    h.b = __builtin_bit_cast(v4u, b);
}

// The planes of a held chunk.
template <typename T>
__device__ __forceinline__ void planes(const Held<T>& h, v4u o[Operand<T>::kPlanes]) {
    if constexpr (sizeof(T) == 4) {
        const Split8 s = split8(__builtin_bit_cast(v4f, h.a), __builtin_bit_cast(v4f, h.b));
        o[0] = __builtin_bit_cast(v4u, s.h);
        o[1] = __builtin_bit_cast(v4u, s.m);
        o[2] = __builtin_bit_cast(v4u, s.l);
    } else if constexpr (__is_same(T, e4m3_wide)) {
        const int lo = (int)(uint32_t)h.a, hi = (int)(uint32_t)(h.a >> 32);
        const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8(lo, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(lo, true);
        const v2f c = __builtin_amdgcn_cvt_pk_f32_fp8(hi, false), d = __builtin_amdgcn_cvt_pk_f32_fp8(hi, true);
        o[0] = (v4u){bf16_pair(a[0], a[1]), bf16_pair(b[0], b[1]), bf16_pair(c[0], c[1]), bf16_pair(d[0], d[1])};
    } else {
        o[0] = h.a;
    }
}
// The same to LDS, `plane` bytes apart. SILU, of 16-bit rows: silu in fp32 as two limbs of the rows' type, its rounding and what
// that left over (0 of an infinity), so that the product is as of the fp32 value and not of one rounded once more.
template <typename T, bool SILU = false>
__device__ __forceinline__ void put(char* at, int plane, const Held<T>& h) {
    constexpr int P = SILU ? 2 : Operand<T>::kPlanes;
    v4u o[P];
    if constexpr (SILU) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float a, b, ha, hb;
            unpack2<T>(h.a[e], a, b);
            a = silu(a);
            b = silu(b);
            o[0][e] = pack2<T>(a, b);
            unpack2<T>(o[0][e], ha, hb);
            a -= ha;
            b -= hb;
            o[1][e] = pack2<T>(a == a ? a : 0.f, b == b ? b : 0.f);
        }
    } else {
        planes(h, o);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) *reinterpret_cast<v4u*>(at + p * plane) = o[p];
}

// ---------------------------------------------------------------- LDS tiles
// R rows of C chunks of 16 bytes. Chunks are moved within a row by an XOR with the row number so that the
// lanes of an access meet different banks: ROWS tiles are read one chunk a lane down 32 rows, COLS tiles by the
// transposing read, four rows of two chunks per 16 lanes.
template <int R, int C, bool COLS>
struct Tile {
    static constexpr int kBytes = R * C * 16;
    // The chunk that lies at a place of the row, and the place of a chunk.
    __device__ static __forceinline__ int chunk(int row, int place) {
        if constexpr (COLS)
            return place ^ (C >= 16 ? ((row & 1) << 2) ^ ((row & 2) ? 10 : 0) : (C == 8 ? 2 * (row & 3) : (row & 2)));
        return place ^ (C >= 16 ? (row & 15) : (C == 8 ? (row & 7) ^ ((row >> 3) & 1) : ((row >> 1) & 3) ^ ((row >> 3) & 1)));
    }
    __device__ static __forceinline__ int at(int row, int c) { return (row * C + chunk(row, c)) * 16; }
};

typedef short v4s __attribute__((ext_vector_type(4)));
__device__ __forceinline__ v4s read_tr(const char* lds) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)lds);
}

// One lane's eight elements of the 32 x 16 operand at (row i0, element k0): lane i + 32 h holds k0 + 8 h .. + 7 of
// row i0 + i. A COLS tile holds k down its rows: 16 lanes fetch a 4 x 16 block and receive its transpose.
template <int R, int C, bool COLS>
__device__ __forceinline__ v4u fragment(const char* tile, int i0, int k0, int lane) {
    if constexpr (!COLS) {
        return *reinterpret_cast<const v4u*>(tile + Tile<R, C, false>::at(i0 + (lane & 31), (k0 >> 3) + (lane >> 5)));
    } else {
        const int t = lane & 15, q = lane >> 4;
        const int k = k0 + 8 * (q >> 1) + (t >> 2), col = i0 + 16 * (q & 1) + 4 * (t & 3);
        const v4s a = read_tr(tile + Tile<R, C, true>::at(k, col >> 3) + 2 * (col & 7));
        const v4s b = read_tr(tile + Tile<R, C, true>::at(k + 4, col >> 3) + 2 * (col & 7));
        typedef short v8s __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(v4u, (v8s)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

typedef f16 v8h __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));

template <typename T>
__device__ __forceinline__ v16f mfma16(v4u a, v4u b, v16f c) {
    if constexpr (__is_same(T, f16))
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    else
        return mfma_32x32x16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c);
}

// The products of one chunk: MT x NT tiles of 32 x 32, elements [k_begin, k_begin + STEPS * step) of the chunk. The
// column operand comes first, so that a lane ends with four neighbouring columns of one row at a time: register q of
// acc[m][n] is row lane & 31, column 8 (q >> 2) + 4 (lane >> 5) + (q & 3) of the tile.
template <typename T>
constexpr int kStep = __is_same(T, e4m3) ? 64 : 16;              // elements of the sum per instruction

// One step's operands: 8 (e4m3: 32, each half of the wave its own) neighbouring elements of a row per lane.
// PA, PB: planes of the operands, one each, three each, or two of one of them.
template <typename T, int PA, int PB, int RA, int CA, bool COLS_A, int RB, int CB, bool COLS_B, int MT, int NT>
struct Fragments {
    static constexpr int W = __is_same(T, e4m3) ? 2 : 1;
    static_assert((PA == 3 && PB == 3) || PA * PB <= 2, "no other order of products is written");
    v4u a[PA * W][MT], b[PB * W][NT];

    __device__ __forceinline__ void load(const char* ta, const char* tb, int m0, int n0, int k0, int lane) {
        if constexpr (__is_same(T, e4m3)) {
            const int c = (k0 >> 4) + 2 * (lane >> 5);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    a[h][m] = *reinterpret_cast<const v4u*>(ta + Tile<RA, CA, false>::at(m0 + 32 * m + (lane & 31), c + h));
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    b[h][n] = *reinterpret_cast<const v4u*>(tb + Tile<RB, CB, false>::at(n0 + 32 * n + (lane & 31), c + h));
            }
        } else {
            constexpr int kA = Tile<RA, CA, COLS_A>::kBytes, kB = Tile<RB, CB, COLS_B>::kBytes;
#pragma unroll
            for (int p = 0; p < (PA > PB ? PA : PB); ++p) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    if (p < PA) a[p][m] = fragment<RA, CA, COLS_A>(ta + p * kA, m0 + 32 * m, k0, lane);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    if (p < PB) b[p][n] = fragment<RB, CB, COLS_B>(tb + p * kB, n0 + 32 * n, k0, lane);
            }
        }
    }
    __device__ __forceinline__ void products(v16f acc[MT][NT]) const {
        if constexpr (__is_same(T, e4m3)) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const v8i x = __builtin_shufflevector(__builtin_bit_cast(v4i, a[0][m]), __builtin_bit_cast(v4i, a[1][m]), 0,
                                                          1, 2, 3, 4, 5, 6, 7);
                    const v8i w = __builtin_shufflevector(__builtin_bit_cast(v4i, b[0][n]), __builtin_bit_cast(v4i, b[1][n]), 0,
                                                          1, 2, 3, 4, 5, 6, 7);
                    acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, acc[m][n], 0, 0, 0, 0x7f7f7f7f, 0,
                                                                                0x7f7f7f7f);
                }
        } else {
            // limb products from the smallest up; of one instruction after another none waits for the one before
            constexpr int kProducts = PA == 3 ? 6 : PA * PB;
            constexpr int pa[6] = {0, 1, 2, 0, 1, 0}, pb[6] = {2, 1, 0, 1, 0, 0};
#pragma unroll
            for (int q = 0; q < kProducts; ++q)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        acc[m][n] = mfma16<T>(b[PA == 3 ? pb[q] : PB - 1 - q > 0 ? PB - 1 - q : 0][n],
                                              a[PA == 3 ? pa[q] : PA - 1 - q > 0 ? PA - 1 - q : 0][m], acc[m][n]);
        }
    }
};

template <typename T, int PA, int PB, int RA, int CA, bool COLS_A, int RB, int CB, bool COLS_B, int MT, int NT, int STEPS>
__device__ __forceinline__ void chunk_products(const char* ta, const char* tb, int m0, int n0, int k_begin, int lane,
                                               v16f acc[MT][NT]) {
    using F = Fragments<T, PA, PB, RA, CA, COLS_A, RB, CB, COLS_B, MT, NT>;
    if constexpr (MT * NT > 4) {
        // few waves per SIMD: the next step's operands are on their way during this one's products, and no more of
        // them (the barrier), or the accumulators would spill
        F f[2];
        f[0].load(ta, tb, m0, n0, k_begin, lane);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (s + 1 < STEPS) f[(s + 1) & 1].load(ta, tb, m0, n0, k_begin + (s + 1) * kStep<T>, lane);
            f[s & 1].products(acc);
            __builtin_amdgcn_sched_barrier(0);
        }
    } else {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            F f;
            f.load(ta, tb, m0, n0, k_begin + s * kStep<T>, lane);
            f.products(acc);
        }
    }
}

// Waves at their products go before waves of the CU's other workgroups that split operands into limbs, so that the
// matrix cores are fed first. fp32 24,000 x 1440 -> 320 (us, without / with): 148 / 143, input gradient 165 / 161, weights 183 /
// 180; 2304 -> 512 372 / 357, 346 / 333, 344 / 344. Of 16 and 8 bits nothing is split, and it costs 1 %: 271 / 280, 70.8 / 71.7.
template <typename T>
__device__ __forceinline__ void before_products() {
    if constexpr (Operand<T>::kPlanes > 1) __builtin_amdgcn_s_setprio(1);
}
template <typename T>
__device__ __forceinline__ void after_products() {
    if constexpr (Operand<T>::kPlanes > 1) __builtin_amdgcn_s_setprio(0);
}

// ---------------------------------------------------------------- staging without registers
// Operands whose 16-byte chunks are aligned and whole (launch_rows, launch_weight) go from memory to LDS directly:
// lane l of a wave fills the 16 bytes at 16 l of a stretch of 1 KB, so the chunk that belongs there by the tile's XOR is
// the one it loads. Chunks outside the operand come from a block of zeros.
__device__ const v4u kZeroChunk = {0, 0, 0, 0};
__device__ __forceinline__ void to_lds(const void* from, char* stretch) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)stretch, 16, 0, 0);
}

// ---------------------------------------------------------------- which rows a workgroup owns
__device__ __forceinline__ int64_t clamp_slot(int64_t v, int64_t slots) { return v < 0 ? 0 : (v > slots ? slots : v); }

struct Range {
    int group;                     // `groups`: the slots of no group; -1: nothing
    int64_t begin, end;            // its places in order
    int64_t index;                 // of this piece among the group's
};
// The t-th piece of `size` places of the groups 0 .. groups. The same in all threads.
__device__ __forceinline__ Range find_piece(const int32_t* ptr, int groups, int64_t slots, int size, int64_t t) {
    const int lane = threadIdx.x & 63;
    int64_t before = 0;
    for (int g0 = 0; g0 <= groups; g0 += 64) {
        const int g = g0 + lane;
        int64_t b = 0, e = 0;
        if (g <= groups) {
            b = clamp_slot(ptr[g], slots);
            e = g < groups ? clamp_slot(ptr[g + 1], slots) : slots;
        }
        const int c = e > b ? (int)((e - b + size - 1) / size) : 0;
        int s = c;
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(s, o, 64);
            if (lane >= o) s += u;
        }
        const int total = __shfl(s, 63, 64);
        if (t < before + total) {
            const int l = __builtin_ctzll(__ballot(before + s > t));
            return {g0 + l, __shfl(b, l, 64), __shfl(e, l, 64), t - (before + __shfl(s, l, 64) - __shfl(c, l, 64))};
        }
        before += total;
    }
    return {-1, 0, 0, 0};
}

// Workgroups that follow each other on one XCD (every eighth) take neighbouring items, so that tiles of the same
// rows and of the same weights meet in its L2.
__device__ __forceinline__ int64_t xcd_item(int64_t items) {
    const int64_t b = blockIdx.x, per = items / 8, rest = items % 8, x = b % 8;
    return x * per + (x < rest ? x : rest) + b / 8;
}

// ---------------------------------------------------------------- forward and input gradient
// WM x WN x WK waves of MT x NT tiles. COLS_B: the weights lie (sum, column), as the input gradient reads them.
// DIRECT_A, DIRECT_B: the operand is staged without registers. SILU: 16-bit rows through silu, in two limbs.
template <typename T, bool COLS_B, int WM, int WN, int WK, int MT, int NT, int C, bool SILU>
struct RowsKernel {
    using Op = Operand<T>;
    static constexpr int BM = 32 * MT * WM, BN = 32 * NT * WN, BK = C * Op::kElems;
    static constexpr int PA = SILU ? 2 : Op::kPlanes, PB = Op::kPlanes;
    static constexpr int kWaves = WM * WN * WK, kThreads = 64 * kWaves;
    static constexpr int CB = COLS_B ? BN / 8 : C, RB = COLS_B ? BK : BN;
    using TA = Tile<BM, C, false>;
    using TB = Tile<RB, CB, COLS_B>;
    static constexpr int kLdsA = PA * TA::kBytes, kLdsB = PB * TB::kBytes;
    // finished sums on their way out: 32 rows of a wave's columns at a time, rows four floats apart in the banks
    static constexpr int kOutLd = 32 * NT + 4, kOut = 32 * kOutLd * 4;
    static constexpr int kLds = kLdsA + kLdsB > kWaves * kOut ? kLdsA + kLdsB : kWaves * kOut;
    static constexpr int NA = BM * C / kThreads, NB = RB * CB / kThreads;   // chunks per thread
    static_assert(NA * kThreads == BM * C && NB * kThreads == RB * CB, "whole rounds of chunks");
    static_assert(WK == 1 || (WM == 1 && WN == 1 && MT == 1 && NT == 1), "split chunks: one tile");
};

// Out-of-range sums of limbs: a value past bf16's largest, or an infinity, has a NaN limb, so 32 x 32 tiles with a sum that is
// not finite are formed again by plain products of the fp32 operands, and such sums take the value found there. A wave does
// its own tile, through `lds` of 64 rows of kPlainLd floats: put(lds, from) stores the kPlain steps of the sum from `from`
// on, 32 values of each operand. The sum goes over the steps [first, first + run) of every `turn` (run a multiple of kPlain)
// before `end`, in order. Loops stay rolled, so that the path takes no registers from the products. 24,000 x 1440 -> 320,
// both directions, with nothing finite in it: 6.9 ms against 0.5 (and 117 with a lane per sum).
constexpr int kPlain = 8, kPlainLd = kPlain + 1;
__device__ __forceinline__ bool finite(float v) { return __builtin_fabsf(v) <= 0x1.fffffep+127f; }
__device__ __forceinline__ bool all_finite(const v16f& v) {
    bool f = true;
#pragma unroll
    for (int q = 0; q < 16; ++q) f = f && finite(v[q]);
    return f;
}
template <typename Put>
__device__ __forceinline__ void plain_tile(float* lds, int64_t first, int64_t run, int64_t turn, int64_t end, int lane, Put put,
                                           v16f& acc) {
    v16f s = {};
    for (int64_t at = first; at < end; at += turn)
        for (int64_t from = at; from < at + run && from < end; from += kPlain) {
            put(lds, from);
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int i = 0; i < kPlain; ++i) {
                const float a = lds[(lane & 31) * kPlainLd + i];
#pragma unroll
                for (int q = 0; q < 16; ++q)
                    s[q] = fmaf(a, lds[(32 + 8 * (q >> 2) + 4 * (lane >> 5) + (q & 3)) * kPlainLd + i], s[q]);
            }
            __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
    for (int q = 0; q < 16; ++q) acc[q] = finite(acc[q]) ? acc[q] : s[q];
}

// The epilogue of the eight columns from col of slot a, and their store.
template <typename T, typename Out, bool COLS_B>
__device__ __forceinline__ void finish(const GroupedArgs& g, int group, int32_t a, int col, float v[8]) {
    const int left = g.n - col;
    if (left <= 0) return;
    if constexpr (kIsQ8<T>) {
        const float sx = g.xs[a / g.xdiv];
        float s[8];
        load_piece(g.ws + (int64_t)group * g.n + col, left, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // one after the other where their product leaves the normal range, in which the result may still lie
            const float f = sx * s[e];
            v[e] = __builtin_amdgcn_classf(f, 0x108) ? v[e] * f : v[e] * sx * s[e];
        }
    }
    if (g.bias) {
        float s[8];
        load_piece((const Out*)g.bias + group * g.ld_b + col, left, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += s[e];
    }
    if constexpr (COLS_B) {
        if (g.z) {
            float z[8];
            load_piece((const T*)g.z + (int64_t)(a / g.zdiv) * g.ld_z + col, left, z);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= silu_slope(z[e]);
        }
    }
    store_piece((Out*)g.y + a * g.ld_y + col, left, v);
}

// A 32 x 32 tile of fp32 rows, where there are few: rows and weights go from memory to the matrix cores without LDS, and
// without a wait in common. Lane i + 32 h holds 16 values of row i and of weight row i; each wave takes every WK-th 128-byte
// stretch of all of them (32 whole lines an operand), the next one on its way while it multiplies the last. The order of
// k within a stretch is the lanes', the same for both operands. 21 rows in three groups (us, staged / so): 864 -> 192 10.9
// / 8.7, 1440 -> 320 15.8 / 11.7, 2304 -> 512 21.4 / 15.8; 100 rows 2048 -> 2048, 288 workgroups, 27.5 / 33.5: an access of 64
// lanes touches 32 lines. 16-bit rows gain a tenth up to 1440 columns and lose as much from 2304 on: they are staged.
template <int WK>
__device__ __forceinline__ void few_rows(const float* x, const float* w, int k, int x_op, int wave, int lane, v16f acc[1][1]) {
    constexpr int N = 2, E = 8, kLine = 2 * N * E;
    using F = Fragments<float, 3, 3, 32, 1, false, 32, 1, false, 1, 1>;
    const int half = N * E * (lane >> 5);
    struct Run {
        Held<float> a[N], b[N];
    };
    auto load = [&](Run& r, int turn) {
        const int p = (turn * WK + wave) * kLine + half;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            r.a[i] = hold(x + p + i * E);
            r.b[i] = hold(w + p + i * E);
        }
    };
    auto multiply = [&](Run& r) {
        if (x_op) {
#pragma unroll
            for (int i = 0; i < N; ++i) apply_silu(r.a[i]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v4u a[3], b[3];
            planes(r.a[i], a);
            planes(r.b[i], b);
            F f;
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                f.a[p][0] = a[p];
                f.b[p][0] = b[p];
            }
            f.products(acc);
        }
    };
    const int whole = k / kLine;                                 // stretches; this wave's: wave, wave + WK, ...
    const int turns = whole > wave ? (whole - wave + WK - 1) / WK : 0;
    // no branch between a load and its use: behind one the compiler waits for every load on its way
    Run r0, r1;
    int turn = 0;
    if (turns) load(r0, 0);
    for (; turn + 2 < turns; turn += 2) {
        load(r1, turn + 1);
        multiply(r0);
        load(r0, turn + 2);
        multiply(r1);
    }
    if (turn + 1 < turns) {
        load(r1, turn + 1);
        multiply(r0);
        multiply(r1);
    } else if (turn < turns) {
        multiply(r0);
    }
    if (k % kLine && whole % WK == wave) {                       // the last stretch, in part
        const int p = whole * kLine + half;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            r0.a[i] = hold(x + p + i * E, k - p - i * E);
            r0.b[i] = hold(w + p + i * E, k - p - i * E);
        }
        multiply(r0);
    }
}

template <typename T, typename Out, bool COLS_B, int WM, int WN, int WK, int MT, int NT, int C, bool DIRECT_A, bool DIRECT_B,
          bool FEW = false, bool SILU = false>
__global__ __launch_bounds__((RowsKernel<T, COLS_B, WM, WN, WK, MT, NT, C, SILU>::kThreads), (DIRECT_A ? 4 : 2)) void
    grouped_rows_kernel(GroupedArgs g) {
    using K = RowsKernel<T, COLS_B, WM, WN, WK, MT, NT, C, SILU>;
    static_assert(!SILU || (sizeof(T) == 2 && !DIRECT_A && !COLS_B), "rows of 16 bits, through registers");
    __shared__ __attribute__((aligned(256))) char lds[K::kLds];
    __shared__ int32_t slot_of[K::BM];
    const int64_t item = xcd_item(g.tiles * g.col_tiles);
    const int col0 = (int)(item % g.col_tiles) * K::BN;
    const Range r = find_piece(g.ptr, g.groups, g.slots, K::BM, item / g.col_tiles);
    if (r.group < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t place0 = r.begin + r.index * K::BM;
    for (int i = tid; i < K::BM; i += K::kThreads) {
        int32_t a = -1;
        if (place0 + i < r.end) a = g.order[place0 + i];
        slot_of[i] = a >= 0 && a < g.slots ? a : -1;
    }
    __syncthreads();
    if (r.group == g.groups) {
        Out* y = (Out*)g.y;
        for (int i = wave; i < K::BM; i += K::kWaves) {
            const int32_t a = slot_of[i];
            if (a < 0) continue;
            for (int c = lane; c < K::BN; c += 64)
                if (col0 + c < g.n) y[a * g.ld_y + col0 + c] = from_f<Out>(0.f);
        }
        return;
    }
    const T* w = (const T*)g.w + r.group * g.w_group;
    const T* x = (const T*)g.x;

    // This thread's chunks: chunk tid % C of row tid / C, the next ones kThreads / C rows on (directly: the same places of
    // the tile, and the chunk that the XOR puts there, the same in all of the thread's rows). Rows of x and columns of the
    // weights that are not there repeat one that is: what comes of them is not stored.
    const T* ap[K::NA];
    uint32_t b_off[K::NB];                   // bytes from the group's weights
    const int a_col = (DIRECT_A ? K::TA::chunk(tid / C, tid % C) : tid % C) * K::Op::kElems;
    const int b_chunk = DIRECT_B ? K::TB::chunk(tid / K::CB, tid % K::CB) : tid % K::CB;
    const int b_col = COLS_B ? col0 + 8 * b_chunk : b_chunk * K::Op::kElems;     // along the row
    const char* wb = (const char*)w;
#pragma unroll
    for (int i = 0; i < K::NA; ++i) {
        const int32_t a = slot_of[tid / C + i * (K::kThreads / C)];
        ap[i] = x + (int64_t)(a < 0 ? 0 : a / g.xdiv) * g.ld_x + a_col;
    }
    if constexpr (DIRECT_B) {
#pragma unroll
        for (int i = 0; i < K::NB; ++i) {
            const int row = tid / K::CB + i * (K::kThreads / K::CB);
            const int wr = COLS_B || col0 + row < g.n ? row : 0, wc = COLS_B && b_col >= g.n ? 0 : b_col;
            b_off[i] = (uint32_t)(((COLS_B ? wr : col0 + wr) * g.ld_w + wc) * sizeof(T));
        }
    }
    const int64_t w_step = (COLS_B ? g.ld_w : 1) * (int64_t)sizeof(T);           // one place of the sum
    // the next chunk in registers; whole chunks are loaded without a branch per lane
    Held<T> ha[DIRECT_A ? 1 : K::NA], hb[DIRECT_B ? 1 : K::NB];
    const bool cols_whole = !COLS_B || col0 + K::BN <= g.n;
    auto fetch = [&](int k0) {
        if (k0 >= g.k) return;
        if (k0 + K::BK <= g.k && cols_whole) {
            if constexpr (!DIRECT_A) {
#pragma unroll
                for (int i = 0; i < K::NA; ++i) ha[i] = hold(ap[i] + k0);
            }
            if constexpr (!DIRECT_B) {
#pragma unroll
                for (int i = 0; i < K::NB; ++i) {
                    const int row = tid / K::CB + i * (K::kThreads / K::CB);
                    hb[i] = hold(COLS_B ? w + (k0 + row) * g.ld_w + b_col
                                             : w + (col0 + row < g.n ? col0 + row : col0) * g.ld_w + b_col + k0);
                }
            }
        } else {
            if constexpr (!DIRECT_A) {
#pragma unroll
                for (int i = 0; i < K::NA; ++i) ha[i] = hold(ap[i] + k0, g.k - a_col - k0);
            }
            if constexpr (!DIRECT_B) {
#pragma unroll
                for (int i = 0; i < K::NB; ++i) {
                    const int row = tid / K::CB + i * (K::kThreads / K::CB);
                    if constexpr (COLS_B)
                        hb[i] = hold(w + (k0 + row) * g.ld_w + b_col, k0 + row < g.k ? g.n - b_col : 0);
                    else
                        hb[i] = hold(w + (col0 + row) * g.ld_w + b_col + k0, col0 + row < g.n ? g.k - b_col - k0 : 0);
                }
            }
        }
    };
    v16f acc[MT][NT] = {};
    const int wk = wave % WK, wn = wave / WK % WN, wm = wave / WK / WN;
    // WHOLE: the chunk ends within the sum; else what lies past its end is zeros, in both operands
    auto stage_a = [&](int k0, char* to, auto whole) {
        if constexpr (DIRECT_A) {
#pragma unroll
            for (int i = 0; i < K::NA; ++i)
                to_lds(decltype(whole)::value || a_col + k0 < g.k ? (const void*)(ap[i] + k0) : &kZeroChunk,
                       to + (i * K::kThreads + wave * 64) * 16);
        } else {
            if constexpr (__is_same(T, float)) {
                if (g.x_op) {
#pragma unroll
                    for (int i = 0; i < K::NA; ++i) apply_silu(ha[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < K::NA; ++i)
                put<T, SILU>(to + K::TA::at(tid / C + i * (K::kThreads / C), tid % C), K::TA::kBytes, ha[i]);
        }
    };
    auto stage_b = [&](int k0, char* to, auto whole) {
        if constexpr (DIRECT_B) {
            const char* base = wb + k0 * w_step;
#pragma unroll
            for (int i = 0; i < K::NB; ++i) {
                const int at = COLS_B ? tid / K::CB + i * (K::kThreads / K::CB) : b_col;     // place in the chunk
                to_lds(decltype(whole)::value || at + k0 < g.k ? (const void*)(base + b_off[i]) : &kZeroChunk,
                       to + (i * K::kThreads + wave * 64) * 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < K::NB; ++i)
                put(to + K::TB::at(tid / K::CB + i * (K::kThreads / K::CB), tid % K::CB), K::TB::kBytes, hb[i]);
        }
    };
    if constexpr (FEW) {
        static_assert(WK > 1 && !COLS_B, "rows of the sum on both sides");
        const int32_t a = slot_of[lane & 31];
        const int col = col0 + (lane & 31);
        few_rows<WK>(x + (int64_t)(a < 0 ? 0 : a / g.xdiv) * g.ld_x, w + (col < g.n ? col : col0) * g.ld_w, g.k, g.x_op, wave, lane,
                     acc);
    } else {
        fetch(0);
        for (int k0 = 0; k0 < g.k; k0 += K::BK) {
            if (k0 + K::BK <= g.k) {
                stage_a(k0, lds, std::true_type{});
                stage_b(k0, lds + K::kLdsA, std::true_type{});
            } else {
                stage_a(k0, lds, std::false_type{});
                stage_b(k0, lds + K::kLdsA, std::false_type{});
            }
            __syncthreads();
            fetch(k0 + K::BK);
            before_products<T>();
            chunk_products<T, K::PA, K::PB, K::BM, C, false, K::RB, K::CB, COLS_B, MT, NT, K::BK / WK / kStep<T>>(
                lds, lds + K::kLdsA, 32 * MT * wm, 32 * NT * wn, wk * (K::BK / WK), lane, acc);
            after_products<T>();
            __syncthreads();
        }
    }

    if constexpr (__is_same(T, float)) {
        // the steps of the sum that this wave's products took, in runs of `run`
        constexpr int run = FEW ? 32 : K::BK / WK;
        static_assert(run % kPlain == 0 && 2 * 32 * kPlainLd * 4 <= K::kOut, "room for the steps in the wave's rows");
        float* steps = reinterpret_cast<float*>(lds) + wave * (K::kOut / 4);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int row0 = 32 * (MT * wm + m);
            const bool there = slot_of[row0 + (lane & 31)] >= 0;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (!__any(there && !all_finite(acc[m][n]))) continue;
                const int c0 = col0 + 32 * (NT * wn + n);
                // eight steps of eight rows a turn
                plain_tile(steps, wk * run, run, WK * run, g.k, lane,
                           [&](float* to, int64_t from) {
                               const int i = lane & 7;
                               const bool in = from + i < g.k;
#pragma unroll 1
                               for (int r = lane >> 3; r < 32; r += 8) {
                                   const int32_t a = slot_of[row0 + r];
                                   const float v = in && a >= 0 ? x[(int64_t)(a / g.xdiv) * g.ld_x + from + i] : 0.f;
                                   to[r * kPlainLd + i] = g.x_op ? silu(v) : v;
                                   const int64_t c = c0 + r;
                                   to[(32 + r) * kPlainLd + i] =
                                       in && c < g.n ? (COLS_B ? w[(from + i) * g.ld_w + c] : w[c * g.ld_w + from + i]) : 0.f;
                               }
                           },
                           acc[m][n]);
            }
        }
    }

    // Out through LDS: whole rows of eight columns a lane, so that the stores (and the reads of z) are whole lines
    float* out = reinterpret_cast<float*>(lds) + wave * (K::kOut / 4);
    if constexpr (WK > 1) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            st4(out + (lane & 31) * K::kOutLd + 8 * q + 4 * (lane >> 5),
                (v4f){acc[0][0][4 * q], acc[0][0][4 * q + 1], acc[0][0][4 * q + 2], acc[0][0][4 * q + 3]});
        __syncthreads();
        const int row = tid >> 2, c = 8 * (tid & 3);
        if (tid < 128 && slot_of[row] >= 0) {
            float v[8] = {};
#pragma unroll
            for (int u = 0; u < WK; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += reinterpret_cast<const float*>(lds)[u * (K::kOut / 4) + row * K::kOutLd + c + e];
            finish<T, Out, COLS_B>(g, r.group, slot_of[row], col0 + c, v);
        }
    } else {
        constexpr int kLanes = 4 * NT;                           // lanes per row, eight columns each
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    st4(out + (lane & 31) * K::kOutLd + 32 * n + 8 * q + 4 * (lane >> 5),
                        (v4f){acc[m][n][4 * q], acc[m][n][4 * q + 1], acc[m][n][4 * q + 2], acc[m][n][4 * q + 3]});
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < 32 * kLanes / 64; ++i) {
                const int row = lane / kLanes + i * (64 / kLanes), c = 8 * (lane % kLanes);
                const v4f lo = ld4(out + row * K::kOutLd + c), hi = ld4(out + row * K::kOutLd + c + 4);
                float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                const int32_t a = slot_of[32 * (MT * wm + m) + row];
                if (a >= 0) finish<T, Out, COLS_B>(g, r.group, a, col0 + 32 * NT * wn + c, v);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// ---------------------------------------------------------------- weight gradient
// 128 x 128 tiles (n, k), the sum down the places of order. The places are cut into equal shares (weight_shares),
// wherever the groups end: a workgroup per share and tile goes through the groups of its share.
// A group that lies within one share is finished there; of the others each share leaves a partial result, two at most (of its
// first and its last group), which grouped_join_kernel adds in order: no atomics. 200,000 slots, 512 x 2304, eight
// groups, bf16: 673 us in 128 x 128 tiles, against 780 us with chunks of single groups (2.25 rounds of workgroups of
// unlike length), and 578 us in 256 x 256 tiles: 816 TFLOP/s.
// TILE 256 (16-bit operands staged without registers): 256 x 256 by eight waves of 128 x 64, into two buffers in turn, the next
// slots on their way during the present ones' products. It spills 46 registers, the 128 x 128 tile staged so 25 to 27: places of
// the results, stored before the loop over the groups and read where the results are, none in the loop over the slots.
// The tile's padding is multiplied too: 1440 x 320 becomes 1536 x 384, 28 % more.
// SILU: x through silu, in two limbs.
template <typename T, int TILE, bool SILU>
struct WeightKernel {
    using Op = Operand<T>;
    static constexpr int P = Op::kPlanes, PX = SILU ? 2 : P, BK = P == 3 ? 32 : 64, CT = TILE / 8;
    static constexpr int WM = 2, WN = TILE / 64, MT = TILE / 64, NT = 2, kThreads = 64 * WM * WN;
    using TT = Tile<BK, CT, true>;
    static constexpr int kLds = (P + PX) * TT::kBytes, NC = BK * CT / kThreads;
};

template <typename T, bool DIRECT, int TILE, bool SILU>
__global__ __launch_bounds__((WeightKernel<T, TILE, SILU>::kThreads), (DIRECT && TILE == 128 ? 4 : 2)) void grouped_weight_kernel(
    GroupedWArgs g) {
    using K = WeightKernel<T, TILE, SILU>;
    static_assert(!SILU || (sizeof(T) == 2 && !DIRECT), "rows of 16 bits, through registers");
    constexpr bool kTwo = TILE == 256;
    static_assert(DIRECT || !kTwo, "two buffers are filled without registers");
    // two arrays, not one of twice the size: reads of one need not wait for what is on its way into the other
    __shared__ __attribute__((aligned(256))) char lds[K::kLds];
    __shared__ __attribute__((aligned(256))) char lds_2[kTwo ? K::kLds : 16];
    const int64_t per = (int64_t)g.row_tiles * g.col_tiles;
    const int64_t item = xcd_item(per * (g.shares > 1 ? g.shares : g.groups));
    const int row0 = (int)(item % per / g.col_tiles) * TILE, col0 = (int)(item % g.col_tiles) * TILE;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *x = (const T*)g.x, *dy = (const T*)g.dy;
    constexpr int kB = K::P * K::TT::kBytes;                     // where x lies behind dy
    const int unit = (int)(item / per);                          // share or group
    int64_t s0 = 0, s1 = g.slots;
    int group = unit, last = unit;
    if (g.shares > 1) {
        const int64_t lo = clamp_slot(g.ptr[0], g.slots), hi = clamp_slot(g.ptr[g.groups], g.slots);
        s0 = lo + unit * g.share;
        s1 = s0 + g.share < hi ? s0 + g.share : hi;
        if (s0 >= s1) return;
        // the first group that ends behind s0
        last = g.groups - 1;
        for (group = 0; group <= last; group += 64) {
            const int e = group + lane;
            const uint64_t m = __ballot(e <= last && g.ptr[e + 1] > s0);
            if (m) {
                group += __builtin_ctzll(m);
                break;
            }
        }
    }

    // chunk tid % CT (directly: the one the XOR puts there, the same in all of the thread's rows, four apart)
    const int row_t = tid / K::CT, chunk = DIRECT ? K::TT::chunk(row_t, tid % K::CT) : tid % K::CT;
    const int ca = row0 + 8 * chunk, cb = col0 + 8 * chunk;
    const bool sums = g.db && col0 == 0;
    const int64_t stride = (int64_t)g.n * g.k + (g.db ? g.n : 0);
    const int wn = wave % K::WN, wm = wave / K::WN, slots = (int)g.slots;
    float colsum[8];
    int32_t next[K::NC];
    const uint32_t ld_a = (uint32_t)(g.ld_dy * sizeof(T)), ld_b = (uint32_t)(g.ld_x * sizeof(T));
    const int32_t* order;
    int rows;                                                    // of the present group in this share
    // The slots of the thread's rows from p on: fetched without a branch or a test, either of which would wait for them
    // (and for the operands on their way before them) at once; slot() tests one where it is used, -1: no row.
    auto find = [&](int p) {
#pragma unroll
        for (int i = 0; i < K::NC; ++i) {
            const int at = p + row_t + i * (K::kThreads / K::CT);
            next[i] = order[at < rows ? at : 0];
        }
    };
    auto slot = [&](int p, int i) {
        return p + row_t + i * (K::kThreads / K::CT) < rows && next[i] < slots ? next[i] : -1;
    };
    Held<T> ha[DIRECT ? 1 : K::NC], hb[DIRECT ? 1 : K::NC];
    auto fetch = [&](int p) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int i = 0; i < K::NC; ++i) {
                const int32_t a = slot(p, i);
                ha[i] = hold(dy + (a >= 0 ? a * g.ld_dy + ca : 0), a >= 0 ? g.n - ca : 0);
                const uint32_t ra = (uint32_t)((uint64_t)(uint32_t)a * g.div_mul >> g.div_shift);
                hb[i] = hold(x + (a >= 0 ? (int64_t)ra * g.ld_x + cb : 0), a >= 0 ? g.k - cb : 0);
            }
        }
    };
    auto add_columns = [&](v4u lo, v4u hi) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (sizeof(T) == 4) {
                colsum[e] += __builtin_bit_cast(v4f, lo)[e];
                colsum[4 + e] += __builtin_bit_cast(v4f, hi)[e];
            } else {
                float u, v;
                unpack2<T>(lo[e], u, v);
                colsum[2 * e] += u;
                colsum[2 * e + 1] += v;
            }
        }
    };
    for (; group <= last; ++group) {
        const int64_t g0 = clamp_slot(g.ptr[group], g.slots), g1 = clamp_slot(g.ptr[group + 1], g.slots);
        const int64_t p0 = g0 > s0 ? g0 : s0, p1 = g1 < s1 ? g1 : s1;
        if (g.shares > 1) {
            if (p0 >= s1) break;
            if (p0 >= p1) continue;                              // a group without slots: grouped_join_kernel
        }
        rows = p1 > p0 ? (int)(p1 - p0) : 0;
        order = rows ? g.order + p0 : g.ptr;                     // something to read where there is nothing
        v16f acc[K::MT][K::NT] = {};
#pragma unroll
        for (int e = 0; e < 8; ++e) colsum[e] = 0.f;
        // DIRECT: the rows from p on, into LDS
        auto stage = [&](int p, char* to) {
#pragma unroll
            for (int i = 0; i < K::NC; ++i) {
                // strides below 2^31 bytes: one multiply-add an address
                const int32_t s = slot(p, i);
                const uint32_t a = (uint32_t)s, ra = (uint32_t)((uint64_t)a * g.div_mul >> g.div_shift);
                const char* pa = (const char*)(dy + ca) + (uint64_t)a * ld_a;
                const char* pb = (const char*)(x + cb) + (uint64_t)ra * ld_b;
                char* at = to + (i * K::kThreads + wave * 64) * 16;
                to_lds(s >= 0 && ca < g.n ? pa : (const char*)&kZeroChunk, at);
                to_lds(s >= 0 && cb < g.k ? pb : (const char*)&kZeroChunk, at + kB);
            }
        };
        auto products = [&](const char* from) {
            if (DIRECT && sums) {                                // the thread's own chunks again, from LDS
#pragma unroll
                for (int i = 0; i < K::NC; ++i) {
                    const v4u v = *reinterpret_cast<const v4u*>(from + (i * K::kThreads + tid) * 16);
                    add_columns(v, v);
                }
            }
            chunk_products<T, K::P, K::PX, K::BK, K::CT, true, K::BK, K::CT, true, K::MT, K::NT, K::BK / 16>(
                from, from + kB, 32 * K::MT * wm, 32 * K::NT * wn, 0, lane, acc);
        };
        find(0);
        if constexpr (kTwo) {
            stage(0, lds);
            find(K::BK);
            int p = 0;
            for (; p + K::BK < rows; p += 2 * K::BK) {
                __syncthreads();
                stage(p + K::BK, lds_2);
                find(p + 2 * K::BK);
                products(lds);
                __syncthreads();
                if (p + 2 * K::BK < rows) {
                    stage(p + 2 * K::BK, lds);
                    find(p + 3 * K::BK);
                }
                products(lds_2);
            }
            __syncthreads();
            if (p < rows) products(lds);
        } else {
            fetch(0);
            if constexpr (!DIRECT) find(K::BK);
            for (int p = 0; p < rows; p += K::BK) {
                if constexpr (DIRECT) {
                    stage(p, lds);
                    find(p + K::BK);
                } else {
                    if constexpr (__is_same(T, float)) {
                        if (g.x_op) {
#pragma unroll
                            for (int i = 0; i < K::NC; ++i) apply_silu(hb[i]);
                        }
                    }
                    if (sums) {
#pragma unroll
                        for (int i = 0; i < K::NC; ++i) {
                            if constexpr (sizeof(T) == 4) add_columns(ha[i].a, ha[i].b);
                            else add_columns(ha[i].a, ha[i].a);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < K::NC; ++i) {
                        const int at = K::TT::at(row_t + i * (K::kThreads / K::CT), chunk);
                        put(lds + at, K::TT::kBytes, ha[i]);
                        put<T, SILU>(lds + kB + at, K::TT::kBytes, hb[i]);
                    }
                }
                __syncthreads();
                if (!DIRECT && p + K::BK < rows) {
                    fetch(p + K::BK);
                    find(p + 2 * K::BK);
                }
                before_products<T>();
                products(lds);
                after_products<T>();
                __syncthreads();
            }
        }
        if constexpr (__is_same(T, float)) {
            constexpr int kWaves = K::kThreads / 64;
            static_assert(K::kLds >= kWaves * 2 * 32 * kPlainLd * 4, "room for the steps of all waves");
            float* steps = reinterpret_cast<float*>(lds) + wave * 2 * 32 * kPlainLd;
#pragma unroll
            for (int m = 0; m < K::MT; ++m)
#pragma unroll
                for (int n = 0; n < K::NT; ++n) {
                    if (!__any(!all_finite(acc[m][n]))) continue;
                    const int row = row0 + 32 * (K::MT * wm + m) + (lane & 31), col = col0 + 32 * (K::NT * wn + n) + (lane & 31);
                    // a slot's 32 values of each operand by half a wave
                    plain_tile(steps, 0, kPlain, kPlain, rows, lane,
                               [&](float* to, int64_t from) {
#pragma unroll 1
                                   for (int i = lane >> 5; i < kPlain; i += 2) {
                                       int32_t a = from + i < rows ? order[from + i] : -1;
                                       if (a >= slots) a = -1;
                                       to[(lane & 31) * kPlainLd + i] = a >= 0 && row < g.n ? dy[a * g.ld_dy + row] : 0.f;
                                       const float v = a >= 0 && col < g.k ? x[(int64_t)(a / g.xdiv) * g.ld_x + col] : 0.f;
                                       to[(32 + (lane & 31)) * kPlainLd + i] = g.x_op ? silu(v) : v;
                                   }
                               },
                               acc[m][n]);
                }
        }
        float* part = g0 >= s0 && g1 <= s1 ? nullptr : g.part + (2 * (int64_t)unit + (p0 > s0)) * stride;
        T* dw = (T*)g.dw + (int64_t)group * g.n * g.k;
        // out through LDS as in the forward: 32 rows of 64 columns of a wave at a time
        constexpr int kLd = 68;
        static_assert(K::kLds >= K::WN * 32 * kLd * 4, "room for the rows of the waves of one turn");
        float* out = reinterpret_cast<float*>(lds) + wn * 32 * kLd;
#pragma unroll
        for (int turn = 0; turn < K::WM; ++turn) {
            __syncthreads();
            if (wm != turn) continue;
#pragma unroll
            for (int m = 0; m < K::MT; ++m) {
#pragma unroll
                for (int n = 0; n < K::NT; ++n)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        st4(out + (lane & 31) * kLd + 32 * n + 8 * q + 4 * (lane >> 5),
                            (v4f){acc[m][n][4 * q], acc[m][n][4 * q + 1], acc[m][n][4 * q + 2], acc[m][n][4 * q + 3]});
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = (lane >> 3) + 8 * i, row = row0 + 32 * (K::MT * wm + m) + at, c = 8 * (lane & 7);
                    const int col = col0 + 64 * wn + c, left = g.k - col;
                    const v4f lo = ld4(out + at * kLd + c), hi = ld4(out + at * kLd + c + 4);
                    float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    if (row >= g.n || left <= 0) continue;
                    if (part)
                        store_piece(part + (int64_t)row * g.k + col, left, v);
                    else
                        store_piece(dw + (int64_t)row * g.k + col, left, v);
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
        if (sums) {
            __syncthreads();
            float* red = reinterpret_cast<float*>(lds);          // 16 threads per chunk of eight columns
#pragma unroll
            for (int e = 0; e < 8; ++e) red[row_t * TILE + 8 * chunk + e] = colsum[e];
            __syncthreads();
            if (tid < TILE && row0 + tid < g.n) {
                float s = 0.f;
                for (int i = 0; i < K::kThreads / K::CT; ++i) s += red[i * TILE + tid];
                if (part)
                    part[(int64_t)g.n * g.k + row0 + tid] = s;
                else
                    ((T*)g.db)[(int64_t)group * g.n + row0 + tid] = from_f<T>(s);
            }
        }
        __syncthreads();                                             // LDS is free for the next group
    }
}

// dW and db of the groups that lie in several shares: their partial sums, in order. Zeros for groups without slots.
template <typename T>
__global__ __launch_bounds__(256) void grouped_join_kernel(GroupedWArgs g) {
    const int group = blockIdx.y;
    const int64_t lo = clamp_slot(g.ptr[0], g.slots), hi = clamp_slot(g.ptr[g.groups], g.slots);
    int64_t b = clamp_slot(g.ptr[group], g.slots), e = clamp_slot(g.ptr[group + 1], g.slots);
    b = b > lo ? b : lo;
    e = e < hi ? e : hi;
    const bool none = e <= b;
    const int64_t first = none ? 0 : (b - lo) / g.share, last = none ? 0 : (e - 1 - lo) / g.share;
    if ((!none && first == last) || last >= g.shares) return;
    const int64_t nk = (int64_t)g.n * g.k, stride = nk + (g.db ? g.n : 0);
    const float* head = g.part + (2 * first + (b > lo + first * g.share)) * stride;
    const float* rest = g.part + 2 * (first + 1) * stride;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < stride; i += (int64_t)gridDim.x * 256) {
        float s = none ? 0.f : head[i];
#pragma unroll 4
        for (int64_t c = 0; c < last - first; ++c) s += rest[2 * c * stride + i];
        if (i < nk)
            ((T*)g.dw)[group * nk + i] = from_f<T>(s);
        else
            ((T*)g.db)[(int64_t)group * g.n + i - nk] = from_f<T>(s);
    }
}

// ---------------------------------------------------------------- launches
// Instantiated per element type in a file of its own (grouped_f32.hip, ...).
template <typename T, typename Out, bool COLS_B, int WM, int WN, int WK, int MT, int NT, int C, bool DIRECT_A, bool DIRECT_B,
          bool FEW = false, bool SILU = false>
static int launch_rows_shape(GroupedArgs g, hipStream_t st) {
    using K = RowsKernel<T, COLS_B, WM, WN, WK, MT, NT, C, SILU>;
    const int64_t most = g.groups + (int64_t)1;
    g.tiles = g.slots / K::BM + (most < g.slots ? most : g.slots);
    g.col_tiles = (g.n + K::BN - 1) / K::BN;
    const int64_t grid = g.tiles * g.col_tiles;
    if (grid > 0x7fffffff) return FACE_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((grouped_rows_kernel<T, Out, COLS_B, WM, WN, WK, MT, NT, C, DIRECT_A, DIRECT_B, FEW, SILU>),
                       dim3((unsigned)grid), dim3(K::kThreads), 0, st, g);
    FACE_LAUNCH_CHECK();
    return 0;
}

// Whether rows of `width` elements at p, `ld` apart, are whole 16-byte chunks at 16-byte addresses.
template <typename T>
static inline bool whole_chunks(const void* p, int64_t ld, int64_t width) {
    constexpr int E = 16 / sizeof(T);
    return sizeof(T) < 4 && !__is_same(T, e4m3_wide) && (uintptr_t)p % 16 == 0 && ld % E == 0 && width % E == 0;
}

template <typename T, typename Out, bool COLS_B, int MT, int NT>
static int launch_rows_large(GroupedArgs g, hipStream_t st) {
    constexpr int C = sizeof(T) == 4 ? 4 : 8;
    if constexpr (sizeof(T) < 4 && !__is_same(T, e4m3_wide)) {
        const bool a = whole_chunks<T>(g.x, g.ld_x, g.k);
        const bool b = whole_chunks<T>(g.w, g.ld_w, COLS_B ? g.n : g.k) && g.w_group % (16 / (int)sizeof(T)) == 0 &&
                       (COLS_B ? 64 : (int64_t)g.n) * g.ld_w * (int64_t)sizeof(T) < ((int64_t)1 << 31);
        if constexpr (sizeof(T) == 2 && !COLS_B) {
            if (g.x_op)
                return b ? launch_rows_shape<T, Out, COLS_B, 2, 2, 1, MT, NT, C, false, true, false, true>(g, st)
                         : launch_rows_shape<T, Out, COLS_B, 2, 2, 1, MT, NT, C, false, false, false, true>(g, st);
        }
        if (a && b) return launch_rows_shape<T, Out, COLS_B, 2, 2, 1, MT, NT, C, true, true>(g, st);
        if (b) return launch_rows_shape<T, Out, COLS_B, 2, 2, 1, MT, NT, C, false, true>(g, st);
    }
    return launch_rows_shape<T, Out, COLS_B, 2, 2, 1, MT, NT, C, false, false>(g, st);
}

// The tile: of a workgroup's chunks each waits `wait` ns for memory and barriers and takes `work` ns for each of the
// workgroups that a CU has to do, so a launch takes about chunks (wait + work max(1, tiles / CUs)); the shape with the
// least is launched. Fitted to 400 sizes of 21 to 100,000 slots and widths of 97 to 2304, on which its choice is 0.7 % slower
// than the best on average (whole rounds of workgroups in place of the quotient: 2 % for fp32, 0.8 % for the others), 17 %
// at worst (us; 32 x 32 split eight ways / 64 x 64 / 128 x 64 / 128 x 128):
//   fp32, 2304 -> 512:    21 slots 16 / 60 / 87 / 125, 3,000 slots 90 / 80 / 89 / 129, 12,000 slots 311 / 203 / 211 / 182
//   fp32, 1440 -> 320:    1,344 slots 23 / 40 / 57 / 83, 12,000 slots 128 / 89 / 82 / 106
//   bf16, 2304 -> 512:    21 slots 9.0 / 18 / 22 / 30, 3,000 slots 33 / 27 / 32 / 41, 12,000 slots 99 / 47 / 50 / 46
//   bf16, 2304 <- 512:    400 slots 12.7 / 8.2 / 9.6 / 12, 12,000 slots 182 / 55 / 51 / 42
//   e4m3, 2304 -> 512:    21 slots 6.5 / 10 / 13 / 16, 3,000 slots 25 / 15 / 18 / 23, 12,000 slots 79 / 28 / 28 / 28
struct RowsShape {
    int rows, cols, bytes, wait, work;       // bytes: of a row's chunk in the 16-bit or 8-bit operand (of 32 bits: half)
};
// Tiles of rows x cols: a group ends in the middle of one on average.
static inline int64_t expected_tiles(int64_t slots, int64_t groups, int n, int rows, int cols) {
    groups = groups < slots ? groups : slots;
    const int64_t t = slots / rows + groups / 2;
    return (t > groups ? t : groups) * ((n + cols - 1) / cols);
}
template <typename T, bool COLS_B>
static inline int rows_shape(int64_t slots, int64_t groups, int n, int k) {
    constexpr RowsShape f32[4] = {{32, 32, 256, 320, 570}, {64, 64, 64, 350, 310}, {128, 64, 64, 400, 580}, {128, 128, 64, 440, 1130}};
    constexpr RowsShape low[4] = {{32, 32, 512, 680, COLS_B ? 550 : 280}, {64, 64, 128, 170, 190}, {128, 64, 128, 720, 190},
                                  {128, 128, 128, 780, 290}};
    const double cus = (double)device_cu_count();
    int best = 0;
    double least = 0;
    for (int i = 0; i < 4; ++i) {
        const RowsShape& s = sizeof(T) == 4 ? f32[i] : low[i];
        const double load = (double)expected_tiles(slots, groups, n, s.rows, s.cols) / cus;
        const int64_t chunk = s.bytes / (__is_same(T, e4m3) ? 1 : 2), chunks = (k + chunk - 1) / chunk;
        const double ns = (double)chunks * (s.wait + s.work * (load > 1 ? load : 1));
        if (i == 0 || ns < least) {
            least = ns;
            best = i;
        }
    }
    return best;
}

template <typename T, typename Out, bool COLS_B>
int launch_rows(GroupedArgs g, hipStream_t st) {
    switch (rows_shape<T, COLS_B>(g.slots, g.groups, g.n, g.k)) {
        case 0:
            if constexpr (sizeof(T) == 4 && !COLS_B)
                if (expected_tiles(g.slots, g.groups, g.n, 32, 32) <= device_cu_count())
                    return launch_rows_shape<T, Out, COLS_B, 1, 1, 8, 1, 1, 16, false, false, true>(g, st);
            if constexpr (sizeof(T) == 2 && !COLS_B)
                if (g.x_op) return launch_rows_shape<T, Out, COLS_B, 1, 1, 8, 1, 1, 32, false, false, false, true>(g, st);
            return launch_rows_shape<T, Out, COLS_B, 1, 1, 8, 1, 1, (sizeof(T) == 4 ? 16 : 32), false, false>(g, st);
        case 1: return launch_rows_large<T, Out, COLS_B, 1, 1>(g, st);
        case 2: return launch_rows_large<T, Out, COLS_B, 2, 1>(g, st);
        default: return launch_rows_large<T, Out, COLS_B, 2, 2>(g, st);
    }
}

// Whether the weight gradient of 16-bit rows takes 256 x 256 tiles: half the reads per product, but one workgroup per CU, whose
// end nothing hides. Both ways (us, 128 / 256, joins included): 200,000 slots 2304 x 512 730 / 584, 2304 x 2304 3627 / 2327,
// 512 x 512 186 / 174, 100,000 slots 2304 x 512 361 / 311, 8,000 slots 2304 x 2304 164 / 160; 24,000 slots 2304 x 512 in 16
// groups 147 / 153, 100,000 slots 512 x 512 109 / 111, 3,000 slots 2304 x 2304 93 / 96, 24,000 slots 512 x 512 52 / 62.
static inline bool weight_large(int64_t slots, int n, int k) {
    auto up = [](int64_t v, int64_t to) { return (v + to - 1) / to * to; };
    return n >= 512 && k >= 512 && (double)slots * n * k >= 4e10 &&
           up(n, 256) * up(k, 256) * 8 <= up(n, 128) * up(k, 128) * 9;          // an eighth more area at most
}
// Shares of its slots. A workgroup takes about `slot` us a slot, and a share costs 0.08 us and the bytes of a partial result
// written and read at 4 TB/s, so that s shares take slots slot / s + s (0.08 + 2e-6 n k): the s with the least, and no more
// than fill the chip once (three workgroups per CU of 16-bit rows staged without registers, two of others, one of 256 x 256). One workgroup per
// group and tile instead, without partial results, where the largest group (taken as half the slots, or all of one) is done
// no later than the shares and the 9 us of their join, and up to 512 slots, which need no workspace then. Measured (us,
// shares of 256 slots or more that fill the chip / this rule):
//   bf16: 1,600 slots in 16 groups 512 x 512 35 / 10, 800 in one 2304 x 512 28 / 20, 8,000 in three 97 x 192 28 / 26,
//         24,000 in three 512 x 512 56 / 50, 100,000 in eight 1440 x 320 200 / 208, 97 x 96 46 / 50
//   fp32: 800 in three 2304 x 512 53 / 30, in one 192 x 97 30 / 24, 8,000 in 32 864 x 192 65 / 58, 100,000 in eight 192 x 97
//         67 / 71; the same within 1 % from 24,000 slots of 1440 x 320 on
// 16-bit rows staged through registers take 195 of them, two workgroups per CU; shares for three / for two (us, SiLU on load in
// one limb): 200,000 slots in eight 2304 x 512 1650 / 1452, 100,000 512 x 512 198 / 168, 1440 x 320 411 / 368; without SiLU
// 513 x 97 111 / 89, 321 x 1440 420 / 433.
static inline int weight_shares(int64_t slots, int groups, int n, int k, int dtype, bool large, bool direct) {
    const int tile = large ? 256 : 128;
    const double tiles = (double)((n + tile - 1) / tile) * ((k + tile - 1) / tile);
    const double fill = (large ? 1 : dtype != FACE_F32 && direct ? 3 : 2) * device_cu_count() / tiles;
    const double slot = dtype == FACE_F32 ? 0.06 : (direct ? 0.0175 : 0.035);
    const double all = (double)slots * slot, join = 0.08 + 2e-6 * n * k;
    double s = __builtin_sqrt(all / join);
    s = __builtin_floor(s < fill ? s : fill);
    return slots <= 512 || s < 2 || (groups > 1 ? all / 2 : all) <= all / s + s * join + 9 ? 1 : (int)s;
}

template <typename T, bool DIRECT, int TILE, bool SILU = false>
static int launch_weight_tile(GroupedWArgs g, hipStream_t st) {
    g.shares = weight_shares(g.slots, g.groups, g.n, g.k, sizeof(T) == 4 ? FACE_F32 : FACE_BF16, TILE == 256, DIRECT);
    g.share = (g.slots + g.shares - 1) / g.shares;
    g.row_tiles = (g.n + TILE - 1) / TILE;
    g.col_tiles = (g.k + TILE - 1) / TILE;
    const int64_t grid = (int64_t)(g.shares > 1 ? g.shares : g.groups) * g.row_tiles * g.col_tiles;
    if (grid > 0x7fffffff) return FACE_ERR_UNSUPPORTED;
    // ceil(2^(31 + s) / xdiv) with 2^s >= xdiv is exact for every numerator below 2^31
    uint32_t s = 0;
    while (((int64_t)1 << s) < g.xdiv) ++s;
    g.div_mul = (uint32_t)((((uint64_t)1 << (31 + s)) + g.xdiv - 1) / g.xdiv);
    g.div_shift = 31 + s;
    hipLaunchKernelGGL((grouped_weight_kernel<T, DIRECT, TILE, SILU>), dim3((unsigned)grid),
                       dim3(WeightKernel<T, TILE, SILU>::kThreads), 0, st, g);
    FACE_LAUNCH_CHECK();
    if (g.shares > 1) {
        const int64_t blocks = ((int64_t)g.n * g.k + 1023) / 1024;
        hipLaunchKernelGGL(grouped_join_kernel<T>, dim3((unsigned)(blocks < 4096 ? blocks : 4096), g.groups), dim3(256), 0, st,
                           g);
        FACE_LAUNCH_CHECK();
    }
    return 0;
}

template <typename T>
int launch_weight(GroupedWArgs g, hipStream_t st) {
    if constexpr (sizeof(T) < 4) {
        if (g.x_op) return launch_weight_tile<T, false, 128, true>(g, st);
        if (whole_chunks<T>(g.x, g.ld_x, g.k) && whole_chunks<T>(g.dy, g.ld_dy, g.n) &&
            g.ld_x < ((int64_t)1 << 30) && g.ld_dy < ((int64_t)1 << 30))
            return weight_large(g.slots, g.n, g.k) ? launch_weight_tile<T, true, 256>(g, st)
                                                   : launch_weight_tile<T, true, 128>(g, st);
    }
    return launch_weight_tile<T, false, 128>(g, st);
}

}  // namespace face

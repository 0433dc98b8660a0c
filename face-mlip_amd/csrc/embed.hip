// Rows of a table by index, scaled, and the table's gradient:
//
//   y[i] = scale T[idx i], 0 where idx lies outside [0, V);   dT[v] = scale sum over the i with idx i = v of dy[i]
//
// The sums go in the order of the rows, split at places that the sizes alone set and joined in a fixed order: no
// atomics, the same bits every time. Two ways:
//   * few entries, or few rows: a wave takes a chunk of rows and, entry by entry, finds the chunk's rows of it with a
//     ballot per 64 indices; partial sums per chunk and entry, joined by columns. Nothing is sorted.
//   * else the indices are sorted first (a stable radix sort of 8 bits a pass, or one workgroup up to 1024 rows); groups of
//     lanes sum equal shares of the sorted rows, entry after entry. What begins and ends within a share is done; the
//     sums that go on into the next share are joined afterwards, short runs by a few lanes, long ones by a workgroup.
// Sums in fp32. Bound by bytes, the rows of y and of dy, once each, and by the launches of the sort. A million rows x 64 fp32 of
// 14,161 entries: forward 45 us (256 MB), gradient 117: 2 x (7 + 4 + 15) for the sort, 55 for the sums (256 MB, 4.7 TB/s), 10 for
// what goes on. 100,000 x 256 bf16 of three entries: 11 us, gradient 18 + 5 (51 MB each). 21 x 96: 2.0 and 2.8 us, the launches.
#include "kept.h"

namespace face {

// Rows of y and of dy past this pass the caches by (64 MB of pairs' rows, both directions, 77 us for 81 with ordinary accesses, 256 MB
// 158 for 211).
constexpr int64_t kEmbedStream = (int64_t)48 << 20;

// R rows per group of lanes, a workgroup's groups side by side, so that the rows' indices, then their entries, are on
// their way together.
template <typename T, typename I, int R, bool NT, bool CUT>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const T* __restrict__ table, int64_t ld, const I* __restrict__ index,
                                                        int64_t N, int64_t V, int F, float factor, int lg, T* __restrict__ y,
                                                        int32_t* __restrict__ key) {
    constexpr int E = Sixteen<T>::E;
    const int groups = 256 >> lg, lane = threadIdx.x & ((1 << lg) - 1);
    const int64_t n0 = row_block() * groups * R + (threadIdx.x >> lg);
    I v[R];
    bool in[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t n = n0 + i * groups;
        v[i] = n < N ? index[n] : (I)-1;
        in[i] = v[i] >= 0 && v[i] < V;
        if (key && lane == 0 && n < N) key[n] = in[i] ? (int32_t)v[i] : -1;
    }
    for (int c = E * lane; c < F; c += E << lg) {
        Sixteen<T> r[R];
#pragma unroll
        for (int i = 0; i < R; ++i) r[i] = hold16<false, CUT>(table + (in[i] ? (int64_t)v[i] : 0) * ld, c, in[i] ? F : 0);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t n = n0 + i * groups;
            float x[E];
            values16<T>(r[i], x);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = in[i] ? x[e] * factor : 0.f;
            if (n < N) store16<NT, CUT>(y + n * F, c, F, x);
        }
    }
}

// ---------------------------------------------------------------- few entries or few rows
// A lane's sums in fp32, to columns [c, c + E) of a row of F.
template <int E>
__device__ __forceinline__ void store_sums(float* row, int c, int F, const float x[E]) {
    store16<false, true>(row, c, F, x);
    if constexpr (E == 8) store16<false, true>(row, c + 4, F, x + 4);
}

// A wave: rows [chunk R, chunk R + R), entries [block TV, block TV + TV), 64 times sixteen bytes of the columns. Partial sums
// (chunks, V, F), or with one chunk the result.
template <typename T>
__global__ __launch_bounds__(256) void embed_scan_kernel(const int32_t* __restrict__ key, const T* __restrict__ dy, int64_t ld,
                                                         int64_t N, int64_t R, int64_t chunks, int64_t V, int64_t TV,
                                                         int64_t blocks, int F, float factor, float* __restrict__ part,
                                                         T* __restrict__ out) {
    constexpr int E = Sixteen<T>::E;
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (id >= chunks * blocks) return;
    const int64_t chunk = id / blocks, b = id - chunk * blocks;
    const int64_t n0 = chunk * R, n1 = n0 + R < N ? n0 + R : N;
    const int64_t v1 = (b + 1) * TV < V ? (b + 1) * TV : V;
    const int c = E * (lane + 64 * (int)blockIdx.y), left = F - c;
    for (int64_t v = b * TV; v < v1; ++v) {
        float s[E] = {};
        for (int64_t a = n0; a < n1; a += 64) {
            uint64_t m = __ballot(a + lane < n1 && key[a + lane < n1 ? a + lane : a] == (int32_t)v);
            while (m) {
                constexpr int U = 8;
                Sixteen<T> r[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    r[u] = {};
                    if (m) {
                        const int i = __builtin_ctzll(m);
                        m &= m - 1;
                        r[u] = hold16<false, true>(dy + (a + i) * ld, c, F);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float x[E];
                    values16<T>(r[u], x);
#pragma unroll
                    for (int e = 0; e < E; ++e) s[e] += x[e];
                }
            }
        }
        if (left <= 0) continue;
        if (part) {
            store_sums<E>(part + (chunk * V + v) * F, c, F, s);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) s[e] *= factor;
            store16<false, true>(out + v * F, c, F, s);
        }
    }
}

// out[c] = factor times the sum over `rows` of part (rows, cols): 64 threads per column, each a sum of every 64th
// row, then a tree.
template <typename T>
__global__ __launch_bounds__(1024) void embed_join_kernel(const float* __restrict__ part, int64_t rows, int64_t cols, float factor,
                                                          T* __restrict__ out) {
    __shared__ float sums[64][17];
    const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4;
    const int64_t c = (int64_t)blockIdx.x * 16 + cx;
    float a = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (int64_t r = ry; r < rows; r += 64) a += part[r * cols + c];
    }
    sums[ry][cx] = a;
    __syncthreads();
    for (int o = 32; o > 0; o >>= 1) {
        if (ry < o) sums[ry][cx] += sums[ry + o][cx];
        __syncthreads();
    }
    if (ry == 0 && c < cols) out[c] = from_f<T>(factor * sums[0][cx]);
}

// ---------------------------------------------------------------- sort
// (key, row) pairs by key, stably; a key outside [0, V) counts as V. Pairs come from the indices in the first pass.
constexpr int kSortThreads = 512, kSortWaves = kSortThreads / kWave, kSortBits = 8;
constexpr int64_t kSortOne = 1024;               // one workgroup does it all up to here (24 us with the sums; 48 for 4000, in passes 26)

__device__ __forceinline__ uint32_t sort_key(const int32_t* key, int64_t a, uint32_t V) {
    const uint32_t k = (uint32_t)key[a];
    return k < V ? k : V;
}
static inline int64_t sort_segment(int64_t N) {
    const int64_t s = (N + 1023) / 1024;
    return s > 2048 ? (s + 511) / 512 * 512 : 2048;
}

__global__ __launch_bounds__(1024) void sort_one_kernel(const int32_t* __restrict__ key, int N, uint32_t V, int n2,
                                                        int32_t* __restrict__ key_out, int32_t* __restrict__ row_out) {
    __shared__ uint64_t p[kSortOne];
    for (int i = threadIdx.x; i < n2; i += 1024) p[i] = i < N ? (uint64_t)sort_key(key, i, V) << 32 | (uint32_t)i : ~0ull;
    __syncthreads();
    for (int k = 2; k <= n2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int t = threadIdx.x; t < n2 / 2; t += 1024) {
                const int i = 2 * t - (t & (j - 1)), o = i + j;
                const uint64_t a = p[i], b = p[o];
                if ((a > b) == ((i & k) == 0)) {
                    p[i] = b;
                    p[o] = a;
                }
            }
            __syncthreads();
        }
    for (int i = threadIdx.x; i < N; i += 1024) {
        key_out[i] = (int32_t)(p[i] >> 32);
        row_out[i] = (int32_t)(uint32_t)p[i];
    }
}

__device__ __forceinline__ uint64_t same_digit(uint32_t d, bool some, int bits) {
    uint64_t m = __ballot(some);
    for (int b = 0; b < bits; ++b) {
        const uint64_t v = __ballot((d >> b) & 1);
        m &= (d >> b) & 1 ? v : ~v;
    }
    return m;
}
// A segment is shared out to the waves, a wave's share taken 64 keys at a time; up to kSortHeld of these are loaded together
// (one by one, a million keys were placed in 16.6 us a pass for 15.4).
constexpr int kSortHeld = 8;
struct SortShare {
    int64_t begin, end;
};
__device__ __forceinline__ SortShare sort_share(int64_t a0, int64_t a1) {
    const int64_t per = (a1 - a0 + kSortThreads - 1) / kSortThreads * kWave;
    const int64_t b = a0 + threadIdx.x / kWave * per;
    return {b, b + per < a1 ? b + per : a1};
}
__device__ __forceinline__ void sort_hold(const int32_t* key, int64_t a, const SortShare& s, uint32_t V, uint32_t k[kSortHeld]) {
#pragma unroll
    for (int i = 0; i < kSortHeld; ++i) {
        const int64_t at = a + i * kWave + threadIdx.x % kWave;
        k[i] = at < s.end ? sort_key(key, at, V) : 0;
    }
}
// Counts of the wave's share's digits, cnt[digits] in LDS. `k`: the share's first kSortHeld loads.
__device__ __forceinline__ void sort_count(const int32_t* key, const SortShare& s, uint32_t V, int shift, int bits, int* cnt,
                                           const uint32_t k0[kSortHeld]) {
    const int lane = threadIdx.x % kWave;
    uint32_t k[kSortHeld];
#pragma unroll
    for (int i = 0; i < kSortHeld; ++i) k[i] = k0[i];
    for (int64_t a = s.begin; a < s.end; a += kSortHeld * kWave) {
        if (a != s.begin) sort_hold(key, a, s, V, k);
#pragma unroll
        for (int i = 0; i < kSortHeld; ++i) {
            if (a + i * kWave >= s.end) break;
            const bool some = a + i * kWave + lane < s.end;
            const uint32_t d = some ? (k[i] >> shift) & ((1u << bits) - 1) : 0;
            const uint64_t m = same_digit(d, some, bits);
            if (some && (m & ((1ull << lane) - 1)) == 0) cnt[d] += __popcll(m);
            __builtin_amdgcn_wave_barrier();
        }
    }
}
// Workgroups behind the segments' clear the table's gradient: entries without a row.
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const int32_t* __restrict__ key, int64_t N, int64_t seg, int segs,
                                                                  uint32_t V, int shift, int bits, int32_t* __restrict__ count,
                                                                  char* __restrict__ out, int64_t out_bytes) {
    __shared__ int cnt[kSortWaves << kSortBits];
    if ((int)blockIdx.x >= segs) {
        const int64_t begin = ((int64_t)(blockIdx.x - segs) * kSortThreads + threadIdx.x) * 16;
        for (int64_t at = begin; at < out_bytes; at += (int64_t)(gridDim.x - segs) * kSortThreads * 16) {
            if (at + 16 <= out_bytes)
                st16(out + at, (v4u){0, 0, 0, 0});
            else
                for (int64_t i = at; i < out_bytes; i += 2) *(uint16_t*)(out + i) = 0;
        }
        return;
    }
    const int D = 1 << bits;
    const int64_t a0 = blockIdx.x * seg, a1 = a0 + seg < N ? a0 + seg : N;
    const SortShare s = sort_share(a0, a1);
    uint32_t k[kSortHeld];
    sort_hold(key, s.begin, s, V, k);
    for (int i = threadIdx.x; i < kSortWaves * D; i += kSortThreads) cnt[i] = 0;
    __syncthreads();
    sort_count(key, s, V, shift, bits, cnt + threadIdx.x / kWave * D, k);
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kSortThreads) {
        int c = 0;
        for (int w = 0; w < kSortWaves; ++w) c += cnt[w * D + d];
        count[(int64_t)d * segs + blockIdx.x] = c;
    }
}
// Exclusive sums of a value per thread over a workgroup of 256, and the total. `part`: LDS, 4.
__device__ __forceinline__ int sums_before(int c, int* part, int& total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    int s = c;
    for (int o = 1; o < kWave; o <<= 1) {
        const int t = __shfl_up(s, o, kWave);
        if (lane >= o) s += t;
    }
    __syncthreads();
    if (lane == kWave - 1) part[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < 4; ++w) {
        before += w < wave ? part[w] : 0;
        total += part[w];
    }
    return before + s - c;
}
// count (D, segs): every digit's row becomes its exclusive sums, tot its total. A workgroup per digit, four segments a
// thread at a time.
__global__ __launch_bounds__(256) void sort_rows_kernel(int32_t* __restrict__ count, int segs, int32_t* __restrict__ tot) {
    __shared__ int part[4];
    int32_t* row = count + (int64_t)blockIdx.x * segs;
    int run = 0;
    for (int b0 = 0; b0 < segs; b0 += 1024) {
        const int b = b0 + 4 * threadIdx.x;
        int c[4], sum = 0, total;
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = b + i < segs ? row[b + i] : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += c[i];
        int at = run + sums_before(sum, part, total);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (b + i < segs) row[b + i] = at;
            at += c[i];
        }
        run += total;
    }
    if (threadIdx.x == 0) tot[blockIdx.x] = run;
}
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(const int32_t* __restrict__ key, const int32_t* __restrict__ row,
                                                                  int64_t N, int64_t seg, uint32_t V, int shift, int bits,
                                                                  const int32_t* __restrict__ count,
                                                                  const int32_t* __restrict__ tot, int32_t* __restrict__ key_out,
                                                                  int32_t* __restrict__ row_out) {
    __shared__ int cnt[kSortWaves << kSortBits], begin[1 << kSortBits];
    const int D = 1 << bits, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int64_t a0 = blockIdx.x * seg, a1 = a0 + seg < N ? a0 + seg : N;
    const SortShare s = sort_share(a0, a1);
    uint32_t k[kSortHeld];
    int32_t r[kSortHeld];
    auto hold_rows = [&](int64_t a) {
#pragma unroll
        for (int i = 0; i < kSortHeld; ++i) {
            const int64_t at = a + i * kWave + lane;
            r[i] = row && at < s.end ? row[at] : (int32_t)at;
        }
    };
    sort_hold(key, s.begin, s, V, k);
    hold_rows(s.begin);
    const int mine_tot = (int)threadIdx.x < D ? tot[threadIdx.x] : 0;
    const int mine_count = (int)threadIdx.x < D ? count[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] : 0;
    for (int i = threadIdx.x; i < kSortWaves * D; i += kSortThreads) cnt[i] = 0;
    __syncthreads();
    sort_count(key, s, V, shift, bits, cnt + wave * D, k);
    if ((int)threadIdx.x < D) begin[threadIdx.x] = mine_tot;
    __syncthreads();
    if (wave == 0) {                             // exclusive sums of the digits' totals
        int run = 0;
        for (int d0 = 0; d0 < D; d0 += kWave) {
            const int d = d0 + lane, c = d < D ? begin[d] : 0;
            int t = c;
            for (int o = 1; o < kWave; o <<= 1) {
                const int w = __shfl_up(t, o, kWave);
                if (lane >= o) t += w;
            }
            if (d < D) begin[d] = run + t - c;
            run += __shfl(t, kWave - 1, kWave);
        }
    }
    __syncthreads();
    if ((int)threadIdx.x < D) {
        int at = begin[threadIdx.x] + mine_count;
        for (int w = 0; w < kSortWaves; ++w) {
            const int c = cnt[w * D + threadIdx.x];
            cnt[w * D + threadIdx.x] = at;
            at += c;
        }
    }
    __syncthreads();
    volatile int* mine = cnt + wave * D;
    for (int64_t a = s.begin; a < s.end; a += kSortHeld * kWave) {
        if (s.end - s.begin > kSortHeld * kWave) {
            sort_hold(key, a, s, V, k);
            hold_rows(a);
        }
#pragma unroll
        for (int i = 0; i < kSortHeld; ++i) {
            if (a + i * kWave >= s.end) break;
            const bool some = a + i * kWave + lane < s.end;
            const uint32_t d = some ? (k[i] >> shift) & (D - 1) : 0;
            const uint64_t m = same_digit(d, some, bits);
            const int rank = __popcll(m & ((1ull << lane) - 1));
            if (some) {
                const int at = mine[d];
                key_out[at + rank] = (int32_t)k[i];
                row_out[at + rank] = r[i];
                __builtin_amdgcn_wave_barrier(); // every lane has read the place before the first one moves it on
                if (rank == 0) mine[d] = at + __popcll(m);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// ---------------------------------------------------------------- sums of sorted rows
template <typename T>
__global__ __launch_bounds__(256) void embed_zero_kernel(T* __restrict__ out, int64_t n) {
    const int64_t i = kPiece * (row_block() * 256 + threadIdx.x);
    if (i >= n) return;
    const float none[kPiece] = {};
    store_piece(out + i, n - i < kPiece ? (int)(n - i) : kPiece, none);
}

// Groups of LC lanes, C sorted rows each. part (shares, 2, F): a run that comes from the share before (0), one that begins
// here and goes on (1). The next rows' numbers are on their way while the present ones are added.
template <typename T, int LC, bool NT, bool CUT>
__global__ __launch_bounds__(256) void embed_runs_kernel(const int32_t* __restrict__ key, const int32_t* __restrict__ row,
                                                         const T* __restrict__ dy, int64_t ld, int64_t N, int64_t C, int V, int F,
                                                         float factor, float* __restrict__ part, T* __restrict__ out) {
    constexpr int E = Sixteen<T>::E, U = 8;
    const int64_t s = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LC;
    const int64_t begin = s * C, end = begin + C < N ? begin + C : N;
    const int c = E * ((int)(threadIdx.x % LC) + LC * (int)blockIdx.y), left = F - c;
    if (begin >= N || left <= 0) return;
    int cur = key[begin];
    if (cur >= V) return;
    bool from_before = begin > 0 && key[begin - 1] == cur;
    float acc[E] = {};
    auto flush = [&](bool goes_on) {
        if (from_before || goes_on) {
            store_sums<E>(part + (2 * s + (from_before ? 0 : 1)) * F, c, F, acc);
        } else {
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = factor * acc[e];
            store16<false, true>(out + (int64_t)cur * F, c, F, o);
        }
    };
    int k[U], next_k[U];
    int32_t at[U], next_at[U];
    auto numbers = [&](int64_t p, int kk[U], int32_t rr[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t q = p + u < end ? p + u : end - 1;
            kk[u] = key[q];
            rr[u] = row[q];
        }
    };
    numbers(begin, k, at);
    for (int64_t p = begin; p < end; p += U) {
        Sixteen<T> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) r[u] = hold16<NT, CUT>(dy + (int64_t)at[u] * ld, c, F);
        if (p + U < end) numbers(p + U, next_k, next_at);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p + u >= end) break;
            if (k[u] != cur) {
                flush(false);
                cur = k[u];
                from_before = false;
                if (cur >= V) return;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = 0.f;
            }
            float x[E];
            values16<T>(r[u], x);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += x[e];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k[u] = next_k[u];
            at[u] = next_at[u];
        }
    }
    flush(end < N && key[end] == cur);
}

// A workgroup: 64 shares, 16 pieces of the columns. 16 lanes look at a share; one whose last run begins there and goes on
// has that run's sum joined from the following shares': in order by its lanes where there are few, else by the
// whole workgroup, every 64th by the same lanes, then a tree.
constexpr int kJoinShort = 8;
template <typename T>
__global__ __launch_bounds__(1024) void embed_runs_join_kernel(const int32_t* __restrict__ key, int64_t N, int64_t C, int64_t shares,
                                                               int V, int F, float factor, const float* __restrict__ part,
                                                               T* __restrict__ out) {
    __shared__ int64_t long_first[64], long_last[64];
    __shared__ int longs;
    __shared__ float tree[64][16 * kPiece + 1];
    const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int64_t s = (int64_t)blockIdx.x * 64 + group;
    const int c = kPiece * (lane + 16 * (int)blockIdx.y), left = F - c;
    if (threadIdx.x == 0) longs = 0;
    __syncthreads();
    if (s + 1 < shares) {
        const int64_t begin = s * C, end = begin + C;                    // not the last share: a whole one
        const int k = key[end - 1];
        // how many of the next shares begin with k: their first keys together, then by halves
        const int64_t probe = s + 1 + lane < shares ? s + 1 + lane : shares - 1;
        const int first = key[probe * C], at_begin = key[begin], before = begin > 0 ? key[begin - 1] : -1;
        const uint32_t same = (uint32_t)(__ballot(first == k && s + 1 + lane < shares) >> (threadIdx.x & 48)) & 0xffffu;
        if (k < V && (same & 1) && (at_begin != k || before != k)) {
            int64_t lo = s + __builtin_ctz(~same);                       // the last of the next sixteen
            if (same == 0xffffu) {
                int64_t hi = shares - 1;
                while (lo < hi) {
                    const int64_t mid = (lo + hi + 1) >> 1;
                    if (key[mid * C] == k) lo = mid;
                    else hi = mid - 1;
                }
            }
            if (lo - s > kJoinShort) {
                if (lane == 0) {
                    const int i = atomicAdd(&longs, 1);
                    long_first[i] = s;
                    long_last[i] = lo;
                }
            } else if (left > 0) {
                float a[kPiece];
                load_piece(part + (2 * s + 1) * F + c, left, a);
                for (int64_t j = s + 1; j <= lo; ++j) {
                    float x[kPiece];
                    load_piece(part + 2 * j * F + c, left, x);
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) a[e] += x[e];
                }
#pragma unroll
                for (int e = 0; e < kPiece; ++e) a[e] *= factor;
                store_piece(out + (int64_t)k * F + c, left, a);
            }
        }
    }
    __syncthreads();
    for (int i = 0; i < longs; ++i) {            // each its own rows of out: their order does not matter
        const int64_t first = long_first[i], last = long_last[i];
        float a[kPiece] = {};
        if (left > 0) {
            if (group == 0) load_piece(part + (2 * first + 1) * F + c, left, a);
#pragma unroll 4
            for (int64_t j = first + 1 + group; j <= last; j += 64) {
                float x[kPiece];
                load_piece(part + 2 * j * F + c, left, x);
#pragma unroll
                for (int e = 0; e < kPiece; ++e) a[e] += x[e];
            }
        }
#pragma unroll
        for (int e = 0; e < kPiece; ++e) tree[group][lane + 16 * e] = a[e];
        __syncthreads();
        for (int o = 32; o > 0; o >>= 1) {
            if (group < o)
#pragma unroll
                for (int e = 0; e < kPiece; ++e) tree[group][lane + 16 * e] += tree[group + o][lane + 16 * e];
            __syncthreads();
        }
        if (group == 0 && left > 0) {
#pragma unroll
            for (int e = 0; e < kPiece; ++e) a[e] = factor * tree[0][lane + 16 * e];
            store_piece(out + (int64_t)key[first * C + C - 1] * F + c, left, a);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- plans
struct EmbedPlan {
    bool scan;
    int64_t R, chunks, TV, blocks;               // scan
    int lanes, tiles;                            // sorted: lanes of a group, tiles of the columns
    int64_t C, shares;
    int64_t sort_bytes, bytes;                   // workspace
};
static inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

static EmbedPlan embed_plan(int64_t N, int64_t V, int F, int size) {
    EmbedPlan p = {};
    const int64_t sixteens = ((int64_t)F * size + 15) / 16;
    // Few rows: a wave per entry looks through all of them. Few entries: a wave per chunk looks for all of them. Else sorted.
    // us, this way / sorted: 1024 rows x 96 fp32 of 200 entries 7 / 24, 2048 of 14,161 16 / 32, but x 2304 bf16 76 / 42; 100,000
    // rows x 96 fp32 of 8 entries 22 / 33, of 16 28 / 33, of 64 65 / 34, x 1440 118 / 119, 157 / 127, 325 / 121.
    const int64_t tiles = (sixteens + 63) / 64;
    const bool few_rows = N <= 512 || (V > 8 && N <= 2048 && V * tiles * N <= (int64_t)36 << 20);
    if (V <= 8 || few_rows) {
        p.scan = true;
        if (few_rows) {
            p.R = N < 1 ? 1 : N;
            p.chunks = 1;
            p.TV = (V + (1 << 22) - 1) >> 22;        // one, but for millions of entries: a grid's dimension ends at 2^32 threads
        } else {
            const int64_t r = N * tiles / 2048 / 64 * 64;
            p.R = r < 64 ? 64 : (r > 1024 ? 1024 : r);
            p.chunks = (N + p.R - 1) / p.R;
            p.TV = V;
        }
        p.blocks = (V + p.TV - 1) / p.TV;
        p.bytes = p.chunks > 1 ? 4 * p.chunks * V * F : 0;
        return p;
    }
    p.lanes = 8;
    while (p.lanes < 64 && p.lanes < sixteens) p.lanes *= 2;
    p.tiles = (int)((sixteens + p.lanes - 1) / p.lanes);
    const int64_t c = N * p.tiles * p.lanes / 64 / 2048;
    p.C = c < 16 ? 16 : (c > 512 ? 512 : (c + 7) / 8 * 8);
    p.shares = (N + p.C - 1) / p.C;
    const int64_t seg = sort_segment(N), segs = (N + seg - 1) / seg;
    p.sort_bytes = 4 * up256(4 * N) + (N > kSortOne ? up256(4 * (segs + 1) << kSortBits) : 0);
    p.bytes = p.sort_bytes + up256(8 * p.shares * F);
    return p;
}

// Sorted pairs of `key` in work, where key_out and row_out point then; out (V, F) is cleared on the way.
template <typename T>
static void embed_sort(const int32_t* key, int64_t N, int64_t V, int F, T* out, char* work, const int32_t*& key_out,
                       const int32_t*& row_out, hipStream_t st) {
    constexpr int size = (int)sizeof(T);
    const int64_t n = up256(4 * N);
    int32_t* k[2] = {(int32_t*)work, (int32_t*)(work + n)};
    int32_t* r[2] = {(int32_t*)(work + 2 * n), (int32_t*)(work + 3 * n)};
    if (N <= kSortOne) {
        int n2 = 2;
        while (n2 < N) n2 *= 2;
        hipLaunchKernelGGL(sort_one_kernel, dim3(1), dim3(1024), 0, st, key, (int)N, (uint32_t)V, n2, k[0], r[0]);
        hipLaunchKernelGGL(embed_zero_kernel<T>, row_grid((V * F + 256 * kPiece - 1) / (256 * kPiece)), dim3(256), 0, st, out,
                           V * F);
        key_out = k[0];
        row_out = r[0];
        return;
    }
    int bits = 1;
    while (V >> bits) ++bits;                    // keys up to V
    const int passes = (bits + kSortBits - 1) / kSortBits, per = (bits + passes - 1) / passes;
    const int64_t seg = sort_segment(N), bytes = V * F * size, zeros = (bytes + 16 * kSortThreads - 1) / (16 * kSortThreads);
    const int segs = (int)((N + seg - 1) / seg);
    int32_t *tot = (int32_t*)(work + 4 * n), *count = tot + (1 << kSortBits);
    const int32_t *from = key, *rows = nullptr;
    for (int i = 0; i < passes; ++i) {
        const int D = 1 << per;
        hipLaunchKernelGGL(sort_count_kernel, dim3(segs + (i ? 0 : (unsigned)(zeros < 2048 ? zeros : 2048))), dim3(kSortThreads), 0, st,
                           from, N, seg, segs, (uint32_t)V, i * per, per, count, (char*)out, bytes);
        hipLaunchKernelGGL(sort_rows_kernel, dim3(D), dim3(256), 0, st, count, segs, tot);
        hipLaunchKernelGGL(sort_place_kernel, dim3(segs), dim3(kSortThreads), 0, st, from, rows, N, seg, (uint32_t)V, i * per, per,
                           count, tot, k[i & 1], r[i & 1]);
        from = k[i & 1];
        rows = r[i & 1];
    }
    key_out = from;
    row_out = rows;
}

template <typename T>
static int launch_embed_bwd(const int32_t* key, const T* dy, int64_t ld, int64_t N, int64_t V, int F, float factor, T* out,
                            char* work, hipStream_t st) {
    const EmbedPlan p = embed_plan(N, V, F, (int)sizeof(T));
    if (p.scan) {
        float* part = p.chunks > 1 ? (float*)work : nullptr;
        const dim3 grid((unsigned)((p.chunks * p.blocks + 3) / 4), (unsigned)((F + 64 * Sixteen<T>::E - 1) / (64 * Sixteen<T>::E)));
        hipLaunchKernelGGL(embed_scan_kernel<T>, grid, dim3(256), 0, st, key, dy, ld, N, p.R, p.chunks, V, p.TV, p.blocks, F, factor,
                           part, out);
        if (part)
            hipLaunchKernelGGL(embed_join_kernel<T>, dim3((unsigned)((V * F + 15) / 16)), dim3(1024), 0, st, part, p.chunks, V * F,
                               factor, out);
        FACE_LAUNCH_CHECK();
        return 0;
    }
    const int32_t *keys, *rows;
    embed_sort<T>(key, N, V, F, out, work, keys, rows, st);
    float* part = (float*)(work + p.sort_bytes);
    const dim3 grid((unsigned)((p.shares * p.lanes + 255) / 256), (unsigned)p.tiles);
    const bool nt = N * F * (int64_t)sizeof(T) > kEmbedStream;
#define FACE_RUNS(L_)                                                                                                     \
    if (p.lanes == L_)                                                                                                    \
        with_forms(nt, F % Sixteen<T>::E, [&](auto nt_, auto cut_) {                                                      \
            hipLaunchKernelGGL((embed_runs_kernel<T, L_, nt_.value, cut_.value>), grid, dim3(256), 0, st, keys, rows, dy, ld, N, p.C, \
                               (int)V, F, factor, part, out);                                                             \
        });
    FACE_RUNS(8) FACE_RUNS(16) FACE_RUNS(32) FACE_RUNS(64)
#undef FACE_RUNS
    if (p.shares > 1)
        hipLaunchKernelGGL(embed_runs_join_kernel<T>, dim3((unsigned)((p.shares + 63) / 64), (unsigned)((F + 127) / 128)), dim3(1024),
                           0, st, keys, N, p.C, p.shares, (int)V, F, factor, part, out);
    FACE_LAUNCH_CHECK();
    return 0;
}

static int embed_args(int64_t N, int64_t V, int32_t F, int32_t dtype) {
    if (N < 0 || V <= 0 || F <= 0) return FACE_ERR_ARG;
    if (dtype != FACE_F32 && dtype != FACE_BF16 && dtype != FACE_F16) return FACE_ERR_ARG;
    if (N > (int64_t)0x7fffffff || V > (int64_t)0x7ffffffe || F > (1 << 20)) return FACE_ERR_UNSUPPORTED;
    return 0;
}

}  // namespace face

using namespace face;

extern "C" int face_embed_fwd(const void* table, int64_t ld_t, const void* index, int32_t wide, int64_t N, int64_t V, int32_t F,
                              int32_t dtype, float factor, void* y, int32_t* key, void* stream) {
    if (int rc = embed_args(N, V, F, dtype)) return rc;
    if (ld_t < F || (wide != 0 && wide != 1)) return FACE_ERR_ARG;
    if (N == 0) return 0;
    if (!table || !index || !y) return FACE_ERR_ARG;
    const hipStream_t st = (hipStream_t)stream;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t sixteens = ((int64_t)F * sizeof(T) + 15) / 16;
        int lg = 0;
        while (lg < 8 && (1 << lg) < sixteens) ++lg;
        const bool nt = N * F * (int64_t)sizeof(T) > kEmbedStream, cut = F % Sixteen<T>::E;
        const int64_t groups = 256 >> lg, many = nt || N >= groups * 4096 ? 4 : 1;   // four rows a group once that fills the card
        const dim3 grid = row_grid((N + groups * many - 1) / (groups * many));
        auto launch = [&](auto* i) {
            using I = std::remove_cv_t<std::remove_pointer_t<decltype(i)>>;
            with_forms(nt, cut, [&](auto nt_, auto cut_) {
                auto* kern = many > 1 ? embed_fwd_kernel<T, I, 4, nt_.value, cut_.value> : embed_fwd_kernel<T, I, 1, false, cut_.value>;
                hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, (const T*)table, ld_t, i, N, V, F, factor, lg, (T*)y, key);
            });
        };
        if (wide)
            launch((const int64_t*)index);
        else
            launch((const int32_t*)index);
        FACE_LAUNCH_CHECK();
        return 0;
    });
}

extern "C" int64_t face_embed_bwd_work(int64_t N, int64_t V, int32_t F) {
    if (N <= 0 || V <= 0 || F <= 0 || embed_args(N, V, F, FACE_F32)) return 0;
    const int64_t a = embed_plan(N, V, F, 2).bytes, b = embed_plan(N, V, F, 4).bytes;
    return a > b ? a : b;
}

extern "C" int face_embed_bwd(const int32_t* key, const void* dy, int64_t ld_dy, int64_t N, int64_t V, int32_t F, int32_t dtype,
                              float factor, void* dtable, void* work, int64_t work_bytes, void* stream) {
    if (int rc = embed_args(N, V, F, dtype)) return rc;
    if (ld_dy < F || !dtable || (N && (!key || !dy))) return FACE_ERR_ARG;
    const int64_t need = face_embed_bwd_work(N, V, F);
    if (work_bytes < need || (need && !work)) return FACE_ERR_ARG;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return launch_embed_bwd<T>(key, (const T*)dy, ld_dy, N, V, F, factor, (T*)dtable, (char*)work, (hipStream_t)stream);
    });
}

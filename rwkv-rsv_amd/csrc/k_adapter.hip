// Low-rank adapters of many requests beside a shared projection
// (rsv_adapter_multi): for every row t of a packed batch, with a =
// row_adapter[t],
//   h[t, r] = sum_k x[t, k] A[a, r, k]                       (r < R_a)
//   out[t, n] = epi(y[t, n] + scale[a] * sum_r h[t, r] B[a, n, r]).
//
// Which rows share an adapter is only known on the device.  Rows are taken in
// windows of 64, one lane each: a wave finds the window's distinct adapters
// and their rows from the ids' bits with ballots (ad_window), so there is no
// sorting pass and a captured call follows the ids of its replay.  A window
// with D adapters has its blocks dealt out among the D, so one adapter of 64
// rows and 64 adapters of one row both fill the chip.
#include <algorithm>

#include "rsv_common.h"

namespace rsv {

typedef _Float16 ad_h8 __attribute__((ext_vector_type(8)));
typedef float ad_f4 __attribute__((ext_vector_type(4)));

constexpr int kWin = 64;
constexpr int kBare = -1;  // the group of a window's rows without an adapter

// The groups of a window: one per distinct adapter, in the order of their
// first rows, then (with `bare`) one of the rows that have none.
struct AdWindow {
    uint32_t id;        // the lane's adapter,
    int rank;           // its own rank
    float scale;        // and its scale
    uint64_t same;      // lanes with this lane's adapter
    uint64_t leaders;   // the first lane of each adapter
    uint64_t none;      // lanes of rows without an adapter
    int groups;
};
struct AdGroup {
    int a;          // adapter, or kBare
    int R;          // its rank; 0: rows that y passes through
    float scale;
    int cnt;        // its rows
    int row;        // lane p < cnt: the window row of the group's p-th row
};

__device__ __forceinline__ uint64_t ad_lane64(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

__device__ __forceinline__ AdWindow ad_window(const AdapterJobs &J, int win, bool bare) {
    const int lane = threadIdx.x & 63, t = win * kWin + lane;
    AdWindow w;
    w.id = t < J.rows ? J.row_adapter[t] : 0xFFFFFFFFu;
    const bool has = w.id < (uint32_t)J.n_adapter;
    // one load behind the id's, together with each other
    w.rank = has ? J.ranks ? (int)min(J.ranks[w.id], (uint32_t)J.rank) : J.rank : 0;
    w.scale = has ? J.scale[w.id] : 0.0f;
    w.same = __ballot(has);
    w.none = __ballot(t < J.rows && !has);
    for (int b = 0; (J.n_adapter - 1) >> b; b++) {
        const uint64_t ones = __ballot(w.id >> b & 1);
        w.same &= w.id >> b & 1 ? ones : ~ones;
    }
    w.leaders = __ballot(has && (w.same & ((1ull << lane) - 1)) == 0);
    w.groups = __popcll(w.leaders) + (bare && w.none ? 1 : 0);
    return w;
}

__device__ __forceinline__ AdGroup ad_group(const AdWindow &w, int g) {
    const int lane = threadIdx.x & 63;
    const uint64_t below = (1ull << lane) - 1;
    AdGroup r;
    uint64_t mask = w.none;
    r.a = kBare;
    r.R = 0;
    r.scale = 0.0f;
    if (g < __popcll(w.leaders)) {
        const uint64_t me = __ballot((w.leaders >> lane & 1) && __popcll(w.leaders & below) == g);
        const int l = __ffsll((long long)me) - 1;
        r.a = __builtin_amdgcn_readlane((int)w.id, l);
        r.R = __builtin_amdgcn_readlane(w.rank, l);
        r.scale = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w.scale), l));
        mask = ad_lane64(w.same, l);
    }
    r.cnt = __popcll(mask);
    // lane p receives the p-th row: a permutation of the lanes, the group's rows first
    const int to = mask >> lane & 1 ? __popcll(mask & below) : r.cnt + __popcll(~mask & below);
    r.row = __builtin_amdgcn_ds_permute(to * 4, lane);
    return r;
}

__device__ __forceinline__ float ad_load(const void *p, int f16, size_t i) {
    return f16 ? (float)((const _Float16 *)p)[i] : ((const float *)p)[i];
}

__device__ __forceinline__ float ad_epi(float z, int epi) {
    return epi == GE_RELU2 ? (z > 0.0f ? z * z : z == z ? 0.0f : z) : z;
}

// Products of a 16-rank tile with MT 16-row tiles over k in [k0, k1), one
// wave: acc[m][j][e] += x[row l%16 of tile m] . A[rank 16 j + 4 (l/16) + e].
// Lane (i = l%16, g = l/16) supplies k 8g..8g+7 of each 32: the rank rows as
// the left operand, the batch rows as the right one.  fp16 x goes through
// v_mfma_f32_16x16x32_f16 (products of fp16 are exact in fp32), fp32 x through
// eight v_mfma_f32_16x16x4_f32 with A widened, so both sum in fp32.
template <int RT, int MT, bool X16, int DEP>
__device__ __forceinline__ void ad_dots(const _Float16 *__restrict__ A, const void *__restrict__ x, const size_t (&xrow)[MT],
                                        const bool (&live)[MT], int R, int K, int k0, int k1, ad_f4 (&acc)[MT][RT]) {
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    constexpr ad_h8 zero = {};
    for (int kb = k0; kb < k1; kb += 32 * DEP) {
        ad_h8 a[DEP][RT];
        ad_h8 xh[DEP][MT];
        ad_f4 xf[DEP][MT][2];
#pragma unroll
        for (int s = 0; s < DEP; s++) {
            const int k = kb + 32 * s + 8 * g;
            const bool in = k < k1;
#pragma unroll
            for (int j = 0; j < RT; j++)
                a[s][j] = in && 16 * j + i < R ? *(const ad_h8 *)(A + (size_t)(16 * j + i) * K + k) : zero;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const bool on = in && live[m];
                if constexpr (X16) {
                    xh[s][m] = on ? *(const ad_h8 *)((const _Float16 *)x + xrow[m] + k) : zero;
                } else {
                    const ad_f4 *p = (const ad_f4 *)((const float *)x + xrow[m] + k);
                    xf[s][m][0] = on ? p[0] : (ad_f4){0, 0, 0, 0};
                    xf[s][m][1] = on ? p[1] : (ad_f4){0, 0, 0, 0};
                }
            }
        }
#pragma unroll
        for (int s = 0; s < DEP; s++) {
#pragma unroll
            for (int j = 0; j < RT; j++) {
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    if constexpr (X16) {
                        acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[s][j], xh[s][m], acc[m][j], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)a[s][j][e], xf[s][m][e >> 2][e & 3], acc[m][j], 0, 0, 0);
                    }
                }
            }
        }
    }
}

// ------------------------------------------------ few rows: one launch
// A decode step (at most 64 rows): one block takes one adapter's rows and a
// piece of n, forms the whole h itself (8 waves over k, their sums added in
// wave order) and goes on to its outputs.  Splitting A over blocks instead
// takes a second launch; reading it again from L2 per piece of n costs less.
constexpr int kRowsThreads = 512;

template <int RC>
__device__ __forceinline__ void ad_up_rows(const AdapterJob &j, const float *h, int hs, int R, int rank, const _Float16 *B,
                                           float scale, const size_t *yrow, int rows, int n0, int n1) {
    for (int n = n0 + (int)threadIdx.x; n < n1; n += kRowsThreads) {
        float s[RC] = {};
        for (int r = 0; r < R; r += 8) {
            const ad_h8 b = *(const ad_h8 *)(B + (size_t)n * rank + r);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = r + e < R ? (float)b[e] : 0.0f;
#pragma unroll
                for (int c = 0; c < RC; c++) s[c] += h[c * hs + r + e] * v;
            }
        }
#pragma unroll
        for (int c = 0; c < RC; c++) {
            if (c >= rows) break;
            const size_t at = yrow[c] + n;
            float z = ad_load(j.y, j.y16, at);
            if (R) z += scale * s[c];
            z = ad_epi(z, j.epi);
            if (j.o16)
                ((_Float16 *)j.out)[at] = (_Float16)z;
            else
                ((float *)j.out)[at] = z;
        }
    }
}

template <int RT, bool X16>
__global__ __launch_bounds__(kRowsThreads) void k_adapter_rows(AdapterJobs J) {
    constexpr int HS = 16 * RT + 4, RG = RT < 4 ? RT : 4;
    __shared__ float red[8][16][16 * RG + 4];
    __shared__ __align__(16) float h[16 * HS];
    __shared__ size_t yrow[16];
    const AdapterJob &j = J.j[blockIdx.z];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int win = blockIdx.y, G = gridDim.x;
    const AdWindow w = ad_window(J, win, j.out != j.y || j.epi != GE_STORE);
    if (w.groups == 0) return;
    const int C = max(1, min(G / w.groups, (j.n + 255) / 256));
    if (blockIdx.x >= (unsigned)(w.groups * C)) return;
    const int piece = ((j.n + C - 1) / C + 63) / 64 * 64;
    const int n0 = (int)(blockIdx.x / w.groups) * piece, n1 = min(j.n, n0 + piece);
    const int ks = ((j.k + 7) / 8 + 31) / 32 * 32;  // k of a wave
    for (int gi = blockIdx.x % w.groups; gi < w.groups; gi += G) {
        const AdGroup grp = ad_group(w, gi);
        const int R = grp.R;
        const float scale = grp.scale;
        const _Float16 *A = j.a + (size_t)max(grp.a, 0) * J.rank * j.k, *B = j.b + (size_t)max(grp.a, 0) * j.n * J.rank;
        for (int p0 = 0; p0 < grp.cnt; p0 += 16) {
            const int rows = min(16, grp.cnt - p0);
            const size_t row = (size_t)win * kWin + __shfl(grp.row, p0 + i);
            const size_t xrow[1] = {row * j.k};
            const bool live[1] = {i < rows};
            __syncthreads();  // the tile before is done with h and yrow
            if (wave == 0 && g == 0) yrow[i] = row * j.n;
            if (R) {
                ad_f4 acc[1][RT] = {};
                ad_dots<RT, 1, X16, (RT <= 2 ? 5 : RT <= 4 ? 2 : 1)>(A, j.x, xrow, live, R, j.k, wave * ks, min(j.k, (wave + 1) * ks), acc);
#pragma unroll
                for (int q = 0; q < RT; q += RG) {
#pragma unroll
                    for (int t = 0; t < RG; t++) *(ad_f4 *)&red[wave][i][16 * t + 4 * g] = acc[0][q + t];
                    __syncthreads();
                    for (int v = threadIdx.x; v < 16 * 16 * RG; v += kRowsThreads) {
                        const int hr = v / (16 * RG), hc = v % (16 * RG);
                        float s = 0.0f;
#pragma unroll
                        for (int u = 0; u < 8; u++) s += red[u][hr][hc];
                        h[hr * HS + 16 * q + hc] = s;
                    }
                    __syncthreads();
                }
            } else {
                __syncthreads();
            }
            if (rows == 1)
                ad_up_rows<1>(j, h, HS, R, J.rank, B, scale, yrow, rows, n0, n1);
            else if (rows <= 4)
                ad_up_rows<4>(j, h, HS, R, J.rank, B, scale, yrow, rows, n0, n1);
            else
                ad_up_rows<16>(j, h, HS, R, J.rank, B, scale, yrow, rows, n0, n1);
        }
    }
}

// ------------------------------------------------ many rows: two launches
// h of a window's rows: 4 waves over a slice of k, their sums added in wave
// order into slice q of the work area, h[q][t][r].  The slice count of a group
// follows from the window's groups (ad_slices), so the second launch knows it.
constexpr int kDownThreads = 256;

__device__ __forceinline__ int ad_slices(int G, int groups, int k) { return max(1, min(G / max(groups, 1), (k + 511) / 512)); }

template <int RT, int MT, bool X16>
__device__ __forceinline__ void ad_down_tiles(const AdapterJobs &J, const AdapterJob &j, const AdGroup &grp, int win, int p0, int R,
                                              const _Float16 *A, int k0, int k1, float *hq, float (*red)[16][16 * (RT < 4 ? RT : 4) + 4]) {
    constexpr int RG = RT < 4 ? RT : 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    size_t xrow[MT];
    bool live[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        xrow[m] = ((size_t)win * kWin + __shfl(grp.row, p0 + 16 * m + i)) * j.k;
        live[m] = p0 + 16 * m + i < grp.cnt;
    }
    const int ks = ((k1 - k0 + 3) / 4 + 31) / 32 * 32;
    ad_f4 acc[MT][RT] = {};
    ad_dots<RT, MT, X16, (RT * MT <= 4 ? 4 : RT * MT <= 8 ? 2 : 1)>(A, j.x, xrow, live, R, j.k, min(k1, k0 + wave * ks), min(k1, k0 + (wave + 1) * ks), acc);
#pragma unroll
    for (int m = 0; m < MT; m++) {
#pragma unroll
        for (int q = 0; q < RT; q += RG) {
            __syncthreads();
#pragma unroll
            for (int t = 0; t < RG; t++) *(ad_f4 *)&red[wave][i][16 * t + 4 * g] = acc[m][q + t];
            __syncthreads();
            for (int v = threadIdx.x; v < 16 * 16 * RG; v += kDownThreads) {
                const int hr = v / (16 * RG), hc = v % (16 * RG), p = p0 + 16 * m + hr, r = 16 * q + hc;
                const int row = __shfl(grp.row, p & 63);  // every lane of the wave gets here: 256 divides 256 RG
                if (p < grp.cnt && r < R) hq[((size_t)win * kWin + row) * J.rank + r] = (red[0][hr][hc] + red[1][hr][hc]) + (red[2][hr][hc] + red[3][hr][hc]);
            }
        }
    }
}

template <int RT, bool X16>
__global__ __launch_bounds__(kDownThreads) void k_adapter_down(AdapterJobs J) {
    constexpr int RG = RT < 4 ? RT : 4;
    __shared__ float red[4][16][16 * RG + 4];
    const AdapterJob &j = J.j[blockIdx.z];
    const int win = blockIdx.y, G = gridDim.x;
    const AdWindow w = ad_window(J, win, false);
    if (w.groups == 0) return;
    const int Q = ad_slices(G, w.groups, j.k), q = blockIdx.x / w.groups;
    if (q >= Q) return;
    const int ks = ((j.k + Q - 1) / Q + 127) / 128 * 128, k0 = q * ks, k1 = min(j.k, k0 + ks);
    float *hq = j.h + (size_t)q * J.rows * J.rank;
    for (int gi = blockIdx.x % w.groups; gi < w.groups; gi += G) {
        const AdGroup grp = ad_group(w, gi);
        const int R = grp.R;
        const _Float16 *A = j.a + (size_t)grp.a * J.rank * j.k;
        if (R == 0) continue;
        if (grp.cnt <= 16)
            ad_down_tiles<RT, 1, X16>(J, j, grp, win, 0, R, A, k0, k1, hq, red);
        else if (grp.cnt <= 32)
            ad_down_tiles<RT, 2, X16>(J, j, grp, win, 0, R, A, k0, k1, hq, red);
        else
            ad_down_tiles<RT, 4, X16>(J, j, grp, win, 0, R, A, k0, k1, hq, red);
    }
}

// The outputs of a window's rows in a piece of n.  h's slices are added in
// order and split into two fp16 numbers, hi + lo, after each row is scaled by
// a power of two to [2^9, 2^10): 22 bits of every element that counts in its
// row's sum, so the products run on v_mfma_f32_16x16x32_f16 with fp32's
// accuracy.  B's rows are the left operand: a lane holds four neighbouring n
// of one row, 16-byte loads of y and stores of out.
constexpr int kUpThreads = 256, kUpN = 128;

template <int RU>  // 32-rank units
__global__ __launch_bounds__(kUpThreads) void k_adapter_up(AdapterJobs J, int G) {
    constexpr int HS = 32 * RU + 8;
    __shared__ __align__(16) _Float16 hi[kWin][HS], lo[kWin][HS];
    __shared__ float back[kWin];  // scale times the row's power of two
    __shared__ int rowof[kWin];
    const AdapterJob &j = J.j[blockIdx.z];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int win = blockIdx.y, n0 = blockIdx.x * kUpN;
    if (n0 >= j.n) return;
    const AdWindow w = ad_window(J, win, j.out != j.y || j.epi != GE_STORE);
    const int Q = ad_slices(G, __popcll(w.leaders), j.k);
    const ad_h8 zero = {};
    for (int gi = 0; gi < w.groups; gi++) {
        const AdGroup grp = ad_group(w, gi);
        const int R = grp.R;
        const float scale = grp.scale;
        const _Float16 *B = j.b + (size_t)max(grp.a, 0) * j.n * J.rank;
        __syncthreads();
        if (threadIdx.x < kWin) rowof[threadIdx.x] = grp.row;
        __syncthreads();
        if (R) {
            const int p = threadIdx.x >> 2, c = threadIdx.x & 3;  // four threads a row, 8 RU ranks each
            float v[8 * RU];
            float top = 0.0f;
            const size_t at = ((size_t)win * kWin + rowof[p]) * J.rank;
#pragma unroll
            for (int e = 0; e < 8 * RU; e++) {
                const int r = (e >> 3) * 32 + c * 8 + (e & 7);
                float s = 0.0f;
                if (p < grp.cnt && r < R) {
                    for (int q = 0; q < Q; q++) s += j.h[(size_t)q * J.rows * J.rank + at + r];
                }
                v[e] = s;
                top = fabsf(s) < INFINITY ? fmaxf(top, fabsf(s)) : top;
            }
            top = fmaxf(top, __shfl_xor(top, 1));
            top = fmaxf(top, __shfl_xor(top, 2));
            int ex = 0;
            if (top > 0.0f) ex = max(ilogbf(top) - 9, -126);
            const float down = ldexpf(1.0f, -ex);
#pragma unroll
            for (int e = 0; e < 8 * RU; e++) {
                const int r = (e >> 3) * 32 + c * 8 + (e & 7);
                const float s = v[e] * down;
                const _Float16 a = (_Float16)s;
                hi[p][r] = a;
                lo[p][r] = fabsf(s) < INFINITY ? (_Float16)(s - (float)a) : (_Float16)0.0f;
            }
            if (c == 0) back[p] = scale * ldexpf(1.0f, ex);
        }
        __syncthreads();
        const int tiles = (grp.cnt + 15) / 16;
        for (int nt = wave; nt < kUpN / 16; nt += kUpThreads / 64) {
            const int n = n0 + 16 * nt;
            if (n >= j.n) break;
            ad_h8 b[RU];
#pragma unroll
            for (int u = 0; u < RU; u++) {
                const int r = 32 * u + 8 * g;
                b[u] = r < R && n + i < j.n ? *(const ad_h8 *)(B + (size_t)(n + i) * J.rank + r) : zero;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (r + e >= R) b[u][e] = (_Float16)0.0f;
            }
            for (int m = 0; m < tiles; m++) {
                const int p = 16 * m + i, nn = n + 4 * g;
                ad_f4 acc = {0, 0, 0, 0};
                if (R) {
#pragma unroll
                    for (int u = 0; u < RU; u++) {
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[u], *(const ad_h8 *)&lo[p][32 * u + 8 * g], acc, 0, 0, 0);
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[u], *(const ad_h8 *)&hi[p][32 * u + 8 * g], acc, 0, 0, 0);
                    }
                }
                if (p >= grp.cnt || nn >= j.n) continue;
                const size_t at = ((size_t)win * kWin + rowof[p]) * j.n + nn;
                float z[4];
                if (j.y16) {
                    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
                    const h4 y = *(const h4 *)((const _Float16 *)j.y + at);
                    for (int e = 0; e < 4; e++) z[e] = (float)y[e];
                } else {
                    const ad_f4 y = *(const ad_f4 *)((const float *)j.y + at);
                    for (int e = 0; e < 4; e++) z[e] = y[e];
                }
                for (int e = 0; e < 4; e++) z[e] = ad_epi(R ? z[e] + back[p] * acc[e] : z[e], j.epi);
                if (j.o16) {
                    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
                    h4 o;
                    for (int e = 0; e < 4; e++) o[e] = (_Float16)z[e];
                    *(h4 *)((_Float16 *)j.out + at) = o;
                } else {
                    *(ad_f4 *)((float *)j.out + at) = (ad_f4){z[0], z[1], z[2], z[3]};
                }
            }
        }
    }
}

// Blocks of a window in the first of the two launches: about 512 in all.
static int down_blocks(uint64_t rows, uint64_t njobs) {
    const uint64_t wins = (rows + kWin - 1) / kWin;
    return (int)std::max<uint64_t>(1, std::min<uint64_t>(32, 512 / (wins * njobs)));
}

uint64_t adapter_work_words(const rsv_adapter_job *, uint64_t njobs, uint64_t rank, uint64_t rows) {
    if (rows <= kWin) return 1;
    return njobs * rank * rows * down_blocks(rows, njobs);
}

template <int RT, bool X16>
static void rows_rt(rsv_ctx *ctx, const AdapterJobs &J, dim3 grid) {
    hipLaunchKernelGGL((k_adapter_rows<RT, X16>), grid, dim3(kRowsThreads), 0, ctx->stream, J);
}
template <int RT, bool X16>
static void down_rt(rsv_ctx *ctx, const AdapterJobs &J, dim3 grid) {
    hipLaunchKernelGGL((k_adapter_down<RT, X16>), grid, dim3(kDownThreads), 0, ctx->stream, J);
}
#define AD_RT(f, x16, ...)                                      \
    do {                                                        \
        if (J.rank <= 16) f<1, x16>(__VA_ARGS__);               \
        else if (J.rank <= 32) f<2, x16>(__VA_ARGS__);          \
        else if (J.rank <= 64) f<4, x16>(__VA_ARGS__);          \
        else f<8, x16>(__VA_ARGS__);                            \
    } while (0)

int launch_adapter(rsv_ctx *ctx, AdapterJobs &J, float *work) {
    const int wins = (J.rows + kWin - 1) / kWin;
    const int G = down_blocks(J.rows, J.njob);
    int nmax = 0;
    for (int i = 0; i < J.njob; i++) {
        J.j[i].h = work + (size_t)i * J.rank * J.rows * G;
        nmax = std::max(nmax, J.j[i].n);
    }
    // jobs of one x type go together (each launch's kernel takes one)
    for (int x16 = 0; x16 < 2; x16++) {
        AdapterJobs S = J;
        S.njob = 0;
        for (int i = 0; i < J.njob; i++)
            if (J.j[i].x16 == x16) S.j[S.njob++] = J.j[i];
        if (!S.njob) continue;
        if (J.rows <= kWin) {
            const dim3 grid(std::max(1, 256 / S.njob), 1, S.njob);
            if (x16) AD_RT(rows_rt, true, ctx, S, grid);
            else AD_RT(rows_rt, false, ctx, S, grid);
        } else {
            const dim3 grid(G, wins, S.njob);
            if (x16) AD_RT(down_rt, true, ctx, S, grid);
            else AD_RT(down_rt, false, ctx, S, grid);
        }
    }
    if (J.rows > kWin) {
        const dim3 grid((nmax + kUpN - 1) / kUpN, wins, J.njob);
        if (J.rank <= 32) hipLaunchKernelGGL((k_adapter_up<1>), grid, dim3(kUpThreads), 0, ctx->stream, J, G);
        else if (J.rank <= 64) hipLaunchKernelGGL((k_adapter_up<2>), grid, dim3(kUpThreads), 0, ctx->stream, J, G);
        else hipLaunchKernelGGL((k_adapter_up<4>), grid, dim3(kUpThreads), 0, ctx->stream, J, G);
    }
    RSV_HIP(hipGetLastError());
    return 0;
}

}  // namespace rsv

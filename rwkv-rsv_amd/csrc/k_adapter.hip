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
typedef _Float16 ad_h4 __attribute__((ext_vector_type(4)));
typedef float ad_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t ad_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t ad_u2 __attribute__((ext_vector_type(2)));

constexpr int kWin = 64;
constexpr int kBare = -1;  // the group of a window's rows without an adapter

// The groups of a window: one per distinct adapter, in the order of their
// first rows, then (with `bare`) one of the rows that have none.
struct AdWindow {
    uint32_t id;        // the lane's adapter,
    uint32_t rank;      // its own rank
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
    w.id = J.row_adapter[min(t, J.rows - 1)];
    const bool has = t < J.rows && w.id < (uint32_t)J.n_adapter;
    // one load behind the id's, together with each other; waited for at their use
    const uint32_t known = min(w.id, (uint32_t)J.n_adapter - 1);
    w.rank = J.ranks ? J.ranks[known] : J.rank;
    w.scale = J.scale[known];
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

__device__ __forceinline__ AdGroup ad_group(const AdapterJobs &J, const AdWindow &w, int g) {
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
        r.R = (int)min((uint32_t)__builtin_amdgcn_readlane((int)w.rank, l), (uint32_t)J.rank);
        r.scale = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w.scale), l));
        mask = ad_lane64(w.same, l);
    }
    r.cnt = __popcll(mask);
    // lane p receives the p-th row: a permutation of the lanes, the group's rows first
    const int to = mask >> lane & 1 ? __popcll(mask & below) : r.cnt + __popcll(~mask & below);
    r.row = __builtin_amdgcn_ds_permute(to * 4, lane);
    return r;
}

__device__ __forceinline__ float ad_epi(float z, int epi) {
    return epi == GE_RELU2 ? (z > 0.0f ? z * z : z == z ? 0.0f : z) : z;
}

// Memory through buffer resources: an offset past the size reads as zero and
// is not written, so tails, masked rows and ranks past an adapter's own need
// no branches around the loads.  A resource covers one adapter's matrix or one
// window's rows, at most 2^30 bytes; kOff added to an offset below that, once
// or twice, stays past every size.
constexpr uint32_t kOff = 0x40000000u;
constexpr int kNt = 2;  // non-temporal: outputs that stream past the caches (r/k/v of 4096 rows: 111 -> 83 us)
struct AdBuf {
    __amdgpu_buffer_rsrc_t r;
    __device__ __forceinline__ AdBuf(const void *p, size_t bytes) : r(__builtin_amdgcn_make_buffer_rsrc((void *)p, (short)0, (int)bytes, 0x00020000)) {}
    __device__ __forceinline__ ad_h8 h8(uint32_t at) const { return __builtin_bit_cast(ad_h8, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0)); }
    __device__ __forceinline__ ad_f4 f4(uint32_t at) const { return __builtin_bit_cast(ad_f4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0)); }
    __device__ __forceinline__ ad_h4 h4(uint32_t at) const { return __builtin_bit_cast(ad_h4, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0)); }
    __device__ __forceinline__ float f1(uint32_t at) const { return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0)); }
    __device__ __forceinline__ float h1(uint32_t at) const { return (float)__builtin_bit_cast(_Float16, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0)); }
    __device__ __forceinline__ void put(ad_f4 v, uint32_t at) const { __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(ad_u4, v), r, at, 0, kNt); }
    __device__ __forceinline__ void put(ad_h4 v, uint32_t at) const { __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(ad_u2, v), r, at, 0, kNt); }
    __device__ __forceinline__ void put(float v, uint32_t at) const { __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), r, at, 0, 0); }
    __device__ __forceinline__ void put(_Float16 v, uint32_t at) const { __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, v), r, at, 0, 0); }
};
// A window's rows of [rows, n].
__device__ __forceinline__ AdBuf ad_rows(const AdapterJobs &J, const void *p, int n, int f16, int win) {
    const size_t row = (size_t)n * (f16 ? 2 : 4);
    return AdBuf((const char *)p + (size_t)win * kWin * row, min(kWin, J.rows - win * kWin) * row);
}

// Products of a 16-rank tile with MT 16-row tiles over k in [k0, k1), one
// wave: acc[m][j][e] += x[row l%16 of tile m] . A[rank 16 j + 4 (l/16) + e].
// Lane (i = l%16, g = l/16) supplies k 8g..8g+7 of each 32: the rank rows as
// the left operand, the batch rows as the right one.  fp16 x goes through
// v_mfma_f32_16x16x32_f16 (products of fp16 are exact in fp32), fp32 x through
// eight v_mfma_f32_16x16x4_f32 with A widened, so both sum in fp32.  DEP steps
// of 32 k are in flight at once.  xrow: byte offsets of the rows (kOff: none).
template <int RT, int MT, bool X16, int DEP>
__device__ __forceinline__ void ad_dots(const AdBuf &A, const AdBuf &x, const uint32_t (&xrow)[MT], int K, int k0, int k1,
                                        ad_f4 (&acc)[MT][RT]) {
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    uint32_t arow[RT];
#pragma unroll
    for (int j = 0; j < RT; j++) arow[j] = (16 * j + i) * K * 2u;
    for (int kb = k0; kb < k1; kb += 32 * DEP) {
        ad_h8 a[DEP][RT];
        ad_h8 xh[DEP][MT];
        ad_f4 xf[DEP][MT][2];
#pragma unroll
        for (int s = 0; s < DEP; s++) {
            if (kb + 32 * s >= k1) break;
            const uint32_t k = kb + 32 * s + 8 * g;
            const bool in = (int)k < k1;
            const uint32_t ka = in ? 2 * k : 2 * kOff, kx = in ? (X16 ? 2 : 4) * k : 2 * kOff;
#pragma unroll
            for (int j = 0; j < RT; j++) a[s][j] = A.h8(arow[j] + ka);
#pragma unroll
            for (int m = 0; m < MT; m++) {
                if constexpr (X16) {
                    xh[s][m] = x.h8(xrow[m] + kx);
                } else {
                    xf[s][m][0] = x.f4(xrow[m] + kx);
                    xf[s][m][1] = x.f4(xrow[m] + kx + 16);
                }
            }
        }
#pragma unroll
        for (int s = 0; s < DEP; s++) {
            if (kb + 32 * s >= k1) break;
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
// takes a second launch; reading it again from L2 per piece of n costs less
// (ffn.key of 8 rows with 8 adapters: 36 us as two launches, 7.4 as one).
// Bound by latency: the ids, their ranks and scales, the matrices (all loads of
// a block in flight at once), the sums over the waves and the outputs follow
// one another, 5.6 us for one token, 10.8 for r/k/v of 64 rows and 48 adapters
// (22 MB, 2.1 TB/s).
constexpr int kRowsThreads = 512;

// A thread's B rows for NP neighbouring passes over n (n, n + kRowsThreads, ..).
template <int RT, int NP>
struct AdB {
    ad_h8 v[NP][2 * RT];
    __device__ __forceinline__ void load(const AdBuf &B, int R, int rank, int n, int n1) {
#pragma unroll
        for (int q = 0; q < NP; q++) {
            const int at = n + q * kRowsThreads;
            const uint32_t row = at < n1 ? at * rank * 2u : kOff;
#pragma unroll
            for (int c = 0; c < 2 * RT; c++) {
                v[q][c] = B.h8(8 * c < R ? row + 16 * c : kOff);
            }
        }
    }
};

// Outputs of `rows` rows (at most RC at a time) at the passes that bv holds.
template <int RC, int RT, int NP>
__device__ __forceinline__ void ad_up_rows(const AdapterJob &j, const AdBuf &yb, const AdBuf &ob, const float *h, int hs, int R,
                                           const AdB<RT, NP> &bv, float scale, const uint32_t *rows_of, int rows, int n, int n1) {
    float y[NP][RC];
    uint32_t at[NP][RC];  // elements of the window
#pragma unroll
    for (int q = 0; q < NP; q++) {
#pragma unroll
        for (int c = 0; c < RC; c++) {
            const int nn = n + q * kRowsThreads;
            at[q][c] = nn < n1 && c < rows ? rows_of[c] * j.n + nn : kOff;
            y[q][c] = j.y16 ? yb.h1(2 * at[q][c]) : yb.f1(4 * min(at[q][c], kOff / 2));
        }
    }
#pragma unroll
    for (int q = 0; q < NP; q++) {
        if (n - (int)threadIdx.x + q * kRowsThreads >= n1) break;
        if constexpr (RC > 1) __builtin_amdgcn_sched_barrier(0);
        float s[RC] = {};
#pragma unroll
        for (int r8 = 0; r8 < 2 * RT; r8++) {
            if (8 * r8 >= R) continue;
            const bool part = 8 * r8 + 8 > R;
            if constexpr (RT > 1) __builtin_amdgcn_sched_barrier(0);  // h's reads stay by their products: all at once they would spill
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = part && 8 * r8 + e >= R ? 0.0f : (float)bv.v[q][r8][e];
#pragma unroll
                for (int c = 0; c < RC; c++) s[c] += h[c * hs + 8 * r8 + e] * v;
            }
        }
#pragma unroll
        for (int c = 0; c < RC; c++) {
            const float z = ad_epi(R ? y[q][c] + scale * s[c] : y[q][c], j.epi);
            if (j.o16)
                ob.put((_Float16)z, 2 * at[q][c]);
            else
                ob.put(z, 4 * min(at[q][c], kOff / 2));
        }
    }
}

template <int RT, bool X16>
__global__ __launch_bounds__(kRowsThreads) void k_adapter_rows(AdapterJobs J) {
    constexpr int HS = 16 * RT + 4, RG = RT < 4 ? RT : 4;
    constexpr int NP = RT == 1 ? 5 : RT == 2 ? 3 : 1;  // B rows held from the start
    __shared__ float red[8][16][16 * RG + 4];
    __shared__ __align__(16) float h[16 * HS];
    __shared__ uint32_t rows_of[16];
    const AdapterJob &j = J.j[blockIdx.z];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int win = blockIdx.y, G = gridDim.x;
    const AdBuf xb = ad_rows(J, j.x, j.k, X16, win), yb = ad_rows(J, j.y, j.n, j.y16, win), ob = ad_rows(J, j.out, j.n, j.o16, win);
    const AdWindow w = ad_window(J, win, j.out != j.y || j.epi != GE_STORE);
    if (w.groups == 0) return;
    const int C = max(1, min(G / w.groups, (j.n + 255) / 256));
    if (blockIdx.x >= (unsigned)(w.groups * C)) return;
    const int piece = ((j.n + C - 1) / C + 63) / 64 * 64;
    const int n0 = (int)(blockIdx.x / w.groups) * piece, n1 = min(j.n, n0 + piece);
    const int ks = ((j.k + 7) / 8 + 31) / 32 * 32;  // k of a wave
    for (int gi = blockIdx.x % w.groups; gi < w.groups; gi += G) {
        const AdGroup grp = ad_group(J, w, gi);
        const int R = grp.R;
        const float scale = grp.scale;
        const AdBuf A(j.a + (size_t)max(grp.a, 0) * J.rank * j.k, (size_t)R * j.k * 2);
        const AdBuf B(j.b + (size_t)max(grp.a, 0) * j.n * J.rank, (size_t)j.n * J.rank * 2);
        AdB<RT, NP> bv;
        bv.load(B, R, J.rank, n0 + threadIdx.x, n1);
        for (int p0 = 0; p0 < grp.cnt; p0 += 16) {
            const int rows = min(16, grp.cnt - p0);
            const uint32_t row = __shfl(grp.row, p0 + i);
            const uint32_t xrow[1] = {i < rows ? row * j.k * (X16 ? 2 : 4) : kOff};
            __syncthreads();  // the tile before is done with h and rows_of
            if (wave == 0 && g == 0) rows_of[i] = row;
            if (R) {
                ad_f4 acc[1][RT] = {};
                ad_dots<RT, 1, X16, (RT == 1 ? 10 : RT == 2 ? 6 : RT == 4 ? 4 : 2)>(A, xb, xrow, j.k, wave * ks, min(j.k, (wave + 1) * ks), acc);
#pragma unroll
                for (int q = 0; q < RT; q += RG) {
#pragma unroll
                    for (int t = 0; t < RG; t++) *(ad_f4 *)&red[wave][i][16 * t + 4 * g] = acc[0][q + t];
                    __syncthreads();
                    for (int v = threadIdx.x; v < rows * 16 * RG; v += kRowsThreads) {
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
            for (int n = n0 + (int)threadIdx.x; n - (int)threadIdx.x < n1; n += NP * kRowsThreads) {
                if (n - (int)threadIdx.x > n0 || p0 > 0) bv.load(B, R, J.rank, n, n1);
                if (rows == 1)
                    ad_up_rows<1, RT, NP>(j, yb, ob, h, HS, R, bv, scale, rows_of, rows, n, n1);
                else if (rows == 2)
                    ad_up_rows<2, RT, NP>(j, yb, ob, h, HS, R, bv, scale, rows_of, rows, n, n1);
                else
                    for (int c = 0; c < rows; c += 4) ad_up_rows<4, RT, NP>(j, yb, ob, h + c * HS, HS, R, bv, scale, rows_of + c, rows - c, n, n1);
            }
        }
    }
}

// ------------------------------------------------ many rows: two launches
// h of a window's rows: 4 waves over a slice of k, their sums added in wave
// order into slice q of the work area, h[q][t][r].  A wave's part of k is at
// most 320, loaded in two batches; fewer and longer slices cost less than the
// reading of more partial sums by the second launch (r/k/v of 4096 rows: 99,
// 83, 77, 81 us at slices of 320, 640, 1280, 2560; 517 rows of k = 10240: 41,
// 31, 25, 28).
constexpr int kDownThreads = 256, kDownWaves = kDownThreads / 64;

// Lines of 128 bytes a row (64 k of fp16, 32 of fp32) whose operands fit about 128 registers.
constexpr int ad_lines(int RT, int MT, bool x16) {
    const int d = 128 / (8 * MT + (x16 ? 8 : 4) * RT);
    return d < 1 ? 1 : d > 3 ? 3 : d;
}

// ad_dots for whole windows: x comes as eight lanes a row, whole lines, and
// through LDS (a wave's own 16 x 128 bytes) into the operands' layout.  rows:
// byte offsets of rows l/8 and 8 + l/8 of each tile.
template <int RT, int MT, bool X16, int NL>
__device__ __forceinline__ void ad_dots_lines(const AdBuf &A, const AdBuf &x, const uint32_t (&rows)[MT][2], int K, int k0, int k1,
                                              ad_f4 (&acc)[MT][RT], float (*tile)[36]) {
    constexpr int LK = X16 ? 64 : 32, ST = LK / 32;  // k of a line, its steps of 32
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    uint32_t arow[RT];
#pragma unroll
    for (int j = 0; j < RT; j++) arow[j] = (16 * j + i) * K * 2u;
    for (int kb = k0; kb < k1; kb += LK * NL) {
        ad_h8 a[NL][ST][RT];
        ad_f4 q[NL][MT][2];
#pragma unroll
        for (int l = 0; l < NL; l++) {
            if (kb + LK * l >= k1) break;
            const uint32_t kx = kb + LK * l + (lane & 7) * (X16 ? 8 : 4), ox = (int)kx < k1 ? kx * (X16 ? 2 : 4) : 2 * kOff;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                q[l][m][0] = x.f4(rows[m][0] + ox);
                q[l][m][1] = x.f4(rows[m][1] + ox);
            }
#pragma unroll
            for (int s = 0; s < ST; s++) {
                const uint32_t k = kb + LK * l + 32 * s + 8 * g, oa = (int)k < k1 ? 2 * k : 2 * kOff;
#pragma unroll
                for (int j = 0; j < RT; j++) a[l][s][j] = A.h8(arow[j] + oa);
            }
        }
#pragma unroll
        for (int l = 0; l < NL; l++) {
            if (kb + LK * l >= k1) break;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                *(ad_f4 *)&tile[lane >> 3][4 * (lane & 7)] = q[l][m][0];
                *(ad_f4 *)&tile[8 + (lane >> 3)][4 * (lane & 7)] = q[l][m][1];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                const ad_f4 x0 = *(const ad_f4 *)&tile[i][X16 ? 4 * g : 8 * g], x1 = *(const ad_f4 *)&tile[i][X16 ? 16 + 4 * g : 8 * g + 4];
#pragma unroll
                for (int j = 0; j < RT; j++) {
                    if constexpr (X16) {
                        acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[l][0][j], __builtin_bit_cast(ad_h8, x0), acc[m][j], 0, 0, 0);
                        acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[l][ST - 1][j], __builtin_bit_cast(ad_h8, x1), acc[m][j], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)a[l][0][j][e], e < 4 ? x0[e & 3] : x1[e & 3], acc[m][j], 0, 0, 0);
                    }
                }
            }
        }
    }
}

template <int RT, int MT, bool X16>
__device__ __forceinline__ void ad_down_tiles(const AdapterJobs &J, const AdapterJob &j, const AdGroup &grp, int win, int R,
                                              const AdBuf &A, const AdBuf &x, int k0, int k1, float *hq, float (*red)[16][16 * (RT < 4 ? RT : 4) + 4],
                                              float (*tile)[16][36]) {
    constexpr int RG = RT < 4 ? RT : 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    uint32_t rows[MT][2];
#pragma unroll
    for (int m = 0; m < MT; m++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int p = 16 * m + 8 * h + (lane >> 3);
            const uint32_t row = __shfl(grp.row, p);
            rows[m][h] = p < grp.cnt ? row * j.k * (X16 ? 2 : 4) : kOff;
        }
    }
    const int ks = ((k1 - k0 + kDownWaves - 1) / kDownWaves + 63) / 64 * 64;
    ad_f4 acc[MT][RT] = {};
    ad_dots_lines<RT, MT, X16, ad_lines(RT, MT, X16)>(A, x, rows, j.k, min(k1, k0 + wave * ks), min(k1, k0 + (wave + 1) * ks), acc, tile[wave]);
#pragma unroll
    for (int m = 0; m < MT; m++) {
        if (16 * m >= grp.cnt) break;
#pragma unroll
        for (int q = 0; q < RT; q += RG) {
            __syncthreads();
#pragma unroll
            for (int t = 0; t < RG; t++) *(ad_f4 *)&red[wave][i][16 * t + 4 * g] = acc[m][q + t];
            __syncthreads();
            // four neighbouring ranks a thread
            for (int v = threadIdx.x; v < 16 * 4 * RG; v += kDownThreads) {
                const int hr = v / (4 * RG), hc = 4 * (v % (4 * RG)), p = 16 * m + hr, r = 16 * q + hc;
                ad_f4 s = {0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < kDownWaves; u++) s += *(const ad_f4 *)&red[u][hr][hc];
                const int row = __builtin_amdgcn_ds_bpermute(4 * (p & 63), grp.row);
                // the second launch reads whole eights of ranks
                if (p < grp.cnt && r < (R + 7) / 8 * 8) *(ad_f4 *)&hq[((size_t)win * kWin + row) * J.rank + r] = s;
            }
        }
    }
}

// grid (slices, windows, slots x jobs): slot s takes the window's groups s, s +
// slots, ... (slots in the slowest dimension, so that the blocks that find no
// group do not leave whole XCDs idle)
template <int RT, bool X16>
__global__ __launch_bounds__(kDownThreads) void k_adapter_down(AdapterJobs J, int slots) {
    constexpr int RG = RT < 4 ? RT : 4;
    __shared__ float red[kDownWaves][16][16 * RG + 4];
    __shared__ __align__(16) float tile[kDownWaves][16][36];
    const int slot = blockIdx.z / J.njob;
    const AdapterJob &j = J.j[blockIdx.z % J.njob];
    const int win = blockIdx.y, q = blockIdx.x, k0 = q * J.slice, k1 = min(j.k, k0 + J.slice);
    if (k0 >= j.k) return;
    const AdWindow w = ad_window(J, win, false);
    float *hq = j.h + (size_t)q * J.rows * J.rank;
    const AdBuf x = ad_rows(J, j.x, j.k, X16, win);
    for (int gi = slot; gi < w.groups; gi += slots) {
        const AdGroup grp = ad_group(J, w, gi);
        const int R = grp.R;
        if (R == 0) continue;
        const AdBuf A(j.a + (size_t)grp.a * J.rank * j.k, (size_t)R * j.k * 2);
        if (grp.cnt <= 16)
            ad_down_tiles<RT, 1, X16>(J, j, grp, win, R, A, x, k0, k1, hq, red, tile);
        else if (grp.cnt <= 32)
            ad_down_tiles<RT, 2, X16>(J, j, grp, win, R, A, x, k0, k1, hq, red, tile);
        else
            ad_down_tiles<RT, 4, X16>(J, j, grp, win, R, A, x, k0, k1, hq, red, tile);
    }
}

// The two launches are bound by memory: r/k/v of 4096 rows (fp16 x, fp32 y and
// out in place) move 325 MB in 18.4 + 46.4 us (5.0 TB/s; a copy reaches 5.1);
// 517 rows of k = 10240 take 9.3 + 8.7, mostly ramp and tail.  Windows of many
// adapters with a row each keep too few bytes in flight (256 rows of 256
// adapters, r/k/v: 72 us, 1.7 TB/s); two to four times the slots below make
// that 73 to 76.
//
// The outputs of a window's rows in a piece of n.  h's slices are added in
// order and split into two fp16 numbers, hi + lo, after each row is scaled by
// a power of two to [2^9, 2^10): 22 bits of every element that counts in its
// row's sum, so the products run on v_mfma_f32_16x16x32_f16 with fp32's
// accuracy.  B's rows are the left operand: a lane holds four neighbouring n
// of one row.
constexpr int kUpThreads = 256, kUpN = 128;

// h of row p of a group into hi, lo and back: four lanes a row (c), eights of
// ranks each.  src: the window row; live: the row is the group's.
template <int RU>
__device__ __forceinline__ void ad_stage(const AdapterJobs &J, const AdapterJob &j, int win, int Q, int R, int p, int c,
                                         uint32_t src, bool live, _Float16 (*hi)[32 * RU + 8], _Float16 (*lo)[32 * RU + 8], float *back) {
    const uint32_t hrow = live ? src * J.rank * 4u + 32 * c : kOff;
    ad_f4 v[RU][2] = {};
#pragma unroll 8
    for (int q = 0; q < Q; q++) {
        const AdBuf hb = ad_rows(J, j.h + (size_t)q * J.rows * J.rank, J.rank, 0, win);
#pragma unroll
        for (int u = 0; u < RU; u++) {
            const uint32_t o = 32 * u + 8 * c < R ? hrow + 128 * u : kOff;
            v[u][0] += hb.f4(o);
            v[u][1] += hb.f4(o + 16);
        }
    }
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < 8 * RU; e++) {
        float &s = ((float *)v)[e];
        if ((e >> 3) * 32 + c * 8 + (e & 7) >= R) s = 0.0f;
        top = fabsf(s) < INFINITY ? fmaxf(top, fabsf(s)) : top;
    }
    top = fmaxf(top, __shfl_xor(top, 1));
    top = fmaxf(top, __shfl_xor(top, 2));
    // the row's power of two from its exponent bits: 2^ex with top / 2^ex in [2^9, 2^10)
    const int ex = max((int)(__float_as_uint(top) >> 23) - 127 - 9, -126);
    const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
#pragma unroll
    for (int u = 0; u < RU; u++) {
        ad_h8 a, z;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float s = ((const float *)v[u])[e] * down;
            a[e] = (_Float16)s;
            z[e] = fabsf(s) < INFINITY ? (_Float16)(s - (float)a[e]) : (_Float16)0.0f;
        }
        *(ad_h8 *)&hi[p][32 * u + 8 * c] = a;
        *(ad_h8 *)&lo[p][32 * u + 8 * c] = z;
    }
    if (c == 0) back[p] = __uint_as_float((uint32_t)(127 + ex) << 23);
}

// Four neighbouring n of a row of y (elements at `at` of the window), and the outputs.
__device__ __forceinline__ ad_f4 ad_y4(const AdapterJob &j, const AdBuf &yb, uint32_t at) {
    if (j.y16) {
        const ad_h4 v = yb.h4(2 * at);
        return (ad_f4){(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
    }
    return yb.f4(4 * at);
}
__device__ __forceinline__ void ad_out4(const AdapterJob &j, const AdBuf &ob, ad_f4 z, uint32_t at) {
#pragma unroll
    for (int e = 0; e < 4; e++) z[e] = ad_epi(z[e], j.epi);
    if (j.o16)
        ob.put((ad_h4){(_Float16)z[0], (_Float16)z[1], (_Float16)z[2], (_Float16)z[3]}, 2 * at);
    else
        ob.put(z, 4 * at);
}
template <int RU>
__device__ __forceinline__ void ad_clear_past(ad_h8 (&b)[RU], int R, int g) {  // what lies past the adapter's own rank
    if (R % 8 == 0) return;
#pragma unroll
    for (int u = 0; u < RU; u++)
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (32 * u + 8 * g + e >= R) b[u][e] = (_Float16)0.0f;
}

template <int RU, bool ONE>  // 32-rank units; one block for all groups of a window
__global__ __launch_bounds__(kUpThreads, RU <= 2 ? 4 : 2) void k_adapter_up(AdapterJobs J, int slots) {
    constexpr int HS = 32 * RU + 8;
    __shared__ __align__(16) _Float16 hi[kWin][HS], lo[kWin][HS];
    __shared__ float back[kWin];  // the row's power of two
    __shared__ __align__(16) float tile[kUpThreads / 64][16][36];
    const int slot = ONE ? 0 : blockIdx.z / J.njob, step = ONE ? 1 : slots;
    const AdapterJob &j = J.j[ONE ? blockIdx.z : blockIdx.z % J.njob];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int win = blockIdx.y, n0 = blockIdx.x * kUpN;
    if (n0 >= j.n) return;
    const AdWindow w = ad_window(J, win, j.out != j.y || j.epi != GE_STORE);
    const int Q = (j.k + J.slice - 1) / J.slice;
    const AdBuf yb = ad_rows(J, j.y, j.n, j.y16, win), ob = ad_rows(J, j.out, j.n, j.o16, win);
    for (int gi = slot; gi < w.groups; gi += step) {
        const AdGroup grp = ad_group(J, w, gi);
        const int R = grp.R, tiles = (grp.cnt + 15) / 16;
        const AdBuf B(j.b + (size_t)max(grp.a, 0) * j.n * J.rank, R ? (size_t)j.n * J.rank * 2 : 0);
        // everything the block reads is asked for before the first wait: a
        // wave's two neighbouring 16-n tiles of B, its 32 n of y as eight lanes
        // a row (a whole 128-byte line of fp32: 64 bytes a row at a time took
        // 71 us for r/k/v of 4096 rows, this 55) ...
        const int n = n0 + 32 * wave, yn = n + 4 * (lane & 7), yrow = lane >> 3;
        ad_h8 b[2][RU];
        ad_f4 y[4][2];
        uint32_t at[4][2];  // elements of the window
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int nb = n + 16 * t + i;
#pragma unroll
            for (int u = 0; u < RU; u++) {
                const int r = 32 * u + 8 * g;
                b[t][u] = B.h8(r < R && nb < j.n ? (nb * J.rank + r) * 2u : kOff);
            }
        }
#pragma unroll
        for (int m = 0; m < 4; m++) {
            if (m >= tiles) break;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int p = 16 * m + 8 * t + yrow;
                const uint32_t row = __shfl(grp.row, p);
                at[m][t] = p < grp.cnt && yn < j.n ? row * j.n + yn : kOff / 2;
                y[m][t] = ad_y4(j, yb, at[m][t]);
            }
        }
        // ... and the slices of h: four threads a row, eights of ranks each
        if (gi != slot) __syncthreads();
        if (R) {
            const int p = threadIdx.x >> 2;
            const uint32_t src = __builtin_amdgcn_ds_bpermute(4 * p, grp.row);  // all lanes take part
            ad_stage<RU>(J, j, win, Q, R, p, threadIdx.x & 3, src, p < grp.cnt, hi, lo, back);
            __syncthreads();
            ad_clear_past(b[0], R, g);
            ad_clear_past(b[1], R, g);
        }
#pragma unroll
        for (int m = 0; m < 4; m++) {
            if (m >= tiles) break;
            const int p = 16 * m + i;
            ad_f4 acc[2] = {};
            if (R) {
#pragma unroll
                for (int u = 0; u < RU; u++) {
                    const ad_h8 l = *(const ad_h8 *)&lo[p][32 * u + 8 * g], a = *(const ad_h8 *)&hi[p][32 * u + 8 * g];
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[t][u], l, acc[t], 0, 0, 0);
                        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[t][u], a, acc[t], 0, 0, 0);
                    }
                }
            }
            // the tile through LDS: from (row, 4 n) of 16 rows to eight lanes a row
            if (R) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int t = 0; t < 2; t++) *(ad_f4 *)&tile[wave][i][16 * t + 4 * g] = grp.scale * (back[p] * acc[t]);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
#pragma unroll
            for (int t = 0; t < 2; t++) {
                ad_f4 z = y[m][t];
                if (R) z += *(const ad_f4 *)&tile[wave][8 * t + yrow][4 * (lane & 7)];
                ad_out4(j, ob, z, at[m][t]);
            }
        }
    }
}

// k of a slice in the first of the two launches: long slices leave the second
// launch fewer partial sums to read, but a launch that would leave most of the
// chip idle is over sooner with short ones.
static uint64_t down_slice(const rsv_adapter_job *jobs, uint64_t njobs, uint64_t rows) {
    uint64_t blocks = 0;
    for (uint64_t i = 0; i < njobs; i++) blocks += (rows + kWin - 1) / kWin * ((jobs[i].k + 1279) / 1280);
    return blocks <= 32 ? 640 : 1280;
}

uint64_t adapter_work_words(const rsv_adapter_job *jobs, uint64_t njobs, uint64_t rank, uint64_t rows) {
    if (rows <= kWin) return 1;
    const uint64_t slice = down_slice(jobs, njobs, rows);
    uint64_t n = 0;
    for (uint64_t i = 0; i < njobs; i++) n += (jobs[i].k + slice - 1) / slice * rank * rows;
    return n;
}

template <int RT, bool X16>
static void rows_rt(rsv_ctx *ctx, const AdapterJobs &J, dim3 grid) {
    hipLaunchKernelGGL((k_adapter_rows<RT, X16>), grid, dim3(kRowsThreads), 0, ctx->stream, J);
}
template <int RT, bool X16>
static void down_rt(rsv_ctx *ctx, const AdapterJobs &J, dim3 grid, int slots) {
    hipLaunchKernelGGL((k_adapter_down<RT, X16>), grid, dim3(kDownThreads), 0, ctx->stream, J, slots);
}
template <int RU>
static void up_ru(rsv_ctx *ctx, const AdapterJobs &J, dim3 grid, int slots) {
    if (slots == 1)
        hipLaunchKernelGGL((k_adapter_up<RU, true>), grid, dim3(kUpThreads), 0, ctx->stream, J, 1);
    else
        hipLaunchKernelGGL((k_adapter_up<RU, false>), grid, dim3(kUpThreads), 0, ctx->stream, J, slots);
}
#define AD_RT(f, x16, ...)                                      \
    do {                                                        \
        if (J.rank <= 16) f<1, x16>(__VA_ARGS__);               \
        else if (J.rank <= 32) f<2, x16>(__VA_ARGS__);          \
        else if (J.rank <= 64) f<4, x16>(__VA_ARGS__);          \
        else f<8, x16>(__VA_ARGS__);                            \
    } while (0)

int launch_adapter(rsv_ctx *ctx, AdapterJobs &J, const rsv_adapter_job *jobs, float *work) {
    const int wins = (J.rows + kWin - 1) / kWin;
    J.slice = (int)down_slice(jobs, J.njob, J.rows);
    int nmax = 0, qmax = 0;
    for (int i = 0; i < J.njob; i++) {
        const int q = (J.j[i].k + J.slice - 1) / J.slice;
        J.j[i].h = work;
        work += (size_t)q * J.rank * J.rows;
        nmax = std::max(nmax, J.j[i].n);
        qmax = std::max(qmax, q);
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
            // slots a window: about 512 blocks in all, and two where a packed chunk has
            // windows with the end of one request and the start of the next (75 -> 70 us at 4096 rows)
            const int slots = std::max(2, std::min(kWin, 512 / (wins * S.njob * qmax)));
            const dim3 grid(qmax, wins, slots * S.njob);
            if (x16) AD_RT(down_rt, true, ctx, S, grid, slots);
            else AD_RT(down_rt, false, ctx, S, grid, slots);
        }
    }
    if (J.rows > kWin) {
        const int chunks = (nmax + kUpN - 1) / kUpN;
        const int slots = std::max(1, std::min(kWin, 1024 / (chunks * wins * J.njob)));
        const dim3 grid(chunks, wins, slots * J.njob);
        if (J.rank <= 32) up_ru<1>(ctx, J, grid, slots);
        else if (J.rank <= 64) up_ru<2>(ctx, J, grid, slots);
        else up_ru<4>(ctx, J, grid, slots);
    }
    RSV_HIP(hipGetLastError());
    return 0;
}

}  // namespace rsv

// What a served step takes from its logits rows: draws from given random
// numbers (rsv_sample_rand_batch) and log-probabilities of given tokens
// (rsv_token_logprobs).
#include <algorithm>
#include <type_traits>

#include "k_dpp.h"
#include "rsv_common.h"

namespace rsv {

constexpr float kLog2e = 1.44269504088896340736f;

// A logit as the row's order sees it: NaN as -inf, -0 as +0.
__device__ __forceinline__ float lg_clean(float l) { return l == l ? l + 0.0f : -INFINITY; }
template <bool F16>
__device__ __forceinline__ float lg_value(const void *p, size_t i) {
    return lg_clean(F16 ? (float)((const _Float16 *)p)[i] : ((const float *)p)[i]);
}
// One of 16 bytes' logits as it is.
template <bool F16>
__device__ __forceinline__ float raw_value(const uint4 &q, int x) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[x >> 1] >> (16 * (x & 1))));
    else return __uint_as_float(w[x]);
}
// Order-preserving bits: larger logit, larger key.
__device__ __forceinline__ uint32_t lg_key(float l) {
    const uint32_t b = __float_as_uint(l);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lg_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// 16 bytes of a row's logits as floats (8 halves or 4 floats).
template <bool F16>
__device__ __forceinline__ void lg_unpack(uint4 q, float (&v)[F16 ? 8 : 4]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (F16) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            v[e] = lg_clean((float)__builtin_bit_cast(_Float16, h));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = lg_clean(__uint_as_float(w[e]));
    }
}

// ------------------------------------------------------------- draws
// Two launches.  k_draw_scan: a block per (row, piece of 8192 tokens) leaves
// the piece's maximum, its sum of weights and, where the row's settings cut
// anything, its histogram over eighths of an octave of weight.  k_draw_pick: a
// block per row finds the cut from the histograms and resolves it inside the
// one bin that holds it.  So the row is read once, and then the pieces that
// have tokens in that bin:
// - at most 256 tokens from the maximum down to the bin (peaked rows, small
//   top-k): listed together, they settle both cuts and the draw (kAll);
// - otherwise the bin's tokens are listed (in LDS, 4096 at a time), the cut is
//   narrowed to one key, the draw's piece follows from the pieces' kept sums and
//   the token from that piece alone.
//
// Bounds.  Many rows without cuts stream: 256 rows of 65536 fp32 logits take 21
// us in the first launch (3.2 TB/s; the rest is 64-bit float work) and 6.6 in
// the second.  Rows with cuts are bound by the second launch's chain of reads,
// barriers and LDS round trips on one CU: of one peaked row's 13 us, 3 are the
// settings, the pieces and the table, 3 the bin, 6 the listing, 2 the rest; 64
// mixed rows take 7.6 + 22.  A piece's own list of its largest tokens, made by
// the first launch, saved 5 us of listing and cost 1.6 there and 1 to 5 in rows
// that it did not settle.  256 threads: what all waves do alike costs a SIMD's
// issue slots once a wave, and 16 waves a block took four times as long for it.
//
// A token's weight is 2^x, x = l log2(e) / T, held as an integer with `bits`
// bits below E, a whole octave above the piece's largest x.  With c = 1024
// log2(e) / T: q = l c rounded to an integer (adding 1.5 2^52 leaves it in the
// sum's low bits, right for |l c| < 2^51), r = l c - q in one rounding, and
//   2^x = 2^(q >> 10) tab[q & 1023] (1 + r ln2/1024 + ...),
// a Taylor polynomial of degree 3 in an argument below 3.4e-4 (6e-16 off).
// Adding 2^52 to the scaled weight leaves the integer in the low bits.  Eight
// 64-bit float operations a token; exp() takes about four times as many.
// Weights that round to nothing have no share: below 2^-49 of the piece's
// largest, 2^-38 in rows with cuts (whose bins leave a weight 37 bits beside a
// count).  Integers add up the same in any order; pieces are put together in 64-bit
// floats in the pieces' order, which depends on n alone.  Bins follow q, so
// they mean the same in every piece.
//
// Tokens 36.5 T and more below a piece's maximum (2^-52) have no weight and
// stand in no bin.  Rows that are only settled by their maximum (+inf, or
// |l c| past 2^50, where different logits are 36 T apart) are `sharp`: tokens
// at the maximum weigh 2^(bits - 1), the others nothing.
constexpr int kPiece = 8192, kGroup = 1024, kGroups = kPiece / kGroup;
constexpr int kScanThreads = 512, kPickThreads = 256;
constexpr int kBins = 512, kSteps = 1024, kBinShift = 7, kMaxPieces = (int)(kLogitsMaxN / kPiece);
constexpr int kSharpDown = kSteps - 1;  // a sharp maximum stands in its first octave's last bin
constexpr int kDeepBin = 50 * 8;  // from here on weights vanish beside the maximum's
constexpr int kPlainBits = 48;    // weights of a row without cuts
constexpr int kCutBits = 37;      // with cuts: a bin packs its sum (8192 2^37 = 2^50) and above it its count
constexpr int kInBits = 40;       // inside a bin, below the bin's octave: up to 2^20 tokens
constexpr uint64_t kSumMask = ((uint64_t)1 << 50) - 1;
constexpr int kList = 4096, kListRoom = kList + 8;  // a bin's tokens held in LDS; half a piece and a vector

struct DrawPiece {
    float m;        // largest logit (-inf: nothing to draw)
    uint32_t idx;   // its lowest token (greedy rows)
    double e;       // 1024 E
    uint64_t sum, group[kGroups];  // of the piece and of each 1024 tokens (plain rows)
};
struct DrawWork {
    DrawPiece *piece;   // [rows, P]
    uint64_t *hist;     // [rows, P, kBins]
};
struct DrawRow {
    double T, c;
    float min_p;     // > 0: active
    uint32_t top_k;  // > 0 and < n: active
    float top_p;     // < 1: active
    bool greedy, cuts;
};

__device__ __forceinline__ DrawRow draw_row(const float *f, int n) {
    DrawRow d;
    const float T = f[0], p = f[2], m = f[3];
    const uint32_t k = __float_as_uint(f[1]);
    d.greedy = !(T > 0.0f);
    d.T = T;
    d.c = kSteps * 1.4426950408889634074 / (double)T;
    d.top_k = k < (uint32_t)n ? k : 0;
    d.top_p = p < 1.0f ? fmaxf(p, 0.0f) : 1.0f;
    d.min_p = m > 0.0f && T < INFINITY ? fminf(m, 1.0f) : 0.0f;
    d.cuts = !d.greedy && (d.top_k || d.top_p < 1.0f || d.min_p > 0.0f);
    return d;
}

constexpr double kInfE = 1e300;
constexpr double kRound = 6755399441055744.0;  // 1.5 2^52
__device__ __forceinline__ bool draw_sharp(float m, double c) { return m == INFINITY || fabs((double)m * c) >= 1125899906842624.0; }
__device__ __forceinline__ double draw_e(float m, double c) {
    return m == INFINITY ? kInfE : kSteps * (floor(rint((double)m * c) * (1.0 / kSteps)) + 1.0);
}
// The logit from which tokens carry weight beside a maximum m; -inf never does.
constexpr float kLeast = -3.402823466e38f;
__device__ __forceinline__ float draw_low(float m, const DrawRow &d) {
    return m == INFINITY ? m : fmaxf((float)((double)m - 36.5 * d.T), kLeast);
}

// What weights are taken against: a piece's octave or a bin's.
struct DrawUnit {
    double c;
    uint32_t e;      // low word of E + kRound
    float m;         // sharp: the one logit that weighs
    bool sharp;
    __device__ DrawUnit(double c_, double e_, float m_) : c(c_), e((uint32_t)__double_as_longlong(e_ + kRound)), m(m_), sharp(draw_sharp(m_, c_)) {}
    // q - E, at most 0 (and not below -60 octaves, where nothing is left to weigh)
    __device__ int steps(float l, double &r) const {
        const double t = fma((double)l, c, kRound);
        r = fma((double)l, c, kRound - t);
        return max((int)((uint32_t)__double_as_longlong(t) - e), -60 * kSteps);
    }
};
__device__ __forceinline__ uint64_t draw_value(int k, double r, int bits, const double *tab) {
    constexpr double a1 = 0.69314718055994530942 / kSteps, a2 = a1 * a1 / 2.0, a3 = a2 * a1 / 3.0;
    const double p = fma(r, fma(r, fma(r, a3, a2), a1), 1.0);
    const double t = __longlong_as_double(__double_as_longlong(tab[k & (kSteps - 1)]) + ((int64_t)((k >> 10) + bits) << 52));
    return (uint64_t)__double_as_longlong(fma(t, p, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
}
// A token's weight; l at or above draw_low of the unit's maximum.
__device__ __forceinline__ uint64_t draw_weight(const DrawUnit &u, float l, int bits, const double *tab, int &down) {
    if (u.sharp) {
        down = kSharpDown;
        return l == u.m ? 1ull << (bits - 1) : 0;
    }
    double r;
    const int k = u.steps(l, r);
    down = -k;
    return draw_value(k, r, bits, tab);
}
// 2^(i / 1024), made by the compiler: the series of exp, smallest terms first.
struct DrawTable {
    double v[kSteps];
    constexpr DrawTable() : v() {
        for (int i = 0; i < kSteps; i++) {
            const double x = 0.69314718055994530942 * i / kSteps;
            double t[24] = {1.0}, sum = 0.0;
            for (int k = 1; k < 24; k++) t[k] = t[k - 1] * x / k;
            for (int k = 23; k >= 0; k--) sum += t[k];
            v[i] = sum;
        }
    }
};
__device__ const DrawTable kDrawTable{};
template <int NT>
__device__ __forceinline__ void draw_table(double *tab) {
#pragma unroll
    for (int i = 0; i < kSteps / 2; i += NT)
        if (kSteps / 2 % NT == 0 || i + (int)threadIdx.x < kSteps / 2) ((double2 *)tab)[i + threadIdx.x] = ((const double2 *)kDrawTable.v)[i + threadIdx.x];
}

// Sums over a wave by row shifts and broadcasts: the inclusive scan, whose last
// lane holds the sum.
template <int CTRL, int RM, typename T>
__device__ __forceinline__ T dpp64(T v) {
    static_assert(sizeof(T) == 8);
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, RM, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, RM, 0xF, false);
    return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    v += dpp64<0x111, 0xF>(v);
    v += dpp64<0x112, 0xF>(v);
    v += dpp64<0x114, 0xF>(v);
    v += dpp64<0x118, 0xF>(v);
    v += dpp64<0x142, 0xA>(v);
    v += dpp64<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint32_t wave_scan32(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
    return v;
}
template <typename T>
__device__ __forceinline__ T lane_of(T v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
    return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
}

// A piece's tokens over NT threads: a wave has a contiguous part, lane l the
// 16-byte vectors l, l + 64, ... of it, from the border at or before the piece's
// first token on, and thread t one more behind them where the row does not start
// at a border; tokens that are not the piece's
// are -inf.  Vectors stay inside the tensor's memory, whose end is padded.
template <bool F16, int NT>
struct PieceView {
    static constexpr int V = F16 ? 8 : 4, NV = kPiece / NT / V + 1, N = NV * V;
    const uint4 *q;
    int first, off, len;  // token of the border, piece's first token behind it, its tokens
    bool whole;           // nothing to mask: NV - 1 full vectors
    __device__ __forceinline__ PieceView(const void *logits, size_t base, int p, int n) {
        const size_t at = base + (size_t)p * kPiece;
        off = (int)(at % V);
        first = p * kPiece - off;
        len = min(kPiece, n - p * kPiece);
        whole = off == 0 && len == kPiece;
        q = (const uint4 *)((const char *)logits + (at - off) * (F16 ? 2 : 4));
    }
    static __device__ __forceinline__ int vec(int b) {
        const int t = threadIdx.x;
        return b == NV - 1 ? NT * (NV - 1) + t : (t >> 6) * (64 * (NV - 1)) + 64 * b + (t & 63);
    }
    __device__ __forceinline__ int token(int x) const { return first + vec(x / V) * V + x % V; }
    // past the piece's end its last vector again
    __device__ __forceinline__ void load(uint4 (&r)[NV]) const {
        const int last = (len + off - 1) / V;
#pragma unroll
        for (int b = 0; b < NV - 1; b++) r[b] = q[min(vec(b), last)];
        if (off) r[NV - 1] = q[min(vec(NV - 1), last)];
    }
    // which of a thread's tokens X0 to X1 - 1 are in a range: X1 - 1 in the lowest bit; a NaN is not
    template <int X0, int X1>
    static __device__ __forceinline__ uint32_t within(const uint4 (&r)[NV], float lo, float hi) {
        uint32_t hits = 0;
#pragma unroll
        for (int x = X0; x < X1; x++) {
            const float l = raw_value<F16>(r[x / V], x % V);
            hits = hits + hits + (__builtin_amdgcn_fmed3f(l, lo, hi) == l);
        }
        return hits;
    }
    // takes a neighbour's tokens out of within<0, N - V> and within<N - V, N>
    __device__ __forceinline__ void own(uint32_t &hits, uint32_t &more) const {
        uint32_t mask = 0;
#pragma unroll
        for (int b = 0; b < NV; b++) {
            const int i = vec(b) * V;  // behind the border
            const int lo = min(max(off - i, 0), V), hi = min(max(len + off - i, 0), V);
            const uint32_t in = hi > lo ? (1u << (V - lo)) - (1u << (V - hi)) : 0;
            if (b == NV - 1)
                more &= in;
            else
                mask = mask << V | in;
        }
        hits &= mask;
    }
    // sets what is not the piece's to -inf
    __device__ __forceinline__ void edges(uint4 (&r)[NV]) const {
        if (off == 0) r[NV - 1] = make_uint4(0,0,0,0);
        if (whole) {
            constexpr uint32_t none = F16 ? 0xFC00FC00u : 0xFF800000u;
            r[NV - 1] = make_uint4(none, none, none, none);
            return;
        }
#pragma unroll
        for (int b = 0; b < NV; b++) {
            const int i = vec(b) * V;
            if (i >= off && i + V <= len + off) continue;
            uint32_t w[4] = {r[b].x, r[b].y, r[b].z, r[b].w};
#pragma unroll
            for (int x = 0; x < V; x++) {
                if (i + x >= off && i + x < len + off) continue;
                if constexpr (F16)
                    w[x >> 1] = x & 1 ? (w[x >> 1] & 0xFFFFu) | 0xFC000000u : (w[x >> 1] & 0xFFFF0000u) | 0xFC00u;
                else
                    w[x] = 0xFF800000u;
            }
            r[b] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    __device__ __forceinline__ void values(uint4 (&r)[NV], float (&v)[N]) const {
        edges(r);
#pragma unroll
        for (int b = 0; b < NV; b++) {
            float w[V];
            lg_unpack<F16>(r[b], w);
#pragma unroll
            for (int x = 0; x < V; x++) v[b * V + x] = w[x];
        }
    }
};

template <bool F16>
__global__ __launch_bounds__(kScanThreads) void k_draw_scan(const void *__restrict__ logits, int n, int P,
                                                            const float *__restrict__ filter, DrawWork W) {
    constexpr int NT = kScanThreads, NW = NT / 64;
    __shared__ double tab[kSteps];
    __shared__ uint64_t hist[kBins];
    __shared__ uint64_t group[kGroups];
    __shared__ float sm[NW];
    __shared__ uint32_t si[NW];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x / P;
    const int p = blockIdx.x % P;
    using View = PieceView<F16, NT>;
    const View view(logits, row * n, p, n);
    uint4 raw[View::NV];
    view.load(raw);
    const DrawRow d = draw_row(filter + 4 * row, n);
    if (!d.greedy) draw_table<NT>(tab);
    if (d.cuts)
        for (int b = tid; b < kBins; b += NT) hist[b] = 0;
    float v[View::N];
    view.values(raw, v);
    float m = v[0];
#pragma unroll
    for (int x = 1; x < View::N; x++) m = fmaxf(m, v[x]);
    m = wave_max_last(m);
    if (lane == 63) sm[wave] = m;
    __syncthreads();
    m = sm[0];
#pragma unroll
    for (int w = 1; w < NW; w++) m = fmaxf(m, sm[w]);
    DrawPiece *out = W.piece + row * P + p;
    if (d.greedy) {
        uint32_t idx = 0xFFFFFFFFu;
#pragma unroll
        for (int x = View::N - 1; x >= 0; x--)
            if (v[x] == m) idx = min(idx, (uint32_t)view.token(x));  // where all are -inf the draw does not look
        for (int s = 32; s; s >>= 1) idx = min(idx, (uint32_t)__shfl_xor((int)idx, s));
        if (lane == 0) si[wave] = idx;
        __syncthreads();
        for (int w = 0; w < NW; w++) idx = min(idx, si[w]);
        if (tid == 0) out->m = m, out->idx = idx, out->e = 0.0;
        return;
    }
    if (m == -INFINITY) {
        if (tid == 0) out->m = m, out->e = -kInfE, out->sum = 0;
        return;
    }
    const double e = draw_e(m, d.c);
    const DrawUnit unit(d.c, e, m);
    float low = draw_low(m, d);
    // below this nothing survives min-p, whatever the row's maximum
    if (d.min_p > 0.0f) {
        const float f = (float)((double)m + d.T * log((double)d.min_p));
        low = fmaxf(low, f - fabsf(f) * 2.4e-7f);  // NaN beside an infinite m: low stays
    }
    if (d.cuts) {
        auto add = [&](int down, uint64_t w) { atomicAdd((unsigned long long *)&hist[down >> kBinShift], (unsigned long long)(w | 1ull << 50)); };
        if (unit.sharp) {
#pragma unroll
            for (int x = 0; x < View::N; x++)
                if (v[x] >= low) add(kSharpDown, v[x] == m ? 1ull << (kCutBits - 1) : 0);
        } else {  // every lane weighs, what is below `low` goes nowhere
#pragma unroll
            for (int x = 0; x < View::N; x++) {
                if (x >= View::N - View::V && view.off == 0) continue;
                double r;
                const int k = unit.steps(v[x], r);
                const uint64_t w = draw_value(k, r, kCutBits, tab);
                if (v[x] >= low) add(-k, w);
            }
        }
        __syncthreads();
        const size_t at = (row * P + p) * kBins;
        for (int b = tid; b < kBins; b += NT) W.hist[at + b] = hist[b];
        if (tid == 0) out->m = m, out->e = e;
    } else {
        // a wave's part is a group, if the row starts at a border
        static_assert(kPiece / NW == kGroup);
        uint64_t s = 0;
        if (unit.sharp) {
#pragma unroll
            for (int x = 0; x < View::N; x++) s += v[x] == m ? 1ull << (kPlainBits - 1) : 0;
        } else {  // every lane weighs, what lies below `low` for nothing
#pragma unroll
            for (int x = 0; x < View::N; x++) {
                if (x >= View::N - View::V && view.off == 0) continue;  // nothing there
                double r;
                const int k = unit.steps(v[x], r);
                const uint64_t w = draw_value(k, r, kPlainBits, tab);
                s += v[x] >= low ? w : 0;
            }
        }
        s = wave_scan(s);
        if (lane == 63) group[wave] = s;
        __syncthreads();
        if (tid < kGroups) out->group[tid] = group[tid];
        if (tid == 0) {
            uint64_t s = 0;
            for (int g = 0; g < kGroups; g++) s += group[g];
            out->m = m, out->e = e, out->sum = s;
        }
    }
}

// ---- the second launch
// A cut of the row's order: kept are keys above `key`, and of its own tokens
// those up to index `last`.
struct DrawCut {
    uint32_t key, last;
    __device__ bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= last); }
};

constexpr int kSorted = kPickThreads;  // tokens put in order each against all others: 256 comparisons a lane at most
constexpr int kWhole = 1024;  // tokens listed down from the maximum, for a second cut among them
constexpr int kFew = 8;  // pieces whose histograms and tokens are held at once (n <= 65536)
// Eight bins a lane, with a gap behind each eight against bank conflicts.
__device__ __forceinline__ int bin_at(int b) { return b + (b >> 3); }
constexpr int kBinRoom = kBins + kBins / 8;

// A piece without its groups.
struct DrawHead {
    float m;
    uint32_t idx;
    double e;
    uint64_t sum;
};
struct __align__(16) PickShared {
    double tab[kSteps];
    uint64_t hist[kFew * kBins];   // of the row's pieces, where they are few
    DrawHead piece[kMaxPieces];
    double scale[kMaxPieces];      // a piece's unit in the row's
    int shift[kMaxPieces];         // its first bin among the row's
    uint64_t kept[kMaxPieces];     // its kept sum, in its unit
    double sum[kBinRoom];          // the row's bins, in the row's unit
    uint32_t cnt[kBinRoom];
    uint64_t sub_sum[kBinRoom];    // of a key range's parts
    uint32_t sub_cnt[kBinRoom];
    union {
        struct {
            uint32_t list_key[kListRoom], list_idx[kListRoom];  // tokens of one bin
            uint64_t order[kSorted], weight[kSorted];
            uint32_t entry[kSorted], by_idx[kSorted];
        };
        float tok[kPiece + kPiece / 8 + 16];  // at last the draw's piece
    };
    uint32_t list_n;
    int todo[kMaxPieces], ntodo;   // pieces that have tokens in a bin
    double before_d;
    uint64_t before_u, wave_total[kPickThreads / 64];
    uint32_t at, ties;
    DrawCut cut;
};

// In wave 0: the first of 512 parts (eight a lane) at which `before` and what
// has gone by reach the goal, or the last part that holds anything.
template <typename T>
__device__ __forceinline__ int first_part(const T (&own)[8], const bool (&some)[8], T before, T goal, T &gone) {
    T s = own[0];
    bool any = some[0];
#pragma unroll
    for (int j = 1; j < 8; j++) s += own[j], any = any || some[j];
    const T run = before + wave_scan(s);
    const uint64_t anys = __ballot(any), hits = __ballot(any && run >= goal);
    if (anys == 0) return -1;
    const int lane = hits ? __ffsll((long long)hits) - 1 : 63 - __clzll((long long)anys);
    T b = run - s;
    int last = 0;
    bool done = false;
    gone = b;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (!done && some[j]) last = j, gone = b;
        done = done || (some[j] && b + own[j] >= goal);
        b += own[j];
    }
    gone = lane_of(gone, lane);
    return (hits ? 0 : kBins) + 8 * lane + __builtin_amdgcn_readlane(last, lane);
}

template <bool F16>
__global__ __launch_bounds__(kPickThreads) void k_draw_pick(const void *__restrict__ logits, int n, int P,
                                                            const float *__restrict__ filter,
                                                            const float *__restrict__ rnd, uint32_t *__restrict__ token,
                                                            float *__restrict__ logp, DrawWork W) {
    constexpr int NT = kPickThreads, NW = NT / 64;
    using View = PieceView<F16, NT>;
    __shared__ PickShared S;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x, base = row * n;
    const uint64_t *hist = W.hist + row * P * kBins;
    // read ahead of the settings: rows without cuts leave them unused
    uint4 ahead[kFew * kBins / 2 / NT];
    if (P <= kFew) {
#pragma unroll
        for (int x = 0; x < kFew * kBins / 2 / NT; x++)
            if (tid + NT * x < P * kBins / 2) ahead[x] = ((const uint4 *)hist)[tid + NT * x];
    }
    DrawHead mine_p{-INFINITY, 0, -kInfE, 0};
    if (tid < P) {
        const DrawPiece &q = W.piece[row * P + tid];
        mine_p = DrawHead{q.m, q.idx, q.e, q.sum};
    }
    const DrawRow d = draw_row(filter + 4 * row, n);
    const float u = rnd[row];
    if (d.cuts && P <= kFew) {
#pragma unroll
        for (int x = 0; x < kFew * kBins / 2 / NT; x++) {
            const bool in = tid + NT * x < P * kBins / 2;
            ((uint4 *)S.hist)[tid + NT * x] = in ? ahead[x] : make_uint4(0, 0, 0, 0);
        }
    }
    if (!d.greedy) draw_table<NT>(S.tab);
    if (tid < kMaxPieces) S.piece[tid] = mine_p;
    __syncthreads();
    float m = -INFINITY;
    double e = -kInfE;
    uint32_t first = 0xFFFFFFFFu;
    for (int p0 = 0; p0 < P; p0 += 8) {
#pragma unroll
        for (int x = 0; x < 8; x++) {
            const DrawHead &q = S.piece[p0 + x];
            if (q.m > m) m = q.m, first = q.idx;
            e = fmax(e, q.e);
        }
    }
    if (m == -INFINITY || d.greedy) {
        if (tid == 0) {
            token[row] = m == -INFINITY ? 0xFFFFFFFFu : first;
            if (logp) logp[row] = m == -INFINITY ? -INFINITY : 0.0f;
        }
        return;
    }
    if (tid < kMaxPieces) {
        const int o = (int)fmin((e - mine_p.e) * (1.0 / kSteps), 4000.0);  // octaves below the row's
        S.scale[tid] = o < 1000 ? ldexp(1.0, -o) : 0.0;
        S.shift[tid] = mine_p.m > -INFINITY ? min(8 * o, kBins) : kBins;
        S.kept[tid] = d.cuts ? 0 : mine_p.sum;
    }
    __syncthreads();
    const DrawUnit unit(d.c, e, m);
    const float low = draw_low(m, d);
    const double uu = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    // ln of the probability of l among kept weights of this sum in the row's
    // unit: total 2^(E - bits), the maximum lies `below` octaves under E
    auto log_p = [&](float l, double total, int bits) {
        double below = 1.0;
        if (!unit.sharp) {
            double r;
            below = -(double)unit.steps(m, r);
            below = (below - r) / kSteps;
        }
        return (float)((l == m ? 0.0 : ((double)l - (double)m) / d.T) - (log(ldexp(total, -bits)) + below * 0.69314718055994530942));
    };
    const double inv_c = d.T * (0.69314718055994530942 / kSteps);
    DrawCut cut{0, 0xFFFFFFFFu};
    int cbin = kBins;  // the cut's bin; kBins: no cut
    if (d.cuts) {
        auto piece_bin = [&](int p, int b) { return P <= kFew ? S.hist[p * kBins + b] : hist[p * kBins + b]; };
        for (int bin = tid; bin < kBins; bin += NT) {
            double s = 0.0;
            uint32_t c = 0;
            for (int p0 = 0; p0 < P; p0 += 8) {
                uint64_t h[8];
                if (P <= kFew) {
#pragma unroll
                    for (int x = 0; x < 8; x++) h[x] = S.hist[x * kBins + max(bin - S.shift[x], 0)];
                } else {
#pragma unroll
                    for (int x = 0; x < 8; x++) h[x] = hist[min(p0 + x, P - 1) * kBins + max(bin - S.shift[p0 + x], 0)];
                }
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const uint64_t in = bin >= S.shift[p0 + x] ? h[x] : 0;  // past the last piece the shift is kBins
                    s += (double)(in & kSumMask) * S.scale[p0 + x];
                    c += (uint32_t)(in >> 50);
                }
            }
            S.sum[bin_at(bin)] = s;
            S.cnt[bin_at(bin)] = c;
        }
        if (d.min_p > 0.0f) {  // the smallest float whose weight is at least min_p
            const double lim = m == INFINITY ? INFINITY : (double)m + d.T * log((double)d.min_p);
            float f = (float)lim;
            if ((double)f < lim) f = lg_unkey(lg_key(f + 0.0f) + 1);
            f = fminf(f + 0.0f, m);
            if (f >= low) {
                double r;
                cut.key = lg_key(f);
                cbin = (unit.sharp ? kSharpDown : -unit.steps(f, r)) >> kBinShift;
            }
        }
        // Stage 0: top-k (min-p has set its key already); stage 1: top-p of what
        // that leaves.  Each finds the goal's bin, narrows its keys to one by
        // passes over the bin's tokens (kNarrow), finds the last of that key's
        // tokens if some have to go (kTies), and sums up what the pieces keep
        // (kKeep).
        enum { kNext, kNarrow, kTies, kKeep, kAll };
        int mode = kNext, stage = -1, bin = 0, sh = 0;
        uint32_t klo = 0, khi = 0, top_key = 0, cnt = 0, ties = 0, count = 0, ilo = 0, ihi = 0, step = 0;
        uint64_t want = 0, before = 0;
        double row_goal = 0.0;  // kAll: top-p's of the whole row
        bool limited = false;
        DrawCut lim = cut;
        // a thread's place among the list's tokens that are in, and (upper half) by index
        auto sort = [&](bool in, uint32_t key, uint32_t idx, uint32_t have) {
            S.order[tid] = in ? (uint64_t)key << 32 | (uint32_t)~idx : 0;
            __syncthreads();
#pragma unroll
            for (int x0 = 0; x0 < kSorted; x0 += 64) {
                if (x0 >= (int)have) break;
                const uint64_t own = S.order[x0 + lane];
                uint32_t c = 0, by_idx = 0;
                for (int y0 = 0; y0 < (int)have; y0 += 8 * NW) {
#pragma unroll
                    for (int y = 0; y < 8; y++) {
                        const uint64_t o = S.order[y0 + 8 * wave + y];
                        c += o > own;
                        by_idx += (uint32_t)o > (uint32_t)own;
                    }
                }
                atomicAdd(&S.sub_cnt[x0 + lane], c | by_idx << 16);
            }
            __syncthreads();
            return S.sub_cnt[tid];
        };
        auto block_scan = [&](uint64_t v, uint64_t &all) {
            const uint64_t pre = wave_scan(v);
            if (lane == 63) S.wave_total[wave] = pre;
            __syncthreads();
            uint64_t b = pre;
            all = 0;
#pragma unroll
            for (int y = 0; y < NW; y++) {
                if (y < wave) b += S.wave_total[y];
                all += S.wave_total[y];
            }
            return b;
        };
        bool listed = false;  // the list holds all tokens with keys from list_lo to list_hi
        uint32_t list_lo = 0, list_hi = 0;
        bool above = false;   // list what is above the bin too
        bool fresh = true;    // before the row's first cut
        for (;;) {
            const bool by_count = stage == 0;
            if (mode == kNext) {
                if (++stage == 2) break;
                const bool counts = stage == 0;
                if (counts ? d.top_k == 0 && cbin == kBins : d.top_p >= 1.0f) continue;
                bool select = !counts || d.top_k;
                double before_d = 0.0, goal = d.top_k;
                __syncthreads();
                if (select) {
                    if (wave == 0) {
                        double own[8], total = 0.0;
                        bool some[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const int b = 8 * lane + j;
                            own[j] = counts ? (double)S.cnt[bin_at(b)] : b < cbin ? S.sum[bin_at(b)] : 0.0;
                            some[j] = own[j] > 0.0;
                            total += own[j];
                        }
                        if (!counts) {  // of all that the cut so far leaves
                            if (cbin < kBins) total = (double)S.kept[lane] * S.scale[lane] + (double)S.kept[lane + 64] * S.scale[lane + 64];
                            goal = (double)d.top_p * lane_of(wave_scan(total), 63);
                        }
                        double gone = 0.0;
                        int at = first_part(own, some, 0.0, goal, gone);
                        if (at < 0 || at >= kBins) {  // not reached
                            at = kBins;
                            gone = 0.0;
#pragma unroll
                            for (int j = 0; j < 8; j++) gone += own[j];
                            gone = lane_of(wave_scan(gone), 63);
                        }
                        if (lane == 0) S.at = at, S.before_d = gone, S.before_u = __builtin_bit_cast(uint64_t, goal);
                    }
                    __syncthreads();
                    bin = S.at;
                    before_d = S.before_d;
                    goal = __builtin_bit_cast(double, S.before_u);
                    if (!counts && bin == kBins) bin = cbin;  // not above the cut's bin: in it
                    // a count that ends below the cut, or among tokens without weight, cuts nothing
                    select = bin <= cbin && bin < kDeepBin;
                }
                if (!select) {
                    if (cbin == kBins) continue;
                    bin = cbin;
                }
                // the bin's keys: its borders in l, exactly, from the floats around them
                uint32_t low_key = lg_key(m);
                top_key = low_key;
                if (!unit.sharp) {
                    uint32_t at[2];
#pragma unroll
                    for (int side = 0; side < 2; side++) {  // the first key of this bin, of the bin above
                        const int steps = (bin + 1 - side) << kBinShift;
                        float f = (float)((e - steps + 0.5) * inv_c);
                        f = f == f ? fminf(fmaxf(f, kLeast), -kLeast) : 0.0f;
                        const uint32_t k0 = lg_key(f + 0.0f) - 32;
                        const float l = lg_unkey(k0 + lane);
                        double r;
                        const uint64_t yes = __ballot(l > m || (l >= low && -unit.steps(l, r) < steps));
                        at[side] = k0 + (yes ? __ffsll((long long)yes) - 1 : 64);
                    }
                    low_key = at[0];
                    top_key = max(at[0], min(at[1] - 1, top_key));
                }
                cnt = S.cnt[bin_at(bin)];
                if (select) {
                    limited = bin == cbin;
                    lim = cut;
                    klo = limited ? max(low_key, lim.key) : low_key;
                    khi = max(top_key, klo);
                    // the goal inside the bin: a count, or weights kInBits below the octave that holds the bin's top
                    const double left = fmax(goal - before_d, 0.0);
                    want = counts ? (uint64_t)left : (uint64_t)ceil(ldexp(left, (bin >> 3) + kInBits - kCutBits));
                    before = 0;
                    mode = kNarrow;
                    above = counts && d.top_p < 1.0f && before_d + cnt <= kWhole;
                } else {
                    mode = kKeep;
                }
                if (fresh) {  // few tokens down to the bin: they settle the row
                    fresh = false;
                    uint32_t c = 0;
#pragma unroll
                    for (int j = 0; j < 8; j++) c += 8 * lane + j <= bin ? S.cnt[9 * lane + j] : 0;
                    if (__builtin_amdgcn_readlane((int)wave_scan32(c), 63) <= kSorted) {
                        if (mode == kKeep) klo = cut.key, khi = max(top_key, klo);
                        mode = kAll;
                        above = true;
                        row_goal = goal;
                    }
                }
                if (mode != kKeep) continue;
            }
            if (mode == kKeep) {  // whole bins; the cut's own token by token
                for (int p = wave; p < P; p += NW) {
                    uint64_t s = 0;
                    const int top = cbin - S.shift[p];
#pragma unroll
                    for (int x = 0; x < kBins; x += 64) s += x + lane < top ? piece_bin(p, x + lane) & kSumMask : 0;
                    s = wave_scan(s);
                    if (lane == 63) S.kept[p] = s;
                }
                klo = cut.key;
                khi = max(top_key, klo);
            } else if (mode == kNarrow) {
                sh = 0;
                while ((khi - klo) >> sh >= kBins) sh++;
            } else if (mode == kTies) {
                step = (ihi - ilo) / kBins + 1;
            }
            // a pass over the bin's tokens with keys in [klo, khi]: from the list,
            // into which a bin of at most kList tokens goes whole, a larger one
            // half a piece at a time
            const bool held = listed && klo >= list_lo && khi <= list_hi;
            __syncthreads();
            if (mode != kKeep)
                for (int b = tid; b < kBinRoom; b += NT) S.sub_sum[b] = 0, S.sub_cnt[b] = 0;
            if (tid == 0) S.ntodo = 0, S.list_n = held ? S.list_n : 0, S.before_u = 0;
            __syncthreads();
            int chunks = 1;
            bool direct = false;
            if (!held) {
                list_lo = klo;
                list_hi = above ? lg_key(m) : khi;
                if (tid < P) {
                    const int b = bin - S.shift[tid];
                    if (above ? lg_key(mine_p.m) >= klo : b >= 0 && piece_bin(tid, b)) S.todo[atomicAdd(&S.ntodo, 1)] = tid;
                }
                above = false;
                __syncthreads();
                listed = cnt <= kList;
                if (!listed)
                    chunks = 2 * S.ntodo;  // kListRoom tokens each at most
            }
            const DrawUnit in_unit(d.c, e - (double)kSteps * (bin >> 3), m);
            for (int ch = 0; ch < chunks; ch++) {
                if (!held) {
                    const int t0 = listed ? 0 : ch >> 1, t1 = listed ? S.ntodo : t0 + 1;
                    // half a piece is each thread's first or last 16 tokens, these with what lies behind the last border
                    constexpr int PT = kPiece / NT;
                    static_assert(PT == 32);
                    const uint32_t half = listed ? ~0u : ch & 1 ? 0xFFFFu : 0xFFFF0000u;
                    const float llo = lg_unkey(list_lo), lhi = lg_unkey(list_hi);
                    if (ch) {
                        __syncthreads();
                        if (tid == 0) S.list_n = 0;
                        __syncthreads();
                    }
                    constexpr int AT = 4;  // pieces in flight
                    for (int t = t0; t < t1; t += AT) {
                        uint4 raw[AT][View::NV];
#pragma unroll
                        for (int a = 0; a < AT; a++)
                            if (t + a < t1) View(logits, base, S.todo[t + a], n).load(raw[a]);
                        uint32_t hits[AT], more[AT], own = 0;
#pragma unroll
                        for (int a = 0; a < AT; a++) {
                            hits[a] = more[a] = 0;
                            if (t + a >= t1) continue;
                            const View view(logits, base, S.todo[t + a], n);
                            hits[a] = View::template within<0, PT>(raw[a], llo, lhi) & half;
                            if (view.off && (half & 1)) more[a] = View::template within<PT, View::N>(raw[a], llo, lhi);
                            if (!view.whole) view.own(hits[a], more[a]);
                            own += __popc(hits[a]) + __popc(more[a]);
                        }
                        const uint32_t end = wave_scan32(own), all = __builtin_amdgcn_readlane((int)end, 63);
                        if (all == 0) continue;
                        uint32_t at = 0;
                        if (lane == 0) at = atomicAdd(&S.list_n, all);
                        at = __builtin_amdgcn_readfirstlane((int)at) + end - own;
#pragma unroll
                        for (int a = 0; a < AT; a++) {
                            if (t + a >= t1) continue;
                            const View view(logits, base, S.todo[t + a], n);
                            for (uint32_t h = hits[a]; h;) {
                                const int z = __clz((int)h);
                                h &= ~(0x80000000u >> z);
                                if (at < kListRoom) S.list_idx[at++] = view.token(z);
                            }
                            for (uint32_t h = more[a]; h;) {
                                const int z = __clz((int)h);
                                h &= ~(0x80000000u >> z);
                                if (at < kListRoom) S.list_idx[at++] = view.token(z + PT - (32 - View::V));
                            }
                        }
                    }
                    __syncthreads();
                }
                const uint32_t have = min(S.list_n, (uint32_t)kListRoom);
                if (!held)  // their keys, all loads at once; below a thread meets its own
                    for (uint32_t x = tid; x < have; x += NT) S.list_key[x] = lg_key(lg_value<F16>(logits, base + S.list_idx[x]));
                if (mode == kAll) {
                    // each token against all others, in the row's order and by index: both cuts and the draw
                    const bool in = tid < (int)have;
                    const uint32_t k = in ? S.list_key[tid] : 0, i = in ? S.list_idx[tid] : 0;
                    int down;
                    const uint64_t w = in ? draw_weight(unit, lg_unkey(k), kPlainBits, S.tab, down) : 0;
                    const uint32_t at = sort(in, k, i, have);
                    if (in) {
                        S.weight[at & 0xFFFF] = w;
                        S.entry[at & 0xFFFF] = at >> 16;
                        S.by_idx[at >> 16] = tid;
                    }
                    __syncthreads();
                    // a thread has a place in the row's order ...
                    uint64_t all, total;
                    const uint64_t mine = in && (!d.top_k || tid < (int)d.top_k) ? S.weight[tid] : 0;
                    const uint64_t ahead = block_scan(mine, all) - mine;
                    const double lim_p = stage == 1 ? ldexp(row_goal, kPlainBits - kCutBits) : (double)d.top_p * (double)all;
                    if (in) S.order[S.entry[tid]] = d.top_p >= 1.0f || tid == 0 || (double)ahead < lim_p ? mine : 0;
                    __syncthreads();
                    // ... and now one by index
                    const uint64_t kept = in ? S.order[tid] : 0, run = block_scan(kept, total);
                    const uint64_t goal = min((uint64_t)(uu * (double)total), total - 1);
                    if (kept && run - kept <= goal && goal < run) {
                        const uint32_t x = S.by_idx[tid];
                        token[row] = S.list_idx[x];
                        if (logp) logp[row] = log_p(lg_unkey(S.list_key[x]), (double)total, kPlainBits);
                    }
                    return;
                }
                if (mode == kNarrow && listed && have <= kSorted) {  // the cut without more passes
                    const uint32_t k = S.list_key[tid], i = S.list_idx[tid];
                    const bool in = tid < (int)have && k >= klo && k <= khi && !(limited && !lim.keeps(k, i));
                    int down;
                    const uint64_t w = !in ? 0 : by_count ? 1 : draw_weight(in_unit, lg_unkey(k), kInBits, S.tab, down);
                    S.weight[tid] = 0;
                    if (tid == 0) S.cut = DrawCut{klo, 0xFFFFFFFFu};
                    const uint32_t at = sort(in, k, i, have) & 0xFFFF;
                    if (in) S.weight[at] = w, S.entry[at] = tid;
                    __syncthreads();
                    uint64_t all;
                    const uint64_t mine = S.weight[tid], run = block_scan(mine, all);
                    const uint64_t to = min(want > before ? want - before : 1, all);
                    if (mine && run - mine < to && to <= run) S.cut = DrawCut{S.list_key[S.entry[tid]], S.list_idx[S.entry[tid]]};
                    __syncthreads();
                    cut = S.cut;
                    cbin = bin;
                    cnt = S.cnt[bin_at(bin)];
                    mode = kKeep;
                    direct = true;
                    break;
                }
                for (uint32_t x = tid; x < have; x += NT) {
                    const uint32_t k = S.list_key[x], i = S.list_idx[x];
                    if (k < klo || k > khi) continue;
                    if (mode == kTies) {
                        if (i >= ilo && i <= ihi) atomicAdd(&S.sub_cnt[bin_at((i - ilo) / step)], 1u);
                        continue;
                    }
                    const bool keep = mode == kKeep;
                    if (keep ? !cut.keeps(k, i) : limited && !lim.keeps(k, i)) continue;
                    const int part = bin_at((int)((khi - k) >> sh)), p = i / kPiece;
                    if (!keep) atomicAdd(&S.sub_cnt[part], 1u);
                    if (!keep && by_count) continue;
                    int down;
                    const DrawUnit to = keep ? DrawUnit(d.c, S.piece[p].e, S.piece[p].m) : in_unit;
                    const uint64_t w = draw_weight(to, lg_unkey(k), keep ? kCutBits : kInBits, S.tab, down);
                    atomicAdd((unsigned long long *)(keep ? &S.kept[p] : &S.sub_sum[part]), (unsigned long long)w);
                }
            }
            if (direct) continue;
            __syncthreads();
            if (mode == kKeep) {
                mode = kNext;
            } else if (mode == kNarrow) {
                if (wave == 0) {
                    uint64_t own[8], gone = before;
                    uint32_t c[8];
                    bool some[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        c[j] = S.sub_cnt[9 * lane + j];
                        own[j] = by_count ? c[j] : S.sub_sum[9 * lane + j];
                        some[j] = c[j] != 0;
                    }
                    const int at = first_part(own, some, before, want, gone);
                    if (lane == 0) S.at = at < 0 ? 0 : at & (kBins - 1), S.before_u = gone, S.ties = at < 0 ? 0 : S.sub_cnt[bin_at(at & (kBins - 1))];
                }
                __syncthreads();
                before = S.before_u;
                cnt = ties = S.ties;
                khi -= S.at << sh;
                if (sh) {
                    klo = max(klo, khi - ((1u << sh) - 1u));
                } else {
                    // one key is left; its tokens weigh the same, so a division tells how many stay
                    const uint64_t left = want > before ? want - before : 0;
                    const uint64_t w = by_count ? 1 : (uint64_t)rint((double)S.sub_sum[bin_at(S.at)] / (double)max(ties, 1u));
                    count = w ? (uint32_t)fmin(ceil((double)left / (double)w), (double)n) : 1;
                    if (count * w < left) count++;  // the division's rounding
                    else if (count && (count - 1) * w >= left) count--;
                    count = max(count, 1u);
                    klo = khi;
                    cut = DrawCut{khi, limited && lim.key == khi ? lim.last : 0xFFFFFFFFu};
                    cbin = bin;
                    cnt = S.cnt[bin_at(bin)];
                    mode = count < ties ? kTies : kKeep;
                    ilo = 0;
                    ihi = n - 1;
                }
            } else {
                if (tid == 0) {
                    uint32_t b = 0, got = 0;
                    while (b < kBins - 1 && got + S.sub_cnt[bin_at(b)] < count) got += S.sub_cnt[bin_at(b++)];
                    S.at = b;
                    S.ties = got;
                }
                __syncthreads();
                count -= S.ties;
                ilo += S.at * step;
                ihi = min(ihi, ilo + step - 1);
                if (ilo >= ihi) {
                    cut.last = ilo;
                    mode = kKeep;
                }
            }
        }
        if (cbin == kBins) {  // nothing was cut
            for (int p = wave; p < P; p += NW) {
                uint64_t s = 0;
                if (S.shift[p] < kBins || S.scale[p] > 0.0)
#pragma unroll
                    for (int x = 0; x < kBins; x += 64) s += piece_bin(p, x + lane) & kSumMask;
                s = wave_scan(s);
                if (lane == 63) S.kept[p] = s;
            }
            __syncthreads();
        }
    }
    // the draw's piece: every wave goes through them, the same way
    const int bits = d.cuts ? kCutBits : kPlainBits;
    double total = 0.0;
    for (int p0 = 0; p0 < P; p0 += 8) {
#pragma unroll
        for (int x = 0; x < 8; x++) total += (double)S.kept[p0 + x] * S.scale[p0 + x];
    }
    const double target = uu * total;
    double run = 0.0, gone = 0.0;
    int piece = -1;
    for (int p0 = 0; p0 < P; p0 += 8) {
#pragma unroll
        for (int x = 0; x < 8; x++) {
            const double s = (double)S.kept[p0 + x] * S.scale[p0 + x];
            if (s > 0.0 && run <= target) piece = p0 + x, gone = run;
            run += s;
        }
    }
    const DrawUnit pu(d.c, S.piece[piece].e, S.piece[piece].m);
    const float plow = draw_low(S.piece[piece].m, d);
    uint64_t goal = (uint64_t)fmax((target - gone) / S.scale[piece], 0.0);
    if (goal >= S.kept[piece]) goal = S.kept[piece] - 1;
    // The token.  A plain row's piece has sums by groups of 1024 tokens (where
    // the row starts at a 16-byte border), and threads take four tokens of the
    // group each.  Otherwise they take 32 of the piece through LDS and weigh
    // those that are kept.
    const bool grouped = !d.cuts && base % View::V == 0;
    auto weight = [&](float l) {
        int down;
        return draw_weight(pu, l, bits, S.tab, down);
    };
    auto find = [&](uint64_t mine, uint64_t b, auto walk) {  // walk(up to): the token of a thread's own at which its sum passes it
        const uint64_t pre = wave_scan(mine);
        if (lane == 63) S.wave_total[wave] = pre;
        __syncthreads();
        b += pre - mine;
#pragma unroll
        for (int y = 0; y < NW; y++)
            if (y < wave) b += S.wave_total[y];
        if (goal < b || goal >= b + mine) return;
        float l;
        token[row] = walk(goal - b, l);
        if (logp) logp[row] = log_p(l, total, bits);
    };
    if (grouped) {
        constexpr int V = 4;
        static_assert(kGroup == NT * V);
        const uint64_t *group = W.piece[row * P + piece].group;
        uint64_t gs[kGroups], b = 0, run_g = 0;
        int g = 0;
#pragma unroll
        for (int x = 0; x < kGroups; x++) gs[x] = group[x];
#pragma unroll
        for (int x = 0; x < kGroups; x++) {
            if (run_g <= goal) g = x, b = run_g;
            run_g += gs[x];
        }
        const int i0 = piece * kPiece + g * kGroup + tid * V;
        float v[V];
        uint64_t w[V], mine = 0;
#pragma unroll
        for (int x = 0; x < V; x++) v[x] = i0 + x < n ? lg_value<F16>(logits, base + i0 + x) : -INFINITY;
#pragma unroll
        for (int x = 0; x < V; x++) w[x] = v[x] >= plow ? weight(v[x]) : 0, mine += w[x];
        find(mine, b, [&](uint64_t left, float &l) {
            int hit = V - 1;
            l = v[V - 1];
            uint64_t up = mine;
#pragma unroll
            for (int x = V - 1; x >= 0; x--) {
                if (left < up && w[x]) hit = x, l = v[x];
                up -= w[x];
            }
            return (uint32_t)(i0 + hit);
        });
    } else {
        const float lc = cbin == kBins ? plow : lg_unkey(cut.key);  // kept: above it, or at it up to index cut.last
        const View view(logits, base, piece, n);
        uint4 raw[View::NV];
        view.load(raw);
        // position j of the view (token view.first + j) at j + 4 (j / 32): 16-byte writes and reads, all banks
#pragma unroll
        for (int x = 0; x < View::N; x += 4) {
            const int j = View::vec(x / View::V) * View::V + x % View::V;
            float4 l;
            l.x = raw_value<F16>(raw[x / View::V], x % View::V);
            l.y = raw_value<F16>(raw[x / View::V], x % View::V + 1);
            l.z = raw_value<F16>(raw[x / View::V], x % View::V + 2);
            l.w = raw_value<F16>(raw[x / View::V], x % View::V + 3);
            if (j < kPiece + view.off) *(float4 *)&S.tok[j + 4 * (j >> 5)] = l;
        }
        __syncthreads();
        constexpr int PT = kPiece / NT;
        const uint32_t i0 = view.first + tid * PT;
        const float4 *own4 = (const float4 *)(S.tok + (PT + 4) * tid);
        const float *own = (const float *)own4;
        uint32_t keep = 0, more = 0;
#pragma unroll
        for (int x = 0; x < PT; x += 4) {
            const float4 q = own4[x / 4];
            const float l[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int y = 0; y < 4; y++) keep |= l[y] > lc || (l[y] == lc && i0 + x + y <= cut.last) ? 1u << (x + y) : 0;
        }
        // the piece's own only
        const int skip = tid ? 0 : view.off, end = view.off + view.len - tid * PT;
        keep = end <= 0 ? 0 : keep >> skip << skip & (end < PT ? (1u << end) - 1 : ~0u);
        // the last thread has the tokens behind the last border too
        if (view.off && tid == NT - 1)
            for (int x = 0; x < end - PT; x++) {
                const float l = own[PT + 4 + x];
                more |= l > lc || (l == lc && i0 + PT + x <= cut.last) ? 1u << x : 0;
            }
        uint64_t mine = 0;
        for (uint32_t k = keep; k; k &= k - 1) mine += weight(own[__ffs((int)k) - 1]);
        for (uint32_t k = more; k; k &= k - 1) mine += weight(own[PT + 3 + __ffs((int)k)]);
        find(mine, 0, [&](uint64_t left, float &l) {
            uint64_t up = 0;
            int x = 0;
            for (uint32_t k = keep, z = 0; z < 2; k = more, z++) {
                for (; k && left >= up; k &= k - 1) {
                    x = __ffs((int)k) - 1 + (z ? PT : 0);
                    l = own[x + 4 * (x / PT)];
                    up += weight(l);
                }
            }
            return i0 + x;
        });
    }
}

static int draw_pieces(uint64_t n) { return (int)((n + kPiece - 1) / kPiece); }

// ------------------------------------------------- log-probabilities
// logp = (l[tok] - m) - ln(sum exp(l - m)); rank = tokens ahead of tok in the
// row's order (larger logit, or equal and a lower index).
struct LpPart {
    float m, s;
    uint32_t ahead, pad;
};
constexpr int kLpThreads = 256;

__device__ __forceinline__ float lp_exp(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }
__device__ __forceinline__ void lp_join(LpPart &a, const LpPart &b) {
    const float m = fmaxf(a.m, b.m);
    a.s = (a.m == m ? a.s : a.s * lp_exp(a.m - m)) + (b.m == m ? b.s : b.s * lp_exp(b.m - m));
    a.m = m;
    a.ahead += b.ahead;
}
// More logits into a running (maximum, sum relative to it).
template <int N>
__device__ __forceinline__ void lp_add(LpPart &a, const float (&v)[N], float thr) {
    float m = a.m;
#pragma unroll
    for (int e = 0; e < N; e++) m = fmaxf(m, v[e]);
#pragma unroll
    for (int e = 0; e < N; e++) a.ahead += !(v[e] <= thr);
    if (m == -INFINITY) return;
    if (m > a.m) {
        a.s *= lp_exp(a.m - m);
        a.m = m;
    }
    if (m < INFINITY) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < N; e++) s += lp_exp(v[e] - m);
        a.s += s;
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) a.s += v[e] == m ? 1.0f : 0.0f;
    }
}

__device__ __forceinline__ void lp_write(const LpPart &a, float lt, float *logp, uint32_t *rank, size_t row) {
    logp[row] = lt == -INFINITY ? -INFINITY : (lt == a.m ? 0.0f : lt - a.m) - logf(a.s);
    if (rank) rank[row] = a.ahead;
}

// A block per (row, piece of 16-byte vectors); with one piece a row, the
// result itself.  Bound by the read: 2048 rows of 65536 fp32 logits take 96 us
// (5.6 TB/s, above the 5.1 of a copy).  Few rows are two short launches, 4.0 +
// 2.6 us for 8 rows; one exp2 a token, the maximum carried per thread.
template <bool F16>
__global__ __launch_bounds__(kLpThreads) void k_logprob(const void *__restrict__ logits, int n, int P,
                                                        const uint32_t *__restrict__ token, float *__restrict__ logp,
                                                        uint32_t *__restrict__ rank, LpPart *__restrict__ part) {
    constexpr int V = F16 ? 8 : 4, SZ = F16 ? 2 : 4, UN = 4;
    __shared__ LpPart sh[kLpThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x / P, base = row * n;
    const int p = blockIdx.x % P;
    const uint32_t tok = token[row];
    if (tok >= (uint32_t)n) {
        if (p == 0 && tid == 0) {
            logp[row] = 0.0f;
            if (rank) rank[row] = 0;
        }
        return;
    }
    const float lt = lg_value<F16>(logits, base + tok);
    // ahead of tok: from lt on at lower indexes, above lt at higher ones; `from`
    // is the number below lt (NaN, which everything passes, below -inf)
    const float from = lt == -INFINITY ? NAN : lg_unkey(lg_key(lt) - (lt == 0.0f ? 2 : 1));  // no -0 here
    // whole vectors lie between the row's first and last 16-byte border
    const int head = min(n, (int)((V - base % V) % V)), nv = (n - head) / V, tail0 = head + nv * V;
    const int per = (nv + P - 1) / P, v0 = min(nv, p * per), v1 = min(nv, v0 + per);
    LpPart a{-INFINITY, 0.0f, 0, 0};
    const uint4 *q = (const uint4 *)((const char *)logits + (base + head) * SZ);
    for (int v = v0 + tid; v < v1; v += kLpThreads * UN) {
        uint4 w[UN];
#pragma unroll
        for (int j = 0; j < UN; j++)
            if (v + kLpThreads * j < v1) w[j] = q[v + kLpThreads * j];
#pragma unroll
        for (int j = 0; j < UN; j++) {
            const int vi = v + kLpThreads * j;
            if (vi >= v1) break;
            float x[V];
            lg_unpack<F16>(w[j], x);
            const int i = head + vi * V;
            lp_add(a, x, i + V <= (int)tok ? from : lt);
            if (i <= (int)tok && i + V > (int)tok) {  // tok's own vector: equal logits before it
#pragma unroll
                for (int e = 0; e < V; e++) a.ahead += i + e < (int)tok && x[e] == lt;
            }
        }
    }
    if (p == 0) {
        const int i = tid < head ? tid : tail0 + tid - head;
        if (i < n && tid < head + n - tail0) {
            const float x[1] = {lg_value<F16>(logits, base + i)};
            lp_add(a, x, i < (int)tok ? from : lt);
        }
    }
    for (int d = 32; d; d >>= 1) {
        const LpPart b{__shfl_xor(a.m, d), __shfl_xor(a.s, d), (uint32_t)__shfl_xor((int)a.ahead, d), 0};
        lp_join(a, b);
    }
    if (lane == 0) sh[wave] = a;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kLpThreads / 64; w++) lp_join(a, sh[w]);
        if (P == 1)
            lp_write(a, lt, logp, rank, row);
        else
            part[row * P + p] = a;
    }
}

template <bool F16>
__global__ __launch_bounds__(64) void k_logprob_join(const void *__restrict__ logits, int n, int P,
                                                     const uint32_t *__restrict__ token, float *__restrict__ logp,
                                                     uint32_t *__restrict__ rank, const LpPart *__restrict__ part) {
    const size_t row = blockIdx.x;
    const uint32_t tok = token[row];
    if (tok >= (uint32_t)n) return;
    const float lt = lg_value<F16>(logits, row * n + tok);
    LpPart a = (int)threadIdx.x < P ? part[row * P + threadIdx.x] : LpPart{-INFINITY, 0.0f, 0, 0};
    for (int d = 32; d; d >>= 1) {
        const LpPart b{__shfl_xor(a.m, d), __shfl_xor(a.s, d), (uint32_t)__shfl_xor((int)a.ahead, d), 0};
        lp_join(a, b);
    }
    if (threadIdx.x == 0) lp_write(a, lt, logp, rank, row);
}

// Pieces of a row: about 1024 blocks in all, at least 4 KB each, at most a wave's lanes.
static int logprob_pieces(uint64_t n, uint64_t rows) {
    return (int)std::max<uint64_t>(1, std::min<uint64_t>({(1024 + rows - 1) / rows, n / 2048, 64}));
}

// ------------------------------------------------------------- launchers
uint64_t logits_work_words(uint64_t n, uint64_t rows) {
    const uint64_t draw = rows * draw_pieces(n) * (sizeof(DrawPiece) + kBins * 8) / 4;
    const uint64_t lp = rows * logprob_pieces(n, rows) * sizeof(LpPart) / 4;
    return std::max(draw, lp);
}

template <bool F16>
static void draw_launch(rsv_ctx *ctx, const void *logits, int n, int P, const float *filter, const float *rnd,
                        uint32_t *token, float *logp, const DrawWork &W, uint64_t rows) {
    hipLaunchKernelGGL((k_draw_scan<F16>), dim3((unsigned)(rows * P)), dim3(kScanThreads), 0, ctx->stream, logits, n, P, filter, W);
    hipLaunchKernelGGL((k_draw_pick<F16>), dim3((unsigned)rows), dim3(kPickThreads), 0, ctx->stream, logits, n, P, filter, rnd,
                       token, logp, W);
}

int launch_draw(rsv_ctx *ctx, const void *logits, int f16, uint32_t *token, uint64_t n, const float *filter,
                const float *rnd, float *logp, float *work, uint64_t rows) {
    const int P = draw_pieces(n);
    DrawWork W;
    W.hist = (uint64_t *)work;
    W.piece = (DrawPiece *)(W.hist + rows * P * kBins);
    if (f16)
        draw_launch<true>(ctx, logits, (int)n, P, filter, rnd, token, logp, W, rows);
    else
        draw_launch<false>(ctx, logits, (int)n, P, filter, rnd, token, logp, W, rows);
    RSV_HIP(hipGetLastError());
    return 0;
}

template <bool F16>
static void logprob_launch(rsv_ctx *ctx, const void *logits, const uint32_t *token, int n, float *logp, uint32_t *rank,
                           LpPart *part, uint64_t rows) {
    const int P = logprob_pieces(n, rows);
    hipLaunchKernelGGL((k_logprob<F16>), dim3((unsigned)(rows * P)), dim3(kLpThreads), 0, ctx->stream, logits, n, P, token, logp, rank, part);
    if (P > 1)
        hipLaunchKernelGGL((k_logprob_join<F16>), dim3((unsigned)rows), dim3(64), 0, ctx->stream, logits, n, P, token, logp, rank, part);
}

int launch_logprobs(rsv_ctx *ctx, const void *logits, int f16, const uint32_t *token, uint64_t n, float *logp,
                    uint32_t *rank, float *work, uint64_t rows) {
    if (f16)
        logprob_launch<true>(ctx, logits, token, (int)n, logp, rank, (LpPart *)work, rows);
    else
        logprob_launch<false>(ctx, logits, token, (int)n, logp, rank, (LpPart *)work, rows);
    RSV_HIP(hipGetLastError());
    return 0;
}

}  // namespace rsv

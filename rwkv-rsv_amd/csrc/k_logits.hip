// What a served step takes from its logits rows: draws from given random
// numbers (rsv_sample_rand_batch) and log-probabilities of given tokens
// (rsv_token_logprobs).
#include <algorithm>
#include <type_traits>

#include "rsv_common.h"

namespace rsv {

constexpr float kLog2e = 1.44269504088896340736f;

// A logit as the row's order sees it: NaN as -inf, -0 as +0.
__device__ __forceinline__ float lg_clean(float l) { return l == l ? l + 0.0f : -INFINITY; }
template <bool F16>
__device__ __forceinline__ float lg_value(const void *p, size_t i) {
    return lg_clean(F16 ? (float)((const _Float16 *)p)[i] : ((const float *)p)[i]);
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
// block per row finds the cut from the histograms, resolves it inside the one
// bin that holds it, takes the draw's piece from the pieces' kept sums and the
// token from that piece alone.  So the row is read once, and then what lies in
// one bin and one piece.
//
// A token's weight is 2^x, x = l log2(e) / T, held as an integer with `bits`
// bits below E, a whole octave above the piece's largest x.  With c = 1024
// log2(e) / T: q = l c rounded to an integer (adding 1.5 2^52 leaves it in the
// sum's low bits, right for |l c| < 2^51), r = l c - q in one rounding, and
//   2^x = 2^(q >> 10) tab[q & 1023] (1 + r ln2/1024 + ...),
// a Taylor polynomial of degree 3 in an argument below 3.4e-4 (6e-16 off).
// Adding 2^52 to the scaled weight leaves the integer in the low bits.  Eight
// 64-bit float operations a token; exp() takes about four times as many.
// Integers add up the same in any order; pieces are put together in 64-bit
// floats in the pieces' order, which depends on n alone.  Bins follow q, so
// they mean the same in every piece.
//
// Tokens 36.5 T and more below a piece's maximum (2^-52) have no weight and
// stand in no bin.  Rows that are only settled by their maximum (+inf, or
// |l c| past 2^50, where different logits are 36 T apart) are `sharp`: tokens
// at the maximum weigh 2^(bits - 1), the others nothing.
constexpr int kPiece = 8192, kDrawThreads = 1024, kPer = kPiece / kDrawThreads;
constexpr int kBins = 512, kSteps = 1024, kBinShift = 7, kMaxPieces = (int)(kLogitsMaxN / kPiece);
constexpr int kSharpDown = kSteps - 1;  // a sharp maximum stands in its first octave's last bin
constexpr int kDeepBin = 50 * 8;  // from here on weights vanish beside the maximum's
constexpr int kPlainBits = 48;    // weights of a row without cuts
constexpr int kCutBits = 37;      // with cuts: a bin packs its sum (8192 2^37 = 2^50) and above it its count
constexpr int kInBits = 40;       // inside a bin, below the bin's octave: up to 2^20 tokens
constexpr uint64_t kSumMask = ((uint64_t)1 << 50) - 1;
constexpr int kList = 4096;       // a bin's tokens held in LDS

struct DrawPiece {
    float m;        // largest logit (-inf: nothing to draw)
    uint32_t idx;   // its lowest token (greedy rows)
    double e;       // 1024 E
    uint64_t sum;   // plain rows
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
__device__ __forceinline__ void draw_table(double *tab) {
    for (int i = threadIdx.x; i < kSteps; i += kDrawThreads) tab[i] = exp2((double)i / kSteps);
}

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// The tokens of a piece that a lane holds, kPer of them, those past the row's
// end as -inf.  `aligned`: rows start at 16-byte borders.
template <bool F16>
__device__ __forceinline__ int piece_token(bool aligned, int e) {
    constexpr int V = F16 ? 8 : 4;
    return aligned ? ((int)threadIdx.x + kDrawThreads * (e / V)) * V + e % V : (int)threadIdx.x + kDrawThreads * e;
}
template <bool F16>
__device__ __forceinline__ void piece_load(const void *logits, size_t base, int i0, int n, bool aligned, float (&v)[kPer]) {
    constexpr int V = F16 ? 8 : 4;
    if (aligned && i0 + kPiece <= n) {
#pragma unroll
        for (int b = 0; b < kPer / V; b++) {
            float w[V];
            const size_t at = base + i0 + (threadIdx.x + kDrawThreads * b) * V;
            lg_unpack<F16>(*(const uint4 *)((const char *)logits + at * (F16 ? 2 : 4)), w);
#pragma unroll
            for (int e = 0; e < V; e++) v[b * V + e] = w[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            const int i = i0 + piece_token<F16>(aligned, e);
            v[e] = i < n ? lg_value<F16>(logits, base + i) : -INFINITY;
        }
    }
}

template <bool F16>
__global__ __launch_bounds__(kDrawThreads) void k_draw_scan(const void *__restrict__ logits, int n, int P, bool aligned,
                                                            const float *__restrict__ filter, DrawWork W) {
    __shared__ double tab[kSteps];
    __shared__ uint64_t hist[kBins];
    __shared__ uint64_t ss[16];
    __shared__ float sm[16];
    __shared__ uint32_t si[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x / P;
    const int p = blockIdx.x % P, i0 = p * kPiece;
    float v[kPer];
    piece_load<F16>(logits, row * n, i0, n, aligned, v);
    const DrawRow d = draw_row(filter + 4 * row, n);
    if (!d.greedy) draw_table(tab);
    if (d.cuts)
        for (int b = tid; b < kBins; b += kDrawThreads) hist[b] = 0;
    float m = v[0];
#pragma unroll
    for (int e = 1; e < kPer; e++) m = fmaxf(m, v[e]);
    for (int s = 32; s; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
    if (lane == 0) sm[wave] = m;
    __syncthreads();
    for (int w = 0; w < 16; w++) m = fmaxf(m, sm[w]);
    DrawPiece *out = W.piece + row * P + p;
    if (d.greedy) {
        uint32_t idx = 0xFFFFFFFFu;
#pragma unroll
        for (int e = kPer - 1; e >= 0; e--)
            if (v[e] == m) idx = i0 + piece_token<F16>(aligned, e);
        for (int s = 32; s; s >>= 1) idx = min(idx, (uint32_t)__shfl_xor((int)idx, s));
        if (lane == 0) si[wave] = idx;
        __syncthreads();
        for (int w = 0; w < 16; w++) idx = min(idx, si[w]);
        if (tid == 0) *out = DrawPiece{m, idx, 0.0, 0};
        return;
    }
    if (m == -INFINITY) {
        if (tid == 0) *out = DrawPiece{m, 0, -kInfE, 0};
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
#pragma unroll
        for (int t = 0; t < kPer; t++) {
            if (!(v[t] >= low)) continue;
            int down;
            const uint64_t w = draw_weight(unit, v[t], kCutBits, tab, down);
            atomicAdd((unsigned long long *)&hist[down >> kBinShift], (unsigned long long)(w | 1ull << 50));
        }
        __syncthreads();
        const size_t at = (row * P + p) * kBins;
        for (int b = tid; b < kBins; b += kDrawThreads) W.hist[at + b] = hist[b];
        if (tid == 0) *out = DrawPiece{m, 0, e, 0};
    } else {
        uint64_t s = 0;
#pragma unroll
        for (int t = 0; t < kPer; t++) {
            if (!(v[t] >= low)) continue;
            int down;
            s += draw_weight(unit, v[t], kPlainBits, tab, down);
        }
        s = wave_sum(s);
        if (lane == 0) ss[wave] = s;
        __syncthreads();
        if (tid == 0) {
            s = 0;
            for (int w = 0; w < 16; w++) s += ss[w];
            *out = DrawPiece{m, 0, e, s};
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

struct PickShared {
    double tab[kSteps];
    DrawPiece piece[kMaxPieces];
    uint64_t kept[kMaxPieces];  // kept sums of the pieces, in their units
    double sum[kBins];          // the row's bins, in the row's unit
    uint32_t cnt[kBins];
    uint64_t sub_sum[kBins];    // of a key range's parts
    uint32_t sub_cnt[kBins];
    uint32_t list_key[kList], list_idx[kList];  // tokens of one bin
    uint32_t list_n;
    int todo[kMaxPieces], ntodo;  // pieces that have tokens in a bin
    double before_d, red[16];
    uint64_t before_u;
    uint32_t at, ties, klo, khi;
};

template <bool F16>
__global__ __launch_bounds__(kDrawThreads) void k_draw_pick(const void *__restrict__ logits, int n, int P, bool aligned,
                                                            const float *__restrict__ filter,
                                                            const float *__restrict__ rnd, uint32_t *__restrict__ token,
                                                            float *__restrict__ logp, DrawWork W) {
    __shared__ PickShared S;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x, base = row * n;
    const DrawRow d = draw_row(filter + 4 * row, n);
    const uint64_t *hist = W.hist + row * P * kBins;
    float u = rnd[row];
    if (tid < P) S.piece[tid] = W.piece[row * P + tid];
    if (!d.greedy) draw_table(S.tab);
    __syncthreads();
    float m = -INFINITY;
    double e = -kInfE;
    uint32_t first = 0xFFFFFFFFu;
    for (int p = 0; p < P; p++) {
        if (S.piece[p].m > m) m = S.piece[p].m, first = S.piece[p].idx;
        e = fmax(e, S.piece[p].e);
    }
    if (m == -INFINITY || d.greedy) {
        if (tid == 0) {
            token[row] = m == -INFINITY ? 0xFFFFFFFFu : first;
            if (logp) logp[row] = m == -INFINITY ? -INFINITY : 0.0f;
        }
        return;
    }
    // a piece's unit below the row's in octaves, and its first bin among the row's
    auto octaves = [&](int p) { return (int)fmin((e - S.piece[p].e) * (1.0 / kSteps), 4000.0); };
    auto shift = [&](int p) { return min(8 * octaves(p), kBins); };
    const DrawUnit unit(d.c, e, m);
    const float low = draw_low(m, d);
    DrawCut cut{0, 0xFFFFFFFFu};
    int cbin = kBins;  // the cut's bin; kBins: no cut
    if (d.cuts) {
        if (tid < kBins) {
            double s = 0.0;
            uint32_t c = 0;
            for (int p0 = 0; p0 < P; p0 += 8) {
                uint64_t h[8];
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const int p = p0 + x, b = p < P && S.piece[p].m > -INFINITY ? tid - shift(p) : -1;
                    h[x] = b >= 0 ? hist[p * kBins + b] : 0;
                }
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    if (p0 + x >= P) break;
                    s += ldexp((double)(h[x] & kSumMask), -octaves(p0 + x));
                    c += (uint32_t)(h[x] >> 50);
                }
            }
            S.sum[tid] = s;
            S.cnt[tid] = c;
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
        // the keys of a bin into S.klo .. S.khi: its borders in l, exactly, from the floats around them
        auto bin_keys = [&](int bin) {
            __syncthreads();
            if (wave == 0) {
                if (unit.sharp) {
                    if (lane == 0) S.klo = S.khi = lg_key(m);
                } else {
                    uint32_t at[2];
#pragma unroll
                    for (int side = 0; side < 2; side++) {  // the first key of this bin, of the bin above
                        const int steps = (bin + 1 - side) << kBinShift;
                        float f = (float)((e - steps + 0.5) / d.c);
                        f = f == f ? fminf(fmaxf(f, kLeast), -kLeast) : 0.0f;
                        const uint32_t k0 = lg_key(f + 0.0f) - 32;
                        const float l = lg_unkey(k0 + lane);
                        double r;
                        const uint64_t yes = __ballot(l > m || (l >= low && -unit.steps(l, r) < steps));
                        at[side] = k0 + (yes ? __ffsll((long long)yes) - 1 : 64);
                    }
                    if (lane == 0) S.klo = at[0], S.khi = min(at[1] - 1, lg_key(m));
                }
            }
            __syncthreads();
        };
        // fn(key, index, logit) for a bin's tokens with keys in [klo, khi], from
        // the pieces that have any, AT pieces in flight
        auto row_pass = [&](auto at_c, int bin, uint32_t klo, uint32_t khi, auto fn) {
            constexpr int AT = decltype(at_c)::value;
            __syncthreads();
            if (tid == 0) S.ntodo = 0;
            __syncthreads();
            if (tid < P) {
                const int b = bin - shift(tid);
                if (S.piece[tid].m > -INFINITY && b >= 0 && hist[tid * kBins + b]) S.todo[atomicAdd(&S.ntodo, 1)] = tid;
            }
            __syncthreads();
            const float llo = lg_unkey(klo), lhi = lg_unkey(khi);
            for (int t = 0; t < S.ntodo; t += AT) {
                float v[AT][kPer];
#pragma unroll
                for (int a = 0; a < AT; a++)
                    if (t + a < S.ntodo) piece_load<F16>(logits, base, S.todo[t + a] * kPiece, n, aligned, v[a]);
#pragma unroll
                for (int a = 0; a < AT; a++) {
                    if (t + a >= S.ntodo) break;
                    const int i0 = S.todo[t + a] * kPiece;
#pragma unroll
                    for (int x = 0; x < kPer; x++)
                        if (v[a][x] >= llo && v[a][x] <= lhi) fn(lg_key(v[a][x]), (uint32_t)(i0 + piece_token<F16>(aligned, x)));
                }
            }
        };
        int listed = -1;  // the bin in the list, with its keys from list_lo to list_hi
        uint32_t list_lo = 0, list_hi = 0;
        auto holds = [&](int bin, uint32_t klo, uint32_t khi) { return listed == bin && klo >= list_lo && khi <= list_hi; };
        auto bin_pass = [&](int bin, uint32_t klo, uint32_t khi, auto fn) {
            if (holds(bin, klo, khi)) {
                for (uint32_t i = tid; i < S.list_n; i += kDrawThreads) {
                    const uint32_t k = S.list_key[i];
                    if (k >= klo && k <= khi) fn(k, S.list_idx[i]);
                }
            } else {
                row_pass(std::integral_constant<int, 1>{}, bin, klo, khi, fn);
            }
        };
        // stage 0: top-k (min-p has set its key already); stage 1: top-p of what that leaves
        for (int stage = 0; stage < 2; stage++) {
            const bool by_count = stage == 0;
            if (by_count ? d.top_k == 0 && cbin == kBins : d.top_p >= 1.0f) continue;
            if (!by_count || d.top_k) {
                double goal = d.top_k;
                if (!by_count) {
                    double s = 0.0;
                    if (cbin < kBins)
                        for (int p = tid; p < P; p += kDrawThreads) s += ldexp((double)S.kept[p], -octaves(p));
                    else if (tid < kBins)
                        s = S.sum[tid];
                    s = wave_sum(s);
                    __syncthreads();
                    if (lane == 0) S.red[wave] = s;
                    __syncthreads();
                    goal = 0.0;
                    for (int w = 0; w < 16; w++) goal += S.red[w];
                    goal *= (double)d.top_p;
                }
                // the first bin at which the running count or sum reaches the goal
                __syncthreads();
                if (wave == 0) {
                    double own[8], s = 0.0;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int b = 8 * lane + j;
                        own[j] = by_count ? (double)S.cnt[b] : b < cbin ? S.sum[b] : 0.0;
                        s += own[j];
                    }
                    double run = s;
                    for (int o = 1; o < 64; o <<= 1) {
                        const double x = __shfl_up(run, o);
                        if (lane >= o) run += x;
                    }
                    const uint64_t hit = __ballot(run >= goal && run > 0.0);
                    if (hit == 0 && lane == 63) S.at = kBins, S.before_d = run;
                    if (hit && lane == __ffsll((long long)hit) - 1) {
                        double b = run - s, last_b = b;
                        int last = 0;
                        bool done = false;
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            if (!done && own[j] > 0.0) last = j, last_b = b;
                            done = done || (own[j] > 0.0 && b + own[j] >= goal);
                            b += own[j];
                        }
                        S.at = 8 * lane + last;
                        S.before_d = last_b;
                    }
                }
                __syncthreads();
                int bin = S.at;
                const double before_d = S.before_d;
                if (!by_count && bin == kBins) bin = cbin;  // not above the cut's bin: in it
                // a count that ends below the cut, or among tokens without weight, cuts nothing
                if (bin <= cbin && bin < kDeepBin) {
                    const bool limited = bin == cbin;
                    const DrawCut lim = cut;
                    bin_keys(bin);
                    const uint32_t klo0 = limited ? max(S.klo, lim.key) : S.klo;
                    uint32_t klo = klo0, khi = max(S.khi, klo0);
                    // the goal inside the bin: a count, or weights kInBits below the octave that holds the bin's top
                    const double left = fmax(goal - before_d, 0.0);
                    const uint64_t want = by_count ? (uint64_t)left : (uint64_t)ceil(ldexp(left, (bin >> 3) + kInBits - kCutBits));
                    const DrawUnit in_unit(d.c, e - (double)kSteps * (bin >> 3), m);
                    uint64_t before = 0;
                    uint32_t cnt = S.cnt[bin], ties = 0;
                    for (;;) {  // keys are narrowed by 512 parts of their range until one is left
                        if (cnt <= kList && !holds(bin, klo, khi)) {
                            __syncthreads();
                            if (tid == 0) S.list_n = 0;
                            row_pass(std::integral_constant<int, 4>{}, bin, klo, khi, [&](uint32_t k, uint32_t i) {
                                const uint32_t x = atomicAdd(&S.list_n, 1u);
                                if (x < kList) S.list_key[x] = k, S.list_idx[x] = i;
                            });
                            __syncthreads();
                            listed = S.list_n <= kList ? bin : -1;
                            list_lo = klo;
                            list_hi = khi;
                        }
                        int sh = 0;
                        while ((khi - klo) >> sh >= kBins) sh++;
                        __syncthreads();
                        if (tid < kBins) S.sub_sum[tid] = 0, S.sub_cnt[tid] = 0;
                        __syncthreads();
                        bin_pass(bin, klo, khi, [&](uint32_t k, uint32_t i) {
                            if (limited && !lim.keeps(k, i)) return;
                            const uint32_t b = (khi - k) >> sh;
                            int down;
                            atomicAdd(&S.sub_cnt[b], 1u);
                            if (!by_count)
                                atomicAdd((unsigned long long *)&S.sub_sum[b], (unsigned long long)draw_weight(in_unit, lg_unkey(k), kInBits, S.tab, down));
                        });
                        __syncthreads();
                        if (wave == 0) {
                            uint64_t own[8], s = 0;
                            uint32_t c[8], some = 0;
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                c[j] = S.sub_cnt[8 * lane + j];
                                own[j] = by_count ? c[j] : S.sub_sum[8 * lane + j];
                                some |= c[j];
                                s += own[j];
                            }
                            uint64_t run = s;
                            for (int o = 1; o < 64; o <<= 1) {
                                const uint64_t x = __shfl_up(run, o);
                                if (lane >= o) run += x;
                            }
                            if (lane == 0) S.at = 0, S.ties = 0, S.before_u = before;  // stands if the range is empty
                            const uint64_t any = __ballot(some != 0), hit = __ballot(some != 0 && before + run >= want);
                            if (lane == (hit ? __ffsll((long long)hit) : 64 - __clzll((long long)any)) - 1) {
                                uint64_t b = before + run - s, last_b = b;
                                uint32_t last = 0, last_c = 0;
                                bool done = false;
#pragma unroll
                                for (int j = 0; j < 8; j++) {
                                    if (!done && c[j]) last = j, last_c = c[j], last_b = b;
                                    done = done || (c[j] && b + own[j] >= want);
                                    b += own[j];
                                }
                                S.at = 8 * lane + last;
                                S.ties = last_c;
                                S.before_u = last_b;
                            }
                        }
                        __syncthreads();
                        before = S.before_u;
                        cnt = ties = S.ties;
                        khi -= S.at << sh;
                        if (sh == 0) break;
                        klo = max(klo, khi - ((1u << sh) - 1u));
                    }
                    // one key is left; its tokens weigh the same, so a division tells how many stay
                    int down;
                    const uint64_t w = by_count ? 1 : draw_weight(in_unit, lg_unkey(khi), kInBits, S.tab, down);
                    uint32_t c = want > before && w ? (uint32_t)min((unsigned long long)((want - before + w - 1) / w), (unsigned long long)n) : 1;
                    cut = DrawCut{khi, limited && lim.key == khi ? lim.last : 0xFFFFFFFFu};
                    cbin = bin;
                    if (c < ties) {  // the index of the c-th token of this key, by 512 parts of the index range
                        uint32_t lo = 0, hi = (uint32_t)n - 1;
                        while (lo < hi) {
                            const uint32_t step = (hi - lo) / kBins + 1;
                            __syncthreads();
                            if (tid < kBins) S.sub_cnt[tid] = 0;
                            __syncthreads();
                            bin_pass(bin, khi, khi, [&](uint32_t, uint32_t i) {
                                if (i >= lo && i <= hi) atomicAdd(&S.sub_cnt[(i - lo) / step], 1u);
                            });
                            __syncthreads();
                            if (tid == 0) {
                                uint32_t b = 0, got = 0;
                                while (b < kBins - 1 && got + S.sub_cnt[b] < c) got += S.sub_cnt[b++];
                                S.at = b;
                                S.ties = got;
                            }
                            __syncthreads();
                            c -= S.ties;
                            lo += S.at * step;
                            hi = min(hi, lo + step - 1);
                        }
                        cut.last = lo;
                    }
                }
            }
            if (cbin == kBins) continue;
            // kept sums of the pieces: whole bins, and the cut's own bin token by token
            bin_keys(cbin);
            for (int p = wave; p < P; p += 16) {
                uint64_t s = 0;
                const int top = S.piece[p].m > -INFINITY ? cbin - shift(p) : 0;
#pragma unroll
                for (int x = 0; x < kBins; x += 64) s += x + lane < top ? hist[p * kBins + x + lane] & kSumMask : 0;
                s = wave_sum(s);
                if (lane == 0) S.kept[p] = s;
            }
            const uint32_t top_key = S.khi;
            __syncthreads();
            bin_pass(cbin, cut.key, top_key, [&](uint32_t k, uint32_t i) {
                if (!cut.keeps(k, i)) return;
                const int p = i / kPiece;
                const DrawUnit pu(d.c, S.piece[p].e, S.piece[p].m);
                int down;
                atomicAdd((unsigned long long *)&S.kept[p], (unsigned long long)draw_weight(pu, lg_unkey(k), kCutBits, S.tab, down));
            });
            __syncthreads();
        }
    }
    // Where no cut was found (all tokens stay) a row with cuts has its sums in the bins.
    const int bits = d.cuts ? kCutBits : kPlainBits;
    if (cbin == kBins) {
        for (int p = wave; p < P; p += 16) {
            uint64_t s = S.piece[p].sum;
            if (d.cuts) {
                s = 0;
                if (S.piece[p].m > -INFINITY)
                    for (int x = lane; x < kBins; x += 64) s += hist[p * kBins + x] & kSumMask;
                s = wave_sum(s);
            }
            if (lane == 0) S.kept[p] = s;
        }
        __syncthreads();
    }
    // the draw's piece
    double total = 0.0;
    for (int p = 0; p < P; p++) total += ldexp((double)S.kept[p], -octaves(p));
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    const double target = (double)u * total;
    double run = 0.0, at = 0.0;
    int piece = 0;
    for (int p = 0; p < P; p++) {
        if (S.kept[p] == 0) continue;
        piece = p;
        at = run;
        run += ldexp((double)S.kept[p], -octaves(p));
        if (run > target) break;
    }
    // its token: lanes hold tokens of the piece in index order
    const DrawUnit pu(d.c, S.piece[piece].e, S.piece[piece].m);
    const float plow = draw_low(S.piece[piece].m, d);
    uint64_t goal = (uint64_t)fmax(ldexp(target - at, octaves(piece)), 0.0);
    if (goal >= S.kept[piece]) goal = S.kept[piece] - 1;
    float v[kPer];
    uint64_t w[kPer], mine = 0;
    const int i0 = piece * kPiece + tid * kPer;
#pragma unroll
    for (int x = 0; x < kPer; x++) v[x] = i0 + x < n ? lg_value<F16>(logits, base + i0 + x) : -INFINITY;
#pragma unroll
    for (int x = 0; x < kPer; x++) {
        int down;
        w[x] = 0;
        if (v[x] >= plow && cut.keeps(lg_key(v[x]), i0 + x)) w[x] = draw_weight(pu, v[x], bits, S.tab, down);
        mine += w[x];
    }
    uint64_t pre = mine;
    for (int s = 1; s < 64; s <<= 1) {
        const uint64_t o = __shfl_up(pre, s);
        if (lane >= s) pre += o;
    }
    uint64_t *wave_total = S.sub_sum;
    if (lane == 63) wave_total[wave] = pre;
    __syncthreads();
    uint64_t b = pre - mine;
    for (int x = 0; x < wave; x++) b += wave_total[x];
    if (goal >= b && goal < b + mine) {
        int hit = -1;
        float l = 0.0f;
#pragma unroll
        for (int x = 0; x < kPer; x++) {
            b += w[x];
            if (hit < 0 && goal < b) hit = x, l = v[x];
        }
        token[row] = i0 + hit;
        if (logp) {  // the sum is total 2^(E - bits); the maximum lies `below` octaves under E
            double r = 0.0, below = 1.0;
            if (!unit.sharp) below = -(unit.steps(m, r) + 0.0) / kSteps, below -= r / kSteps;
            const double z = l == m ? 0.0 : ((double)l - (double)m) / d.T;
            logp[row] = (float)(z - (log(ldexp(total, -bits)) + below * 0.69314718055994530942));
        }
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
// result itself.
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
static void draw_launch(rsv_ctx *ctx, const void *logits, int n, int P, bool aligned, const float *filter, const float *rnd,
                        uint32_t *token, float *logp, const DrawWork &W, uint64_t rows) {
    hipLaunchKernelGGL((k_draw_scan<F16>), dim3((unsigned)(rows * P)), dim3(kDrawThreads), 0, ctx->stream, logits, n, P, aligned, filter, W);
    hipLaunchKernelGGL((k_draw_pick<F16>), dim3((unsigned)rows), dim3(kDrawThreads), 0, ctx->stream, logits, n, P, aligned, filter, rnd,
                       token, logp, W);
}

int launch_draw(rsv_ctx *ctx, const void *logits, int f16, uint32_t *token, uint64_t n, const float *filter,
                const float *rnd, float *logp, float *work, uint64_t rows) {
    const int P = draw_pieces(n);
    DrawWork W;
    W.hist = (uint64_t *)work;
    W.piece = (DrawPiece *)(W.hist + rows * P * kBins);
    const bool aligned = n * (f16 ? 2 : 4) % 16 == 0;
    if (f16)
        draw_launch<true>(ctx, logits, (int)n, P, aligned, filter, rnd, token, logp, W, rows);
    else
        draw_launch<false>(ctx, logits, (int)n, P, aligned, filter, rnd, token, logp, W, rows);
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

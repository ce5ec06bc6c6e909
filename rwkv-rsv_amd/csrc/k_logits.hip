// What a served step takes from its logits rows: draws from given random
// numbers (rsv_sample_rand_batch) and log-probabilities of given tokens
// (rsv_token_logprobs).
#include <algorithm>

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
// A token's weight is 2^x, x = l * log2(e) / T, held as an integer with 48 bits
// below the octave E above the piece's largest (E - x > 0).  With c = 64
// log2(e) / T, q = floor(l c) and r = l c - q (one rounding) the weight is
// 2^(q/64) 2^(r/64): a 64-entry table and a Taylor polynomial of degree 5 in
// r ln2 / 64 < 0.011 (2e-15 off).  Adding 2^52 to the scaled weight leaves the
// integer in the low bits of the sum.  Integers add up the same in any order;
// pieces are put together in 64-bit floats in the pieces' order, which
// depends on n alone.  Bins follow q, so they mean the same in every piece.
constexpr int kPiece = 8192, kDrawThreads = 1024, kPer = kPiece / kDrawThreads;
constexpr int kBins = 512, kBits = 48, kMaxPieces = (int)(kLogitsMaxN / kPiece);
constexpr int kList = 4096;  // a bin's tokens held in LDS

struct DrawPiece {
    float m;        // largest logit (-inf: nothing to draw)
    uint32_t idx;   // its lowest token
    double e64;     // 64 E
    uint64_t sum;
    uint32_t cnt, pad;  // tokens in the histogram
};
struct DrawWork {
    DrawPiece *piece;   // [rows, P]
    uint64_t *sum;      // [rows, P, kBins]
    uint16_t *cnt;      // [rows, P, kBins]
};
struct DrawRow {
    double T, c64;
    float min_p;    // > 0: active
    uint32_t top_k;  // > 0 and < n: active
    float top_p;    // < 1: active
    bool greedy, cuts;
};

__device__ __forceinline__ DrawRow draw_row(const float *f, int n) {
    DrawRow d;
    const float T = f[0], p = f[2], m = f[3];
    const uint32_t k = __float_as_uint(f[1]);
    d.greedy = !(T > 0.0f);
    d.T = T;
    d.c64 = 64.0 * 1.4426950408889634074 / (double)T;
    d.top_k = k < (uint32_t)n ? k : 0;
    d.top_p = p < 1.0f ? fmaxf(p, 0.0f) : 1.0f;
    d.min_p = m > 0.0f && T < INFINITY ? fminf(m, 1.0f) : 0.0f;
    d.cuts = !d.greedy && (d.top_k || d.top_p < 1.0f || d.min_p > 0.0f);
    return d;
}

// 64 E of a piece (or its inf tokens): whole octaves strictly above its maximum.
constexpr double kInfE = 1e300;
__device__ __forceinline__ double draw_e64(float m, double c64) {
    return m == INFINITY ? kInfE : 64.0 * (floor(floor((double)m * c64) * 0.015625) + 1.0);
}
// q of a token in a piece with this maximum; +inf tokens stand one step below
// kInfE, the others of such a piece carry no weight.
__device__ __forceinline__ double draw_q(float l, double c64, bool inf) {
    return inf ? l == INFINITY ? kInfE : -kInfE : floor((double)l * c64);
}
// A token's bin below the piece's octave: 0 .. kBins - 1, the last one open.
__device__ __forceinline__ int draw_bin(double q, double e64) {
    const double down = e64 - 1.0 - q;  // 0, 1, ...
    return down < (double)(8 * kBins) ? max((int)down, 0) >> 3 : kBins - 1;
}
// r of a token; where a step is no longer seen beside l c (|l c| > 2^53),
// tokens of different logits are whole octaves apart and any r will do
__device__ __forceinline__ double draw_frac(float l, double c64, double q) {
    return fmin(fmax(fma((double)l, c64, -q), 0.0), 1.0);
}
__device__ __forceinline__ uint64_t draw_weight(float l, double c64, double q, double e64, bool inf, const double *tab) {
    const double down = e64 - q;
    if (!(down < 64.0 * kBits + 64.0)) return 0;
    if (inf) return 1ull << (kBits - 1);
    const int k = -(int)down;  // -64 kBits - 63 .. 0
    const double r = draw_frac(l, c64, q) * (0.69314718055994530942 / 64.0);
    double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const double t = ldexp(tab[k & 63], (k >> 6) + kBits);
    return (uint64_t)__double_as_longlong(fma(t, p, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
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
    __shared__ double tab[64];
    __shared__ float sm[16];
    __shared__ uint32_t si[16];
    __shared__ uint64_t ss[16];
    __shared__ uint64_t hsum[kBins];
    __shared__ uint32_t hcnt[kBins];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x / P;
    const int p = blockIdx.x % P, i0 = p * kPiece;
    float v[kPer];
    piece_load<F16>(logits, row * n, i0, n, aligned, v);
    const DrawRow d = draw_row(filter + 4 * row, n);
    if (tid < 64) tab[tid] = exp2((double)tid / 64.0);
    if (d.cuts)
        for (int b = tid; b < kBins; b += kDrawThreads) hsum[b] = 0, hcnt[b] = 0;
    float m = v[0];
#pragma unroll
    for (int e = 1; e < kPer; e++) m = fmaxf(m, v[e]);
    for (int s = 32; s; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
    if (lane == 0) sm[wave] = m;
    __syncthreads();
    for (int w = 0; w < 16; w++) m = fmaxf(m, sm[w]);
    uint32_t idx = 0xFFFFFFFFu;
    if (d.greedy) {
#pragma unroll
        for (int e = kPer - 1; e >= 0; e--)
            if (v[e] == m) idx = i0 + piece_token<F16>(aligned, e);
        for (int s = 32; s; s >>= 1) idx = min(idx, (uint32_t)__shfl_xor((int)idx, s));
        if (lane == 0) si[wave] = idx;
        __syncthreads();
        for (int w = 0; w < 16; w++) idx = min(idx, si[w]);
    }
    DrawPiece *out = W.piece + row * P + p;
    const bool inf = m == INFINITY;
    const double e64 = draw_e64(m, d.c64);
    if (d.greedy || m == -INFINITY) {
        if (tid == 0) *out = DrawPiece{m, idx, m == -INFINITY ? -kInfE : e64, 0, 0, 0};
        if (d.greedy) return;
    }
    // below this nothing survives min-p, whatever the row's maximum
    const float low = d.min_p > 0.0f ? (float)((double)m + d.T * log((double)d.min_p)) : -INFINITY;
    const float floor_l = low - fabsf(low) * 2.4e-7f;
    uint64_t s = 0;
    uint32_t c = 0;
    if (m > -INFINITY) {
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            if (v[e] == -INFINITY || (d.min_p > 0.0f && v[e] < floor_l)) continue;
            const double q = draw_q(v[e], d.c64, inf);
            const uint64_t w = draw_weight(v[e], d.c64, q, e64, inf, tab);
            s += w;
            c++;
            if (d.cuts) {
                const int b = draw_bin(q, e64);
                atomicAdd((unsigned long long *)&hsum[b], (unsigned long long)w);
                atomicAdd(&hcnt[b], 1u);
            }
        }
        s = wave_sum(s);
        c = wave_sum(c);
        if (lane == 0) ss[wave] = s, si[wave] = c;
    }
    __syncthreads();
    if (tid == 0 && m > -INFINITY) {
        s = 0;
        c = 0;
        for (int w = 0; w < 16; w++) s += ss[w], c += si[w];
        *out = DrawPiece{m, idx, e64, s, c, 0};
    }
    if (d.cuts) {
        const size_t at = (row * P + p) * kBins;
        for (int b = tid; b < kBins; b += kDrawThreads) {
            W.sum[at + b] = hsum[b];
            W.cnt[at + b] = (uint16_t)hcnt[b];
        }
    }
}

// ---- the second launch
// A cut of the row's order: kept are keys above `key`, and of its own tokens
// those up to index `last`.
struct DrawCut {
    uint32_t key, last;
};
__device__ __forceinline__ bool cut_keeps(const DrawCut &c, uint32_t key, uint32_t i) {
    return key > c.key || (key == c.key && i <= c.last);
}

struct PickShared {
    double tab[64];
    DrawPiece piece[kMaxPieces];
    uint64_t kept[kMaxPieces];      // kept sums of the pieces
    double sum[kBins];              // of the row's bins, below the row's octave
    uint32_t cnt[kBins];
    uint64_t sub_sum[kBins];        // of a key range's parts
    uint32_t sub_cnt[kBins];
    uint32_t list_key[kList], list_idx[kList];
    uint32_t list_n;
    int list_bin;
    int todo[kMaxPieces], ntodo;    // pieces that have tokens in the bin asked for
    double red_d[16];
    uint64_t red_u[16];
    uint32_t red_i[16];
    double pick_before;
    uint32_t pick_at, pick_cnt;
    uint32_t token;
    float logit;
};

template <bool F16>
struct Picker {
    PickShared &S;
    const void *logits;
    size_t base, row;
    int n, P;
    bool aligned;
    DrawRow d;
    DrawWork W;
    float m;
    double e64;

    __device__ bool inf() const { return m == INFINITY; }
    // where bins of a piece start among the row's
    __device__ int shift(int p) const {
        const double s = (e64 - S.piece[p].e64) * 0.125;
        return s < (double)kBins ? (int)s : kBins;
    }
    __device__ int bin_of(float l) const { return draw_bin(draw_q(l, d.c64, inf()), e64); }
    // A weight with kBinBits bits below the octave that holds this bin's top:
    // a bin can hold all 2^20 tokens of a row.
    static constexpr int kBinBits = 40;
    __device__ double bin_top64(int bin) const { return e64 - 64.0 * (bin >> 3); }
    __device__ uint64_t weight_at(float l, double top64) const {
        return draw_weight(l, d.c64, draw_q(l, d.c64, inf()), top64, inf(), S.tab) >> (kBits - kBinBits);
    }

    // fn(key, index, logit) for every token of a bin; from the list in LDS if it holds this bin
    template <typename Fn>
    __device__ void for_bin(int bin, Fn fn) {
        if (S.list_bin == bin) {
            for (uint32_t i = threadIdx.x; i < S.list_n; i += kDrawThreads)
                fn(S.list_key[i], S.list_idx[i], lg_unkey(S.list_key[i]));
            return;
        }
        __syncthreads();
        if (threadIdx.x == 0) S.ntodo = 0;
        __syncthreads();
        if ((int)threadIdx.x < P) {
            const int p = threadIdx.x, b = bin - shift(p);
            // the row's last bin gathers what the pieces have from there on
            if (S.piece[p].m > -INFINITY && (bin == kBins - 1 || (b >= 0 && W.cnt[(row * P + p) * kBins + b])))
                S.todo[atomicAdd(&S.ntodo, 1)] = p;
        }
        __syncthreads();
        constexpr int AT = 4;  // pieces in flight
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
                for (int e = 0; e < kPer; e++) {
                    const int i = i0 + piece_token<F16>(aligned, e);
                    if (i < n && bin_of(v[a][e]) == bin) fn(lg_key(v[a][e]), (uint32_t)i, v[a][e]);
                }
            }
        }
    }

    __device__ void gather(int bin) {
        __syncthreads();
        if (S.list_bin == bin || S.cnt[bin] > kList) return;
        if (threadIdx.x == 0) S.list_n = 0;
        __syncthreads();
        for_bin(bin, [&](uint32_t key, uint32_t i, float) {
            const uint32_t at = atomicAdd(&S.list_n, 1u);
            if (at < kList) S.list_key[at] = key, S.list_idx[at] = i;
        });
        __syncthreads();
        if (threadIdx.x == 0) S.list_bin = S.list_n <= kList ? bin : -1;
        __syncthreads();
    }

    // The first bin at which the running count (by_count) or sum reaches the goal, with what goes before it.
    __device__ int find_bin(bool by_count, double goal, double &before) {
        __syncthreads();
        if (threadIdx.x < 64) {
            const int lane = threadIdx.x;
            double own[8], s = 0.0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                own[j] = by_count ? (double)S.cnt[8 * lane + j] : S.sum[8 * lane + j];
                s += own[j];
            }
            double run = s;
            for (int o = 1; o < 64; o <<= 1) {
                const double v = __shfl_up(run, o);
                if (lane >= o) run += v;
            }
            const uint64_t hit = __ballot(run >= goal && run > 0.0);
            const uint64_t some = __ballot(s > 0.0);
            const int at = hit ? __ffsll((long long)hit) - 1 : 63 - __clzll((long long)some);
            if (lane == at) {
                double b = run - s;  // at most a rounding off the lane below's run
                int j = 0, last = 0;
                double last_b = b;
                for (; j < 8; j++) {
                    if (own[j] > 0.0) last = j, last_b = b;
                    if (own[j] > 0.0 && b + own[j] >= goal) break;
                    b += own[j];
                }
                S.pick_at = 8 * lane + last;
                S.pick_before = last_b;
            }
        }
        __syncthreads();
        before = S.pick_before;
        return (int)S.pick_at;
    }

    // Within a bin: the token at which the goal is reached.  Keys are narrowed
    // by 512 parts of their range until one key is left; its tokens weigh the
    // same, so a division tells how many of them stay.  before and goal count
    // tokens or, with weights, are integers below the bin's top.
    __device__ DrawCut resolve(int bin, bool by_count, uint64_t goal, const DrawCut &lim, bool limited) {
        const double top64 = bin_top64(bin);
        uint32_t klo = 0xFFFFFFFFu, khi = 0;
        gather(bin);
        for_bin(bin, [&](uint32_t key, uint32_t i, float) {
            if (limited && !cut_keeps(lim, key, i)) return;
            klo = min(klo, key);
            khi = max(khi, key);
        });
        for (int s = 32; s; s >>= 1) {
            klo = min(klo, (uint32_t)__shfl_xor((int)klo, s));
            khi = max(khi, (uint32_t)__shfl_xor((int)khi, s));
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) S.red_i[threadIdx.x >> 6] = klo, S.red_u[threadIdx.x >> 6] = khi;
        __syncthreads();
        for (int w = 0; w < 16; w++) klo = min(klo, S.red_i[w]), khi = max(khi, (uint32_t)S.red_u[w]);
        uint64_t before = 0;
        uint32_t ties = 0;
        for (;;) {
            int sh = 0;
            while ((khi - klo) >> sh >= kBins) sh++;
            __syncthreads();
            for (int b = threadIdx.x; b < kBins; b += kDrawThreads) S.sub_sum[b] = 0, S.sub_cnt[b] = 0;
            __syncthreads();
            for_bin(bin, [&](uint32_t key, uint32_t i, float l) {
                if (key < klo || key > khi || (limited && !cut_keeps(lim, key, i))) return;
                const uint32_t b = (khi - key) >> sh;
                atomicAdd(&S.sub_cnt[b], 1u);
                if (!by_count) atomicAdd((unsigned long long *)&S.sub_sum[b], (unsigned long long)weight_at(l, top64));
            });
            __syncthreads();
            if (threadIdx.x < 64) {
                const int lane = threadIdx.x;
                uint64_t own[8], s = 0;
                uint32_t any = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    own[j] = by_count ? S.sub_cnt[8 * lane + j] : S.sub_sum[8 * lane + j];
                    any |= S.sub_cnt[8 * lane + j];
                    s += own[j];
                }
                uint64_t run = s;
                for (int o = 1; o < 64; o <<= 1) {
                    const uint64_t v = __shfl_up(run, o);
                    if (lane >= o) run += v;
                }
                const uint64_t hit = __ballot(any && before + run >= goal);
                const uint64_t some = __ballot(any != 0);
                const int at = hit ? __ffsll((long long)hit) - 1 : 63 - __clzll((long long)some);
                if (lane == at) {
                    uint64_t b = before + run - s, last_b = b;
                    int last = 0;
                    for (int j = 0; j < 8; j++) {
                        if (S.sub_cnt[8 * lane + j] == 0) continue;
                        last = j, last_b = b;
                        if (b + own[j] >= goal) break;
                        b += own[j];
                    }
                    S.pick_at = 8 * lane + last;
                    S.pick_cnt = S.sub_cnt[8 * lane + last];
                    S.red_u[0] = last_b;
                }
            }
            __syncthreads();
            before = S.red_u[0];
            ties = S.pick_cnt;
            const uint32_t b = S.pick_at;
            const uint32_t top = khi - (b << sh);
            klo = sh == 0 ? top : max(klo, top - ((1u << sh) - 1u));
            khi = top;
            if (sh == 0) break;
        }
        uint64_t w = 1, left = goal > before ? goal - before : 0;
        if (!by_count) w = weight_at(lg_unkey(klo), top64);
        uint64_t c = w ? (left + w - 1) / w : 0;
        c = c < 1 ? 1 : c;
        DrawCut r{klo, 0xFFFFFFFFu};
        if (limited && lim.key == klo) r.last = lim.last;
        if (c < ties) r.last = nth_tie(bin, klo, (uint32_t)c);
        return r;
    }

    // Index of the c-th token of a key that lies in this bin.
    __device__ uint32_t nth_tie(int bin, uint32_t key, uint32_t c) {
        uint32_t lo = 0, hi = (uint32_t)n - 1;  // the smallest index i with c ties up to it
        while (lo < hi) {
            const uint32_t step = (hi - lo) / kBins + 1;  // parts of the index range
            __syncthreads();
            for (int b = threadIdx.x; b < kBins; b += kDrawThreads) S.sub_cnt[b] = 0;
            __syncthreads();
            for_bin(bin, [&](uint32_t k, uint32_t i, float) {
                if (k == key && i >= lo && i <= hi) atomicAdd(&S.sub_cnt[(i - lo) / step], 1u);
            });
            __syncthreads();
            if (threadIdx.x == 0) {
                uint32_t b = 0, got = 0;
                while (b < kBins - 1 && got + S.sub_cnt[b] < c) got += S.sub_cnt[b++];
                S.pick_at = b;
                S.pick_cnt = got;
            }
            __syncthreads();
            c -= S.pick_cnt;
            lo += S.pick_at * step;
            hi = min(hi, lo + step - 1);
        }
        return lo;
    }

    // The kept part of a cut's own bin, in the row's units.
    __device__ double bin_sum(int bin, const DrawCut &c) {
        const double top64 = bin_top64(bin);
        uint64_t s = 0;
        for_bin(bin, [&](uint32_t key, uint32_t i, float l) {
            if (cut_keeps(c, key, i)) s += weight_at(l, top64);
        });
        s = wave_sum(s);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) S.red_u[threadIdx.x >> 6] = s;
        __syncthreads();
        s = 0;
        for (int w = 0; w < 16; w++) s += S.red_u[w];
        __syncthreads();
        return ldexp((double)s, kBits - kBinBits - (bin >> 3));
    }
};

template <bool F16>
__global__ __launch_bounds__(kDrawThreads) void k_draw_pick(const void *__restrict__ logits, int n, int P, bool aligned,
                                                            const float *__restrict__ filter,
                                                            const float *__restrict__ rnd, uint32_t *__restrict__ token,
                                                            float *__restrict__ logp, DrawWork W) {
    __shared__ PickShared S;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x;
    Picker<F16> K{S, logits, row * n, row, n, P, aligned, draw_row(filter + 4 * row, n), W, -INFINITY, -kInfE};
    const DrawRow &d = K.d;
    if (tid < P) S.piece[tid] = W.piece[row * P + tid];
    if (tid >= kDrawThreads - 64) S.tab[tid & 63] = exp2((double)(tid & 63) / 64.0);
    if (tid == 0) S.list_bin = -1;
    __syncthreads();
    uint32_t first = 0xFFFFFFFFu;
    for (int p = 0; p < P; p++)
        if (S.piece[p].m > K.m) K.m = S.piece[p].m, first = S.piece[p].idx;
    for (int p = 0; p < P; p++) K.e64 = fmax(K.e64, S.piece[p].e64);
    if (K.m == -INFINITY || d.greedy) {
        if (tid == 0) {
            token[row] = K.m == -INFINITY ? 0xFFFFFFFFu : first;
            if (logp) logp[row] = K.m == -INFINITY ? -INFINITY : 0.0f;
        }
        return;
    }
    auto octaves = [&](int p) {  // of a piece's unit below the row's
        return (int)fmin((K.e64 - S.piece[p].e64) * 0.015625, 4000.0);
    };
    DrawCut cut{0, 0xFFFFFFFFu};
    int cbin = kBins;  // the bin of the cut
    if (d.cuts) {
        if (tid < kBins) {
            double s = 0.0;
            uint32_t c = 0;
            for (int p = 0; p < P; p++) {
                if (S.piece[p].m == -INFINITY) continue;
                const int sh = K.shift(p);
                const size_t at = (row * P + p) * kBins;
                if (tid < sh || tid == kBins - 1) continue;
                s += ldexp((double)W.sum[at + tid - sh], -octaves(p));
                c += W.cnt[at + tid - sh];
            }
            S.sum[tid] = s;
            S.cnt[tid] = c;
            c = wave_sum(c);
            if (lane == 0) S.red_i[wave] = c;
        }
        __syncthreads();
        if (tid == 0) {  // the last bin: all the others; 63 octaves down, no weight is left
            uint32_t c = 0;
            for (int p = 0; p < P; p++) c += S.piece[p].cnt;
            for (int w = 0; w < kBins / 64; w++) c -= S.red_i[w];
            S.cnt[kBins - 1] = c;
        }
        __syncthreads();
        double before;
        if (d.min_p > 0.0f) {  // the smallest float whose weight is at least min_p
            const double lim = K.inf() ? INFINITY : (double)K.m + d.T * log((double)d.min_p);
            float f = (float)lim;
            if ((double)f < lim) f = lg_unkey(lg_key(f + 0.0f) + 1);
            f = fminf(f + 0.0f, K.m);
            if (f > -INFINITY) {
                cut.key = lg_key(f);
                cbin = K.bin_of(f);
            }
        }
        if (d.top_k) {
            const int b = K.find_bin(true, (double)d.top_k, before);
            if (b <= cbin && before + S.cnt[b] >= (double)d.top_k) {
                const DrawCut c = K.resolve(b, true, d.top_k - (uint64_t)before, cut, false);
                if (c.key >= cut.key) cut = c, cbin = b;
            }
        }
        if (d.top_p < 1.0f) {
            double total;
            if (cbin < kBins) {  // the cut's bin counts as far as it is kept
                const double part = K.bin_sum(cbin, cut);
                __syncthreads();
                if (tid < kBins && tid >= cbin) S.sum[tid] = tid == cbin ? part : 0.0;
                __syncthreads();
            }
            total = 0.0;
            {
                double s = tid < kBins ? S.sum[tid] : 0.0;
                s = wave_sum(s);
                if (lane == 0) S.red_d[wave] = s;
                __syncthreads();
                for (int w = 0; w < kBins / 64; w++) total += S.red_d[w];
            }
            const double goal = (double)d.top_p * total;
            const int b = K.find_bin(false, goal, before);
            const double left = fmax(goal - before, 0.0);
            const bool lim = b == cbin;
            cut = K.resolve(b, false, (uint64_t)ceil(ldexp(left, (b >> 3) + K.kBinBits - kBits)), cut, lim);
            cbin = b;
        }
    }
    // kept sums of the pieces
    if (cbin < kBins) {
        K.gather(cbin);
        for (int p = wave; p < P; p += 16) {
            uint64_t s = 0;
            if (S.piece[p].m > -INFINITY) {
                const int sh = K.shift(p), top = min(kBins, cbin - sh);
                for (int b = lane; b < top; b += 64) s += W.sum[(row * P + p) * kBins + b];
            }
            s = wave_sum(s);
            if (lane == 0) S.kept[p] = s;
        }
        __syncthreads();
        K.for_bin(cbin, [&](uint32_t key, uint32_t i, float l) {
            if (!cut_keeps(cut, key, i)) return;
            const int p = i / kPiece;
            const uint64_t w = draw_weight(l, d.c64, draw_q(l, d.c64, S.piece[p].m == INFINITY), S.piece[p].e64, S.piece[p].m == INFINITY, S.tab);
            atomicAdd((unsigned long long *)&S.kept[p], (unsigned long long)w);
        });
    } else if (tid < P) {
        S.kept[tid] = S.piece[tid].sum;
    }
    __syncthreads();
    // the draw's piece
    double total = 0.0;
    for (int p = 0; p < P; p++) total += ldexp((double)S.kept[p], -octaves(p));
    float u = rnd[row];
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    const double target = (double)u * total;
    double run = 0.0, at = 0.0;
    int piece = 0;
    for (int p = 0; p < P; p++) {
        const double s = ldexp((double)S.kept[p], -octaves(p));
        if (S.kept[p]) piece = p, at = run;
        if (S.kept[p] && run + s > target) break;
        run += s;
    }
    // its token: lanes hold tokens of the piece in index order
    const float pm = S.piece[piece].m;
    const bool pinf = pm == INFINITY;
    const double pe = S.piece[piece].e64;
    uint64_t goal = (uint64_t)fmax(ldexp(target - at, octaves(piece)), 0.0);
    if (goal >= S.kept[piece]) goal = S.kept[piece] - 1;
    float v[kPer];
    uint64_t w[kPer], mine = 0;
    const int i0 = piece * kPiece + tid * kPer;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        v[e] = i0 + e < n ? lg_value<F16>(logits, K.base + i0 + e) : -INFINITY;
        const bool keep = v[e] > -INFINITY && cut_keeps(cut, lg_key(v[e]), i0 + e);
        w[e] = keep ? draw_weight(v[e], d.c64, draw_q(v[e], d.c64, pinf), pe, pinf, S.tab) : 0;
        mine += w[e];
    }
    uint64_t pre = mine;
    for (int s = 1; s < 64; s <<= 1) {
        const uint64_t o = __shfl_up(pre, s);
        if (lane >= s) pre += o;
    }
    __syncthreads();
    if (lane == 63) S.red_u[wave] = pre;
    __syncthreads();
    uint64_t b = pre - mine;
    for (int x = 0; x < wave; x++) b += S.red_u[x];
    if (goal >= b && goal < b + mine) {
        int hit = 0;
        for (int e = 0; e < kPer; e++) {
            if (goal < b + w[e]) {
                hit = e;
                break;
            }
            b += w[e];
        }
        float l = v[0];
#pragma unroll
        for (int e = 1; e < kPer; e++) l = hit == e ? v[e] : l;
        token[row] = i0 + hit;
        if (logp) {  // in units of the row's octave: total 2^-kBits 2^E
            const double z = l == K.m ? 0.0 : ((double)l - (double)K.m) / d.T;
            double me = -1.0;  // the maximum's octaves below E, as draw_weight takes them
            if (!K.inf()) {
                const double q = draw_q(K.m, d.c64, false);
                me = (q - K.e64 + draw_frac(K.m, d.c64, q)) / 64.0;
            }
            logp[row] = (float)(z - (log(ldexp(total, -kBits)) - me * 0.69314718055994530942));
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
    const uint64_t draw = rows * draw_pieces(n) * (sizeof(DrawPiece) + kBins * 10) / 4;
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
    W.sum = (uint64_t *)work;
    W.piece = (DrawPiece *)(W.sum + rows * P * kBins);
    W.cnt = (uint16_t *)(W.piece + rows * P);
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

// What a served step takes from its logits rows: draws from given random
// numbers (rsv_sample_rand_batch) and log-probabilities of given tokens
// (rsv_token_logprobs).
#include "rsv_common.h"

namespace rsv {

// A logit as the row's order sees it: NaN as -inf, -0 as +0.
__device__ __forceinline__ float lg_value(const void *p, int f16, size_t i) {
    const float l = f16 ? (float)((const _Float16 *)p)[i] : ((const float *)p)[i];
    return l == l ? l + 0.0f : -INFINITY;
}
// Order-preserving bits: larger logit, larger key.
__device__ __forceinline__ uint32_t lg_key(float l) {
    const uint32_t b = __float_as_uint(l);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lg_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// exp((l - m) / T); 1 at the maximum, 0 where l is -inf
__device__ __forceinline__ double lg_exp(float l, float m, double T) {
    return l == m ? 1.0 : l == -INFINITY ? 0.0 : exp(((double)l - (double)m) / T);
}

// ------------------------------------------------------------- draws
// Sums are integers: a weight is exp((l - m)/T) with `bits` bits after the
// point (62 - ceil(log2 n), so that a row's sum is at most 2^62), so no order
// of additions changes a draw.
struct DrawRow {
    float m;
    double T, min_p;
    uint32_t key;   // kept: keys above this one,
    uint64_t ties;  // and the first `ties` tokens of this key
};
__device__ __forceinline__ uint64_t dr_weight(const DrawRow &d, float l, int bits) {
    const double e = lg_exp(l, d.m, d.T);
    return e >= d.min_p ? (uint64_t)__double2ull_rn(ldexp(e, bits)) : 0;
}

constexpr int kDrawThreads = 1024;

template <typename T>
__device__ T block_sum(T v, T *sh) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    T s = 0;
    for (int w = 0; w < kDrawThreads / 64; w++) s += sh[w];
    return s;
}

// One block a row; every pass reads the row again.
__global__ __launch_bounds__(kDrawThreads) void k_draw_row(const void *__restrict__ logits, int f16, int n,
                                                           const float *__restrict__ filter,
                                                           const float *__restrict__ rnd, uint32_t *__restrict__ token,
                                                           float *__restrict__ logp, int bits) {
    __shared__ uint64_t hist[256];
    __shared__ uint64_t sh[16], sh2[16];
    __shared__ uint32_t shk[16], shi[16];
    __shared__ uint64_t s_before, s_pick;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x, base = row * n;
    // the maximum and its lowest index
    uint32_t bk = 0, bi = 0xFFFFFFFFu;
    for (int i = tid; i < n; i += kDrawThreads) {
        const uint32_t k = lg_key(lg_value(logits, f16, base + i));
        if (k > bk) bk = k, bi = i;
    }
    for (int d = 32; d; d >>= 1) {
        const uint32_t ok = __shfl_xor(bk, d), oi = __shfl_xor(bi, d);
        if (ok > bk || (ok == bk && oi < bi)) bk = ok, bi = oi;
    }
    if (lane == 0) shk[wave] = bk, shi[wave] = bi;
    __syncthreads();
    for (int w = 0; w < 16; w++)
        if (shk[w] > bk || (shk[w] == bk && shi[w] < bi)) bk = shk[w], bi = shi[w];
    DrawRow d;
    d.m = lg_unkey(bk);
    const float T = filter[4 * row];
    const uint32_t top_k = __float_as_uint(filter[4 * row + 1]);
    const float top_p = filter[4 * row + 2], min_p = filter[4 * row + 3];
    if (d.m == -INFINITY || !(T > 0.0f)) {
        if (tid == 0) {
            token[row] = d.m == -INFINITY ? 0xFFFFFFFFu : bi;
            if (logp) logp[row] = d.m == -INFINITY ? -INFINITY : 0.0f;
        }
        return;
    }
    d.T = T;
    d.min_p = min_p > 0.0f ? fmin((double)min_p, 1.0) : 0.0;
    d.key = 0;
    d.ties = ~0ull;
    if (top_k > 0 && top_k < (uint32_t)n) {  // the key of rank top_k - 1, 8 bits a pass
        uint64_t before = 0;
        uint32_t prefix = 0;
        for (int sft = 24; sft >= 0; sft -= 8) {
            __syncthreads();
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kDrawThreads) {
                const uint32_t k = lg_key(lg_value(logits, f16, base + i));
                if (sft == 24 || (k >> (sft + 8)) == prefix) atomicAdd((unsigned long long *)&hist[(k >> sft) & 255], 1ull);
            }
            __syncthreads();
            if (tid == 0) {
                int b = 255;
                uint64_t at = before;
                while (b > 0 && at + hist[b] < top_k) at += hist[b--];
                s_before = at;
                s_pick = b;
            }
            __syncthreads();
            before = s_before;
            prefix = prefix << 8 | (uint32_t)s_pick;
        }
        d.key = prefix;
        d.ties = top_k - before;
    }
    auto tie_count = [&](uint32_t key, uint64_t most) {  // tokens of this key, at most `most`
        uint64_t c = 0;
        for (int i = tid; i < n; i += kDrawThreads) c += lg_key(lg_value(logits, f16, base + i)) == key;
        c = block_sum(c, sh);
        return c < most ? c : most;
    };
    auto sum_above = [&](uint32_t key) {
        uint64_t s = 0;
        for (int i = tid; i < n; i += kDrawThreads) {
            const float l = lg_value(logits, f16, base + i);
            if (lg_key(l) > key) s += dr_weight(d, l, bits);
        }
        return block_sum(s, sh);
    };
    d.ties = tie_count(d.key, d.ties);
    const uint64_t wt0 = dr_weight(d, lg_unkey(d.key), bits);
    uint64_t total = sum_above(d.key) + (d.ties ? d.ties * wt0 : 0);
    if (top_p < 1.0f) {  // the token at which the sum in the row's order reaches P
        const uint64_t P = top_p > 0.0f ? (uint64_t)ceil((double)top_p * (double)total) : 0;
        const uint32_t k_key = d.key;
        const uint64_t k_ties = d.ties;
        uint64_t before = 0;
        uint32_t prefix = 0;
        for (int sft = 24; sft >= 0; sft -= 8) {
            __syncthreads();
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kDrawThreads) {
                const float l = lg_value(logits, f16, base + i);
                const uint32_t k = lg_key(l);
                if (k > k_key && (sft == 24 || (k >> (sft + 8)) == prefix))
                    atomicAdd((unsigned long long *)&hist[(k >> sft) & 255], (unsigned long long)dr_weight(d, l, bits));
            }
            __syncthreads();
            if (tid == 0) {
                if (k_ties && (sft == 24 || (k_key >> (sft + 8)) == prefix)) hist[(k_key >> sft) & 255] += k_ties * wt0;
                int b = 255;
                uint64_t at = before;
                // the largest key stands in the first bin that is not empty
                while (b > 0 && (hist[b] == 0 || at + hist[b] < P)) at += hist[b--];
                s_before = at;
                s_pick = b;
            }
            __syncthreads();
            before = s_before;
            prefix = prefix << 8 | (uint32_t)s_pick;
        }
        d.key = prefix;
        const uint64_t wt = dr_weight(d, lg_unkey(prefix), bits);
        uint64_t c = wt ? (P > before ? (P - before + wt - 1) / wt : 0) : 0;
        if (before == 0 && c == 0) c = 1;
        d.ties = prefix == k_key ? (c < k_ties ? c : k_ties) : tie_count(prefix, c);
        total = before + d.ties * wt;
    }
    // the draw, in index order: each wave holds a contiguous piece
    const uint64_t wt = dr_weight(d, lg_unkey(d.key), bits);
    float u = rnd[row];
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    uint64_t target = (uint64_t)((double)u * (double)total);
    if (target >= total) target = total - 1;
    const int seg = ((n + 16 * 64 - 1) / (16 * 64)) * 64;
    const int i0 = wave * seg;
    uint64_t sw = 0, sc = 0;
    for (int i = i0 + lane; i < min(n, i0 + seg); i += 64) {
        const float l = lg_value(logits, f16, base + i);
        const uint32_t k = lg_key(l);
        if (k > d.key) sw += dr_weight(d, l, bits);
        sc += k == d.key;
    }
    for (int s = 32; s; s >>= 1) sw += __shfl_xor(sw, s), sc += __shfl_xor(sc, s);
    __syncthreads();
    if (lane == 0) sh[wave] = sw, sh2[wave] = sc;
    __syncthreads();
    uint64_t cum = 0, tie = 0;
    for (int w = 0; w < wave; w++) {
        const uint64_t kept = tie < d.ties ? min((unsigned long long)sh2[w], (unsigned long long)(d.ties - tie)) : 0;
        cum += sh[w] + kept * wt;
        tie += sh2[w];
    }
    const uint64_t kept = tie < d.ties ? min((unsigned long long)sh2[wave], (unsigned long long)(d.ties - tie)) : 0;
    if (target < cum || target >= cum + sh[wave] + kept * wt) return;
    for (int i = i0; i < i0 + seg; i += 64) {
        const float l = i + lane < n ? lg_value(logits, f16, base + i + lane) : -INFINITY;
        const uint32_t k = lg_key(l);
        const bool same = i + lane < n && k == d.key;
        const uint64_t before_ties = tie + __popcll(__ballot(same) & ((1ull << lane) - 1));
        uint64_t w = k > d.key ? dr_weight(d, l, bits) : same && before_ties < d.ties ? wt : 0;
        uint64_t pre = w;
        for (int s = 1; s < 64; s <<= 1) {
            const uint64_t o = __shfl_up(pre, s);
            if (lane >= s) pre += o;
        }
        const uint64_t hit = __ballot(cum + pre > target);
        if (hit) {
            if (lane == __ffsll((long long)hit) - 1) {
                token[row] = i + lane;
                if (logp) {
                    const double z = l == d.m ? 0.0 : ((double)l - (double)d.m) / d.T;
                    logp[row] = (float)(z - log(ldexp((double)total, -bits)));
                }
            }
            return;
        }
        cum += __shfl(pre, 63);
        tie += __popcll(__ballot(same));
    }
}

int launch_draw(rsv_ctx *ctx, const void *logits, int f16, uint32_t *token, uint64_t n, const float *filter,
                const float *rnd, float *logp, float *, uint64_t rows) {
    int lg = 0;
    while ((1ull << lg) < n) lg++;
    hipLaunchKernelGGL(k_draw_row, dim3((unsigned)rows), dim3(kDrawThreads), 0, ctx->stream, logits, f16, (int)n, filter,
                       rnd, token, logp, 62 - lg);
    RSV_HIP(hipGetLastError());
    return 0;
}

// ------------------------------------------------- log-probabilities
// logp = (l[tok] - m) - ln(sum exp(l - m)); rank = tokens ahead of tok in the
// row's order (larger logit, or equal and a lower index).  One block a row.
__global__ __launch_bounds__(kDrawThreads) void k_logprob_row(const void *__restrict__ logits, int f16, int n,
                                                              const uint32_t *__restrict__ token,
                                                              float *__restrict__ logp, uint32_t *__restrict__ rank) {
    __shared__ float shf[16];
    __shared__ uint32_t shu[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x, base = row * n;
    const uint32_t tok = token[row];
    if (tok >= (uint32_t)n) {
        if (tid == 0) {
            logp[row] = 0.0f;
            if (rank) rank[row] = 0;
        }
        return;
    }
    const float lt = lg_value(logits, f16, base + tok);
    float m = -INFINITY;
    uint32_t ahead = 0;
    for (int i = tid; i < n; i += kDrawThreads) {
        const float l = lg_value(logits, f16, base + i);
        m = fmaxf(m, l);
        ahead += l > lt || (l == lt && i < (int)tok);
    }
    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (lane == 0) shf[wave] = m;
    ahead = block_sum(ahead, shu);
    for (int w = 0; w < 16; w++) m = fmaxf(m, shf[w]);
    float s = 0.0f;
    for (int i = tid; i < n; i += kDrawThreads) {
        const float l = lg_value(logits, f16, base + i);
        s += l == m ? 1.0f : expf(l - m);
    }
    __syncthreads();
    s = block_sum(s, shf);
    if (tid == 0) {
        logp[row] = lt == -INFINITY ? -INFINITY : (lt == m ? 0.0f : lt - m) - logf(s);
        if (rank) rank[row] = ahead;
    }
}

int launch_logprobs(rsv_ctx *ctx, const void *logits, int f16, const uint32_t *token, uint64_t n, float *logp,
                    uint32_t *rank, float *, uint64_t rows) {
    hipLaunchKernelGGL(k_logprob_row, dim3((unsigned)rows), dim3(kDrawThreads), 0, ctx->stream, logits, f16, (int)n,
                       token, logp, rank);
    RSV_HIP(hipGetLastError());
    return 0;
}

uint64_t logits_work_words(uint64_t, uint64_t) { return 0; }

}  // namespace rsv

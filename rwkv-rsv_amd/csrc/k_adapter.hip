// Low-rank adapters of many requests beside a shared projection
// (rsv_adapter_multi): out[t] = epi(y[t] + scale[a] * (x[t] A_a^T) B_a^T) with
// a = row_adapter[t], for a list of jobs over the same rows.
#include <algorithm>

#include "rsv_common.h"

namespace rsv {

__device__ __forceinline__ float ad_load(const void *p, int f16, size_t i) {
    return f16 ? (float)((const _Float16 *)p)[i] : ((const float *)p)[i];
}

// h[t, r] = sum_k x[t, k] A[a, r, k]: one block per (row, job), one wave per r.
__global__ __launch_bounds__(256) void k_adapter_down(AdapterJobs J) {
    const int t = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const AdapterJob &j = J.j[blockIdx.y];
    const uint32_t a = J.row_adapter[t];
    if (a >= (uint32_t)J.n_adapter) return;
    const int R = J.ranks ? (int)min(J.ranks[a], (uint32_t)J.rank) : J.rank;
    for (int r = wave; r < R; r += 4) {
        const _Float16 *w = j.a + ((size_t)a * J.rank + r) * j.k;
        float s = 0.0f;
        for (int k = lane; k < j.k; k += 64) s += ad_load(j.x, j.x16, (size_t)t * j.k + k) * (float)w[k];
        for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
        if (lane == 0) j.h[(size_t)t * J.rank + r] = s;
    }
}

// out[t, n] = epi(y[t, n] + scale * sum_r h[t, r] B[a, n, r]).
__global__ __launch_bounds__(256) void k_adapter_up(AdapterJobs J) {
    const int t = blockIdx.x;
    const AdapterJob &j = J.j[blockIdx.z];
    const int n = blockIdx.y * 256 + threadIdx.x;
    if (n >= j.n) return;
    const uint32_t a = J.row_adapter[t];
    const size_t at = (size_t)t * j.n + n;
    float z = ad_load(j.y, j.y16, at);
    if (a < (uint32_t)J.n_adapter) {
        const int R = J.ranks ? (int)min(J.ranks[a], (uint32_t)J.rank) : J.rank;
        const _Float16 *w = j.b + ((size_t)a * j.n + n) * J.rank;
        float s = 0.0f;
        for (int r = 0; r < R; r++) s += j.h[(size_t)t * J.rank + r] * (float)w[r];
        z += J.scale[a] * s;
    }
    if (j.epi == GE_RELU2) z = z > 0.0f ? z * z : z == z ? 0.0f : z;
    if (j.o16)
        ((_Float16 *)j.out)[at] = (_Float16)z;
    else
        ((float *)j.out)[at] = z;
}

uint64_t adapter_work_words(const rsv_adapter_job *, uint64_t njobs, uint64_t rank, uint64_t rows) {
    return njobs * rank * rows;
}

int launch_adapter(rsv_ctx *ctx, AdapterJobs &J, float *work) {
    int nmax = 0;
    for (int i = 0; i < J.njob; i++) {
        J.j[i].h = work + (size_t)i * J.rank * J.rows;
        nmax = std::max(nmax, J.j[i].n);
    }
    hipLaunchKernelGGL(k_adapter_down, dim3(J.rows, J.njob), dim3(256), 0, ctx->stream, J);
    hipLaunchKernelGGL(k_adapter_up, dim3(J.rows, (nmax + 255) / 256, J.njob), dim3(256), 0, ctx->stream, J);
    RSV_HIP(hipGetLastError());
    return 0;
}

}  // namespace rsv

// A projection with a low-rank adapter chosen per row (include/fortis_step.h, fortis_plan_linear_adapters):
//     Y[r] = act(X[r] W^T + b + s_i (X[r] A_i^T) U_i^T),  i = index[r], no adapter where i is outside [0, nadapt)
#include "common.h"

#define AD_THREADS 256

// H[r][j] = s_i X[r] . A_i[j]; rows without an adapter are not written.
__global__ __launch_bounds__(AD_THREADS) void adapt_low_simple_kernel(AdaptDesc d, const float* __restrict__ X, const int* __restrict__ index,
                                                                      float* __restrict__ H, long B)
{
    const long e = (long)blockIdx.x * AD_THREADS + threadIdx.x;
    if (e >= B * d.rank) return;
    const long r = e / d.rank, j = e % d.rank;
    const int i = index[r];
    if (i < 0 || i >= d.nadapt) return;
    const float *x = X + r * d.K, *a = d.A + ((long)i * d.rank + j) * d.K;
    float acc = 0.f;
    for (long k = 0; k < d.K; k++) acc = fmaf(x[k], a[k], acc);
    H[e] = acc * d.scale[i];
}
__global__ __launch_bounds__(AD_THREADS) void adapt_simple_kernel(AdaptDesc d, const float* __restrict__ X, const int* __restrict__ index,
                                                                  const float* __restrict__ H, float* __restrict__ Y, long B)
{
    const long e = (long)blockIdx.x * AD_THREADS + threadIdx.x;
    if (e >= B * d.N) return;
    const long r = e / d.N, n = e % d.N;
    const float *x = X + r * d.K, *w = d.W + n * d.K;
    float acc = 0.f;
    for (long k = 0; k < d.K; k++) acc = fmaf(x[k], w[k], acc);
    const int i = index[r];
    if (i >= 0 && i < d.nadapt) {
        const float *h = H + r * d.rank, *u = d.U + ((long)i * d.N + n) * d.rank;
        for (long j = 0; j < d.rank; j++) acc = fmaf(h[j], u[j], acc);
    }
    Y[e] = fortis_act_any(acc + (d.bias ? d.bias[n] : 0.f), d.act, d.alpha);
}

long fortis_adapters_workspace(const AdaptDesc& d, long B) { return B * d.rank * 4; }

void fortis_launch_linear_adapters(const AdaptDesc& d, const float* X, const int* index, float* Y, long B, void* ws, hipStream_t s)
{
    float* H = (float*)ws;
    hipLaunchKernelGGL(adapt_low_simple_kernel, dim3((unsigned)cdiv(B * d.rank, AD_THREADS)), dim3(AD_THREADS), 0, s, d, X, index, H, B);
    hipLaunchKernelGGL(adapt_simple_kernel, dim3((unsigned)cdiv(B * d.N, AD_THREADS)), dim3(AD_THREADS), 0, s, d, X, index, H, Y, B);
    HIP_OK(hipGetLastError());
}

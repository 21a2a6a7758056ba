// Group normalisation with an activation (include/fortis_step.h, fortis_plan_group_norm):
//     y = act(gamma_c (x - mean_{n,g}) / sqrt(var_{n,g} + eps) + beta_c)
// over the S * C / G values of every (sample, group), channels last or first.
#include "common.h"

#define GN_THREADS 256

// One workgroup per (sample, group), two reads of the input.  Sums are taken about the group's first value in float64.
__global__ __launch_bounds__(GN_THREADS) void norm_simple_kernel(NormDesc d, const float* __restrict__ x, float* __restrict__ y)
{
    __shared__ double red[2][GN_THREADS];
    const long n = blockIdx.x / d.G, g = blockIdx.x % d.G;
    const long cg = d.C / d.G, count = d.S * cg;
    auto at = [&](long e) {
        return d.first ? ((n * d.C + g * cg) * d.S + e) : ((n * d.S + e / cg) * d.C + g * cg + e % cg);
    };
    const float pivot = x[at(0)];
    double s1 = 0, s2 = 0;
    for (long e = threadIdx.x; e < count; e += GN_THREADS) {
        const double v = (double)x[at(e)] - (double)pivot;
        s1 += v; s2 += v * v;
    }
    red[0][threadIdx.x] = s1; red[1][threadIdx.x] = s2;
    __syncthreads();
    for (int o = GN_THREADS / 2; o; o >>= 1) {
        if ((int)threadIdx.x < o) { red[0][threadIdx.x] += red[0][threadIdx.x + o]; red[1][threadIdx.x] += red[1][threadIdx.x + o]; }
        __syncthreads();
    }
    const double dm = red[0][0] / (double)count, raw = red[1][0] / (double)count - dm * dm;
    const double var = raw < 0 ? 0 : raw;       // a NaN stays one
    const float rstd = (float)(1.0 / sqrt(var + (double)d.eps));
    for (long e = threadIdx.x; e < count; e += GN_THREADS) {
        const long a = at(e), c = g * cg + (d.first ? e / d.S : e % cg);
        const float v = (float)(((double)x[a] - (double)pivot) - dm) * rstd;
        y[a] = fortis_act_silu(fmaf(v, d.gamma ? d.gamma[c] : 1.f, d.beta ? d.beta[c] : 0.f), d.act, d.alpha);
    }
}

long fortis_norm_workspace(const NormDesc&) { return 0; }

void fortis_launch_group_norm(const NormDesc& d, const float* x, float* y, void*, hipStream_t s)
{
    hipLaunchKernelGGL(norm_simple_kernel, dim3((unsigned)(d.NB * d.G)), dim3(GN_THREADS), 0, s, d, x, y);
    HIP_OK(hipGetLastError());
}

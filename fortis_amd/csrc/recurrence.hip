// Gated linear recurrence (include/fortis_step.h, fortis_plan_recurrence):
//     f = 1 / (1 + exp(-g_t)),  h_t = f h_(t-1) + (1 - f) x_t
// per sequence and channel, rows of 2 * ch features (g first, x behind).
#include "common.h"

#define RC_THREADS 256

// (f, (1 - f) x) of one step; 1 - f as sigmoid(-g), which keeps its digits where f is close to 1.
__device__ __forceinline__ void rc_step(float g, float x, float& f, float& b)
{
    float hi, lo;
    fortis_sigmoids(g, hi, lo);
    f = g >= 0.f ? hi : lo;
    b = (g >= 0.f ? lo : hi) * x;
}

// One lane per (sequence, channel) walks its steps.
__global__ __launch_bounds__(RC_THREADS) void recurrence_simple_kernel(RecurDesc d, const float* __restrict__ src, float* __restrict__ dst,
                                                                       const float* h_in, float* h_out, const int* __restrict__ lengths)
{
    const long e = (long)blockIdx.x * RC_THREADS + threadIdx.x;
    if (e >= d.nseq * d.ch) return;
    const long s = e / d.ch, c = e % d.ch;
    long len = d.len;
    if (lengths) { const long l = lengths[s]; len = l < 0 ? 0 : l < len ? l : len; }
    float h = h_in ? h_in[e] : 0.f;
    for (long i = 0; i < len; i++) {
        const long t = d.reverse ? len - 1 - i : i, row = d.time_major ? t * d.nseq + s : s * d.len + t;
        float f, b;
        rc_step(src[row * 2 * d.ch + c], src[row * 2 * d.ch + d.ch + c], f, b);
        h = fmaf(f, h, b);
        dst[row * d.ch + c] = h;
    }
    if (h_out) h_out[e] = h;
}

long fortis_recurrence_workspace(const RecurDesc&) { return 0; }

void fortis_launch_recurrence(const RecurDesc& d, const float* src, float* dst, const float* h_in, float* h_out, const int* lengths, void*, hipStream_t s)
{
    hipLaunchKernelGGL(recurrence_simple_kernel, dim3((unsigned)cdiv(d.nseq * d.ch, RC_THREADS)), dim3(RC_THREADS), 0, s, d, src, dst, h_in, h_out, lengths);
    HIP_OK(hipGetLastError());
}

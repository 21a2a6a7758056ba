// Fused GEMM + bias + activation on the fp32 matrix cores:
//     C[B][N] = epi(A[B][K] . W[N][K]^T)
// One kernel replaces the reference's cuBLAS SGEMM (runtime/fortis_rt.c:45-75) AND the separate
// epilogue kernel fortis-fuse emits behind it (compiler/FortisFuse.cpp:685-692, 721-760: load C,
// add bias, activation, store), which re-reads and re-writes every activation once per layer.
//
// Tiling for CDNA4 (64-lane waves, v_mfma_f32_32x32x2f32, 4 SIMDs per CU):
//   workgroup tile 128 x 128 (halves and quarters of it at the tail of a launch), 256 threads =
//   4 waves in a 2 x 2 grid, each wave TM x TN MFMA tiles of 32 x 32; k is consumed in slabs of BK
//   staged through LDS, double buffered (global -> registers -> LDS while the previous slab is
//   multiplied).
//   Both operands are k-contiguous in memory (A row-major, W[N][K]), so both are staged the same
//   way, and a lane reads 4 consecutive k as one 16-byte LDS load that feeds 4 MFMAs: MFMA step s
//   of an 8-wide k group uses k = 4h + s for lane half h, identically for A and B.
//   LDS rows are padded by 4 floats so the 16-byte reads of consecutive rows fall in different banks.
#include "gemm_dev.h"

// Persistent kernel: the grid is exactly the number of workgroups the chip holds at once (slots), and
// every workgroup walks the phases taking item (round * slots + its place).  Whole rounds of full
// blocks come first; what is left over is cut into halves and quarters so that the last rounds still
// give every workgroup (hence every CU) the same amount of work -- with plain one-tile-per-workgroup
// launches a 1.5-round problem costs 2 rounds.
// Within a round the places are numbered so that each XCD (workgroup id mod 8) gets a contiguous band
// of items: the band's A rows and all of W stay in that XCD's L2.
template <int GM_BK>
__global__ __launch_bounds__(GM_THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) void gemm_kernel(const float* __restrict__ A, const float* __restrict__ W,
                                                          float* __restrict__ C, long B, long N, long K,
                                                          GemmSched sc, GemmEpi epi)
{
    extern __shared__ float4 smem4[];
    float* smem = (float*)smem4;
    const long w = blockIdx.x;
    for (int p = 0; p < sc.nphase; p++) {
        const int level = sc.ph[p].level;
        const long base = sc.ph[p].base, count = sc.ph[p].count;
        if (level == 0) {
            // whole rounds: count is a multiple of slots, this workgroup's place is the same in each
            const long place = (w & 7) * (sc.slots / 8) + (w >> 3);
            const long rounds = count / sc.slots;
            v4f ra[2 * GM_BK / 16], rw[2 * GM_BK / 16];
            for (long r = 0; r < rounds; r++) {
                const long tile = base + r * sc.slots + place, next = tile + sc.slots;
                const long tm = tile / sc.tiles_n, tn = tile - tm * sc.tiles_n;
                const long tmn = next / sc.tiles_n, tnn = next - tmn * sc.tiles_n;
                gemm_tile<2, 2, GM_BK, GemmPlain>(A, W, C, B, N, K, tm * 128, tn * 128, epi, smem, ra, rw,
                                       r > 0, r + 1 < rounds, tmn * 128, tnn * 128, GemmPlain());
            }
            continue;
        }
        // a partial round of halves or quarters
        const long per_xcd = (count + 7) / 8;
        if ((w >> 3) >= per_xcd) continue;
        const long item = (w & 7) * per_xcd + (w >> 3);
        if (item >= count) continue;
        const long tile = base + (level == 1 ? (item >> 1) : (item >> 2));
        const long tm = tile / sc.tiles_n, tn = tile - tm * sc.tiles_n;
        if (level == 1) {
            const long m0 = tm * 128, n0 = tn * 128 + (item & 1) * 64;
            if (m0 >= B || n0 >= N) continue;
            v4f ra[2 * GM_BK / 16], rw[GM_BK / 16];
            gemm_tile<2, 1, GM_BK, GemmPlain>(A, W, C, B, N, K, m0, n0, epi, smem, ra, rw, false, false, 0, 0, GemmPlain());
        } else {
            const long m0 = tm * 128 + ((item >> 1) & 1) * 64, n0 = tn * 128 + (item & 1) * 64;
            if (m0 >= B || n0 >= N) continue;
            v4f ra[GM_BK / 16], rw[GM_BK / 16];
            gemm_tile<1, 1, GM_BK, GemmPlain>(A, W, C, B, N, K, m0, n0, epi, smem, ra, rw, false, false, 0, 0, GemmPlain());
        }
    }
}

// Small batches (B <= 16; the reference's generated warp-per-output kernel for batch < 32,
// compiler/FortisFuse.cpp:667-719): one wave per output column n.  The lanes stride over k with 16-byte
// loads of W[n][:] (1 KiB per wave per step, fully coalesced) and of the few A rows (the same for every
// wave: served by the caches), then the 64 partial sums are folded with a shuffle tree.  Memory-bound on
// reading W once; a 128 x 128 MFMA tile would be 1 % useful.
template <int BR>
__global__ __launch_bounds__(256) void gemm_small_kernel(const float* __restrict__ A, const float* __restrict__ W,
                                                         float* __restrict__ C, int B, long N, long K, GemmEpi epi)
{
    const int lane = threadIdx.x & 63;
    const long n = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= N) return;
    float acc[BR];
#pragma unroll
    for (int r = 0; r < BR; r++) acc[r] = 0.f;
    const float* wrow = W + n * K;
    for (long k0 = lane * 4; k0 < K; k0 += 256) {
        const v4f w = *(const v4f*)(wrow + k0);
#pragma unroll
        for (int r = 0; r < BR; r++) {
            const v4f a = *(const v4f*)(A + (long)(r < B ? r : 0) * K + k0);
            acc[r] = fmaf(w.w, a.w, fmaf(w.z, a.z, fmaf(w.y, a.y, fmaf(w.x, a.x, acc[r]))));
        }
    }
#pragma unroll
    for (int r = 0; r < BR; r++)
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) acc[r] += __shfl_xor(acc[r], off, 64);
    if (lane == 0) {
        const float bv = epi.bias ? epi.bias[n] : 0.f;
#pragma unroll
        for (int r = 0; r < BR; r++) {
            if (r >= B) break;
            float v = gemm_act(acc[r] + bv, epi.act, epi.alpha);
            if (epi.out_scale) v = v * epi.out_scale[n];
            if (n >= epi.mask_from) v = v > 0.f ? v : 0.f;
            C[(long)r * N + n] = v;
        }
    }
}

// Generic guarded fallback for K not a multiple of 4 (16-byte row loads impossible): one thread
// per output element, fp32 FMA chain.  Correct for any shape; not a fast path.
__global__ void gemm_naive_kernel(const float* __restrict__ A, const float* __restrict__ W, float* __restrict__ C,
                                  long B, long N, long K, GemmEpi epi)
{
    const long idx = (long)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx >= B * N) return;
    const long m = idx / N, n = idx - m * N;
    float acc = 0.f;
    for (long k = 0; k < K; k++) acc = fmaf(A[m * K + k], W[n * K + k], acc);
    float v = gemm_act(acc + (epi.bias ? epi.bias[n] : 0.f), epi.act, epi.alpha);
    if (epi.out_scale) v = v * epi.out_scale[n];
    if (n >= epi.mask_from) v = v > 0.f ? v : 0.f;
    C[idx] = v;
}

// Test hook: the schedule as (level, first tile, items) triples; returns the number of phases.
extern "C" int fortis_gemm_schedule(long B, long N, long slots, long* triples)
{
    if (B <= 0 || N <= 0 || slots < 8 || slots % 8) return -1;
    GemmSched sc;
    gemm_make_sched(B, N, slots, &sc);
    for (int p = 0; p < sc.nphase; p++) { triples[3 * p] = sc.ph[p].level; triples[3 * p + 1] = sc.ph[p].base; triples[3 * p + 2] = sc.ph[p].count; }
    return sc.nphase;
}

// slots = workgroups resident at once (occupancy x CUs), a multiple of 8
template <int BK>
static void launch_tiled(const float* A, const float* W, float* C, long B, long N, long K, const GemmEpi& epi, hipStream_t s)
{
    const size_t shmem = (size_t)2 * (128 + 128) * (BK + 4) * sizeof(float);
    static long slots = 0;
    if (!slots) {
        HIP_OK(hipFuncSetAttribute((const void*)gemm_kernel<BK>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shmem));
        int occ = 0, dev = 0;
        hipDeviceProp_t prop;
        HIP_OK(hipGetDevice(&dev));
        HIP_OK(hipGetDeviceProperties(&prop, dev));
        HIP_OK(hipOccupancyMaxActiveBlocksPerMultiprocessor(&occ, (const void*)gemm_kernel<BK>, GM_THREADS, shmem));
        if (occ < 1) occ = 1;
        slots = (long)occ * prop.multiProcessorCount / 8 * 8;
        if (slots < 8) slots = 8;
    }
    GemmSched sc;
    gemm_make_sched(B, N, slots, &sc);
    long items = 0;
    for (int p = 0; p < sc.nphase; p++) items = sc.ph[p].count > items ? sc.ph[p].count : items;
    const long grid = items < slots ? cdiv(items, 8) * 8 : slots;
    hipLaunchKernelGGL((gemm_kernel<BK>), dim3((unsigned)grid), dim3(GM_THREADS), shmem, s, A, W, C, B, N, K, sc, epi);
    HIP_OK(hipGetLastError());
}

int fortis_launch_gemm(const float* A, const float* W, const float* bias, float* C, long B, long N, long K,
                       int act, float alpha, const float* out_scale, long mask_tail, hipStream_t s)
{
    if (B <= 0 || N <= 0 || K <= 0) return -1;
    GemmEpi epi = { bias, out_scale, act, alpha, mask_tail > 0 ? N - mask_tail : N };
    const bool vec_ok = (K % 4 == 0) && K < (1L << 22) && N < (1L << 24) && (((uintptr_t)A | (uintptr_t)W) % 16 == 0);
    if (!vec_ok) {
        hipLaunchKernelGGL(gemm_naive_kernel, dim3((unsigned)cdiv(B * N, 256)), dim3(256), 0, s, A, W, C, B, N, K, epi);
        HIP_OK(hipGetLastError());
        return 0;
    }
    if (B <= 16) {
        const dim3 grid((unsigned)cdiv(N, 4)), block(256);
        if (B == 1) hipLaunchKernelGGL(gemm_small_kernel<1>, grid, block, 0, s, A, W, C, (int)B, N, K, epi);
        else if (B <= 4) hipLaunchKernelGGL(gemm_small_kernel<4>, grid, block, 0, s, A, W, C, (int)B, N, K, epi);
        else hipLaunchKernelGGL(gemm_small_kernel<16>, grid, block, 0, s, A, W, C, (int)B, N, K, epi);
        HIP_OK(hipGetLastError());
        return 0;
    }
    static int bk = 0;
    if (!bk) { const char* e = getenv("FORTIS_GEMM_BK"); bk = (e && atoi(e) == 16) ? 16 : 32; }
    if (bk == 16) launch_tiled<16>(A, W, C, B, N, K, epi, s);
    else launch_tiled<32>(A, W, C, B, N, K, epi, s);
    return 0;
}

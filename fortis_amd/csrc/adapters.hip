// A projection with a low-rank adapter chosen per row (include/fortis_step.h, fortis_plan_linear_adapters):
//     Y[r] = act(X[r] W^T + b + s_i (X[r] A_i^T) U_i^T),  i = index[r], no adapter where i is outside [0, nadapt)
// fp32 throughout, sums on the fp32 matrix instructions.
//
// Few rows (up to AD_FEW_ROWS): bound by latency and by reading W and the named adapters once.  One launch forms the
// low-rank rows H[r] = s_i X[r] A_i^T with a wave per row and four ranks, a second the outputs: a workgroup owns 16 rows
// by 16 columns and its eight waves divide K, so that all of a wave's loads are in flight at once.
//
// Narrow layers (K and N up to 64, ranks up to 16): bound by reading X and writing Y.  One launch does it all: W lies in LDS, a wave
// takes 16 rows at a time from X to Y.
//
// Many rows: bound by the matrix pipes.  Rows are sorted by adapter inside windows of AD_WINDOW rows (one launch), H is
// formed for 16 sorted rows at a time, and the GEMM tile of gemm.hip runs over the sorted rows: a row of A is found through
// the permutation, and behind the k loop each wave adds, per 32 rows and adapter among them, H U_i^T with the H of other
// adapters' rows as zeros.  Sorted rows leave one or two adapters to a block of 32; rows that were not sorted would leave up to
// 32.  A window keeps a tile's rows and the rows it writes within a few megabytes of each other.  Sorting places equal
// adapters in any order: a row's sums do not depend on its place.
#include "gemm_dev.h"

#define AD_THREADS 256
#define AD_WINDOW 2048          // rows sorted together; a multiple of the tile's 128
// Few rows against sorted ones, us at rank 16, 8 / 64 adapters:
//   K = N = 256     512 rows 12.5 : 23 / 12.4 : 32      1024 rows 20 : 23 / 19 : 27
//   K = N = 768     512 rows 25 : 33 / 25 : 39          1024 rows 44 : 34 / 45 : 38
//   K = N = 2048    256 rows 74 : 73 / 75 : 115         512 rows 140 : 74 / 143 : 95      1024 rows 273 : 97 / 277 : 107
// The limit holds for K = N = 256.  Wider layers would change over sooner, as W is read again for every 16 rows: between 512 and
// 1024 rows at 768, at 256 rows at 2048.
#define AD_FEW_ROWS 1024

static inline long up(long n, long m) { return (n + m - 1) / m * m; }

// ---- weights, laid out once --------------------------------------------------------------------------------------
// W [N][ldw], A [nadapt][R16][Ka], U [nadapt][N][Rp], padded with zeros.
// Where one launch pays, us for the narrow form / the others: 24576 rows of 64 -> 64, rank 8 with 8 adapters in any order 18 / 31 (sorted
// rows), 27 -> 64 13 / 32, but 128 -> 128 41 / 37 and 128 -> 128 with rank 64 and 24 adapters 207 / 84 (every adapter among 16 rows is a
// product of its own); 500 rows of 128 -> 128 24 / 9 (few rows).
#define NARROW_K 64
#define NARROW_N 64
#define NARROW_RANK 16
AdaptPitch fortis_adapters_pitch(long K, long N, long rank, bool finite)
{
    // (an adapter with an infinity or a NaN in U would reach other rows through 0 times U in all forms but the few-rows one)
    const int narrow = finite && K <= NARROW_K && N <= NARROW_N && rank <= NARROW_RANK;
    return { up(K, 4), up(K, 16), up(rank, 16), up(rank, narrow ? 16 : 8), narrow, finite };
}
// Where rank j of a row of U lies: in order, but 4 x 4 transposed within sixteen for the narrow form, whose instruction c then
// multiplies ranks 4 c .. 4 c + 3 and which leaves out the instructions behind the last rank.
// (H of the few-rows form lies alike.)
__host__ __device__ __forceinline__ static int adapt_place(int narrow, int j) { return narrow ? j / 16 * 16 + j % 4 * 4 + j % 16 / 4 : j; }
long fortis_adapters_place(const AdaptPitch& p, long j) { return adapt_place(p.narrow, (int)j); }

// Elements k .. k + 3 of a row of K floats at p; what lies at or beyond K is 0.  How rows lie: ROW4 K is a multiple of 4; ROWANY
// rows start at any float and K is at least 4: the 16 bytes are loaded where they are; ROWTINY K < 4.
enum { ROW4 = 0, ROWANY = 1, ROWTINY = 2 };
template <int ROW> __device__ __forceinline__ v4f load_row4(const float* p, long k, long K)
{
    if constexpr (ROW == ROWANY) return shift_row4(*(const v4f_any*)(p + (k <= K - 4 ? k : K - 4)), k, K);
    v4f v;
    if constexpr (ROW == ROWTINY) {
#pragma unroll
        for (int c = 0; c < 4; c++) { const float t = p[k + c < K ? k + c : K - 1]; v[c] = k + c < K ? t : 0.f; }
    } else {
        v = *(const v4f*)(p + (k < K ? k : 0));
        if (k >= K) v = (v4f)(0.f);
    }
    return v;
}

// ---- few rows ----------------------------------------------------------------------------------------------------
// H[r][4 q .. 4 q + 3], one wave each: lanes stride over k.  48 rows of 768 with rank 16 (2.5 MB): 3.9 us, the launch and one
// round of loads.
template <int ROW>
__global__ __launch_bounds__(AD_THREADS) void adapt_low_rows_kernel(AdaptDesc d, const float* __restrict__ X, const int* __restrict__ index,
                                                                    float* __restrict__ H, long B)
{
    const int lane = threadIdx.x & 63;
    const long quads = d.p.Rp / 4, id = (long)blockIdx.x * (AD_THREADS / 64) + (threadIdx.x >> 6);
    if (id >= B * quads) return;
    const long r = id / quads, q = id - r * quads;
    const int i = index[r];
    if (i < 0 || i >= d.nadapt) return;
    const float* x = X + r * d.K;
    const float* a = d.A + ((long)i * d.p.R16 + 4 * q) * d.p.Ka;
    float s[4] = { 0.f, 0.f, 0.f, 0.f };
    for (long k = lane * 4; k < d.p.Ka; k += 256) {
        const v4f xv = load_row4<ROW>(x, k, d.K);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const v4f av = *(const v4f*)(a + j * d.p.Ka + k);
            s[j] = fmaf(xv[3], av[3], fmaf(xv[2], av[2], fmaf(xv[1], av[1], fmaf(xv[0], av[0], s[j]))));
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) s[j] += __shfl_xor(s[j], o, 64);
    if (lane < 4) {
        const float v = lane == 0 ? s[0] : lane == 1 ? s[1] : lane == 2 ? s[2] : s[3];
        H[r * d.p.Rp + adapt_place(d.p.narrow, (int)(4 * q) + lane)] = 4 * q + lane < d.rank ? v * d.scale[i] : 0.f;
    }
}

// 16 rows x 16 columns of Y; wave w takes the 16-wide k groups w, w + 8, ...  A lane reads four consecutive k of a row of X
// and of W as one 16-byte load each and feeds four matrix instructions: instruction c multiplies k = 16 g + 4 q + c for lane
// quarter q on both sides.
// One row of 768 -> 768: 5.7 us (2.4 MB of W at 0.42 TB/s: one launch's start, the loads and a join); 48 rows with the launch in front
// 9.8 us, 7.4 MB at 0.75 TB/s.
// What the outputs' adapters add is formed while those loads travel.  FUSED (a few products at most, FEW_FUSED): every
// workgroup forms H of its rows itself, one product a wave at a time, and the launch in front is not needed.
#define FEW_WAVES 8
#define FEW_FUSED 32            // rows x ranks
template <int ROW, bool FUSED>
__global__ __launch_bounds__(64 * FEW_WAVES) void adapt_few_kernel(AdaptDesc d, const float* __restrict__ X, const int* __restrict__ index,
                                                                   const float* __restrict__ H, float* __restrict__ Y, long B)
{
    __shared__ float part[FEW_WAVES][16][17];
    __shared__ __attribute__((aligned(16))) float sH[FUSED ? FEW_FUSED : 4];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, lr = lane & 15, lq = lane >> 4;
    const unsigned tn = (unsigned)(d.N + 15) / 16;
    const long m0 = (long)(blockIdx.x / tn) * 16, n0 = (long)(blockIdx.x % tn) * 16;
    // this thread's output (the first 256 threads)
    const long m = m0 + t / 16, n = n0 + t % 16;
    const bool out = t < 256 && m < B && n < d.N;
    int i = out ? index[m] : -1;
    const float bias = out && d.bias ? d.bias[n] : 0.f;
    const float* x = X + (m0 + lr < B ? m0 + lr : B - 1) * d.K;
    const float* w = d.W + (n0 + lr < d.N ? n0 + lr : d.N - 1) * d.p.ldw;
    const int groups = (int)d.p.Ka / 16, Rp = (int)d.p.Rp;
    constexpr int AHEAD = 6;
    v4f xv[AHEAD], wv[AHEAD];
    auto fetch = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const int k = (g + u * FEW_WAVES) * 16 + 4 * lq;
            xv[u] = load_row4<ROW>(x, k, d.K);
            wv[u] = load_row4<ROW4>(w, k, d.p.ldw);
        }
    };
    fetch(wave);
    if constexpr (FUSED) {
        for (int e = wave; e < (int)B * Rp; e += FEW_WAVES) {
            const int r = e / Rp, j = e - r * Rp, a = index[r];
            float s = 0.f;
            if (a >= 0 && a < d.nadapt && j < d.rank) {
                const float *xr = X + r * d.K, *ar = d.A + ((long)a * d.p.R16 + j) * d.p.Ka;
                for (int k = lane * 4; k < (int)d.p.Ka; k += 256) {
                    const v4f p = load_row4<ROW>(xr, k, d.K), q = *(const v4f*)(ar + k);
                    s = fmaf(p[3], q[3], fmaf(p[2], q[2], fmaf(p[1], q[1], fmaf(p[0], q[0], s))));
                }
                s *= d.scale[a];
#pragma unroll
                for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
            }
            if (lane == 0) sH[r * Rp + adapt_place(d.p.narrow, j)] = s;
        }
    }
    if (i >= d.nadapt) i = -1;
    const float* u = d.U + ((long)(i < 0 ? 0 : i) * d.N + n) * Rp;
    float low = 0.f;
    if (!FUSED && i >= 0) {
        const float* h = H + m * Rp;
        for (int j = 0; j < Rp; j += 4) {
            const v4f hv = *(const v4f*)(h + j), uv = *(const v4f*)(u + j);
            low = fmaf(hv[3], uv[3], fmaf(hv[2], uv[2], fmaf(hv[1], uv[1], fmaf(hv[0], uv[0], low))));
        }
    }
    v4f acc = (v4f)(0.f);
    for (int g = wave; g < groups; g += FEW_WAVES * AHEAD) {
        if (g > wave) fetch(g);
#pragma unroll
        for (int u = 0; u < AHEAD; u++)
#pragma unroll
            for (int c = 0; c < 4; c++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[u][c], wv[u][c], acc, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; r++) part[wave][4 * lq + r][lr] = acc[r];
    __syncthreads();
    if (!out) return;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < FEW_WAVES; k++) v += part[k][t / 16][t % 16];
    if (FUSED && i >= 0) {
        const float* h = sH + m * Rp;
        for (int j = 0; j < Rp; j += 4) {
            const v4f hv = *(const v4f*)(h + j), uv = *(const v4f*)(u + j);
            low = fmaf(hv[3], uv[3], fmaf(hv[2], uv[2], fmaf(hv[1], uv[1], fmaf(hv[0], uv[0], low))));
        }
    }
    Y[m * d.N + n] = fortis_act_any(v + low + bias, d.act, d.alpha);
}

// ---- narrow layers -----------------------------------------------------------------------------------------------
// A wave owns 16 rows: their X as KG operands of four k (k = 16 g + 4 q + c, as above).  Per adapter among the rows: all
// are multiplied with its A, the products change places through the wave's own piece of LDS into
// operands of the second product, where those of other adapters' rows are zeros.  Loads of X start before W is brought to LDS.
// 71040 rows of 27 -> 64 with 15 adapters of rank 4 in bands (26 MB): 13.0 us, 2.0 TB/s, bound by a wave's chain of loads, two products
// and the way through LDS between them, and by a second round: 1110 workgroups, of which 1024 are resident (106 registers); 32 rows
// a wave gain 0.3 us there and lose where neighbours' adapters differ, adapter operands loaded a block of rows ahead cost 1.6.
#define NARROW_WAVE_FLOATS(KG, SC) (16 * 20 + ((SC) ? 16 * (16 * (KG) + 4) : 0))
template <int KG, int NT, bool SC>
__global__ __launch_bounds__(AD_THREADS, 3) void adapt_narrow_kernel(AdaptDesc d, const float* __restrict__ X, const int* __restrict__ index,
                                                                  float* __restrict__ Y, long B, FastDiv byK)
{
    extern __shared__ float4 smem4[];
    constexpr int LDW = 16 * KG + 4, ROWS = 16;
    float* sW = (float*)smem4;                                                                 // [16 NT][LDW]
    float* sH = sW + 16 * NT * LDW + (threadIdx.x >> 6) * NARROW_WAVE_FLOATS(KG, SC);      // [ROWS][20] for this wave
    float* sX = sH + ROWS * 20;                                                                // SC: [ROWS][LDW], zeros behind K
    const int lane = threadIdx.x & 63, lr = lane & 15, lq = lane >> 4;
    const int K = (int)d.K, N = (int)d.N;
    const long step = (long)gridDim.x * (AD_THREADS / 64) * ROWS;
    long m0 = ((long)blockIdx.x * (AD_THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * ROWS;
    v4f xv[KG];
    int i = -1;                                                                                // adapter of row lane % 16
    auto fetch = [&](long m) __attribute__((always_inline)) {
        const int n = B - m < ROWS ? (int)(B - m) : ROWS, row = lane & (ROWS - 1);
        i = row < n ? index[m + row] : -1;
        const float* p = X + m * K;
        if constexpr (SC) {
            // the rows' floats in the order of memory, whatever K is
#pragma unroll
            for (int u = 0; u < 4 * KG; u++) {
                const int e = lane + 64 * u;
                xv[u / 4][u % 4] = p[e < n * K ? e : n * K - 1];
            }
        } else {
#pragma unroll
            for (int g = 0; g < KG; g++) xv[g] = load_row4<ROW4>(p + (lr < n ? lr : n - 1) * K, 16 * g + 4 * lq, K);
        }
    };
    if (m0 < B) fetch(m0);
    if constexpr (SC) {
        for (int e = lane; e < ROWS * LDW; e += 64) sX[e] = 0.f;
    }
    float bv[NT];
    int ucol[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        bv[t] = d.bias && 16 * t + lr < N ? d.bias[16 * t + lr] : 0.f;
        ucol[t] = (16 * t + lr < N ? 16 * t + lr : N - 1) * (int)d.p.Rp + 4 * lq;
    }
    for (int e = threadIdx.x; e < 16 * NT * 4 * KG; e += AD_THREADS) {
        const int n = e / (4 * KG), k = e % (4 * KG) * 4;
        *(v4f*)(sW + n * LDW + k) = load_row4<ROW4>(d.W + (n < N ? n : N - 1) * d.p.ldw, k, d.p.ldw);
    }
    __syncthreads();
    auto turn = [&]() __attribute__((always_inline)) {         // the wave's LDS writes before its reads
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    while (m0 < B) {
        v4f acc[NT];
        if (i >= d.nadapt) i = -1;
        unsigned live = (unsigned)__ballot(i >= 0) & (unsigned)((1ull << ROWS) - 1);
        if constexpr (SC) {
#pragma unroll
            for (int u = 0; u < 4 * KG; u++) {
                const unsigned e = lane + 64 * u, r = fortis_div(e, byK);
                if (e < (unsigned)(ROWS * K)) sX[r * LDW + e - r * K] = xv[u / 4][u % 4];
            }
            turn();
#pragma unroll
            for (int g = 0; g < KG; g++) xv[g] = *(const v4f*)(sX + lr * LDW + 16 * g + 4 * lq);
            __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (int t = 0; t < NT; t++) acc[t] = (v4f)(0.f);
#pragma unroll
        for (int g = 0; g < KG; g++)
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const v4f w = *(const v4f*)(sW + (16 * t + lr) * LDW + 16 * g + 4 * lq);
#pragma unroll
                for (int c = 0; c < 4; c++) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[g][c], w[c], acc[t], 0, 0, 0);
            }
        while (live) {
            const int a = __builtin_amdgcn_readlane(i, __builtin_ctz(live));
            const unsigned rows = (unsigned)__ballot(i == a) & (unsigned)((1ull << ROWS) - 1);
            live &= ~rows;
            const float sc = d.scale[a];
            const int rank = (int)d.rank;
            const float* A = d.A + (long)a * d.p.R16 * d.p.Ka;                                  // uniform
            const float* U = d.U + (long)a * N * d.p.Rp;
            v4f h = (v4f)(0.f), av[KG], uv[NT];
#pragma unroll
            for (int g = 0; g < KG; g++) av[g] = 16 * g < d.p.Ka ? *(const v4f*)(A + lr * (int)d.p.Ka + 4 * lq + 16 * g) : (v4f)(0.f);
#pragma unroll
            for (int t = 0; t < NT; t++) uv[t] = *(const v4f*)(U + ucol[t]);
#pragma unroll
            for (int g = 0; g < KG; g++)
#pragma unroll
                for (int c = 0; c < 4; c++) h = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[g][c], av[g][c], h, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; r++) sH[(4 * lq + r) * 20 + lr] = h[r] * sc;
            turn();
#pragma unroll
            for (int c = 0; c < 4; c++) {
                if (4 * c >= rank) break;
                const float hv = sH[lr * 20 + 4 * c + lq];
                const float hc = (rows >> lr) & 1 && 4 * c + lq < rank ? hv : 0.f;
#pragma unroll
                for (int t = 0; t < NT; t++) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(hc, uv[t][c], acc[t], 0, 0, 0);
            }
            __builtin_amdgcn_wave_barrier();
        }
        float* y = Y + m0 * N;                                                                 // uniform
        const int n = B - m0 < ROWS ? (int)(B - m0) : ROWS;
        m0 += step;
        if (m0 < B) fetch(m0);
        const float alpha = d.alpha;
        fortis_with_act(d.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int m = 4 * lq + r;
                if (m >= n) continue;
                float* row = y + m * N + lr;
#pragma unroll
                for (int t = 0; t < NT; t++)
                    if (16 * t + lr < N) row[16 * t] = fortis_act_any(acc[t][r] + bv[t], decltype(act)::value, alpha);
            }
        });
    }
}
template <int KG, int NT, bool SC>
static void launch_narrow(const AdaptDesc& d, const float* X, const int* index, float* Y, long B, hipStream_t s)
{
    const size_t shmem = (size_t)(16 * NT * (16 * KG + 4) + (AD_THREADS / 64) * NARROW_WAVE_FLOATS(KG, SC)) * 4;
    static bool set = false;
    if (!set) { HIP_OK(hipFuncSetAttribute((const void*)adapt_narrow_kernel<KG, NT, SC>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shmem)); set = true; }
    const long wgs = cdiv(B, 16 * (AD_THREADS / 64));
    hipLaunchKernelGGL((adapt_narrow_kernel<KG, NT, SC>), dim3((unsigned)(wgs < 2048 ? wgs : 2048)), dim3(AD_THREADS), shmem, s, d, X, index, Y, B, fortis_fast_div((unsigned)d.K));
}
template <int KG, bool SC>
static void narrow_by_columns(const AdaptDesc& d, const float* X, const int* index, float* Y, long B, hipStream_t s)
{
    if (d.N <= 16) launch_narrow<KG, 1, SC>(d, X, index, Y, B, s);
    else if (d.N <= 32) launch_narrow<KG, 2, SC>(d, X, index, Y, B, s);
    else launch_narrow<KG, 4, SC>(d, X, index, Y, B, s);
}

// ---- many rows ---------------------------------------------------------------------------------------------------
// Rows of a window in order of their adapter, those without one behind: perm[p] = row inside the window, key[p] = its
// adapter or -1.  A counting sort in LDS, one workgroup a window: 4.7 us whether 3 windows or 12, its barriers and atomics in
// turn (rows of one adapter 1.5 us more when they were counted a second time instead of keeping what the first count returned).
__global__ __launch_bounds__(1024) void adapt_sort_kernel(const int* __restrict__ index, int* __restrict__ perm, int* __restrict__ key, long B, int nadapt)
{
    extern __shared__ int bin[];        // [nadapt + 1], then 16 wave sums
    const int tid = threadIdx.x, bins = nadapt + 1;
    int* wsum = bin + bins;
    const long r0 = (long)blockIdx.x * AD_WINDOW;
    for (int b = tid; b < bins; b += 1024) bin[b] = 0;
    __syncthreads();
    int mine[AD_WINDOW / 1024], place[AD_WINDOW / 1024];      // bin, and how many of the bin came before
#pragma unroll
    for (int k = 0; k < AD_WINDOW / 1024; k++) {
        const long r = r0 + tid + k * 1024;
        mine[k] = -1;
        if (r < B) {
            const int i = index[r];
            mine[k] = i >= 0 && i < nadapt ? i : nadapt;
            place[k] = atomicAdd(&bin[mine[k]], 1);
        }
    }
    __syncthreads();
    // exclusive sums of the bins: `per` neighbouring bins a thread
    const int per = (bins + 1023) / 1024, b0 = tid * per;
    int sum = 0;
    for (int b = b0; b < b0 + per && b < bins; b++) sum += bin[b];
    int run = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int t = __shfl_up(run, o, 64); if ((tid & 63) >= o) run += t; }
    if ((tid & 63) == 63) wsum[tid >> 6] = run;
    __syncthreads();
    int before = run - sum;
    for (int w = 0; w < (tid >> 6); w++) before += wsum[w];
    for (int b = b0; b < b0 + per && b < bins; b++) { const int t = bin[b]; bin[b] = before; before += t; }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < AD_WINDOW / 1024; k++) {
        if (mine[k] < 0) continue;
        const int p = bin[mine[k]] + place[k];
        perm[r0 + p] = tid + k * 1024;
        key[r0 + p] = mine[k] < nadapt ? mine[k] : -1;
    }
}

// H of 16 sorted rows: KS waves divide the 16-wide k groups, 16 ranks at a time; per adapter among the rows all 16 are
// multiplied with its A and its own rows kept.  Bound by reading X, and by how many loads a compute unit holds: 24576 rows of 768 with 24
// adapters of rank 16 (75 MB) 24 us behind the sort, 3.1 TB/s; with 32 rows a workgroup 27, and
// 4099 rows of 556 9 instead of 7.5 (but 8192 x 2048 -> 512 with rank 32, whose X is read once per 16 ranks, 207 us in all instead of 220).
#define LOW_ROWS 16
template <int KS, bool SC>
__global__ __launch_bounds__(64 * KS) void adapt_low_sorted_kernel(AdaptDesc d, const float* __restrict__ X, const int* __restrict__ perm,
                                                                      const int* __restrict__ key, float* __restrict__ H, long B)
{
    __shared__ float part[KS][LOW_ROWS][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lq = lane >> 4;
    const long p0 = (long)blockIdx.x * LOW_ROWS, base = p0 / AD_WINDOW * AD_WINDOW;
    const int kk = lane < LOW_ROWS && p0 + lane < B ? key[p0 + lane] : -1;
    const float* x = X + (base + perm[p0 + lr < B ? p0 + lr : B - 1]) * d.K;
    const int groups = (int)d.p.Ka / 16;
    constexpr int AHEAD = 6;
    v4f xv[AHEAD];
    auto fetch = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const int k = (g + u * KS) * 16 + 4 * lq;
            xv[u] = load_row4<SC ? ROWANY : ROW4>(x, k, d.K);
        }
    };
    // rows that one set of loads holds whole are read once for all their adapters
    const bool whole = groups <= KS * AHEAD;
    unsigned live = (unsigned)__ballot(kk >= 0);
    if (whole && live) fetch(wave);
    while (live) {
        const int a = __builtin_amdgcn_readlane(kk, __builtin_ctz(live));
        const unsigned rows = (unsigned)__ballot(kk == a);
        live &= ~rows;
        const float sc = d.scale[a];
        for (long j0 = 0; j0 < d.rank; j0 += 16) {
            const float* w = d.A + ((long)a * d.p.R16 + j0 + lr) * d.p.Ka;
            v4f acc = (v4f)(0.f);
            for (int g = wave; g < groups; g += KS * AHEAD) {
                v4f wv[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; u++) wv[u] = load_row4<ROW4>(w, (g + u * KS) * 16 + 4 * lq, d.p.Ka);
                if (!whole) fetch(g);
#pragma unroll
                for (int u = 0; u < AHEAD; u++)
#pragma unroll
                    for (int c = 0; c < 4; c++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[u][c], wv[u][c], acc, 0, 0, 0);
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; r++) part[wave][4 * lq + r][lr] = acc[r];
            __syncthreads();
            for (int e = threadIdx.x; e < 16 * LOW_ROWS; e += 64 * KS) {
                const int m = e >> 4, j = e & 15;
                if (!((rows >> m) & 1) || j0 + j >= d.p.Rp) continue;
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < KS; w++) v += part[w][m][j];
                H[(p0 + m) * d.p.Rp + j0 + j] = j0 + j < d.rank ? v * sc : 0.f;
            }
        }
    }
}

// The GEMM tile over sorted rows.  24576 x 768 -> 768 with 24 adapters of rank 16: 240 us, 126 TFLOP/s of the 149 that a large product
// reaches (the same layer without adapters 227: what is added is 2.1 % of the multiplications, rows found through the list and
// written row by row the rest); 4099 x 556 -> 368: 29 us, 390 tiles of 64 x 64 on 256 compute units.  (SC spills 12 vector registers.)
template <bool SC> struct AdaptRows {
    static constexpr bool kPlain = false, kAnyRow = SC;
    const int *perm, *key;
    const float *H, *U;
    long ldw, B, N, Rp;
    __device__ __forceinline__ long base(long m0) const { return m0 / AD_WINDOW * AD_WINDOW; }
    __device__ __forceinline__ unsigned rel(long m) const { return (unsigned)perm[m]; }
    template <int TM, int TN> __device__ __forceinline__ void add(v16f (&acc)[TM][TN], long m, long n, int lr, int lh) const
    {
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const long pb = m + i * 32;
            if (pb >= B) continue;
            const long p = pb + lr < B ? pb + lr : B - 1;
            const int kk = pb + lr < B ? key[p] : -1;
            const float* h = H + p * Rp + 4 * lh;
            unsigned live = (unsigned)__ballot(kk >= 0);
            while (live) {
                const int a = __builtin_amdgcn_readlane(kk, __builtin_ctz(live));
                const unsigned rows = (unsigned)__ballot(kk == a);
                live &= ~rows;
                const bool mine = (rows >> lr) & 1;
                const float* u[TN];
#pragma unroll
                for (int j = 0; j < TN; j++) u[j] = U + ((long)a * N + (n + j * 32 + lr < N ? n + j * 32 + lr : N - 1)) * Rp + 4 * lh;
                for (long k = 0; k < Rp; k += 8) {
                    v4f hv = *(const v4f*)(h + k), uv[TN];
                    if (!mine) hv = (v4f)(0.f);
#pragma unroll
                    for (int j = 0; j < TN; j++) uv[j] = *(const v4f*)(u[j] + k);
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int j = 0; j < TN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(hv[c], uv[j][c], acc[i][j], 0, 0, 0);
                }
            }
        }
    }
    template <int ACT, int TM, int TN>
    __device__ __forceinline__ void store_act(const v16f (&acc)[TM][TN], float* C, long m, long n, int lr, int lh, const GemmEpi& epi) const
    {
        float bv[TN];
#pragma unroll
        for (int j = 0; j < TN; j++) bv[j] = epi.bias && n + j * 32 + lr < N ? epi.bias[n + j * 32 + lr] : 0.f;
        const long b = base(m);
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const long p = m + i * 32 + 8 * q + 4 * lh;
                const int4 to = *(const int4*)(perm + p);             // the list is a whole number of windows long
                const int row[4] = { to.x, to.y, to.z, to.w };
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    if (p + c >= B) continue;
                    float* y = C + (b + row[c]) * N + n + lr;
#pragma unroll
                    for (int j = 0; j < TN; j++)
                        if (n + j * 32 + lr < N) y[j * 32] = fortis_act_any(acc[i][j][4 * q + c] + bv[j], ACT, epi.alpha);
                }
            }
    }
    template <int TM, int TN>
    __device__ __forceinline__ void store(const v16f (&acc)[TM][TN], float* C, long, long, long m, long n, int lr, int lh, const GemmEpi& epi) const
    {
        if (epi.act == FORTIS_ACT_RELU) store_act<FORTIS_ACT_RELU>(acc, C, m, n, lr, lh, epi);
        else if (epi.act == FORTIS_ACT_LEAKY) store_act<FORTIS_ACT_LEAKY>(acc, C, m, n, lr, lh, epi);
        else if (epi.act == FORTIS_ACT_SILU) store_act<FORTIS_ACT_SILU>(acc, C, m, n, lr, lh, epi);
        else store_act<FORTIS_ACT_NONE>(acc, C, m, n, lr, lh, epi);
    }
};

#define AD_BK 32
// The phases of gemm.hip's persistent kernel.
template <bool SC>
__global__ __launch_bounds__(GM_THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) void adapt_gemm_kernel(const float* __restrict__ A, const float* __restrict__ W,
                                                          float* __restrict__ C, long B, long N, long K, GemmSched sc, GemmEpi epi, AdaptRows<SC> ext)
{
    extern __shared__ float4 smem4[];
    float* smem = (float*)smem4;
    const long w = blockIdx.x;
    for (int p = 0; p < sc.nphase; p++) {
        const int level = sc.ph[p].level;
        const long base = sc.ph[p].base, count = sc.ph[p].count;
        if (level == 0) {
            const long place = (w & 7) * (sc.slots / 8) + (w >> 3);
            const long rounds = count / sc.slots;
            v4f ra[2 * AD_BK / 16], rw[2 * AD_BK / 16];
            for (long r = 0; r < rounds; r++) {
                const long tile = base + r * sc.slots + place, next = tile + sc.slots;
                const long tm = tile / sc.tiles_n, tn = tile - tm * sc.tiles_n;
                const long tmn = next / sc.tiles_n, tnn = next - tmn * sc.tiles_n;
                gemm_tile<2, 2, AD_BK>(A, W, C, B, N, K, tm * 128, tn * 128, epi, smem, ra, rw, r > 0, r + 1 < rounds, tmn * 128, tnn * 128, ext);
            }
            continue;
        }
        const long per_xcd = (count + 7) / 8;
        if ((w >> 3) >= per_xcd) continue;
        const long item = (w & 7) * per_xcd + (w >> 3);
        if (item >= count) continue;
        const long tile = base + (level == 1 ? (item >> 1) : (item >> 2));
        const long tm = tile / sc.tiles_n, tn = tile - tm * sc.tiles_n;
        if (level == 1) {
            const long m0 = tm * 128, n0 = tn * 128 + (item & 1) * 64;
            if (m0 >= B || n0 >= N) continue;
            v4f ra[2 * AD_BK / 16], rw[AD_BK / 16];
            gemm_tile<2, 1, AD_BK>(A, W, C, B, N, K, m0, n0, epi, smem, ra, rw, false, false, 0, 0, ext);
        } else {
            const long m0 = tm * 128 + ((item >> 1) & 1) * 64, n0 = tn * 128 + (item & 1) * 64;
            if (m0 >= B || n0 >= N) continue;
            v4f ra[AD_BK / 16], rw[AD_BK / 16];
            gemm_tile<1, 1, AD_BK>(A, W, C, B, N, K, m0, n0, epi, smem, ra, rw, false, false, 0, 0, ext);
        }
    }
}
template <bool SC>
static void launch_adapt_gemm(const AdaptDesc& d, const float* X, float* Y, long B, const AdaptRows<SC>& ext, hipStream_t s)
{
    const size_t shmem = (size_t)2 * (128 + 128) * (AD_BK + 4) * sizeof(float);
    static long slots = 0;
    if (!slots) {
        HIP_OK(hipFuncSetAttribute((const void*)adapt_gemm_kernel<SC>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shmem));
        int occ = 0, dev = 0;
        hipDeviceProp_t prop;
        HIP_OK(hipGetDevice(&dev));
        HIP_OK(hipGetDeviceProperties(&prop, dev));
        HIP_OK(hipOccupancyMaxActiveBlocksPerMultiprocessor(&occ, (const void*)adapt_gemm_kernel<SC>, GM_THREADS, shmem));
        if (occ < 1) occ = 1;
        slots = (long)occ * prop.multiProcessorCount / 8 * 8;
        if (slots < 8) slots = 8;
    }
    GemmSched sc;
    gemm_make_sched(B, d.N, slots, &sc);
    long items = 0;
    for (int p = 0; p < sc.nphase; p++) items = sc.ph[p].count > items ? sc.ph[p].count : items;
    const long grid = items < slots ? cdiv(items, 8) * 8 : slots;
    const GemmEpi epi = { d.bias, nullptr, d.act, d.alpha, d.N };
    hipLaunchKernelGGL((adapt_gemm_kernel<SC>), dim3((unsigned)grid), dim3(GM_THREADS), shmem, s, X, d.W, Y, B, d.N, d.K, sc, epi, ext);
}

// A launch has to stay under 2^32 work-items, and both forms have many to a row: more than AD_PIECE rows, or few_piece(), go through
// in pieces, one behind the other through the same scratch.
#define AD_PIECE (1L << 26)     // sorted rows: up to 32 work-items each; a multiple of AD_WINDOW
// few rows: 16 work-items a row and rank, 512 a tile of 16 rows and 16 columns; a multiple of 16 and at least 2048 (N < 2^19)
static long few_piece(const AdaptDesc& d)
{
    const long by_rank = (1L << 27) / d.p.Rp / 16 * 16, by_columns = (1L << 22) / cdiv(d.N, 16) * 16;
    return by_rank < by_columns ? by_rank : by_columns;
}
// Both forms' scratch: a step that has been re-sized to fewer rows may take the other one.
long fortis_adapters_workspace(const AdaptDesc& d, long B)
{
    const long n = B < AD_PIECE ? B : AD_PIECE;
    return up(n, AD_WINDOW) * 8 + n * d.p.Rp * 4;
}
template <int ROW>
static void launch_few(const AdaptDesc& d, const float* X, const int* index, float* Y, long B, bool fused, void* ws, hipStream_t s)
{
    float* H = (float*)ws;
    const dim3 grid((unsigned)(cdiv(B, 16) * cdiv(d.N, 16))), block(64 * FEW_WAVES);
    if (fused) {
        hipLaunchKernelGGL((adapt_few_kernel<ROW, true>), grid, block, 0, s, d, X, index, (const float*)H, Y, B);
        return;
    }
    hipLaunchKernelGGL((adapt_low_rows_kernel<ROW>), dim3((unsigned)cdiv(B * (d.p.Rp / 4), AD_THREADS / 64)), dim3(AD_THREADS), 0, s, d, X, index, H, B);
    hipLaunchKernelGGL((adapt_few_kernel<ROW, false>), grid, block, 0, s, d, X, index, (const float*)H, Y, B);
}
template <bool SC>
static void launch_sorted(const AdaptDesc& d, const float* X, const int* index, float* Y, long B, void* ws, hipStream_t s)
{
    const long Bw = up(B, AD_WINDOW);
    int *perm = (int*)ws, *key = perm + Bw;
    float* H = (float*)(key + Bw);
    hipLaunchKernelGGL(adapt_sort_kernel, dim3((unsigned)(Bw / AD_WINDOW)), dim3(1024), (size_t)(d.nadapt + 1 + 16) * 4, s, index, perm, key, B, (int)d.nadapt);
    // Waves by K: each loads six groups of 16 at once; up to 12 groups are left to one wave, 24 to two.  One / two / four / eight
    // waves take, in all, with N = 256 and 24 adapters of rank 16, us:
    //   24576 rows   K = 96  39 / 42 / 49 / 56          K = 192  53 / 50 / 57 / 67          K = 384  79 / 76 / 74 / 84   K = 768  130 / 126 / 124 / 119
    //   4096 rows    K = 96  17.9 / 18.3 / 18.4 / 19.9  K = 192  22.1 / 20.2 / 20.4 / 22.2  K = 384  32 / 28 / 25 / 27   K = 768  52 / 43 / 39 / 36
    const dim3 blocks((unsigned)cdiv(B, LOW_ROWS));
    if (d.p.Ka <= 12 * 16) hipLaunchKernelGGL((adapt_low_sorted_kernel<1, SC>), blocks, dim3(64), 0, s, d, X, (const int*)perm, (const int*)key, H, B);
    else if (d.p.Ka <= 24 * 16) hipLaunchKernelGGL((adapt_low_sorted_kernel<2, SC>), blocks, dim3(128), 0, s, d, X, (const int*)perm, (const int*)key, H, B);
    else hipLaunchKernelGGL((adapt_low_sorted_kernel<8, SC>), blocks, dim3(512), 0, s, d, X, (const int*)perm, (const int*)key, H, B);
    const AdaptRows<SC> ext = { perm, key, H, d.U, d.p.ldw, B, d.N, d.p.Rp };
    launch_adapt_gemm<SC>(d, X, Y, B, ext, s);
}
template <bool SC>
static void launch_adapters(const AdaptDesc& d, const float* X, const int* index, float* Y, long B, void* ws, hipStream_t s)
{
    if (B > AD_FEW_ROWS && d.p.narrow) {
        if (d.K <= 16) narrow_by_columns<1, SC>(d, X, index, Y, B, s);
        else if (d.K <= 32) narrow_by_columns<2, SC>(d, X, index, Y, B, s);
        else narrow_by_columns<4, SC>(d, X, index, Y, B, s);
        return;
    }
    // by all rows: the pieces of a call take one form
    const bool few = d.K < 4 || B <= AD_FEW_ROWS || !d.p.finite, fused = B * d.p.Rp <= FEW_FUSED;
    const long piece = few ? few_piece(d) : AD_PIECE;
    for (long r = 0; r < B; r += piece) {
        const long n = B - r < piece ? B - r : piece;
        const float* x = X + r * d.K;
        float* y = Y + r * d.N;
        if (!few) launch_sorted<SC>(d, x, index + r, y, n, ws, s);
        else if (d.K < 4) launch_few<ROWTINY>(d, x, index + r, y, n, fused, ws, s);
        else launch_few<SC ? ROWANY : ROW4>(d, x, index + r, y, n, fused, ws, s);
    }
}
void fortis_launch_linear_adapters(const AdaptDesc& d, const float* X, const int* index, float* Y, long B, void* ws, hipStream_t s)
{
    if (d.K % 4 == 0) launch_adapters<false>(d, X, index, Y, B, ws, s);
    else launch_adapters<true>(d, X, index, Y, B, ws, s);
    HIP_OK(hipGetLastError());
}

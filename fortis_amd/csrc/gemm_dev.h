// The tile of the fp32 matrix-core GEMM and its work list, shared by the plain GEMM (gemm.hip) and the projection with
// adapters (adapters.hip).  gemm.hip describes the tiling.
#pragma once
#include "common.h"

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));   // native vector: selects and copies stay in registers

#define GM_THREADS 256

// Four floats from any float on, and what a load from the last four floats of a row of K has to become to stand for k .. k + 3.
typedef v4f v4f_any __attribute__((aligned(4)));
__device__ __forceinline__ v4f shift_row4(v4f t, long k, long K)
{
    const int s = k <= K - 4 ? 0 : (int)(k - (K - 4));
    v4f v;
    v[0] = s == 0 ? t[0] : s == 1 ? t[1] : s == 2 ? t[2] : s == 3 ? t[3] : 0.f;
    v[1] = s == 0 ? t[1] : s == 1 ? t[2] : s == 2 ? t[3] : 0.f;
    v[2] = s == 0 ? t[2] : s == 1 ? t[3] : 0.f;
    v[3] = s == 0 ? t[3] : 0.f;
    return v;
}

struct GemmEpi {
    const float* bias;
    const float* out_scale;
    int act;
    float alpha;
    long mask_from;   // columns >= mask_from get ReLU (N when unused)
};

__device__ __forceinline__ float gemm_act(float v, int act, float alpha)
{
    if (act == FORTIS_ACT_RELU) return v > 0.f ? v : 0.f;
    if (act == FORTIS_ACT_LEAKY) return v > 0.f ? v : alpha * v;
    return v;
}

// Epilogue of a tile with all its rows and nothing but bias and activation: per element one add, the activation
// (MODE 0 none, 1 max(v, 0), 2 max(v, alpha v) for 0 <= alpha <= 1, 3 the general form) and a store to
// uniform row base + one of TM*TN per-lane 32-bit offsets.
template <int TM, int TN, int MODE>
__device__ __forceinline__ void gemm_store_plain(const v16f (&acc)[TM][TN], float* cb, unsigned Nu, const float* bias,
                                                 int wm, int wn, int lr, int lh, int ncols, const GemmEpi& epi)
{
    const float alpha = epi.alpha;
#pragma unroll
    for (int j = 0; j < TN; j++) {
        if (wn + j * 32 + lr >= ncols) continue;                         // column past the end of C
        const float bv = bias ? bias[wn + j * 32 + lr] : 0.f;
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const unsigned off = (unsigned)(wm + i * 32 + 4 * lh) * Nu + (unsigned)(wn + j * 32 + lr);
#pragma unroll
            for (int r = 0; r < 16; r++) {
                float v = acc[i][j][r] + bv;
                if (MODE == 1) v = fmaxf(v, 0.f);
                else if (MODE == 2) v = fmaxf(v, alpha * v);
                else if (MODE == 3) v = gemm_act(v, epi.act, alpha);
                float* rb = cb + (size_t)((unsigned)(8 * (r >> 2) + (r & 3)) * Nu);     // uniform row base
                rb[off] = v;
            }
        }
    }
}

// Workgroup barrier that orders LDS traffic only: global loads issued earlier stay in flight across it
// (__syncthreads() would also wait for every outstanding global load).
__device__ __forceinline__ void lds_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// One output tile of (64 TM) x (64 TN) at (m0, n0), by the whole workgroup.
//
// Schedule of one k slab (NKG groups of 8 k, one group = TM*TN*4 MFMAs per wave):
//   top      global loads of the next slab -> staging registers (ra, rw)
//   group g  LDS reads of the fragments of group g+1, then the MFMAs of group g
//   before the last group: staging registers -> other LDS buffer, barrier, LDS reads of the next slab's group 0
// so every LDS read has a whole group of MFMAs to arrive, and the barrier is followed by MFMAs that
// were already fed.  The staging registers belong to the caller: when `preloaded`, they already hold
// this tile's slab 0, and when `has_next`, the last slab's "next slab" is slab 0 of tile (m0n, n0n),
// whose latency then hides behind this tile's epilogue.
//
// Ext says how the rows of A and C are found and what joins the sums; GemmPlain is a GEMM of consecutive rows.  Another
// one (kPlain false) gives
//   base(m0), rel(m)   A's row of tile row m is base(m0) + rel(m)
//   ldw                pitch of W's rows
//   kAnyRow            A's rows start at any float (K no multiple of 4 but at least 4; ldw is one, W's rows end in zeros)
//   add(acc, ...)      sums that join before the epilogue
//   store(acc, ...)    the epilogue
struct GemmPlain { static constexpr bool kPlain = true, kAnyRow = false; };
template <int TM, int TN, int GM_BK, class Ext>
__device__ __forceinline__ void gemm_tile(const float* __restrict__ A, const float* __restrict__ W,
                                          float* __restrict__ C, long B, long N, long K,
                                          long m0, long n0, const GemmEpi& epi, float* smem,
                                          v4f (&ra)[TM * GM_BK / 16], v4f (&rw)[TN * GM_BK / 16],
                                          bool preloaded, bool has_next, long m0n, long n0n, const Ext& ext)
{
    constexpr int BM = 64 * TM, BN = 64 * TN;
    constexpr int GM_LDK = GM_BK + 4;                   // LDS row pitch: +4 floats staggers the banks
    constexpr int F4R = GM_BK / 4;                      // v4f per staged row
    constexpr int LA = TM * GM_BK / 16;                 // v4f loads per thread per slab (A)
    constexpr int LW = TN * GM_BK / 16;
    constexpr int NKG = GM_BK / 8;
    static_assert(NKG % 2 == 0, "fragment sets alternate per k group");
    float* sA = smem;                                   // [2][BM][GM_LDK]
    float* sW = sA + 2 * BM * GM_LDK;                   // [2][BN][GM_LDK]

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave & 1) * (BM / 2), wn = (wave >> 1) * (BN / 2);
    const int lr = lane & 31, lh = lane >> 5;

    v16f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;

    // staging map: v4f index f = tid + t*256 -> row = f / F4R, kq = f % F4R.
    // A thread's byte offsets inside the tile's rows are fixed for the whole tile (32 bits: rows past
    // the end of A or W are clamped to the last one -- their products land in rows/columns of the tile
    // that are never stored), so a load is uniform base + k0 plus a per-thread 32-bit offset.
    long ldw = K;
    if constexpr (!Ext::kPlain) ldw = ext.ldw;
    auto abase = [&](long mt) __attribute__((always_inline)) { if constexpr (Ext::kPlain) return A + mt * K; else return A + ext.base(mt) * K; };
    auto offsets = [&](long mt, long nt, unsigned (&oa)[LA], unsigned (&ow)[LW]) __attribute__((always_inline)) {
        const int lastm = (int)(B - 1 - mt < BM - 1 ? B - 1 - mt : BM - 1);
        const int lastn = (int)(N - 1 - nt < BN - 1 ? N - 1 - nt : BN - 1);
#pragma unroll
        for (int t = 0; t < LA; t++) {
            const int f = tid + t * GM_THREADS, row = f / F4R, kq = f % F4R;
            if constexpr (Ext::kPlain) oa[t] = ((unsigned)(row < lastm ? row : lastm) * (unsigned)K + kq * 4) * 4u;
            else oa[t] = (ext.rel(mt + (row < lastm ? row : lastm)) * (unsigned)K + (Ext::kAnyRow ? 0 : kq * 4)) * 4u;
        }
#pragma unroll
        for (int t = 0; t < LW; t++) {
            const int f = tid + t * GM_THREADS, row = f / F4R, kq = f % F4R;
            ow[t] = ((unsigned)(row < lastn ? row : lastn) * (unsigned)ldw + kq * 4) * 4u;
        }
    };
    // Every staged chunk of a thread sits at the same k inside the slab (GM_THREADS is a multiple of F4R).
    static_assert(GM_THREADS % F4R == 0, "a thread's chunks share their k position");
    const int kq4 = (tid % F4R) * 4;
    // ONE load site and ONE store site per slab, whatever the slab is (a full one, the one that runs past K,
    // slab 0 of the next tile): the compiler otherwise merges the register sets of the different sites with
    // copies placed right behind the loads, and every wave then waits for its loads before it multiplies.
    // A chunk at or beyond K reads the row's chunk 0 instead (a valid address) and is zeroed when stored.
    auto load_slab = [&](const float* Ab, const float* Wb, const unsigned (&oa)[LA], const unsigned (&ow)[LW], long k0) __attribute__((always_inline)) {
        const char* wb = (const char*)(Wb + k0);
        if constexpr (Ext::kAnyRow) {
            // from the row's last four floats at most; moved into place when stored
            const unsigned ok = (unsigned)(k0 + kq4 <= K - 4 ? k0 + kq4 : K - 4) * 4u;
#pragma unroll
            for (int t = 0; t < LA; t++) ra[t] = *(const v4f_any*)((const char*)Ab + oa[t] + ok);
        } else {
            const char* ab = (const char*)(Ab + k0);
#pragma unroll
            for (int t = 0; t < LA; t++) ra[t] = *(const v4f*)(ab + oa[t]);
        }
#pragma unroll
        for (int t = 0; t < LW; t++) rw[t] = *(const v4f*)(wb + ow[t]);
    };
    // Before the load of a slab that runs past K (the last one of a tile, after which these offsets are not
    // used again): chunks at or beyond K are pointed at their row's chunk 0.
    auto clamp_offsets = [&](long k0, unsigned (&oa)[LA], unsigned (&ow)[LW]) __attribute__((always_inline)) {
        if (k0 + GM_BK > K) {
            asm volatile("" ::: "memory");               // stays a branch
            const unsigned adj = k0 + kq4 < K ? 0u : (unsigned)kq4 * 4u;
            if constexpr (!Ext::kAnyRow) {
#pragma unroll
                for (int t = 0; t < LA; t++) oa[t] -= adj;
            }
#pragma unroll
            for (int t = 0; t < LW; t++) ow[t] -= adj;
        }
    };
    // k0: the slab the staging registers hold
    auto store_slab = [&](int buf, long k0) __attribute__((always_inline)) {
        float* a = sA + buf * BM * GM_LDK;
        float* w = sW + buf * BN * GM_LDK;
        if (k0 + GM_BK > K) {
            // only the slab that runs past K comes here; the empty asm keeps this a branch (as a select it
            // would cost every slab one instruction per staged register)
            asm volatile("" ::: "memory");
            if (k0 + kq4 >= K) {
                const v4f zero = (v4f)(0.f);
#pragma unroll
                for (int t = 0; t < LA; t++) ra[t] = zero;
#pragma unroll
                for (int t = 0; t < LW; t++) rw[t] = zero;
            }
            if constexpr (Ext::kAnyRow) {
                if (k0 + kq4 < K) {
#pragma unroll
                    for (int t = 0; t < LA; t++) ra[t] = shift_row4(ra[t], k0 + kq4, K);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < LA; t++) {
            const int f = tid + t * GM_THREADS, row = f / F4R, kq = f % F4R;
            *(v4f*)(a + row * GM_LDK + kq * 4) = ra[t];
        }
#pragma unroll
        for (int t = 0; t < LW; t++) {
            const int f = tid + t * GM_THREADS, row = f / F4R, kq = f % F4R;
            *(v4f*)(w + row * GM_LDK + kq * 4) = rw[t];
        }
    };
    v4f fa[2][TM], fw[2][TN];
    auto read_frag = [&](int set, int buf, int kg) __attribute__((always_inline)) {
        const float* a = sA + buf * BM * GM_LDK + (wm + lr) * GM_LDK + 4 * lh + kg * 8;
        const float* w = sW + buf * BN * GM_LDK + (wn + lr) * GM_LDK + 4 * lh + kg * 8;
#pragma unroll
        for (int i = 0; i < TM; i++) fa[set][i] = *(const v4f*)(a + i * 32 * GM_LDK);
#pragma unroll
        for (int j = 0; j < TN; j++) fw[set][j] = *(const v4f*)(w + j * 32 * GM_LDK);
    };
    auto multiply = [&](int set) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[set][i][c], fw[set][j][c], acc[i][j], 0, 0, 0);
    };

    const int nslab = (int)((K + GM_BK - 1) / GM_BK);
    unsigned oa[LA], ow[LW];
    offsets(m0, n0, oa, ow);
    const float* Ab = abase(m0);
    const float* Wb = W + n0 * ldw;
    if (!preloaded) {
        clamp_offsets(0, oa, ow);
        load_slab(Ab, Wb, oa, ow, 0);
    }
    store_slab(0, 0);
    lds_barrier();
    read_frag(0, 0, 0);
    // one k slab out of LDS buffer `buf` (a literal at both call sites, so every LDS address below is a
    // constant offset from the thread's base and no address arithmetic is left in the loop)
    auto slab = [&](int sl, int buf) __attribute__((always_inline)) {
        const bool more = sl + 1 < nslab;
        long knext = (long)(sl + 1) * GM_BK;
        if (!more && has_next) {
            // the staging registers now fetch slab 0 of the next tile: its offsets replace this tile's
            offsets(m0n, n0n, oa, ow);
            Ab = abase(m0n);
            Wb = W + n0n * ldw;
            knext = 0;
        }
        if (more || has_next) {
            clamp_offsets(knext, oa, ow);
            load_slab(Ab, Wb, oa, ow, knext);
        }
#pragma unroll
        for (int kg = 0; kg + 1 < NKG; kg++) {
            read_frag((kg + 1) & 1, buf, kg + 1);
            multiply(kg & 1);
        }
        // the staged slab goes to LDS as late as possible: its loads have had NKG - 1 groups of MFMAs to arrive
        if (more) store_slab(buf ^ 1, knext);
        lds_barrier();
        if (more) read_frag(0, buf ^ 1, 0);
        multiply((NKG - 1) & 1);
    };
    for (int sl = 0; sl < nslab; sl += 2) {
        slab(sl, 0);
        if (sl + 1 < nslab) slab(sl + 1, 1);
    }

    if constexpr (!Ext::kPlain) {
        ext.add(acc, m0 + wm, n0 + wn, lr, lh);
        ext.store(acc, C, B, N, m0 + wm, n0 + wn, lr, lh, epi);
        return;
    }
    // epilogue: lane holds column n = lr of 16 rows per MFMA tile.
    // Tiles with all their rows and a plain bias + activation epilogue (every hidden layer) take a path
    // with one add and the activation per element; everything else takes the guarded one.
    const bool plain = !epi.out_scale && epi.mask_from >= N && m0 + BM <= B;
    const int ncols = (int)(N - n0 < BN ? N - n0 : BN);                 // columns of this tile that exist
    if (plain) {
        float* cb = C + m0 * N + n0;                                    // uniform
        const float* bias = epi.bias ? epi.bias + n0 : nullptr;
        if (epi.act == FORTIS_ACT_RELU) gemm_store_plain<TM, TN, 1>(acc, cb, (unsigned)N, bias, wm, wn, lr, lh, ncols, epi);
        else if (epi.act == FORTIS_ACT_LEAKY && epi.alpha >= 0.f && epi.alpha <= 1.f) gemm_store_plain<TM, TN, 2>(acc, cb, (unsigned)N, bias, wm, wn, lr, lh, ncols, epi);
        else if (epi.act == FORTIS_ACT_NONE) gemm_store_plain<TM, TN, 0>(acc, cb, (unsigned)N, bias, wm, wn, lr, lh, ncols, epi);
        else gemm_store_plain<TM, TN, 3>(acc, cb, (unsigned)N, bias, wm, wn, lr, lh, ncols, epi);
        return;
    }
#pragma unroll
    for (int j = 0; j < TN; j++) {
        const long n = n0 + wn + j * 32 + lr;
        if (n >= N) continue;
        const float bv = epi.bias ? epi.bias[n] : 0.f;
        const float sv = epi.out_scale ? epi.out_scale[n] : 1.f;
        const bool relu_tail = n >= epi.mask_from;
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const long m = m0 + wm + i * 32 + 8 * (r >> 2) + 4 * lh + (r & 3);
                if (m >= B) continue;
                float v = gemm_act(acc[i][j][r] + bv, epi.act, epi.alpha);
                if (epi.out_scale) v = v * sv;
                if (relu_tail) v = v > 0.f ? v : 0.f;
                C[m * N + n] = v;
            }
    }
}

// Work list of one launch.  Tiles are numbered row-major over 128 x 128 blocks of C; a phase hands
// out items of 1 (level 0), 1/2 (level 1: 128 x 64) or 1/4 (level 2: 64 x 64) of such a block.
struct GemmPhase { int level, pad; long base, count; };
struct GemmSched { int nphase, tiles_n; long slots; GemmPhase ph[4]; };

// Work list for C[B][N] on `slots` resident workgroups (a multiple of 8): whole rounds of 128 x 128 tiles,
// then one round of halves if at least half a round is left, one round of quarters if at least a quarter
// round is left, and the rest as quarters.
static void gemm_make_sched(long B, long N, long slots, GemmSched* out)
{
    GemmSched sc = {};
    sc.tiles_n = (int)cdiv(N, 128);
    sc.slots = slots;
    const long total = cdiv(B, 128) * sc.tiles_n;
    long base = total / slots * slots, rem = total - base;
    auto phase = [&](int level, long b, long count) { GemmPhase ph = { level, 0, b, count }; sc.ph[sc.nphase++] = ph; };
    if (base) phase(0, 0, base);
    if (2 * rem >= slots) { phase(1, base, slots); base += slots / 2; rem -= slots / 2; }
    if (4 * rem >= slots) { phase(2, base, slots); base += slots / 4; rem -= slots / 4; }
    if (rem) phase(2, base, 4 * rem);
    *out = sc;
}

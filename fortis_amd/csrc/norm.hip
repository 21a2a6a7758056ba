// Group normalisation with an activation (include/fortis_step.h, fortis_plan_group_norm):
//     y = act(gamma_c (x - mean_{n,g}) / sqrt(var_{n,g} + eps) + beta_c)
// over the S * C / G values of every (sample, group) -- an "instance" below -- channels last or first.
//
// Memory-bound: 8 bytes and about ten operations a value.  Three forms:
//   lanes    up to 2048 values an instance (512 vectors): 1 to 64 lanes hold it in registers, one read, one write, no barrier.
//            71040 rows of 64 in heads of 16, SiLU: 9.2 us, 3.9 TB/s (a copy of as many bytes 5.4 us), bound by issuing vector instructions:
//            some 265 for a wave's 256 values, 7.7 us at four cycles each;
//   block    up to 32768: one workgroup holds an instance (or the neighbouring instances whose channels share 128-byte
//            lines) in registers, one read, one write.  512 x 8 instances of 16384, channels first: 102 us, 5.2 TB/s;
//   split    beyond, and where few workgroups would have much each (a compute unit alone moves some 25 GB/s: eight instances of
//            32768 take 8.3 us in the block form, 7.6-7.7 in two launches): one launch sums over chunks of every sample, a second joins
//            a sample's chunk sums and normalises.  The input is read twice, the second time from the caches as far as they
//            hold it.  287496 x 64 in 8 groups: 36.2 us, 13 of them the sums (the first read runs at what HBM gives), the rest
//            the second at 6 TB/s; 65536 x 32: 10.8 us, both launches bound by their start and two barriers, the second by the join as well: each of
//            its 256 workgroups adds up 256 partial sums of eight groups.
// Sums.  Where the values stay in registers the mean comes first, summed about the instance's first value as a pivot, and the
// squares of what is left after it second, in float32.  The split form has to take both sums in one read: every thread sums at
// most 64 values about the first one it meets, and from there on everything is joined in float64 about the instance's first
// value, where cancellation costs digits that are there to spare.  The mean is subtracted as a float32 pair.
#include "common.h"

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
template <int V> struct VecOf { typedef float T; };
template <> struct VecOf<2> { typedef v2f T; };
template <> struct VecOf<4> { typedef v4f T; };
template <int V> struct Vals { float v[V]; };
template <int V> __device__ __forceinline__ Vals<V> ld(const float* p)
{
    Vals<V> r;
    const typename VecOf<V>::T t = *(const typename VecOf<V>::T*)p;
    __builtin_memcpy(r.v, &t, sizeof t);
    return r;
}
template <int V, bool STREAM = false> __device__ __forceinline__ void st(float* p, const Vals<V>& r)
{
    typename VecOf<V>::T t;
    __builtin_memcpy(&t, r.v, sizeof t);
    if constexpr (STREAM) __builtin_nontemporal_store(t, (typename VecOf<V>::T*)p);
    else *(typename VecOf<V>::T*)p = t;
}

#define GN_LANES_VECS 512      // vectors of an instance in the lanes form: 64 lanes x 8
#define GN_BLOCK_VALUES 32768  // values of a workgroup in the block form: 1024 threads x 32
#define GN_BLOCK_ALONE 8192    // up to this many the block form is taken however few workgroups there are
#define GN_BLOCK_FULL 256      // workgroups that keep every compute unit busy
#define GN_LINE 32             // channels whose floats fill a 128-byte line

// Sum over the 2^k lanes around this one (L = 2^k).
template <int L> __device__ __forceinline__ float sum_lanes(float v)
{
#pragma unroll
    for (int o = L / 2; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// The values of an instance held in registers, less their mean, in two steps.  The first mean is summed about a pivot, the instance's
// first value, which may lie far outside (sqrt(n) spreads): it is off by some u |pivot - mean|.  It is subtracted as a pair
// (hi, lo), and what the differences still sum to corrects it.
struct Centre { float hi, lo; };
__device__ __forceinline__ Centre centre(float pivot, float mean)       // pivot + mean to twice float32's digits
{
    Centre c;
    c.hi = pivot + mean;
    const float b = c.hi - pivot;
    c.lo = (pivot - (c.hi - b)) + (mean - b);
    return c;
}

struct NormArgs {
    NormDesc d;
    const float* x;
    float* y;
    long cg, count;             // channels a group, values an instance
    FastDiv row;                // vectors of an instance's row (channels last), or of a channel (channels first)
    FastDiv group;              // groups of a sample
};
// (64-bit divisions take a hundred instructions each; counts that reach 2^31 are rare enough to pay for them)
__device__ __forceinline__ long div_up31(long n, const FastDiv& f) { return n < (1L << 31) ? (long)fortis_div((unsigned)n, f) : n / (long)f.d; }

// ---- lanes form --------------------------------------------------------------------------------------------------
// Element e (vectors of V) of an instance: position e / (cg / V), channel V * (e % (cg / V)); channels first: V values of
// channel e / (S / V).  L lanes share an instance, E vectors a lane; a wave takes 64 / L neighbouring instances at a time.
template <int V, int L, int E>
__global__ __launch_bounds__(256) void norm_lanes_kernel(NormArgs a, long total)
{
    const NormDesc& d = a.d;
    const int lane = threadIdx.x & 63, sub = lane & (L - 1);
    const unsigned nv = (unsigned)(a.count / V);
    const long step = (long)gridDim.x * (256 / L);
    for (long first = (long)blockIdx.x * (256 / L); first < total; first += step) {
        const long inst = first + threadIdx.x / L;
        const bool on = inst < total;
        const long n = on ? div_up31(inst, a.group) : 0;
        const int g = on ? (int)(inst - n * d.G) : 0;
        const long base = d.first ? (n * d.C + g * a.cg) * d.S : n * d.S * d.C + g * a.cg;
        Vals<V> v[E];
        unsigned ch[E];
        long at[E];
        bool have[E];
#pragma unroll
        for (int k = 0; k < E; k++) {
            const unsigned e = sub + k * L;
            have[k] = on && e < nv;
            const unsigned q = fortis_div(e, a.row);
            if (d.first) { at[k] = base + (long)e * V; ch[k] = (unsigned)(g * a.cg) + q; }
            else { const unsigned c = (e - q * a.row.d) * V; at[k] = base + (long)q * d.C + c; ch[k] = (unsigned)(g * a.cg) + c; }
            if (have[k]) v[k] = ld<V>(a.x + at[k]);
        }
        Vals<V> ga[E], be[E];
        auto scales = [&](int k) __attribute__((always_inline)) {
            if (d.first) {
                const float gs = d.gamma[ch[k]], bs = d.beta[ch[k]];
#pragma unroll
                for (int c = 0; c < V; c++) { ga[k].v[c] = gs; be[k].v[c] = bs; }
            } else { ga[k] = ld<V>(d.gamma + ch[k]); be[k] = ld<V>(d.beta + ch[k]); }
        };
        constexpr bool EARLY = E <= 2;      // few enough to travel beside the values: 9.7 -> 9.1 us for 71040 rows of 64
        if constexpr (EARLY) {
#pragma unroll
            for (int k = 0; k < E; k++) if (have[k]) scales(k);
        }
        const float pivot = __shfl(v[0].v[0], lane & ~(L - 1), 64);
        const float inv = 1.f / (float)a.count;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < E; k++)
#pragma unroll
            for (int c = 0; c < V; c++) s += have[k] ? v[k].v[c] - pivot : 0.f;
        const Centre mid = centre(pivot, sum_lanes<L>(s) * inv);
        float s2 = 0.f;
        s = 0.f;
#pragma unroll
        for (int k = 0; k < E; k++)
#pragma unroll
            for (int c = 0; c < V; c++) {
                v[k].v[c] = (v[k].v[c] - mid.hi) - mid.lo;
                const float t = have[k] ? v[k].v[c] : 0.f;
                s += t;
                s2 = fmaf(t, t, s2);
            }
        const float off = sum_lanes<L>(s) * inv, rstd = 1.f / sqrtf(fmaf(-off, off, sum_lanes<L>(s2) * inv) + d.eps);
        fortis_with_act(d.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < E; k++) {
            if (!have[k]) continue;
            if constexpr (!EARLY) scales(k);
            Vals<V> o;
#pragma unroll
            for (int c = 0; c < V; c++) o.v[c] = fortis_act_any(fmaf((v[k].v[c] - off) * rstd, ga[k].v[c], be[k].v[c]), decltype(act)::value, d.alpha);
            st<V>(a.y + at[k], o);
        }
        });
    }
}

// ---- block form --------------------------------------------------------------------------------------------------
// Sums of two floats per thread over the workgroup's T threads, the same order in every call; red: T / 64 pairs.
template <int T> __device__ __forceinline__ float2 sum_block(float v, float w, float2* red)
{
    v = sum_lanes<64>(v); w = sum_lanes<64>(w);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(v, w);
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < T / 64; k++) { s.x += red[k].x; s.y += red[k].y; }
    __syncthreads();
    return s;
}
// One instance per workgroup: vectors e = thread + k T of it.
template <int V, int T, int E>
__global__ __launch_bounds__(T) void norm_block_kernel(NormArgs a, long total)
{
    __shared__ float2 red[T / 64];
    const NormDesc& d = a.d;
    const unsigned nv = (unsigned)(a.count / V);
    for (long inst = blockIdx.x; inst < total; inst += gridDim.x) {
        const long n = div_up31(inst, a.group);
        const int g = (int)(inst - n * d.G);
        const float* x = a.x + (d.first ? (n * d.C + g * a.cg) * d.S : n * d.S * d.C + g * a.cg);
        float* y = a.y + (x - a.x);
        Vals<V> v[E];
        const unsigned gc = (unsigned)(g * a.cg);
        // element e of the instance: where it lies and its (first) channel
        auto place = [&](unsigned e, long& at, unsigned& ch) __attribute__((always_inline)) {
            const unsigned q = fortis_div(e, a.row);
            if (d.first) { at = (long)e * V; ch = gc + q; }
            else { const unsigned c = (e - q * a.row.d) * V; at = (long)q * d.C + c; ch = gc + c; }
        };
#pragma unroll
        for (int k = 0; k < E; k++) {
            const unsigned e = threadIdx.x + k * T;
            long at;
            unsigned ch;
            place(e, at, ch);
            if (e < nv) v[k] = ld<V>(x + at);
            if (k % 8 == 7) asm volatile("" ::: "memory");       // eight addresses at a time
        }
        const float pivot = x[0], inv = 1.f / (float)a.count;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < E; k++)
#pragma unroll
            for (int c = 0; c < V; c++) s += threadIdx.x + k * T < nv ? v[k].v[c] - pivot : 0.f;
        const Centre mid = centre(pivot, sum_block<T>(s, 0.f, red).x * inv);
        float s2 = 0.f;
        s = 0.f;
#pragma unroll
        for (int k = 0; k < E; k++)
#pragma unroll
            for (int c = 0; c < V; c++) {
                v[k].v[c] = (v[k].v[c] - mid.hi) - mid.lo;
                const float t = threadIdx.x + k * T < nv ? v[k].v[c] : 0.f;
                s += t;
                s2 = fmaf(t, t, s2);
            }
        const float2 sums = sum_block<T>(s, s2, red);
        const float off = sums.x * inv, rstd = 1.f / sqrtf(fmaf(-off, off, sums.y * inv) + d.eps);
        fortis_with_act(d.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < E; k++) {
            unsigned e = threadIdx.x + k * T, ch;
            if (e >= nv) continue;
            asm volatile("" : "+v"(e));          // formed again: E addresses kept in registers would spill
            long at;
            place(e, at, ch);
            Vals<V> o;
#pragma unroll
            for (int c = 0; c < V; c++) {
                const unsigned i = ch + (d.first ? 0 : c);
                o.v[c] = fortis_act_any(fmaf((v[k].v[c] - off) * rstd, d.gamma[i], d.beta[i]), decltype(act)::value, d.alpha);
            }
            st<V>(y + at, o);
        }
        });
    }
}
// Channels last, `gs` neighbouring groups of one sample per workgroup: a thread keeps its column of V channels, which lie in one group, and takes every rows-th position.
template <int V, int T, int E>
__global__ __launch_bounds__(T) void norm_block_groups_kernel(NormArgs a, int gs, FastDiv slices, long total)
{
    __shared__ float2 part[T], sums[T];
    const NormDesc& d = a.d;
    const int tid = threadIdx.x;
    for (long item = blockIdx.x; item < total; item += gridDim.x) {
        const long n = div_up31(item, slices);
        const int g0 = (int)(item - n * slices.d) * gs, ng = d.G - g0 < gs ? (int)(d.G - g0) : gs;
        const int cgv = (int)(a.cg / V), wv = ng * cgv, rows = (int)((unsigned)T / (unsigned)wv);
        const int row = (int)((unsigned)tid / (unsigned)wv), col = tid - row * wv, gl = (int)((unsigned)col / (unsigned)cgv);
        const bool on = row < rows;
        const unsigned c0 = (unsigned)(g0 * a.cg) + col * V;
        const long base = n * d.S * d.C + c0;
        Vals<V> v[E];
#pragma unroll
        for (int k = 0; k < E; k++)
            if (on && row + k * rows < d.S) v[k] = ld<V>(a.x + base + (long)(row + k * rows) * d.C);
        Vals<V> ga, be;
        if (on) { ga = ld<V>(d.gamma + c0); be = ld<V>(d.beta + c0); }
        const float pivot = a.x[n * d.S * d.C + (g0 + gl) * a.cg], inv = 1.f / (float)a.count;
        // the group's sum: its threads are (row, columns gl cgv .. + cgv); one wave adds each group's partial sums
        auto group_sum = [&](float s, float s2) __attribute__((always_inline)) {
            part[tid] = on ? make_float2(s, s2) : make_float2(0.f, 0.f);
            __syncthreads();
            for (int g = tid >> 6; g < ng; g += T / 64) {
                float t = 0.f, t2 = 0.f;
                for (unsigned i = tid & 63; i < (unsigned)(rows * cgv); i += 64) {
                    const unsigned r = i / (unsigned)cgv;
                    const float2 q = part[r * wv + g * cgv + i - r * cgv];
                    t += q.x; t2 += q.y;
                }
                t = sum_lanes<64>(t); t2 = sum_lanes<64>(t2);
                if ((tid & 63) == 0) sums[g] = make_float2(t, t2);
            }
            __syncthreads();
            return sums[gl];
        };
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < E; k++)
#pragma unroll
            for (int c = 0; c < V; c++) s += on && row + k * rows < d.S ? v[k].v[c] - pivot : 0.f;
        const Centre mid = centre(pivot, group_sum(s, 0.f).x * inv);
        float s2 = 0.f;
        s = 0.f;
#pragma unroll
        for (int k = 0; k < E; k++)
#pragma unroll
            for (int c = 0; c < V; c++) {
                v[k].v[c] = (v[k].v[c] - mid.hi) - mid.lo;
                const float t = on && row + k * rows < d.S ? v[k].v[c] : 0.f;
                s += t;
                s2 = fmaf(t, t, s2);
            }
        const float2 both = group_sum(s, s2);
        const float off = both.x * inv, rstd = 1.f / sqrtf(fmaf(-off, off, both.y * inv) + d.eps);
        if (!on) continue;
        fortis_with_act(d.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < E; k++) {
            if (row + k * rows >= d.S) continue;
            Vals<V> o;
#pragma unroll
            for (int c = 0; c < V; c++) o.v[c] = fortis_act_any(fmaf((v[k].v[c] - off) * rstd, ga.v[c], be.v[c]), decltype(act)::value, d.alpha);
            st<V>(a.y + base + (long)(row + k * rows) * d.C, o);
        }
        });
    }
}

// ---- split form --------------------------------------------------------------------------------------------------
#define GS_THREADS 1024
#define GS_FOLD 16             // batches of loads between two moves of a thread's float32 sums into its float64 ones
#define GS_AHEAD 4             // loads a thread has in flight
struct SplitShape {
    long chunks, per;        // chunks of a sample (an instance with channels first), positions (vectors) a chunk
    int V;                   // floats a thread loads at a time
    int gs, slices;          // channels last: groups and workgroups across the channels
    int blocks;              // workgroups across one group's channels (1 unless a group is wider than 1024 vectors)
    long parts;              // partial sums an instance has
    FastDiv by_chunks, by_across, by_blocks, by_cg;
};
// Where a workgroup of the split form stands (channels last).
struct SplitPlace { long n, c_lo; int chunk, g0, ng, wv, rows, col, row, bl; };
template <int V> __device__ __forceinline__ SplitPlace split_place(const NormArgs& a, const SplitShape& h)
{
    SplitPlace p;
    const NormDesc& d = a.d;
    const unsigned rest = fortis_div(blockIdx.x, h.by_chunks), n = fortis_div(rest, h.by_across), across = rest - n * h.by_across.d;
    const unsigned sl = fortis_div(across, h.by_blocks);
    p.chunk = (int)(blockIdx.x - rest * h.by_chunks.d);
    p.n = n;
    p.bl = (int)(across - sl * h.by_blocks.d);
    p.g0 = (int)sl * h.gs;
    p.ng = d.G - p.g0 < h.gs ? (int)(d.G - p.g0) : h.gs;
    p.c_lo = (long)p.g0 * a.cg + (long)p.bl * GS_THREADS * V;                  // first channel of the workgroup
    const long c_hi = h.blocks > 1 ? ((long)p.g0 + 1) * a.cg : (long)(p.g0 + p.ng) * a.cg;
    p.wv = (int)((c_hi - p.c_lo) / V < GS_THREADS ? (c_hi - p.c_lo) / V : GS_THREADS);
    p.rows = (int)((unsigned)GS_THREADS / (unsigned)p.wv);
    p.row = (int)(threadIdx.x / (unsigned)p.wv);
    p.col = (int)threadIdx.x - p.row * p.wv;
    return p;
}

// Partial sums of `n` values about P: a1 = sum(v - P), a2 = sum((v - P)^2), from sums about a pivot of the thread's own.
__device__ __forceinline__ void about(float pivot, long n, double s1, double s2, double P, double& a1, double& a2)
{
    const double dn = (double)n;
    a1 = a2 = 0.0;
    if (n == 0) return;
    // centred, s2 - s1^2 / n, and moved to P, + t1^2 / n, where t1 - s1 = n (pivot - P): no division
    const double d = (double)pivot - P;
    a1 = dn * d + s1;
    a2 = s2 + d * (s1 + a1);
}
__device__ __forceinline__ double sum_wave(double v)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Channels last.  The slice's columns (V channels each) by rows of the chunk; a thread keeps its column.  ONE: a column's V
// channels lie in one group (they do unless the slice is all channels and V does not divide cg) and are summed together.
template <int V, bool ONE>
__global__ __launch_bounds__(GS_THREADS) void norm_sums_kernel(NormArgs a, SplitShape h, double2* __restrict__ out)
{
    __shared__ double2 part[GS_THREADS];
    const NormDesc& d = a.d;
    const int tid = threadIdx.x;
    const SplitPlace w = split_place<V>(a, h);
    const long r0 = (long)w.chunk * h.per, r1 = r0 + h.per < d.S ? r0 + h.per : d.S;
    const float* xs = a.x + w.n * d.S * d.C;
    constexpr int D = ONE ? 1 : V;              // sums a thread keeps
    float P[D];                                 // the groups' first values: what the sums are joined about
#pragma unroll
    for (int c = 0; c < D; c++) {
        const int g = h.blocks > 1 ? w.g0 : (int)fortis_div((unsigned)(w.c_lo + w.col * V + c), h.by_cg);
        P[c] = xs[g * a.cg];
    }
    float p[D], s1[V], s2[V];
    double d1[D], d2[D];
    long cnt = 0;
#pragma unroll
    for (int c = 0; c < V; c++) s1[c] = s2[c] = 0.f;
#pragma unroll
    for (int c = 0; c < D; c++) { p[c] = 0.f; d1[c] = d2[c] = 0; }
    auto take = [&](const Vals<V>& v) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < V; c++) { const float t = v.v[c] - p[ONE ? 0 : c]; s1[c] += t; s2[c] = fmaf(t, t, s2[c]); }
    };
    auto fold = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < V; c++) { d1[ONE ? 0 : c] += (double)s1[c]; d2[ONE ? 0 : c] += (double)s2[c]; s1[c] = s2[c] = 0.f; }
    };
    // whole passes of the workgroup over `rows` positions: uniform base + a 32-bit offset of the thread's own
    const unsigned off = ((unsigned)w.row * (unsigned)d.C + (unsigned)w.col * V) * 4u;
    const char* base = (const char*)(xs + w.c_lo + r0 * d.C);
    const long pass = (long)w.rows * d.C * 4;
    long left = r1 - r0;
    if (w.row < w.rows) {
        if (w.row < left) {
            const Vals<V> f = ld<V>((const float*)(base + off));
#pragma unroll
            for (int c = 0; c < D; c++) p[c] = f.v[c];
        }
        for (int batch = 1; left >= GS_AHEAD * w.rows; batch++) {
            Vals<V> v[GS_AHEAD];
#pragma unroll
            for (int k = 0; k < GS_AHEAD; k++) v[k] = ld<V>((const float*)(base + k * pass + off));
#pragma unroll
            for (int k = 0; k < GS_AHEAD; k++) take(v[k]);
            cnt += GS_AHEAD;
            base += GS_AHEAD * pass;
            left -= GS_AHEAD * w.rows;
            if (batch % GS_FOLD == 0) fold();
        }
        Vals<V> v[GS_AHEAD];
#pragma unroll
        for (int k = 0; k < GS_AHEAD; k++)
            if (w.row + k * w.rows < left) v[k] = ld<V>((const float*)(base + k * pass + off));
#pragma unroll
        for (int k = 0; k < GS_AHEAD; k++)
            if (w.row + k * w.rows < left) { take(v[k]); cnt++; }
        fold();
    }
    for (int c = 0; c < D; c++) {
        // component c of every column; the groups then take the components one after the other
        double a1 = 0, a2 = 0;
#pragma unroll
        for (int k = 0; k < D; k++) if (k == c) about(p[k], ONE ? V * cnt : cnt, d1[k], d2[k], (double)P[k], a1, a2);
        __syncthreads();
        part[tid] = make_double2(a1, a2);
        __syncthreads();
        for (int q = tid >> 6; q < w.ng; q += GS_THREADS / 64) {
            // columns that hold a channel of group g0 + q in component c (ONE: in any)
            const int lo = h.blocks > 1 ? 0 : (int)(q * a.cg), hi = h.blocks > 1 ? w.wv * V : lo + (int)a.cg;
            const int k0 = ONE ? lo / V : (lo - c + V - 1 + V) / V - 1, k1 = ONE ? hi / V : (hi - c + V - 1 + V) / V - 1;
            double t1 = 0, t2 = 0;
            const int width = k1 - k0;
            for (int i = tid & 63; i < w.rows * width; i += 64) {
                const int r = (int)((unsigned)i / (unsigned)width);
                const double2 t = part[r * w.wv + k0 + i - r * width];
                t1 += t.x; t2 += t.y;
            }
            t1 = sum_wave(t1); t2 = sum_wave(t2);
            if ((tid & 63) == 0) {
                double2* o = out + (w.n * d.G + w.g0 + q) * h.parts + w.chunk * h.blocks + w.bl;
                if (c == 0) *o = make_double2(t1, t2);
                else *o = make_double2(o->x + t1, o->y + t2);
            }
        }
    }
}
// Channels first: chunks of `per` vectors of an instance, which is contiguous.
template <int V>
__global__ __launch_bounds__(GS_THREADS) void norm_sums_first_kernel(NormArgs a, SplitShape h, double2* __restrict__ out)
{
    __shared__ double2 part[GS_THREADS / 64];
    const int tid = threadIdx.x;
    const unsigned inst = fortis_div(blockIdx.x, h.by_chunks), chunk = blockIdx.x - inst * h.by_chunks.d;
    const float* x = a.x + inst * a.count;
    const long nv = a.count / V, e0 = chunk * h.per, e1 = e0 + h.per < nv ? e0 + h.per : nv;
    const float P = x[0];
    float p = 0.f, s1 = 0.f, s2 = 0.f;
    double d1 = 0, d2 = 0;
    long cnt = 0;
    auto take = [&](const Vals<V>& v) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < V; c++) { const float t = v.v[c] - p; s1 += t; s2 = fmaf(t, t, s2); }
        cnt += V;
    };
    auto fold = [&]() __attribute__((always_inline)) { d1 += (double)s1; d2 += (double)s2; s1 = s2 = 0.f; };
    const float* base = x + e0 * V;
    long left = e1 - e0;
    if (tid < left) p = base[tid * V];
    for (; left >= GS_AHEAD * GS_THREADS; left -= GS_AHEAD * GS_THREADS, base += GS_AHEAD * GS_THREADS * V) {
        Vals<V> v[GS_AHEAD];
#pragma unroll
        for (int k = 0; k < GS_AHEAD; k++) v[k] = ld<V>(base + (k * GS_THREADS + tid) * V);
#pragma unroll
        for (int k = 0; k < GS_AHEAD; k++) take(v[k]);
        if (cnt % 64 == 0) fold();
    }
    {
        Vals<V> v[GS_AHEAD];
#pragma unroll
        for (int k = 0; k < GS_AHEAD; k++)
            if (k * GS_THREADS + tid < left) v[k] = ld<V>(base + (k * GS_THREADS + tid) * V);
#pragma unroll
        for (int k = 0; k < GS_AHEAD; k++)
            if (k * GS_THREADS + tid < left) take(v[k]);
        fold();
    }
    double a1, a2;
    about(p, cnt, d1, d2, (double)P, a1, a2);
    a1 = sum_wave(a1); a2 = sum_wave(a2);
    if ((tid & 63) == 0) part[tid >> 6] = make_double2(a1, a2);
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < GS_THREADS / 64; w++) { a1 += part[w].x; a2 += part[w].y; }
        out[(long)inst * h.parts + chunk] = make_double2(a1, a2);
    }
}

// mean (as a pair) and 1 / sqrt(var + eps) of an instance from its partial sums, by one wave.
struct Stat { float hi, lo, rstd, pad; };
__device__ __forceinline__ Stat join(const double2* part, long parts, double pivot, double count, float eps)
{
    double t1 = 0, t2 = 0;
    for (long i = threadIdx.x & 63; i < parts; i += 256) {         // four loads at once: one after the other they take 3 us for 256
        double2 q[4];
#pragma unroll
        for (int k = 0; k < 4; k++) q[k] = part[i + 64 * k < parts ? i + 64 * k : i];
#pragma unroll
        for (int k = 0; k < 4; k++) if (i + 64 * k < parts) { t1 += q[k].x; t2 += q[k].y; }
    }
    t1 = sum_wave(t1) / count; t2 = sum_wave(t2) / count;
    double var = t2 - t1 * t1;
    if (var < 0) var = 0;                                  // a NaN stays one
    const double mean = pivot + t1;
    Stat s;
    s.hi = (float)mean; s.lo = (float)(mean - (double)s.hi); s.rstd = 1.f / sqrtf((float)(var + (double)eps)); s.pad = 0.f;
    return s;
}
// Channels last: the same chunks and columns as the sums, last position first (what the caches still hold).  The first loads
// travel while the sums are joined.
template <int V, bool STREAM>
__global__ __launch_bounds__(GS_THREADS) void norm_apply_kernel(NormArgs a, SplitShape h, const double2* __restrict__ in)
{
    __shared__ Stat stat[GS_THREADS];
    const NormDesc& d = a.d;
    const SplitPlace w = split_place<V>(a, h);
    const long r0 = (long)w.chunk * h.per, r1 = r0 + h.per < d.S ? r0 + h.per : d.S, c0 = w.c_lo + w.col * V;
    const bool on = w.row < w.rows;
    // passes of the workgroup over `rows` positions, GS_AHEAD at a time, the last ones first
    const unsigned off = ((unsigned)w.row * (unsigned)d.C + (unsigned)w.col * V) * 4u;
    const long pass = (long)w.rows * d.C * 4, first = (w.n * d.S + r0) * d.C + w.c_lo;
    const int batch = GS_AHEAD * w.rows, total = (int)(r1 - r0);
    int at = (total - 1) / batch * batch;                    // first position of the batch
    const char* x = (const char*)(a.x + first) + (long)(at / w.rows) * pass;
    char* y = (char*)(a.y + first) + (long)(at / w.rows) * pass;
    Vals<V> v[GS_AHEAD];
    if (on) {                                                // the last batch may be short
#pragma unroll
        for (int k = 0; k < GS_AHEAD; k++)
            if (at + w.row + k * w.rows < total) v[k] = ld<V>((const float*)(x + k * pass + off));
    }
    Vals<V> ga, bt;
    if (on) { ga = ld<V>(d.gamma + c0); bt = ld<V>(d.beta + c0); }
    for (int q = threadIdx.x >> 6; q < w.ng; q += GS_THREADS / 64) {
        const Stat s = join(in + (w.n * d.G + w.g0 + q) * h.parts, h.parts, (double)a.x[w.n * d.S * d.C + (w.g0 + q) * a.cg], (double)a.count, d.eps);
        if ((threadIdx.x & 63) == 0) stat[q] = s;
    }
    __syncthreads();
    if (!on) return;
    float hi[V], lo[V], sc[V], be[V];
#pragma unroll
    for (int c = 0; c < V; c++) {
        const Stat s = stat[h.blocks > 1 ? 0 : (int)fortis_div((unsigned)(c0 + c), h.by_cg) - w.g0];
        hi[c] = s.hi; lo[c] = s.lo;
        sc[c] = s.rstd * ga.v[c];
        be[c] = bt.v[c];
    }
    const float alpha = d.alpha;
    fortis_with_act(d.act, [&](auto act) __attribute__((always_inline)) {
        auto put = [&](int k) __attribute__((always_inline)) {
            Vals<V> o;
#pragma unroll
            for (int c = 0; c < V; c++) o.v[c] = fortis_act_any(fmaf((v[k].v[c] - hi[c]) - lo[c], sc[c], be[c]), decltype(act)::value, alpha);
            st<V, STREAM>((float*)(y + k * pass + off), o);
        };
#pragma unroll
        for (int k = 0; k < GS_AHEAD; k++)
            if (at + w.row + k * w.rows < total) put(k);
        while ((at -= batch) >= 0) {
            x -= GS_AHEAD * pass;
            y -= GS_AHEAD * pass;
#pragma unroll
            for (int k = 0; k < GS_AHEAD; k++) v[k] = ld<V>((const float*)(x + k * pass + off));
#pragma unroll
            for (int k = 0; k < GS_AHEAD; k++) put(k);
        }
    });
}
template <int V, bool STREAM>
__global__ __launch_bounds__(GS_THREADS) void norm_apply_first_kernel(NormArgs a, SplitShape h, const double2* __restrict__ in)
{
    __shared__ Stat stat;
    const NormDesc& d = a.d;
    const int tid = threadIdx.x;
    const unsigned inst = fortis_div(blockIdx.x, h.by_chunks), chunk = blockIdx.x - inst * h.by_chunks.d;
    const unsigned g = inst - fortis_div(inst, a.group) * a.group.d;
    const float* x = a.x + inst * a.count;
    float* y = a.y + inst * a.count;
    const long nv = a.count / V, e0 = chunk * h.per, e1 = e0 + h.per < nv ? e0 + h.per : nv;
    const bool small = nv < (1L << 31);
    const long total = e1 - e0;
    long at = (total - 1) / (GS_AHEAD * GS_THREADS) * (GS_AHEAD * GS_THREADS);       // first vector of the batch, the last one first
    const float* xb = x + (e0 + at) * V;
    float* yb = y + (e0 + at) * V;
    Vals<V> v[GS_AHEAD];
#pragma unroll
    for (int k = 0; k < GS_AHEAD; k++)
        if (at + k * GS_THREADS + tid < total) v[k] = ld<V>(xb + (k * GS_THREADS + tid) * V);
    if (tid < 64) {
        const Stat s = join(in + (long)inst * h.parts, h.parts, (double)x[0], (double)a.count, d.eps);
        if (tid == 0) stat = s;
    }
    __syncthreads();
    const Stat s = stat;
    const float alpha = d.alpha;
    const long c0 = g * a.cg;
    fortis_with_act(d.act, [&](auto act) __attribute__((always_inline)) {
        auto put = [&](int k) __attribute__((always_inline)) {
            const long e = e0 + at + k * GS_THREADS + tid;
            const long c = c0 + (small ? (long)fortis_div((unsigned)e, a.row) : e / (d.S / V));
            const float sc = s.rstd * d.gamma[c], be = d.beta[c];
            Vals<V> o;
#pragma unroll
            for (int q = 0; q < V; q++) o.v[q] = fortis_act_any(fmaf((v[k].v[q] - s.hi) - s.lo, sc, be), decltype(act)::value, alpha);
            st<V, STREAM>(yb + (k * GS_THREADS + tid) * V, o);
        };
#pragma unroll
        for (int k = 0; k < GS_AHEAD; k++)
            if (at + k * GS_THREADS + tid < total) put(k);
        while ((at -= GS_AHEAD * GS_THREADS) >= 0) {
            xb -= GS_AHEAD * GS_THREADS * V;
            yb -= GS_AHEAD * GS_THREADS * V;
#pragma unroll
            for (int k = 0; k < GS_AHEAD; k++) v[k] = ld<V>(xb + (k * GS_THREADS + tid) * V);
#pragma unroll
            for (int k = 0; k < GS_AHEAD; k++) put(k);
        }
    });
}

// ---- choice ------------------------------------------------------------------------------------------------------
static NormDesc norm_normal(const NormDesc& in)
{
    NormDesc d = in;
    if (d.S == 1) d.first = 0;          // the two orders are the same
    return d;
}
static SplitShape split_shape(const NormDesc& d)
{
    SplitShape h = {};
    const long cg = d.C / d.G;
    // Workgroups of 1024 threads: one for every compute unit.  64, 128, 256 and 512 of them take 15.1, 12.6, 11.1 and 16.3 us for 65536 x 32
    // channels last, 61, 40, 36 and 42 for 287496 x 64.
    const long want = 256;
    if (d.first) {
        h.V = d.S % 4 == 0 ? 4 : d.S % 2 == 0 ? 2 : 1;
        const long nv = cg * d.S / h.V, insts = d.NB * d.G;
        h.chunks = cdiv(want, insts);
        if (h.chunks > cdiv(nv, GS_THREADS)) h.chunks = cdiv(nv, GS_THREADS);
        h.per = cdiv(nv, h.chunks);
        h.chunks = cdiv(nv, h.per);
        h.gs = h.slices = h.blocks = 1;
        h.parts = h.chunks;
        h.by_chunks = fortis_fast_div((unsigned)h.chunks);
        return h;
    }
    h.V = d.C % 4 == 0 && d.C <= 4 * GS_THREADS ? 4 : cg % 4 == 0 ? 4 : cg % 2 == 0 ? 2 : 1;
    const long fit = GS_THREADS * h.V;                  // channels a workgroup spans
    h.gs = (int)(d.C <= fit ? d.G : cg <= fit ? fit / cg : 1);
    // The second launch keeps its groups' statistics in an array of GS_THREADS; with groups narrower than V channels there would be up
    // to four times as many.  (V divides C and GS_THREADS cg: every slice is whole vectors.)
    if (h.gs > GS_THREADS) h.gs = GS_THREADS;
    h.slices = (int)cdiv(d.G, h.gs);
    h.blocks = (int)cdiv(cg, fit);
    const long across = (long)h.slices * h.blocks * d.NB;
    const long width = (long)h.gs * cg < fit ? (long)h.gs * cg : fit;
    const long pass = GS_THREADS / cdiv(width, h.V) ? GS_THREADS / cdiv(width, h.V) : 1;      // rows a pass of the workgroup covers
    h.chunks = cdiv(want, across);
    if (h.chunks > cdiv(d.S, pass)) h.chunks = cdiv(d.S, pass);
    h.per = cdiv(d.S, h.chunks);
    h.chunks = cdiv(d.S, h.per);
    h.parts = h.chunks * h.blocks;
    h.by_chunks = fortis_fast_div((unsigned)h.chunks);
    h.by_across = fortis_fast_div((unsigned)(h.slices * h.blocks));
    h.by_blocks = fortis_fast_div((unsigned)h.blocks);
    h.by_cg = fortis_fast_div((unsigned)cg);
    return h;
}

// Which form a problem takes.  S = 1 may be re-sized to other row counts later and is decided by the width of a group alone.
enum NormKind { NORM_LANES, NORM_BLOCK, NORM_GROUPS, NORM_SPLIT };
struct NormForm { NormKind kind; int V, gs; };
static NormForm norm_form(const NormDesc& d)
{
    const long cg = d.C / d.G, count = d.S * cg;
    // a vector stays inside a group and a position (channels last) or inside a channel (channels first)
    const long along = d.first ? d.S : cg;
    NormForm f = { NORM_LANES, along % 4 == 0 ? 4 : along % 2 == 0 ? 2 : 1, 1 };
    if (d.first || d.S == 1 || d.G == 1 || cg >= 4 * GN_LINE) {
        // instances whose memory comes in long pieces
        if (count <= GN_LANES_VECS * f.V) return f;
        f.kind = count <= GN_BLOCK_ALONE || (count <= GN_BLOCK_VALUES && (d.S == 1 || d.NB * d.G >= GN_BLOCK_FULL)) ? NORM_BLOCK : NORM_SPLIT;
        return f;
    }
    // Channels last and narrow groups: neighbouring groups share lines.  Instances of a few values are left to lanes all the
    // same (a sample's are next to each other in a wave); otherwise a workgroup takes the groups of one line, or more of them
    // as long as there are workgroups enough: 512 samples of 128 x 256 in groups of 32 channels take 36.1 us with a group
    // each and 33.6 with four.
    if (count <= 256) return f;
    auto fits = [&](long gs) { return gs * cg / f.V <= 1024 && d.S <= 1024 / (gs * cg / f.V) * 8; };
    f.gs = (int)cdiv(GN_LINE, cg);
    if (f.gs > d.G) f.gs = (int)d.G;
    while (2 * f.gs <= d.G && fits(2 * f.gs) && d.NB * cdiv(d.G, 2 * f.gs) >= 2 * GN_BLOCK_FULL) f.gs *= 2;
    const bool enough = d.S * f.gs * cg <= GN_BLOCK_ALONE || d.NB * cdiv(d.G, f.gs) >= GN_BLOCK_FULL;
    f.kind = fits(f.gs) && enough ? NORM_GROUPS : NORM_SPLIT;
    return f;
}

long fortis_norm_workspace(const NormDesc& in)
{
    const NormDesc d = norm_normal(in);
    if (norm_form(d).kind != NORM_SPLIT) return 0;
    return d.NB * d.G * split_shape(d).parts * (long)sizeof(double2);
}

template <int V> static void launch_lanes(const NormArgs& a, long total, hipStream_t s)
{
    const long nv = a.count / V;
    auto grid = [&](int L) { const long g = cdiv(total, 256 / L); return dim3((unsigned)(g < 8192 ? g : 8192)); };
#define GN_LANES(L, E) hipLaunchKernelGGL((norm_lanes_kernel<V, L, E>), grid(L), dim3(256), 0, s, a, total)
    if (nv <= 1) GN_LANES(1, 1);
    else if (nv <= 2) GN_LANES(2, 1);
    else if (nv <= 4) GN_LANES(4, 1);
    else if (nv <= 8) GN_LANES(8, 1);
    else if (nv <= 16) GN_LANES(16, 1);
    else if (nv <= 32) GN_LANES(32, 1);
    else if (nv <= 64) GN_LANES(64, 1);
    else if (nv <= 128) GN_LANES(64, 2);
    else if (nv <= 256) GN_LANES(64, 4);
    else GN_LANES(64, 8);
#undef GN_LANES
}
template <int V> static void launch_block(const NormArgs& a, NormKind kind, int gs, hipStream_t s)
{
    const NormDesc& d = a.d;
    if (kind == NORM_BLOCK) {
        const long total = d.NB * d.G, nv = a.count / V;
        const dim3 grid((unsigned)(total < 65536 ? total : 65536));
        if (nv <= 256 * 4) hipLaunchKernelGGL((norm_block_kernel<V, 256, 4>), grid, dim3(256), 0, s, a, total);
        else if (nv <= 256 * 8) hipLaunchKernelGGL((norm_block_kernel<V, 256, 8>), grid, dim3(256), 0, s, a, total);
        else if (nv <= 1024 * 4) hipLaunchKernelGGL((norm_block_kernel<V, 1024, 4>), grid, dim3(1024), 0, s, a, total);
        else if (nv <= 1024 * 8) hipLaunchKernelGGL((norm_block_kernel<V, 1024, 8>), grid, dim3(1024), 0, s, a, total);
        if constexpr (V <= 2) if (nv > 1024 * 8 && nv <= 1024 * 16) hipLaunchKernelGGL((norm_block_kernel<V, 1024, 16>), grid, dim3(1024), 0, s, a, total);
        // (32 single values a thread do not fit in 128 registers: 26 are spilled)
        if constexpr (V == 1) if (nv > 1024 * 16) hipLaunchKernelGGL((norm_block_kernel<V, 1024, 32>), grid, dim3(1024), 0, s, a, total);
        return;
    }
    const long nslices = cdiv(d.G, gs), total = d.NB * nslices;
    const FastDiv slices = fortis_fast_div((unsigned)nslices);
    const long wv = gs * a.cg / V;
    const dim3 grid((unsigned)(total < 65536 ? total : 65536));
    if (wv <= 256 && d.S <= 256 / wv * 4) hipLaunchKernelGGL((norm_block_groups_kernel<V, 256, 4>), grid, dim3(256), 0, s, a, gs, slices, total);
    else if (d.S <= 1024 / wv * 4) hipLaunchKernelGGL((norm_block_groups_kernel<V, 1024, 4>), grid, dim3(1024), 0, s, a, gs, slices, total);
    else hipLaunchKernelGGL((norm_block_groups_kernel<V, 1024, 8>), grid, dim3(1024), 0, s, a, gs, slices, total);
}
template <int V> static void launch_split(NormArgs a, const SplitShape& h, void* ws, hipStream_t s)
{
    const NormDesc& d = a.d;
    double2* part = (double2*)ws;
    // An output that the eight L2s (32 MB) cannot hold is written past them: it would only push out the input that the second
    // launch is about to read (287496 x 64, 74 MB: 49.7 us through the caches, 40.5 us past them; 65536 x 32, 8 MB: no difference,
    // and the next kernel finds it there).
    const bool stream = d.NB * d.S * d.C * 4 > (32L << 20);
    // A launch has to stay under 2^32 work-items: as many samples at a time as 2^21 workgroups take.
    const long wgs = d.first ? d.G * h.chunks : (long)h.slices * h.blocks * h.chunks, piece = (1L << 21) / wgs;
    for (long n = 0; n < d.NB; n += piece, a.x += piece * d.S * d.C, a.y += piece * d.S * d.C, part += piece * d.G * h.parts) {
        const dim3 grid((unsigned)((d.NB - n < piece ? d.NB - n : piece) * wgs));
        if (d.first) {
            hipLaunchKernelGGL((norm_sums_first_kernel<V>), grid, dim3(GS_THREADS), 0, s, a, h, part);
            if (stream) hipLaunchKernelGGL((norm_apply_first_kernel<V, true>), grid, dim3(GS_THREADS), 0, s, a, h, (const double2*)part);
            else hipLaunchKernelGGL((norm_apply_first_kernel<V, false>), grid, dim3(GS_THREADS), 0, s, a, h, (const double2*)part);
            continue;
        }
        if (a.cg % V == 0) hipLaunchKernelGGL((norm_sums_kernel<V, true>), grid, dim3(GS_THREADS), 0, s, a, h, part);
        else if constexpr (V > 1) hipLaunchKernelGGL((norm_sums_kernel<V, false>), grid, dim3(GS_THREADS), 0, s, a, h, part);
        if (stream) hipLaunchKernelGGL((norm_apply_kernel<V, true>), grid, dim3(GS_THREADS), 0, s, a, h, (const double2*)part);
        else hipLaunchKernelGGL((norm_apply_kernel<V, false>), grid, dim3(GS_THREADS), 0, s, a, h, (const double2*)part);
    }
}

void fortis_launch_group_norm(const NormDesc& in, const float* x, float* y, void* ws, hipStream_t s)
{
    NormArgs a = { norm_normal(in), x, y, in.C / in.G, in.S * (in.C / in.G), {}, fortis_fast_div((unsigned)in.G) };
    const NormDesc& d = a.d;
    const NormForm f = norm_form(d);
    if (f.kind == NORM_SPLIT) {
        const SplitShape h = split_shape(d);
        if (d.first && d.S / h.V < (1L << 31)) a.row = fortis_fast_div((unsigned)(d.S / h.V));
        if (h.V == 4) launch_split<4>(a, h, ws, s);
        else if (h.V == 2) launch_split<2>(a, h, ws, s);
        else launch_split<1>(a, h, ws, s);
    } else {
        a.row = fortis_fast_div((unsigned)((d.first ? d.S : a.cg) / f.V));
        if (f.kind == NORM_LANES) {
            if (f.V == 4) launch_lanes<4>(a, d.NB * d.G, s);
            else if (f.V == 2) launch_lanes<2>(a, d.NB * d.G, s);
            else launch_lanes<1>(a, d.NB * d.G, s);
        } else if (f.V == 4) launch_block<4>(a, f.kind, f.gs, s);
        else if (f.V == 2) launch_block<2>(a, f.kind, f.gs, s);
        else launch_block<1>(a, f.kind, f.gs, s);
    }
    HIP_OK(hipGetLastError());
}

// Gated linear recurrence (include/fortis_step.h, fortis_plan_recurrence):
//     f = 1 / (1 + exp(-g_t)),  h_t = f h_(t-1) + (1 - f) x_t
// per sequence and channel, rows of 2 * ch features (g first, x behind).
//
// Memory-bound: 12 bytes and about 25 instructions a value.  A lane owns one or two neighbouring channels of a sequence and
// walks its steps with two batches of loads in flight.  4736 columns of up to 15 levels of 64 channels: 7.9 us, 3.8 TB/s (with 8 to 15 steps the
// one round's last loads are its own first batch again and the rest's travel behind it); one step: 3.3 us, the launch; 4736 x 60 x 64: 43.7 us, 5.0 TB/s.
// Where sequences and channels alone do not fill the chip, every sequence is cut into K chunks: a step is the map
// h -> f h + b, maps compose to (F, B), so one launch composes every chunk's steps, one wave per sequence and channel scans the
// K compositions and leaves the state in front of every chunk, and a third launch walks the chunks from there: 8 bytes a value
// more.  2 x 32768 steps of 384 channels: 90 us = 37 (201 MB at 5.4 TB/s) + 5 + 48 (302 MB at 6.3, the input partly from the
// memory-side cache); in one read it could not be under 57 us at a copy's rate.  (Reading once would take chunks handed out by an
// atomic ticket, each waiting only for chunks that running workgroups hold; not built.)
// All compositions happen in a fixed order: results repeat bit for bit.
#include "common.h"

#define RC_THREADS 256
#define RC_AHEAD 4              // steps whose loads are in flight together

typedef float v2f __attribute__((ext_vector_type(2)));
template <int V> struct VecOf { typedef float T; };
template <> struct VecOf<2> { typedef v2f T; };

struct RecurArgs {
    RecurDesc d;
    const float* src;
    float* dst;
    const float* h_in;
    float* h_out;
    const int* lengths;
    float2* maps;               // [nseq * ch][chunks]: (F, B) of a chunk, then (h in front of it, unused)
    long chunks, per;           // chunks of a sequence, steps a chunk
    long first;                 // lane that the launch starts with
};

template <int V> __device__ __forceinline__ void load(float (&o)[V], const float* p)
{
    const typename VecOf<V>::T t = *(const typename VecOf<V>::T*)p;
    __builtin_memcpy(o, &t, sizeof t);
}
template <int V, bool STREAM> __device__ __forceinline__ void store(float* p, const float (&o)[V])
{
    typename VecOf<V>::T t;
    __builtin_memcpy(&t, o, sizeof t);
    if constexpr (STREAM) __builtin_nontemporal_store(t, (typename VecOf<V>::T*)p);
    else *(typename VecOf<V>::T*)p = t;
}
__device__ __forceinline__ long steps_of(const RecurArgs& a, long s)
{
    if (!a.lengths) return a.d.len;
    const long l = a.lengths[s];
    return l < 0 ? 0 : l < a.d.len ? l : a.d.len;
}

// One lane, V channels, the steps of one chunk.  APPLY: from the state in front, writing every step; otherwise the map of the
// chunk's steps.
template <int V, bool APPLY, bool STREAM>
__global__ __launch_bounds__(RC_THREADS) void recurrence_walk_kernel(RecurArgs a)
{
    const RecurDesc& d = a.d;
    const long lanes = d.nseq * d.ch / V;
    const long id = a.first + (long)blockIdx.x * RC_THREADS + threadIdx.x;
    if (id >= lanes * a.chunks) return;
    const long k = id / lanes, e = (id - k * lanes) * V;      // chunk, first of the lane's values in [nseq][ch]
    const long s = e / d.ch, c = e - s * d.ch;
    const long len = steps_of(a, s);
    const long i0 = k * a.per, i1 = i0 + a.per < len ? i0 + a.per : len;
    float h[V], F[V];
#pragma unroll
    for (int v = 0; v < V; v++) { h[v] = -0.f; F[v] = 1.f; }     // the identity to the bit: 1 h + -0 is h, also for h = -0
    if (APPLY) {
        if (a.chunks > 1) {
#pragma unroll
            for (int v = 0; v < V; v++) h[v] = a.maps[(e + v) * a.chunks + k].x;
        } else if (a.h_in) load<V>(h, a.h_in + e);
        else {
#pragma unroll
            for (int v = 0; v < V; v++) h[v] = 0.f;
        }
    }
    if (i0 < i1) {
        const long row0 = d.time_major ? s : s * d.len, rstep = d.time_major ? d.nseq : 1;
        const long t0 = d.reverse ? len - 1 - i0 : i0, dir = d.reverse ? -rstep : rstep;
        const float* p = a.src + (row0 + t0 * rstep) * 2 * d.ch + c;
        float* q = a.dst + (row0 + t0 * rstep) * d.ch + c;
        const long ps = dir * 2 * d.ch, qs = dir * d.ch, n = i1 - i0;
        float g[2][RC_AHEAD][V], x[2][RC_AHEAD][V];
        auto step = [&](int set, int u, float* at) __attribute__((always_inline)) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                float hi, lo;
                const float gv = g[set][u][v];
                fortis_sigmoids<false>(gv, hi, lo);
                const float f = gv >= 0.f ? hi : lo, b = (gv >= 0.f ? lo : hi) * x[set][u][v];
                h[v] = fmaf(f, h[v], b);
                if (!APPLY) F[v] *= f;
            }
            if (APPLY) store<V, STREAM>(at, h);
        };
        // Two register sets: a batch's loads are issued before the batch in front of it is worked on.  No branch goes round a load
        // in this loop (the last round reads its own first batch again): one would make every wait a wait for all loads in flight.
        auto fetch = [&](int set, const float* at) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < RC_AHEAD; u++) { load<V>(g[set][u], at + u * ps); load<V>(x[set][u], at + u * ps + d.ch); }
        };
        const long rounds = n / (2 * RC_AHEAD);
        if (rounds > 0) fetch(0, p);
        for (long r = 0; r < rounds; r++) {
            fetch(1, p + RC_AHEAD * ps);
#pragma unroll
            for (int u = 0; u < RC_AHEAD; u++) step(0, u, q + u * qs);
            const float* next = r + 1 < rounds ? p + 2 * RC_AHEAD * ps : p;
            fetch(0, next);
#pragma unroll
            for (int u = 0; u < RC_AHEAD; u++) step(1, u, q + (RC_AHEAD + u) * qs);
            p += 2 * RC_AHEAD * ps;
            q += 2 * RC_AHEAD * qs;
        }
        const int rest = (int)(n - rounds * 2 * RC_AHEAD);
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int u = 0; u < RC_AHEAD; u++)
                if (k * RC_AHEAD + u < rest) { load<V>(g[k][u], p + (k * RC_AHEAD + u) * ps); load<V>(x[k][u], p + (k * RC_AHEAD + u) * ps + d.ch); }
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int u = 0; u < RC_AHEAD; u++)
                if (k * RC_AHEAD + u < rest) step(k, u, q + (k * RC_AHEAD + u) * qs);
    }
    if (APPLY) {
        if (a.chunks == 1 && a.h_out) store<V, false>(a.h_out + e, h);
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) a.maps[(e + v) * a.chunks + k] = make_float2(F[v], h[v]);
    }
}

// One wave per (sequence, channel): the maps of its chunks become the states in front of them.
__global__ __launch_bounds__(RC_THREADS) void recurrence_scan_kernel(RecurArgs a)
{
    const long e = (long)blockIdx.x * (RC_THREADS / 64) + (threadIdx.x >> 6);
    if (e >= a.d.nseq * a.d.ch) return;
    const int lane = threadIdx.x & 63;
    const long q = (a.chunks + 63) / 64, k0 = lane * q, k1 = k0 + q < a.chunks ? k0 + q : a.chunks;
    float2* m = a.maps + e * a.chunks;
    float F = 1.f, B = -0.f;
    for (long k = k0; k < k1; k++) { const float2 w = m[k]; B = fmaf(w.x, B, w.y); F *= w.x; }
    // inclusive scan over the lanes: (F, B) after (Fp, Bp) is (F Fp, F Bp + B)
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const float Fp = __shfl_up(F, o, 64), Bp = __shfl_up(B, o, 64);
        if (lane >= o) { B = fmaf(F, Bp, B); F *= Fp; }
    }
    const float h0 = a.h_in ? a.h_in[e] : 0.f;
    if (a.h_out && lane == 63) a.h_out[e] = fmaf(F, h0, B);
    float Fx = __shfl_up(F, 1, 64), Bx = __shfl_up(B, 1, 64);
    if (lane == 0) { Fx = 1.f; Bx = -0.f; }
    float h = fmaf(Fx, h0, Bx);
    for (long k = k0; k < k1; k++) {
        const float2 w = m[k];
        m[k] = make_float2(h, 0.f);
        h = fmaf(w.x, h, w.y);
    }
}

struct RecurShape { int V; long chunks, per; };
static RecurShape recur_shape(const RecurDesc& d)
{
    RecurShape r;
    const long values = d.nseq * d.ch, full = 256 * 8 * 64;      // lanes that keep the memory busy: eight waves a compute unit (twelve and sixteen: no faster)
    // One channel a lane until two still give every SIMD four waves: 4736 x 64 values over 15 and 60 levels take 8.0 and 43.5 us with
    // one, 9.4 and 45.7 with two (four: 10.6 and 54).
    r.V = d.ch % 2 == 0 && values / 2 >= 2 * full ? 2 : 1;
    r.chunks = 1;
    // One chunk costs 70 ns a step, two more launches 5 us: 64, 128 and 512 steps of 1 x 64 channels take 6.0, 10.1 and 36.7 us in one chunk,
    // 7.9, 8.1 and 8.9 in chunks of 8, 8.8, 8.9 and 9.7 of 16, 10.8, 11.0 and 11.6 of 32.  Where the scan has many to go through longer chunks
    // win: 4 x 4096 steps of 64 take 15.1, 12.2 and 12.8 us.  One walk against chunks, us at 100, 200 and 1000 steps:
    //   4096 values   9.8 : 9.5   17 : 10.8   87 : 20          32768 values  11.4 : 19.7   21 : 31   92 : 93
    //   16384 values  10.5 : 14.6   19 : 17.7   88 : 51        65472 values  13.8 : 36.5   23 : 53   174 : 242
    // From about 16384 values on the limit on their number asks for chunks too soon where the sequences are short, from 32768 on always.
    const long least = d.len > 512 ? 16 : 8;
    if (d.len > 96 && values / r.V < full / 2) r.chunks = cdiv(full, values / r.V);
    if (r.chunks > cdiv(d.len, least)) r.chunks = cdiv(d.len, least);
    r.per = cdiv(d.len, r.chunks);
    r.chunks = cdiv(d.len, r.per);
    return r;
}

long fortis_recurrence_workspace(const RecurDesc& d)
{
    const RecurShape r = recur_shape(d);
    return r.chunks > 1 ? d.nseq * d.ch * r.chunks * (long)sizeof(float2) : 0;
}

// A launch has to stay under 2^32 work-items.
#define RC_PIECE (1L << 31)
template <class K> static void launch_walk(K kernel, RecurArgs a, long lanes, hipStream_t s)
{
    for (a.first = 0; a.first < lanes; a.first += RC_PIECE) {
        const long n = lanes - a.first < RC_PIECE ? lanes - a.first : RC_PIECE;
        hipLaunchKernelGGL(kernel, dim3((unsigned)cdiv(n, RC_THREADS)), dim3(RC_THREADS), 0, s, a);
    }
}
template <int V> static void launch_walks(const RecurArgs& a, hipStream_t s)
{
    const long lanes = a.d.nseq * a.d.ch / V * a.chunks;
    if (a.chunks > 1) {
        launch_walk(recurrence_walk_kernel<V, false, false>, a, lanes, s);
        hipLaunchKernelGGL(recurrence_scan_kernel, dim3((unsigned)cdiv(a.d.nseq * a.d.ch, RC_THREADS / 64)), dim3(RC_THREADS), 0, s, a);
    }
    // an output that the eight L2s (32 MB) cannot hold is written past them: 106 -> 96 us for 2 x 32768 x 384
    if (a.d.nseq * a.d.len * a.d.ch * 4 > (32L << 20)) launch_walk(recurrence_walk_kernel<V, true, true>, a, lanes, s);
    else launch_walk(recurrence_walk_kernel<V, true, false>, a, lanes, s);
}
void fortis_launch_recurrence(const RecurDesc& d, const float* src, float* dst, const float* h_in, float* h_out, const int* lengths, void* ws, hipStream_t s)
{
    const RecurShape r = recur_shape(d);
    const RecurArgs a = { d, src, dst, h_in, h_out, lengths, (float2*)ws, r.chunks, r.per, 0 };
    if (r.V == 2) launch_walks<2>(a, s);
    else launch_walks<1>(a, s);
    HIP_OK(hipGetLastError());
}

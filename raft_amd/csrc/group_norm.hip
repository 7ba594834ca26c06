// Group normalisation with an activation, channels last, forward and backward.
//
// x is a matrix of N*P rows (sample n, position p) of C channels; groups of D = C / G neighbouring channels share mean and
// variance over P*D values:
//   xh = (x - mean) * rstd,  z = xh * w[c] + b[c],  y = act(z)
//   g = dy * act'(z):  db[c] = sum g,  dw[c] = sum g * xh,
//   dx = rstd * (g * w - s1 - xh * s2),  s1 = mean over the group of g * w,  s2 = mean over the group of g * w * xh.
// Memory bound: 8 operations a value forward, some 20 backward.
// A workgroup that can hold all rows of a sample's channel slab in registers reads them once and does everything in one launch.
// Else there are three: sums of row ranges per channel, one small launch that joins them per group, one pass that writes.  That
// pass reads x again out of the 256 MB last-level cache as far as it fits; it loads and stores past the replacement order, so the
// results do not displace what is still to be read (12 x 64 x 200 x 360 float32, forward: 75 us that pass without it, 65 with).
#include "common.h"
#include "elem.h"
#include <type_traits>

namespace raftcorr {

// How the rows of one sample are dealt to the threads of a workgroup.  T threads read T vectors of V elements in a row, which is
// R = T * V / Cs whole rows of the slab's Cs channels; one iteration later a thread is R rows further and on the same channels.
// Vectors may run over the end of a row where rows are dense (Cs == C == row stride): any channel count is read in full vectors.
struct NormGeom {
    int64_t P;                   // rows a sample
    int64_t x_batch, x_row;      // strides in elements
    int64_t d_batch, d_row;      // the same of dy (backward)
    int C, G, D, N;
    int Cs, nslab;               // channels of a slab (the last may be smaller), slabs
    int T, R;                    // threads at work, rows an iteration (first slabs)
    int S;                       // row ranges a sample is split into
    int64_t rows;                // rows of a range
    int n0, n1;                  // first sample and samples of a launch
};

enum {
    kThreads = 256,
    kWaves = 4,                  // workgroups a CU (registers: 128 a thread)
    kUnroll = 4,                 // vectors of x that a thread has on their way at once, forward
    kMostRanges = 1024,          // workgroups of a pass over everything ...
    kFewRanges = 768,            // ... and while these leave a range below kRangeBytes: each workgroup costs a launch, its coefficients and a join
    kRangeBytes = 192 << 10,     // (forward + backward in us; 12 x 128 x 50 x 90 float16: 17.2 + 22.9, with 1024 18.7 + 24.1;
                                 // 12 x 64 x 200 x 360 float32: with 512 117 + 199, with 1024 109 + 184)
};

// the same backward, of x and of dy each
template <int V> constexpr int unroll_bwd() { return V == 8 ? 2 : 4; }

static int gcd_(int a, int b) { while (b) { const int t = a % b; a = b; b = t; } return a; }

// slab widths for vectors of V: whole rows if their pattern fits the workgroup, else column slabs of 256 vectors
static void slab_geom(NormGeom& g, int V)
{
    const int pattern = g.C / gcd_(g.C, V);          // threads after which the channel pattern repeats
    if (pattern <= kThreads) {
        g.Cs = g.C; g.nslab = 1;
        // 8 vectors of 16 bytes are a line: rounds of whole lines, or two rounds would each write a part of one
        // (96 channels in 16 bits, 2 x 272 x 480: the writing pass takes 16 us with 240 threads, 21 with 252)
        const int lines = pattern * (8 / gcd_(pattern, 8));
        g.T = lines <= kThreads ? kThreads / lines * lines : kThreads / pattern * pattern;
    } else {
        g.Cs = V * kThreads; g.nslab = (g.C + g.Cs - 1) / g.Cs;
        g.T = kThreads;
    }
    g.R = g.T * V / g.Cs;
}

// the slab of this workgroup: first channel, width, threads, rows an iteration
template <int V> __device__ __forceinline__ void slab_of(const NormGeom& g, int slab, int& c0, int& cs, int& T, int& R)
{
    c0 = slab * g.Cs;
    cs = min(g.Cs, g.C - c0);
    T = g.T; R = g.R;
    if (cs != g.Cs) { const int cols = cs / V; R = kThreads / cols; T = R * cols; }   // last slab: V divides its width (or V == 1)
}

// Row lane and column of each of a thread's V slots (slot j: value t * V + j of a round), by one division and counting.
template <int V> struct Slots {
    int lane[V], col[V];
    __device__ __forceinline__ Slots(int t, int cs)
    {
        const unsigned f = (unsigned)t * V;
        int l = (int)(f / (unsigned)cs), k = (int)(f % (unsigned)cs);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            lane[j] = l; col[j] = k;
            if (++k == cs) { k = 0; ++l; }                          // only where the slab is the whole row
        }
    }
};

// sum over the row lanes of a quantity of each slot: slot f = t * V + j of thread t holds channel f % cs, row lane f / cs.
// buf: blockDim * V values; afterwards buf[c] is channel c's sum.  Fixed order.
template <int V, typename S> __device__ __forceinline__ void reduce_columns(const S (&val)[V], S* buf, int T, int R, int cs)
{
    const int t = threadIdx.x;
    __syncthreads();
    if (t < T)
#pragma unroll
        for (int j = 0; j < V; ++j) buf[t * V + j] = val[j];
    for (int rows = R; rows > 1;) {
        const int half = (rows + 1) / 2;
        __syncthreads();
        for (int f = t; f < (rows - half) * cs; f += blockDim.x) buf[f] += buf[f + half * cs];
        rows = half;
    }
    __syncthreads();
}

// Tensors beyond the last-level cache (256 MB) leave it with what a pass read last, and the next pass begins there (`backwards`).
// What it could not hold anyway goes past it instead of displacing the rest: a summing pass keeps only its last kKept bytes, from
// the workgroup `kept` on, and streams the others.  Forward of 802 MB float32 with its reading order 406 us | 420 without both;
// backward of 221 MB twice 176 | 184, of 802 MB twice 675 | 698, of 200 MB bfloat16 twice 168 | 176.
// Kept 128 MB: 423, 181, 691, 172; 160: 420, 178, 685, 169; 192: 411, 177, 679, 166; 240: 404, 177, 670, 170.
// Below 256 MB nothing is streamed: forward of 252 MB 124 us | 130, backward of 126 MB twice 104 | 117.
constexpr int64_t kCache = 256LL << 20, kKept = 224LL << 20;

template <bool ONCE, typename T_, int V>
__device__ __forceinline__ void load_next(Vec<T_, V>& v, const T_*& p, int64_t step)
{
    v = ONCE ? load_vec_once<T_, V>(p) : load_vec<T_, V>(p);
    p += step;
}

// first of a summing launch's workgroups whose rows stay in the cache; bytes: of all that the pass reads
static unsigned kept_from(int64_t bytes, unsigned blocks)
{
    return bytes <= kCache ? 0 : blocks - (unsigned)((double)blocks * kKept / (double)bytes);
}

// ---- forward ------------------------------------------------------------------------------------------------------------

// Sum and sum of squares of each channel over one row range -> part[n][s][c].  In 64 bits (full rate here, three operations a value):
// no mean is large enough to cancel the squares, and the statistics are exact enough for ReLU's gradient to tell on which side of
// zero each z lies (see NormCoef).
template <typename T_, int V>
__global__ __launch_bounds__(kThreads, kWaves) void norm_stats_kernel(const T_* __restrict__ x, NormGeom g, double2* __restrict__ part,
                                                              unsigned kept)
{
    constexpr int U = kUnroll;
    __shared__ double buf[kThreads * V];
    const int s = blockIdx.x % g.S, slab = blockIdx.x / g.S % g.nslab;
    const int64_t n = g.n0 + blockIdx.x / g.S / g.nslab;
    int c0, cs, T, R;
    slab_of<V>(g, slab, c0, cs, T, R);
    const int t = threadIdx.x;
    const int64_t r1 = min(g.P, (s + 1) * g.rows);
    double sum[V] = {}, squares[V] = {};
    if (t < T) {
        const Slots<V> q(t, cs);
        const int (&lane)[V] = q.lane;
        auto add = [&](T_ e, int j) {
            const double d = (double)to_float(e);
            sum[j] += d;
            squares[j] += d * d;
        };
        const int64_t step = (int64_t)R * g.x_row;
        int64_t r = s * g.rows;
        const T_* p = x + n * g.x_batch + (r + lane[0]) * g.x_row + c0 + q.col[0];
        for (; r + (int64_t)U * R <= r1; r += U * R) {
            Vec<T_, V> v[U];
            if (blockIdx.x >= kept) {
#pragma unroll
                for (int u = 0; u < U; ++u) load_next<false, T_, V>(v[u], p, step);
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u) load_next<true, T_, V>(v[u], p, step);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < V; ++j) add(v[u][j], j);
        }
        // what is left, all loads at once again; a vector that the range's end cuts comes value by value
        Vec<T_, V> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u * R + lane[V - 1] < r1) v[u] = load_vec<T_, V>(p + u * step);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = r + u * R;
            if (at + lane[V - 1] < r1) {
#pragma unroll
                for (int j = 0; j < V; ++j) add(v[u][j], j);
            } else if (at + lane[0] < r1) {
                for (int j = 0; j < V; ++j)
                    if (at + lane[j] < r1) add(p[u * step + j], j);
            }
        }
    }
    double2* out = part + (n * g.S + s) * g.C + c0;
    reduce_columns<V>(sum, buf, T, R, cs);
    for (int c = t; c < cs; c += kThreads) out[c].x = buf[c];
    reduce_columns<V>(squares, buf, T, R, cs);
    for (int c = t; c < cs; c += kThreads) out[c].y = buf[c];
}

template <typename S> __device__ __forceinline__ S wave_sum(S v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// sum of v over the workgroup's threads (whole waves), in every thread; buf: one value a wave
template <typename S> __device__ __forceinline__ S block_sum(S v, S* buf)
{
    v = wave_sum(v);
    const int waves = blockDim.x / 64;
    if (waves == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x / 64] = v;
    __syncthreads();
    v = buf[0];
    for (int w = 1; w < waves; ++w) v += buf[w];
    return v;
}

// (mean, rstd) from a group's sum and sum of squares, inv = 1 / (P D)
__device__ __forceinline__ double2 statistics(double sum, double squares, double inv, double eps)
{
    const double mean = sum * inv, var = squares * inv - mean * mean;
    return make_double2(mean, 1.0 / sqrt((var < 0.0 ? 0.0 : var) + eps));       // (a NaN stays one)
}

// part -> (mean, rstd) of each (n, group); one workgroup each, so that all its reads are on their way at once
__global__ __launch_bounds__(1024) void norm_join_kernel(const double2* __restrict__ part, NormGeom g, double eps, double2* __restrict__ stats)
{
    __shared__ double buf[16];
    const int64_t n = g.n0 + blockIdx.x / (unsigned)g.G;
    const unsigned group = blockIdx.x % (unsigned)g.G;
    const double2* p = part + n * g.S * g.C + (int64_t)group * g.D;
    const unsigned count = (unsigned)g.S * g.D, D = g.D;
    double a = 0.0, q = 0.0;
#pragma unroll 4
    for (unsigned k = threadIdx.x; k < count; k += blockDim.x) {
        const double2 v = p[(int64_t)(k / D) * g.C + k % D];
        a += v.x;
        q += v.y;
    }
    a = block_sum(a, buf);
    q = block_sum(q, buf);
    if (threadIdx.x == 0) stats[n * g.G + group] = statistics(a, q, 1.0 / ((double)g.P * (double)g.D), eps);
}

template <int ACT> __device__ __forceinline__ float activate(float z)
{
    if (ACT == RAFTCORR_ACT_RELU) return z < 0.f ? 0.f : z;                    // (a NaN stays one)
    if (ACT == RAFTCORR_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + expf(-z));
    return z;
}

template <int ACT> __device__ __forceinline__ float slope(float z)
{
    if (ACT == RAFTCORR_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + expf(-z));
        return s * (1.f + z * (1.f - s));
    }
    return 1.f;
}

// What the slots need of their channels is worked out once a channel and handed to them through shared memory: with loads by every
// slot for itself 12 x 128 x 50 x 90 float16 takes 20.1 us forward and 28.1 backward, this way 17.2 and 22.9.
// [mean][rstd w][b], each cs floats
__device__ __forceinline__ void stage_forward(float* lds, int c, int cs, double2 st, const float* weight, const float* bias, int channel)
{
    lds[c] = (float)st.x;
    lds[cs + c] = (float)st.y * (weight ? weight[channel] : 1.f);
    lds[2 * cs + c] = bias ? bias[channel] : 0.f;
}

extern __shared__ float staged[];

template <typename T_, int V, int ACT>
__global__ __launch_bounds__(kThreads, kWaves) void norm_apply_kernel(const T_* __restrict__ x, NormGeom g, const double2* __restrict__ stats,
                                                              const float* __restrict__ weight, const float* __restrict__ bias,
                                                              T_* __restrict__ y, int backwards)
{
    constexpr int U = kUnroll;
    const unsigned block = backwards ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    const int s = block % g.S, slab = block / g.S % g.nslab;
    const int64_t n = g.n0 + block / g.S / g.nslab;
    int c0, cs, T, R;
    slab_of<V>(g, slab, c0, cs, T, R);
    const int t = threadIdx.x;
    for (int c = t; c < cs; c += kThreads) stage_forward(staged, c, cs, stats[n * g.G + (c0 + c) / g.D], weight, bias, c0 + c);
    __syncthreads();
    if (t >= T) return;
    const int64_t r1 = min(g.P, (s + 1) * g.rows);
    float mean[V], a[V], b[V];
    const Slots<V> q(t, cs);
    const int (&lane)[V] = q.lane;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        mean[j] = staged[q.col[j]];
        a[j] = staged[cs + q.col[j]];
        b[j] = staged[2 * cs + q.col[j]];
    }
    const int64_t step = (int64_t)R * g.x_row, ystep = (int64_t)R * g.C;
    const T_* p = x + n * g.x_batch + (s * g.rows + lane[0]) * g.x_row + c0 + q.col[0];
    T_* o = y + (n * g.P + s * g.rows + lane[0]) * g.C + c0 + q.col[0];
    int64_t r = s * g.rows;
    for (; r + (int64_t)U * R <= r1; r += U * R) {
        Vec<T_, V> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) { v[u] = load_vec_once<T_, V>(p); p += step; }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Vec<T_, V> w;
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = from_float<T_>(activate<ACT>((to_float(v[u][j]) - mean[j]) * a[j] + b[j]));
            store_vec_once<T_, V>(o, w);
            o += ystep;
        }
    }
    Vec<T_, V> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (r + u * R + lane[V - 1] < r1) v[u] = load_vec_once<T_, V>(p + u * step);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = r + u * R;
        if (at + lane[V - 1] < r1) {
            Vec<T_, V> w;
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = from_float<T_>(activate<ACT>((to_float(v[u][j]) - mean[j]) * a[j] + b[j]));
            store_vec_once<T_, V>(o + u * ystep, w);
        } else if (at + lane[0] < r1) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (at + lane[j] < r1) o[u * ystep + j] = from_float<T_>(activate<ACT>((to_float(p[u * step + j]) - mean[j]) * a[j] + b[j]));
        }
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------------

// What a channel's slots need.  ReLU passes a gradient where z = (x - mean) rstd w + b > 0, that is where x is above (for w < 0:
// below) the point mean - b / (rstd w).  That point is computed in 64 bits and rounded down to a float32 `edge`, and x, with its
// sign turned for w < 0, is compared with it: the right side for every x, one operation instead of two.  With z in float32 one in
// some 10^8 values would land on the wrong side, and its whole gradient with it.
//   g = dy act'(z):  ReLU: dy where x * k0 > k1 (turn, edge);  SiLU: z = (x - mean) * k0 + k1 (rstd w, b)
//   dx = g * a - b - (x - mean) * c,  a = rstd w, b = rstd s1, c = rstd^2 s2
enum { kMean, kSlope0, kSlope1, kSums, kA = kSums, kB, kC, kFields };          // rows of `staged`; the sums need the first three

__device__ __forceinline__ float round_down(double d)
{
    const float f = (float)d;
    if (!((double)f > d)) return f;
    const uint32_t u = __float_as_uint(f);
    return __uint_as_float(f > 0.f ? u - 1 : f < 0.f ? u + 1 : 0x80000001u);
}

template <int ACT>
__device__ __forceinline__ void stage_backward(float* lds, int c, int cs, double2 st, const float* weight, const float* bias, int channel)
{
    const float w = weight ? weight[channel] : 1.f, b = bias ? bias[channel] : 0.f;
    lds[kMean * cs + c] = (float)st.x;
    if (ACT == RAFTCORR_ACT_RELU) {
        const float turn = w < 0.f ? -1.f : 1.f;
        const double at = st.x - (b != 0.f ? (double)b / ((double)w * st.y) : 0.0);
        lds[kSlope0 * cs + c] = turn;
        lds[kSlope1 * cs + c] = w == 0.f ? (b > 0.f ? -__builtin_inff() : __builtin_inff()) : round_down(turn * at);
    } else if (ACT == RAFTCORR_ACT_SILU) {
        lds[kSlope0 * cs + c] = (float)st.y * w;
        lds[kSlope1 * cs + c] = b;
    }
}

__device__ __forceinline__ void stage_gradient(float* lds, int c, int cs, double2 st, const float* weight, float s1, float s2, int channel)
{
    const float rstd = (float)st.y;
    lds[kA * cs + c] = rstd * (weight ? weight[channel] : 1.f);
    lds[kB * cs + c] = rstd * s1;
    lds[kC * cs + c] = rstd * rstd * s2;
}

// a slot's share of them
template <int ACT> struct NormCoef {
    float mean, k0, k1;
    __device__ __forceinline__ void take(const float* lds, int col, int cs)
    {
        mean = lds[kMean * cs + col];
        k0 = ACT == RAFTCORR_ACT_NONE ? 0.f : lds[kSlope0 * cs + col];
        k1 = ACT == RAFTCORR_ACT_NONE ? 0.f : lds[kSlope1 * cs + col];
    }
    // g = dy * act'(z), d = x - mean
    __device__ __forceinline__ float through(float x, float d, float dy) const
    {
        if (ACT == RAFTCORR_ACT_RELU) return x * k0 > k1 ? dy : 0.f;
        return dy * slope<ACT>(d * k0 + k1);
    }
};

// sum of g and of g * xh of each channel over one row range -> part[n][s][c]
template <typename T_, int V, int ACT>
__global__ __launch_bounds__(kThreads, kWaves) void norm_bwd_sums_kernel(const T_* __restrict__ x, const T_* __restrict__ dy, NormGeom g,
                                                                 const double2* __restrict__ stats, const float* __restrict__ weight,
                                                                 const float* __restrict__ bias, float2* __restrict__ part,
                                                                 unsigned kept)
{
    constexpr int U = unroll_bwd<V>();
    __shared__ float buf[kThreads * V];
    const int s = blockIdx.x % g.S, slab = blockIdx.x / g.S % g.nslab;
    const int64_t n = g.n0 + blockIdx.x / g.S / g.nslab;
    int c0, cs, T, R;
    slab_of<V>(g, slab, c0, cs, T, R);
    const int t = threadIdx.x;
    const int64_t r1 = min(g.P, (s + 1) * g.rows);
    for (int c = t; c < cs; c += kThreads) stage_backward<ACT>(staged, c, cs, stats[n * g.G + (c0 + c) / g.D], weight, bias, c0 + c);
    __syncthreads();
    float sum[V] = {}, dot[V] = {};                          // of g and of g * (x - mean)
    if (t < T) {
        NormCoef<ACT> k[V];
        const Slots<V> q(t, cs);
        const int (&lane)[V] = q.lane;
#pragma unroll
        for (int j = 0; j < V; ++j) k[j].take(staged, q.col[j], cs);
        auto add = [&](float xv, float dv, int j, float& a, float& b) {
            const float d = xv - k[j].mean, e = k[j].through(xv, d, dv);
            a += e;
            b += e * d;
        };
        const int64_t step = (int64_t)R * g.x_row, dstep = (int64_t)R * g.d_row;
        const T_* p = x + n * g.x_batch + (s * g.rows + lane[0]) * g.x_row + c0 + q.col[0];
        const T_* d = dy + n * g.d_batch + (s * g.rows + lane[0]) * g.d_row + c0 + q.col[0];
        int64_t r = s * g.rows;
        for (; r + (int64_t)U * R <= r1; r += U * R) {
            Vec<T_, V> v[U], w[U];
            if (blockIdx.x >= kept) {
#pragma unroll
                for (int u = 0; u < U; ++u) { load_next<false, T_, V>(v[u], p, step); load_next<false, T_, V>(w[u], d, dstep); }
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u) { load_next<true, T_, V>(v[u], p, step); load_next<true, T_, V>(w[u], d, dstep); }
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float a = 0.f, b = 0.f;                      // the chunk by itself first: long sums lose less
#pragma unroll
                for (int u = 0; u < U; ++u) add(to_float(v[u][j]), to_float(w[u][j]), j, a, b);
                sum[j] += a;
                dot[j] += b;
            }
        }
        Vec<T_, V> v[U], w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u * R + lane[V - 1] < r1) {
                v[u] = load_vec<T_, V>(p + u * step);
                w[u] = load_vec<T_, V>(d + u * dstep);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = r + u * R;
            if (at + lane[V - 1] < r1) {
#pragma unroll
                for (int j = 0; j < V; ++j) add(to_float(v[u][j]), to_float(w[u][j]), j, sum[j], dot[j]);
            } else if (at + lane[0] < r1) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (at + lane[j] < r1) add(to_float(p[u * step + j]), to_float(d[u * dstep + j]), j, sum[j], dot[j]);
            }
        }
    }
    float2* out = part + (n * g.S + s) * g.C + c0;
    reduce_columns<V>(sum, buf, T, R, cs);
    for (int c = t; c < cs; c += kThreads) out[c].x = buf[c];
    reduce_columns<V>(dot, buf, T, R, cs);
    for (int c = t; c < cs; c += kThreads) out[c].y = buf[c] * (float)stats[n * g.G + (c0 + c) / g.D].y;
}

// part -> (s1, s2) of each (n, group) and, in further workgroups with dweight / dbias, a channel's sums over all samples
__global__ __launch_bounds__(1024) void norm_bwd_join_kernel(const float2* __restrict__ part, NormGeom g, const float* __restrict__ weight,
                                                             float2* __restrict__ coef, float* __restrict__ dweight, float* __restrict__ dbias)
{
    __shared__ float buf[16];
    const unsigned T = blockDim.x, groups = (unsigned)g.n1 * g.G;
    float a = 0.f, b = 0.f;
    if (blockIdx.x < groups) {
        const int64_t n = g.n0 + blockIdx.x / (unsigned)g.G;
        const unsigned group = blockIdx.x % (unsigned)g.G;
        const int c0 = (int)group * g.D;
        const float2* p = part + n * g.S * g.C + c0;
        const unsigned count = (unsigned)g.S * g.D, D = g.D;
#pragma unroll 4
        for (unsigned k = threadIdx.x; k < count; k += T) {
            const unsigned c = k % D;
            const float2 v = p[(int64_t)(k / D) * g.C + c];
            const float w = weight ? weight[c0 + c] : 1.f;
            a += v.x * w;
            b += v.y * w;
        }
        const float inv = 1.f / ((float)g.P * (float)g.D);
        a = block_sum(a, buf) * inv;
        b = block_sum(b, buf) * inv;
        if (threadIdx.x == 0) coef[n * g.G + group] = make_float2(a, b);
        return;
    }
    const unsigned c = blockIdx.x - groups;
#pragma unroll 4
    for (int64_t k = threadIdx.x; k < (int64_t)g.N * g.S; k += T) {
        const float2 v = part[k * g.C + c];
        a += v.x;
        b += v.y;
    }
    a = block_sum(a, buf);
    b = block_sum(b, buf);
    if (threadIdx.x == 0) {
        if (dbias) dbias[c] = a;
        if (dweight) dweight[c] = b;
    }
}

template <typename T_, int V, int ACT>
__global__ __launch_bounds__(kThreads, kWaves) void norm_bwd_apply_kernel(const T_* __restrict__ x, const T_* __restrict__ dy, NormGeom g,
                                                                  const double2* __restrict__ stats, const float* __restrict__ weight,
                                                                  const float* __restrict__ bias, const float2* __restrict__ coef,
                                                                  T_* __restrict__ dx, int backwards)
{
    constexpr int U = unroll_bwd<V>();
    const unsigned block = backwards ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    const int s = block % g.S, slab = block / g.S % g.nslab;
    const int64_t n = g.n0 + block / g.S / g.nslab;
    int c0, cs, T, R;
    slab_of<V>(g, slab, c0, cs, T, R);
    const int t = threadIdx.x;
    for (int c = t; c < cs; c += kThreads) {
        const int64_t group = n * g.G + (c0 + c) / g.D;
        stage_backward<ACT>(staged, c, cs, stats[group], weight, bias, c0 + c);
        stage_gradient(staged, c, cs, stats[group], weight, coef[group].x, coef[group].y, c0 + c);
    }
    __syncthreads();
    if (t >= T) return;
    const int64_t r1 = min(g.P, (s + 1) * g.rows);
    NormCoef<ACT> k[V];
    float ka[V], kb[V], kc[V];
    const Slots<V> q(t, cs);
    const int (&lane)[V] = q.lane;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        k[j].take(staged, q.col[j], cs);
        ka[j] = staged[kA * cs + q.col[j]];
        kb[j] = staged[kB * cs + q.col[j]];
        kc[j] = staged[kC * cs + q.col[j]];
    }
    auto grad = [&](float xv, float dv, int j) {
        const float d = xv - k[j].mean;
        return k[j].through(xv, d, dv) * ka[j] - kb[j] - d * kc[j];
    };
    const int64_t step = (int64_t)R * g.x_row, dstep = (int64_t)R * g.d_row, ostep = (int64_t)R * g.C;
    const T_* p = x + n * g.x_batch + (s * g.rows + lane[0]) * g.x_row + c0 + q.col[0];
    const T_* d = dy + n * g.d_batch + (s * g.rows + lane[0]) * g.d_row + c0 + q.col[0];
    T_* o = dx + (n * g.P + s * g.rows + lane[0]) * g.C + c0 + q.col[0];
    int64_t r = s * g.rows;
    for (; r + (int64_t)U * R <= r1; r += U * R) {
        Vec<T_, V> v[U], w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u] = load_vec_once<T_, V>(p); p += step;
            w[u] = load_vec_once<T_, V>(d); d += dstep;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Vec<T_, V> f;
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = from_float<T_>(grad(to_float(v[u][j]), to_float(w[u][j]), j));
            store_vec_once<T_, V>(o, f);
            o += ostep;
        }
    }
    Vec<T_, V> v[U], w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (r + u * R + lane[V - 1] < r1) {
            v[u] = load_vec_once<T_, V>(p + u * step);
            w[u] = load_vec_once<T_, V>(d + u * dstep);
        }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = r + u * R;
        if (at + lane[V - 1] < r1) {
            Vec<T_, V> f;
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = from_float<T_>(grad(to_float(v[u][j]), to_float(w[u][j]), j));
            store_vec_once<T_, V>(o + u * ostep, f);
        } else if (at + lane[0] < r1) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (at + lane[j] < r1) o[u * ostep + j] = from_float<T_>(grad(to_float(p[u * step + j]), to_float(d[u * dstep + j]), j));
        }
    }
}


// ---- small: one workgroup holds a slab of whole groups of one sample --------------------------------------------------------

// Slab of a workgroup: whole groups, whole vectors, 32 or 64 bytes of each row at least.  T threads, K rounds.
struct SmallGeom { int Cs, nslab, T, K, lds; };

// most threads of such a workgroup: the slots' sums take 32 KB
template <int V> constexpr int small_threads() { return V == 8 ? 512 : 1024; }
// of the variant with K rounds: the largest K only come with 256
template <int V, int K, bool BACKWARD> constexpr int small_bound() { return K > (BACKWARD ? 4 : 8) ? 256 : small_threads<V>(); }

// sum over each group's channels of buf[c] (times weight[c]) / count -> out[group]: a thread a group of few channels, a wave a larger one
template <typename S> __device__ __forceinline__ void small_groups(const S* buf, const float* weight, S inv, S* out, int cs, int D)
{
    if (D <= 16) {
        for (int k = threadIdx.x; k < cs / D; k += blockDim.x) {
            S a = 0;
            for (int c = k * D; c < k * D + D; ++c) a += buf[c] * (weight ? weight[c] : 1.f);
            out[k] = a * inv;
        }
    } else {
        const int l = threadIdx.x & 63;
        for (int k = threadIdx.x / 64; k < cs / D; k += blockDim.x / 64) {
            S a = 0;
            for (int c = l; c < D; c += 64) a += buf[k * D + c] * (weight ? weight[k * D + c] : 1.f);
            a = wave_sum(a) * inv;
            if (l == 0) out[k] = a;
        }
    }
    __syncthreads();
}

template <typename T_, int V, int ACT, int K>
__global__ __launch_bounds__((small_bound<V, K, false>())) void norm_small_kernel(const T_* __restrict__ x, NormGeom g, const float* __restrict__ weight,
                                                                        const float* __restrict__ bias, double eps, T_* __restrict__ y,
                                                                        double2* __restrict__ stats)
{
    extern __shared__ double small_buf[];              // blockDim * V slots, two values a group, the channels' three
    double* buf = small_buf;
    const int64_t n = g.n0 + blockIdx.x / (unsigned)g.nslab;
    const int c0 = (int)(blockIdx.x % (unsigned)g.nslab) * g.Cs, cs = min(g.Cs, g.C - c0), cols = cs / V;
    const int R = blockDim.x / cols, T = R * cols, t = threadIdx.x, P = (int)g.P;
    double* group_mean = buf + blockDim.x * V;
    double* group_rstd = group_mean + g.Cs / g.D;
    const int r0 = t / cols, c = t % cols * V;          // the thread's first row and its channels in the slab
    const bool work = t < T;
    Vec<T_, V> v[K];
    const T_* p = x + n * g.x_batch + r0 * g.x_row + c0 + c;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (work && r0 + k * R < P) v[k] = load_vec<T_, V>(p + (int64_t)k * R * g.x_row);
    double sum[V] = {}, squares[V] = {};
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (work && r0 + k * R < P)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const double e = (double)to_float(v[k][j]);
                sum[j] += e;
                squares[j] += e * e;
            }
    reduce_columns<V>(sum, buf, T, R, cs);
    small_groups(buf, nullptr, 1.0, group_mean, cs, g.D);
    reduce_columns<V>(squares, buf, T, R, cs);
    small_groups(buf, nullptr, 1.0, group_rstd, cs, g.D);
    const double inv = 1.0 / ((double)P * (double)g.D);
    float* lds = (float*)(group_rstd + g.Cs / g.D);
    for (int i = t; i < cs; i += blockDim.x) {
        const int k = i / g.D;
        const double2 st = statistics(group_mean[k], group_rstd[k], inv, eps);
        if (i % g.D == 0) stats[n * g.G + c0 / g.D + k] = st;
        stage_forward(lds, i, cs, st, weight, bias, c0 + i);
    }
    __syncthreads();
    if (!work) return;
    float mean[V], a[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { mean[j] = lds[c + j]; a[j] = lds[cs + c + j]; b[j] = lds[2 * cs + c + j]; }
#pragma unroll
    for (int k = 0; k < K; ++k) keep_packed(v[k]);
    T_* o = y + (n * P + r0) * g.C + c0 + c;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (r0 + k * R < P) {
            Vec<T_, V> w;
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = from_float<T_>(activate<ACT>((to_float(v[k][j]) - mean[j]) * a[j] + b[j]));
            store_vec<T_, V>(o + (int64_t)k * R * g.C, w);
        }
}

// dx, and each channel's sums of g and g * xh over the sample -> part[n][c] (or, for one sample, dbias and dweight themselves)
template <typename T_, int V, int ACT, int K>
__global__ __launch_bounds__((small_bound<V, K, true>())) void norm_small_bwd_kernel(const T_* __restrict__ x, const T_* __restrict__ dy, NormGeom g,
                                                              const double2* __restrict__ stats, const float* __restrict__ weight,
                                                              const float* __restrict__ bias, T_* __restrict__ dx, float2* __restrict__ part,
                                                              float* __restrict__ dweight, float* __restrict__ dbias)
{
    extern __shared__ double small_buf[];
    float* buf = (float*)small_buf;
    const int64_t n = g.n0 + blockIdx.x / (unsigned)g.nslab;
    const int c0 = (int)(blockIdx.x % (unsigned)g.nslab) * g.Cs, cs = min(g.Cs, g.C - c0), cols = cs / V;
    const int R = blockDim.x / cols, T = R * cols, t = threadIdx.x, P = (int)g.P;
    float* s1 = buf + blockDim.x * V;
    float* s2 = s1 + g.Cs / g.D;
    const int r0 = t / cols, c = t % cols * V;
    const bool work = t < T;
    Vec<T_, V> v[K], d[K];
    const T_* p = x + n * g.x_batch + r0 * g.x_row + c0 + c;
    const T_* q = dy + n * g.d_batch + r0 * g.d_row + c0 + c;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (work && r0 + k * R < P) {
            v[k] = load_vec<T_, V>(p + (int64_t)k * R * g.x_row);
            d[k] = load_vec<T_, V>(q + (int64_t)k * R * g.d_row);
        }
    float* lds = s2 + g.Cs / g.D;
    for (int i = t; i < cs; i += blockDim.x) stage_backward<ACT>(lds, i, cs, stats[n * g.G + (c0 + i) / g.D], weight, bias, c0 + i);
    __syncthreads();
    NormCoef<ACT> e[V];
    float a[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        a[j] = b[j] = 0.f;
        e[j].take(lds, c + j, cs);
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (work && r0 + k * R < P) {
                const float xv = to_float(v[k][j]), m = xv - e[j].mean, h = e[j].through(xv, m, to_float(d[k][j]));
                a[j] += h;
                b[j] += h * m;
            }
    }
    const float inv = 1.f / ((float)P * (float)g.D);
    const float* w = weight ? weight + c0 : nullptr;
    reduce_columns<V>(a, buf, T, R, cs);
    for (int i = t; i < cs; i += blockDim.x) {
        if (part) part[n * g.C + c0 + i].x = buf[i];
        if (dbias) dbias[c0 + i] = buf[i];
    }
    small_groups(buf, w, inv, s1, cs, g.D);
    reduce_columns<V>(b, buf, T, R, cs);
    for (int i = t; i < cs; i += blockDim.x) {
        buf[i] *= (float)stats[n * g.G + (c0 + i) / g.D].y;
        if (part) part[n * g.C + c0 + i].y = buf[i];
        if (dweight) dweight[c0 + i] = buf[i];
    }
    __syncthreads();
    if (!dx) return;
    small_groups(buf, w, inv, s2, cs, g.D);
    for (int i = t; i < cs; i += blockDim.x)
        stage_gradient(lds, i, cs, stats[n * g.G + (c0 + i) / g.D], weight, s1[i / g.D], s2[i / g.D], c0 + i);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) { keep_packed(v[k]); keep_packed(d[k]); }
    if (!work) return;
    float ka[V], kb[V], kc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { ka[j] = lds[kA * cs + c + j]; kb[j] = lds[kB * cs + c + j]; kc[j] = lds[kC * cs + c + j]; }
    T_* o = dx + (n * P + r0) * g.C + c0 + c;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (r0 + k * R < P) {
            Vec<T_, V> f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xv = to_float(v[k][j]), m = xv - e[j].mean;
                f[j] = from_float<T_>(e[j].through(xv, m, to_float(d[k][j])) * ka[j] - kb[j] - m * kc[j]);
            }
            store_vec<T_, V>(o + (int64_t)k * R * g.C, f);
        }
}

// ---- host ---------------------------------------------------------------------------------------------------------------

// Full vectors (16 bytes) wherever the mapping allows them: rows dense, or a channel count that whole vectors divide.  Addresses
// need no more than the element's own alignment (global loads take any).
static bool full_vectors(const NormGeom& g, int V) { return (g.x_row == g.C && g.d_row == g.C && g.C / gcd_(g.C, V) <= kThreads) || g.C % V == 0; }

static NormGeom norm_geom(int N, int64_t P, int C, int G, int64_t x_batch, int64_t x_row, int64_t d_batch, int64_t d_row, int dtype, int& V)
{
    NormGeom g{};
    g.N = N; g.P = P; g.C = C; g.G = G; g.D = C / G;
    g.x_batch = x_batch; g.x_row = x_row; g.d_batch = d_batch; g.d_row = d_row;
    V = dtype == RAFTCORR_DTYPE_FP32 ? 4 : 8;
    if (!full_vectors(g, V)) V = 1;
    slab_geom(g, V);
    const int64_t chunk = (int64_t)g.R * kUnroll, most = (P + chunk - 1) / chunk;
    const int64_t bytes = (int64_t)N * P * C * (dtype == RAFTCORR_DTYPE_FP32 ? 4 : 2);
    int64_t S = (bytes > (int64_t)kFewRanges * kRangeBytes ? kMostRanges : kFewRanges) / ((int64_t)N * g.nslab);
    S = S < 1 ? 1 : S > most ? most : S;
    g.rows = (most + S - 1) / S * chunk;                 // whole rounds: only a sample's last range has a rest
    g.S = (int)((P + g.rows - 1) / g.rows);
    return g;
}

// the most row ranges that any layout of these sizes is cut into
static int64_t norm_part_bytes(int N, int C) { const int64_t S = kMostRanges / N; return (S < 1 ? 1 : S) * N * C * (int64_t)sizeof(double2); }

// The one-launch form: K rounds of T threads hold P rows of a slab (K = 0: they do not).  A thread holds 16 vectors, forward of x and
// backward 8 of x and 8 of dy; few threads with many vectors, whose sums take fewer steps to join, before many threads with half.
static SmallGeom small_geom(const NormGeom& g, int V, int bytes, bool backward)
{
    SmallGeom q{};
    const int unit = g.D / gcd_(g.D, V) * V;
    if (g.C % V) return q;
    // 64 bytes of a row; forward 32 while 64 would make few workgroups (us, 32 | 64: 8 x 64 x 1000 rows float32 7.9 | 8.7,
    // 12 x 96 x 1125 rows 11.2 | 9.7; backward 8 x 64 x 1000 rows 14.6 | 12.9)
    const int least = (!backward && (int64_t)g.N * g.C * bytes <= 48 * 64 ? 32 : 64) / bytes;
    q.Cs = unit * ((least + unit - 1) / unit);
    if (q.Cs > g.C) q.Cs = g.C;
    q.nslab = (g.C + q.Cs - 1) / q.Cs;
    const int cols = q.Cs / V;
    for (const int T : {256, V == 8 ? small_threads<8>() : small_threads<1>()}) {
        if (cols > T) continue;
        const int64_t K = (g.P + T / cols - 1) / (T / cols);
        if (K <= (T == 256 ? 16 : 8) / (backward ? 2 : 1)) {
            q.T = T;
            q.lds = (T * V + 2 * (q.Cs / g.D)) * (int)(backward ? sizeof(float) : sizeof(double)) + (backward ? (int)kFields : 3) * q.Cs * (int)sizeof(float);
            if (q.lds <= 64 << 10) q.K = K <= 2 ? 2 : K <= 4 ? 4 : K <= 8 ? 8 : 16;
            return q;
        }
    }
    return q;
}

// Calls launch(geometry of some samples, its workgroups) until all samples are through: a launch takes less than 2^32 threads.
template <typename F> static void by_samples(NormGeom g, int64_t blocks, unsigned threads, F launch)
{
    const int64_t most = ((1LL << 32) - 1) / threads / blocks;          // at least 3: `blocks` workgroups a sample are 2^20 at most
    for (int64_t n = 0; n < g.N; n += most) {
        g.n0 = (int)n;
        g.n1 = (int)(g.N - n < most ? g.N - n : most);
        launch(g, (unsigned)(g.n1 * blocks));
    }
}

size_t group_norm_workspace_bytes(int N, int C, int G) { return (size_t)(norm_part_bytes(N, C) + (int64_t)N * G * (int64_t)sizeof(float2)); }

// threads of a joining workgroup over `count` partial sums: whole waves, four values a thread while there are no more than 1024
static unsigned join_threads(int64_t count)
{
    const int64_t waves = (count + 255) / 256;
    return 64 * (unsigned)(waves < 1 ? 1 : waves > 16 ? 16 : waves);
}

template <typename T_, int V, int ACT>
static void fwd_launch(const void* x_, const NormGeom& g, const float* w, const float* b, double eps, void* y_, double2* stats, double2* part, hipStream_t s)
{
    const T_* x = (const T_*)x_;
    T_* y = (T_*)y_;
    const SmallGeom q = small_geom(g, V, sizeof(T_), false);
    if (q.K) {
        NormGeom h = g;
        h.Cs = q.Cs; h.nslab = q.nslab;
        by_samples(h, q.nslab, q.T, [&](const NormGeom& h, unsigned blocks) {
            if (q.K == 2) norm_small_kernel<T_, V, ACT, 2><<<blocks, q.T, q.lds, s>>>(x, h, w, b, eps, y, stats);
            else if (q.K == 4) norm_small_kernel<T_, V, ACT, 4><<<blocks, q.T, q.lds, s>>>(x, h, w, b, eps, y, stats);
            else if (q.K == 8) norm_small_kernel<T_, V, ACT, 8><<<blocks, q.T, q.lds, s>>>(x, h, w, b, eps, y, stats);
            else norm_small_kernel<T_, V, ACT, 16><<<blocks, q.T, q.lds, s>>>(x, h, w, b, eps, y, stats);
        });
        return;
    }
    const unsigned threads = join_threads((int64_t)g.S * g.D);
    const int64_t bytes = (int64_t)g.N * g.P * g.C * (int64_t)sizeof(T_);
    const int backwards = bytes > kCache;
    by_samples(g, (int64_t)g.nslab * g.S, kThreads, [&](const NormGeom& h, unsigned blocks) {
        norm_stats_kernel<T_, V><<<blocks, kThreads, 0, s>>>(x, h, part, kept_from(bytes, blocks));
    });
    by_samples(g, g.G, threads, [&](const NormGeom& h, unsigned blocks) { norm_join_kernel<<<blocks, threads, 0, s>>>(part, h, eps, stats); });
    by_samples(g, (int64_t)g.nslab * g.S, kThreads, [&](const NormGeom& h, unsigned blocks) {
        norm_apply_kernel<T_, V, ACT><<<blocks, kThreads, 3 * g.Cs * sizeof(float), s>>>(x, h, stats, w, b, y, backwards);
    });
}

template <typename T_, int V, int ACT>
static void bwd_launch(const void* x_, const void* dy_, const NormGeom& g, const float* w, const float* b, const double2* stats, void* dx_,
                       float* dw, float* db, float2* part, float2* coef, hipStream_t s)
{
    const T_ *x = (const T_*)x_, *dy = (const T_*)dy_;
    T_* dx = (T_*)dx_;
    const SmallGeom q = small_geom(g, V, sizeof(T_), true);
    if (q.K) {
        NormGeom h = g;
        h.Cs = q.Cs; h.nslab = q.nslab; h.S = 1; h.rows = g.P;
        const bool join = (dw || db) && g.N > 1;
        float2* sums = join ? part : nullptr;
        float *dw1 = join ? nullptr : dw, *db1 = join ? nullptr : db;
        by_samples(h, q.nslab, q.T, [&](const NormGeom& h, unsigned blocks) {
            if (q.K == 2) norm_small_bwd_kernel<T_, V, ACT, 2><<<blocks, q.T, q.lds, s>>>(x, dy, h, stats, w, b, dx, sums, dw1, db1);
            else if (q.K == 4) norm_small_bwd_kernel<T_, V, ACT, 4><<<blocks, q.T, q.lds, s>>>(x, dy, h, stats, w, b, dx, sums, dw1, db1);
            else norm_small_bwd_kernel<T_, V, ACT, 8><<<blocks, q.T, q.lds, s>>>(x, dy, h, stats, w, b, dx, sums, dw1, db1);
        });
        h.n1 = 0;                                                      // the channels' sums alone
        if (join) norm_bwd_join_kernel<<<g.C, join_threads(g.N), 0, s>>>(part, h, w, coef, dw, db);
        return;
    }
    // the groups' sums, and in the last launch the channels'
    const int64_t most = (int64_t)g.S * g.D > (dw || db ? (int64_t)g.S * g.N : 0) ? (int64_t)g.S * g.D : (int64_t)g.S * g.N;
    const unsigned threads = join_threads(most);
    const int64_t bytes = 2 * (int64_t)g.N * g.P * g.C * (int64_t)sizeof(T_);
    const int backwards = bytes > kCache;
    by_samples(g, (int64_t)g.nslab * g.S, kThreads, [&](const NormGeom& h, unsigned blocks) {
        norm_bwd_sums_kernel<T_, V, ACT><<<blocks, kThreads, kSums * g.Cs * sizeof(float), s>>>(x, dy, h, stats, w, b, part, kept_from(bytes, blocks));
    });
    by_samples(g, g.G, threads, [&](const NormGeom& h, unsigned blocks) {
        const bool last = h.n0 + h.n1 == g.N && (dw || db);
        norm_bwd_join_kernel<<<blocks + (last ? g.C : 0), threads, 0, s>>>(part, h, w, coef, dw, db);
    });
    if (dx) by_samples(g, (int64_t)g.nslab * g.S, kThreads, [&](const NormGeom& h, unsigned blocks) {
        norm_bwd_apply_kernel<T_, V, ACT><<<blocks, kThreads, kFields * g.Cs * sizeof(float), s>>>(x, dy, h, stats, w, b, coef, dx, backwards);
    });
}

// f(a value of the element type, the vector's length, the activation) for the run-time ones
template <typename F> static void dispatch(int dtype, int V, int act, F f)
{
    auto with_act = [&](auto t, auto v) {
        if (act == RAFTCORR_ACT_RELU) f(t, v, std::integral_constant<int, RAFTCORR_ACT_RELU>());
        else if (act == RAFTCORR_ACT_SILU) f(t, v, std::integral_constant<int, RAFTCORR_ACT_SILU>());
        else f(t, v, std::integral_constant<int, RAFTCORR_ACT_NONE>());
    };
    auto with_vector = [&](auto t) {
        constexpr int full = 16 / (int)sizeof(t);
        if (V == full) with_act(t, std::integral_constant<int, full>());
        else with_act(t, std::integral_constant<int, 1>());
    };
    if (dtype == RAFTCORR_DTYPE_FP32) with_vector(float());
    else if (dtype == RAFTCORR_DTYPE_FP16) with_vector(_Float16());
    else with_vector(__bf16());
}

int launch_group_norm_fwd(const void* x, int64_t x_batch, int64_t x_row, int dtype, int N, int64_t P, int C, int G, const float* w,
                          const float* b, double eps, int act, void* y, double* stats, void* workspace, hipStream_t s)
{
    int V;
    const NormGeom g = norm_geom(N, P, C, G, x_batch, x_row, x_batch, x_row, dtype, V);
    if (V > 1 && small_geom(g, 1, dtype == RAFTCORR_DTYPE_FP32 ? 4 : 2, false).K && C % V) V = 1;
    double2* part = (double2*)workspace;
    double2* st = (double2*)stats;
    dispatch(dtype, V, act, [&](auto t, auto v, auto a) {
        fwd_launch<decltype(t), decltype(v)::value, decltype(a)::value>(x, g, w, b, eps, y, st, part, s);
    });
    return check_launch("group_norm_fwd");
}

int launch_group_norm_bwd(const void* x, int64_t x_batch, int64_t x_row, const void* dy, int64_t d_batch, int64_t d_row, int dtype, int N,
                          int64_t P, int C, int G, const float* w, const float* b, int act, const double* stats, void* dx, float* dw,
                          float* db, void* workspace, hipStream_t s)
{
    int V;
    const NormGeom g = norm_geom(N, P, C, G, x_batch, x_row, d_batch, d_row, dtype, V);
    if (V > 1 && small_geom(g, 1, dtype == RAFTCORR_DTYPE_FP32 ? 4 : 2, true).K && C % V) V = 1;
    float2* part = (float2*)workspace;
    float2* coef = (float2*)((char*)workspace + norm_part_bytes(N, C));
    const double2* st = (const double2*)stats;
    dispatch(dtype, V, act, [&](auto t, auto v, auto a) {
        bwd_launch<decltype(t), decltype(v)::value, decltype(a)::value>(x, dy, g, w, b, st, dx, dw, db, part, coef, s);
    });
    return check_launch("group_norm_bwd");
}

}  // namespace raftcorr

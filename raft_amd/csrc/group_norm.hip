// Group normalisation with an activation, channels last, forward and backward.
//
// x is a matrix of N*P rows (sample n, position p) of C channels; groups of D = C / G neighbouring channels share mean and
// variance over P*D values:
//   xh = (x - mean) * rstd,  z = xh * w[c] + b[c],  y = act(z)
//   g = dy * act'(z):  db[c] = sum g,  dw[c] = sum g * xh,
//   dx = rstd * (g * w - s1 - xh * s2),  s1 = mean over the group of g * w,  s2 = mean over the group of g * w * xh.
// Memory bound: 8 operations a value forward, some 20 backward.  Three launches each: sums of row ranges per channel, one small
// launch that joins them per group, one pass that writes.
#include "common.h"
#include "elem.h"

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
};

enum { kThreads = 256, kUnroll = 8 };

static int gcd_(int a, int b) { while (b) { const int t = a % b; a = b; b = t; } return a; }

// slab widths for vectors of V: whole rows if their pattern fits the workgroup, else column slabs of 256 vectors
static void slab_geom(NormGeom& g, int V)
{
    const int pattern = g.C / gcd_(g.C, V);          // threads after which the channel pattern repeats
    if (pattern <= kThreads) {
        g.Cs = g.C; g.nslab = 1;
        g.T = kThreads / pattern * pattern;
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

// sum over the row lanes of NQ quantities a slot: slot f = t * V + j of thread t holds channel f % cs, row lane f / cs.
// buf: NQ * kThreads * V floats; afterwards buf[q * kThreads * V + c] is channel c's sum.  Fixed order.
template <int V, int NQ> __device__ __forceinline__ void reduce_columns(float (&val)[NQ][V], float* buf, int T, int R, int cs)
{
    const int t = threadIdx.x;
    __syncthreads();
    if (t < T)
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int j = 0; j < V; ++j) buf[q * kThreads * V + t * V + j] = val[q][j];
    for (int rows = R; rows > 1;) {
        const int half = (rows + 1) / 2;
        __syncthreads();
        for (int f = t; f < (rows - half) * cs; f += kThreads)
#pragma unroll
            for (int q = 0; q < NQ; ++q) buf[q * kThreads * V + f] += buf[q * kThreads * V + f + half * cs];
        rows = half;
    }
    __syncthreads();
}

// ---- forward ------------------------------------------------------------------------------------------------------------

// mean and sum of squared deviations of each channel over one row range -> part[n][s][c].  A thread takes 8 rows at a time (two
// passes over them in registers) and joins the result with what it has: no sum of squares that a large mean would cancel.
template <typename T_, int V>
__global__ __launch_bounds__(kThreads) void norm_stats_kernel(const T_* __restrict__ x, NormGeom g, float2* __restrict__ part)
{
    __shared__ float buf[2 * kThreads * V];
    const int s = blockIdx.x % g.S, slab = blockIdx.x / g.S % g.nslab;
    const int64_t n = blockIdx.x / g.S / g.nslab;
    int c0, cs, T, R;
    slab_of<V>(g, slab, c0, cs, T, R);
    const int t = threadIdx.x;
    const int64_t r0 = s * g.rows, r1 = min(g.P, r0 + g.rows);
    float mean[1][V] = {}, m2[1][V] = {};
    int cnt[V];
    int lane[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { lane[j] = (t * V + j) / cs; cnt[j] = 0; }
    if (t < T) {
        const int64_t step = (int64_t)R * g.x_row;
        const T_* p = x + n * g.x_batch + (r0 + lane[0]) * g.x_row + c0 + (t * V) % cs;
        int64_t r = r0;
        int k = 0;
        for (; r + (int64_t)kUnroll * R <= r1; r += kUnroll * R) {
            Vec<T_, V> v[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) { v[u] = load_vec<T_, V>(p); p += step; }
            const float fa = (float)kUnroll / (float)(k + kUnroll), fb = fa * (float)k;
            k += kUnroll;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float a = 0.f, q = 0.f;
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) a += to_float(v[u][j]);
                a *= 1.f / kUnroll;
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) { const float d = to_float(v[u][j]) - a; q += d * d; }
                const float d = a - mean[0][j];
                mean[0][j] += d * fa;
                m2[0][j] += q + d * d * fb;
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) cnt[j] = k;
        for (; r < r1; r += R) {
            const float f = 1.f / (float)(k + 1);
            ++k;
            if (r + lane[V - 1] < r1) {
                const Vec<T_, V> v = load_vec<T_, V>(p);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = to_float(v[j]) - mean[0][j];
                    mean[0][j] += d * f;
                    m2[0][j] += d * (to_float(v[j]) - mean[0][j]);
                    cnt[j] = k;
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (r + lane[j] < r1) {
                        const float e = to_float(p[j]), d = e - mean[0][j];
                        mean[0][j] += d * f;
                        m2[0][j] += d * (e - mean[0][j]);
                        cnt[j] = k;
                    }
            }
            p += step;
        }
    }
    // join the row lanes: mean of the means, then the deviations around it
    float w[1][V];
#pragma unroll
    for (int j = 0; j < V; ++j) w[0][j] = mean[0][j] * (float)cnt[j];
    reduce_columns<V, 1>(w, buf, T, R, cs);
    float* keep = buf + kThreads * V;
    const float inv = 1.f / (float)(r1 - r0);
    for (int c = t; c < cs; c += kThreads) keep[c] = buf[c] * inv;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float d = t < T ? mean[0][j] - keep[(t * V + j) % cs] : 0.f;
        w[0][j] = m2[0][j] + d * d * (float)cnt[j];
    }
    reduce_columns<V, 1>(w, buf, T, R, cs);
    for (int c = t; c < cs; c += kThreads)
        part[(n * g.S + s) * g.C + c0 + c] = make_float2(keep[c], buf[c]);
}

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// part -> (mean, rstd) of each (n, group); one wave each
__global__ __launch_bounds__(kThreads) void norm_join_kernel(const float2* __restrict__ part, NormGeom g, float eps, float2* __restrict__ stats)
{
    const int64_t i = (int64_t)blockIdx.x * (kThreads / 64) + threadIdx.x / 64;
    if (i >= (int64_t)g.N * g.G) return;
    const int64_t n = i / g.G;
    const float2* p = part + n * g.S * g.C + i % g.G * g.D;
    const int l = threadIdx.x & 63, count = g.S * g.D;
    const float full = (float)g.rows, last = (float)(g.P - (g.S - 1) * g.rows);
    float a = 0.f;
    for (int k = l; k < count; k += 64) {
        const int s = k / g.D;
        a += p[(int64_t)s * g.C + k % g.D].x * (s == g.S - 1 ? last : full);
    }
    const float inv = 1.f / ((float)g.P * (float)g.D);
    const float mean = wave_sum(a) * inv;
    float q = 0.f;
    for (int k = l; k < count; k += 64) {
        const int s = k / g.D;
        const float2 v = p[(int64_t)s * g.C + k % g.D];
        const float d = v.x - mean;
        q += v.y + d * d * (s == g.S - 1 ? last : full);
    }
    const float var = wave_sum(q) * inv;
    if (l == 0) stats[i] = make_float2(mean, 1.f / sqrtf(var + eps));
}

template <int ACT> __device__ __forceinline__ float activate(float z)
{
    if (ACT == RAFTCORR_ACT_RELU) return z < 0.f ? 0.f : z;                    // (a NaN stays one)
    if (ACT == RAFTCORR_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + expf(-z));
    return z;
}

template <int ACT> __device__ __forceinline__ float slope(float z)
{
    if (ACT == RAFTCORR_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (ACT == RAFTCORR_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + expf(-z));
        return s * (1.f + z * (1.f - s));
    }
    return 1.f;
}

template <typename T_, int V, int ACT>
__global__ __launch_bounds__(kThreads) void norm_apply_kernel(const T_* __restrict__ x, NormGeom g, const float2* __restrict__ stats,
                                                              const float* __restrict__ weight, const float* __restrict__ bias,
                                                              T_* __restrict__ y)
{
    const int s = blockIdx.x % g.S, slab = blockIdx.x / g.S % g.nslab;
    const int64_t n = blockIdx.x / g.S / g.nslab;
    int c0, cs, T, R;
    slab_of<V>(g, slab, c0, cs, T, R);
    const int t = threadIdx.x;
    if (t >= T) return;
    const int64_t r1 = min(g.P, (s + 1) * g.rows);
    float mean[V], a[V], b[V];
    int lane[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        lane[j] = (t * V + j) / cs;
        const int c = c0 + (t * V + j) % cs;
        const float2 st = stats[n * g.G + c / g.D];
        mean[j] = st.x;
        a[j] = weight ? st.y * weight[c] : st.y;
        b[j] = bias ? bias[c] : 0.f;
    }
    const int64_t step = (int64_t)R * g.x_row, ystep = (int64_t)R * g.C;
    const T_* p = x + n * g.x_batch + (s * g.rows + lane[0]) * g.x_row + c0 + (t * V) % cs;
    T_* o = y + (n * g.P + s * g.rows + lane[0]) * g.C + c0 + (t * V) % cs;
    int64_t r = s * g.rows;
    for (; r + (int64_t)kUnroll * R <= r1; r += kUnroll * R) {
        Vec<T_, V> v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) { v[u] = load_vec<T_, V>(p); p += step; }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            Vec<T_, V> w;
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = from_float<T_>(activate<ACT>((to_float(v[u][j]) - mean[j]) * a[j] + b[j]));
            store_vec<T_, V>(o, w);
            o += ystep;
        }
    }
    for (; r < r1; r += R) {
        if (r + lane[V - 1] < r1) {
            const Vec<T_, V> v = load_vec<T_, V>(p);
            Vec<T_, V> w;
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = from_float<T_>(activate<ACT>((to_float(v[j]) - mean[j]) * a[j] + b[j]));
            store_vec<T_, V>(o, w);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (r + lane[j] < r1) o[j] = from_float<T_>(activate<ACT>((to_float(p[j]) - mean[j]) * a[j] + b[j]));
        }
        p += step;
        o += ystep;
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------------

// what a slot needs of its channel
struct NormCoef { float mean, rstd, w, b; };

__device__ __forceinline__ NormCoef coef_of(const NormGeom& g, const float2* stats, const float* weight, const float* bias, int64_t n, int c)
{
    const float2 st = stats[n * g.G + c / g.D];
    return NormCoef{st.x, st.y, weight ? weight[c] : 1.f, bias ? bias[c] : 0.f};
}

// sum of g and of g * xh of each channel over one row range -> part[n][s][c]
template <typename T_, int V, int ACT>
__global__ __launch_bounds__(kThreads) void norm_bwd_sums_kernel(const T_* __restrict__ x, const T_* __restrict__ dy, NormGeom g,
                                                                 const float2* __restrict__ stats, const float* __restrict__ weight,
                                                                 const float* __restrict__ bias, float2* __restrict__ part)
{
    __shared__ float buf[2 * kThreads * V];
    const int s = blockIdx.x % g.S, slab = blockIdx.x / g.S % g.nslab;
    const int64_t n = blockIdx.x / g.S / g.nslab;
    int c0, cs, T, R;
    slab_of<V>(g, slab, c0, cs, T, R);
    const int t = threadIdx.x;
    const int64_t r1 = min(g.P, (s + 1) * g.rows);
    float sum[2][V] = {};
    if (t < T) {
        NormCoef k[V];
        int lane[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            lane[j] = (t * V + j) / cs;
            k[j] = coef_of(g, stats, weight, bias, n, c0 + (t * V + j) % cs);
        }
        auto add = [&](float xv, float dv, int j, float& a, float& b) {
            const float xh = (xv - k[j].mean) * k[j].rstd;
            const float e = dv * slope<ACT>(xh * k[j].w + k[j].b);
            a += e;
            b += e * xh;
        };
        const int64_t step = (int64_t)R * g.x_row, dstep = (int64_t)R * g.d_row;
        const T_* p = x + n * g.x_batch + (s * g.rows + lane[0]) * g.x_row + c0 + (t * V) % cs;
        const T_* d = dy + n * g.d_batch + (s * g.rows + lane[0]) * g.d_row + c0 + (t * V) % cs;
        int64_t r = s * g.rows;
        for (; r + (int64_t)(kUnroll / 2) * R <= r1; r += kUnroll / 2 * R) {
            Vec<T_, V> v[kUnroll / 2], w[kUnroll / 2];
#pragma unroll
            for (int u = 0; u < kUnroll / 2; ++u) {
                v[u] = load_vec<T_, V>(p); p += step;
                w[u] = load_vec<T_, V>(d); d += dstep;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float a = 0.f, b = 0.f;                      // the chunk by itself first: long sums lose less
#pragma unroll
                for (int u = 0; u < kUnroll / 2; ++u) add(to_float(v[u][j]), to_float(w[u][j]), j, a, b);
                sum[0][j] += a;
                sum[1][j] += b;
            }
        }
        for (; r < r1; r += R) {
            if (r + lane[V - 1] < r1) {
                const Vec<T_, V> v = load_vec<T_, V>(p), w = load_vec<T_, V>(d);
#pragma unroll
                for (int j = 0; j < V; ++j) add(to_float(v[j]), to_float(w[j]), j, sum[0][j], sum[1][j]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (r + lane[j] < r1) add(to_float(p[j]), to_float(d[j]), j, sum[0][j], sum[1][j]);
            }
            p += step;
            d += dstep;
        }
    }
    reduce_columns<V, 2>(sum, buf, T, R, cs);
    for (int c = t; c < cs; c += kThreads)
        part[(n * g.S + s) * g.C + c0 + c] = make_float2(buf[c], buf[kThreads * V + c]);
}

// part -> (s1, s2) of each (n, group) and, with dweight / dbias, the channels' sums over all samples; one wave each
__global__ __launch_bounds__(kThreads) void norm_bwd_join_kernel(const float2* __restrict__ part, NormGeom g, const float* __restrict__ weight,
                                                                 float2* __restrict__ coef, float* __restrict__ dweight, float* __restrict__ dbias)
{
    int64_t i = (int64_t)blockIdx.x * (kThreads / 64) + threadIdx.x / 64;
    const int l = threadIdx.x & 63;
    float a = 0.f, b = 0.f;
    if (i < (int64_t)g.N * g.G) {
        const int64_t n = i / g.G;
        const int c0 = (int)(i % g.G) * g.D;
        for (int64_t k = l; k < (int64_t)g.S * g.D; k += 64) {
            const int c = c0 + (int)(k % g.D);
            const float2 v = part[(n * g.S + k / g.D) * g.C + c];
            const float w = weight ? weight[c] : 1.f;
            a += v.x * w;
            b += v.y * w;
        }
        const float inv = 1.f / ((float)g.P * (float)g.D);
        a = wave_sum(a) * inv;
        b = wave_sum(b) * inv;
        if (l == 0) coef[i] = make_float2(a, b);
        return;
    }
    i -= (int64_t)g.N * g.G;
    if (i >= g.C || !(dweight || dbias)) return;
    for (int64_t k = l; k < (int64_t)g.N * g.S; k += 64) {
        const float2 v = part[k * g.C + i];
        a += v.x;
        b += v.y;
    }
    a = wave_sum(a);
    b = wave_sum(b);
    if (l == 0) {
        if (dbias) dbias[i] = a;
        if (dweight) dweight[i] = b;
    }
}

template <typename T_, int V, int ACT>
__global__ __launch_bounds__(kThreads) void norm_bwd_apply_kernel(const T_* __restrict__ x, const T_* __restrict__ dy, NormGeom g,
                                                                  const float2* __restrict__ stats, const float* __restrict__ weight,
                                                                  const float* __restrict__ bias, const float2* __restrict__ coef,
                                                                  T_* __restrict__ dx)
{
    const int s = blockIdx.x % g.S, slab = blockIdx.x / g.S % g.nslab;
    const int64_t n = blockIdx.x / g.S / g.nslab;
    int c0, cs, T, R;
    slab_of<V>(g, slab, c0, cs, T, R);
    const int t = threadIdx.x;
    if (t >= T) return;
    const int64_t r1 = min(g.P, (s + 1) * g.rows);
    NormCoef k[V];
    float2 m[V];
    int lane[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        lane[j] = (t * V + j) / cs;
        const int c = c0 + (t * V + j) % cs;
        k[j] = coef_of(g, stats, weight, bias, n, c);
        m[j] = coef[n * g.G + c / g.D];
    }
    auto grad = [&](float xv, float dv, int j) {
        const float xh = (xv - k[j].mean) * k[j].rstd;
        const float e = dv * slope<ACT>(xh * k[j].w + k[j].b);
        return k[j].rstd * (e * k[j].w - m[j].x - xh * m[j].y);
    };
    const int64_t step = (int64_t)R * g.x_row, dstep = (int64_t)R * g.d_row, ostep = (int64_t)R * g.C;
    const T_* p = x + n * g.x_batch + (s * g.rows + lane[0]) * g.x_row + c0 + (t * V) % cs;
    const T_* d = dy + n * g.d_batch + (s * g.rows + lane[0]) * g.d_row + c0 + (t * V) % cs;
    T_* o = dx + (n * g.P + s * g.rows + lane[0]) * g.C + c0 + (t * V) % cs;
    int64_t r = s * g.rows;
    for (; r + (int64_t)(kUnroll / 2) * R <= r1; r += kUnroll / 2 * R) {
        Vec<T_, V> v[kUnroll / 2], w[kUnroll / 2];
#pragma unroll
        for (int u = 0; u < kUnroll / 2; ++u) {
            v[u] = load_vec<T_, V>(p); p += step;
            w[u] = load_vec<T_, V>(d); d += dstep;
        }
#pragma unroll
        for (int u = 0; u < kUnroll / 2; ++u) {
            Vec<T_, V> q;
#pragma unroll
            for (int j = 0; j < V; ++j) q[j] = from_float<T_>(grad(to_float(v[u][j]), to_float(w[u][j]), j));
            store_vec<T_, V>(o, q);
            o += ostep;
        }
    }
    for (; r < r1; r += R) {
        if (r + lane[V - 1] < r1) {
            const Vec<T_, V> v = load_vec<T_, V>(p), w = load_vec<T_, V>(d);
            Vec<T_, V> q;
#pragma unroll
            for (int j = 0; j < V; ++j) q[j] = from_float<T_>(grad(to_float(v[j]), to_float(w[j]), j));
            store_vec<T_, V>(o, q);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (r + lane[j] < r1) o[j] = from_float<T_>(grad(to_float(p[j]), to_float(d[j]), j));
        }
        p += step;
        d += dstep;
        o += ostep;
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
    // some four workgroups a CU, each with one unrolled round at least
    const int64_t most = (P + (int64_t)kUnroll * g.R - 1) / ((int64_t)kUnroll * g.R);
    int64_t S = 1024 / ((int64_t)N * g.nslab);
    S = S < 1 ? 1 : S > most ? most : S;
    g.rows = ((P + S - 1) / S + g.R - 1) / g.R * g.R;
    g.S = (int)((P + g.rows - 1) / g.rows);
    return g;
}

// The most row ranges any layout of these sizes is cut into: 1024 / N.
static int64_t norm_part_bytes(int N, int C) { const int64_t S = 1024 / N; return (S < 1 ? 1 : S) * N * C * (int64_t)sizeof(float2); }

size_t group_norm_workspace_bytes(int N, int C, int G) { return (size_t)(norm_part_bytes(N, C) + (int64_t)N * G * (int64_t)sizeof(float2)); }

template <typename T_, int V>
static void fwd_launch(const void* x, const NormGeom& g, const float* w, const float* b, float eps, int act, void* y, float2* stats, float2* part, hipStream_t s)
{
    const unsigned blocks = (unsigned)((int64_t)g.N * g.nslab * g.S), joins = (unsigned)(((int64_t)g.N * g.G + 3) / 4);
    norm_stats_kernel<T_, V><<<blocks, kThreads, 0, s>>>((const T_*)x, g, part);
    norm_join_kernel<<<joins, kThreads, 0, s>>>(part, g, eps, stats);
    if (act == RAFTCORR_ACT_RELU) norm_apply_kernel<T_, V, RAFTCORR_ACT_RELU><<<blocks, kThreads, 0, s>>>((const T_*)x, g, stats, w, b, (T_*)y);
    else if (act == RAFTCORR_ACT_SILU) norm_apply_kernel<T_, V, RAFTCORR_ACT_SILU><<<blocks, kThreads, 0, s>>>((const T_*)x, g, stats, w, b, (T_*)y);
    else norm_apply_kernel<T_, V, RAFTCORR_ACT_NONE><<<blocks, kThreads, 0, s>>>((const T_*)x, g, stats, w, b, (T_*)y);
}

template <typename T_, int V, int ACT>
static void bwd_launch(const void* x, const void* dy, const NormGeom& g, const float* w, const float* b, const float2* stats, void* dx,
                       float* dw, float* db, float2* part, float2* coef, hipStream_t s)
{
    const unsigned blocks = (unsigned)((int64_t)g.N * g.nslab * g.S);
    const unsigned joins = (unsigned)(((int64_t)g.N * g.G + (dw || db ? g.C : 0) + 3) / 4);
    norm_bwd_sums_kernel<T_, V, ACT><<<blocks, kThreads, 0, s>>>((const T_*)x, (const T_*)dy, g, stats, w, b, part);
    norm_bwd_join_kernel<<<joins, kThreads, 0, s>>>(part, g, w, coef, dw, db);
    if (dx) norm_bwd_apply_kernel<T_, V, ACT><<<blocks, kThreads, 0, s>>>((const T_*)x, (const T_*)dy, g, stats, w, b, coef, (T_*)dx);
}

int launch_group_norm_fwd(const void* x, int64_t x_batch, int64_t x_row, int dtype, int N, int64_t P, int C, int G, const float* w,
                          const float* b, float eps, int act, void* y, float* stats, void* workspace, hipStream_t s)
{
    int V;
    const NormGeom g = norm_geom(N, P, C, G, x_batch, x_row, x_batch, x_row, dtype, V);
    float2* part = (float2*)workspace;
    float2* st = (float2*)stats;
    if (dtype == RAFTCORR_DTYPE_FP32) {
        if (V == 4) fwd_launch<float, 4>(x, g, w, b, eps, act, y, st, part, s); else fwd_launch<float, 1>(x, g, w, b, eps, act, y, st, part, s);
    } else if (dtype == RAFTCORR_DTYPE_FP16) {
        if (V == 8) fwd_launch<_Float16, 8>(x, g, w, b, eps, act, y, st, part, s); else fwd_launch<_Float16, 1>(x, g, w, b, eps, act, y, st, part, s);
    } else {
        if (V == 8) fwd_launch<__bf16, 8>(x, g, w, b, eps, act, y, st, part, s); else fwd_launch<__bf16, 1>(x, g, w, b, eps, act, y, st, part, s);
    }
    return check_launch("group_norm_fwd");
}

template <typename T_, int V>
static void bwd_by_act(int act, const void* x, const void* dy, const NormGeom& g, const float* w, const float* b, const float2* stats, void* dx,
                       float* dw, float* db, float2* part, float2* coef, hipStream_t s)
{
    if (act == RAFTCORR_ACT_RELU) bwd_launch<T_, V, RAFTCORR_ACT_RELU>(x, dy, g, w, b, stats, dx, dw, db, part, coef, s);
    else if (act == RAFTCORR_ACT_SILU) bwd_launch<T_, V, RAFTCORR_ACT_SILU>(x, dy, g, w, b, stats, dx, dw, db, part, coef, s);
    else bwd_launch<T_, V, RAFTCORR_ACT_NONE>(x, dy, g, w, b, stats, dx, dw, db, part, coef, s);
}

int launch_group_norm_bwd(const void* x, int64_t x_batch, int64_t x_row, const void* dy, int64_t d_batch, int64_t d_row, int dtype, int N,
                          int64_t P, int C, int G, const float* w, const float* b, int act, const float* stats, void* dx, float* dw,
                          float* db, void* workspace, hipStream_t s)
{
    int V;
    const NormGeom g = norm_geom(N, P, C, G, x_batch, x_row, d_batch, d_row, dtype, V);
    float2* part = (float2*)workspace;
    float2* coef = (float2*)((char*)workspace + norm_part_bytes(N, C));
    const float2* st = (const float2*)stats;
    if (dtype == RAFTCORR_DTYPE_FP32) {
        if (V == 4) bwd_by_act<float, 4>(act, x, dy, g, w, b, st, dx, dw, db, part, coef, s);
        else bwd_by_act<float, 1>(act, x, dy, g, w, b, st, dx, dw, db, part, coef, s);
    } else if (dtype == RAFTCORR_DTYPE_FP16) {
        if (V == 8) bwd_by_act<_Float16, 8>(act, x, dy, g, w, b, st, dx, dw, db, part, coef, s);
        else bwd_by_act<_Float16, 1>(act, x, dy, g, w, b, st, dx, dw, db, part, coef, s);
    } else {
        if (V == 8) bwd_by_act<__bf16, 8>(act, x, dy, g, w, b, st, dx, dw, db, part, coef, s);
        else bwd_by_act<__bf16, 1>(act, x, dy, g, w, b, st, dx, dw, db, part, coef, s);
    }
    return check_launch("group_norm_bwd");
}

}  // namespace raftcorr

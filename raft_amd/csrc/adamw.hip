// The AdamW step of many tensors, with moments in 32 or in 8 bits and the gradients clipped by their global norm.
//
//   c = min(1, max_norm / (|g| + 1e-6)),  m = b1 m + (1 - b1) c g,  v = b2 v + (1 - b2) (c g)^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Memory bound: 28 bytes a float32 parameter with 32-bit moments, 16 with 8-bit ones.  Launches: sums of squares of the gradients
// (only with clipping), one workgroup that counts the steps and joins the sums, the update; each takes the tensors' addresses by
// value, as many as 4 KB of kernel arguments hold, so a captured graph depends on no table.
//
// The moments of a bucket of tensors lie in flat buffers; tensor i starts at a multiple of 512 values.  A wave takes 512
// neighbouring values ("tile") of one tensor, 8 a lane.
//
// 8-bit moments: 64 neighbouring values share one exponent byte E, the exponent field of the largest one's float32.  A code c
// stands for c units below 8, else for (8 + (c & 7)) << ((c >> 3) - 1) units: three bits behind the leading one, 15 (first moment, sign
// in bit 7) or 31 (second) binades, the unit 2^(E - 127 - 16) or 2^(E - 127 - 32).  Scales are powers of two: nothing but the
// last step rounds.  That step rounds up with the probability of the rest it drops: with b2 = 0.999 a step moves v by a
// thousandth, a code is 6 to 12 % wide, and rounding to the nearest would hold v where it is for good.  The 16 random bits of a
// value come from (seed, step, position) alone.  A second moment that is not zero keeps at least one unit: m / (sqrt(0) + eps)
// would be a huge step.  E = 255 (something not finite in the block) decodes as NaN, all 64; E = 0 (all below 2^-126) as zero.
// The new moments are summed in 64 bits (full rate here), rounded to 32, used for the update, then coded.
//
// A code is the upper bits of a float32 whose unit is 2^-129: subnormal below 8 units, three mantissa bits above.  So the float with
// the bits c << 20, times a power of two, is the value; and the other way round the value times that power, its bits, the random
// bits added below the code's last one, shifted down by 20, is the code.  No case apart for small codes.
#include "common.h"
#include "elem.h"
#include <type_traits>

namespace raftcorr {

enum { kTile = RAFTCORR_ADAMW_TILE, kBlock = RAFTCORR_ADAMW_BLOCK, kLane = 8, kWg = 256, kWaves = kWg / 64 };
static_assert(kTile == 64 * kLane && kBlock % kLane == 0 && kTile % kBlock == 0, "a lane's values share a block, a wave's tile holds whole blocks");

// ---- gradient norm ------------------------------------------------------------------------------------------------------

enum { kNormTensors = 240, kRun = 4 };
struct NormTable {
    const void* grad[kNormTensors];
    uint32_t first[kNormTensors];             // first tile of each tensor, counted from the first tensor of the launch
    uint16_t tail[kNormTensors];              // values in its last tile
};

// the tensor a tile belongs to: the last of `count` that starts at or before it
__device__ __forceinline__ int tensor_of(const uint32_t* first, int count, uint32_t tile)
{
    int lo = 0, hi = count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (first[mid] <= tile) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// partial[block] = sum of squares over the tiles of the block's waves, in 64 bits.  A wave takes `run` neighbouring tiles: it looks
// its tensor up once and has the loads of four tiles on their way at a time.
template <typename T>
__global__ __launch_bounds__(kWg) void adamw_norm_kernel(NormTable tab, int count, uint32_t tiles, uint32_t run, double* __restrict__ partial)
{
    __shared__ double part[kWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63;
    double sum = 0.0;
    uint32_t tile = (blockIdx.x * kWaves + wave) * run;
    const uint32_t end = min(tile + run, tiles);
    if (tile < end) {
        int i = tensor_of(tab.first, count, tile);
        while (tile < end) {
            const uint32_t first = tab.first[i], next = i + 1 < count ? tab.first[i + 1] : tiles;
            const T* g = (const T*)tab.grad[i] + (int64_t)(tile - first) * kTile + lane * kLane;
            const uint32_t full = min(end, next - 1);          // whole tiles up to here
            for (; tile + kRun <= full; tile += kRun, g += kRun * kTile) {
                Vec<T, kLane> v[kRun];
#pragma unroll
                for (int u = 0; u < kRun; ++u) v[u] = load_vec<T, kLane>(g + u * kTile);
#pragma unroll
                for (int u = 0; u < kRun; ++u)
#pragma unroll
                    for (int j = 0; j < kLane; ++j) { const double e = (double)to_float(v[u][j]); sum += e * e; }
            }
            for (; tile < full; ++tile, g += kTile) {
                const Vec<T, kLane> v = load_vec<T, kLane>(g);
#pragma unroll
                for (int j = 0; j < kLane; ++j) { const double e = (double)to_float(v[j]); sum += e * e; }
            }
            if (tile < end) {                                   // the tensor's last tile
                const int have = (int)tab.tail[i] - lane * kLane;
                if (have >= kLane) {
                    const Vec<T, kLane> v = load_vec<T, kLane>(g);
#pragma unroll
                    for (int j = 0; j < kLane; ++j) { const double e = (double)to_float(v[j]); sum += e * e; }
                } else {
                    for (int j = 0; j < have; ++j) { const double e = (double)to_float(g[j]); sum += e * e; }
                }
                ++tile;
                ++i;
            }
        }
    }
    sum = wave_sum(sum);
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = part[0];
        for (int w = 1; w < kWaves; ++w) s += part[w];
        partial[blockIdx.x] = s;
    }
}

// ---- steps, bias corrections, clipping coefficient ----------------------------------------------------------------------

enum { kStepTensors = 960 };
struct StepTable { int32_t slot[kStepTensors]; };

enum { kCountWg = 1024 };

// b^t for a whole t
__device__ __forceinline__ double power(double b, uint32_t t)
{
    double p = 1.0;
    for (; t; t >>= 1, b *= b)
        if (t & 1) p *= b;
    return p;
}

// counts the tensors' steps; scale[slot] = (lr / (1 - b1^t), 1 / sqrt(1 - b2^t)); joins the partial sums (partials > 0)
__global__ __launch_bounds__(kCountWg) void adamw_count_kernel(StepTable tab, int count, float* __restrict__ steps, float2* __restrict__ scale,
                                                               double lr, const float* __restrict__ lr_device, double b1, double b2,
                                                               const double* __restrict__ partial, int partials, double max_norm,
                                                               double* __restrict__ clip, float* __restrict__ norm)
{
    __shared__ double part[kCountWg / 64];
    double sum = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < partials; i += kCountWg) sum += partial[i];
    if (lr_device) lr = (double)*lr_device;
    if ((int)threadIdx.x < count) {
        const int slot = tab.slot[threadIdx.x];
        const float t = steps[slot] + 1.f;
        steps[slot] = t;
        scale[slot] = make_float2((float)(lr / (1.0 - power(b1, (uint32_t)t))), (float)(1.0 / sqrt(1.0 - power(b2, (uint32_t)t))));
    }
    if (!partials) return;
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < kCountWg / 64; ++w) sum += part[w];
    sum = sqrt(sum);
    const double c = max_norm / (sum + 1e-6);
    *clip = c > 1.0 ? 1.0 : c;                  // (a NaN stays one)
    *norm = (float)sum;
}

// ---- update -------------------------------------------------------------------------------------------------------------

enum { kUpdateTensors = 140 };
struct UpdateTable {
    uint64_t p[kUpdateTensors], g[kUpdateTensors];
    uint32_t first[kUpdateTensors], state[kUpdateTensors];      // first tile in the launch, first tile in the bucket's buffers
    uint32_t slot_tail[kUpdateTensors];                         // step counter << 10 | values in the last tile
};

struct UpdateArgs {
    void* m;
    void* v;
    uint8_t* me;
    uint8_t* ve;
    const float* steps;
    const float2* scale;
    const double* clip;
    const float* lr_device;
    double b1, b2;
    float lr, eps, wd;
    uint32_t seed, count, tiles;
};
static_assert(sizeof(UpdateTable) + sizeof(UpdateArgs) <= 4096 && sizeof(NormTable) + 24 <= 4096 && sizeof(StepTable) + 96 <= 4096, "kernel arguments");

// Scrambles 32 bits: shifts and odd multipliers (the leading binary digits of sqrt 2 and sqrt 3).
__device__ __forceinline__ uint32_t mix(uint32_t x)
{
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ x >> 16;
}
constexpr uint32_t kGolden = 0x9E3779B9u;       // leading binary digits of the golden ratio: neighbouring positions land far apart

// the largest of the values of a block's lanes
__device__ __forceinline__ uint32_t block_max(uint32_t v)
{
#pragma unroll
    for (int o = 1; o < kBlock / kLane; o <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    return v;
}

// 2^e for -1022 <= e <= 1023
__device__ __forceinline__ double exp2i(int e) { return __longlong_as_double((long long)(e + 1023) << 52); }

template <typename T> __device__ __forceinline__ T round_param(float x, uint32_t) { return (T)x; }
// bfloat16 parameters are rounded up with the probability of what is dropped: a step of 2^-9 of a weight would be lost otherwise
// (infinities and NaN as they are: x comes out of a sum, its NaN have their upper mantissa bit set)
template <> __device__ __forceinline__ __bf16 round_param<__bf16>(float x, uint32_t bits16)
{
    const uint32_t w = __float_as_uint(x);
    return __builtin_bit_cast(__bf16, (uint16_t)((w + (__builtin_isfinite(x) ? bits16 : 0u)) >> 16));
}

// m / (sqrt(v) r + eps) within four units of 2^-24.  The root instruction takes subnormals for zero: with eps >= 1e-12 that is below
// the rounding of the sum (EXACT = false), else they are scaled.
template <bool EXACT> __device__ __forceinline__ float quotient(float m, float v, float r, float eps)
{
    float s;
    if (EXACT) {
        const bool low = v < 0x1p-96f;
        s = __builtin_amdgcn_sqrtf(low ? v * 0x1p64f : v) * (low ? 0x1p-32f : 1.f);
    } else {
        s = __builtin_amdgcn_sqrtf(v);
    }
    return m * __builtin_amdgcn_rcpf(s * r + eps);
}

// byte j of w as a code of the first / second moment: the float whose bits are the code << 20 (and the sign)
__device__ __forceinline__ float code_float_signed(uint32_t w, int j) { return __uint_as_float((uint32_t)((int32_t)(w << (24 - 8 * j)) >> 4) & 0x87F00000u); }
__device__ __forceinline__ float code_float(uint32_t w, int j) { return __uint_as_float((j < 3 ? w << (20 - 8 * j) : w >> 4) & 0x0FF00000u); }

// the upper bytes of four words as one word
__device__ __forceinline__ uint32_t upper_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x07030C0Cu), __builtin_amdgcn_perm(b, a, 0x0C0C0703u), 0x07060100u);
}

// x + the lower / upper half of bits << 4, in one instruction.  (Together with maxima as float operations
// and the padding's masks off the usual path: 105 M bfloat16 parameters with 8-bit moments 277 us instead of 290.)
__device__ __forceinline__ uint32_t add_low(uint32_t x, uint32_t bits)
{
    uint32_t r;
    asm("v_mad_u32_u16 %0, %1, 16, %2" : "=v"(r) : "v"(bits), "v"(x));
    return r;
}
__device__ __forceinline__ uint32_t add_high(uint32_t x, uint32_t bits)
{
    uint32_t r;
    asm("v_mad_u32_u16 %0, %1, 16, %2 op_sel:[1,0,0,0]" : "=v"(r) : "v"(bits), "v"(x));
    return r;
}

// what the update reads and writes: past the caches' replacement order (ONCE), or to be found there later
template <bool ONCE, typename T> __device__ __forceinline__ Vec<T, kLane> load_lane(const T* p) { return ONCE ? load_vec_once<T, kLane>(p) : load_vec<T, kLane>(p); }
template <bool ONCE, typename T> __device__ __forceinline__ void store_lane(T* p, const Vec<T, kLane>& v) { if (ONCE) store_vec_once<T, kLane>(p, v); else store_vec<T, kLane>(p, v); }

template <typename T, int BITS, bool ONCE>
__global__ __launch_bounds__(kWg) void adamw_update_kernel(UpdateTable tab, UpdateArgs a)
{
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63;
    const uint32_t tile = blockIdx.x * kWaves + wave;
    if (tile >= a.tiles) return;
    const int lo = tensor_of(tab.first, (int)a.count, tile);
    const uint32_t first = tab.first[lo], next = lo + 1 < (int)a.count ? tab.first[lo + 1] : a.tiles;
    const uint32_t slot = tab.slot_tail[lo] >> 10;
    const int have = min(kLane, (tile + 1 == next ? (int)(tab.slot_tail[lo] & 1023) : kTile) - lane * kLane);      // may be <= 0
    T* p = (T*)tab.p[lo] + (int64_t)(tile - first) * kTile + lane * kLane;
    const T* g = (const T*)tab.g[lo] + (int64_t)(tile - first) * kTile + lane * kLane;
    const int64_t pos = ((int64_t)tab.state[lo] + (tile - first)) * kTile + lane * kLane;
    Vec<T, kLane> pv, gv;
    if (have == kLane) {
        pv = load_lane<ONCE>(p);
        gv = load_lane<ONCE>(g);
    } else {
#pragma unroll
        for (int j = 0; j < kLane; ++j) { pv[j] = j < have ? p[j] : (T)0.f; gv[j] = j < have ? g[j] : (T)0.f; }
    }
    const float2 sc = a.scale[slot];
    const double clip = a.clip ? *a.clip : 1.0;
    const float lr = a.lr_device ? *a.lr_device : a.lr, keep = 1.f - lr * a.wd;
    uint32_t bits[kLane];
    if (BITS == 8 || sizeof(T) == 2) {
        const uint32_t t = (uint32_t)a.steps[slot];
        const uint32_t key = mix(mix(a.seed + kGolden * t) + (uint32_t)(pos >> 32)) + (uint32_t)pos * kGolden;
#pragma unroll
        for (int j = 0; j < kLane; ++j) bits[j] = mix(key + j * kGolden);
    }
    float mf[kLane], vf[kLane];
    if (BITS == 32) {
        float* ms = (float*)a.m + pos;
        float* vs = (float*)a.v + pos;
        Vec<float, kLane> mv = load_lane<ONCE>(ms), vv = load_lane<ONCE>(vs);
        const float b1 = (float)a.b1, b2 = (float)a.b2, c1 = (float)(1.0 - a.b1), c2 = (float)(1.0 - a.b2), cf = (float)clip;
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            const float e = to_float(gv[j]) * cf;
            mf[j] = b1 * mv[j] + c1 * e;
            vf[j] = b2 * vv[j] + c2 * e * e;
            mv[j] = mf[j];
            vv[j] = vf[j];
            if (j >= have) mv[j] = vv[j] = 0.f;                // padding stays zero whatever the coefficient
        }
        store_lane<ONCE>(ms, mv);                     // a tile's state is the bucket's own: whole, padding included
        store_lane<ONCE>(vs, vv);
    } else {
        uint8_t* ms = (uint8_t*)a.m + pos;
        uint8_t* vs = (uint8_t*)a.v + pos;
        const Vec<uint32_t, 2> mw = load_vec<uint32_t, 2>((const uint32_t*)ms), vw = load_vec<uint32_t, 2>((const uint32_t*)vs);
        const int me = a.me[pos / kBlock], ve = a.ve[pos / kBlock];
        // value of the float with bits c << 20: unit 2^-129; b1 and b2 go into the factor (an exact product)
        const double bad = __builtin_nan("");
        const double mscale = me == 255 ? bad : me == 0 ? 0.0 : a.b1 * exp2i(me - 127 - 16 + 129);
        const double vscale = ve == 255 ? bad : ve == 0 ? 0.0 : a.b2 * exp2i(ve - 127 - 32 + 129);
        const double c1 = (1.0 - a.b1) * clip, c2 = (1.0 - a.b2) * clip * clip;
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            const double e = (double)to_float(gv[j]);
            mf[j] = (float)(c1 * e + mscale * (double)code_float_signed(mw[j / 4], j % 4));
            vf[j] = (float)(c2 * e * e + vscale * (double)code_float(vw[j / 4], j % 4));
        }
        if (have < kLane) {                                             // padding stays zero whatever the coefficient
#pragma unroll
            for (int j = 0; j < kLane; ++j)
                if (j >= have) mf[j] = vf[j] = 0.f;
        }
        float mx = fabsf(mf[0]), vx = vf[0];                            // NaN is the largest, then infinity
#pragma unroll
        for (int j = 1; j < kLane; ++j) {
            mx = __builtin_elementwise_maximum(mx, fabsf(mf[j]));
            vx = __builtin_elementwise_maximum(vx, vf[j]);
        }
        const int mn = (int)(block_max(__float_as_uint(mx) & 0x7FFFFFFFu) >> 23), vn = (int)(block_max(__float_as_uint(vx) & 0x7FFFFFFFu) >> 23);
        const uint32_t mlive = mn != 0 && mn != 255 ? ~0u : 0u, vlive = vn != 0 && vn != 255 ? ~0u : 0u;
        Vec<uint32_t, 2> mo, vo;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint32_t mc[4], vc[4];                              // the code in the upper byte
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = 4 * w + i;
                const uint32_t mb = add_low(__float_as_uint(ldexpf(mf[j], 127 + 16 - 129 - mn)), bits[j]);
                const uint32_t vb = add_high(__float_as_uint(ldexpf(vf[j], 127 + 32 - 129 - vn)), bits[j]);
                mc[i] = (mb & 0x80000000u) | (mb << 4 & 0x7FFFFFFFu);
                vc[i] = max(vb, min(__float_as_uint(vf[j]), 1u) << 20) << 4;
            }
            mo[w] = upper_bytes(mc[0], mc[1], mc[2], mc[3]) & mlive;
            vo[w] = upper_bytes(vc[0], vc[1], vc[2], vc[3]) & vlive;
        }
        store_vec<uint32_t, 2>((uint32_t*)ms, mo);
        store_vec<uint32_t, 2>((uint32_t*)vs, vo);
        if (lane % (kBlock / kLane) == 0) { a.me[pos / kBlock] = (uint8_t)mn; a.ve[pos / kBlock] = (uint8_t)vn; }
    }
    float q[kLane];
    if (a.eps >= 1e-12f) {
#pragma unroll
        for (int j = 0; j < kLane; ++j) q[j] = quotient<false>(mf[j], vf[j], sc.y, a.eps);
    } else {
#pragma unroll
        for (int j = 0; j < kLane; ++j) q[j] = quotient<true>(mf[j], vf[j], sc.y, a.eps);
    }
#pragma unroll
    for (int j = 0; j < kLane; ++j) pv[j] = round_param<T>(to_float(pv[j]) * keep - sc.x * q[j], sizeof(T) == 2 ? mix(bits[j] + kGolden) & 0xFFFF : 0);
    if (have == kLane) store_lane<ONCE>(p, pv);
    else
        for (int j = 0; j < kLane; ++j) if (j < have) p[j] = pv[j];
}

// ---- 8-bit moments as numbers ---------------------------------------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(kWg) void adamw_decode_kernel(const uint8_t* __restrict__ m, const uint8_t* __restrict__ v,
                                                           const uint8_t* __restrict__ me, const uint8_t* __restrict__ ve, int64_t count,
                                                           T* __restrict__ mo, T* __restrict__ vo)
{
    const int64_t pos = ((int64_t)blockIdx.x * kWg + threadIdx.x) * kLane;
    if (pos >= count) return;
    const Vec<uint32_t, 2> mw = load_vec<uint32_t, 2>((const uint32_t*)(m + pos)), vw = load_vec<uint32_t, 2>((const uint32_t*)(v + pos));
    const int em = me[pos / kBlock], ev = ve[pos / kBlock];
    const double bad = __builtin_nan("");
    const double mscale = em == 255 ? bad : em == 0 ? 0.0 : exp2i(em - 127 - 16 + 129), vscale = ev == 255 ? bad : ev == 0 ? 0.0 : exp2i(ev - 127 - 32 + 129);
    Vec<T, kLane> a, b;
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
        a[j] = from_float<T>((float)(mscale * (double)code_float_signed(mw[j / 4], j % 4)));
        b[j] = from_float<T>((float)(vscale * (double)code_float(vw[j / 4], j % 4)));
    }
    store_vec_once<T, kLane>(mo + pos, a);
    store_vec_once<T, kLane>(vo + pos, b);
}

// ---- host ---------------------------------------------------------------------------------------------------------------

static int64_t tiles_of(int64_t n) { return (n + kTile - 1) / kTile; }

// how many tensors from the i-th on one launch takes, and their tiles: `most` of them, less than 2^32 threads
static int launch_share(const int64_t* numels, int i, int count, int most, int64_t& tiles)
{
    int n = 0;
    for (tiles = 0; i + n < count && n < most && tiles + tiles_of(numels[i + n]) < 1 << 26; ++n) tiles += tiles_of(numels[i + n]);
    return n;
}

// neighbouring tiles a wave of the norm pass takes: some 2048 workgroups, whole rounds of loads
static uint32_t norm_run(int64_t tiles)
{
    const int64_t run = tiles / (2048 * kWaves);
    return run < 1 ? 1 : (uint32_t)((run + kRun - 1) / kRun * kRun);
}
static int64_t norm_blocks(int64_t tiles) { const int64_t waves = (tiles + norm_run(tiles) - 1) / norm_run(tiles); return (waves + kWaves - 1) / kWaves; }

int64_t adamw_norm_partials(const int64_t* numels, int count)
{
    int64_t blocks = 0;
    for (int i = 0; i < count;) {
        int64_t tiles;
        i += launch_share(numels, i, count, kNormTensors, tiles);
        blocks += norm_blocks(tiles);
    }
    return blocks;
}

int launch_adamw_norm(const void* const* grads, const int64_t* numels, int count, int dtype, double* partial, hipStream_t s)
{
    for (int i = 0; i < count;) {
        NormTable tab;
        uint32_t tiles = 0;
        int64_t all;
        const int n = launch_share(numels, i, count, kNormTensors, all);
        for (int k = 0; k < n; ++k) {
            const int64_t t = tiles_of(numels[i + k]);
            tab.grad[k] = grads[i + k];
            tab.first[k] = tiles;
            tab.tail[k] = (uint16_t)(numels[i + k] - (t - 1) * kTile);
            tiles += (uint32_t)t;
        }
        const unsigned blocks = (unsigned)norm_blocks(tiles);
        if (dtype == RAFTCORR_DTYPE_FP32) adamw_norm_kernel<float><<<blocks, kWg, 0, s>>>(tab, n, tiles, norm_run(tiles), partial);
        else adamw_norm_kernel<__bf16><<<blocks, kWg, 0, s>>>(tab, n, tiles, norm_run(tiles), partial);
        partial += blocks;
        i += n;
    }
    return check_launch("adamw_norm");
}

int launch_adamw_step(void* const* params, const void* const* grads, const int64_t* numels, const int64_t* offsets, const int32_t* slots,
                      int count, int dtype, int bits, void* m, void* v, uint8_t* me, uint8_t* ve, float* steps, float* scale,
                      double lr, const float* lr_device, double b1, double b2, double eps, double wd, uint32_t seed,
                      const double* partial, int partials, double max_norm, double* clip, float* norm, hipStream_t s)
{
    for (int i = 0; i < count; i += kStepTensors) {
        StepTable tab;
        const int n = count - i < kStepTensors ? count - i : kStepTensors;
        for (int k = 0; k < n; ++k) tab.slot[k] = slots[i + k];
        adamw_count_kernel<<<1, kCountWg, 0, s>>>(tab, n, steps, (float2*)scale, lr, lr_device, b1, b2, partial, i == 0 ? partials : 0,
                                             max_norm, clip, norm);
    }
    // More than the 256 MB last-level cache keeps from one step to the next: nothing of it is worth a place there.  With the norm pass, in
    // us, so | kept: 105 M values bfloat16 444 | 487 (32 bits), 289 | 314 (8); float32 627 | 647; 5 M float32 41 | 38.
    int64_t values = 0;
    for (int i = 0; i < count; ++i) values += numels[i];
    const bool once = values * (2 * (dtype == RAFTCORR_DTYPE_FP32 ? 4 : 2) + (bits == 32 ? 8 : 2)) > 256 << 20;
    for (int i = 0; i < count;) {
        UpdateTable tab;
        uint32_t tiles = 0;
        int64_t all;
        const int n = launch_share(numels, i, count, kUpdateTensors, all);
        for (int k = 0; k < n; ++k) {
            const int64_t t = tiles_of(numels[i + k]);
            tab.p[k] = (uint64_t)params[i + k];
            tab.g[k] = (uint64_t)grads[i + k];
            tab.first[k] = tiles;
            tab.state[k] = (uint32_t)(offsets[i + k] / kTile);
            tab.slot_tail[k] = (uint32_t)slots[i + k] << 10 | (uint32_t)(numels[i + k] - (t - 1) * kTile);
            tiles += (uint32_t)t;
        }
        const UpdateArgs a{m, v, me, ve, steps, (const float2*)scale, partials ? clip : nullptr, lr_device, b1, b2,
                           (float)lr, (float)eps, (float)wd, seed, (uint32_t)n, tiles};
        const unsigned blocks = (tiles + kWaves - 1) / kWaves;
        auto launch = [&](auto t, auto once) {
            if (bits == 32) adamw_update_kernel<decltype(t), 32, decltype(once)::value><<<blocks, kWg, 0, s>>>(tab, a);
            else adamw_update_kernel<decltype(t), 8, decltype(once)::value><<<blocks, kWg, 0, s>>>(tab, a);
        };
        if (dtype == RAFTCORR_DTYPE_FP32) { if (once) launch(float(), std::true_type()); else launch(float(), std::false_type()); }
        else { if (once) launch(__bf16(), std::true_type()); else launch(__bf16(), std::false_type()); }
        i += n;
    }
    return check_launch("adamw_step");
}

int launch_adamw_decode(const uint8_t* m, const uint8_t* v, const uint8_t* me, const uint8_t* ve, int64_t count, int dtype, void* mo, void* vo,
                        hipStream_t s)
{
    const unsigned blocks = (unsigned)((count / kLane + kWg - 1) / kWg);
    if (dtype == RAFTCORR_DTYPE_FP32) adamw_decode_kernel<float><<<blocks, kWg, 0, s>>>(m, v, me, ve, count, (float*)mo, (float*)vo);
    else adamw_decode_kernel<__bf16><<<blocks, kWg, 0, s>>>(m, v, me, ve, count, (__bf16*)mo, (__bf16*)vo);
    return check_launch("adamw_decode");
}

}  // namespace raftcorr

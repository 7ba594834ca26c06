// The AdamW step of many tensors, with moments in 32 or in 8 bits and the gradients clipped by their global norm.
//
//   c = min(1, max_norm / (|g| + 1e-6)),  m = b1 m + (1 - b1) c g,  v = b2 v + (1 - b2) (c g)^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Memory bound: 28 bytes a float32 parameter with 32-bit moments, 16 with 8-bit ones, some 20 operations.  Launches: sums of
// squares of the gradients (only with clipping), one workgroup that counts the steps and joins the sums, the update; each takes
// the tensors' addresses by value, as many as 4 KB of kernel arguments hold, so a captured graph depends on no table.
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
#include "common.h"
#include "elem.h"

namespace raftcorr {

enum { kTile = RAFTCORR_ADAMW_TILE, kBlock = RAFTCORR_ADAMW_BLOCK, kLane = 8, kWg = 256, kWaves = kWg / 64 };
static_assert(kTile == 64 * kLane && kBlock % kLane == 0 && kTile % kBlock == 0, "a lane's values share a block, a wave's tile holds whole blocks");

// ---- gradient norm ------------------------------------------------------------------------------------------------------

enum { kNormTensors = 240 };
struct NormTable {
    const void* grad[kNormTensors];
    uint32_t first[kNormTensors];             // first tile of each tensor, counted from the first tensor of the launch
    uint16_t tail[kNormTensors];              // values in its last tile
};

// the tensor a tile belongs to: the last one that starts at or before it
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

// partial[block] = sum of squares over the tiles of the block's waves, in 64 bits
template <typename T>
__global__ __launch_bounds__(kWg) void adamw_norm_kernel(NormTable tab, int count, uint32_t tiles, double* __restrict__ partial)
{
    __shared__ double part[kWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63;
    double sum = 0.0;
    for (uint32_t tile = blockIdx.x * kWaves + wave; tile < tiles; tile += gridDim.x * kWaves) {
        const int i = tensor_of(tab.first, count, tile);
        const uint32_t next = i + 1 < count ? tab.first[i + 1] : tiles;
        const int values = tile + 1 == next ? tab.tail[i] : kTile;
        const T* g = (const T*)tab.grad[i] + (int64_t)(tile - tab.first[i]) * kTile + lane * kLane;
        const int have = values - lane * kLane;
        if (have >= kLane) {
            const Vec<T, kLane> v = load_vec<T, kLane>(g);
#pragma unroll
            for (int j = 0; j < kLane; ++j) { const double e = (double)to_float(v[j]); sum += e * e; }
        } else {
            for (int j = 0; j < have; ++j) { const double e = (double)to_float(g[j]); sum += e * e; }
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

// counts the tensors' steps; scale[slot] = (lr / (1 - b1^t), 1 / sqrt(1 - b2^t)); joins the partial sums (partials > 0)
__global__ __launch_bounds__(kWg) void adamw_count_kernel(StepTable tab, int count, float* __restrict__ steps, float2* __restrict__ scale,
                                                          double lr, const float* __restrict__ lr_device, double b1, double b2,
                                                          const double* __restrict__ partial, int partials, double max_norm,
                                                          double* __restrict__ clip, float* __restrict__ norm)
{
    if (lr_device) lr = (double)*lr_device;
    for (int i = threadIdx.x; i < count; i += kWg) {
        const int slot = tab.slot[i];
        const float t = steps[slot] + 1.f;
        steps[slot] = t;
        scale[slot] = make_float2((float)(lr / (1.0 - pow(b1, (double)t))), (float)(1.0 / sqrt(1.0 - pow(b2, (double)t))));
    }
    if (!partials) return;
    __shared__ double part[kWaves];
    double sum = 0.0;
    for (int i = threadIdx.x; i < partials; i += kWg) sum += partial[i];
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < kWaves; ++w) sum += part[w];
    sum = sqrt(sum);
    const double c = max_norm / (sum + 1e-6);
    *clip = c > 1.0 ? 1.0 : c;                  // (a NaN stays one)
    *norm = (float)sum;
}

// ---- update -------------------------------------------------------------------------------------------------------------

enum { kStepWords = 32, kUpdateTensors = 120 };
struct UpdateTensor {
    void* p;
    const void* g;
    uint32_t first, state;                      // first tile in the launch, first tile in the bucket's buffers
    uint32_t slot, tail;
};
struct UpdateTable { UpdateTensor t[kUpdateTensors]; };

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

// the largest of 8 lanes' values (the lanes of one block)
__device__ __forceinline__ float block_max(float v)
{
#pragma unroll
    for (int o = 1; o < kBlock / kLane; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// |x| of exponent at most E, in units of 2^(E - 127 - top), to its code: below 8 units 8 is added, which lines the units up with the
// same bit of the word that ends the three mantissa bits above; the random bits then carry into it or not.
__device__ __forceinline__ uint32_t encode(float x, int shift, uint32_t bits16)
{
    const float u = ldexpf(x, shift);
    const bool low = u < 8.f;
    const uint32_t w = __float_as_uint(low ? u + 8.f : u) + (bits16 << 4);
    return (w >> 20) - ((0x41000000u >> 20) - (low ? 0u : 8u));
}

__device__ __forceinline__ double decode(uint32_t code, int shift)
{
    const uint32_t units = code < 8 ? code : 8 + (code & 7);
    return ldexp((double)units, shift + (code < 8 ? 0 : (int)(code >> 3) - 1));
}

template <typename T> __device__ __forceinline__ T round_param(float x, uint32_t) { return (T)x; }
// bfloat16 parameters are rounded up with the probability of what is dropped: a step of 2^-9 of a weight would be lost otherwise
template <> __device__ __forceinline__ __bf16 round_param<__bf16>(float x, uint32_t bits16)
{
    const uint32_t w = __float_as_uint(x);
    if ((w & 0x7F800000u) == 0x7F800000u) return (__bf16)x;                   // infinities and NaN as they are
    return __builtin_bit_cast(__bf16, (uint16_t)((w + bits16) >> 16));
}

template <typename T, int BITS>
__global__ __launch_bounds__(kWg) void adamw_update_kernel(UpdateTable tab, UpdateArgs a)
{
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x & 63;
    const uint32_t tile = blockIdx.x * kWaves + wave;
    if (tile >= a.tiles) return;
    int lo = 0, hi = (int)a.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (tab.t[mid].first <= tile) lo = mid; else hi = mid;
    }
    const uint32_t first = tab.t[lo].first, next = lo + 1 < (int)a.count ? tab.t[lo + 1].first : a.tiles;
    const uint32_t slot = tab.t[lo].slot;
    const int have = min(kLane, (tile + 1 == next ? (int)tab.t[lo].tail : kTile) - lane * kLane);      // may be <= 0
    T* p = (T*)tab.t[lo].p + (int64_t)(tile - first) * kTile + lane * kLane;
    const T* g = (const T*)tab.t[lo].g + (int64_t)(tile - first) * kTile + lane * kLane;
    const int64_t pos = ((int64_t)tab.t[lo].state + (tile - first)) * kTile + lane * kLane;
    Vec<T, kLane> pv, gv;
    if (have == kLane) {
        pv = load_vec<T, kLane>(p);
        gv = load_vec<T, kLane>(g);
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
        const uint32_t key = mix(mix(a.seed + kGolden * t) + (uint32_t)(pos >> 32));
#pragma unroll
        for (int j = 0; j < kLane; ++j) bits[j] = mix(((uint32_t)pos + j) * kGolden + key);
    }
    float mf[kLane], vf[kLane];
    if (BITS == 32) {
        float* ms = (float*)a.m + pos;
        float* vs = (float*)a.v + pos;
        Vec<float, kLane> mv = load_vec<float, kLane>(ms), vv = load_vec<float, kLane>(vs);
        const float b1 = (float)a.b1, b2 = (float)a.b2, c1 = (float)(1.0 - a.b1), c2 = (float)(1.0 - a.b2), cf = (float)clip;
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            const float e = to_float(gv[j]) * cf;
            mf[j] = b1 * mv[j] + c1 * e;
            vf[j] = b2 * vv[j] + c2 * e * e;
            mv[j] = mf[j];
            vv[j] = vf[j];
        }
        store_vec<float, kLane>(ms, mv);                       // a tile's state is the bucket's own: whole, padding included
        store_vec<float, kLane>(vs, vv);
    } else {
        uint8_t* ms = (uint8_t*)a.m + pos;
        uint8_t* vs = (uint8_t*)a.v + pos;
        Vec<uint8_t, kLane> mv = load_vec<uint8_t, kLane>(ms), vv = load_vec<uint8_t, kLane>(vs);
        const int me = a.me[pos / kBlock], ve = a.ve[pos / kBlock];
        const double bad = __builtin_nan(""), c1 = 1.0 - a.b1, c2 = 1.0 - a.b2;
        float mx = 0.f, vx = 0.f;
        bool finite = true;
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            double m = me == 255 ? bad : me == 0 ? 0.0 : decode(mv[j] & 127, me - 127 - 16);
            if (mv[j] & 128) m = -m;
            const double v = ve == 255 ? bad : ve == 0 ? 0.0 : decode(vv[j], ve - 127 - 32);
            const double e = (double)to_float(gv[j]) * clip;
            mf[j] = (float)(a.b1 * m + c1 * e);
            vf[j] = (float)(a.b2 * v + c2 * e * e);
            mx = fmaxf(mx, fabsf(mf[j]));
            vx = fmaxf(vx, vf[j]);
            finite = finite && mf[j] - mf[j] == 0.f && vf[j] - vf[j] == 0.f;
        }
        mx = block_max(finite ? mx : __builtin_inff());
        vx = block_max(finite ? vx : __builtin_inff());
        const int mn = (int)(__float_as_uint(mx) >> 23), vn = (int)(__float_as_uint(vx) >> 23);
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            uint32_t m = 0, v = 0;
            if (mn != 0 && mn != 255) m = encode(fabsf(mf[j]), 127 + 16 - mn, bits[j] & 0xFFFF) | (mf[j] < 0.f ? 128u : 0u);
            if (vn != 0 && vn != 255) {
                v = encode(vf[j], 127 + 32 - vn, bits[j] >> 16);
                if (v == 0 && vf[j] > 0.f) v = 1;
            }
            mv[j] = (uint8_t)m;
            vv[j] = (uint8_t)v;
        }
        store_vec<uint8_t, kLane>(ms, mv);
        store_vec<uint8_t, kLane>(vs, vv);
        if (lane % (kBlock / kLane) == 0) { a.me[pos / kBlock] = (uint8_t)mn; a.ve[pos / kBlock] = (uint8_t)vn; }
    }
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
        const float n = to_float(pv[j]) * keep - sc.x * mf[j] / (sqrtf(vf[j]) * sc.y + a.eps);
        pv[j] = round_param<T>(n, sizeof(T) == 2 ? mix(bits[j] + kGolden) & 0xFFFF : 0);
    }
    if (have == kLane) store_vec<T, kLane>(p, pv);
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
    const Vec<uint8_t, kLane> mc = load_vec<uint8_t, kLane>(m + pos), vc = load_vec<uint8_t, kLane>(v + pos);
    const int em = me[pos / kBlock], ev = ve[pos / kBlock];
    Vec<T, kLane> a, b;
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
        float x = em == 255 ? __builtin_nanf("") : em == 0 ? 0.f : (float)decode(mc[j] & 127, em - 127 - 16);
        if (mc[j] & 128) x = -x;
        a[j] = from_float<T>(x);
        b[j] = from_float<T>(ev == 255 ? __builtin_nanf("") : ev == 0 ? 0.f : (float)decode(vc[j], ev - 127 - 32));
    }
    store_vec<T, kLane>(mo + pos, a);
    store_vec<T, kLane>(vo + pos, b);
}

// ---- host ---------------------------------------------------------------------------------------------------------------

static int64_t tiles_of(int64_t n) { return (n + kTile - 1) / kTile; }

// workgroups of the norm pass over `tiles` tiles
static int64_t norm_blocks(int64_t tiles) { const int64_t b = (tiles + kWaves - 1) / kWaves; return b < 1024 ? b : 1024; }

int64_t adamw_norm_partials(const int64_t* numels, int count)
{
    int64_t blocks = 0;
    for (int i = 0; i < count;) {
        int64_t tiles = 0;
        const int n = count - i < kNormTensors ? count - i : kNormTensors;
        for (int k = 0; k < n; ++k) tiles += tiles_of(numels[i + k]);
        blocks += norm_blocks(tiles);
        i += n;
    }
    return blocks;
}

int launch_adamw_norm(const void* const* grads, const int64_t* numels, int count, int dtype, double* partial, hipStream_t s)
{
    for (int i = 0; i < count;) {
        NormTable tab;
        uint32_t tiles = 0;
        const int n = count - i < kNormTensors ? count - i : kNormTensors;
        for (int k = 0; k < n; ++k) {
            const int64_t t = tiles_of(numels[i + k]);
            tab.grad[k] = grads[i + k];
            tab.first[k] = tiles;
            tab.tail[k] = (uint16_t)(numels[i + k] - (t - 1) * kTile);
            tiles += (uint32_t)t;
        }
        const unsigned blocks = (unsigned)norm_blocks(tiles);
        if (dtype == RAFTCORR_DTYPE_FP32) adamw_norm_kernel<float><<<blocks, kWg, 0, s>>>(tab, n, tiles, partial);
        else adamw_norm_kernel<__bf16><<<blocks, kWg, 0, s>>>(tab, n, tiles, partial);
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
        adamw_count_kernel<<<1, kWg, 0, s>>>(tab, n, steps, (float2*)scale, lr, lr_device, b1, b2, partial, i == 0 ? partials : 0,
                                             max_norm, clip, norm);
    }
    for (int i = 0; i < count;) {
        UpdateTable tab;
        uint32_t tiles = 0;
        const int n = count - i < kUpdateTensors ? count - i : kUpdateTensors;
        for (int k = 0; k < n; ++k) {
            const int64_t t = tiles_of(numels[i + k]);
            tab.t[k] = UpdateTensor{params[i + k], grads[i + k], tiles, (uint32_t)(offsets[i + k] / kTile), (uint32_t)slots[i + k],
                                    (uint32_t)(numels[i + k] - (t - 1) * kTile)};
            tiles += (uint32_t)t;
        }
        const UpdateArgs a{m, v, me, ve, steps, (const float2*)scale, partials ? clip : nullptr, lr_device, b1, b2,
                           (float)lr, (float)eps, (float)wd, seed, (uint32_t)n, tiles};
        const unsigned blocks = (tiles + kWaves - 1) / kWaves;
        if (dtype == RAFTCORR_DTYPE_FP32) {
            if (bits == 32) adamw_update_kernel<float, 32><<<blocks, kWg, 0, s>>>(tab, a);
            else adamw_update_kernel<float, 8><<<blocks, kWg, 0, s>>>(tab, a);
        } else {
            if (bits == 32) adamw_update_kernel<__bf16, 32><<<blocks, kWg, 0, s>>>(tab, a);
            else adamw_update_kernel<__bf16, 8><<<blocks, kWg, 0, s>>>(tab, a);
        }
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

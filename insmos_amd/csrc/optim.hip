// insmos_amd/csrc/optim.hip -- one AdamW / Adam step over a list of tensors, moments in 32 or in 8 bits, with the clip by the
// gradients' global norm (the optimiser of models/models.py:185-190 as one short chain of launches instead of a chain per tensor).
//
//   g' = c g (+ wd p when the decay is coupled),  c = min(1, max_norm / (|g| + 1e-6)) or 1
//   m  = b1 m + (1 - b1) g'        v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd or 1) - lr / (1 - b1^t) * (m / (sqrt(v) / sqrt(1 - b2^t) + eps))
//
// Bound: HBM.  An element moves 28 bytes with fp32 tensors and moments (p, m, v read and written, g read; + 4 when the norm is
// taken), 16 with moments in 8 bits; the arithmetic is some 45 (32 bits) or 75 (8 bits) vector instructions per element.
//
// Layout: the moments (and fp32 master weights) of a list lie in ONE buffer each; tensor i starts at a multiple of 256 elements, so
// their accesses are 16-byte ones whatever the tensors are, and only p and g come with an address each.  The addresses travel as
// kernel arguments, up to 140 tensors per launch: no table in device memory to fill, nothing kept between calls, and a captured
// graph holds what it needs.  What depends on the step (t, the bias corrections, c) is computed on the device by k_adamw_prepare,
// from a step counter in device memory: a replayed graph advances, and the host waits for nothing.
//
// 8 bits: 256 consecutive elements share an fp32 scale, largest / 448 (e4m3's largest number), for m and for s = sqrt(v) each.  s and not
// v, because its range within a block is the root of v's, and 3 mantissa bits of s are what the step divides by.  With b2 = 0.999 an
// update moves s by 1/2000 of itself or less, far below the distance of neighbouring codes (1/8 to 1/16): rounded to nearest, s would
// never move.  So codes are rounded up or down at random, with the right mean: 16 bits each from a hash of (position, step, seed) --
// the same call gives the same bits.  s > 0 never becomes 0 (m / eps would be an enormous step); what is not finite becomes NaN (0x7f) and
// stays out of its block's scale.  m, s and the update itself are fp32; only what is stored is rounded.
#include <cmath>
#include "common.h"

namespace insmos {
namespace {

constexpr int OPT_BLOCK = 256;      // elements per scale and alignment of a tensor in the state buffers
constexpr int STEP_CHUNK = 4096;    // elements per workgroup of the step: 4 x (4 per lane x 256 lanes)
constexpr int NORM_CHUNK = 8192;    // ... of the norm (one 8-byte partial sum each); 16 bytes a lane and load
constexpr int64_t PART = 1 << 30;   // a longer tensor travels as several entries of this many elements

// A launch's arguments may have 4 KB: 140 entries of 28 bytes for the step, 250 of 16 for the norm.
struct StepList {
    static constexpr int MOST = 140;
    void* p[MOST];
    const void* g[MOST];
    uint32_t n[MOST];
    uint32_t off[MOST];              // start in the state buffers, in blocks of 256
    uint32_t first[MOST + 1];        // first workgroup of every entry
    int count;
    void set(int i, void* param, const void* grad, int64_t numel, int64_t state_off) {
        p[i] = param; g[i] = grad; n[i] = (uint32_t)numel; off[i] = (uint32_t)(state_off / OPT_BLOCK);
    }
};
struct NormList {
    static constexpr int MOST = 250;
    const void* g[MOST];
    uint32_t n[MOST];
    uint32_t first[MOST + 1];
    int count;
    void set(int i, void*, const void* grad, int64_t numel, int64_t) { g[i] = grad; n[i] = (uint32_t)numel; }
};
struct StepVals {   // what the launches of one step share (device memory)
    float clip, keep, size, root;        // c, factor of p, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    uint32_t key;                        // hash of step and seed
    int skip;
};

typedef float of32x4 __attribute__((ext_vector_type(4)));
typedef float of32x8 __attribute__((ext_vector_type(8)));
template <class T, int V> struct VecOf { typedef T t __attribute__((ext_vector_type(V))); };

// A published mixer of 32 bits (C. Wellons, 2018: shifts and factors found by a search for the least bias), over position, step and seed.
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x ^= x >> 16; x *= 0x7FEB352Du;
    x ^= x >> 15; x *= 0x846CA68Bu;
    return x ^ (x >> 16);
}
// The tensor a workgroup works on: how many of the list's starts are not behind it.  Every lane looks at a few of them at once (a search, whose
// reads wait for each other, cost 0.6 to 1 us more per launch: 250 tensors' norm 9.5 -> 8.6 us, 140 tensors' update 21.3 -> 20.3).
template <class List>
__device__ __forceinline__ int tensor_of(const List& L, uint32_t b) {
    const int lane = threadIdx.x & 63;
    int t = -1;
#pragma unroll
    for (int i = 0; i < List::MOST; i += 64) {
        const bool in = i + lane < L.count;
        const uint32_t first = L.first[min(i + lane, List::MOST)];
        t += __builtin_popcountll(__ballot(in && first <= b));
    }
    return __builtin_amdgcn_readfirstlane(t);
}
// V (4 or 8) elements of a tensor from element i on; zeros past its end; `wide` = the tensor's address allows one access
template <int V, class T>
__device__ __forceinline__ typename VecOf<float, V>::t load_v(const T* __restrict__ p, uint32_t i, uint32_t n, bool wide) {
    typedef typename VecOf<float, V>::t FV;
    if (wide && i + V <= n) return __builtin_convertvector(*(const typename VecOf<T, V>::t*)(p + i), FV);
    FV r;
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = i + j < n ? (float)p[i + j] : 0.f;
    return r;
}
template <int V, class T>
__device__ __forceinline__ void store_v(T* __restrict__ p, uint32_t i, uint32_t n, bool wide, typename VecOf<float, V>::t v) {
    typedef typename VecOf<T, V>::t TV;
    if (wide && i + V <= n) { *(TV*)(p + i) = __builtin_convertvector(v, TV); return; }
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (i + j < n) p[i + j] = (T)v[j];
}
// (a vector of 32 bytes is two accesses of 16)
template <class T, int V>
__device__ __forceinline__ bool is_wide(const void* a) { return ((uintptr_t)a & (V * sizeof(T) < 16 ? V * sizeof(T) - 1 : 15)) == 0; }

// ---- the gradients' sum of squares: one fp64 partial per workgroup (fixed order: the same bits every time) ------------------
// Four squares are added in fp32 (their rounding errors have no direction and average out) and the sums in fp64: a quarter of the
// fp64 work.  Sums near fp32's limits are taken in fp64.
template <int V>
__device__ __forceinline__ void add_squares(double& s, const typename VecOf<float, V>::t v) {
#pragma unroll
    for (int h = 0; h < V; h += 4) {
        const float q = fmaf(v[h], v[h], v[h + 1] * v[h + 1]) + fmaf(v[h + 2], v[h + 2], v[h + 3] * v[h + 3]);
        if (q >= 1e-30f && q <= 1e37f) s += (double)q;
        else
#pragma unroll
            for (int j = 0; j < 4; ++j) s = fma((double)v[h + j], (double)v[h + j], s);
    }
}
template <class T>
__global__ void __launch_bounds__(256) k_grad_sumsq(const NormList L, double* __restrict__ partial) {
    constexpr int V = 16 / sizeof(T), STEP = 256 * V;
    typedef typename VecOf<float, V>::t FV;
    typedef typename VecOf<T, V>::t TV;
    const int t = tensor_of(L, blockIdx.x);
    const T* g = (const T*)L.g[t];
    const uint32_t n = L.n[t], base = (blockIdx.x - L.first[t]) * NORM_CHUNK;
    const bool wide = is_wide<T, V>(g);
    double s = 0.0;
    if (wide && base + NORM_CHUNK <= n) {   // a whole chunk: all loads in flight
        TV v[NORM_CHUNK / STEP];
#pragma unroll
        for (int u = 0; u < NORM_CHUNK / STEP; ++u) v[u] = *(const TV*)(g + base + u * STEP + threadIdx.x * V);
#pragma unroll
        for (int u = 0; u < NORM_CHUNK / STEP; ++u) add_squares<V>(s, __builtin_convertvector(v[u], FV));
    } else {
        for (int u = 0; u < NORM_CHUNK / STEP; ++u) {
            const uint32_t i = base + u * STEP + threadIdx.x * V;
            if (i < n) add_squares<V>(s, load_v<V>(g, i, n, wide));
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    __shared__ double w[4];
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = (w[0] + w[1]) + (w[2] + w[3]);
}
__device__ __forceinline__ double sum_partials(const double* __restrict__ partial, int64_t n, double* w) {
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += partial[i];
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
    for (int q = 0; q < 16; ++q) s += w[q];
    return s;
}
__global__ void __launch_bounds__(1024) k_grad_norm(const double* __restrict__ partial, int64_t n, float* __restrict__ norm) {
    __shared__ double w[16];
    const double s = sum_partials(partial, n, w);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

struct PrepareP {
    const double* partial;   // sums of squares to add up, or null
    int64_t n_partial;
    const float* norm_in;    // the norm itself, or null
    float* norm_out;         // or null
    const float* lr_dev;     // or null: lr
    double lr, b1, b2, wd, max_norm;
    int decoupled, clip, skip_nonfinite;
    uint32_t seed;
    int32_t* step;
    StepVals* vals;
};
__global__ void __launch_bounds__(1024) k_adamw_prepare(const PrepareP A) {
    __shared__ double w[16];
    double norm = 0.0;
    if (A.partial) norm = sqrt(sum_partials(A.partial, A.n_partial, w));
    if (threadIdx.x > 1) return;
    if (A.norm_in) norm = (double)*A.norm_in;
    StepVals v;
    v.skip = A.skip_nonfinite && !((float)norm <= 3.402823466e38f);   // (what norm_out says)
    const int t = *A.step + (v.skip ? 0 : 1);
    const double power = pow(threadIdx.x ? A.b2 : A.b1, (double)t), power2 = __shfl(power, 1);   // lane 0: b1^t, lane 1: b2^t
    if (threadIdx.x) return;
    if (A.norm_out) *A.norm_out = (float)norm;
    *A.step = t;
    const double lr = A.lr_dev ? (double)*A.lr_dev : A.lr;
    v.clip = 1.f;
    if (A.clip) {
        const float c = (float)(A.max_norm / (norm + 1e-6));
        v.clip = c >= 1.f ? 1.f : c;   // (a norm that is NaN stays one)
    }
    v.keep = A.decoupled ? (float)(1.0 - lr * A.wd) : 1.f;
    v.size = (float)(lr / (1.0 - power));
    v.root = (float)(1.0 / sqrt(1.0 - power2));
    v.key = mix32(mix32((uint32_t)t) ^ A.seed);
    *A.vals = v;
}

struct StepP {
    const StepVals* vals;
    void* m;          // float or e4m3 codes
    void* v;          // float: v; e4m3 codes: sqrt(v)
    float* scales;    // 8 bits: [2][n_blocks]
    int64_t n_blocks;
    float* masters;   // fp32 weights in the state layout, or null
    float b1, a1, b2, a2, eps, wd;   // a = 1 - b; wd: the coupled decay (0 when decoupled)
    int coupled;
};

// 20 bits of mantissa are rounded away: x (>= 0) in units of the block's scale -> e4m3 code.  e4m3's smallest normal number 2^-6 is
// taken to fp32's 2^-126, so that exponent and first three mantissa bits ARE the code, below the normal numbers too.
__device__ __forceinline__ uint32_t code_of(float a, float inv, uint32_t u16) {
    const float y = fminf(a * inv, 448.f) * 0x1p-120f;
    return (__float_as_uint(y) + (u16 << 4)) >> 20;
}
// the largest value of each half of the wave, in all of its lanes: rotations within the rows of 16, then the rows of a half exchanged
__device__ __forceinline__ uint32_t half_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, false));   // row_ror:8, 4, 2, 1
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, false));
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}
__device__ __forceinline__ of32x8 decode8(uint2 c, float scale) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, true);
    const auto d = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, false), e = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, true);
    of32x8 r = {a[0] * scale, a[1] * scale, b[0] * scale, b[1] * scale, d[0] * scale, d[1] * scale, e[0] * scale, e[1] * scale};
    return r;
}
// Root and quotient with one correction of v_rsq's / v_rcp's result: the correctly rounded value but for about one argument in a million (one
// unit in the last place off there), at half of the general functions' instructions.  x in 2^-96 .. 2^96; d = a root of that times a factor + eps.
__device__ __forceinline__ float root_of(float x) {
    const float y = __builtin_amdgcn_rsqf(x), s = x * y;
    return fmaf(fmaf(-s, s, x), 0.5f * y, s);
}
__device__ __forceinline__ float quotient(float a, float d) {
    const float y = __builtin_amdgcn_rcpf(d), q = a * y;
    return fmaf(fmaf(-d, q, a), y, q);
}

// Moments in 32 bits: 4 elements a lane.  Bound by HBM: 120 M bf16 parameters with fp32 masters 610 us (5.5 TB/s), 140 tensors of 3.6 M fp32 values
// 21 us (4.8).
template <class T, bool MASTER>
__global__ void __launch_bounds__(256) k_adamw(const StepList L, const StepP A) {
    const StepVals S = *A.vals;
    if (S.skip) return;
    const int t = tensor_of(L, blockIdx.x);
    T* p = (T*)L.p[t];
    const T* g = (const T*)L.g[t];
    const uint32_t n = L.n[t], base = (blockIdx.x - L.first[t]) * STEP_CHUNK;
    const bool wide = is_wide<T, 4>(p) && is_wide<T, 4>(g);
    const int64_t off = (int64_t)L.off[t] * OPT_BLOCK;
#pragma unroll
    for (int u = 0; u < STEP_CHUNK / 1024; ++u) {
        const uint32_t i = base + u * 1024 + threadIdx.x * 4;
        if ((i & ~(uint32_t)(OPT_BLOCK - 1)) >= n) break;   // (a wave's 256 elements are one block of the state)
        const int64_t s = off + i;
        const of32x4 gr = load_v<4>(g, i, n, wide), pr = MASTER ? *(const of32x4*)(A.masters + s) : load_v<4>((const T*)p, i, n, wide);
        of32x4 m = *(const of32x4*)((const float*)A.m + s), v = *(const of32x4*)((const float*)A.v + s), np;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float gj = gr[j] * S.clip;
            if (A.coupled) gj = gj + A.wd * pr[j];
            m[j] = A.b1 * m[j] + A.a1 * gj;
            v[j] = A.b2 * v[j] + A.a2 * (gj * gj);
            np[j] = pr[j] * S.keep - S.size * (m[j] / (sqrtf(v[j]) * S.root + A.eps));
            if (i + j >= n) m[j] = v[j] = np[j] = 0.f;   // behind the tensor's end the state holds zeros
        }
        if (MASTER) *(of32x4*)(A.masters + s) = np;
        store_v<4>(p, i, n, wide, np);
        *(of32x4*)((float*)A.m + s) = m;
        *(of32x4*)((float*)A.v + s) = v;
    }
}

// Moments in 8 bits: 8 elements a lane, a block is half a wave.  Bound by the vector instructions (some 75 per element, the hash's two products
// and the codes among them) as much as by its bytes: 200 M bf16 parameters 395 us, their 2 GB at 5.5 TB/s 364; with 4 elements a lane, the general
// root and division and the wave's maximum through the LDS 546.
template <class T, bool MASTER>
__global__ void __launch_bounds__(256) k_adamw8(const StepList L, const StepP A) {
    const StepVals S = *A.vals;
    if (S.skip) return;
    const int t = tensor_of(L, blockIdx.x);
    T* p = (T*)L.p[t];
    const T* g = (const T*)L.g[t];
    const uint32_t n = L.n[t], base = (blockIdx.x - L.first[t]) * STEP_CHUNK;
    const bool wide = is_wide<T, 8>(p) && is_wide<T, 8>(g);
    constexpr uint32_t INF = 0x7F800000u;
#pragma unroll
    for (int u = 0; u < STEP_CHUNK / 2048; ++u) {
        const uint32_t i = base + u * 2048 + threadIdx.x * 8, from = i & ~(uint32_t)(OPT_BLOCK - 1);
        if (from >= n) break;   // (the same for the half wave: what follows exchanges values within halves)
        const int64_t b = (int64_t)L.off[t] + from / OPT_BLOCK, s = b * OPT_BLOCK + (i - from);
        const of32x8 gr = load_v<8>(g, i, n, wide), pr = MASTER ? *(const of32x8*)(A.masters + s) : load_v<8>((const T*)p, i, n, wide);
        of32x8 m = decode8(*(const uint2*)((const uint8_t*)A.m + s), A.scales[b]);
        of32x8 v = decode8(*(const uint2*)((const uint8_t*)A.v + s), A.scales[A.n_blocks + b]);
        of32x8 root, np;
        float least = 1.f, most = 1.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float gj = gr[j] * S.clip;
            if (A.coupled) gj = gj + A.wd * pr[j];
            m[j] = A.b1 * m[j] + A.a1 * gj;
            v[j] = A.b2 * (v[j] * v[j]) + A.a2 * (gj * gj);
            least = fminf(least, v[j]);
            most = fmaxf(most, v[j]);
            if (!(v[j] == v[j])) most = 3e38f;
        }
        if (least >= 0x1p-96f && most <= 0x1p96f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                root[j] = root_of(v[j]);
                np[j] = pr[j] * S.keep - S.size * quotient(m[j], root[j] * S.root + A.eps);
            }
        } else {   // zeros (no gradient ever), far values
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                root[j] = sqrtf(v[j]);
                np[j] = pr[j] * S.keep - S.size * (m[j] / (root[j] * S.root + A.eps));
            }
        }
        if (from + OPT_BLOCK > n) {   // behind the tensor's end the state holds zeros
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j >= n) m[j] = root[j] = np[j] = 0.f;
        }
        if (MASTER) *(of32x8*)(A.masters + s) = np;
        store_v<8>(p, i, n, wide, np);
        // Largest magnitudes as integers (the same order as the floats'; inf and NaN are above all finite ones).  sqrt(v) has no sign but that
        // of a NaN.
        uint32_t am[8], ar[8], hm = 0, hs = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            am[j] = __float_as_uint(m[j]) & 0x7FFFFFFFu;
            ar[j] = __float_as_uint(root[j]) & 0x7FFFFFFFu;
            hm = max(hm, am[j]);
            hs = max(hs, ar[j]);
        }
        uint32_t tm = half_max(hm), ts = half_max(hs);
        const bool fine = max(tm, ts) < INF;   // (the same for the half wave)
        if (!fine) {
            hm = hs = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                hm = max(hm, am[j] < INF ? am[j] : 0u);
                hs = max(hs, ar[j] < INF ? ar[j] : 0u);
            }
            tm = half_max(hm);
            ts = half_max(hs);
        }
        const float km = fmaxf(__uint_as_float(tm) * (1.f / 448.f), 0x1p-126f), ks = fmaxf(__uint_as_float(ts) * (1.f / 448.f), 0x1p-126f);
        const int inv = (int)__float_as_uint(1.f / ((threadIdx.x & 1) ? ks : km));   // both divisions at once, in the odd and the even lanes
        const float im = __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, inv, 0xA0, 0xf, 0xf, false));   // quad_perm:[0,0,2,2]
        const float is = __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, inv, 0xF5, 0xf, 0xf, false));   // quad_perm:[1,1,3,3]
        const uint32_t at = (uint32_t)s + (uint32_t)((uint64_t)s >> 32) * 0x9E3779B1u + S.key;   // (8 | s: no carry in s + j)
        uint32_t cm[2] = {0, 0}, cs[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t h = mix32(at + j);
            uint32_t a = code_of(__uint_as_float(am[j]), im, h & 0xFFFFu), r = code_of(__uint_as_float(ar[j]), is, h >> 16);
            r = max(r, min(ar[j], 1u));
            if (!fine) {
                if (am[j] >= INF) a = 0x7Fu;
                if (ar[j] >= INF) r = 0x7Fu;
            }
            a |= (__float_as_uint(m[j]) >> 24) & 0x80u;
            cm[j / 4] |= a << (8 * (j % 4));
            cs[j / 4] |= r << (8 * (j % 4));
        }
        *(uint2*)((uint8_t*)A.m + s) = make_uint2(cm[0], cm[1]);
        *(uint2*)((uint8_t*)A.v + s) = make_uint2(cs[0], cs[1]);
        if (i == from) {
            A.scales[b] = km;
            A.scales[A.n_blocks + b] = ks;
        }
    }
}

size_t dtype_size(int dtype) { return dtype == INSMOS_F32 ? 4 : 2; }

// Calls fn(list, workgroups) for every launch that `tensors` need; INSMOS_EINVAL at a bad entry.
template <class List, class F>
int each_launch(const InsmosOptTensor* tensors, int n_tensors, int64_t chunk, bool params, int dtype, int64_t n_state, F fn) {
    List L;
    L.count = 0;
    uint32_t blocks = 0;
    auto flush = [&]() -> int {
        if (!L.count) return INSMOS_OK;
        L.first[L.count] = blocks;
        const int rc = fn(L, blocks);
        L.count = 0;
        blocks = 0;
        return rc;
    };
    const size_t size = dtype_size(dtype);
    for (int i = 0; i < n_tensors; ++i) {
        const InsmosOptTensor& t = tensors[i];
        if (t.numel < 0 || t.numel > (int64_t)1 << 40) return INSMOS_EINVAL;
        if (t.numel == 0) continue;
        if (!t.grad || (uintptr_t)t.grad % size) return INSMOS_EINVAL;
        if (params && (!t.param || (uintptr_t)t.param % size || t.state_off < 0 || t.state_off % OPT_BLOCK ||
                       t.state_off + (t.numel + OPT_BLOCK - 1) / OPT_BLOCK * OPT_BLOCK > n_state))
            return INSMOS_EINVAL;
        for (int64_t at = 0; at < t.numel; at += PART) {
            const int64_t n = t.numel - at < PART ? t.numel - at : PART;
            const uint32_t need = (uint32_t)((n + chunk - 1) / chunk);
            if (L.count == List::MOST || (uint64_t)blocks + need > 0x7FFFFFFFull / 256) {   // (2^31 threads are a launch's most)
                const int rc = flush();
                if (rc != INSMOS_OK) return rc;
            }
            L.set(L.count, (char*)t.param + at * size, (const char*)t.grad + at * size, n, t.state_off + at);
            L.first[L.count++] = blocks;
            blocks += need;
        }
    }
    return flush();
}

template <class T>
int launch_sumsq(const NormList& L, uint32_t blocks, double* partial, hipStream_t s) {
    ProfScope ps(KK_ADAMW, s);
    const auto kernel = k_grad_sumsq<T>;
    INSMOS_LAUNCH(kernel, dim3(blocks), dim3(256), 0, s, L, partial);
    HIP_TRY(hipGetLastError());
    return INSMOS_OK;
}
int sumsq(const InsmosOptTensor* tensors, int n, int dtype, double* partial, hipStream_t s, int64_t* used) {
    int64_t at = 0;
    const int rc = each_launch<NormList>(tensors, n, NORM_CHUNK, false, dtype, 0, [&](const NormList& L, uint32_t blocks) -> int {
        double* q = partial + at;
        at += blocks;
        return dtype == INSMOS_F32 ? launch_sumsq<float>(L, blocks, q, s)
               : dtype == INSMOS_BF16 ? launch_sumsq<__bf16>(L, blocks, q, s) : launch_sumsq<_Float16>(L, blocks, q, s);
    });
    *used = at;
    return rc;
}
template <class T, bool MASTER>
int launch_step(const StepList& L, uint32_t blocks, const StepP& P, int bits, hipStream_t s) {
    ProfScope ps(KK_ADAMW, s);
    const auto kernel = bits == 32 ? k_adamw<T, MASTER> : k_adamw8<T, MASTER>;
    INSMOS_LAUNCH(kernel, dim3(blocks), dim3(256), 0, s, L, P);
    HIP_TRY(hipGetLastError());
    return INSMOS_OK;
}
template <class T>
int launch_step_t(const StepList& L, uint32_t blocks, const StepP& P, int bits, hipStream_t s) {
    return P.masters ? launch_step<T, true>(L, blocks, P, bits, s) : launch_step<T, false>(L, blocks, P, bits, s);
}
bool good_list(const InsmosOptTensor* t, int n, int dtype) {
    return (t || !n) && n >= 0 && (dtype == INSMOS_F32 || dtype == INSMOS_BF16 || dtype == INSMOS_F16);
}
}  // namespace
}  // namespace insmos

using namespace insmos;

extern "C" size_t insmos_grad_sumsq_partials(const InsmosOptTensor* tensors_host, int n_tensors) {
    if (!good_list(tensors_host, n_tensors, INSMOS_F32)) return 0;
    size_t total = 0;
    for (int i = 0; i < n_tensors; ++i)   // (a size that is out of range is refused by the calls that take the list)
        if (tensors_host[i].numel > 0 && tensors_host[i].numel <= (int64_t)1 << 40)
            total += (size_t)((tensors_host[i].numel + NORM_CHUNK - 1) / NORM_CHUNK);   // (a PART is whole chunks)
    return total;
}
extern "C" int insmos_grad_sumsq(const InsmosOptTensor* tensors_host, int n_tensors, int dtype, double* partials, int64_t n_partials,
                                 void* stream) {
    const size_t need = insmos_grad_sumsq_partials(tensors_host, n_tensors);
    if (!good_list(tensors_host, n_tensors, dtype) || (need && !partials) || n_partials < 0) return INSMOS_EINVAL;
    const int bad = each_launch<NormList>(tensors_host, n_tensors, NORM_CHUNK, false, dtype, 0, [](const NormList&, uint32_t) { return INSMOS_OK; });
    if (bad != INSMOS_OK) return bad;
    if ((size_t)n_partials < need) return INSMOS_EWORKSPACE;
    int64_t used = 0;
    return sumsq(tensors_host, n_tensors, dtype, partials, (hipStream_t)stream, &used);
}
extern "C" int insmos_grad_norm(const double* partials, int64_t n_partials, float* norm, void* stream) {
    if (n_partials < 0 || (n_partials && !partials) || !norm) return INSMOS_EINVAL;
    ProfScope ps(KK_ADAMW, (hipStream_t)stream);
    INSMOS_LAUNCH(k_grad_norm, dim3(1), dim3(1024), 0, (hipStream_t)stream, partials, n_partials, norm);
    HIP_TRY(hipGetLastError());
    return INSMOS_OK;
}
extern "C" size_t insmos_adamw_ws_bytes(const InsmosOptTensor* tensors_host, int n_tensors) {
    return pad256(sizeof(StepVals)) + pad256(insmos_grad_sumsq_partials(tensors_host, n_tensors) * sizeof(double));
}
extern "C" int insmos_adamw_step(const InsmosOptTensor* tensors_host, int n_tensors, int dtype, int state_bits, void* exp_avg,
                                 void* exp_avg_sq, float* scales, int64_t n_state, float* masters, int32_t* step, double lr,
                                 const float* lr_dev, double beta1, double beta2, double eps, double weight_decay, int decoupled,
                                 double max_norm, const float* norm_in, int skip_nonfinite, unsigned seed, float* norm_out, void* ws,
                                 size_t ws_bytes, void* stream) {
    if (!good_list(tensors_host, n_tensors, dtype) || (state_bits != 32 && state_bits != 8) || !step || n_state < 0 ||
        n_state % OPT_BLOCK || n_state > (int64_t)1 << 40 || (n_state && (!exp_avg || !exp_avg_sq)) || (state_bits == 8 && n_state && !scales) ||
        (masters && dtype == INSMOS_F32) || !ws)
        return INSMOS_EINVAL;
    if ((uintptr_t)exp_avg % 16 || (uintptr_t)exp_avg_sq % 16 || (uintptr_t)masters % 16 || (uintptr_t)ws % 16) return INSMOS_EINVAL;
    if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !(weight_decay >= 0.0) || max_norm != max_norm)
        return INSMOS_EINVAL;
    // every entry is looked at before the first launch: a refused call has changed nothing
    const int bad = each_launch<StepList>(tensors_host, n_tensors, STEP_CHUNK, true, dtype, n_state, [](const StepList&, uint32_t) { return INSMOS_OK; });
    if (bad != INSMOS_OK) return bad;
    if (ws_bytes < insmos_adamw_ws_bytes(tensors_host, n_tensors)) return INSMOS_EWORKSPACE;
    const hipStream_t s = (hipStream_t)stream;
    StepVals* vals = (StepVals*)ws;
    double* partial = (double*)((char*)ws + pad256(sizeof(StepVals)));
    const bool clip = max_norm > 0.0, norm = !norm_in && (clip || skip_nonfinite || norm_out);
    PrepareP Q = {};
    if (norm) {
        const int rc = sumsq(tensors_host, n_tensors, dtype, partial, s, &Q.n_partial);
        if (rc != INSMOS_OK) return rc;
        Q.partial = partial;
    }
    Q.norm_in = norm_in;
    Q.norm_out = norm_out;
    Q.lr_dev = lr_dev;
    Q.lr = lr; Q.b1 = beta1; Q.b2 = beta2; Q.wd = weight_decay; Q.max_norm = max_norm;
    Q.decoupled = decoupled != 0; Q.clip = clip; Q.skip_nonfinite = skip_nonfinite != 0;
    Q.seed = seed;
    Q.step = step;
    Q.vals = vals;
    {
        ProfScope ps(KK_ADAMW, s);
        INSMOS_LAUNCH(k_adamw_prepare, dim3(1), dim3(1024), 0, s, Q);
        HIP_TRY(hipGetLastError());
    }
    StepP P = {};
    P.vals = vals;
    P.m = exp_avg; P.v = exp_avg_sq; P.scales = scales; P.n_blocks = n_state / OPT_BLOCK;
    P.masters = masters;
    P.b1 = (float)beta1; P.a1 = (float)(1.0 - beta1);
    P.b2 = (float)beta2; P.a2 = (float)(1.0 - beta2);
    P.eps = (float)eps;
    P.wd = (float)weight_decay;
    P.coupled = !decoupled && weight_decay != 0.0;
    return each_launch<StepList>(tensors_host, n_tensors, STEP_CHUNK, true, dtype, n_state, [&](const StepList& L, uint32_t blocks) -> int {
        if (dtype == INSMOS_F32) return launch_step<float, false>(L, blocks, P, state_bits, s);
        return dtype == INSMOS_BF16 ? launch_step_t<__bf16>(L, blocks, P, state_bits, s) : launch_step_t<_Float16>(L, blocks, P, state_bits, s);
    });
}

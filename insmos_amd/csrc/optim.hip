// insmos_amd/csrc/optim.hip -- one AdamW / Adam step over a list of tensors, moments in 32 or in 8 bits, with the clip by the
// gradients' global norm (the optimiser of models/models.py:185-190 as one short chain of launches instead of a chain per tensor).
//
//   g' = c g (+ wd p when the decay is coupled),  c = min(1, max_norm / (|g| + 1e-6)) or 1
//   m  = b1 m + (1 - b1) g'        v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd or 1) - lr / (1 - b1^t) * (m / (sqrt(v) / sqrt(1 - b2^t) + eps))
//
// Bound: HBM.  An element moves 28 bytes with fp32 tensors and moments (p, m, v read and written, g read; + 4 when the norm is
// taken), 16 with moments in 8 bits; the arithmetic is some 20 (32 bits) or 80 (8 bits) vector instructions per element.
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
constexpr int NORM_CHUNK = 8192;    // ... of the norm (one 8-byte partial sum each)
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
typedef __bf16 obf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 of16x4 __attribute__((ext_vector_type(4)));
template <class T> struct Vec4;
template <> struct Vec4<float> { typedef of32x4 t; };
template <> struct Vec4<__bf16> { typedef obf16x4 t; };
template <> struct Vec4<_Float16> { typedef of16x4 t; };

__device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x ^= x >> 16; x *= 0x7FEB352Du;
    x ^= x >> 15; x *= 0x846CA68Bu;
    return x ^ (x >> 16);
}
// the tensor a workgroup works on (the argument arrays are read through scalar loads: the index is the same for all lanes)
template <class List>
__device__ __forceinline__ int tensor_of(const List& L, uint32_t b) {
    int lo = 0, hi = L.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (L.first[mid] <= b) lo = mid; else hi = mid;
    }
    return lo;
}
// four elements of a tensor from element i on; zeros past its end; `wide` = the tensor's address allows one access
template <class T>
__device__ __forceinline__ of32x4 load4(const T* __restrict__ p, uint32_t i, uint32_t n, bool wide) {
    if (wide && i + 4 <= n) return __builtin_convertvector(*(const typename Vec4<T>::t*)(p + i), of32x4);
    of32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (i + j < n) r[j] = (float)p[i + j];
    return r;
}
template <class T>
__device__ __forceinline__ void store4(T* __restrict__ p, uint32_t i, uint32_t n, bool wide, of32x4 v) {
    if (wide && i + 4 <= n) { *(typename Vec4<T>::t*)(p + i) = __builtin_convertvector(v, typename Vec4<T>::t); return; }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (i + j < n) p[i + j] = (T)v[j];
}
template <class T>
__device__ __forceinline__ bool is_wide(const void* a) { return ((uintptr_t)a & (4 * sizeof(T) - 1)) == 0; }

// ---- the gradients' sum of squares: one fp64 partial per workgroup (fixed order: the same bits every time) ------------------
// Four squares are added in fp32 (their rounding errors have no direction and average out) and the sums in fp64: a quarter of the
// fp64 work.  Sums near fp32's limits are taken in fp64.
__device__ __forceinline__ void add_squares(double& s, const of32x4 v) {
    const float q = fmaf(v[0], v[0], v[1] * v[1]) + fmaf(v[2], v[2], v[3] * v[3]);
    if (q >= 1e-30f && q <= 1e37f) s += (double)q;
    else
#pragma unroll
        for (int j = 0; j < 4; ++j) s = fma((double)v[j], (double)v[j], s);
}
template <class T>
__global__ void __launch_bounds__(256) k_grad_sumsq(const NormList L, double* __restrict__ partial) {
    const int t = tensor_of(L, blockIdx.x);
    const T* g = (const T*)L.g[t];
    const uint32_t n = L.n[t], base = (blockIdx.x - L.first[t]) * NORM_CHUNK;
    const bool wide = is_wide<T>(g);
    double s = 0.0;
    if (wide && base + NORM_CHUNK <= n) {   // a whole chunk: all loads in flight
        of32x4 v[NORM_CHUNK / 1024];
#pragma unroll
        for (int u = 0; u < NORM_CHUNK / 1024; ++u)
            v[u] = __builtin_convertvector(*(const typename Vec4<T>::t*)(g + base + u * 1024 + threadIdx.x * 4), of32x4);
#pragma unroll
        for (int u = 0; u < NORM_CHUNK / 1024; ++u) add_squares(s, v[u]);
    } else {
        for (int u = 0; u < NORM_CHUNK / 1024; ++u) {
            const uint32_t i = base + u * 1024 + threadIdx.x * 4;
            if (i < n) add_squares(s, load4(g, i, n, wide));
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
    if (threadIdx.x) return;
    if (A.norm_in) norm = (double)*A.norm_in;
    if (A.norm_out) *A.norm_out = (float)norm;
    StepVals v;
    v.skip = A.skip_nonfinite && !(norm <= 1.7976931348623157e308);
    const int t = *A.step + (v.skip ? 0 : 1);
    *A.step = t;
    const double lr = A.lr_dev ? (double)*A.lr_dev : A.lr;
    v.clip = 1.f;
    if (A.clip) {
        const float c = (float)(A.max_norm / (norm + 1e-6));
        v.clip = c >= 1.f ? 1.f : c;   // (a norm that is NaN stays one)
    }
    v.keep = A.decoupled ? (float)(1.0 - lr * A.wd) : 1.f;
    v.size = (float)(lr / (1.0 - pow(A.b1, (double)t)));
    v.root = (float)(1.0 / sqrt(1.0 - pow(A.b2, (double)t)));
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
// the largest of the wave's 64 values in a scalar register (row shifts, then the rows' last lanes handed on)
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false));   // row_shr:1, 2, 4, 8
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false));   // row_bcast:15, 31
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false));
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ of32x4 decode4(uint32_t c, float scale) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    of32x4 r = {lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale};
    return r;
}

template <class T, int BITS, bool MASTER>
__global__ void __launch_bounds__(256) k_adamw(const StepList L, const StepP A) {
    const StepVals S = *A.vals;
    if (S.skip) return;
    const int t = tensor_of(L, blockIdx.x);
    T* p = (T*)L.p[t];
    const T* g = (const T*)L.g[t];
    const uint32_t n = L.n[t], base = (blockIdx.x - L.first[t]) * STEP_CHUNK;
    const uint32_t lane4 = (threadIdx.x & 63) * 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool wide = is_wide<T>(p) && is_wide<T>(g);
#pragma unroll
    for (int u = 0; u < STEP_CHUNK / 1024; ++u) {
        const uint32_t from = base + u * 1024 + wave * 256, i = from + lane4;   // a wave's 256 elements are one block of the state
        if (from >= n) break;
        const int64_t b = (int64_t)L.off[t] + from / OPT_BLOCK, s = b * OPT_BLOCK + lane4;
        of32x4 gr = load4(g, i, n, wide);
        of32x4 pr = MASTER ? *(const of32x4*)(A.masters + s) : load4((const T*)p, i, n, wide);
        of32x4 m, v;
        if (BITS == 32) {
            m = *(const of32x4*)((const float*)A.m + s);
            v = *(const of32x4*)((const float*)A.v + s);
        } else {
            m = decode4(*(const uint32_t*)((const uint8_t*)A.m + s), A.scales[b]);
            v = decode4(*(const uint32_t*)((const uint8_t*)A.v + s), A.scales[A.n_blocks + b]);
            v = v * v;
        }
        of32x4 root, np;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float gj = gr[j] * S.clip;
            if (A.coupled) gj = gj + A.wd * pr[j];
            m[j] = A.b1 * m[j] + A.a1 * gj;
            v[j] = A.b2 * v[j] + A.a2 * (gj * gj);
            root[j] = sqrtf(v[j]);
            np[j] = pr[j] * S.keep - S.size * (m[j] / (root[j] * S.root + A.eps));
        }
        if (from + OPT_BLOCK > n) {   // behind the tensor's end the state holds zeros
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j >= n) m[j] = v[j] = root[j] = np[j] = 0.f;
        }
        if (MASTER) *(of32x4*)(A.masters + s) = np;
        store4(p, i, n, wide, np);
        if (BITS == 32) {
            *(of32x4*)((float*)A.m + s) = m;
            *(of32x4*)((float*)A.v + s) = v;
        } else {
            // Largest magnitudes as integers (the same order as the floats'; inf and NaN are above all finite ones).  sqrt(v) has no
            // sign but that of a NaN.
            uint32_t am[4], ar[4], hm = 0, hs = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                am[j] = __float_as_uint(m[j]) & 0x7FFFFFFFu;
                ar[j] = __float_as_uint(root[j]) & 0x7FFFFFFFu;
                hm = max(hm, am[j]);
                hs = max(hs, ar[j]);
            }
            uint32_t tm = wave_max(hm), ts = wave_max(hs);
            const bool fine = max(tm, ts) < 0x7F800000u;   // (the same for the wave)
            if (!fine) {
                hm = hs = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    hm = max(hm, am[j] < 0x7F800000u ? am[j] : 0u);
                    hs = max(hs, ar[j] < 0x7F800000u ? ar[j] : 0u);
                }
                tm = wave_max(hm);
                ts = wave_max(hs);
            }
            const float km = fmaxf(__uint_as_float(tm) * (1.f / 448.f), 0x1p-126f), ks = fmaxf(__uint_as_float(ts) * (1.f / 448.f), 0x1p-126f);
            const float inv = 1.f / ((threadIdx.x & 1) ? ks : km);   // both divisions at once, in the odd and the even lanes
            const float im = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(inv), 0));
            const float is = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(inv), 1));
            const uint32_t at = (uint32_t)s + (uint32_t)((uint64_t)s >> 32) * 0x9E3779B1u + S.key;   // (256 | s: no carry in s + j)
            uint32_t cm = 0, cs = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t h = mix32(at + j);
                uint32_t a = code_of(__uint_as_float(am[j]), im, h & 0xFFFFu), r = code_of(__uint_as_float(ar[j]), is, h >> 16);
                r = max(r, min(ar[j], 1u));
                if (!fine) {
                    if (am[j] >= 0x7F800000u) a = 0x7Fu;
                    if (ar[j] >= 0x7F800000u) r = 0x7Fu;
                }
                a |= (__float_as_uint(m[j]) >> 24) & 0x80u;
                cm |= a << (8 * j);
                cs |= r << (8 * j);
            }
            *(uint32_t*)((uint8_t*)A.m + s) = cm;
            *(uint32_t*)((uint8_t*)A.v + s) = cs;
            if (lane4 == 0) {
                A.scales[b] = km;
                A.scales[A.n_blocks + b] = ks;
            }
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
template <class T, int BITS, bool MASTER>
int launch_step(const StepList& L, uint32_t blocks, const StepP& P, hipStream_t s) {
    const auto kernel = k_adamw<T, BITS, MASTER>;
    INSMOS_LAUNCH(kernel, dim3(blocks), dim3(256), 0, s, L, P);
    HIP_TRY(hipGetLastError());
    return INSMOS_OK;
}
template <class T>
int launch_step_t(const StepList& L, uint32_t blocks, const StepP& P, int bits, hipStream_t s) {
    if (P.masters) return bits == 32 ? launch_step<T, 32, true>(L, blocks, P, s) : launch_step<T, 8, true>(L, blocks, P, s);
    return bits == 32 ? launch_step<T, 32, false>(L, blocks, P, s) : launch_step<T, 8, false>(L, blocks, P, s);
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
    INSMOS_LAUNCH(k_adamw_prepare, dim3(1), dim3(1024), 0, s, Q);
    HIP_TRY(hipGetLastError());
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
        if (dtype == INSMOS_F32)
            return state_bits == 32 ? launch_step<float, 32, false>(L, blocks, P, s) : launch_step<float, 8, false>(L, blocks, P, s);
        return dtype == INSMOS_BF16 ? launch_step_t<__bf16>(L, blocks, P, state_bits, s) : launch_step_t<_Float16>(L, blocks, P, state_bits, s);
    });
}

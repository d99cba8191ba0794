// insmos_amd/csrc/linear.h -- the tiled matrix product behind insmos_linear / insmos_linear_backward (linear_bf16.hip, linear_f16.hip,
// linear_f32.hip: its instances; linear.hip: entry points and the element-wise parts).
//
//   C[m][n] = epilogue( sum_k A[m][k] B[k][n] )
//
// Both operands may have their contraction index contiguous (KC) or the other one (NC): x W is (KC, NC) for W (cin, cout) and (KC, KC) for
// a transposed (cout, cin) weight, dz W^T the other way round, x^T dz is (NC, NC).  Nothing is transposed in memory.
//
// A tile row of either operand is 128 bytes of LDS (64 16-bit or 32 fp32 values of k for KC, or BK rows of R values for NC); a wave
// instruction moves 64 x 16 bytes from memory straight to LDS (buffer_load ... lds; addresses on 4 bytes), with the buffer's extent as the
// bounds check: rows behind the matrix read as zero, and so does k behind its end (cut() clears a chunk that K ends in).  Two tiles in LDS: one is filled while the other is read.
// The LDS image is written in lane order, so the bank swizzle is in the ADDRESSES READ: 16-byte chunk c of KC row r lies at c ^ (r & 7)
// (the 8 lanes of a read phase then touch 8 different chunks), chunk c of NC row k at c ^ 4 (k & 3 | k >> 1 & 4) (the 8 rows of a
// transposing read touch 8 different 64-byte pieces).  NC operands reach the matrix instructions through ds_read_b64_tr_b16.
//
// v_mfma_f32_32x32x16 (16 bit) / 32x32x2 (fp32) with B as the first operand: a lane then holds 4 consecutive n of one row m, so the
// epilogue loads and stores vectors.  Accumulation is fp32 throughout.
#pragma once
#include "common.h"

namespace insmos {
namespace lin {

#define LIN_LDS __attribute__((address_space(3)))
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
// eight values in memory at the alignment of one (the hardware takes 16-byte accesses at any address)
template <class T> struct Mem8;
template <> struct Mem8<float> { typedef float t __attribute__((ext_vector_type(8), aligned(4))); };
template <> struct Mem8<__bf16> { typedef __bf16 t __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Mem8<_Float16> { typedef _Float16 t __attribute__((ext_vector_type(8), aligned(2))); };

enum { KC = 0, NC = 1 };                                            // which index of an operand is contiguous
enum { T256 = 0, T128, T128X64, T64X128, T128X32, T32X128, FEW };   // tiles (rows x columns); k_linear_few

struct GemmP {
    const void* a;
    const void* b;
    int64_t lda, ldb;
    int M, N, K;
    int splits;           // k is cut into this many parts
    float* part;          // splits > 1: [split][M][ld_part] raw sums
    int64_t ld_part;
    // epilogue (splits == 1; otherwise the join kernel's)
    const void* bias;     // [N] or null
    const void* res;      // [M][ld_res] or null
    int64_t ld_res;
    void* y;
    int64_t ld_y;
    void* slope;          // act'(z) for the backward pass (see Slope), or null
    int64_t ld_slope;     // a multiple of 16 bytes
    int act, res_first;
};

// ---- activations ------------------------------------------------------------------------------------------------------------
// (v_exp and v_rcp: 1 ulp each; exp(-x) = inf gives 0)
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kGelu0 = 0.7978845608028654f, kGelu1 = 0.044715f;   // sqrt(2 / pi) (z + 0.044715 z^3)
// Phi(-|z|) of the normal distribution, and e = exp(-z^2 / 2): a polynomial in t = 1 / (1 + 0.3 |z|) times e, fitted to the least largest relative
// error (1.5e-7 for |z| <= 14, where the value leaves fp32's range).  To that the rounding of e's argument adds up to 5.6e-8 z^2 (1.4e-6 at 5, 1.1e-5 at
// 14), so the tail keeps its size, which 1 + erf(z / sqrt 2) loses, in less than half of erff's instructions.
__device__ __forceinline__ float normal_tail(float z, float& e) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, fabsf(z), 1.f));
    float p = fmaf(0.0356761676f, t, -0.157209128f);
    p = fmaf(p, t, 0.206364304f);
    p = fmaf(p, t, -0.0536939024f);
    p = fmaf(p, t, 0.128567206f);
    p = fmaf(p, t, 0.0999117609f);
    p = fmaf(p, t, 0.120754239f);
    p = fmaf(p, t, 0.11962928f);
    e = __builtin_amdgcn_exp2f((-0.5f * kLog2E) * z * z);
    return p * t * e;
}
// act(z) in place, and act'(z), act != INSMOS_ACT_NONE: z times a weight between 0 and 1; silu's and the tanh form's are sigmoids: (1 + tanh u) / 2
// = sigmoid(2 u).  The choice stands outside the loops: eight values' chains then run side by side (inside, 33953 x 210 x 142 bf16 with gelu took
// 34 us, and 18 without an activation).
__device__ __forceinline__ void activate8(f32x8& v, int act, f32x8& slope) {
    if (act == INSMOS_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float z = v[i];
            slope[i] = z > 0.f ? 1.f : (z != z ? z : 0.f);
            v[i] = z > 0.f ? z : (z != z ? z : 0.f);
        }
    } else if (act == INSMOS_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float z = v[i];
            float e;
            const float tail = normal_tail(z, e), phi = z > 0.f ? 1.f - tail : tail;
            slope[i] = fmaf(z * 0.3989422804014327f, e, phi);
            v[i] = z * phi;
        }
    } else if (act == INSMOS_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float z = v[i], s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2E * z)), y = z * s;
            slope[i] = fmaf(-y, s, y) + s;
            v[i] = y;
        }
    } else {
        constexpr float c0 = 2.f * kGelu0, c1 = 2.f * kGelu0 * kGelu1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float z = v[i], z2 = fminf(z * z, 3e38f);   // (its slope has 0 times the square far out)
            const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * fmaf(-kLog2E * c1, z2, -kLog2E * c0))), y = z * s;
            slope[i] = fmaf(fmaf(-y, s, y), fmaf(3.f * c1, z2, c0), s);
            v[i] = y;
        }
    }
}
// What the backward pass is given of act'(z): the value itself in fp32; with 16-bit types a code of 16 bits (all slopes lie in -0.13 .. 1.13):
//   |s| >= 2^-6   16384 + 2^15 s, rounded: codes 12 100 .. 15 872 and 16 896 .. 53 500
//   |s| <  2^-6   9 bits of mantissa and 23 exponents (the last one's numbers without a leading 1): m = 0 .. 11776, as m + 1 where s < 0 and as
//                 65 534 - m where it is not
//   0             not a number
// So a slope is off by at most 2^-16, and by 2^-10 of itself from 2^-6 down to 2^-28: of silu's and gelu's tails, where the slopes of all of a unit's
// rows may lie, the gradient keeps its size (silu to z = -22, gelu to -6.5), for 791 -> 802 us of the training step 8192 x 2048 x 8192 bf16.  Rounded to bf16 a
// slope would cost what the rounding of dz costs; z rounded to the type ten times the error near 1 (fp16), and the backward would compute the slope again.
//   The first form takes two instructions: clamped to 0 .. 1 (which makes a NaN 0) and added to 2^23, a value is rounded to a whole number that lies
// in the sum's lowest bits.  For the second |s| is moved so that its exponents end where fp32's do: 9 bits are then cut from its bits.
template <class T> struct Slope {
    typedef uint16_t t;
    static constexpr float kNear = 0x1p-6f, kMove = 0x1p-98f;   // 2^-28 -> fp32's smallest normal number
    static __device__ __forceinline__ uint16_t store(float s) {
        const uint32_t wide = __float_as_uint(fmaf(fminf(fmaxf(fmaf(s, 0.5f, 0.25f), 0.f), 1.f), 0x1p16f, 0x1p23f));
        const uint32_t m1 = (__float_as_uint(fabsf(s) * kMove) + 0x6000u) >> 14;   // m + 1
        const uint32_t fine = m1 ^ ~(uint32_t)((int32_t)__float_as_uint(s) >> 31);
        return (uint16_t)(fabsf(s) < kNear ? fine : wide);
    }
    static __device__ __forceinline__ float load(uint16_t c) {
        const bool below = c < 12000, above = c > 53600;
        const uint32_t m = below ? c - 1u : 65534u - c;
        const float fine = __uint_as_float(m << 14) * (below ? -0x1p98f : 0x1p98f);
        return c == 0 ? __builtin_nanf("") : below || above ? fine : (float)c * 0x1p-15f - 0.5f;
    }
};
template <> struct Slope<float> {
    typedef float t;
    static __device__ __forceinline__ float store(float s) { return s; }
    static __device__ __forceinline__ float load(float s) { return s; }
};
// eight values of a row from i on, of which `left` > 0 exist (behind them: the last one again); and the first `left` of eight stored
template <class T>
__device__ __forceinline__ typename Mem8<T>::t load8(const void* q, int64_t i, int left) {
    typedef typename Mem8<T>::t M8;
    if (left >= 8) return *(const M8*)((const T*)q + i);
    M8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = ((const T*)q)[i + min(e, left - 1)];
    return v;
}
template <class V>
__device__ __forceinline__ f32x8 wide(V v) { return __builtin_convertvector(v, f32x8); }
// Values n..n+7 (n < N) of row m from the fp32 sums; b and r: bias and residual (zeros where there is none).  Columns behind N are computed with
// the rest and not stored: only loads and stores differ at the edge (a second, one by one epilogue there held up 4099 x 1000 x 1533 fp16 by 16
// of 53 us, as the last tile column was on its own with it).
template <class T>
__device__ __forceinline__ void epilogue8(const GemmP& p, int m, int n, f32x8 v, f32x8 b, f32x8 r) {
    typedef typename Mem8<T>::t M8;
    const int left = p.N - n;
    v += b;
    if (p.res_first) v += r;
    f32x8 s;
    if (p.slope) {   // (with an activation only)
        typedef typename Slope<T>::t S;
        typedef S S8 __attribute__((ext_vector_type(8), aligned(16)));
        S8 c;
        activate8(v, p.act, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = Slope<T>::store(s[e]);
        S* q = (S*)p.slope + m * p.ld_slope + n;
        if (n + 8 <= p.ld_slope) {   // (the row's rest up to 16 bytes may be written)
            *(S8*)q = c;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) q[e] = c[e];
        }
    } else if (p.act) {
        activate8(v, p.act, s);
    }
    if (!p.res_first) v += r;
    const M8 o = __builtin_convertvector(v, M8);
    T* y = (T*)p.y + m * p.ld_y + n;
    if (left >= 8) {
        *(M8*)y = o;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) y[e] = o[e];
    }
}
template <class T>
__device__ __forceinline__ void epilogue(const GemmP& p, int m, int n, f32x8 v) {
    const f32x8 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    epilogue8<T>(p, m, n, v, p.bias ? wide(load8<T>(p.bias, n, p.N - n)) : zero, p.res ? wide(load8<T>(p.res, m * p.ld_res + n, p.N - n)) : zero);
}

// ---- operands ---------------------------------------------------------------------------------------------------------------
// One operand's tile: R rows (m or n) x BK, filled by NW waves.
template <class T, int LAY, int R, int NW>
struct Tile {
    static constexpr int ES = sizeof(T), BK = 128 / ES, CE = 16 / ES;   // CE: values per 16-byte chunk
    static constexpr int NI = R * 128 / (NW * 1024);                    // wave instructions per tile
    static constexpr int CPR = R * ES / 16, RPI = 64 / CPR;             // NC: chunks per row, rows per instruction
    const char* p;         // the current k tile
    int64_t left, step;    // bytes from p to the operand's end; per k tile
    uint32_t voff, istep;  // this lane's offset; per instruction
    int chunk;             // KC: k of this lane's chunk

    static __device__ __forceinline__ int swizzle(int k) { return ES == 2 ? ((((k & 3) | ((k >> 1) & 4)) << 2)) & (CPR - 1) : 0; }
    __device__ __forceinline__ void init(const void* base, int64_t ld, int r0, int rtot, int K, int kt0, int wave, int lane) {
        // (the bounds check goes by dwords: the one that holds the operand's last value counts as inside)
        if (LAY == KC) {
            p = (const char*)base + (int64_t)r0 * ld * ES;
            left = (((int64_t)(min(R, rtot - r0) - 1) * ld + K) * ES + 3) & ~(int64_t)3;
            step = 128;
            chunk = ((lane & 7) ^ (lane >> 3)) * CE;
            voff = (uint32_t)((wave * 8 + (lane >> 3)) * ld * ES) + chunk * ES;
            istep = (uint32_t)(NW * 8 * ld * ES);
        } else {
            static_assert(NI == 1 || ES == 4 || NW * RPI % 16 == 0, "one swizzle for a lane's instructions");
            p = (const char*)base + (int64_t)r0 * ES;
            left = (((int64_t)(K - 1) * ld + (rtot - r0)) * ES + 3) & ~(int64_t)3;
            step = (int64_t)BK * ld * ES;
            const int k = wave * RPI + lane / CPR;
            chunk = 0;
            voff = (uint32_t)(k * ld * ES) + ((lane % CPR) ^ swizzle(k)) * 16;
            istep = (uint32_t)(NW * RPI * ld * ES);
        }
        p += kt0 * step;
        left -= kt0 * step;
    }
    // The loads of the current k tile: where from (k_left: K minus the tile's first k; without `on` nothing is read), and instruction i.
    struct Source { __amdgpu_buffer_rsrc_t rs; uint32_t v; };
    __device__ __forceinline__ Source source(int k_left, bool on = true) {
        const int bytes = on ? (int)max((int64_t)0, min(left, (int64_t)0x7FFFFFFF)) : 0;
        const Source r = {__builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00027000), LAY == KC && chunk >= k_left ? 0x80000000u : voff};
        p += step;
        left -= step;
        return r;
    }
    __device__ __forceinline__ void load1(const Source& f, LIN_LDS char* __restrict lds, int i, int wave) const {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(f.rs, (LIN_LDS void*)(lds + (i * NW + wave) * 1024), 16, f.v, i * istep, 0, 0);
    }
    __device__ __forceinline__ void load(LIN_LDS char* __restrict lds, int k_left, int wave) {   // all of them
        const Source f = source(k_left);
#pragma unroll
        for (int i = 0; i < NI; ++i) load1(f, lds, i, wave);
    }
    // KC: the chunk that K ends in has brought values from behind the row's end; zeros in their place (k: valid values of the tile)
    static __device__ __forceinline__ void cut(LIN_LDS char* lds, int k) {
        if (LAY != KC || k % CE == 0) return;
        for (int r = threadIdx.x; r < R; r += NW * 64) {
            LIN_LDS char* c = lds + r * 128 + (((k / CE) ^ (r & 7)) << 4);
            for (int e = k % CE; e < CE; ++e) {
                if (ES == 2) *(LIN_LDS short*)(c + e * 2) = 0;
                else *(LIN_LDS float*)(c + e * 4) = 0.f;
            }
        }
    }
};

// What a lane reads of a tile for step s: rows rb + 32 t + lane % 32; k = 16 s + 8 (lane / 32) + 0..7 (16 bit).
template <class T, int LAY, int R, int NT>
struct Frag {
    typedef s16x8 type;
    static constexpr int N = LAY == KC ? 4 : NT;   // addresses: KC one per s (t is a constant offset), NC one per t
    uint32_t off[N];
    __device__ __forceinline__ void init(int rb, int lane) {
        if (LAY == KC) {
#pragma unroll
            for (int s = 0; s < 4; ++s) off[s] = (rb + (lane & 31)) * 128 + (((2 * s + (lane >> 5)) ^ (lane & 7)) << 4);
        } else {
            // a transposing read: lane j of 16 addresses row j / 4, columns 4 (j % 4)..; it receives column j of those four rows
            const int g = lane >> 4, j = lane & 15, k = (g >> 1) * 8 + (j >> 2);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int col = rb + t * 32 + (g & 1) * 16 + 4 * (j & 3);
                off[t] = k * R * 2 + (((col >> 3) ^ Tile<T, NC, R, 1>::swizzle(k)) << 4) + (col & 7) * 2;
            }
        }
    }
    __device__ __forceinline__ s16x8 get(const LIN_LDS char* __restrict lds, int t, int s) const {
        if (LAY == KC) return *(const LIN_LDS s16x8*)(lds + off[s] + t * 4096);
        const LIN_LDS char* q = lds + off[t] + s * (R * 32);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LIN_LDS s16x4*)q);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LIN_LDS s16x4*)(q + R * 8));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};
// fp32: four steps of 32x32x2 take the k of 8 in the order 0 2 | 4 6 | 1 3 | 5 7 (the lower half of the lanes has the first of each pair), so that a
// KC fragment is two 8-byte reads.  (The kernel for few rows and products in parts add in other orders; a z within their rounding of a relu's
// border may be decided either way.)
template <int LAY, int R, int NT>
struct Frag<float, LAY, R, NT> {
    typedef f32x4 type;
    static constexpr int N = LAY == KC ? 8 : 1;
    uint32_t off[N];
    __device__ __forceinline__ void init(int rb, int lane) {
        const int h = lane >> 5;
        if (LAY == KC) {
#pragma unroll
            for (int c = 0; c < N; ++c) off[c] = (rb + (lane & 31)) * 128 + ((c ^ (lane & 7)) << 4) + 8 * h;
        } else {
            off[0] = (2 * h * R + rb + (lane & 31)) * 4;
        }
    }
    __device__ __forceinline__ f32x4 get(const LIN_LDS char* __restrict lds, int t, int s) const {
        f32x4 r;
        if (LAY == KC) {
            typedef float f32x2 __attribute__((ext_vector_type(2)));
            const f32x2 a = *(const LIN_LDS f32x2*)(lds + off[LAY == KC ? 2 * s : 0] + t * 4096);
            const f32x2 b = *(const LIN_LDS f32x2*)(lds + off[LAY == KC ? 2 * s + 1 : 0] + t * 4096);
            r[0] = a[0]; r[1] = b[0]; r[2] = a[1]; r[3] = b[1];
        } else {
            constexpr int K4[4] = {0, 4, 1, 5};
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = *(const LIN_LDS float*)(lds + off[0] + t * 128 + (8 * s + K4[e]) * R * 4);
        }
        return r;
    }
};
template <class T> __device__ __forceinline__ f32x16 mfma(typename Frag<T, KC, 32, 1>::type b, typename Frag<T, KC, 32, 1>::type a, f32x16 c);
template <> __device__ __forceinline__ f32x16 mfma<__bf16>(s16x8 b, s16x8 a, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mfma<_Float16>(s16x8 b, s16x8 a, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mfma<float>(f32x4 b, f32x4 a, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(b[e], a[e], c, 0, 0, 0);
    return c;
}

// ---- the kernel -------------------------------------------------------------------------------------------------------------
struct Item { int tm, tn, split, kt0, kt1; };   // a tile of C and a part of k

template <class T, int LA, int LB, int BM, int BN, int WM, int WN>
struct Gemm {
    static constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, SA = BM * 128, SB = BN * 128, BK = 128 / sizeof(T);
    typedef Tile<T, LA, BM, NW> TA;
    typedef Tile<T, LB, BN, NW> TB;
    typedef Frag<T, LA, BM, TM> FA;
    typedef Frag<T, LB, BN, TN> FB;
    // One k tile: the next one is on its way into wr while rd is read.  (wr and rd never overlap, and __restrict says so: otherwise every
    // LDS read would wait for the loads.)  Four phases; each reads the fragments of the following one between its matrix instructions.  The
    // first still multiplies the previous tile's last fragments, so that the matrix units have work right behind the barrier.
    struct Regs { typename FA::type a[2][TM]; typename FB::type b[2][TN]; };
    static __device__ __forceinline__ void phase(const LIN_LDS char* __restrict rd, const FA& fa, const FB& fb, Regs& r, f32x16 (&acc)[TM][TN], const int s) {
        const int to = s & 1, from = to ^ 1;
#pragma unroll
        for (int j = 0; j < TN; ++j) r.b[to][j] = fb.get(rd + SA, j, s);
#pragma unroll
        for (int i = 0; i < TM; ++i) r.a[to][i] = fa.get(rd, i, s);
        multiply(r, acc, from);
    }
    static __device__ __forceinline__ void multiply(const Regs& r, f32x16 (&acc)[TM][TN], const int from) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = mfma<T>(r.b[from][j], r.a[from][i], acc[i][j]);
    }
    static __device__ __forceinline__ void step(LIN_LDS char* __restrict wr, const LIN_LDS char* __restrict rd, TA& ta, TB& tb, const FA& fa,
                                                const FB& fb, Regs& r, f32x16 (&acc)[TM][TN], bool more, int k_left, int wave) {
        if constexpr (sizeof(T) == 2) {
            if (more) {
                ta.load(wr, k_left, wave);
                tb.load(wr + SA, k_left, wave);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                phase(rd, fa, fb, r, acc, s);
                // reads and matrix instructions in turn, and not the reads in a row in front (1096 -> 1255 TFLOP/s at 8192 x 8192 x 4096, bf16,
                // with the phases' overlap across the barrier)
#pragma unroll
                for (int q = 0; q < TM * TN; ++q) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);   // LDS reads
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // one matrix instruction
                }
            }
        } else {
            // The loads between the matrix instructions of PH phases (in front, a wave that waits for a place in the load queue holds its matrix
            // unit up: 4096 x 4096 x 4096 fp32 1010 -> 980 us; with 16 bits, whose steps are a quarter as long, it is the other way round).
            constexpr int PH = 2, LOADS = TA::NI + TB::NI, EACH = (LOADS + PH - 1) / PH, GAP = TM * TN * 4 / EACH;
            const typename TA::Source sa = ta.source(k_left, more);
            const typename TB::Source sb = tb.source(k_left, more);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
#pragma unroll
                for (int i = s * EACH; i < LOADS && i < (s + 1) * EACH; ++i) {
                    if (i < TA::NI) ta.load1(sa, wr, i, wave);
                    else tb.load1(sb, wr + SA, i - TA::NI, wave);
                }
                phase(rd, fa, fb, r, acc, s);
#pragma unroll
                for (int i = s * EACH; i < LOADS && i < (s + 1) * EACH; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);     // a load
                    __builtin_amdgcn_sched_group_barrier(0x008, GAP, 0);   // matrix instructions
                }
            }
        }
    }
    static __device__ __forceinline__ void fill(LIN_LDS char* __restrict l, const GemmP& p, const Item& it, TA& ta, TB& tb, int wave, int lane) {
        ta.init(p.a, p.lda, it.tm * BM, p.M, p.K, it.kt0, wave, lane);
        tb.init(p.b, p.ldb, it.tn * BN, p.N, p.K, it.kt0, wave, lane);
        ta.load(l, p.K - it.kt0 * BK, wave);
        tb.load(l + SA, p.K - it.kt0 * BK, wave);
    }
    // The epilogue of an item, with the next one's first tile on its way into `l`.  A wave turns its sums, 32 rows at a time, from a lane per row
    // to rows in a row through its part of `turn` (32 rows of TN x 32 floats, 16-byte chunk c of row r at c ^ r): what follows then moves whole
    // lines of C, and in a loop: unrolled over the sums' registers, the code alone cost some 10 us per launch and 4 us per tile.
    static __device__ __forceinline__ void finish(LIN_LDS char* __restrict l, LIN_LDS char* __restrict turn, const GemmP& p, const Item& it, bool more,
                                                  const Item& next, TA& ta, TB& tb, const f32x16 (&acc)[TM][TN], int wave, int lane) {
        static_assert(NW * TN * 4096 <= SA + SB, "`turn` is one tile buffer");
        if (more) fill(l, p, next, ta, tb, wave, lane);
        constexpr int CH = TN * 8, LPR = TN * 4, RPP = 64 / LPR, PASSES = 32 / RPP;   // chunks and lanes per row, rows per pass
        typedef typename Mem8<T>::t M8;
        LIN_LDS char* t = turn + wave * (32 * CH * 16);
        const int n = it.tn * BN + (wave % WN) * (BN / WN) + (lane % LPR) * 8;
        const bool in = n < p.N, plain = p.splits == 1;
        const f32x8 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const f32x8 bias = p.bias && in && plain ? wide(load8<T>(p.bias, n, p.N - n)) : zero;
        float* part = p.part + (int64_t)it.split * p.M * p.ld_part;   // (ld_part: whole groups of 8)
#pragma unroll 1
        for (int i = 0; i < TM; ++i) {
            const int m0 = it.tm * BM + (wave / WN) * (BM / WM) + i * 32 + lane / LPR;
            M8 res[PASSES];   // all of the block's residual is asked for before the first of it is needed
            if (p.res && in && plain) {
#pragma unroll
                for (int q = 0; q < PASSES; ++q) res[q] = load8<T>(p.res, min(m0 + q * RPP, p.M - 1) * p.ld_res + n, p.N - n);
            }
            const int r = lane & 31;
#pragma unroll
            for (int k = 0; k < TM; ++k) {   // (a loop over registers is one over branches)
                if (k != i) continue;
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 v = {acc[k][j][4 * g], acc[k][j][4 * g + 1], acc[k][j][4 * g + 2], acc[k][j][4 * g + 3]};
                        *(LIN_LDS f32x4*)(t + (r * CH + ((j * 8 + 2 * g + (lane >> 5)) ^ (r & (CH - 1)))) * 16) = v;
                    }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < PASSES; ++q) {
                const int row = q * RPP + lane / LPR, m = m0 + q * RPP, c = (lane % LPR) * 2;
                const f32x4 lo = *(const LIN_LDS f32x4*)(t + (row * CH + (c ^ (row & (CH - 1)))) * 16);
                const f32x4 hi = *(const LIN_LDS f32x4*)(t + (row * CH + ((c + 1) ^ (row & (CH - 1)))) * 16);
                const f32x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                if (m < p.M) {
                    if (!plain) {
                        if (n < p.ld_part) *(f32x8*)(part + m * p.ld_part + n) = v;
                    } else if (in) {
                        epilogue8<T>(p, m, n, v, bias, p.res ? wide(res[q]) : zero);
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
};

// Workgroup w runs on XCD w % 8 (each has an L2 of its own), so every XCD gets a contiguous run of items, walked in groups of 8 tile rows: the
// operands of the tiles in flight on one XCD stay in its L2 (groups of 4, 8 or 16: within 3 %).  Bound by the matrix units from a K of some hundreds
// on: 8192 x 4096 x 8192 bf16 with gelu_tanh and a residual 478 .. 494 us = 1113 .. 1150 TFLOP/s (the platform's plain product: 1186), 4096^3 fp32 982 us = 140 of
// 157; below that by the epilogue's lines and vector work (some 12 us per 256 x 256 tile, 8 for two of 128 x 128 side by side).
template <class T, int LA, int LB, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) k_linear_gemm(const GemmP p) {
    typedef Gemm<T, LA, LB, BM, BN, WM, WN> G;
    constexpr int TM = G::TM, TN = G::TN, SA = G::SA, SB = G::SB, BK = G::BK;
    __shared__ __attribute__((aligned(1024))) char lds[2 * (SA + SB)];
    LIN_LDS char* L = (LIN_LDS char*)(LIN_LDS void*)lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int gm = (p.M + BM - 1) / BM, gn = (p.N + BN - 1) / BN, tiles = gm * gn, items = tiles * p.splits;
    const int nk = (p.K + BK - 1) / BK, per_split = (nk + p.splits - 1) / p.splits;
    const int xcd = blockIdx.x & 7, per = items / 8, rest = items % 8;
    const int mine = per + (xcd < rest), base = xcd * per + min(xcd, rest), stride = (gridDim.x - xcd + 7) >> 3;
    auto locate = [&](int q) {   // item q of this XCD
        constexpr int GM = 8;
        const int id = base + q, t = id % tiles, first = t / (GM * gn) * GM, gs = min(GM, gm - first), in = t - first * gn;
        Item it;
        it.tm = first + in % gs;
        it.tn = in / gs;
        it.split = id / tiles;
        it.kt0 = it.split * per_split;
        it.kt1 = min(nk, it.kt0 + per_split);
        return it;
    };
    int q = blockIdx.x >> 3;
    if (q >= mine) return;   // (the same for the workgroup)
    typename G::FA fa;
    typename G::FB fb;
    fa.init(wave / WN * (BM / WM), lane);
    fb.init(wave % WN * (BN / WN), lane);
    typename G::TA ta;
    typename G::TB tb;
    Item it = locate(q);
    G::fill(L, p, it, ta, tb, wave, lane);
    while (true) {
        f32x16 acc[TM][TN];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
        typename G::Regs regs;   // (set 1 is multiplied before it is read for the first time: zeros)
#pragma unroll
        for (int i = 0; i < TM; ++i) regs.a[1][i] = typename G::FA::type{};
#pragma unroll
        for (int j = 0; j < TN; ++j) regs.b[1][j] = typename G::FB::type{};
        uint32_t cur = 0;
        __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): the first tile has arrived
        __syncthreads();
        for (int kt = it.kt0; kt < it.kt1; ++kt) {
            if ((LA == KC || LB == KC) && kt == nk - 1 && p.K % (16 / (int)sizeof(T))) {
                G::TA::cut(L + cur, p.K - kt * BK);
                G::TB::cut(L + cur + SA, p.K - kt * BK);
                __syncthreads();
            }
            G::step(L + (cur ^ (SA + SB)), L + cur, ta, tb, fa, fb, regs, acc, kt + 1 < it.kt1, p.K - (kt + 1) * BK, wave);
            cur ^= SA + SB;
            __builtin_amdgcn_s_waitcnt(0x0F70);   // the next tile has arrived, for every wave, and all are done with this one
            __syncthreads();
        }
        G::multiply(regs, acc, 1);
        q += stride;
        const bool more = q < mine;
        const Item next = more ? locate(q) : it;
        G::finish(L, L + SA + SB, p, it, more, next, ta, tb, acc, wave, lane);
        if (!more) return;
        it = next;
    }
}
// Sums the parts of k: eight columns of a row per lane, S lanes over the parts (each its own in their order, then the S sums in theirs).
template <class T, int S>
__global__ void __launch_bounds__(256) k_linear_join(const GemmP p) {
    constexpr int C = 256 / S;
    const int cols = (int)(p.ld_part / 8), part = threadIdx.x / C;
    const int64_t i = (int64_t)blockIdx.x * C + threadIdx.x % C;
    const bool in = i < (int64_t)p.M * cols;
    const int m = in ? (int)(i / cols) : 0, n = in ? (int)(i % cols) * 8 : 0;
    const float* q = p.part + (int64_t)m * p.ld_part + n;
    const int64_t per = (int64_t)p.M * p.ld_part;
    f32x8 s = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (in) {
#pragma unroll 4
        for (int k = part; k < p.splits; k += S) s += *(const f32x8*)(q + k * per);
    }
    if (S > 1) {
        __shared__ float w[S][C][9];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[part][threadIdx.x % C][e] = s[e];
        __syncthreads();
        if (part) return;
        for (int k = 1; k < S; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += w[k][threadIdx.x][e];
    }
    if (in) epilogue<T>(p, m, n, s);
}

// ---- few rows ---------------------------------------------------------------------------------------------------------------
// Up to 32 rows of x (tokens being generated): the weights' bytes are the time.  One launch, no workspace, any alignment: a workgroup has 32
// columns and all of k, its 8 waves take 128 bytes of k in turn and add up in LDS.  Fragments come straight from memory (KC) or, for weights
// with contiguous columns, through a turn of 16 x 32 values in the wave's own LDS; the whole of a wave's weights is in flight at once.
// Rows and columns behind the matrix repeat the last one and are not stored; k behind its end is zero in both operands.
// 1 x 2048 x 8192 bf16: 7.0 us (4.8 TB/s of weights) against 6.0 + 4.2 with the flat tiles and a join.
// eight values from k on, zeros behind K, one by one
template <class T>
__device__ __forceinline__ s16x8 load_k8(const T* row, int k, int K) {
    s16x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) {   // (K > 0; no branch around the loads)
        const short v = ((const short*)row)[min(k + e, K - 1)];
        r[e] = k + e < K ? v : (short)0;
    }
    return r;
}
template <class T, int LB>
struct Few {   // 16 bit: a chunk is 64 k, four steps of 16
    static constexpr int CHUNK = 64, TURN = 4 * 1024;
    typedef s16x8 type;
    // (whole chunks without a branch: their loads all leave before the first is waited for)
    static __device__ __forceinline__ void load_x(const T* row, int k0, int K, int lane, s16x8 (&f)[4]) {
        typedef short M8 __attribute__((ext_vector_type(8), aligned(2)));
        if (k0 + CHUNK <= K) {
#pragma unroll
            for (int s = 0; s < 4; ++s) f[s] = *(const M8*)((const short*)row + k0 + 16 * s + 8 * (lane >> 5));
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) f[s] = load_k8(row, k0 + 16 * s + 8 * (lane >> 5), K);
        }
    }
    static __device__ __forceinline__ void load_w(const T* w, int64_t ld, int n0, int N, int k0, int K, int lane, s16x8 (&f)[4]) {
        if (LB == KC) {
            load_x(w + (int64_t)min(n0 + (lane & 31), N - 1) * ld, k0, K, lane, f);
        } else {
            typedef short M8 __attribute__((ext_vector_type(8), aligned(2)));
            const int n = n0 + (lane & 3) * 8;
            if (k0 + CHUNK <= K && n0 + 32 <= N) {
#pragma unroll
                for (int s = 0; s < 4; ++s) f[s] = *(const M8*)((const short*)w + (k0 + 16 * s + (lane >> 2)) * ld + n);
            } else {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int k = k0 + 16 * s + (lane >> 2);
                    f[s] = k < K && n < N ? load_k8(w + k * ld, n, N) : s16x8{};
                }
            }
        }
    }
    // the fragments of what load_w loaded
    static __device__ __forceinline__ void turn(LIN_LDS char* l, int lane, s16x8 (&f)[4]) {
        if (LB == KC) return;
#pragma unroll
        for (int s = 0; s < 4; ++s) *(LIN_LDS s16x8*)(l + s * 1024 + lane * 16) = f[s];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int g = lane >> 4, j = lane & 15, k = (g >> 1) * 8 + (j >> 2), col = (g & 1) * 16 + 4 * (j & 3);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LIN_LDS s16x4*)(l + s * 1024 + k * 64 + col * 2));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LIN_LDS s16x4*)(l + s * 1024 + (k + 4) * 64 + col * 2));
            f[s] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
};
template <int LB>
struct Few<float, LB> {   // fp32: a chunk is 32 k, four steps of 8: the lower half of the lanes has the first four of them, in 16-byte loads
    static constexpr int CHUNK = 32, TURN = 0;
    typedef f32x4 type;
    static __device__ __forceinline__ void load_x(const float* row, int k0, int K, int lane, f32x4 (&f)[4]) {
        typedef float M4 __attribute__((ext_vector_type(4), aligned(4)));
        if (k0 + CHUNK <= K) {
#pragma unroll
            for (int s = 0; s < 4; ++s) f[s] = *(const M4*)(row + k0 + 8 * s + 4 * (lane >> 5));
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = k0 + 8 * s + 4 * (lane >> 5) + e;
                    const float v = row[min(k, K - 1)];
                    f[s][e] = k < K ? v : 0.f;
                }
            }
        }
    }
    static __device__ __forceinline__ void load_w(const float* w, int64_t ld, int n0, int N, int k0, int K, int lane, f32x4 (&f)[4]) {
        const int n = min(n0 + (lane & 31), N - 1);
        if (LB == KC) return load_x(w + n * ld, k0, K, lane, f);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int k = k0 + 8 * s + 4 * (lane >> 5) + e;
                const float v = w[min(k, K - 1) * ld + n];
                f[s][e] = k < K ? v : 0.f;
            }
        }
    }
    static __device__ __forceinline__ void turn(LIN_LDS char*, int, f32x4 (&)[4]) {}
};
template <class T, int LB>
__global__ void __launch_bounds__(512) k_linear_few(const GemmP p) {
    typedef Few<T, LB> F;
    constexpr int WAVES = 8;
    __shared__ __attribute__((aligned(1024))) char lds[WAVES * (F::TURN > 4096 ? F::TURN : 4096)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // neighbouring columns on one XCD: they share lines
    const int blocks = gridDim.x, xcd = blockIdx.x & 7, b = xcd * (blocks / 8) + min(xcd, blocks % 8) + (blockIdx.x >> 3), n0 = b * 32;
    const T* x = (const T*)p.a + (int64_t)min(lane & 31, p.M - 1) * p.lda;
    const T* w = (const T*)p.b;
    LIN_LDS char* L = (LIN_LDS char*)(LIN_LDS void*)lds;
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    const int chunks = (p.K + F::CHUNK - 1) / F::CHUNK;
    typename F::type fx[2][4], fw[2][4];
    if (wave < chunks) {
        F::load_w(w, p.ldb, n0, p.N, wave * F::CHUNK, p.K, lane, fw[0]);
        F::load_x(x, wave * F::CHUNK, p.K, lane, fx[0]);
    }
    for (int c = wave; c < chunks; c += 2 * WAVES) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = c + h * WAVES, next = at + WAVES;
            if (at >= chunks) break;
            if (next < chunks) {
                F::load_w(w, p.ldb, n0, p.N, next * F::CHUNK, p.K, lane, fw[h ^ 1]);
                F::load_x(x, next * F::CHUNK, p.K, lane, fx[h ^ 1]);
            }
            F::turn(L + wave * F::TURN, lane, fw[h]);
#pragma unroll
            for (int s = 0; s < 4; ++s) acc = mfma<T>(fw[h][s], fx[h][s], acc);
        }
    }
    __syncthreads();
    // sums of the waves: [wave][row 32][column 32], 16-byte chunk c of row r at c ^ (r & 7)
    const int r = lane & 31;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const f32x4 v = {acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
        *(LIN_LDS f32x4*)(L + wave * 4096 + r * 128 + (((2 * g + (lane >> 5)) ^ (r & 7)) << 4)) = v;
    }
    __syncthreads();
    const int m = threadIdx.x >> 2, c = (threadIdx.x & 3) * 2, n = n0 + c * 4;
    if (m >= p.M || n >= p.N) return;   // (m < 32 of the 128)
    f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
    for (int q = 0; q < WAVES; ++q) {
        lo += *(const LIN_LDS f32x4*)(L + q * 4096 + m * 128 + ((c ^ (m & 7)) << 4));
        hi += *(const LIN_LDS f32x4*)(L + q * 4096 + m * 128 + (((c + 1) ^ (m & 7)) << 4));
    }
    epilogue<T>(p, m, n, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <class T, int LA, int LB, int BM, int BN, int WM, int WN>
int launch_tile(const GemmP& p, int most, hipStream_t s) {
    const int64_t items = (int64_t)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN) * p.splits;
    if (items > 0x7FFFFFFF) return INSMOS_EINVAL;
    ProfScope ps(KK_LINEAR, s);
    ps.meta[0] = p.M; ps.meta[1] = p.N; ps.meta[2] = p.K; ps.meta[3] = p.splits;
    const auto kernel = k_linear_gemm<T, LA, LB, BM, BN, WM, WN>;
    INSMOS_LAUNCH(kernel, dim3((unsigned)(items < most ? items : most)), dim3(64 * WM * WN), 0, s, p);
    HIP_TRY(hipGetLastError());
    return INSMOS_OK;
}
// Launches one product with the given tile; the parts are joined by a second launch.
int launch_gemm_bf16(const GemmP& p, int la, int lb, int tile, hipStream_t s);
int launch_gemm_f16(const GemmP& p, int la, int lb, int tile, hipStream_t s);
int launch_gemm_f32(const GemmP& p, int la, int lb, int tile, hipStream_t s);

template <class T, int LA, int LB>
int launch_gemm_l(const GemmP& p, int tile, hipStream_t s) {
    int rc = INSMOS_EINVAL;
    if constexpr (LA == KC) {
        if (tile == FEW) {
            ProfScope ps(KK_LINEAR, s);
            ps.meta[0] = p.M; ps.meta[1] = p.N; ps.meta[2] = p.K; ps.meta[3] = 1;
            const auto kernel = k_linear_few<T, LB>;
            INSMOS_LAUNCH(kernel, dim3((unsigned)((p.N + 31) / 32)), dim3(512), 0, s, p);
            HIP_TRY(hipGetLastError());
            return INSMOS_OK;
        }
    }
    // persistent: as many workgroups as fit on the CUs at once
    if constexpr (sizeof(T) == 2) {
        if (tile == T256) rc = launch_tile<T, LA, LB, 256, 256, 2, 4>(p, 256, s);
    }
    if (tile == T128) rc = launch_tile<T, LA, LB, 128, 128, 2, 2>(p, 512, s);
    if (tile == T128X64) rc = launch_tile<T, LA, LB, 128, 64, 2, 2>(p, 768, s);
    if (tile == T64X128) rc = launch_tile<T, LA, LB, 64, 128, 1, 4>(p, 768, s);
    if (tile == T128X32) rc = launch_tile<T, LA, LB, 128, 32, 4, 1>(p, 1024, s);
    if (tile == T32X128) rc = launch_tile<T, LA, LB, 32, 128, 1, 4>(p, 1024, s);
    if (rc != INSMOS_OK || p.splits == 1) return rc;
    const int64_t rows8 = (int64_t)p.M * (p.ld_part / 8);
    ProfScope ps(KK_LINEAR, s);
    // many parts are few results: 16 lanes each (469 parts of 64 x 128 fp32: 129 -> 9 us)
    if (p.splits >= 16) {
        const auto kernel = k_linear_join<T, 16>;
        INSMOS_LAUNCH(kernel, dim3((unsigned)((rows8 + 15) / 16)), dim3(256), 0, s, p);
    } else {
        const auto kernel = k_linear_join<T, 1>;
        INSMOS_LAUNCH(kernel, dim3((unsigned)((rows8 + 255) / 256)), dim3(256), 0, s, p);
    }
    HIP_TRY(hipGetLastError());
    return INSMOS_OK;
}
template <class T>
int launch_gemm(const GemmP& p, int la, int lb, int tile, hipStream_t s) {
    if (la == KC && lb == KC) return launch_gemm_l<T, KC, KC>(p, tile, s);
    if (la == KC && lb == NC) return launch_gemm_l<T, KC, NC>(p, tile, s);
    if (la == NC && lb == NC) return launch_gemm_l<T, NC, NC>(p, tile, s);
    return INSMOS_EINVAL;
}
}  // namespace lin
}  // namespace insmos

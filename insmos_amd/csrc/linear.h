// insmos_amd/csrc/linear.h -- the tiled matrix product behind insmos_linear / insmos_linear_backward (linear_bf16.hip, linear_f16.hip,
// linear_f32.hip: its instances; linear.hip: entry points and the element-wise parts).
//
//   C[m][n] = epilogue( sum_k A[m][k] B[k][n] )
//
// Both operands may have their contraction index contiguous (KC) or the other one (NC): x W is (KC, NC) for W (cin, cout) and (KC, KC) for
// a transposed (cout, cin) weight, dz W^T the other way round, x^T dz is (NC, NC).  Nothing is transposed in memory.
//
// A tile row of either operand is 128 bytes of LDS (64 16-bit or 32 fp32 values of k for KC, or BK rows of R values for NC); a wave
// instruction moves 64 x 16 bytes from memory straight to LDS (buffer_load ... lds), with the buffer's extent as the bounds check:
// rows behind the matrix read as zero, and so does k behind its end.  Two tiles in LDS: one is filled while the other is read.
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
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
template <class T> struct Vec;
template <> struct Vec<float> { typedef f32x4 t; };
template <> struct Vec<__bf16> { typedef bf16x4 t; };
template <> struct Vec<_Float16> { typedef f16x4 t; };

enum { KC = 0, NC = 1 };                                            // which index of an operand is contiguous
enum { T256 = 0, T128 = 1, TNARROW = 2, TFLAT = 3 };                // tiles 256x256, 128x128, 128x32 (few columns), 32x128 (few rows)

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
    void* z;              // the value before the activation, or null
    int64_t ld_z;
    int act, res_first;
    int vec;              // y, z, res, bias allow accesses of 4 values
};

// ---- activations ------------------------------------------------------------------------------------------------------------
// (v_exp and v_rcp: 1 ulp each; exp(-x) = inf gives 0)
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __expf(-x)); }
constexpr float kGelu0 = 0.7978845608028654f, kGelu1 = 0.044715f;   // sqrt(2 / pi) (z + 0.044715 z^3)
__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case INSMOS_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
        case INSMOS_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.7071067811865476f));
        case INSMOS_ACT_GELU_TANH: return z * sigmoid(2.f * kGelu0 * (z + kGelu1 * z * z * z));   // (1 + tanh u) / 2 = sigmoid(2 u)
        case INSMOS_ACT_SILU: return z * sigmoid(z);
    }
    return z;
}
__device__ __forceinline__ float slope(float z, int act) {
    switch (act) {
        case INSMOS_ACT_RELU: return z > 0.f ? 1.f : 0.f;
        case INSMOS_ACT_GELU: return 0.5f * (1.f + erff(z * 0.7071067811865476f)) + z * __expf(-0.5f * z * z) * 0.3989422804014327f;
        case INSMOS_ACT_GELU_TANH: {
            const float s = sigmoid(2.f * kGelu0 * (z + kGelu1 * z * z * z));
            return s + z * 2.f * s * (1.f - s) * kGelu0 * (1.f + 3.f * kGelu1 * z * z);
        }
        case INSMOS_ACT_SILU: { const float s = sigmoid(z); return s * (1.f + z * (1.f - s)); }
    }
    return 1.f;
}
// values n..n+3 of row m, from the fp32 sums
template <class T>
__device__ __forceinline__ void epilogue(const GemmP& p, int m, int n, f32x4 v) {
    typedef typename Vec<T>::t T4;
    const T* bias = (const T*)p.bias;
    const T* res = p.res ? (const T*)p.res + (int64_t)m * p.ld_res : nullptr;
    T* y = (T*)p.y + (int64_t)m * p.ld_y;
    T* z = p.z ? (T*)p.z + (int64_t)m * p.ld_z : nullptr;
    if (p.vec && n + 4 <= p.N) {
        if (bias) v += __builtin_convertvector(*(const T4*)(bias + n), f32x4);
        f32x4 r = {0.f, 0.f, 0.f, 0.f};
        if (res) r = __builtin_convertvector(*(const T4*)(res + n), f32x4);
        if (p.res_first) v += r;
        if (z) *(T4*)(z + n) = __builtin_convertvector(v, T4);
        if (p.act) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = activate(v[e], p.act);
        }
        if (res && !p.res_first) v += r;
        *(T4*)(y + n) = __builtin_convertvector(v, T4);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (n + e >= p.N) break;
        float u = v[e];
        if (bias) u += (float)bias[n + e];
        const float r = res ? (float)res[n + e] : 0.f;
        if (p.res_first) u += r;
        if (z) z[n + e] = (T)u;
        u = activate(u, p.act);
        if (res && !p.res_first) u += r;
        y[n + e] = (T)u;
    }
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
        if (LAY == KC) {
            p = (const char*)base + (int64_t)r0 * ld * ES;
            left = ((int64_t)(min(R, rtot - r0) - 1) * ld + (K + CE - 1) / CE * CE) * ES;   // (rows are whole chunks, see loadable())
            step = 128;
            chunk = ((lane & 7) ^ (lane >> 3)) * CE;
            voff = (uint32_t)((wave * 8 + (lane >> 3)) * ld * ES) + chunk * ES;
            istep = (uint32_t)(NW * 8 * ld * ES);
        } else {
            static_assert(NI == 1 || ES == 4 || NW * RPI % 16 == 0, "one swizzle for a lane's instructions");
            p = (const char*)base + (int64_t)r0 * ES;
            // (the check goes by dwords: the one that holds the last value counts as inside)
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
    // k_left: K minus the tile's first k
    __device__ __forceinline__ void load(LIN_LDS char* __restrict lds, int k_left, int wave) {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)max((int64_t)0, min(left, (int64_t)0x7FFFFFFF)), 0x00027000);
        const uint32_t v = LAY == KC && chunk >= k_left ? 0x80000000u : voff;
#pragma unroll
        for (int i = 0; i < NI; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (LIN_LDS void*)(lds + (i * NW + wave) * 1024), 16, v, i * istep, 0, 0);
        p += step;
        left -= step;
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
// fp32: four steps of 32x32x2 take the k of 8 in the order 0 2 | 4 6 | 1 3 | 5 7 (the lower half of the lanes has the first of each pair).  That
// is the order in which 16x16x4 instructions over 8-byte pieces add, which is how the platform's fp32 product usually sums: the two then agree
// to the last bit, and so do a relu's decisions at its border.
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
template <class T, int LA, int LB, int BM, int BN, int WM, int WN>
struct Gemm {
    static constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, SA = BM * 128, SB = BN * 128, BK = 128 / sizeof(T);
    typedef Tile<T, LA, BM, NW> TA;
    typedef Tile<T, LB, BN, NW> TB;
    typedef Frag<T, LA, BM, TM> FA;
    typedef Frag<T, LB, BN, TN> FB;
    // One k tile: the next one is on its way into wr while rd is read.  (wr and rd never overlap, and __restrict says so: otherwise every
    // LDS read would wait for the loads.)
    static __device__ __forceinline__ void step(LIN_LDS char* __restrict wr, const LIN_LDS char* __restrict rd, TA& ta, TB& tb, const FA& fa,
                                                const FB& fb, f32x16 (&acc)[TM][TN], bool more, int k_left, int wave) {
        if (more) {
            ta.load(wr, k_left, wave);
            tb.load(wr + SA, k_left, wave);
        }
        typename FA::type a[2][TM];
        typename FB::type b[2][TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) b[0][j] = fb.get(rd + SA, j, 0);
#pragma unroll
        for (int i = 0; i < TM; ++i) a[0][i] = fa.get(rd, i, 0);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (s < 3) {
#pragma unroll
                for (int j = 0; j < TN; ++j) b[(s + 1) & 1][j] = fb.get(rd + SA, j, s + 1);
#pragma unroll
                for (int i = 0; i < TM; ++i) a[(s + 1) & 1][i] = fa.get(rd, i, s + 1);
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = mfma<T>(b[s & 1][j], a[s & 1][i], acc[i][j]);
            if (sizeof(T) == 2 && s < 3) {
                // the next fragments are read between the matrix instructions and not in a row in front of them (1096 -> 1200 TFLOP/s at
                // 8192 x 8192 x 4096, bf16)
                constexpr int READS = (LA == KC ? TM : 2 * TM) + (LB == KC ? TN : 2 * TN), PER = (READS + TM * TN - 1) / (TM * TN);
#pragma unroll
                for (int q = 0; q < TM * TN; ++q) {
                    __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);   // LDS reads
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);     // one matrix instruction
                }
            }
        }
    }
};

// A work item is a tile of C and a part of k.  Workgroup w runs on XCD w % 8 (each has an L2 of its own), so every XCD gets a contiguous run
// of items, walked in groups of 8 tile rows: the operands of the tiles in flight on one XCD stay in its L2.
template <class T, int LA, int LB, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) k_linear_gemm(const GemmP p) {
    typedef Gemm<T, LA, LB, BM, BN, WM, WN> G;
    constexpr int TM = G::TM, TN = G::TN, SA = G::SA, SB = G::SB, BK = G::BK;
    __shared__ __attribute__((aligned(1024))) char lds[2 * (SA + SB)];
    LIN_LDS char* L = (LIN_LDS char*)(LIN_LDS void*)lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int gm = (p.M + BM - 1) / BM, gn = (p.N + BN - 1) / BN, tiles = gm * gn, items = tiles * p.splits;
    const int nk = (p.K + BK - 1) / BK, per_split = (nk + p.splits - 1) / p.splits;
    const int xcd = blockIdx.x & 7, per = items / 8, rest = items % 8;
    const int mine = per + (xcd < rest), base = xcd * per + min(xcd, rest), stride = (gridDim.x - xcd + 7) >> 3;
    typename G::FA fa;
    typename G::FB fb;
    fa.init(wm * (BM / WM), lane);
    fb.init(wn * (BN / WN), lane);
    typename G::TA ta;
    typename G::TB tb;
    int tm = 0, tn = 0, kt0 = 0, kt1 = 0, split = 0;
    auto begin = [&](int q) {   // the loads' side of item q of this XCD
        const int id = base + q, t = id % tiles;
        split = id / tiles;
        constexpr int GM = 8;
        const int first = t / (GM * gn) * GM, gs = min(GM, gm - first), in = t - first * gn;
        tm = first + in % gs;
        tn = in / gs;
        kt0 = split * per_split;
        kt1 = min(nk, kt0 + per_split);
        ta.init(p.a, p.lda, tm * BM, p.M, p.K, kt0, wave, lane);
        tb.init(p.b, p.ldb, tn * BN, p.N, p.K, kt0, wave, lane);
        ta.load(L, p.K - kt0 * BK, wave);
        tb.load(L + SA, p.K - kt0 * BK, wave);
    };
    int q = blockIdx.x >> 3;
    if (q >= mine) return;   // (the same for the workgroup)
    begin(q);
    while (true) {
        f32x16 acc[TM][TN];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
        uint32_t cur = 0;
        for (int kt = kt0; kt < kt1; ++kt) {
            __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this tile has arrived
            __syncthreads();                      // ... for every wave, and all are done with the other one
            G::step(L + (cur ^ (SA + SB)), L + cur, ta, tb, fa, fb, acc, kt + 1 < kt1, p.K - (kt + 1) * BK, wave);
            cur ^= SA + SB;
        }
        __syncthreads();
        const int m0 = tm * BM + wm * (BM / WM) + (lane & 31), n0 = tn * BN + wn * (BN / WN) + (lane >> 5) * 4, sp = split;
        const bool more = q + stride < mine;
        q += stride;
        if (more) begin(q);   // the next item's first tile is on its way during the epilogue
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int m = m0 + i * 32;
            if (m < p.M) {
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int n = n0 + j * 32 + e * 8;
                        const f32x4 v = {acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
                        if (n >= p.N) continue;
                        if (p.splits > 1) *(f32x4*)(p.part + ((int64_t)sp * p.M + m) * p.ld_part + n) = v;   // (ld_part: a multiple of 4)
                        else epilogue<T>(p, m, n, v);
                    }
            }
        }
        if (!more) return;
    }
}
// Sums the parts of k in their order, four columns a lane.
template <class T>
__global__ void __launch_bounds__(256) k_linear_join(const GemmP p) {
    const int cols = (p.N + 3) / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)p.M * cols) return;
    const int m = (int)(i / cols), n = (int)(i % cols) * 4;
    const float* q = p.part + (int64_t)m * p.ld_part + n;
    const int64_t per = (int64_t)p.M * p.ld_part;
    f32x4 s = *(const f32x4*)q;
    for (int k = 1; k < p.splits; ++k) s += *(const f32x4*)(q + k * per);
    epilogue<T>(p, m, n, s);
}

template <class T, int LA, int LB, int BM, int BN, int WM, int WN>
int launch_tile(const GemmP& p, int most, hipStream_t s) {
    const int64_t items = (int64_t)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN) * p.splits;
    if (items > 0x7FFFFFFF) return INSMOS_EINVAL;
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
    constexpr int MANY = 0x7FFFFFFF;
    int rc = INSMOS_EINVAL;
    if constexpr (sizeof(T) == 2) {
        if (tile == T256) rc = launch_tile<T, LA, LB, 256, 256, 2, 4>(p, 256, s);   // one workgroup per CU, walking its items
    }
    if (tile == T128) rc = launch_tile<T, LA, LB, 128, 128, 2, 2>(p, MANY, s);
    if (tile == TNARROW) rc = launch_tile<T, LA, LB, 128, 32, 4, 1>(p, MANY, s);
    if (tile == TFLAT) rc = launch_tile<T, LA, LB, 32, 128, 1, 4>(p, MANY, s);
    if (rc != INSMOS_OK || p.splits == 1) return rc;
    const int64_t threads = (int64_t)p.M * ((p.N + 3) / 4);
    const auto kernel = k_linear_join<T>;
    INSMOS_LAUNCH(kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, p);
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

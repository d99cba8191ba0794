// insmos_amd/csrc/linear.hip -- insmos_linear / insmos_linear_backward: y = act(x W + b [+ r]) [+ r] and its gradients.
//
//   dz = dy act'(z);   dx = dz W^T;   dW = x^T dz;   db = sum over rows of dz;   dr = dz (residual first) or dy
//
// The three products are linear.h's; here is what surrounds them: the choice of tile and of parts of k, the layout of operands that the
// 16-byte loads cannot take as they are, dz with the column sums (one pass over dy and the slopes), and the argument checks.
#include <algorithm>
#include <cmath>
#include "linear.h"

namespace insmos {
namespace lin {
namespace {

size_t size_of(int dtype) { return dtype == INSMOS_F32 ? 4 : 2; }

// ---- operands that need another layout --------------------------------------------------------------------------------------
// The tile loads move 16 bytes from any address on 4 bytes; 16-bit operands at odd addresses or pitches are copied into rows padded with zeros.
__global__ void __launch_bounds__(256) k_linear_pack(const uint16_t* __restrict__ src, int64_t ld, int64_t rows, int cols, uint16_t* __restrict__ dst,
                                                     int ld_dst) {
    constexpr int V = 8;
    const int per = ld_dst / V;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * per; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per;
        const int c = (int)(i % per) * V;
        typedef uint16_t U8 __attribute__((ext_vector_type(8), aligned(2)));
        U8 v = {0, 0, 0, 0, 0, 0, 0, 0};
        if (c + V <= cols) v = *(const U8*)(src + r * ld + c);
        else
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c + e < cols) v[e] = src[r * ld + c + e];
        typedef uint16_t A8 __attribute__((ext_vector_type(8)));
        *(A8*)(dst + r * ld_dst + c) = v;
    }
}
struct Operand {
    const void* p;
    int64_t ld;
    int lay;
};
int round_up(int v, int to) { return (v + to - 1) / to * to; }
bool loadable(const void* p, int64_t ld, int dtype) { return (uintptr_t)p % 4 == 0 && ld * size_of(dtype) % 4 == 0; }
size_t packed_bytes(int64_t rows, int cols, int dtype) {
    return pad256((size_t)rows * round_up(cols, 16 / (int)size_of(dtype)) * size_of(dtype));
}
// `rows` x `cols` (cols contiguous) as a loadable operand; copies into ws where it is none (any: the kernel takes it as it is)
int operand(const void* p, int64_t ld, int64_t rows, int cols, int lay, int dtype, bool any, Bump& ws, hipStream_t s, Operand* out) {
    *out = {p, ld, lay};
    if (any || loadable(p, ld, dtype)) return INSMOS_OK;
    const int es = (int)size_of(dtype), to = round_up(cols, 16 / es);
    char* d = ws.take<char>((size_t)rows * to * es);
    if (!d) return INSMOS_EWORKSPACE;
    const int64_t groups = (rows * (to / (16 / es)) + 255) / 256;
    const dim3 grid((unsigned)(groups < 1 << 22 ? groups : 1 << 22)), block(256);
    ProfScope ps(KK_LINEAR, s);
    INSMOS_LAUNCH(k_linear_pack, grid, block, 0, s, (const uint16_t*)p, ld, rows, cols, (uint16_t*)d, to);
    HIP_TRY(hipGetLastError());
    *out = {d, to, lay};
    return INSMOS_OK;
}

// ---- tile and parts ---------------------------------------------------------------------------------------------------------
struct Plan { int tile, splits; };
// Up to 32 rows (x W alone) there is a kernel of its own (few_rows).  Otherwise the tile and the number of parts of k with the shortest predicted time:
//   rounds of the workgroups that fit on the chip, each k tiles x max(0.75 us, workgroups per CU x a tile's work at the CU's rate) + a fixed
//   part for its first loads and its epilogue; with parts, their bytes at 4 TB/s and another launch.
// Rates (all CUs together, TFLOP/s) and fixed parts (us) are measured; predicted / measured, us, bf16: 8192 x 1024 x 1024 128x128 24 / 26,
// 256x256 39 / 33; 2048^3 128x64 29 / 32, 128x128 32 / 35; 512 x 4096 x 512 128x64 in 8 parts 18 / 15, 128x128 in 16 23 / 21; fp32:
// 300000 x 128 x 256 128x128 234 / 231, 128x64 212 / 213; 119817 x 64 x 128 128x128 31 / 37, 128x32 29 / 33.
//
// The kernel for few rows or tiles and parts, by predicted times again (us): a workgroup per 32 columns walks all of k, 8 waves taking 128 bytes
// of it in turn, against 13 for two launches or the weights' stream; odd operands, which only the tiles need copied, add that.  Few / tiles, us:
// bf16 1 x 4096 x 4096 12.6 / 13.9, 32 rows 17.8 / 16.4, 8 x 14336 x 4096 38 / 23.5, 4 x 8192 x 8192 26 / 28; fp32 8 x 1024 x 1024 10.8 / 13.5,
// 8 x 2048 x 2048 17.4 / 13.3, 4 x 4096 x 8192 33.5 / 30.
bool few_rows(int M, int N, int K, int dtype, bool odd) {
    if (M > 32) return false;
    const int trips = (int)((K * (int64_t)size_of(dtype) + 1023) / 1024), rounds = (N + 8191) / 8192;
    const double few = 4 + trips * rounds * (dtype == INSMOS_F32 ? 1.7 : 1.1 + 0.0125 * M), bytes = (double)K * N * size_of(dtype);
    return few < fmax(13, 6 + bytes / 6.5e6) + (odd ? 6 + bytes / 2.5e6 : 0);
}
// xw: the first operand has contiguous k; odd: an operand would have to be copied for the tiles
Plan plan_for(int M, int N, int K, int dtype, bool xw, bool odd = false) {
    const int bk = 128 / (int)size_of(dtype), nk = (K + bk - 1) / bk;
    if (xw && few_rows(M, N, K, dtype, odd)) return {FEW, 1};
    struct Shape { int tile, bm, bn, slots; double rate, rate32, fixed; };
    static const Shape shapes[] = {{T256, 256, 256, 256, 1250, 0, 12},     {T128, 128, 128, 512, 1050, 140, 8},    {T128X64, 128, 64, 768, 800, 135, 5},
                                   {T64X128, 64, 128, 768, 800, 135, 5},  {T128X32, 128, 32, 1024, 500, 120, 3}, {T32X128, 32, 128, 1024, 500, 120, 3}};
    static const int parts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256, 384, 512, 768, 1024};
    Plan best = {T128, 1};
    double least = 1e300;
    for (const Shape& c : shapes) {
        const double rate = dtype == INSMOS_F32 ? c.rate32 : c.rate;
        if (rate == 0) continue;
        const int64_t tiles = (int64_t)((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
        const double unit = 2.0 * c.bm * c.bn * bk * 256 / rate * 1e-6;   // us of a k tile on one CU
        for (int want : parts) {
            if (want > 1 && (tiles * want > c.slots || nk / want < 2)) break;
            const int per = (nk + want - 1) / want, splits = (nk + per - 1) / per;   // no part without work
            const int64_t items = tiles * splits, full = items / c.slots, rest = items % c.slots;
            auto round = [&](int64_t n) {   // n workgroups at once
                const double busy = (double)((n + 255) / 256) * unit;
                return per * (busy > 0.75 ? busy : 0.75) + c.fixed;
            };
            double t = full * round(c.slots) + (rest ? round(rest) : 0);
            if (splits > 1) t += (double)splits * M * N * 8 / 4e6 + 3;
            if (t < least) {
                least = t;
                best = {c.tile, splits};
            }
        }
    }
    return best;
}
size_t plan_bytes(const Plan& r, int M, int N) { return r.splits > 1 ? pad256((size_t)r.splits * M * round_up(N, 8) * sizeof(float)) : 0; }
int run_gemm(GemmP p, const Operand& a, const Operand& b, int dtype, const Plan& r, Bump& ws, hipStream_t s) {
    p.a = a.p; p.lda = a.ld;
    p.b = b.p; p.ldb = b.ld;
    p.splits = r.splits;
    if (r.splits > 1) {
        p.ld_part = round_up(p.N, 8);
        p.part = ws.take<float>((size_t)r.splits * p.M * p.ld_part);
        if (!p.part) return INSMOS_EWORKSPACE;
    }
    return dtype == INSMOS_BF16 ? launch_gemm_bf16(p, a.lay, b.lay, r.tile, s)
           : dtype == INSMOS_F16 ? launch_gemm_f16(p, a.lay, b.lay, r.tile, s) : launch_gemm_f32(p, a.lay, b.lay, r.tile, s);
}

// ---- dz and the column sums -------------------------------------------------------------------------------------------------
struct SlopeP {
    const void* dy;
    const void* slope;   // INSMOS_SLOPE_SIGN: y; INSMOS_SLOPE_STORED, INSMOS_SLOPE_GATE: what the forward stored
    void* dz;            // or null: column sums alone
    float* part;         // [row blocks][ld_part] or null
    void* db;            // one row block: the sums' place, in the type, or null
    int64_t ld_dy, ld_slope, ld_dz;
    int64_t M;
    int N, ld_part, kind, rows;   // rows per workgroup
    int lanes;           // column lanes (a power of two <= 32)
};
// 256 lanes = `lanes` over the columns (16 bytes each) x the rest over rows; dz rounds dy act'(z) once to the type (the products read it in that
// type); the column sums are taken before the rounding, in fp32, rows in a fixed order.  Bound by HBM: 8192 x 8192 bf16 89 us (4.5 TB/s for dy, slopes
// and dz), 119817 x 128 fp32 30 us (6.1); four rows per lane are in flight.
template <class T, int KIND>
__global__ void __launch_bounds__(256) k_linear_slope(const SlopeP p) {
    constexpr int V = 16 / sizeof(T), U = 4;   // columns per lane, rows in flight
    typedef T TV __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));   // (16 bytes at any address)
    typedef typename Slope<T>::t S;
    typedef S SV __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr bool STORED = KIND == INSMOS_SLOPE_STORED || KIND == INSMOS_SLOPE_GATE;
    const int lanes = p.lanes, rl = 256 / lanes, cl = threadIdx.x % lanes, r0 = threadIdx.x / lanes;
    const int n = (blockIdx.x * lanes + cl) * V;
    const int64_t from = (int64_t)blockIdx.y * p.rows, to = min(p.M, from + p.rows);
    float sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0.f;
    if (n < p.N) {
        const bool whole = n + V <= p.N;
        for (int64_t m = from + r0; m < to; m += U * rl) {
            TV a[U], y[U];
            SV c[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t q = min(m + u * rl, to - 1);
                const T* dy = (const T*)p.dy + q * p.ld_dy + n;
                if (whole) a[u] = *(const TV*)dy;
                else
#pragma unroll
                    for (int e = 0; e < V; ++e) a[u][e] = n + e < p.N ? dy[e] : (T)0.f;
                if (STORED) c[u] = *(const SV*)((const S*)p.slope + q * p.ld_slope + n);   // (rows of whole chunks)
                if (KIND == INSMOS_SLOPE_SIGN) {
                    const T* yy = (const T*)p.slope + q * p.ld_slope + n;
                    if (whole) y[u] = *(const TV*)yy;
                    else
#pragma unroll
                        for (int e = 0; e < V; ++e) y[u][e] = n + e < p.N ? yy[e] : (T)0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (m + u * rl >= to) break;
                typedef T AV __attribute__((ext_vector_type(16 / sizeof(T))));
                AV out;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float d = (float)a[u][e];
                    if (KIND == INSMOS_SLOPE_STORED && n + e < p.N) d *= Slope<T>::load(c[u][e]);   // (inf and NaN stay what they are)
                    if (KIND == INSMOS_SLOPE_SIGN || (KIND == INSMOS_SLOPE_GATE && n + e < p.N)) {
                        const float v = KIND == INSMOS_SLOPE_SIGN ? (float)y[u][e] : Slope<T>::load(c[u][e]);
                        d = v > 0.f ? d : (v != v ? v : 0.f);   // (where a relu is shut, whatever comes from behind stays there)
                    }
                    sum[e] += d;
                    out[e] = (T)d;
                }
                if (p.dz) *(AV*)((T*)p.dz + (m + u * rl) * p.ld_dz + n) = out;   // (dz rows are padded to whole chunks, with zeros)
            }
        }
    }
    if (!p.part && !p.db) return;
    __shared__ float s[256][V + 1];
#pragma unroll
    for (int e = 0; e < V; ++e) s[threadIdx.x][e] = sum[e];
    __syncthreads();
    for (int h = rl / 2; h; h >>= 1) {
        if (r0 < h) {
#pragma unroll
            for (int e = 0; e < V; ++e) s[threadIdx.x][e] += s[threadIdx.x + h * lanes][e];
        }
        __syncthreads();
    }
    if (r0 == 0) {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (n + e < p.N) {
                if (p.db) ((T*)p.db)[n + e] = (T)s[threadIdx.x][e];
                else p.part[(int64_t)blockIdx.y * p.ld_part + n + e] = s[threadIdx.x][e];
            }
    }
}
// db[n] = sum over the row blocks: 64 lanes per column, then a tree
template <class T>
__global__ void __launch_bounds__(1024) k_linear_colsum(const float* __restrict__ part, int blocks, int N, int ld, T* __restrict__ db) {
    const int n = blockIdx.x * 16 + (threadIdx.x & 15), r = threadIdx.x >> 4;
    float s = 0.f;
    if (n < N) {
#pragma unroll 4
        for (int b = r; b < blocks; b += 64) s += part[(int64_t)b * ld + n];
    }
    __shared__ float w[64][17];
    w[r][threadIdx.x & 15] = s;
    __syncthreads();
#pragma unroll
    for (int h = 32; h; h >>= 1) {
        if (r < h) w[r][threadIdx.x & 15] += w[r + h][threadIdx.x & 15];
        __syncthreads();
    }
    if (r == 0 && n < N) db[n] = (T)w[0][threadIdx.x];
}
struct SlopePlan { int lanes, strips, rows, blocks; };
SlopePlan slope_plan(int64_t M, int N, int dtype) {
    const int v = 16 / (int)size_of(dtype);
    SlopePlan r;
    r.lanes = 1;
    while (r.lanes < 32 && r.lanes * v < N) r.lanes *= 2;
    r.strips = (N + r.lanes * v - 1) / (r.lanes * v);
    const int step = 256 / r.lanes;                       // rows of one pass of a workgroup
    int64_t blocks = 2048 / r.strips;
    if (blocks < 1) blocks = 1;
    int64_t rows = ((M + blocks - 1) / blocks + step - 1) / step * step;
    const int64_t least = (M <= 8 * step ? 8 : 4) * step;   // a trip has four rows in flight; two trips rather than a second workgroup and its launch
    if (rows < least) rows = least;
    if (rows > (int64_t)1 << 30) rows = (int64_t)1 << 30;
    r.rows = (int)rows;
    r.blocks = (int)((M + rows - 1) / rows);
    return r;
}
template <class T>
int run_slope_t(const SlopeP& p, const SlopePlan& r, void* db, hipStream_t s) {
    const auto kernel = p.kind == INSMOS_SLOPE_STORED ? k_linear_slope<T, INSMOS_SLOPE_STORED>
                        : p.kind == INSMOS_SLOPE_GATE ? k_linear_slope<T, INSMOS_SLOPE_GATE>
                        : p.kind == INSMOS_SLOPE_SIGN ? k_linear_slope<T, INSMOS_SLOPE_SIGN> : k_linear_slope<T, INSMOS_SLOPE_NONE>;
    {
        ProfScope ps(KK_LINEAR_SLOPE, s);
        INSMOS_LAUNCH(kernel, dim3(r.strips, r.blocks), dim3(256), 0, s, p);
        HIP_TRY(hipGetLastError());
    }
    if (p.part) {
        ProfScope ps(KK_LINEAR_SLOPE, s);
        const auto sum = k_linear_colsum<T>;
        INSMOS_LAUNCH(sum, dim3((p.N + 15) / 16), dim3(1024), 0, s, (const float*)p.part, r.blocks, p.N, p.ld_part, (T*)db);
        HIP_TRY(hipGetLastError());
    }
    return INSMOS_OK;
}

bool good_shape(int64_t M, int K, int N, int dtype) {
    return M >= 0 && M <= 0x7FFFFF00 && K >= 1 && N >= 1 && K <= 1 << 20 && N <= 1 << 20 &&
           (dtype == INSMOS_F32 || dtype == INSMOS_BF16 || dtype == INSMOS_F16);
}
bool good_matrix(const void* p, int64_t ld, int64_t cols, int dtype) {
    return p && ld >= cols && ld <= (int64_t)1 << 20 && (uintptr_t)p % size_of(dtype) == 0;
}
// dz needs a buffer of its own where there is an activation or dy cannot be loaded as it is
bool needs_dz(const void* dy, int64_t ld_dy, int kind, int dtype) { return kind != INSMOS_SLOPE_NONE || !loadable(dy, ld_dy, dtype); }
// What a forward call takes of ws: copies of operands that the tiles cannot load (a, b: whether x, W are such), and the parts of k.  plan: the call's.
size_t forward_need(int64_t M, int K, int N, int dtype, bool a, bool b, int w_out_in, const Plan& plan) {
    if (plan.tile == FEW) return 0;
    return (a ? packed_bytes(M, K, dtype) : 0) + (!b ? 0 : w_out_in ? packed_bytes(N, K, dtype) : packed_bytes(K, N, dtype)) + plan_bytes(plan, (int)M, N);
}
// What a backward call takes: dz where it has no place of its own, the row blocks' column sums, copies of W and x; and the parts of k, one product's
// after the other's in the same place.
struct BackwardNeed { bool dz, sums, w, x; Plan dx, dw; };
size_t backward_need(int64_t M, int K, int N, int dtype, int w_out_in, const BackwardNeed& n) {
    const size_t p1 = plan_bytes(n.dx, (int)M, K), p2 = w_out_in ? plan_bytes(n.dw, N, K) : plan_bytes(n.dw, K, N);
    return (n.dz ? packed_bytes(M, N, dtype) : 0) + (n.sums ? pad256((size_t)slope_plan(M, N, dtype).blocks * N * sizeof(float)) : 0) +
           (!n.w ? 0 : w_out_in ? packed_bytes(N, K, dtype) : packed_bytes(K, N, dtype)) + (n.x ? packed_bytes(M, K, dtype) : 0) + (p1 > p2 ? p1 : p2);
}
Plan dw_plan(int64_t M, int K, int N, int dtype, int w_out_in) { return w_out_in ? plan_for(N, K, (int)M, dtype, false) : plan_for(K, N, (int)M, dtype, false); }
BackwardNeed backward_needs(const void* dy, int64_t ld_dy, int kind, const void* x, int64_t ld_x, const void* w, int64_t ld_w, int w_out_in, int64_t M, int K, int N,
                            int dtype, bool dx, bool dw, bool db, bool dz) {
    const bool own = (dx || dw) && needs_dz(dy, ld_dy, kind, dtype), odd_w = dx && !loadable(w, ld_w, dtype);   // (what the products read of dz is loadable)
    BackwardNeed n = {own && !dz, db && slope_plan(M, N, dtype).blocks > 1, false, dw && !loadable(x, ld_x, dtype), {FEW, 1}, {FEW, 1}};
    if (dx) n.dx = plan_for((int)M, K, N, dtype, true, odd_w);
    n.w = odd_w && n.dx.tile != FEW;
    if (dw) n.dw = dw_plan(M, K, N, dtype, w_out_in);
    return n;
}
// rows of a buffer in the library's own layout: 16-byte aligned, whole chunks
bool good_rows(const void* p, int64_t ld, int N, int dtype) {
    const int64_t chunk = 16 / (int64_t)size_of(dtype);
    return (uintptr_t)p % 16 == 0 && ld % chunk == 0 && ld >= round_up(N, (int)chunk) && ld <= (int64_t)1 << 20;
}
}  // namespace
}  // namespace lin
}  // namespace insmos

using namespace insmos;
using namespace insmos::lin;

// (an operand of 16 bits may be one that is copied; where such a call takes the kernel for few rows, so do all)
extern "C" size_t insmos_linear_ws_bytes(int64_t M, int K, int N, int dtype) {
    if (!good_shape(M, K, N, dtype) || !M) return 0;
    const Plan plan = plan_for((int)M, N, K, dtype, true);
    const bool odd = dtype != INSMOS_F32;
    return std::max(forward_need(M, K, N, dtype, odd, odd, 0, plan), forward_need(M, K, N, dtype, odd, odd, 1, plan));
}
extern "C" size_t insmos_linear_ws_bytes_for(const void* x, int64_t ld_x, const void* w, int64_t ld_w, int w_out_in, int64_t M, int K, int N, int dtype) {
    if (!good_shape(M, K, N, dtype) || !M) return 0;
    const bool a = !loadable(x, ld_x, dtype), b = !loadable(w, ld_w, dtype);
    return forward_need(M, K, N, dtype, a, b, w_out_in, plan_for((int)M, N, K, dtype, true, a || b));
}
extern "C" int insmos_linear(const void* x, int64_t ld_x, const void* w, int64_t ld_w, int w_out_in, const void* bias, const void* residual,
                             int64_t ld_res, int residual_first, int act, int64_t M, int K, int N, int dtype, void* y, int64_t ld_y,
                             void* slope, int64_t ld_slope, void* ws, size_t ws_bytes, void* stream) {
    if (!good_shape(M, K, N, dtype) || act < INSMOS_ACT_NONE || act > INSMOS_ACT_SILU) return INSMOS_EINVAL;
    if (M == 0) return INSMOS_OK;
    const uintptr_t es = size_of(dtype);
    if (!good_matrix(x, ld_x, K, dtype) || !good_matrix(w, ld_w, w_out_in ? K : N, dtype) || !good_matrix(y, ld_y, N, dtype) ||
        (slope && (act == INSMOS_ACT_NONE || !good_rows(slope, ld_slope, N, dtype))) || (residual && (ld_res < 0 || ld_res > (int64_t)1 << 20 || (uintptr_t)residual % es)) ||
        (uintptr_t)bias % es || (uintptr_t)ws % 16)
        return INSMOS_EINVAL;
    const hipStream_t s = (hipStream_t)stream;
    Bump bump(ws, ws ? ws_bytes : 0);
    Operand a, b;
    const bool odd_x = !loadable(x, ld_x, dtype), odd_w = !loadable(w, ld_w, dtype);
    const Plan plan = plan_for((int)M, N, K, dtype, true, odd_x || odd_w);
    if (bump.cap < forward_need(M, K, N, dtype, odd_x, odd_w, w_out_in, plan)) return INSMOS_EWORKSPACE;   // (before the first launch)
    const bool any = plan.tile == FEW;
    int rc = operand(x, ld_x, M, K, KC, dtype, any, bump, s, &a);
    if (rc == INSMOS_OK) rc = w_out_in ? operand(w, ld_w, N, K, KC, dtype, any, bump, s, &b) : operand(w, ld_w, K, N, NC, dtype, any, bump, s, &b);
    if (rc != INSMOS_OK) return rc;
    GemmP p = {};
    p.M = (int)M; p.N = N; p.K = K;
    p.bias = bias;
    p.res = residual; p.ld_res = ld_res; p.res_first = residual && residual_first;
    p.y = y; p.ld_y = ld_y;
    p.slope = slope; p.ld_slope = ld_slope;
    p.act = act;
    return run_gemm(p, a, b, dtype, plan, bump, s);
}

extern "C" size_t insmos_linear_backward_ws_bytes(int64_t M, int K, int N, int dtype) {
    if (!good_shape(M, K, N, dtype) || !M) return 0;
    const Plan dx = plan_for((int)M, K, N, dtype, true);
    const bool odd = dtype != INSMOS_F32, sums = slope_plan(M, N, dtype).blocks > 1;
    size_t need = 0;
    for (int out_in = 0; out_in < 2; ++out_in)
        need = std::max(need, backward_need(M, K, N, dtype, out_in, {true, sums, odd && dx.tile != FEW, odd, dx, dw_plan(M, K, N, dtype, out_in)}));
    return need;
}
extern "C" size_t insmos_linear_backward_ws_bytes_for(const void* dy, int64_t ld_dy, int slope_kind, const void* x, int64_t ld_x, const void* w, int64_t ld_w,
                                                      int w_out_in, int64_t M, int K, int N, int dtype, int dx, int dw, int db, int dz) {
    if (!good_shape(M, K, N, dtype) || !M) return 0;
    return backward_need(M, K, N, dtype, w_out_in, backward_needs(dy, ld_dy, slope_kind, x, ld_x, w, ld_w, w_out_in, M, K, N, dtype, dx, dw, db, dz));
}
extern "C" int insmos_linear_backward(const void* dy, int64_t ld_dy, const void* slope, int64_t ld_slope, int slope_kind, const void* x,
                                      int64_t ld_x, const void* w, int64_t ld_w, int w_out_in, int64_t M, int K, int N, int dtype, void* dx, int64_t ld_dx, void* dw,
                                      int64_t ld_dw, void* db, void* dz, int64_t ld_dz, void* ws, size_t ws_bytes, void* stream) {
    if (!good_shape(M, K, N, dtype) || M < 1 || slope_kind < INSMOS_SLOPE_NONE || slope_kind > INSMOS_SLOPE_GATE) return INSMOS_EINVAL;
    const int64_t es = size_of(dtype), chunk = 16 / es;
    if (!good_matrix(dy, ld_dy, N, dtype) || (slope_kind == INSMOS_SLOPE_SIGN && !good_matrix(slope, ld_slope, N, dtype)) ||
        (slope_kind >= INSMOS_SLOPE_STORED && (!slope || !good_rows(slope, ld_slope, N, dtype))) || (dx && !good_matrix(dx, ld_dx, K, dtype)) ||
        (dx && !good_matrix(w, ld_w, w_out_in ? K : N, dtype)) || (dw && !good_matrix(x, ld_x, K, dtype)) ||
        (dw && !good_matrix(dw, ld_dw, w_out_in ? K : N, dtype)) || (uintptr_t)db % es || (uintptr_t)ws % 16)
        return INSMOS_EINVAL;
    // dz given: it is an output too; rows padded to whole chunks
    if (dz && !good_rows(dz, ld_dz, N, dtype)) return INSMOS_EINVAL;
    const hipStream_t s = (hipStream_t)stream;
    Bump bump(ws, ws ? ws_bytes : 0);
    int rc = INSMOS_OK;
    const BackwardNeed needs = backward_needs(dy, ld_dy, slope_kind, x, ld_x, w, ld_w, w_out_in, M, K, N, dtype, dx, dw, db, dz);
    if (bump.cap < backward_need(M, K, N, dtype, w_out_in, needs)) return INSMOS_EWORKSPACE;   // (before the first launch)
    const void* d = dy;
    int64_t ld_d = ld_dy;
    const bool own = dz || ((dx || dw) && needs_dz(dy, ld_dy, slope_kind, dtype));
    if (own || db) {
        SlopeP q = {};
        q.dy = dy; q.ld_dy = ld_dy;
        q.slope = slope; q.ld_slope = ld_slope;
        q.kind = slope_kind;
        q.M = M; q.N = N;
        const SlopePlan r = slope_plan(M, N, dtype);
        q.rows = r.rows;
        q.lanes = r.lanes;
        if (own) {
            q.ld_dz = dz ? ld_dz : round_up(N, (int)chunk);
            q.dz = dz ? dz : bump.take<char>((size_t)M * q.ld_dz * es);
            if (!q.dz) return INSMOS_EWORKSPACE;
            d = q.dz;
            ld_d = q.ld_dz;
        }
        if (db && r.blocks == 1) {   // (few rows: a launch less)
            q.db = db;
        } else if (db) {
            q.ld_part = N;
            q.part = bump.take<float>((size_t)r.blocks * N);
            if (!q.part) return INSMOS_EWORKSPACE;
        }
        rc = dtype == INSMOS_F32 ? run_slope_t<float>(q, r, db, s)
             : dtype == INSMOS_BF16 ? run_slope_t<__bf16>(q, r, db, s) : run_slope_t<_Float16>(q, r, db, s);
        if (rc != INSMOS_OK) return rc;
    }
    if (dx) {   // (M, K) = dz (M, N) W^T: k of this product is N
        Operand a, b;
        const bool any = needs.dx.tile == FEW;
        rc = operand(d, ld_d, M, N, KC, dtype, any, bump, s, &a);
        if (rc == INSMOS_OK) rc = w_out_in ? operand(w, ld_w, N, K, NC, dtype, any, bump, s, &b) : operand(w, ld_w, K, N, KC, dtype, any, bump, s, &b);
        if (rc != INSMOS_OK) return rc;
        GemmP p = {};
        p.M = (int)M; p.N = K; p.K = N;
        p.y = dx; p.ld_y = ld_dx;
        const size_t before = bump.off;
        rc = run_gemm(p, a, b, dtype, needs.dx, bump, s);
        if (rc != INSMOS_OK) return rc;
        bump.off = before;   // (dw's parts are written behind this product's, on the same stream)
    }
    if (dw) {   // (K, N) = x^T dz, or its transpose for a (N, K) weight: k of this product is M
        Operand a, b;
        rc = operand(x, ld_x, M, K, NC, dtype, false, bump, s, &a);
        if (rc == INSMOS_OK) rc = operand(d, ld_d, M, N, NC, dtype, false, bump, s, &b);
        if (rc != INSMOS_OK) return rc;
        GemmP p = {};
        p.M = w_out_in ? N : K; p.N = w_out_in ? K : N; p.K = (int)M;
        p.y = dw; p.ld_y = ld_dw;
        rc = w_out_in ? run_gemm(p, b, a, dtype, needs.dw, bump, s) : run_gemm(p, a, b, dtype, needs.dw, bump, s);
    }
    return rc;
}

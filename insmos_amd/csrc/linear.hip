// insmos_amd/csrc/linear.hip -- insmos_linear / insmos_linear_backward: y = act(x W + b [+ r]) [+ r] and its gradients.
//
//   dz = dy act'(z);   dx = dz W^T;   dW = x^T dz;   db = sum over rows of dz;   dr = dz (residual first) or dy
//
// The three products are linear.h's; here is what surrounds them: the choice of tile and of parts of k, the layout of operands that the
// 16-byte loads cannot take as they are, dz with the column sums (one pass over dy and z), and the argument checks.
#include "linear.h"

namespace insmos {
namespace lin {
namespace {

size_t size_of(int dtype) { return dtype == INSMOS_F32 ? 4 : 2; }

// ---- operands that need another layout --------------------------------------------------------------------------------------
// The tile loads move 16 aligned bytes: address and row pitch must be multiples of 16 bytes, and where k is the contiguous index it must be a
// multiple of a chunk (a chunk half behind k would bring the next row's values in).  Other operands are copied into rows padded with zeros;
// the copy's time is that of its bytes, the product's an order more.
template <class T>
__global__ void __launch_bounds__(256) k_linear_pack(const T* __restrict__ src, int64_t ld, int64_t rows, int cols, T* __restrict__ dst, int ld_dst) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    constexpr int V = 16 / sizeof(T);
    const int per = ld_dst / V;
    const int64_t r = i / per;
    const int c = (int)(i % per) * V;
    if (r >= rows) return;
    typedef T TV __attribute__((ext_vector_type(16 / sizeof(T))));
    TV v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = c + e < cols ? src[r * ld + c + e] : (T)0;
    *(TV*)(dst + r * ld_dst + c) = v;
}
struct Operand {
    const void* p;
    int64_t ld;
    int lay;
};
int round_up(int v, int to) { return (v + to - 1) / to * to; }
bool loadable(const void* p, int64_t ld, int contiguous, int lay, int dtype) {
    const int64_t es = size_of(dtype), ce = 16 / es;
    return (uintptr_t)p % 16 == 0 && ld % ce == 0 && (lay == NC || contiguous % ce == 0);
}
size_t packed_bytes(int64_t rows, int cols, int dtype) {
    return pad256((size_t)rows * round_up(cols, 16 / (int)size_of(dtype)) * size_of(dtype));
}
// `rows` x `cols` (cols contiguous) as a loadable operand; copies into ws where it is none (any: the kernel takes it as it is)
int operand(const void* p, int64_t ld, int64_t rows, int cols, int lay, int dtype, bool any, Bump& ws, hipStream_t s, Operand* out) {
    *out = {p, ld, lay};
    if (any || loadable(p, ld, cols, lay, dtype)) return INSMOS_OK;
    const int es = (int)size_of(dtype), to = round_up(cols, 16 / es);
    char* d = ws.take<char>((size_t)rows * to * es);
    if (!d) return INSMOS_EWORKSPACE;
    const int64_t threads = rows * (to / (16 / es));
    if ((threads + 255) / 256 > 0x7FFFFFFF / 256) return INSMOS_EINVAL;
    const dim3 grid((unsigned)((threads + 255) / 256)), block(256);
    if (dtype == INSMOS_F32) INSMOS_LAUNCH(k_linear_pack<uint32_t>, grid, block, 0, s, (const uint32_t*)p, ld, rows, cols, (uint32_t*)d, to);
    else INSMOS_LAUNCH(k_linear_pack<uint16_t>, grid, block, 0, s, (const uint16_t*)p, ld, rows, cols, (uint16_t*)d, to);
    HIP_TRY(hipGetLastError());
    *out = {d, to, lay};
    return INSMOS_OK;
}

// ---- tile and parts ---------------------------------------------------------------------------------------------------------
struct Plan { int tile, splits; };
// Rates of a full chip: 256x256 tiles 1200 TFLOP/s (bf16, one workgroup per CU), 128x128 1050 (two per CU); a launch takes as long as its fullest
// CU, so the larger tile pays only where its tiles fill whole rounds of 256.  Up to 32 rows or columns the flat tiles waste least.
// Where the tiles leave CUs idle, k is cut into parts, each at least 4 k tiles long, until about two workgroups per CU are there.
Plan plan_for(int M, int N, int K, int dtype, bool xw) {   // xw: the first operand has contiguous k
    const int bk = 128 / (int)size_of(dtype), nk = (K + bk - 1) / bk;
    Plan r = {T128, 1};
    int64_t tiles, want = 512;
    const int64_t t128 = (int64_t)((M + 127) / 128) * ((N + 127) / 128), t256 = (int64_t)((M + 255) / 256) * ((N + 255) / 256);
    // (one workgroup per 32 columns walks all of k: 16 x 8192 x 256 takes 25 us that way and 10 in parts)
    if (M <= 32 && xw && (K <= 4096 || N >= 4096)) { r.tile = FEW; return r; }
    if (M <= 32) { r.tile = TFLAT; tiles = (N + 127) / 128; want = 1024; }
    else if (N <= 32) { r.tile = TNARROW; tiles = (M + 127) / 128; want = 1024; }
    else {
        tiles = t128;
        if (dtype != INSMOS_F32) {
            const double c256 = (double)((t256 + 255) / 256) * 4 / 1200, c128 = (double)((t128 + 511) / 512) * 2 / 1050;
            if (c256 <= c128) { r.tile = T256; tiles = t256; want = 256; }
        }
    }
    if (tiles * 2 <= want) {
        int64_t s = want / tiles;
        if (s > nk / 4) s = nk / 4;
        if (s > 1) {
            const int per = (int)((nk + s - 1) / s);
            r.splits = (nk + per - 1) / per;   // no part without work
        }
    }
    return r;
}
size_t plan_bytes(const Plan& r, int M, int N) { return r.splits > 1 ? pad256((size_t)r.splits * M * round_up(N, 8) * sizeof(float)) : 0; }
int run_gemm(GemmP p, const Operand& a, const Operand& b, int dtype, Bump& ws, hipStream_t s) {
    const Plan r = plan_for(p.M, p.N, p.K, dtype, a.lay == KC);
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
    const void* z;       // z, or y for relu; null: no activation
    void* dz;            // or null: column sums alone
    float* part;         // [row blocks][ld_part] or null
    int64_t ld_dy, ld_z, ld_dz;
    int64_t M;
    int N, ld_part, act, rows;   // rows per workgroup
    int lanes;           // column lanes (a power of two <= 32)
};
// 256 lanes = `lanes` over the columns (16 bytes each) x the rest over rows; dz rounds dy act'(z) once to the type (the products read it in that
// type); the column sums are taken before the rounding, in fp32, rows in a fixed order.
template <class T>
__global__ void __launch_bounds__(256) k_linear_slope(const SlopeP p) {
    constexpr int V = 16 / sizeof(T);
    typedef T TV __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));   // (16 bytes at any address)
    const int lanes = p.lanes, rl = 256 / lanes, cl = threadIdx.x % lanes, r0 = threadIdx.x / lanes;
    const int n = (blockIdx.x * lanes + cl) * V;
    const int64_t from = (int64_t)blockIdx.y * p.rows, to = min(p.M, from + p.rows);
    float sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0.f;
    auto row = [&](int64_t m, const float (&d0)[V], const float (&zz)[V]) {
        TV out;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float d = d0[e];
            if (p.act && n + e < p.N) d *= slope(zz[e], p.act);
            sum[e] += d;
            out[e] = (T)d;
        }
        if (p.dz) *(TV*)((T*)p.dz + m * p.ld_dz + n) = out;   // (dz rows are padded to whole chunks, with zeros)
    };
    if (n + V <= p.N) {
        constexpr int U = 4;   // rows in flight
        for (int64_t m = from + r0; m < to; m += U * rl) {
            TV a[U], b[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t q = min(m + u * rl, to - 1);
                a[u] = *(const TV*)((const T*)p.dy + q * p.ld_dy + n);
                b[u] = p.z ? *(const TV*)((const T*)p.z + q * p.ld_z + n) : a[u];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (m + u * rl >= to) break;
                float d[V], zz[V];
#pragma unroll
                for (int e = 0; e < V; ++e) { d[e] = (float)a[u][e]; zz[e] = (float)b[u][e]; }
                row(m + u * rl, d, zz);
            }
        }
    } else if (n < p.N) {
        for (int64_t m = from + r0; m < to; m += rl) {
            const T* dy = (const T*)p.dy + m * p.ld_dy + n;
            const T* z = p.z ? (const T*)p.z + m * p.ld_z + n : nullptr;
            float d[V], zz[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                d[e] = n + e < p.N ? (float)dy[e] : 0.f;
                zz[e] = z && n + e < p.N ? (float)z[e] : 0.f;
            }
            row(m, d, zz);
        }
    }
    if (!p.part) return;
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
            if (n + e < p.N) p.part[(int64_t)blockIdx.y * p.ld_part + n + e] = s[threadIdx.x][e];
    }
}
// db[n] = sum over the row blocks: 16 lanes per column, then a tree
template <class T>
__global__ void __launch_bounds__(256) k_linear_colsum(const float* __restrict__ part, int blocks, int N, int ld, T* __restrict__ db) {
    const int n = blockIdx.x * 16 + (threadIdx.x & 15), r = threadIdx.x >> 4;
    float s = 0.f;
    if (n < N)
        for (int b = r; b < blocks; b += 16) s += part[(int64_t)b * ld + n];
    __shared__ float w[16][17];
    w[r][threadIdx.x & 15] = s;
    __syncthreads();
    if (r == 0 && n < N) {
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < 16; ++q) t += w[q][threadIdx.x & 15];
        db[n] = (T)t;
    }
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
    const int64_t least = 4 * step;
    if (rows < least) rows = least;
    if (rows > (int64_t)1 << 30) rows = (int64_t)1 << 30;
    r.rows = (int)rows;
    r.blocks = (int)((M + rows - 1) / rows);
    return r;
}
template <class T>
int run_slope_t(const SlopeP& p, const SlopePlan& r, void* db, hipStream_t s) {
    const auto kernel = k_linear_slope<T>;
    INSMOS_LAUNCH(kernel, dim3(r.strips, r.blocks), dim3(256), 0, s, p);
    HIP_TRY(hipGetLastError());
    if (db) {
        const auto sum = k_linear_colsum<T>;
        INSMOS_LAUNCH(sum, dim3((p.N + 15) / 16), dim3(256), 0, s, (const float*)p.part, r.blocks, p.N, p.ld_part, (T*)db);
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
bool needs_dz(const void* dy, int64_t ld_dy, int N, int act, int dtype) { return act != INSMOS_ACT_NONE || !loadable(dy, ld_dy, N, KC, dtype); }
}  // namespace
}  // namespace lin
}  // namespace insmos

using namespace insmos;
using namespace insmos::lin;

extern "C" size_t insmos_linear_ws_bytes(int64_t M, int K, int N, int dtype) {
    if (!good_shape(M, K, N, dtype) || !M) return 0;
    return packed_bytes(M, K, dtype) + packed_bytes(K, N, dtype) + packed_bytes(N, K, dtype) + plan_bytes(plan_for((int)M, N, K, dtype, true), (int)M, N);
}
extern "C" int insmos_linear(const void* x, int64_t ld_x, const void* w, int64_t ld_w, int w_out_in, const void* bias, const void* residual,
                             int64_t ld_res, int residual_first, int act, int64_t M, int K, int N, int dtype, void* y, int64_t ld_y, void* z,
                             int64_t ld_z, void* ws, size_t ws_bytes, void* stream) {
    if (!good_shape(M, K, N, dtype) || act < INSMOS_ACT_NONE || act > INSMOS_ACT_SILU) return INSMOS_EINVAL;
    if (M == 0) return INSMOS_OK;
    const uintptr_t es = size_of(dtype);
    if (!good_matrix(x, ld_x, K, dtype) || !good_matrix(w, ld_w, w_out_in ? K : N, dtype) || !good_matrix(y, ld_y, N, dtype) ||
        (z && !good_matrix(z, ld_z, N, dtype)) || (residual && (ld_res < 0 || ld_res > (int64_t)1 << 20 || (uintptr_t)residual % es)) ||
        (uintptr_t)bias % es || (uintptr_t)ws % 16)
        return INSMOS_EINVAL;
    const hipStream_t s = (hipStream_t)stream;
    Bump bump(ws, ws ? ws_bytes : 0);
    Operand a, b;
    const bool any = plan_for((int)M, N, K, dtype, true).tile == FEW;
    int rc = operand(x, ld_x, M, K, KC, dtype, any, bump, s, &a);
    if (rc == INSMOS_OK) rc = w_out_in ? operand(w, ld_w, N, K, KC, dtype, any, bump, s, &b) : operand(w, ld_w, K, N, NC, dtype, any, bump, s, &b);
    if (rc != INSMOS_OK) return rc;
    GemmP p = {};
    p.M = (int)M; p.N = N; p.K = K;
    p.bias = bias;
    p.res = residual; p.ld_res = ld_res; p.res_first = residual && residual_first;
    p.y = y; p.ld_y = ld_y;
    p.z = z; p.ld_z = ld_z;
    p.act = act;
    return run_gemm(p, a, b, dtype, bump, s);
}

extern "C" size_t insmos_linear_backward_ws_bytes(int64_t M, int K, int N, int dtype) {
    if (!good_shape(M, K, N, dtype) || !M) return 0;
    const SlopePlan r = slope_plan(M, N, dtype);
    const Plan dx = plan_for((int)M, K, N, dtype, true), dw = plan_for(K, N, (int)M, dtype, false), dwt = plan_for(N, K, (int)M, dtype, false);
    const size_t w1 = plan_bytes(dw, K, N), w2 = plan_bytes(dwt, N, K);
    return packed_bytes(M, N, dtype) + pad256((size_t)r.blocks * N * sizeof(float)) + packed_bytes(K, N, dtype) + packed_bytes(N, K, dtype) +
           packed_bytes(M, K, dtype) + plan_bytes(dx, (int)M, K) + (w1 > w2 ? w1 : w2);
}
extern "C" int insmos_linear_backward(const void* dy, int64_t ld_dy, const void* z, int64_t ld_z, const void* x, int64_t ld_x, const void* w,
                                      int64_t ld_w, int w_out_in, int act, int64_t M, int K, int N, int dtype, void* dx, int64_t ld_dx, void* dw,
                                      int64_t ld_dw, void* db, void* dz, int64_t ld_dz, void* ws, size_t ws_bytes, void* stream) {
    if (!good_shape(M, K, N, dtype) || M < 1 || act < INSMOS_ACT_NONE || act > INSMOS_ACT_SILU) return INSMOS_EINVAL;
    const int64_t es = size_of(dtype), chunk = 16 / es;
    if (!good_matrix(dy, ld_dy, N, dtype) || (act && !good_matrix(z, ld_z, N, dtype)) || (dx && !good_matrix(dx, ld_dx, K, dtype)) ||
        (dx && !good_matrix(w, ld_w, w_out_in ? K : N, dtype)) || (dw && !good_matrix(x, ld_x, K, dtype)) ||
        (dw && !good_matrix(dw, ld_dw, w_out_in ? K : N, dtype)) || (uintptr_t)db % es || (uintptr_t)ws % 16)
        return INSMOS_EINVAL;
    // dz given: it is an output too; rows padded to whole chunks
    if (dz && ((uintptr_t)dz % 16 || ld_dz % chunk || ld_dz < round_up(N, (int)chunk) || ld_dz > (int64_t)1 << 20)) return INSMOS_EINVAL;
    const hipStream_t s = (hipStream_t)stream;
    Bump bump(ws, ws ? ws_bytes : 0);
    int rc = INSMOS_OK;
    const void* d = dy;
    int64_t ld_d = ld_dy;
    const bool own = dz || ((dx || dw) && needs_dz(dy, ld_dy, N, act, dtype));
    if (own || db) {
        SlopeP q = {};
        q.dy = dy; q.ld_dy = ld_dy;
        q.z = act ? z : nullptr; q.ld_z = ld_z;
        q.act = act;
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
        if (db) {
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
        const int np = round_up(N, (int)chunk);
        const bool any = plan_for((int)M, K, N, dtype, true).tile == FEW;
        rc = operand(d, ld_d, M, own ? np : N, KC, dtype, any, bump, s, &a);   // (own rows end in zeros: N may count as padded there)
        if (rc == INSMOS_OK) rc = w_out_in ? operand(w, ld_w, N, K, NC, dtype, any, bump, s, &b) : operand(w, ld_w, K, N, KC, dtype, any, bump, s, &b);
        if (rc != INSMOS_OK) return rc;
        GemmP p = {};
        p.M = (int)M; p.N = K; p.K = N;
        p.y = dx; p.ld_y = ld_dx;
        rc = run_gemm(p, a, b, dtype, bump, s);
        if (rc != INSMOS_OK) return rc;
    }
    if (dw) {   // (K, N) = x^T dz, or its transpose for a (N, K) weight: k of this product is M
        Operand a, b;
        rc = operand(x, ld_x, M, K, NC, dtype, false, bump, s, &a);
        if (rc == INSMOS_OK) rc = operand(d, ld_d, M, N, NC, dtype, false, bump, s, &b);
        if (rc != INSMOS_OK) return rc;
        GemmP p = {};
        p.M = w_out_in ? N : K; p.N = w_out_in ? K : N; p.K = (int)M;
        p.y = dw; p.ld_y = ld_dw;
        rc = w_out_in ? run_gemm(p, b, a, dtype, bump, s) : run_gemm(p, a, b, dtype, bump, s);
    }
    return rc;
}

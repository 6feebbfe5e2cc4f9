// GS_CXXFLAGS: -Xclang -target-feature -Xclang -packed-fp32-ops
// Dense layer with its epilogue, forward and backward (gfx950).
//
//     z = x W^T + b,   y = act(z) + r          x [M,K], W [N,K], b [N], r, y [M,N]
//     gz = g act'(z),  dx = gz W,  dW = gz^T x,  db = sum_m gz,  dr = g
//
// One product serves all three: C[i,j] = sum_c A(i,c) B(j,c), each operand given either with c contiguous ("rows") or with c as its row index
// ("columns"): y = (x rows, W rows), dx = (gz rows, W columns), dW = (gz columns, x columns).  Products run on the matrix cores with 32-bit sums.
// fp32 operands are split into three bf16 parts, x = x1 + x2 + x3 (each part the rounding of what the ones before left: 24 bits and more in all,
// and bf16 has fp32's exponents), and six products are summed, x1 y1 + x1 y2 + x2 y1 + x2 y2 + x1 y3 + x3 y1; the three left out are below
// 2^-25 |x y| each.  That is 6 / 16 of the bf16 rate, where the fp32 matrix instruction has 1 / 16.  An infinity has no such split (inf * 0): a sum
// that comes out non-finite is done again with fp32 multiply-adds.
#include <hip/hip_runtime.h>

#include "../../include/gshell_hip.h"
#include "common.hpp"

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef __attribute__((ext_vector_type(8))) bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) f16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SOFTPLUS = 2, ACT_SILU = 3, ACT_GELU = 4 };

// act'(z) as the forward pass keeps it for the backward pass: for bf16 layers in fp16 (its 11 bits lose nothing next to bf16's 8; |act'| <= 1.13),
// for fp16 and fp32 layers in fp32 (one more rounding to the layer's own type would cost the gradients as much as their own)
template <typename T> struct dact_type { typedef float type; };
template <> struct dact_type<bf16> { typedef f16 type; };

template <typename T> __device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma<f16>(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// value and derivative of the activation
__device__ __forceinline__ void act_eval(int act, float beta, float z, float& y, float& d) {
    if (act == ACT_RELU) {
        y = z < 0.f ? 0.f : z;
        d = z <= 0.f ? 0.f : 1.f;
    } else if (act == ACT_SOFTPLUS) {
        const float t = expf(-fabsf(beta * z));          // in (0, 1]: neither end of z overflows
        y = fmaxf(z, 0.f) + log1pf(t) / beta;
        d = (z >= 0.f ? 1.f : t) / (1.f + t);
    } else if (act == ACT_SILU) {
        const float s = 1.f / (1.f + expf(-z));
        y = z * s;
        d = s * (1.f + z * (1.f - s));
    } else if (act == ACT_GELU) {
        const float phi = 0.5f * erfcf(z * -0.70710678118654752f);
        y = z * phi;
        d = phi + z * (expf(-0.5f * z * z) * 0.39894228040143268f);
    } else {
        y = z;
        d = 1.f;
    }
}

template <typename T> struct Epilogue {
    const T* bias;                                  // [N] or null
    const T* res;                                   // [M,N], row stride ldr, or null
    T* out;                                         // [M,N], row stride ldo
    typename dact_type<T>::type* dact;              // [M,N] contiguous or null
    float* part;                                    // not null: fp32 sums of this slice of the contraction go to part[split][M][N], nothing else is done
    int64_t ldr, ldo;
    int act;
    float beta;
};

template <typename T> __device__ __forceinline__ void finish(const Epilogue<T>& E, int64_t i, int64_t j, int64_t N, float z) {
    if (E.bias) z += (float)E.bias[j];
    float y, d;
    act_eval(E.act, E.beta, z, y, d);
    if (E.dact) E.dact[i * N + j] = (typename dact_type<T>::type)d;
    if (E.res) y += (float)E.res[i * E.ldr + j];
    E.out[i * E.ldo + j] = (T)y;
}

template <typename T> struct Operand {
    const T* p;
    int64_t ld;
};

// 16 values of the contraction c0 .. c0+15 of line `i` (zero outside of the operand)
template <typename T, bool COLS> __device__ __forceinline__ void fetch16(const Operand<T>& A, int64_t i, int64_t lines, int64_t c0, int64_t c_end, T (&v)[16]) {
    const bool ok = i < lines;
    if (!COLS) {
        const T* q = A.p + i * A.ld + c0;
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = ok && c0 + k < c_end ? q[k] : (T)0.f;
    } else {
        const T* q = A.p + c0 * A.ld + i;
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = ok && c0 + k < c_end ? q[(int64_t)k * A.ld] : (T)0.f;
    }
}

__device__ __forceinline__ short raw(bf16 v) { return __builtin_bit_cast(short, v); }
__device__ __forceinline__ short raw(f16 v) { return __builtin_bit_cast(short, v); }

constexpr int TILE = 128, BK = 32, LDS_ROW = 40;          // 40 shorts a line: 16-byte aligned, and 16 lines read side by side fall on distinct banks

template <typename T> __device__ __forceinline__ void stage16(const T (&v)[16], short* lds) {
    s16x8 a, b;
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = raw(v[k]), b[k] = raw(v[k + 8]);
    *(s16x8*)lds = a;
    *(s16x8*)(lds + 8) = b;
}
template <> __device__ __forceinline__ void stage16<float>(const float (&v)[16], short* lds) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        s16x8 p[3];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float x = v[8 * h + k];
            const bf16 x1 = (bf16)x;
            const float r1 = x - (float)x1;
            const bf16 x2 = (bf16)r1;
            p[0][k] = raw(x1), p[1][k] = raw(x2), p[2][k] = raw((bf16)(r1 - (float)x2));
        }
#pragma unroll
        for (int q = 0; q < 3; ++q) *(s16x8*)(lds + q * TILE * LDS_ROW + 8 * h) = p[q];
    }
}

// A non-finite sum of the split operands, done again in fp32
template <bool ACOLS, bool BCOLS> __device__ __noinline__ float plain_dot(const float* a, int64_t lda, const float* b, int64_t ldb, int64_t i, int64_t j, int64_t c0, int64_t c1) {
    float s = 0.f;
    for (int64_t c = c0; c < c1; ++c) s = fmaf(ACOLS ? a[c * lda + i] : a[i * lda + c], BCOLS ? b[c * ldb + j] : b[j * ldb + c], s);
    return s;
}

template <typename T, bool ACOLS, bool BCOLS>
__global__ void __launch_bounds__(256) k_product(Operand<T> A, Operand<T> B, int64_t M, int64_t N, int64_t K, int64_t slice, Epilogue<T> E) {
    constexpr int P = sizeof(T) == 4 ? 3 : 1;
    __shared__ __attribute__((aligned(16))) short lds_a[P * TILE * LDS_ROW], lds_b[P * TILE * LDS_ROW];
    const int64_t tiles_n = (N + TILE - 1) / TILE;
    const int64_t i0 = (int64_t)(blockIdx.x / tiles_n) * TILE, j0 = (int64_t)(blockIdx.x % tiles_n) * TILE;
    const int64_t c_begin = (int64_t)blockIdx.y * slice, c_end = c_begin + slice < K ? c_begin + slice : K;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int wi = (wave >> 1) * 64, wj = (wave & 1) * 64;
    // rows: two threads share a line; columns: neighbouring threads take neighbouring lines, so that a load of theirs is one stretch of memory
    const int la = ACOLS ? t & 127 : t >> 1, ca = (ACOLS ? t >> 7 : t & 1) * 16;
    const int lb = BCOLS ? t & 127 : t >> 1, cb = (BCOLS ? t >> 7 : t & 1) * 16;
    T va[16], vb[16];
    f32x4 acc[4][4] = {};
    fetch16<T, ACOLS>(A, i0 + la, M, c_begin + ca, c_end, va);
    fetch16<T, BCOLS>(B, j0 + lb, N, c_begin + cb, c_end, vb);
    for (int64_t c = c_begin; c < c_end; c += BK) {
        __syncthreads();
        stage16<T>(va, lds_a + la * LDS_ROW + ca);
        stage16<T>(vb, lds_b + lb * LDS_ROW + cb);
        __syncthreads();
        if (c + BK < c_end) {
            fetch16<T, ACOLS>(A, i0 + la, M, c + BK + ca, c_end, va);
            fetch16<T, BCOLS>(B, j0 + lb, N, c + BK + cb, c_end, vb);
        }
        s16x8 fa[P][4], fb[P][4];
#pragma unroll
        for (int q = 0; q < P; ++q)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                fa[q][u] = *(const s16x8*)(lds_a + q * TILE * LDS_ROW + (wi + u * 16 + (lane & 15)) * LDS_ROW + (lane >> 4) * 8);
                fb[q][u] = *(const s16x8*)(lds_b + q * TILE * LDS_ROW + (wj + u * 16 + (lane & 15)) * LDS_ROW + (lane >> 4) * 8);
            }
        // B goes in as the instruction's first operand: a lane then holds four neighbouring j of one line i
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if (P == 3) {
                    acc[u][w] = mfma<T>(fb[P - 1][w], fa[0][u], acc[u][w]);
                    acc[u][w] = mfma<T>(fb[0][w], fa[P - 1][u], acc[u][w]);
                    acc[u][w] = mfma<T>(fb[P / 2][w], fa[P / 2][u], acc[u][w]);
                    acc[u][w] = mfma<T>(fb[P / 2][w], fa[0][u], acc[u][w]);
                    acc[u][w] = mfma<T>(fb[0][w], fa[P / 2][u], acc[u][w]);
                }
                acc[u][w] = mfma<T>(fb[0][w], fa[0][u], acc[u][w]);
            }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int64_t i = i0 + wi + u * 16 + (lane & 15);
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t j = j0 + wj + w * 16 + (lane >> 4) * 4 + e;
                if (i >= M || j >= N) continue;
                float z = acc[u][w][e];
                if constexpr (P == 3) {
                    if (!(fabsf(z) < __builtin_inff())) z = plain_dot<ACOLS, BCOLS>(A.p, A.ld, B.p, B.ld, i, j, c_begin, c_end);
                }
                if (E.part) E.part[((int64_t)blockIdx.y * M + i) * N + j] = z;
                else finish<T>(E, i, j, N, z);
            }
    }
}

// the slices of a contraction joined in their order, then the epilogue
template <typename T> __global__ void __launch_bounds__(256) k_join(const float* part, int splits, int64_t M, int64_t N, Epilogue<T> E) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= M * N) return;
    float z = 0.f;
    for (int s = 0; s < splits; ++s) z += part[(int64_t)s * M * N + at];
    finish<T>(E, at / N, at % N, N, z);
}

// gz = g act'(z), rounded to the layer's type for the two products that read it, and its column sums (of the unrounded values) by slabs of rows
constexpr int GZ_COLS = 64, GZ_LINES = 4;
template <typename T>
__global__ void __launch_bounds__(256) k_gz(const T* g, int64_t ldg, const typename dact_type<T>::type* dact, int64_t M, int64_t N, int64_t slab, T* gz, float* part) {
    __shared__ float sums[GZ_LINES][GZ_COLS];
    const int64_t j = (int64_t)blockIdx.x * GZ_COLS + (threadIdx.x & 63);
    const int64_t m0 = (int64_t)blockIdx.y * slab, m1 = m0 + slab < M ? m0 + slab : M;
    float s = 0.f;
    if (j < N)
        for (int64_t m = m0 + (threadIdx.x >> 6); m < m1; m += GZ_LINES) {
            float v = (float)g[m * ldg + j];
            if (dact) v *= (float)dact[m * N + j];
            if (gz) gz[m * N + j] = (T)v;
            s += v;
        }
    if (!part) return;
    sums[threadIdx.x >> 6][threadIdx.x & 63] = s;
    __syncthreads();
    if (threadIdx.x < GZ_COLS && j < N) part[(int64_t)blockIdx.y * N + j] = (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
}

template <typename T> __global__ void __launch_bounds__(256) k_column_join(const float* part, int slabs, int64_t N, T* db) {
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (j >= N) return;
    float s = 0.f;
    for (int k = 0; k < slabs; ++k) s += part[(int64_t)k * N + j];
    db[j] = (T)s;
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------------------
constexpr int CUS = 256;

// Slices of the contraction: a grid with fewer tiles than the chip has compute units leaves the rest idle, and a long contraction can be shared out.
static int64_t slices(int64_t M, int64_t N, int64_t K) {
    const int64_t tiles = gs::cdiv(M, TILE) * gs::cdiv(N, TILE);
    if (tiles >= CUS || K <= 512) return 1;
    int64_t s = CUS * 2 / tiles;
    if (s > K / 256) s = K / 256;
    return s < 1 ? 1 : (s > 64 ? 64 : s);
}
static int64_t product_bytes(int64_t M, int64_t N, int64_t K) {
    const int64_t s = slices(M, N, K);
    return s > 1 ? s * M * N * 4 : 0;
}

template <typename T, bool ACOLS, bool BCOLS>
int product(Operand<T> A, Operand<T> B, int64_t M, int64_t N, int64_t K, Epilogue<T> E, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    if (M == 0 || N == 0) return 0;
    const int64_t s = slices(M, N, K), tiles = gs::cdiv(M, TILE) * gs::cdiv(N, TILE);
    GS_REQUIRE(tiles < (1ll << 31), "gs_linear: too many tiles");
    GS_REQUIRE(workspace_bytes >= product_bytes(M, N, K) && (s == 1 || workspace), "gs_linear: workspace too small");
    const int64_t slice = s > 1 ? gs::cdiv(gs::cdiv(K, s), BK) * BK : K;
    const int64_t used = s > 1 ? gs::cdiv(K, slice) : 1;
    Epilogue<T> first = E;
    first.part = s > 1 ? (float*)workspace : nullptr;
    hipLaunchKernelGGL((k_product<T, ACOLS, BCOLS>), dim3((unsigned)tiles, (unsigned)used), dim3(256), 0, stream, A, B, M, N, K, slice, first);
    if (s > 1) hipLaunchKernelGGL(k_join<T>, dim3((unsigned)gs::cdiv(M * N, 256)), dim3(256), 0, stream, (const float*)workspace, (int)used, M, N, E);
    GS_LAUNCH_CHECK();
    return 0;
}

constexpr int64_t GZ_SLAB = 256;
static int64_t gz_slab(int64_t M) { return M / GZ_SLAB < 65535 ? GZ_SLAB : gs::cdiv(M, 65535); }

template <typename T>
int linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* res, int64_t ldr, int64_t M, int64_t N, int64_t K, int act,
               float beta, void* y, int64_t ldy, void* dact, void* ws, int64_t ws_bytes, hipStream_t stream) {
    Epilogue<T> E{(const T*)bias, (const T*)res, (T*)y, (typename dact_type<T>::type*)dact, nullptr, ldr, ldy, act, beta};
    return product<T, false, false>({(const T*)x, ldx}, {(const T*)w, ldw}, M, N, K, E, ws, ws_bytes, stream);
}

static int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }

struct BackwardPlan {
    int64_t gz, cols, prod, total;          // byte offsets of gz, the column sums' slabs and the products' slices
};
static BackwardPlan backward_plan(int64_t M, int64_t N, int64_t K, int64_t es, bool has_dact, bool want_x, bool want_w, bool want_b) {
    BackwardPlan p;
    p.gz = 0;
    p.cols = p.gz + (has_dact ? align256(M * N * es) : 0);
    p.prod = p.cols + (want_b ? align256(gs::cdiv(M, gz_slab(M)) * N * 4) : 0);
    int64_t b = 0;
    if (want_x) b = product_bytes(M, K, N);
    if (want_w && product_bytes(N, K, M) > b) b = product_bytes(N, K, M);
    p.total = p.prod + b;
    return p;
}

template <typename T>
int linear_bwd(const void* g, int64_t ldg, const void* dact, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, void* dx,
               void* dw, void* db, void* ws, int64_t ws_bytes, hipStream_t stream) {
    const BackwardPlan p = backward_plan(M, N, K, sizeof(T), dact != nullptr, dx != nullptr, dw != nullptr, db != nullptr);
    GS_REQUIRE(ws_bytes >= p.total && (ws || p.total == 0), "gs_linear_bwd: workspace too small");
    char* base = (char*)ws;
    const T* gz = (const T*)g;
    int64_t ldgz = ldg;
    if (N > 0 && (dact || db)) {
        const int64_t slab = gz_slab(M), slabs = gs::cdiv(M, slab);
        float* part = db ? (float*)(base + p.cols) : nullptr;
        T* out = dact ? (T*)(base + p.gz) : nullptr;
        if (M > 0)
            hipLaunchKernelGGL(k_gz<T>, dim3((unsigned)gs::cdiv(N, GZ_COLS), (unsigned)slabs), dim3(256), 0, stream, (const T*)g, ldg,
                               (const typename dact_type<T>::type*)dact, M, N, slab, out, part);
        if (db) hipLaunchKernelGGL(k_column_join<T>, dim3((unsigned)gs::cdiv(N, 256)), dim3(256), 0, stream, (const float*)part, (int)slabs, N, (T*)db);
        if (dact) gz = out, ldgz = N;
        GS_LAUNCH_CHECK();
    }
    Epilogue<T> E{};
    int rc = 0;
    if (dx) {
        E.out = (T*)dx, E.ldo = K;
        rc = product<T, false, true>({gz, ldgz}, {(const T*)w, ldw}, M, K, N, E, base + p.prod, ws_bytes - p.prod, stream);
    }
    if (!rc && dw) {
        E.out = (T*)dw, E.ldo = K;
        rc = product<T, true, true>({gz, ldgz}, {(const T*)x, ldx}, N, K, M, E, base + p.prod, ws_bytes - p.prod, stream);
    }
    return rc;
}

static bool sizes_ok(int64_t M, int64_t N, int64_t K) {
    const int64_t top = 1ll << 31;
    return M >= 0 && N >= 0 && K >= 0 && M < top && N < top && K < top;
}

}  // namespace

extern "C" int64_t gs_linear_fwd_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype) {
    return sizes_ok(M, N, K) && dtype >= 0 && dtype <= 2 ? product_bytes(M, N, K) : -1;
}

extern "C" int gs_linear_fwd(const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* bias, const void* residual, int64_t ldr, int64_t M, int64_t N,
                             int64_t K, int dtype, int act, float beta, void* y, int64_t ldy, void* dact, void* workspace, int64_t workspace_bytes, gs_stream_t stream) {
    GS_REQUIRE(sizes_ok(M, N, K), "gs_linear_fwd: sizes are 0 .. 2^31 - 1");
    GS_REQUIRE(dtype >= 0 && dtype <= 2, "gs_linear_fwd: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    GS_REQUIRE(act >= 0 && act <= 4, "gs_linear_fwd: unknown activation");
    GS_REQUIRE(act != ACT_SOFTPLUS || (beta > 0.f && beta < 1e30f), "gs_linear_fwd: softplus needs a positive finite beta");
    if (M == 0 || N == 0) return 0;
    GS_REQUIRE(y && ldy >= N && (!residual || ldr >= 0), "gs_linear_fwd: null output or row stride smaller than a row");
    GS_REQUIRE(K == 0 || (x && weight && ldx >= 0 && ldw >= 0), "gs_linear_fwd: null operand");
    const auto run = dtype == DT_F32 ? linear_fwd<float> : dtype == DT_BF16 ? linear_fwd<bf16> : linear_fwd<f16>;
    return run(x, ldx, weight, ldw, bias, residual, ldr, M, N, K, act, beta, y, ldy, dact, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int64_t gs_linear_bwd_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, int has_dact, int want_x, int want_w, int want_b) {
    if (!sizes_ok(M, N, K) || dtype < 0 || dtype > 2) return -1;
    return backward_plan(M, N, K, dtype == DT_F32 ? 4 : 2, has_dact, want_x, want_w, want_b).total;
}

extern "C" int gs_linear_bwd(const void* g, int64_t ldg, const void* dact, const void* x, int64_t ldx, const void* weight, int64_t ldw, int64_t M, int64_t N, int64_t K,
                             int dtype, void* dx, void* dw, void* db, void* workspace, int64_t workspace_bytes, gs_stream_t stream) {
    GS_REQUIRE(sizes_ok(M, N, K), "gs_linear_bwd: sizes are 0 .. 2^31 - 1");
    GS_REQUIRE(dtype >= 0 && dtype <= 2, "gs_linear_bwd: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    GS_REQUIRE(M == 0 || N == 0 || (g && ldg >= 0), "gs_linear_bwd: null gradient");
    GS_REQUIRE(M == 0 || N == 0 || K == 0 || ((!dx || weight) && (!dw || x)), "gs_linear_bwd: null operand");
    const auto run = dtype == DT_F32 ? linear_bwd<float> : dtype == DT_BF16 ? linear_bwd<bf16> : linear_bwd<f16>;
    return run(g, ldg, dact, x, ldx, weight, ldw, M, N, K, dx, dw, db, workspace, workspace_bytes, (hipStream_t)stream);
}

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

// Value and derivative of the activation.  For 16-bit layers (FAST) the hardware's exp2, log2 and reciprocal (1 ulp each) and erfc by Abramowitz and Stegun
// 7.1.26 (absolute error 1.5e-7): far below the rounding of the result.  For fp32 the library's functions.
template <bool FAST> __device__ __forceinline__ float exp_(float x) { return FAST ? __builtin_amdgcn_exp2f(x * 1.44269504f) : expf(x); }
template <bool FAST> __device__ __forceinline__ float rcp_(float x) { return FAST ? __builtin_amdgcn_rcpf(x) : 1.f / x; }

template <bool FAST> __device__ __forceinline__ void act_relu(float z, float& y, float& d) {
    y = z < 0.f ? 0.f : z;
    d = z <= 0.f ? 0.f : 1.f;
}
template <bool FAST> __device__ __forceinline__ void act_softplus(float beta, float inv_beta, float z, float& y, float& d) {
    const float t = exp_<FAST>(-fabsf(beta * z));          // in [0, 1]: neither end of z overflows
    float l;
    if (FAST) {
        // log(1 + t) from log of the rounded 1 + t, put right by the ratio of t to what was added in fact
        const float u = 1.f + t, added = u - 1.f;
        l = added == 0.f ? t : __builtin_amdgcn_logf(u) * 0.69314718f * t * __builtin_amdgcn_rcpf(added);
    } else {
        l = log1pf(t);
    }
    y = (z < 0.f ? 0.f : z) + l * inv_beta;
    d = (z >= 0.f ? 1.f : t) * rcp_<FAST>(1.f + t);
}
template <bool FAST> __device__ __forceinline__ void act_silu(float z, float& y, float& d) {
    const float s = rcp_<FAST>(1.f + exp_<FAST>(-z));
    y = z * s;
    d = s * (1.f + z * (1.f - s));
}
template <bool FAST> __device__ __forceinline__ void act_gelu(float z, float& y, float& d) {
    const float e = exp_<FAST>(-0.5f * z * z);
    float phi;
    if (FAST) {
        const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * 0.70710678f * fabsf(z));
        const float c = 0.5f * e * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
        phi = z < 0.f ? c : 1.f - c;
    } else {
        phi = 0.5f * erfcf(z * -0.70710678118654752f);
    }
    y = z * phi;
    d = phi + z * (e * 0.39894228040143268f);
}
// V values at once: the choice is the same for the whole launch
template <bool FAST, int V> __device__ __forceinline__ void act_eval(int act, float beta, float inv_beta, float (&z)[V], float (&d)[V]) {
    switch (act) {
        case ACT_RELU:
#pragma unroll
            for (int k = 0; k < V; ++k) act_relu<FAST>(z[k], z[k], d[k]);
            break;
        case ACT_SOFTPLUS:
#pragma unroll
            for (int k = 0; k < V; ++k) act_softplus<FAST>(beta, inv_beta, z[k], z[k], d[k]);
            break;
        case ACT_SILU:
#pragma unroll
            for (int k = 0; k < V; ++k) act_silu<FAST>(z[k], z[k], d[k]);
            break;
        case ACT_GELU:
#pragma unroll
            for (int k = 0; k < V; ++k) act_gelu<FAST>(z[k], z[k], d[k]);
            break;
        default:
#pragma unroll
            for (int k = 0; k < V; ++k) d[k] = 1.f;
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
    float beta, inv_beta;
};

template <typename T, int V> struct __attribute__((packed)) Pack { T v[V]; };          // rows start at any element: the hardware takes unaligned vectors

template <typename T> constexpr int width() { return 16 / (int)sizeof(T); }

// V neighbouring outputs of line i, columns j ..; `in_row`: how many of them are in the row
template <typename T, int V> __device__ __forceinline__ void load_some(const T* p, int64_t in_row, float (&v)[V]) {
    if (in_row >= V) {
        const Pack<T, V> q = *(const Pack<T, V>*)p;
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = (float)q.v[k];
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = k < in_row ? (float)p[k] : 0.f;
    }
}
template <typename T, int V> __device__ __forceinline__ void store_some(T* p, int64_t in_row, const float (&v)[V]) {
    if (in_row >= V) {
        Pack<T, V> q;
#pragma unroll
        for (int k = 0; k < V; ++k) q.v[k] = (T)v[k];
        *(Pack<T, V>*)p = q;
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k < in_row) p[k] = (T)v[k];
    }
}
template <typename T, int V> __device__ __forceinline__ void finish(const Epilogue<T>& E, int64_t i, int64_t j, int64_t N, float (&z)[V]) {
    const int64_t in_row = N - j;
    float d[V], r[V];
    if (E.bias) {
        load_some<T, V>(E.bias + j, in_row, r);
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] += r[k];
    }
    if (E.res) load_some<T, V>(E.res + i * E.ldr + j, in_row, r);
    act_eval<sizeof(T) == 2, V>(E.act, E.beta, E.inv_beta, z, d);
    if (E.dact) store_some<typename dact_type<T>::type, V>(E.dact + i * N + j, in_row, d);
    if (E.res)
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] += r[k];
    store_some<T, V>(E.out + i * E.ldo + j, in_row, z);
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

// A wave's TM x 4 tiles of sums, through 16 KB of LDS of its own, 64 lines at a time: the lanes then hold 16 bytes of neighbouring outputs each, and 8 (16-bit) or 16 (fp32)
// lanes a whole line of 64.  The 16-byte piece p of line l is kept at p ^ (l & 15).  fix(i, j, z): what a sum is replaced by.
template <typename T, int TM, typename F>
__device__ __forceinline__ void store_wave(const Epilogue<T>& E, const f32x4 (&acc)[TM][4], float* lds, int64_t i0, int64_t j0, int64_t M, int64_t N, F fix) {
    constexpr int V = width<T>(), LANES = 64 / V, LINES = 64 / LANES;
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int part = 0; part < TM / 4; ++part) {
#pragma unroll
        for (int p = 0; p < TM / 4; ++p)
            if (p == part)
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int l = u * 16 + (lane & 15);
                        *(f32x4*)(lds + l * 64 + ((w * 4 + (lane >> 4)) ^ (l & 15)) * 4) = acc[p * 4 + u][w];
                    }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int l0 = 0; l0 < 64; l0 += LINES) {
            const int l = l0 + lane / LANES, c = lane % LANES * V;
            const int64_t i = i0 + part * 64 + l, j = j0 + c;
            float z[V];
#pragma unroll
            for (int k = 0; k < V; k += 4) {
                const f32x4 q = *(const f32x4*)(lds + l * 64 + (((c + k) >> 2) ^ (l & 15)) * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) z[k + e] = q[e];
            }
            if (i < M && j < N) {
                fix(i, j, z);
                if (E.part) store_some<float, V>(E.part + ((int64_t)blockIdx.y * M + i) * N + j, N - j, z);
                else finish<T, V>(E, i, j, N, z);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename T, bool ACOLS, bool BCOLS>
__global__ void __launch_bounds__(256) k_product(Operand<T> A, Operand<T> B, int64_t M, int64_t N, int64_t K, int64_t slice, Epilogue<T> E) {
    constexpr int P = sizeof(T) == 4 ? 3 : 1;
    __shared__ __attribute__((aligned(16))) union {
        struct { short a[P * TILE * LDS_ROW], b[P * TILE * LDS_ROW]; } in;
        float out[4 * 64 * 64];
    } lds;
    short *lds_a = lds.in.a, *lds_b = lds.in.b;
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
    __syncthreads();
    store_wave<T, 4>(E, acc, lds.out + wave * 64 * 64, i0 + wi, j0 + wj, M, N, [&](int64_t i, int64_t j, auto& z) {
        if constexpr (P == 3) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (!(fabsf(z[k]) < __builtin_inff()) && j + k < N) z[k] = plain_dot<ACOLS, BCOLS>(A.p, A.ld, B.p, B.ld, i, j + k, c_begin, c_end);
        }
    });
}

// ---- 16-bit products with tiles fed straight into LDS ---------------------------------------------------------------------------------------------------
// Tiles of BM x BN, 64 of the contraction a step, two buffers.  The loads of a step write LDS by themselves (16 bytes a lane, no registers in between) while the step
// before is multiplied; one barrier a step.  Fragments are read one cluster of products ahead, across the barrier too, so the matrix cores do not wait for LDS.
//   rows operand     LDS holds [line][64], 8 pieces of 16 bytes a line, piece p of line l at p ^ (l & 7): the 16 lines of a fragment fall on distinct banks
//   columns operand  LDS holds [64][line]; fragments come out transposed by ds_read_b64_tr_b16 (4 contraction rows x 16 lines a 16-lane group); the 32-byte
//                    piece q of row k sits at q ^ h(k), with h different for the 16 rows that one instruction reads
// Lines and contraction beyond the operand are loaded as zero (an offset outside of the buffer's range).
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) void lds_void;
constexpr int STEP = 64;
constexpr uint32_t OUTSIDE = 0x80000000u;          // every buffer's range: an offset of this size is outside, a tile's own offsets are below

template <bool COLS, int LINES, int THREADS> struct Feed {
    static constexpr int LOADS = LINES * STEP * 2 / (THREADS * 16);
    const char* base;
    int64_t advance;                       // bytes a step
    uint32_t off[LOADS];
    int at[LOADS];                         // the contraction index of the load's first value within the step
    __device__ __forceinline__ void init(const void* p, int64_t ld, int64_t line0, int64_t lines, int64_t c0) {
        const int t = threadIdx.x;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int q = j * THREADS + t;
            if (!COLS) {
                const int l = q >> 3, piece = (q & 7) ^ (l & 7);
                off[j] = line0 + l < lines ? (uint32_t)(l * (int)ld * 2 + piece * 16) : OUTSIDE;
                at[j] = piece * 8;
            } else {
                constexpr int PIECES = LINES / 8;
                const int k = q / PIECES, slot = q % PIECES, h = ((k & 3) | ((k >> 1) & 12)) & (PIECES / 2 - 1);
                const int l = (((slot >> 1) ^ h) * 2 + (slot & 1)) * 8;
                off[j] = line0 + l < lines ? (uint32_t)(k * (int)ld * 2 + l * 2) : OUTSIDE;
                at[j] = k;
            }
        }
        base = (const char*)p + (COLS ? c0 * ld + line0 : line0 * ld + c0) * 2;
        advance = (COLS ? ld * STEP : STEP) * 2;
    }
    // `left`: what is left of the contraction from this step on
    __device__ __forceinline__ void load(short* lds, int64_t left) {
        __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, OUTSIDE, 0x00020000);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(lds + (j * THREADS + wave * 64) * 8), 16, at[j] < left ? off[j] : OUTSIDE, 0, 0, 0);
        base += advance;
    }
};

// the fragment of 16 lines x 32 of the contraction (half `ks` of the step)
template <bool COLS, int LINES> __device__ __forceinline__ s16x8 fragment(const short* lds, int line, int ks) {
    const int lane = threadIdx.x & 63;
    if constexpr (!COLS) {
        const int l = line + (lane & 15);
        return *(const s16x8*)(lds + l * STEP + (((ks * 4 + (lane >> 4)) ^ (l & 7)) * 8));
    } else {
        s16x8 out;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int k = ks * 32 + (lane >> 4) * 8 + half * 4 + ((lane & 15) >> 2);
            const int h = ((k & 3) | ((k >> 1) & 12)) & (LINES / 16 - 1);
            const short* at = lds + k * LINES + ((line >> 4) ^ h) * 16 + (lane & 3) * 4;
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
#pragma unroll
            for (int e = 0; e < 4; ++e) out[half * 4 + e] = v[e];
        }
        return out;
    }
}

// Workgroups are dealt to the 8 XCDs in turn: give each XCD one stretch of the tiles, and walk a stretch in bands of BAND tile rows, so that the operands' lines that
// its workgroups share stay in its own L2.
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t tiles_m, uint32_t tiles_n, uint32_t& ti, uint32_t& tj) {
    constexpr uint32_t XCDS = 8, BAND = 8;
    const uint32_t total = tiles_m * tiles_n, per = total / XCDS, extra = total % XCDS, x = id % XCDS, k = id / XCDS;
    const uint32_t t = x * per + (x < extra ? x : extra) + k;
    const uint32_t band = t / (BAND * tiles_n), first = band * BAND, rows = tiles_m - first < BAND ? tiles_m - first : BAND, in = t - first * tiles_n;
    ti = first + in % rows, tj = in / rows;
}

template <typename T, bool ACOLS, bool BCOLS, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(BM / WM * (BN / WN) * 64, 2) k_product16(Operand<T> A, Operand<T> B, int64_t M, int64_t N, int64_t lines_a, int64_t lines_b, int64_t K, int64_t slice, Epilogue<T> E) {
#if defined(__HIP_DEVICE_COMPILE__)          // the host pass has no type for a buffer's descriptor
    constexpr int THREADS = BM / WM * (BN / WN) * 64, TM = WM / 16, TN = WN / 16, PARTS = TM / 4, CLUSTERS = 2 * PARTS;
    __shared__ __attribute__((aligned(1024))) short a0[BM * STEP], a1[BM * STEP], b0[BN * STEP], b1[BN * STEP];
    uint32_t ti, tj;
    tile_of(blockIdx.x, (uint32_t)((M + BM - 1) / BM), (uint32_t)((N + BN - 1) / BN), ti, tj);
    const int64_t i0 = (int64_t)ti * BM, j0 = (int64_t)tj * BN;
    const int64_t c_begin = (int64_t)blockIdx.y * slice, len = (c_begin + slice < K ? c_begin + slice : K) - c_begin;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave / (BN / WN) * WM, wj = wave % (BN / WN) * WN;
    Feed<ACOLS, BM, THREADS> fa;
    Feed<BCOLS, BN, THREADS> fb;
    fa.init(A.p, A.ld, i0, lines_a, c_begin);
    fb.init(B.p, B.ld, j0, lines_b, c_begin);
    f32x4 acc[TM][TN] = {};
    s16x8 va[2][4], vb[2][TN];
    const int steps = (int)((len + STEP - 1) / STEP);
    int64_t left = len;
    // one cluster: 4 x TN products of half `ks`, part `part` of the wave's lines
    const auto read = [&](const short* a, const short* b, int cluster) __attribute__((always_inline)) {
        const int ks = cluster / PARTS, part = cluster % PARTS;
#pragma unroll
        for (int u = 0; u < 4; ++u) va[cluster & 1][u] = fragment<ACOLS, BM>(a, wi + (part * 4 + u) * 16, ks);
        if (part == 0)
#pragma unroll
            for (int w = 0; w < TN; ++w) vb[ks][w] = fragment<BCOLS, BN>(b, wj + w * 16, ks);
    };
    const auto multiply = [&](int cluster) __attribute__((always_inline)) {
        const int ks = cluster / PARTS, part = cluster % PARTS;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int w = 0; w < TN; ++w) acc[part * 4 + u][w] = mfma<T>(vb[ks][w], va[cluster & 1][u], acc[part * 4 + u][w]);
    };
    const auto step = [&](int k, short* a, short* b, short* a_next, short* b_next) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c + 1 < CLUSTERS; ++c) {
            read(a, b, c + 1);
            multiply(c);
        }
        __syncthreads();          // the next step's tiles have arrived, and nobody reads this step's any more
        if (k + 1 < steps) read(a_next, b_next, 0);
        if (k + 2 < steps) {
            fa.load(a, left);
            fb.load(b, left);
            left -= STEP;
        }
        multiply(CLUSTERS - 1);
    };
    if (steps > 0) {
        fa.load(a0, left);
        fb.load(b0, left);
        left -= STEP;
        __syncthreads();
        if (steps > 1) {
            fa.load(a1, left);
            fb.load(b1, left);
            left -= STEP;
        }
        read(a0, b0, 0);
        for (int k = 0; k < steps; k += 2) {
            step(k, a0, b0, a1, b1);
            if (k + 1 < steps) step(k + 1, a1, b1, a0, b0);
        }
    }
    // after the last barrier nobody reads the tiles: each wave takes a quarter, or half a quarter, of them for its sums
    static_assert(WN == 64 && BM * STEP * 2 * 2 + BN * STEP * 2 * 2 >= THREADS / 64 * 64 * 64 * 4, "LDS for the sums");
    constexpr int SHARE = THREADS / 64 / 4;
    short* mine = wave / SHARE == 0 ? a0 : wave / SHARE == 1 ? a1 : wave / SHARE == 2 ? b0 : b1;
    store_wave<T, TM>(E, acc, (float*)mine + wave % SHARE * 64 * 64, i0 + wi, j0 + wj, M, N, [](int64_t, int64_t, auto&) {});
#endif
}

// rows copied to rows that start on 16 bytes, zeros behind their ends
template <typename T> __global__ void __launch_bounds__(256) k_pack(const T* p, int64_t ld, int64_t rows, int64_t cols, T* out, int64_t ldo) {
    const int64_t vectors = ldo / 8, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= rows * vectors) return;
    const int64_t r = at / vectors, c = at % vectors * 8;
    s16x8 v;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? raw(p[r * ld + c + k]) : (short)0;
    *(s16x8*)(out + r * ldo + c) = v;
}

// the slices of a contraction joined in their order, then the epilogue
template <typename T> __global__ void __launch_bounds__(256) k_join(const float* part, int splits, int64_t M, int64_t N, Epilogue<T> E) {
    constexpr int V = 4;
    const int64_t vectors = (N + V - 1) / V, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= M * vectors) return;
    const int64_t i = at / vectors, j = at % vectors * V;
    float z[V] = {}, q[V];
    for (int s = 0; s < splits; ++s) {
        load_some<float, V>(part + ((int64_t)s * M + i) * N + j, N - j, q);
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] += q[k];
    }
    finish<T, V>(E, i, j, N, z);
}

// gz = g act'(z), rounded to the layer's type for the two products that read it (rows that start on 16 bytes, zeros behind their ends), and its column sums (of
// the unrounded values) by slabs of rows
constexpr int GZ_LANES = 32, GZ_LINES = 8;
template <typename T>
__global__ void __launch_bounds__(256) k_gz(const T* g, int64_t ldg, const typename dact_type<T>::type* dact, int64_t M, int64_t N, int64_t slab, T* gz, int64_t ldgz, float* part) {
    constexpr int V = width<T>();
    __shared__ float sums[GZ_LINES][GZ_LANES * V];
    const int x = threadIdx.x % GZ_LANES, y = threadIdx.x / GZ_LANES;
    const int64_t j = ((int64_t)blockIdx.x * GZ_LANES + x) * V, in_row = N - j;
    const int64_t m0 = (int64_t)blockIdx.y * slab, m1 = m0 + slab < M ? m0 + slab : M;
    float s[V] = {};
    if (in_row > 0)
        for (int64_t m = m0 + y; m < m1; m += GZ_LINES) {
            float v[V], d[V];
            load_some<T, V>(g + m * ldg + j, in_row, v);
            if (dact) {
                load_some<typename dact_type<T>::type, V>(dact + m * N + j, in_row, d);
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] *= d[k];
            }
            if (gz) store_some<T, V>(gz + m * ldgz + j, V, v);
#pragma unroll
            for (int k = 0; k < V; ++k) s[k] += v[k];
        }
    if (!part) return;
#pragma unroll
    for (int k = 0; k < V; ++k) sums[y][x * V + k] = s[k];
    __syncthreads();
    for (int c = threadIdx.x; c < GZ_LANES * V; c += 256) {
        const int64_t at = (int64_t)blockIdx.x * GZ_LANES * V + c;
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < GZ_LINES; ++q) t += sums[q][c];
        if (at < N) part[(int64_t)blockIdx.y * N + at] = t;
    }
}

// the slabs of a column, 32 stretches of them side by side
template <typename T> __global__ void __launch_bounds__(1024) k_column_join(const float* part, int slabs, int64_t N, T* db) {
    __shared__ float sums[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int64_t j = (int64_t)blockIdx.x * 32 + x;
    const int share = (slabs + 31) / 32, k1 = (y + 1) * share < slabs ? (y + 1) * share : slabs;
    float s = 0.f;
    if (j < N)
        for (int k = y * share; k < k1; ++k) s += part[(int64_t)k * N + j];
    sums[y][x] = s;
    __syncthreads();
    if (y == 0 && j < N) {
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < 32; ++q) t += sums[q][x];
        db[j] = (T)t;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------------------
constexpr int CUS = 256;
static int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }
static int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

// How a product is run: the kernel, the slices of its contraction, what is repacked first, and what of the workspace each takes.
struct Plan {
    int tile = TILE;                    // 256, 128: the 16-bit kernels; 0: the kernel for any operands
    int64_t splits = 1, slice = 0;
    int64_t pack_a = 0, pack_b = 0;          // row strides of the repacked operands, 0: as they are
    int64_t at_a = 0, at_b = 0, at_part = 0, bytes = 0;
};
struct Line {          // an operand as the plan sees it
    const void* p;
    int64_t ld, cols;          // row stride, elements of a row that are read
    bool zeros;                // rows have zeros up to a multiple of 8 behind their ends
};
// The 16-bit kernels load 16 bytes at a time into LDS, by 31-bit offsets within a tile.
static bool direct(const Line& a) { return ((uintptr_t)a.p & 15) == 0 && a.ld % 8 == 0 && (a.cols % 8 == 0 || a.zeros) && a.ld < (1 << 21); }

static Plan plan(int es, Line a, int64_t rows_a, Line b, int64_t rows_b, int64_t M, int64_t N, int64_t K) {
    Plan p;
    const bool fast = es == 2 && up8(a.cols) < (1 << 21) && up8(b.cols) < (1 << 21) && K > 0;
    int64_t tiles;
    if (!fast) {
        p.tile = 0;
        tiles = gs::cdiv(M, TILE) * gs::cdiv(N, TILE);
    } else {
        const int64_t big = gs::cdiv(M, 256) * gs::cdiv(N, 256);
        p.tile = big >= 192 ? 256 : 128;
        tiles = p.tile == 256 ? big : gs::cdiv(M, 128) * gs::cdiv(N, 128);
        if (!direct(a)) p.pack_a = up8(a.cols);
        if (!direct(b)) p.pack_b = up8(b.cols);
    }
    const int64_t slots = p.tile == 256 ? CUS : 2 * CUS;
    if (tiles < slots && K >= 512) {
        p.splits = slots / tiles;
        if (p.splits > K / 256) p.splits = K / 256;
        if (p.splits > 256) p.splits = 256;
        if (p.splits < 1) p.splits = 1;
    }
    p.slice = p.splits > 1 ? gs::cdiv(gs::cdiv(K, p.splits), 64) * 64 : K;
    p.splits = p.splits > 1 ? gs::cdiv(K, p.slice) : 1;
    int64_t at = 0;
    p.at_a = at, at += p.pack_a ? align256(rows_a * p.pack_a * es) : 0;
    p.at_b = at, at += p.pack_b ? align256(rows_b * p.pack_b * es) : 0;
    p.at_part = at, at += p.splits > 1 ? align256(p.splits * M * N * 4) : 0;
    p.bytes = at;
    return p;
}

template <typename T> int pack(const void* p, int64_t ld, int64_t rows, int64_t cols, void* out, int64_t ldo, hipStream_t stream) {
    const int64_t blocks = gs::cdiv(rows * (ldo / 8), 256);
    GS_REQUIRE(blocks < (1ll << 31), "gs_linear: operand too large");
    hipLaunchKernelGGL(k_pack<T>, dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)p, ld, rows, cols, (T*)out, ldo);
    return 0;
}

// C [M,N] over a contraction of K.
template <typename T, bool ACOLS, bool BCOLS>
int product(Line a, Line b, int64_t M, int64_t N, int64_t K, Epilogue<T> E, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    if (M == 0 || N == 0) return 0;
    const int64_t rows_a = ACOLS ? K : M, rows_b = BCOLS ? K : N;
    const Plan p = plan(sizeof(T), a, rows_a, b, rows_b, M, N, K);
    GS_REQUIRE(workspace_bytes >= p.bytes && (workspace || p.bytes == 0), "gs_linear: workspace too small");
    char* ws = (char*)workspace;
    const int64_t t = p.tile ? p.tile : TILE, tiles = gs::cdiv(M, t) * gs::cdiv(N, t);
    GS_REQUIRE(tiles < (1ll << 31) && M * gs::cdiv(N, 4) < (255ll << 31), "gs_linear: too many tiles");
    Epilogue<T> first = E;
    first.part = p.splits > 1 ? (float*)(ws + p.at_part) : nullptr;
    const dim3 grid((unsigned)tiles, (unsigned)p.splits);
    if (p.tile == 0) {
        hipLaunchKernelGGL((k_product<T, ACOLS, BCOLS>), grid, dim3(256), 0, stream, (Operand<T>{(const T*)a.p, a.ld}), (Operand<T>{(const T*)b.p, b.ld}), M, N, K, p.slice, first);
    } else if constexpr (sizeof(T) == 2) {
        int64_t lines_a = M, lines_b = N;
        if (p.pack_a) {
            if (const int rc = pack<T>(a.p, a.ld, rows_a, a.cols, ws + p.at_a, p.pack_a, stream)) return rc;
            a = {ws + p.at_a, p.pack_a, a.cols, true};
        }
        if (p.pack_b) {
            if (const int rc = pack<T>(b.p, b.ld, rows_b, b.cols, ws + p.at_b, p.pack_b, stream)) return rc;
            b = {ws + p.at_b, p.pack_b, b.cols, true};
        }
        if (ACOLS && a.zeros) lines_a = up8(M);
        if (BCOLS && b.zeros) lines_b = up8(N);
        const Operand<T> A{(const T*)a.p, a.ld}, B{(const T*)b.p, b.ld};
        if (p.tile == 256)
            hipLaunchKernelGGL((k_product16<T, ACOLS, BCOLS, 256, 256, 128, 64>), grid, dim3(512), 0, stream, A, B, M, N, lines_a, lines_b, K, p.slice, first);
        else
            hipLaunchKernelGGL((k_product16<T, ACOLS, BCOLS, 128, 128, 64, 64>), grid, dim3(256), 0, stream, A, B, M, N, lines_a, lines_b, K, p.slice, first);
    }
    if (p.splits > 1)
        hipLaunchKernelGGL(k_join<T>, dim3((unsigned)gs::cdiv(M * gs::cdiv(N, 4), 256)), dim3(256), 0, stream, (const float*)(ws + p.at_part), (int)p.splits, M, N, E);
    GS_LAUNCH_CHECK();
    return 0;
}

template <typename T>
int linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* res, int64_t ldr, int64_t M, int64_t N, int64_t K, int act,
               float beta, void* y, int64_t ldy, void* dact, void* ws, int64_t ws_bytes, hipStream_t stream) {
    Epilogue<T> E{(const T*)bias, (const T*)res, (T*)y, (typename dact_type<T>::type*)dact, nullptr, ldr, ldy, act, beta, act == ACT_SOFTPLUS ? 1.f / beta : 0.f};
    return product<T, false, false>({x, ldx, K, false}, {w, ldw, K, false}, M, N, K, E, ws, ws_bytes, stream);
}

struct BackwardPlan {
    bool gz_made, pass;                // gz has a place of its own (an activation, or rows that the products cannot read as they are); a pass over g is made
    int64_t ldgz, slab, slabs;
    int64_t gz, cols, prod, total;          // byte offsets of gz, the column sums' slabs and the products' workspace
};
static BackwardPlan backward_plan(const void* g, int64_t ldg, bool has_dact, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, int es,
                                  bool want_x, bool want_w, bool want_b) {
    BackwardPlan p;
    p.gz_made = has_dact || (es == 2 && (want_x || want_w) && !direct({g, ldg, N, false}));
    p.pass = p.gz_made || want_b;
    p.ldgz = p.gz_made ? up8(N) : ldg;
    const int64_t across = gs::cdiv(N, GZ_LANES * 16 / es);
    p.slab = gs::cdiv(gs::cdiv(M * across, 2048), GZ_LINES) * GZ_LINES;
    if (p.slab < 64) p.slab = 64;
    if (M / p.slab >= 65535) p.slab = gs::cdiv(M, 65535);
    p.slabs = gs::cdiv(M, p.slab);
    p.gz = 0;
    p.cols = p.gz + (p.gz_made ? align256(M * p.ldgz * es) : 0);
    p.prod = p.cols + (want_b ? align256(p.slabs * N * 4) : 0);
    const Line gl{p.gz_made ? nullptr : g, p.ldgz, N, p.gz_made};
    int64_t b = 0;
    if (want_x) b = plan(es, gl, M, {w, ldw, K, false}, N, M, K, N).bytes;
    if (want_w) {
        const int64_t c = plan(es, gl, M, {x, ldx, K, false}, M, N, K, M).bytes;
        if (c > b) b = c;
    }
    p.total = p.prod + b;
    return p;
}

template <typename T>
int linear_bwd(const void* g, int64_t ldg, const void* dact, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, void* dx,
               void* dw, void* db, void* ws, int64_t ws_bytes, hipStream_t stream) {
    const BackwardPlan p = backward_plan(g, ldg, dact != nullptr, x, ldx, w, ldw, M, N, K, sizeof(T), dx != nullptr, dw != nullptr, db != nullptr);
    GS_REQUIRE(ws_bytes >= p.total && (ws || p.total == 0), "gs_linear_bwd: workspace too small");
    char* base = (char*)ws;
    Line gz{p.gz_made ? base + p.gz : g, p.ldgz, N, p.gz_made};
    if (N > 0 && p.pass) {
        float* part = db ? (float*)(base + p.cols) : nullptr;
        const int64_t across = gs::cdiv(N, GZ_LANES * width<T>());
        if (M > 0)
            hipLaunchKernelGGL(k_gz<T>, dim3((unsigned)across, (unsigned)p.slabs), dim3(256), 0, stream, (const T*)g, ldg, (const typename dact_type<T>::type*)dact, M, N, p.slab,
                               p.gz_made ? (T*)(base + p.gz) : nullptr, p.ldgz, part);
        if (db) hipLaunchKernelGGL(k_column_join<T>, dim3((unsigned)gs::cdiv(N, 32)), dim3(1024), 0, stream, (const float*)part, (int)p.slabs, N, (T*)db);
        GS_LAUNCH_CHECK();
    }
    Epilogue<T> E{};
    int rc = 0;
    if (dx) {
        E.out = (T*)dx, E.ldo = K;
        rc = product<T, false, true>(gz, {w, ldw, K, false}, M, K, N, E, base + p.prod, ws_bytes - p.prod, stream);
    }
    if (!rc && dw) {
        E.out = (T*)dw, E.ldo = K;
        rc = product<T, true, true>(gz, {x, ldx, K, false}, N, K, M, E, base + p.prod, ws_bytes - p.prod, stream);
    }
    return rc;
}

static bool sizes_ok(int64_t M, int64_t N, int64_t K) {
    const int64_t top = 1ll << 31;
    return M >= 0 && N >= 0 && K >= 0 && M < top && N < top && K < top;
}

}  // namespace

extern "C" int64_t gs_linear_fwd_workspace_bytes(const void* x, int64_t ldx, const void* weight, int64_t ldw, int64_t M, int64_t N, int64_t K, int dtype) {
    if (!sizes_ok(M, N, K) || dtype < 0 || dtype > 2) return -1;
    return M == 0 || N == 0 ? 0 : plan(dtype == DT_F32 ? 4 : 2, {x, ldx, K, false}, M, {weight, ldw, K, false}, N, M, N, K).bytes;
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

extern "C" int64_t gs_linear_bwd_workspace_bytes(const void* g, int64_t ldg, int has_dact, const void* x, int64_t ldx, const void* weight, int64_t ldw, int64_t M, int64_t N,
                                                 int64_t K, int dtype, int want_x, int want_w, int want_b) {
    if (!sizes_ok(M, N, K) || dtype < 0 || dtype > 2) return -1;
    return backward_plan(g, ldg, has_dact, x, ldx, weight, ldw, M, N, K, dtype == DT_F32 ? 4 : 2, want_x, want_w, want_b).total;
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

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
typedef __attribute__((ext_vector_type(4))) short s16x4;

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

// Value and derivative of the activation, on the hardware's exp2, log2 and reciprocal (1 ulp each).  For 16-bit layers (FAST) the exponent's product is rounded, and
// erfc is Abramowitz and Stegun 7.1.26 (absolute error 1.5e-7): far below the rounding of the result.  For fp32 the product's rounding error goes into the
// exponential as a factor, and erfc is the library's.
template <bool FAST> __device__ __forceinline__ float exp_(float x) {
    const float p = x * 1.44269504f;
    const float e = __builtin_amdgcn_exp2f(p);
    if (FAST) return e;
    // x log2(e) = p + r: r is what the product and the constant were rounded by; an infinite x has p right and r nonsense
    const float r = __builtin_fmaf(x, 1.44269504f, -p) + x * 1.92596299e-8f;
    return fabsf(p) < 1000.f ? __builtin_fmaf(e, r * 0.69314718f, e) : e;
}
__device__ __forceinline__ float rcp_(float x) { return __builtin_amdgcn_rcpf(x); }

template <bool FAST> __device__ __forceinline__ void act_relu(float z, float& y, float& d) {
    y = z < 0.f ? 0.f : z;
    d = z <= 0.f ? 0.f : 1.f;
}
template <bool FAST> __device__ __forceinline__ void act_softplus(float beta, float inv_beta, float z, float& y, float& d) {
    const float t = exp_<FAST>(-fabsf(beta * z));          // in [0, 1]: neither end of z overflows
    // log(1 + t) from the logarithm of the rounded 1 + t, put right by the ratio of t to what was added in fact
    const float u = 1.f + t, added = u - 1.f;
    const float l = added == 0.f ? t : __builtin_amdgcn_logf(u) * 0.69314718f * t * rcp_(added);
    y = (z < 0.f ? 0.f : z) + l * inv_beta;
    d = (z >= 0.f ? 1.f : t) * rcp_(1.f + t);
}
template <bool FAST> __device__ __forceinline__ void act_silu(float z, float& y, float& d) {
    const float s = rcp_(1.f + exp_<FAST>(-z));
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
// BATCH x V values at once: the choice is the same for the whole launch
template <bool FAST, int V, int BATCH> __device__ __forceinline__ void act_eval(int act, float beta, float inv_beta, float (&z)[BATCH][V], float (&d)[BATCH][V]) {
    switch (act) {
        case ACT_RELU:
#pragma unroll
            for (int k = 0; k < V * BATCH; ++k) act_relu<FAST>(z[k / V][k % V], z[k / V][k % V], d[k / V][k % V]);
            break;
        case ACT_SOFTPLUS:
#pragma unroll
            for (int k = 0; k < V * BATCH; ++k) act_softplus<FAST>(beta, inv_beta, z[k / V][k % V], z[k / V][k % V], d[k / V][k % V]);
            break;
        case ACT_SILU:
#pragma unroll
            for (int k = 0; k < V * BATCH; ++k) act_silu<FAST>(z[k / V][k % V], z[k / V][k % V], d[k / V][k % V]);
            break;
        default:
#pragma unroll
            for (int k = 0; k < V * BATCH; ++k) act_gelu<FAST>(z[k / V][k % V], z[k / V][k % V], d[k / V][k % V]);
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
// BATCH x V outputs of the lines i[0 .. BATCH-1] (those below M), columns j ..
template <typename T, int V, int BATCH> __device__ __forceinline__ void finish(const Epilogue<T>& E, const int64_t (&i)[BATCH], int64_t j, int64_t M, int64_t N, float (&z)[BATCH][V]) {
    const int64_t in_row = N - j;
    float r[BATCH][V];
    if (E.res)
#pragma unroll
        for (int b = 0; b < BATCH; ++b) load_some<T, V>(E.res + i[b] * E.ldr + j, i[b] < M ? in_row : 0, r[b]);
    if (E.bias) {
        float q[V];
        load_some<T, V>(E.bias + j, in_row, q);
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
#pragma unroll
            for (int k = 0; k < V; ++k) z[b][k] += q[k];
    }
    if (E.act != ACT_NONE) {
        float d[BATCH][V];
        act_eval<sizeof(T) == 2, V, BATCH>(E.act, E.beta, E.inv_beta, z, d);
        if (E.dact)
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
                if (i[b] < M) store_some<typename dact_type<T>::type, V>(E.dact + i[b] * N + j, in_row, d[b]);
    }
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
        if (E.res)
#pragma unroll
            for (int k = 0; k < V; ++k) z[b][k] += r[b][k];
        if (i[b] < M) store_some<T, V>(E.out + i[b] * E.ldo + j, in_row, z[b]);
    }
}

template <typename T> struct Operand {
    const T* p;
    int64_t ld;
};

// Workgroups are dealt to the 8 XCDs in turn: give each XCD one stretch of the tiles, and walk a stretch in bands of BAND tile rows, so that the operands' lines that
// its workgroups share stay in its own L2.
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t tiles_m, uint32_t tiles_n, uint32_t& ti, uint32_t& tj) {
    constexpr uint32_t XCDS = 8, BAND = 8;
    const uint32_t total = tiles_m * tiles_n, per = total / XCDS, extra = total % XCDS, x = id % XCDS, k = id / XCDS;
    const uint32_t t = x * per + (x < extra ? x : extra) + k;
    const uint32_t band = t / (BAND * tiles_n), first = band * BAND, rows = tiles_m - first < BAND ? tiles_m - first : BAND, in = t - first * tiles_n;
    ti = first + in % rows, tj = in / rows;
}

// A wave's TM x 4 tiles of sums, through 16 KB of LDS of its own, 64 lines at a time: the lanes then hold 16 bytes of neighbouring outputs each, and 8 (16-bit) or 16 (fp32)
// lanes a whole line of 64.  The 16-byte piece p of line l is kept at p ^ (l & 15).  fix(i, j, z): what a sum is replaced by.
template <typename T, int TM, int BATCH, typename F>
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
        // BATCH lines a lane side by side, as many as the registers beside the sums hold: what they read of the residual is in flight together

#pragma unroll 1
        for (int l0 = 0; l0 < 64; l0 += LINES * BATCH) {
            const int c = lane % LANES * V;
            const int64_t j = j0 + c;
            int64_t i[BATCH];
            float z[BATCH][V];
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                const int l = l0 + b * LINES + lane / LANES;
                i[b] = i0 + part * 64 + l;
#pragma unroll
                for (int k = 0; k < V; k += 4) {
                    const f32x4 q = *(const f32x4*)(lds + l * 64 + (((c + k) >> 2) ^ (l & 15)) * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[b][k + e] = q[e];
                }
                if (i[b] < M && j < N) fix(i[b], j, z[b]);
            }
            if (E.part) {
#pragma unroll
                for (int b = 0; b < BATCH; ++b)
                    if (i[b] < M && j < N) store_some<float, V>(E.part + ((int64_t)blockIdx.y * M + i[b]) * N + j, N - j, z[b]);
            } else if (j < N) {
                finish<T, V, BATCH>(E, i, j, M, N, z);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- fp32 products ------------------------------------------------------------------------------------------------------------------------------------
// Tiles of 128 x 128, 32 of the contraction a step, two workgroups a compute unit.  While a step is multiplied the next one comes
// to registers and is split there; each of the three parts has a plane of its own in LDS: [line][32], 4 pieces of 16 bytes a line, piece p of line l at p ^ (l >> 1 & 3), so that the 16
// lines of a fragment fall on distinct banks.  96 matrix instructions a wave and step stand against 24 fragments read and 32 values split a lane.
//   rows operand     a lane loads 8 neighbours of the contraction; columns operand: 16 of one line, neighbouring lanes neighbouring lines
// A may have a gate: the factor act'(z) that makes gz of g, so that gz is never stored; the products with dW also add up its columns, for db.
constexpr int TILE = 128, BK = 32;
constexpr int PLANE = TILE * BK;

__device__ __forceinline__ short raw(bf16 v) { return __builtin_bit_cast(short, v); }
__device__ __forceinline__ short raw(f16 v) { return __builtin_bit_cast(short, v); }

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

// the parts of two values, each pair in one register
__device__ __forceinline__ void split2(float x, float y, uint32_t (&part)[3]) {
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        part[q] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), bf16x2));
        if (q == 2) break;
        x -= __builtin_bit_cast(float, part[q] << 16);
        y -= __builtin_bit_cast(float, part[q] & 0xffff0000u);
    }
}
__device__ __forceinline__ int piece_at(int line, int at) { return line * BK + (((at >> 3) ^ ((line >> 1) & 3)) * 8) + (at & 7); }

template <bool COLS, bool GATE> struct Feed32 {
    const float *p, *gate;
    int64_t ld, ldgate, line0, lines, c_end;
    bool whole;                    // every line of the tile is in the operand
    // what is in flight: rows operands 2 pieces of 8 neighbours, of lines 64 apart; columns operands 16 neighbours of one line
    struct Values { float v[16], d[GATE ? 16 : 1]; };
    __device__ __forceinline__ void fetch(int64_t c, Values& V) const {
        const bool all = whole && c + BK <= c_end;
        if constexpr (!COLS) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t l = line0 + j * 64 + (threadIdx.x >> 2), at = c + (threadIdx.x & 3) * 8;
                const int64_t left = all ? 8 : l < lines ? c_end - at : 0;
#pragma unroll
                for (int h = 0; h < 8; h += 4) {
                    load_some<float, 4>(p + l * ld + at + h, left - h, *(float(*)[4])(V.v + 8 * j + h));
                    if constexpr (GATE) load_some<float, 4>(gate + l * ldgate + at + h, left - h, *(float(*)[4])(V.d + 8 * j + h));
                }
            }
        } else {
            const int64_t at = c + (__builtin_amdgcn_readfirstlane(threadIdx.x >> 7)) * 16;          // the same for a wave
            const uint32_t l = threadIdx.x & 127;
            const float* q = p + at * ld + line0;
            const float* e = GATE ? gate + at * ldgate + line0 : nullptr;
            if (all) {
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    V.v[k] = q[l];
                    q += ld;
                    if constexpr (GATE) V.d[k] = e[l], e += ldgate;
                }
            } else {
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const bool ok = line0 + l < lines && at + k < c_end;
                    V.v[k] = ok ? q[l] : 0.f;
                    q += ld;
                    if constexpr (GATE) V.d[k] = ok ? e[l] : 0.f, e += ldgate;
                }
            }
        }
    }
    struct Parts { uint32_t p[3][8]; };          // two neighbours a register
    // split; returns the sum of the values (of one line, for columns operands)
    __device__ __forceinline__ float split(Values& V, Parts& S) const {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float x = V.v[2 * k], y = V.v[2 * k + 1];
            if constexpr (GATE) x *= V.d[2 * k], y *= V.d[2 * k + 1];
            if constexpr (COLS) t += x + y;
            uint32_t part[3];
            split2(x, y, part);
#pragma unroll
            for (int q = 0; q < 3; ++q) S.p[q][k] = part[q];
        }
        return t;
    }
    __device__ __forceinline__ void store(short* lds, const Parts& S) const {
#pragma unroll
        for (int q = 0; q < 3; ++q) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int line = COLS ? threadIdx.x & 127 : h * 64 + (threadIdx.x >> 2), at = COLS ? (threadIdx.x >> 7) * 16 + 8 * h : (threadIdx.x & 3) * 8;
                *(u32x4*)(lds + q * PLANE + piece_at(line, at)) = u32x4{S.p[q][4 * h], S.p[q][4 * h + 1], S.p[q][4 * h + 2], S.p[q][4 * h + 3]};
            }
        }
    }
};

template <bool ACOLS, bool BCOLS, bool GATE>
__global__ void __launch_bounds__(256, 2) k_product32(Operand<float> A, const float* gate, int64_t ldgate, Operand<float> B, int64_t M, int64_t N, int64_t K, int64_t slice, Epilogue<float> E,
                                                      float* column_sums) {
    __shared__ __attribute__((aligned(16))) union {
        struct { short a[3 * PLANE], b[3 * PLANE]; } in;
        float out[4 * 64 * 64];
    } lds;
    uint32_t ti, tj;
    tile_of(blockIdx.x, (uint32_t)((M + TILE - 1) / TILE), (uint32_t)((N + TILE - 1) / TILE), ti, tj);
    const int64_t i0 = (int64_t)ti * TILE, j0 = (int64_t)tj * TILE;
    const int64_t c_begin = (int64_t)blockIdx.y * slice, c_end = c_begin + slice < K ? c_begin + slice : K;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = (wave >> 1) * 64, wj = (wave & 1) * 64;
    Feed32<ACOLS, GATE> fa;
    Feed32<BCOLS, false> fb;
    fa.p = A.p, fa.ld = A.ld, fa.gate = gate, fa.ldgate = ldgate, fa.line0 = i0, fa.lines = M, fa.c_end = c_end, fa.whole = i0 + TILE <= M;
    fb.p = B.p, fb.ld = B.ld, fb.line0 = j0, fb.lines = N, fb.c_end = c_end, fb.whole = j0 + TILE <= N;
    const bool sums = ACOLS && column_sums && tj == 0;
    float total = 0.f;
    f32x4 acc[4][4] = {};
    typename Feed32<ACOLS, GATE>::Values ra;
    typename Feed32<BCOLS, false>::Values rb;
    typename Feed32<ACOLS, GATE>::Parts sa;
    typename Feed32<BCOLS, false>::Parts sb;
    if (c_begin < c_end) {
        fa.fetch(c_begin, ra);
        fb.fetch(c_begin, rb);
        total += fa.split(ra, sa);
        fb.split(rb, sb);
    }
    for (int64_t c = c_begin; c < c_end; c += BK) {
        __syncthreads();
        fa.store(lds.in.a, sa);
        fb.store(lds.in.b, sb);
        __syncthreads();
        // behind the end every value is outside and comes as zero
        fa.fetch(c + BK, ra);
        fb.fetch(c + BK, rb);
        s16x8 vb[3][4];
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
            for (int w = 0; w < 4; ++w) vb[q][w] = *(const s16x8*)(lds.in.b + q * PLANE + piece_at(wj + w * 16 + (lane & 15), (lane >> 4) * 8));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            s16x8 va[3];
#pragma unroll
            for (int q = 0; q < 3; ++q) va[q] = *(const s16x8*)(lds.in.a + q * PLANE + piece_at(wi + u * 16 + (lane & 15), (lane >> 4) * 8));
            // B goes in as the instruction's first operand: a lane then holds four neighbouring j of one line i.  Small terms first.
#pragma unroll
            for (int term = 0; term < 6; ++term) {
                constexpr int PA[6] = {0, 2, 1, 0, 1, 0}, PB[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
                for (int w = 0; w < 4; ++w) acc[u][w] = mfma<bf16>(vb[PB[term]][w], va[PA[term]], acc[u][w]);
            }
        }
        // the next step is split in the shadow of the second half of the products
        total += fa.split(ra, sa);
        fb.split(rb, sb);
#pragma unroll
        for (int k = 0; k < 48; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
#pragma unroll
        for (int k = 0; k < 48; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
        }
    }
    __syncthreads();
    if (sums) {          // two lanes hold the halves of a line's sum
        lds.out[threadIdx.x] = total;
        __syncthreads();
        if (threadIdx.x < TILE && i0 + threadIdx.x < M) column_sums[(int64_t)blockIdx.y * M + i0 + threadIdx.x] = lds.out[threadIdx.x] + lds.out[threadIdx.x + TILE];
        __syncthreads();
    }
    store_wave<float, 4, 4>(E, acc, lds.out + wave * 64 * 64, i0 + wi, j0 + wj, M, N, [&](int64_t i, int64_t j, auto& z) {
        // a sum that is not finite is done again without the split, in fp32
#pragma unroll 1
        for (int k = 0; k < 4; ++k)
            if (!(fabsf(z[k]) < __builtin_inff()) && j + k < N) {
                float t = 0.f;
                for (int64_t c = c_begin; c < c_end; ++c) {
                    float a = ACOLS ? A.p[c * A.ld + i] : A.p[i * A.ld + c];
                    if (GATE) a *= ACOLS ? gate[c * ldgate + i] : gate[i * ldgate + c];
                    t = fmaf(a, BCOLS ? B.p[c * B.ld + j + k] : B.p[(j + k) * B.ld + c], t);
                }
                z[k] = t;
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

template <int LEFT> __device__ __forceinline__ void wait_and_meet() {
    // this wave's loads but for the last LEFT have arrived and its reads of LDS are done; then everybody's
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

template <typename T, bool ACOLS, bool BCOLS, int BM, int BN, int WM, int WN, int BUFFERS>
__global__ void __launch_bounds__(BM / WM * (BN / WN) * 64, BUFFERS == 2 ? 2 : 1) k_product16(Operand<T> A, Operand<T> B, int64_t M, int64_t N, int64_t lines_a, int64_t lines_b, int64_t K, int64_t slice, Epilogue<T> E) {
#if defined(__HIP_DEVICE_COMPILE__)          // the host pass has no type for a buffer's descriptor
    constexpr int THREADS = BM / WM * (BN / WN) * 64, TM = WM / 16, TN = WN / 16, PARTS = TM / 4, CLUSTERS = 2 * PARTS;
    // each buffer (A's tile, then B's) is a variable of its own: the compiler then knows which loads a read of LDS has to wait for
    constexpr int BUFFER = (BM + BN) * STEP;
    __shared__ __attribute__((aligned(1024))) short s0[BUFFER], s1[BUFFER], s2[BUFFERS > 2 ? BUFFER : 8], s3[BUFFERS > 2 ? BUFFER : 8];
    static_assert(BUFFERS == 2 || BUFFERS == 4, "buffers");
    uint32_t ti, tj;
    tile_of(blockIdx.x, (uint32_t)((M + BM - 1) / BM), (uint32_t)((N + BN - 1) / BN), ti, tj);
    const int64_t i0 = (int64_t)ti * BM, j0 = (int64_t)tj * BN;
    const int64_t c_begin = (int64_t)blockIdx.y * slice, len = (c_begin + slice < K ? c_begin + slice : K) - c_begin;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave / (BN / WN) * WM, wj = wave % (BN / WN) * WN;
    Feed<ACOLS, BM, THREADS> fa;
    Feed<BCOLS, BN, THREADS> fb;
    constexpr int LOADS = Feed<ACOLS, BM, THREADS>::LOADS + Feed<BCOLS, BN, THREADS>::LOADS;
    fa.init(A.p, A.ld, i0, lines_a, c_begin);
    fb.init(B.p, B.ld, j0, lines_b, c_begin);
    f32x4 acc[TM][TN] = {};
    s16x8 va[2][4], vb[2][TN];
    const int steps = (int)((len + STEP - 1) / STEP);
    int64_t left = len;
    const auto load = [&](short* s) __attribute__((always_inline)) {
        fa.load(s, left);
        fb.load(s + BM * STEP, left);
        left -= STEP;
    };
    // one cluster: 4 x TN products of half `ks`, part `part` of the wave's lines
    const auto read = [&](const short* s, int cluster) __attribute__((always_inline)) {
        const int ks = cluster / PARTS, part = cluster % PARTS;
#pragma unroll
        for (int u = 0; u < 4; ++u) va[cluster & 1][u] = fragment<ACOLS, BM>(s, wi + (part * 4 + u) * 16, ks);
        if (part == 0)
#pragma unroll
            for (int w = 0; w < TN; ++w) vb[ks][w] = fragment<BCOLS, BN>(s + BM * STEP, wj + w * 16, ks);
    };
    const auto multiply = [&](int cluster) __attribute__((always_inline)) {
        const int ks = cluster / PARTS, part = cluster % PARTS;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int w = 0; w < TN; ++w) acc[part * 4 + u][w] = mfma<T>(vb[ks][w], va[cluster & 1][u], acc[part * 4 + u][w]);
    };
    int k = 0;
    const auto step = [&](short* s, short* next) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c + 1 < CLUSTERS; ++c) {
            read(s, c + 1);
            multiply(c);
        }
        // the next step's tiles have arrived, and nobody reads this step's any more
        wait_and_meet<(BUFFERS - 2) * LOADS>();
        // With four buffers every step loads and reads ahead, behind the end too (nothing but zeros comes from there): without branches the compiler sees which loads a
        // read waits for.  With two it waits for all of them anyway, and the branches keep the loads in front of the last products.
        if (BUFFERS > 2 || ++k < steps) read(next, 0);
        if (BUFFERS > 2 || k + 1 < steps) load(s);
        multiply(CLUSTERS - 1);
    };
    load(s0);
    load(s1);
    if constexpr (BUFFERS > 2) {
        load(s2);
        load(s3);
    }
    wait_and_meet<(BUFFERS - 1) * LOADS>();
    read(s0, 0);
    if constexpr (BUFFERS == 2) {
        while (k < steps) {
            step(s0, s1);
            if (k < steps) step(s1, s0);
        }
    } else {
        for (; k + 4 <= steps; k += 4) {
            step(s0, s1);
            step(s1, s2);
            step(s2, s3);
            step(s3, s0);
        }
        if (k < steps) step(s0, s1);
        if (k + 1 < steps) step(s1, s2);
        if (k + 2 < steps) step(s2, s3);
    }
    wait_and_meet<0>();
    // nobody reads or loads tiles any more: the first two buffers hold the waves' sums
    static_assert(WN == 64 && BUFFER * 2 * 2 == THREADS / 64 * 64 * 64 * 4, "LDS for the sums");
    constexpr int SHARE = THREADS / 64 / 2;
    short* mine = wave < SHARE ? s0 : s1;
    store_wave<T, TM, (BUFFERS > 2 ? 8 : TM > 4 ? 2 : 4)>(E, acc, (float*)mine + wave % SHARE * 64 * 64, i0 + wi, j0 + wj, M, N, [](int64_t, int64_t, auto&) {});
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

// The slices of a contraction joined, then the epilogue.  `groups` lanes of a workgroup share the slices of four outputs in equal stretches, in their order.
template <typename T> __global__ void __launch_bounds__(256) k_join(const float* part, int splits, int groups, int64_t M, int64_t N, Epilogue<T> E) {
    constexpr int V = 4;
    __shared__ f32x4 sums[256];
    const int each = 256 / groups, group = threadIdx.x / each, x = threadIdx.x % each;
    const int64_t vectors = (N + V - 1) / V, at = (int64_t)blockIdx.x * each + x;
    const int share = (splits + groups - 1) / groups, s0 = group * share, s1 = s0 + share < splits ? s0 + share : splits;
    const bool ok = at < M * vectors;
    const int64_t i = ok ? at / vectors : 0, j = ok ? at % vectors * V : 0;
    float z[1][V] = {};
    if (ok)
        for (int s = s0; s < s1; s += 4) {
            float q[4][V];
#pragma unroll
            for (int k = 0; k < 4; ++k) load_some<float, V>(part + ((int64_t)(s + k) * M + i) * N + j, s + k < s1 ? N - j : 0, q[k]);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) z[0][e] += q[k][e];
        }
    if (groups > 1) {
        sums[threadIdx.x] = f32x4{z[0][0], z[0][1], z[0][2], z[0][3]};
        __syncthreads();
        if (group > 0) return;
        for (int g = 1; g < groups; ++g)
#pragma unroll
            for (int e = 0; e < V; ++e) z[0][e] += sums[g * each + x][e];
    }
    const int64_t line[1] = {i};
    if (ok) finish<T, V, 1>(E, line, j, M, N, z);
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
    int tile = TILE;                    // 256 or 128
    bool deep = false;                  // 128 with four buffers, one workgroup a compute unit, rather than two with two buffers each
    int64_t splits = 1, slice = 0;
    int64_t pack_a = 0, pack_b = 0;          // row strides of the repacked operands, 0: as they are
    int64_t at_a = 0, at_b = 0, at_part = 0, at_cols = 0, bytes = 0;
};
struct Line {          // an operand as the plan sees it
    const void* p;
    int64_t ld, cols;          // row stride, elements of a row that are read
    bool zeros;                // rows have zeros up to a multiple of 8 behind their ends
};
// The 16-bit kernels load 16 bytes at a time into LDS, by 31-bit offsets within a tile.
static bool direct(const Line& a) { return ((uintptr_t)a.p & 15) == 0 && a.ld % 8 == 0 && (a.cols % 8 == 0 || a.zeros) && a.ld < (1 << 21); }

static Plan plan(int es, Line a, int64_t rows_a, Line b, int64_t rows_b, int64_t M, int64_t N, int64_t K, bool column_sums = false) {
    Plan p;
    int64_t tiles = gs::cdiv(M, TILE) * gs::cdiv(N, TILE);
    if (es == 2) {
        const int64_t big = gs::cdiv(M, 256) * gs::cdiv(N, 256);
        if (big >= 192) p.tile = 256, tiles = big;
        if (!direct(a)) p.pack_a = up8(a.cols);
        if (!direct(b)) p.pack_b = up8(b.cols);
    }
    if (es == 2 && p.tile == 128) p.deep = tiles <= CUS;
    const int64_t slots = p.tile == 256 || p.deep ? CUS : 2 * CUS, least = p.deep ? 512 : 256;
    if (tiles < slots && K >= 2 * least) {
        p.splits = slots / tiles;
        if (p.splits > K / least) p.splits = K / least;
        if (p.splits > 256) p.splits = 256;
        if (p.splits < 1) p.splits = 1;
    }
    p.slice = p.splits > 1 ? gs::cdiv(gs::cdiv(K, p.splits), 64) * 64 : K;
    p.splits = p.splits > 1 ? gs::cdiv(K, p.slice) : 1;
    int64_t at = 0;
    p.at_a = at, at += p.pack_a ? align256(rows_a * p.pack_a * es) : 0;
    p.at_b = at, at += p.pack_b ? align256(rows_b * p.pack_b * es) : 0;
    p.at_part = at, at += p.splits > 1 ? align256(p.splits * M * N * 4) : 0;
    p.at_cols = at, at += column_sums ? align256(p.splits * M * 4) : 0;
    p.bytes = at;
    return p;
}

template <typename T> int pack(const void* p, int64_t ld, int64_t rows, int64_t cols, void* out, int64_t ldo, hipStream_t stream) {
    const int64_t blocks = gs::cdiv(rows * (ldo / 8), 256);
    GS_REQUIRE(blocks < (1ll << 31), "gs_linear: operand too large");
    hipLaunchKernelGGL(k_pack<T>, dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)p, ld, rows, cols, (T*)out, ldo);
    return 0;
}

// C [M,N] over a contraction of K.  fp32: A times `gate` (row stride ldgate), where there is one, and the sums of A's lines (dW only) to column_join.
template <typename T, bool ACOLS, bool BCOLS>
int product(Line a, Line b, int64_t M, int64_t N, int64_t K, Epilogue<T> E, void* workspace, int64_t workspace_bytes, hipStream_t stream, const float* gate = nullptr,
            int64_t ldgate = 0, T* column_join = nullptr) {
    if (M == 0 || N == 0) return 0;
    const int64_t rows_a = ACOLS ? K : M, rows_b = BCOLS ? K : N;
    const Plan p = plan(sizeof(T), a, rows_a, b, rows_b, M, N, K, column_join != nullptr);
    GS_REQUIRE(workspace_bytes >= p.bytes && (workspace || p.bytes == 0), "gs_linear: workspace too small");
    char* ws = (char*)workspace;
    const int64_t tiles = gs::cdiv(M, p.tile) * gs::cdiv(N, p.tile);
    GS_REQUIRE(tiles < (1ll << 31) && M * gs::cdiv(N, 4) < (31ll << 31), "gs_linear: too many tiles");
    Epilogue<T> first = E;
    first.part = p.splits > 1 ? (float*)(ws + p.at_part) : nullptr;
    const dim3 grid((unsigned)tiles, (unsigned)p.splits);
    if constexpr (sizeof(T) == 4) {
        const Operand<float> A{(const float*)a.p, a.ld}, B{(const float*)b.p, b.ld};
        float* cols = column_join ? (float*)(ws + p.at_cols) : nullptr;
        if (gate) hipLaunchKernelGGL((k_product32<ACOLS, BCOLS, true>), grid, dim3(256), 0, stream, A, gate, ldgate, B, M, N, K, p.slice, first, cols);
        else hipLaunchKernelGGL((k_product32<ACOLS, BCOLS, false>), grid, dim3(256), 0, stream, A, gate, ldgate, B, M, N, K, p.slice, first, cols);
        if (cols) hipLaunchKernelGGL(k_column_join<T>, dim3((unsigned)gs::cdiv(M, 32)), dim3(1024), 0, stream, (const float*)cols, (int)p.splits, M, column_join);
    } else {
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
            hipLaunchKernelGGL((k_product16<T, ACOLS, BCOLS, 256, 256, 128, 64, 2>), grid, dim3(512), 0, stream, A, B, M, N, lines_a, lines_b, K, p.slice, first);
        else if (p.deep)
            hipLaunchKernelGGL((k_product16<T, ACOLS, BCOLS, 128, 128, 64, 64, 4>), grid, dim3(256), 0, stream, A, B, M, N, lines_a, lines_b, K, p.slice, first);
        else
            hipLaunchKernelGGL((k_product16<T, ACOLS, BCOLS, 128, 128, 64, 64, 2>), grid, dim3(256), 0, stream, A, B, M, N, lines_a, lines_b, K, p.slice, first);
    }
    if (p.splits > 1) {
        const int groups = p.splits >= 32 ? 16 : p.splits >= 8 ? 4 : 1;
        hipLaunchKernelGGL(k_join<T>, dim3((unsigned)gs::cdiv(M * gs::cdiv(N, 4), 256 / groups)), dim3(256), 0, stream, (const float*)(ws + p.at_part), (int)p.splits, groups, M, N, E);
    }
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
    bool gz_made, pass, sums_with_w;          // gz has a place of its own; a pass over g is made; db comes with dW
    int64_t ldgz, slab, slabs;
    int64_t gz, cols, prod, total;          // byte offsets of gz, the column sums' slabs and the products' workspace
};
static BackwardPlan backward_plan(const void* g, int64_t ldg, bool has_dact, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, int es,
                                  bool want_x, bool want_w, bool want_b) {
    BackwardPlan p;
    // fp32 products take the gate as they load g, and the sums with dW; 16-bit ones read gz from memory
    p.gz_made = es == 2 && (want_x || want_w) && (has_dact || !direct({g, ldg, N, false}));
    p.sums_with_w = es == 4 && want_w && want_b && K > 0;
    p.pass = p.gz_made || (want_b && !p.sums_with_w);
    p.ldgz = p.gz_made ? up8(N) : ldg;
    const int64_t across = gs::cdiv(N, GZ_LANES * 16 / es);
    p.slab = gs::cdiv(gs::cdiv(M * across, 2048), GZ_LINES) * GZ_LINES;
    if (p.slab < 64) p.slab = 64;
    if (M / p.slab >= 65535) p.slab = gs::cdiv(M, 65535);
    p.slabs = gs::cdiv(M, p.slab);
    p.gz = 0;
    p.cols = p.gz + (p.gz_made ? align256(M * p.ldgz * es) : 0);
    p.prod = p.cols + (want_b && !p.sums_with_w ? align256(p.slabs * N * 4) : 0);
    const Line gl{p.gz_made ? nullptr : g, p.ldgz, N, p.gz_made};
    int64_t b = 0;
    if (want_x) b = plan(es, gl, M, {w, ldw, K, false}, N, M, K, N).bytes;
    if (want_w) {
        const int64_t c = plan(es, gl, M, {x, ldx, K, false}, M, N, K, M, p.sums_with_w).bytes;
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
        float* part = db && !p.sums_with_w ? (float*)(base + p.cols) : nullptr;
        const int64_t across = gs::cdiv(N, GZ_LANES * width<T>());
        if (M > 0)
            hipLaunchKernelGGL(k_gz<T>, dim3((unsigned)across, (unsigned)p.slabs), dim3(256), 0, stream, (const T*)g, ldg, (const typename dact_type<T>::type*)dact, M, N, p.slab,
                               p.gz_made ? (T*)(base + p.gz) : nullptr, p.ldgz, part);
        if (db && !p.sums_with_w) hipLaunchKernelGGL(k_column_join<T>, dim3((unsigned)gs::cdiv(N, 32)), dim3(1024), 0, stream, (const float*)part, (int)p.slabs, N, (T*)db);
        GS_LAUNCH_CHECK();
    }
    Epilogue<T> E{};
    const float* gate = sizeof(T) == 4 ? (const float*)dact : nullptr;
    int rc = 0;
    if (dx) {
        E.out = (T*)dx, E.ldo = K;
        rc = product<T, false, true>(gz, {w, ldw, K, false}, M, K, N, E, base + p.prod, ws_bytes - p.prod, stream, gate, N);
    }
    if (!rc && dw) {
        E.out = (T*)dw, E.ldo = K;
        rc = product<T, true, true>(gz, {x, ldx, K, false}, N, K, M, E, base + p.prod, ws_bytes - p.prod, stream, gate, N, p.sums_with_w ? (T*)db : nullptr);
    }
    return rc;
}

// 16-bit tiles are addressed by 31-bit offsets: 256 rows of 2^21 elements fit
static bool sizes_ok(int64_t M, int64_t N, int64_t K, int dtype) {
    const int64_t top = 1ll << 31, wide = dtype == DT_F32 ? top : 1ll << 21;
    return M >= 0 && N >= 0 && K >= 0 && M < top && N < wide && K < wide;
}

}  // namespace

extern "C" int64_t gs_linear_fwd_workspace_bytes(const void* x, int64_t ldx, const void* weight, int64_t ldw, int64_t M, int64_t N, int64_t K, int dtype) {
    if (dtype < 0 || dtype > 2 || !sizes_ok(M, N, K, dtype)) return -1;
    return M == 0 || N == 0 ? 0 : plan(dtype == DT_F32 ? 4 : 2, {x, ldx, K, false}, M, {weight, ldw, K, false}, N, M, N, K).bytes;
}

extern "C" int gs_linear_fwd(const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* bias, const void* residual, int64_t ldr, int64_t M, int64_t N,
                             int64_t K, int dtype, int act, float beta, void* y, int64_t ldy, void* dact, void* workspace, int64_t workspace_bytes, gs_stream_t stream) {
    GS_REQUIRE(dtype >= 0 && dtype <= 2, "gs_linear_fwd: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    GS_REQUIRE(sizes_ok(M, N, K, dtype), "gs_linear_fwd: sizes are 0 .. 2^31 - 1, of 16-bit rows 0 .. 2^21 - 1");
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
    if (dtype < 0 || dtype > 2 || !sizes_ok(M, N, K, dtype)) return -1;
    return backward_plan(g, ldg, has_dact, x, ldx, weight, ldw, M, N, K, dtype == DT_F32 ? 4 : 2, want_x, want_w, want_b).total;
}

extern "C" int gs_linear_bwd(const void* g, int64_t ldg, const void* dact, const void* x, int64_t ldx, const void* weight, int64_t ldw, int64_t M, int64_t N, int64_t K,
                             int dtype, void* dx, void* dw, void* db, void* workspace, int64_t workspace_bytes, gs_stream_t stream) {
    GS_REQUIRE(dtype >= 0 && dtype <= 2, "gs_linear_bwd: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    GS_REQUIRE(sizes_ok(M, N, K, dtype), "gs_linear_bwd: sizes are 0 .. 2^31 - 1, of 16-bit rows 0 .. 2^21 - 1");
    GS_REQUIRE(M == 0 || N == 0 || (g && ldg >= 0), "gs_linear_bwd: null gradient");
    GS_REQUIRE(M == 0 || N == 0 || K == 0 || ((!dx || weight) && (!dw || x)), "gs_linear_bwd: null operand");
    const auto run = dtype == DT_F32 ? linear_bwd<float> : dtype == DT_BF16 ? linear_bwd<bf16> : linear_bwd<f16>;
    return run(g, ldg, dact, x, ldx, weight, ldw, M, N, K, dx, dw, db, workspace, workspace_bytes, (hipStream_t)stream);
}

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
// 2^-25 |x y| each.  That is 1 / 6 of the bf16 rate, where the fp32 matrix instruction has 1 / 16.  An infinity has no such split (inf * 0): a sum
// that comes out non-finite is done again with the fp32 matrix instruction (nothing but NaN takes 4 .. 11 times an ordinary product: y of 131072 x 256 x 256 0.6 ms, of
// 8192 x 4096 x 4096 8.3 ms; a sum a lane took 100 times).  The matrix cores take parts below 2^-126 as zero: operands
// below 2^-112 keep fewer bits, 2^-17 at 2^-118.
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

// act'(z) as the forward pass keeps it for the backward pass: fp32 for fp16 and fp32 layers (one more rounding to the layer's own type would cost the gradients as much as their
// own), 16 bits for bf16 layers.  |act'| <= 1.13, so down to 2^-14 these are fp16's, 11 bits next to bf16's 8, and down to 2^-17 its subnormals, 8 bits and more; fp16's codes of 2
// and above, which no derivative needs, hold the smaller ones as bf16 does, 8 bits down to 2^-126: in fp16 itself they would be zero below 2^-25 (softplus at beta z = -17.3).
//   |v| >= 2^-17, NaN: the fp16 of v        smaller: sign, 0x4000 | bf16 of |v| (at most 0x3700: no bit is in the other's place)
struct Slope16 {
    uint16_t bits;
    Slope16() = default;
    __device__ __forceinline__ explicit Slope16(float v) {
        const uint16_t small = __builtin_bit_cast(uint16_t, (bf16)v) | 0x4000, large = __builtin_bit_cast(uint16_t, (f16)v);
        bits = fabsf(v) < 0x1p-17f ? small : large;
    }
    __device__ __forceinline__ explicit operator float() const {
        const uint32_t small = (uint32_t)(bits & 0xbfff) << 16;
        return (uint16_t)((bits & 0x7fff) - 0x4000) < 0x3c00 ? __builtin_bit_cast(float, small) : (float)__builtin_bit_cast(f16, bits);
    }
};
template <typename T> struct dact_type { typedef float type; };
template <> struct dact_type<bf16> { typedef Slope16 type; };

template <typename T> __device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma<f16>(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// g act'(z).  Where the derivative is exactly zero nothing passes, an infinity or NaN neither.
__device__ __forceinline__ float gated(float g, float d) { return d == 0.f ? 0.f : g * d; }

// Value and derivative of the activation, on the hardware's exp2, log2 and reciprocal (1 ulp each).  For fp32 what rounds the exponent's product goes into the exponential as a
// factor and erfc is the library's; 16-bit layers (FAST) do without the factor (2^-24 |exponent|) and have a fitted erfc (act_gelu).
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
// softplus's constants: log2(e) beta in two parts (48 bits), 2 / beta
struct Beta {
    float log2e, low, two_over;
};
// With t = exp(-|beta z|) in [0, 1] (neither end of z overflows): log(1 + t) = 2 artanh(q), q = t / (2 + t) <= 1/3, as q times a polynomial in q^2 (fitted at Chebyshev's
// points, relative error 8e-9), and one reciprocal of (1 + t)(2 + t) serves that and the derivative.  Where p is infinite r is nonsense, but t is zero.
template <bool FAST> __device__ __forceinline__ void act_softplus(const Beta& beta, float z, float& y, float& d) {
    const float a = fabsf(z), p = beta.log2e * a;
    float t = __builtin_amdgcn_exp2f(-p);
    if (!FAST) {
        const float r = __builtin_fmaf(a, beta.low, __builtin_fmaf(a, beta.log2e, -p));
        t = __builtin_fmaf(t, __builtin_amdgcn_fmed3f(r * -0.69314718f, -1.f, 1.f), t);
    }
    const float u = 1.f + t, v = 2.f + t, k = rcp_(u * v), q = t * (k * u), w = q * q;
    const float s = fmaf(fmaf(fmaf(fmaf(0.14087328f, w, 0.13980709f), w, 0.20012426f), w, 0.33333158f), w, 1.f);
    y = fmaf(q * s, beta.two_over, fmaxf(z, 0.f));
    d = (z >= 0.f ? 1.f : t) * (k * v);
}
template <bool FAST> __device__ __forceinline__ void act_silu(float z, float& y, float& d) {
    const float s = rcp_(1.f + exp_<FAST>(-z));
    y = z * s;
    d = s * fmaf(z, 1.f - s, 1.f);
}
// FAST: Phi(-|z|) = exp(-z^2 / 2) t q(t), t = 1 / (1 + 0.415 |z| / sqrt 2), q a polynomial of degree 5 fitted to erfcx (the least largest error): 1e-7 off at most, 2.4e-7 with its
// roundings, and 4e-5 of itself (fp16's half step is 2^-11), however far the tail, down to the exponential's end at z = -13
template <bool FAST> __device__ __forceinline__ void act_gelu(float z, float& y, float& d) {
    const float e = exp_<FAST>(-0.5f * z * z);
    float phi;
    if (FAST) {
        const float t = rcp_(fmaf(0.415f * 0.70710678f, fabsf(z), 1.f));
        float c = -0.08539501f;
        for (const float k : {0.26145714f, -0.065672984f, 0.16594572f, 0.105752f, 0.11791308f}) c = fmaf(c, t, k);
        c *= e * t;
        phi = z < 0.f ? c : 1.f - c;
    } else {
        phi = 0.5f * erfcf(z * -0.70710678118654752f);
    }
    y = z * phi;
    d = fmaf(z, e * 0.39894228040143268f, phi);
}
// BATCH x V values at once: the choice is the same for the whole launch
template <bool FAST, int V, int BATCH> __device__ __forceinline__ void act_eval(int act, const Beta& beta, float (&z)[BATCH][V], float (&d)[BATCH][V]) {
    switch (act) {
        case ACT_RELU:
#pragma unroll
            for (int k = 0; k < V * BATCH; ++k) act_relu<FAST>(z[k / V][k % V], z[k / V][k % V], d[k / V][k % V]);
            break;
        case ACT_SOFTPLUS:
#pragma unroll
            for (int k = 0; k < V * BATCH; ++k) act_softplus<FAST>(beta, z[k / V][k % V], z[k / V][k % V], d[k / V][k % V]);
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
    Beta beta;          // of softplus
};

template <typename T, int V> struct __attribute__((packed)) Pack { T v[V]; };          // rows start at any element: the hardware takes unaligned vectors

template <typename T> constexpr int width() { return 16 / (int)sizeof(T); }

// V neighbouring values, of which the first `in_row` are in the row.  Others repeat the row's last one in the load, so that a row's end costs one branch and one wait
// (83195 x 62 -> 103 bf16 with gelu and residual, a step: 134 us for 163).
template <typename T, int V> __device__ __forceinline__ void load_some(const T* p, int64_t in_row, float (&v)[V]) {
    if (in_row >= V) {
        const Pack<T, V> q = *(const Pack<T, V>*)p;
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = (float)q.v[k];
    } else if (in_row > 0) {
        const int n = (int)in_row;
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = (float)p[k < n ? k : n - 1];
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = k < n ? v[k] : 0.f;
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = 0.f;
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
// BATCH x V outputs of the lines i, i + step, .. (those below M), columns j ..; q: their columns' bias.  ALL: every one of them is in the output.
template <typename T, int V, int BATCH, bool ALL = false>
__device__ __forceinline__ void finish(const Epilogue<T>& E, int64_t i, int64_t step, int64_t j, int64_t M, int64_t N, float (&z)[BATCH][V], const float (&q)[V]) {
    const int64_t in_row = ALL ? V : N - j;
    const auto in = [&](int b) __attribute__((always_inline)) { return ALL || i + b * step < M; };
    float r[BATCH][V];
    if (E.res) {
        const T* p = E.res + i * E.ldr + j;
#pragma unroll
        for (int b = 0; b < BATCH; ++b) load_some<T, V>(p + b * (step * E.ldr), in(b) ? in_row : 0, r[b]);
    }
    if (E.bias)
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
#pragma unroll
            for (int k = 0; k < V; ++k) z[b][k] += q[k];
    if (E.act != ACT_NONE) {
        float d[BATCH][V];
        act_eval<sizeof(T) == 2, V, BATCH>(E.act, E.beta, z, d);
        if (E.dact) {
            auto* p = E.dact + i * N + j;
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
                if (in(b)) store_some<typename dact_type<T>::type, V>(p + b * (step * N), in_row, d[b]);
        }
    }
    T* p = E.out + i * E.ldo + j;
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
        if (E.res)
#pragma unroll
            for (int k = 0; k < V; ++k) z[b][k] += r[b][k];
        if (in(b)) store_some<T, V>(p + b * (step * E.ldo), in_row, z[b]);
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

// A wave's sums go to memory through 16 KB of LDS, 64 x 64 at a time: the lanes then hold 16 bytes of neighbouring outputs each, and 8 (16-bit) or 16 (fp32) lanes a whole
// line of 64.  The 16-byte piece p of line l is kept at p ^ (l & 15).
__device__ __forceinline__ int piece_of_sums(int line, int piece) { return line * 64 + (piece ^ (line & 15)) * 4; }
template <int TM> __device__ __forceinline__ void put_sums(const f32x4 (&acc)[TM][4], int first, float* lds) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) *(f32x4*)(lds + piece_of_sums(u * 16 + (lane & 15), w * 4 + (lane >> 4))) = acc[first + u][w];
}
// Lines l_begin .. l_end of them, BATCH lines a lane side by side, as many as the registers hold (one with tiles of 256): what they read of the residual is in flight together.
// A stretch inside of the output goes without checks (131072 x 256 x 256 fp32: y with softplus 164 us for 170, dx 156 for 165, dW 131 for 134).
template <typename T, int BATCH, bool ALL>
__device__ __forceinline__ void drain_lines(const Epilogue<T>& E, const float* lds, int l_begin, int l_end, int64_t i0, int64_t j, int64_t M, int64_t N, const float (&q)[width<T>()]) {
    constexpr int V = width<T>(), LANES = 64 / V, LINES = 64 / LANES;
    const int lane = threadIdx.x & 63, c = lane % LANES * V;
#pragma unroll 1
    for (int l0 = l_begin; l0 < l_end; l0 += LINES * BATCH) {
        float z[BATCH][V];
        const int64_t i = i0 + l0 + lane / LANES;
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int l = l0 + b * LINES + lane / LANES;
#pragma unroll
            for (int k = 0; k < V; k += 4) {
                const f32x4 s = *(const f32x4*)(lds + piece_of_sums(l, (c + k) >> 2));
#pragma unroll
                for (int e = 0; e < 4; ++e) z[b][k + e] = s[e];
            }
        }
        if (E.part) {
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
                if (ALL || i + b * LINES < M) store_some<float, V>(E.part + ((int64_t)blockIdx.y * M + i + b * LINES) * N + j, ALL ? V : N - j, z[b]);
        } else {
            finish<T, V, BATCH, ALL>(E, i, LINES, j, M, N, z, q);
        }
    }
}
template <typename T, int BATCH>
__device__ __forceinline__ void drain_sums(const Epilogue<T>& E, const float* lds, int l_begin, int l_end, int64_t i0, int64_t j0, int64_t M, int64_t N) {
    constexpr int V = width<T>(), LANES = 64 / V;
    const int64_t j = j0 + (threadIdx.x & 63) % LANES * V;
    float q[V] = {};
    if (j >= N) return;
    if (E.bias && !E.part) load_some<T, V>(E.bias + j, N - j, q);
    if (i0 + l_end <= M && j0 + 64 <= N) drain_lines<T, BATCH, true>(E, lds, l_begin, l_end, i0, j, M, N, q);
    else drain_lines<T, BATCH, false>(E, lds, l_begin, l_end, i0, j, M, N, q);
}
template <typename T, int TM, int BATCH>
__device__ __forceinline__ void store_wave(const Epilogue<T>& E, const f32x4 (&acc)[TM][4], float* lds, int64_t i0, int64_t j0, int64_t M, int64_t N) {
#pragma unroll 1
    for (int part = 0; part < TM / 4; ++part) {
#pragma unroll
        for (int p = 0; p < TM / 4; ++p)
            if (p == part) put_sums<TM>(acc, 4 * p, lds);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        drain_sums<T, BATCH>(E, lds, 0, 64, i0 + part * 64, j0, M, N);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// Sums of columns by slabs of rows, joined: 32 columns a workgroup, the slabs in stretches side by side, in their order.  Done by workgroups that a later launch has
// beside its own.
template <typename T> struct Columns {
    const float* part;          // [slabs][N]
    T* db;
    int64_t N;
    int slabs;
    uint32_t blocks;
};
template <typename T> __device__ __forceinline__ void join_columns(const Columns<T>& C, uint32_t block, float* lds) {
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, groups = blockDim.x >> 5;
    const int64_t j = (int64_t)block * 32 + x;
    const int share = (C.slabs + groups - 1) / groups, k0 = y * share, k1 = k0 + share < C.slabs ? k0 + share : C.slabs;
    float s = 0.f;
    if (j < C.N) {
        int k = k0;
        for (; k + 8 <= k1; k += 8) {
            float q[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) q[e] = C.part[(int64_t)(k + e) * C.N + j];
#pragma unroll
            for (int e = 0; e < 8; ++e) s += q[e];
        }
        for (; k < k1; ++k) s += C.part[(int64_t)k * C.N + j];
    }
    lds[y * 33 + x] = s;
    __syncthreads();
    if (y == 0 && j < C.N) {
        float t = 0.f;
        for (int q = 0; q < groups; ++q) t += lds[q * 33 + x];
        C.db[j] = (T)t;
    }
}

// ---- fp32 products ------------------------------------------------------------------------------------------------------------------------------------
// Tiles of LINES x LINES, 32 of the contraction a step.  128: two workgroups a compute unit, a wave multiplies 64 x 64 (96 matrix instructions a step against 24 fragments read and
// 32 values split a lane); 64: up to four, a wave 32 x 32, for products that have few tiles.  While a step is multiplied the next one comes to registers and is split there; each
// of the three parts has a plane of its own in LDS: [line][32], 4 pieces of 16 bytes a line, piece p of line l at p ^ (l >> 1 & 3), so that the 16 lines of a fragment
// fall on distinct banks.
//   rows operand     a lane loads 8 neighbours of the contraction at a time; columns operand: 16 or 8 of one line, neighbouring lanes neighbouring lines
// A may have a gate: the factor act'(z) that makes gz of g, so that gz is never stored; the products with dW also add up its columns, for db.
// 131072 x 256 x 256: y 107 us (161 Tflop/s; the library's fp32 product 155), with softplus and act' kept 164; dx 114 (154), with a gate 156; dW 107 (319), with a gate and db 131.
// 4096 x 4096 x 4096: 780, 660, 680 us (1040); 512 x 512 x 512 11, 12, 12 (20).  At 131072 rows memory needs 52 .. 78 us and the matrix cores 60; both, the splitting and the epilogue (45 us of dx, 71 of y with
// softplus, by leaving it out) share a compute unit and overlap in part.  Tried and left: the weight's parts made once by a launch of their own and loaded straight into LDS, 165
// + 5 us of 184 for dx and 180 + 5 of 184 for y; workgroups that start a quarter of a tile apart, no change.
constexpr int TILE = 128, BK = 32;

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

template <bool COLS, bool GATE, int LINES> struct Feed32 {
    static constexpr int THREADS = 256, PIECES = LINES * BK / THREADS / 8;          // of 8 neighbours, a lane and step
    static constexpr int PLANE = LINES * BK;
    const float *p, *gate;
    int64_t ld, ldgate, line0, lines, c_end;
    bool whole;                    // every line of the tile is in the operand
    struct Values { float v[8 * PIECES], d[GATE ? 8 * PIECES : 1]; };          // in flight
    struct Parts { u32x4 p[3][PIECES]; };
    // the line and the first index of the lane's piece `h`
    static __device__ __forceinline__ int line_of(int h) { return COLS ? threadIdx.x % LINES : h * (THREADS / 4) + (threadIdx.x >> 2); }
    static __device__ __forceinline__ int at_of(int h) { return COLS ? (threadIdx.x / LINES * PIECES + h) * 8 : (threadIdx.x & 3) * 8; }
    __device__ __forceinline__ void fetch(int64_t c, Values& V) const {
        const bool all = whole && c + BK <= c_end;
        if constexpr (!COLS) {
            const auto some = [&](auto left_of) __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < PIECES; ++h) {
                    const int64_t l = line0 + line_of(h), at = c + at_of(h), left = left_of(l, at);
#pragma unroll
                    for (int k = 0; k < 8; k += 4) {
                        load_some<float, 4>(p + l * ld + at + k, left - k, *(float(*)[4])(V.v + 8 * h + k));
                        if constexpr (GATE) load_some<float, 4>(gate + l * ldgate + at + k, left - k, *(float(*)[4])(V.d + 8 * h + k));
                    }
                }
            };
            if (all) some([](int64_t, int64_t) { return (int64_t)8; });
            else some([&](int64_t l, int64_t at) { return l < lines ? c_end - at : 0; });
        } else {
            const int64_t at = c + __builtin_amdgcn_readfirstlane(at_of(0));          // the same for a wave
            const uint32_t l = threadIdx.x % LINES;
            const float* q = p + at * ld + line0;
            const float* e = GATE ? gate + at * ldgate + line0 : nullptr;
            if (all) {
#pragma unroll
                for (int k = 0; k < 8 * PIECES; ++k) {
                    V.v[k] = q[l];
                    q += ld;
                    if constexpr (GATE) V.d[k] = e[l], e += ldgate;
                }
            } else {
                // what is outside repeats the last line, the last of the contraction, and becomes zero
                const uint32_t n = lines - line0 < LINES ? (uint32_t)(lines - line0) : LINES, in = l < n ? l : n - 1;
                const int64_t left = c_end - at;
#pragma unroll
                for (int k = 0; k < 8 * PIECES; ++k) {
                    const int64_t row = k < left ? k : left - 1;
                    V.v[k] = q[row * ld + in];
                    if constexpr (GATE) V.d[k] = e[row * ldgate + in];
                }
#pragma unroll
                for (int k = 0; k < 8 * PIECES; ++k) {
                    const bool ok = l < n && k < left;
                    V.v[k] = ok ? V.v[k] : 0.f;
                    if constexpr (GATE) V.d[k] = ok ? V.d[k] : 0.f;
                }
            }
        }
    }
    // split; returns the sum of the values (of one line, for columns operands)
    __device__ __forceinline__ float split(const Values& V, Parts& S) const {
        float t = 0.f;
#pragma unroll
        for (int h = 0; h < PIECES; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float x = V.v[8 * h + 2 * k], y = V.v[8 * h + 2 * k + 1];
                if constexpr (GATE) x *= V.d[8 * h + 2 * k], y *= V.d[8 * h + 2 * k + 1];
                if constexpr (COLS) t += x + y;
                uint32_t part[3];
                split2(x, y, part);
#pragma unroll
                for (int q = 0; q < 3; ++q) S.p[q][h][k] = part[q];
            }
        return t;
    }
    __device__ __forceinline__ void store(short* lds, const Parts& S) const {
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
            for (int h = 0; h < PIECES; ++h) *(u32x4*)(lds + q * PLANE + piece_at(line_of(h), at_of(h))) = S.p[q][h];
    }
};

// The sums of 16 x 16 outputs (i, j ..) by the fp32 matrix instruction, straight from memory, 64 of the contraction on their way at a time; what is outside counts as zero.  A
// function of its own, called where there are infinities or NaN: its registers are not the products'.
template <bool COLS> __device__ __forceinline__ void load_line(const float* p, int64_t ld, int64_t line, int64_t lines, int64_t c, int64_t c_end, float (&v)[4]) {
    if constexpr (!COLS) {
        load_some<float, 4>(p + line * ld + c, line < lines ? c_end - c : 0, v);
    } else {          // what is outside repeats the last of the contraction or the last line in the load
        const float* q = p + (line < lines ? line : lines - 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = q[(c + e < c_end ? c + e : c_end - 1) * ld];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = line < lines && c + e < c_end ? v[e] : 0.f;
    }
}
template <bool ACOLS, bool BCOLS, bool GATE>
__device__ __noinline__ f32x4 plain_sums(Operand<float> A, const float* gate, int64_t ldgate, Operand<float> B, int64_t i, int64_t j, int64_t M, int64_t N, int64_t c_begin, int64_t c_end) {
    constexpr int U = 4;
    const int lane = threadIdx.x & 63;
    i += lane & 15, j += lane & 15;
    f32x4 sum = {};
    for (int64_t c = c_begin; c < c_end; c += 16 * U) {
        float a[U][4], b[U][4], d[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = c + u * 16 + (lane >> 4) * 4;
            load_line<ACOLS>(A.p, A.ld, i, M, k, c_end, a[u]);
            if (GATE) load_line<ACOLS>(gate, ldgate, i, M, k, c_end, d[u]);
            load_line<BCOLS>(B.p, B.ld, j, N, k, c_end, b[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(b[u][e], GATE ? gated(a[u][e], d[u][e]) : a[u][e], sum, 0, 0, 0);
    }
    return sum;
}

template <bool ACOLS, bool BCOLS, bool GATE, int LINES>
__global__ void __launch_bounds__(256, LINES == 64 ? 4 : 2) k_product32(Operand<float> A, const float* gate, int64_t ldgate, Operand<float> B, int64_t M, int64_t N, int64_t K, int64_t slice,
                                                                       Epilogue<float> E, float* column_sums /* [slices][M], or db itself where there is one slice */) {
    constexpr int F = LINES / 32, PLANE = LINES * BK;          // fragments of a wave, either way
    __shared__ __attribute__((aligned(16))) union {
        struct { short a[3 * PLANE], b[3 * PLANE]; } in;
        float out[LINES * LINES];
    } lds;
    uint32_t ti, tj;
    tile_of(blockIdx.x, (uint32_t)((M + LINES - 1) / LINES), (uint32_t)((N + LINES - 1) / LINES), ti, tj);
    const int64_t i0 = (int64_t)ti * LINES, j0 = (int64_t)tj * LINES;
    const int64_t c_begin = (int64_t)blockIdx.y * slice, c_end = c_begin + slice < K ? c_begin + slice : K;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = (wave >> 1) * (LINES / 2), wj = (wave & 1) * (LINES / 2);
    typedef Feed32<ACOLS, GATE, LINES> FA;
    typedef Feed32<BCOLS, false, LINES> FB;
    FA fa;
    FB fb;
    fa.p = A.p, fa.ld = A.ld, fa.gate = gate, fa.ldgate = ldgate, fa.line0 = i0, fa.lines = M, fa.c_end = c_end, fa.whole = i0 + LINES <= M;
    fb.p = B.p, fb.ld = B.ld, fb.line0 = j0, fb.lines = N, fb.c_end = c_end, fb.whole = j0 + LINES <= N;
    const bool sums = ACOLS && column_sums && tj == 0;
    float total = 0.f;
    f32x4 acc[F][F] = {};
    typename FA::Values ra;
    typename FB::Values rb;
    typename FA::Parts sa;
    typename FB::Parts sb;
    // With two workgroups a unit the next step is split among the second half of the products; with four or more right before it is stored
    constexpr bool AHEAD = LINES == 128;
    const auto split = [&]() __attribute__((always_inline)) {
        total += fa.split(ra, sa);
        fb.split(rb, sb);
    };
    if (c_begin < c_end) {
        fa.fetch(c_begin, ra);
        fb.fetch(c_begin, rb);
        if (AHEAD) split();
    }
    for (int64_t c = c_begin; c < c_end; c += BK) {
        __syncthreads();
        if (!AHEAD) split();
        fa.store(lds.in.a, sa);
        fb.store(lds.in.b, sb);
        __syncthreads();
        // behind the end every value is outside and comes as zero
        fa.fetch(c + BK, ra);
        fb.fetch(c + BK, rb);
        s16x8 vb[3][F];
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
            for (int w = 0; w < F; ++w) vb[q][w] = *(const s16x8*)(lds.in.b + q * PLANE + piece_at(wj + w * 16 + (lane & 15), (lane >> 4) * 8));
#pragma unroll
        for (int u = 0; u < F; ++u) {
            s16x8 va[3];
#pragma unroll
            for (int q = 0; q < 3; ++q) va[q] = *(const s16x8*)(lds.in.a + q * PLANE + piece_at(wi + u * 16 + (lane & 15), (lane >> 4) * 8));
            // B goes in as the instruction's first operand: a lane then holds four neighbouring j of one line i.  Small terms first.
#pragma unroll
            for (int term = 0; term < 6; ++term) {
                constexpr int PA[6] = {0, 2, 1, 0, 1, 0}, PB[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
                for (int w = 0; w < F; ++w) acc[u][w] = mfma<bf16>(vb[PB[term]][w], va[PA[term]], acc[u][w]);
            }
        }
        if constexpr (AHEAD) {
            split();
#pragma unroll
            for (int q = 0; q < 3 * F * F; ++q) {
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            }
#pragma unroll
            for (int q = 0; q < 3 * F * F; ++q) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
            }
        }
    }
    __syncthreads();
    if (sums) {          // 256 / LINES lanes hold parts of a line's sum
        lds.out[threadIdx.x] = total;
        __syncthreads();
        if (threadIdx.x < LINES && i0 + threadIdx.x < M) {
            float t = 0.f;
#pragma unroll
            for (int q = 0; q < 256 / LINES; ++q) t += lds.out[threadIdx.x + q * LINES];
            if (GATE && !(fabsf(t) < __builtin_inff())) {          // again, as gated() has it
                t = 0.f;
                const float *p = A.p + i0 + threadIdx.x, *d = gate + i0 + threadIdx.x;
                for (int64_t c = c_begin; c < c_end; c += 8) {
                    float v[8], e[8];
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const int64_t k = c + q < c_end ? c + q : c_end - 1;
                        v[q] = p[k * A.ld], e[q] = d[k * ldgate];
                    }
#pragma unroll
                    for (int q = 0; q < 8; ++q) t += c + q < c_end ? gated(v[q], e[q]) : 0.f;
                }
            }
            column_sums[(int64_t)blockIdx.y * M + i0 + threadIdx.x] = t;
        }
        __syncthreads();
    }
    // sums that are not finite are done again without the split, 16 x 16 of them a time, and with gated()
    float all = 0.f;
#pragma unroll
    for (int u = 0; u < F; ++u)
#pragma unroll
        for (int w = 0; w < F; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e) all = __builtin_fmaf(acc[u][w][e], 0.f, all);          // zero, or NaN
    if (__ballot(all != 0.f))
#pragma unroll
        for (int u = 0; u < F; ++u)
#pragma unroll
            for (int w = 0; w < F; ++w) {
                bool bad = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) bad |= !(fabsf(acc[u][w][e]) < __builtin_inff());
                if (!__ballot(bad)) continue;
                const f32x4 again = plain_sums<ACOLS, BCOLS, GATE>(A, gate, ldgate, B, i0 + wi + u * 16, j0 + wj + w * 16, M, N, c_begin, c_end);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[u][w][e] = fabsf(acc[u][w][e]) < __builtin_inff() ? acc[u][w][e] : again[e];
            }
    if constexpr (LINES == 128) {
        store_wave<float, 4, 4>(E, acc, lds.out + wave * 64 * 64, i0 + wi, j0 + wj, M, N);
    } else {          // the four waves' sums side by side, then 16 lines each
#pragma unroll
        for (int u = 0; u < F; ++u)
#pragma unroll
            for (int w = 0; w < F; ++w) *(f32x4*)(lds.out + piece_of_sums(wi + u * 16 + (lane & 15), wj / 4 + w * 4 + (lane >> 4))) = acc[u][w];
        __syncthreads();
        drain_sums<float, 4>(E, lds.out, wave * 16, wave * 16 + 16, i0, j0, M, N);
    }
}

// ---- 16-bit products with tiles fed straight into LDS ---------------------------------------------------------------------------------------------------
// Tiles of BM x BN, 64 of the contraction a step, two buffers.  The loads of a step write LDS by themselves (16 bytes a lane, no registers in between) while the step
// before is multiplied; one barrier a step.  Fragments are read one cluster of products ahead, across the barrier too, so the matrix cores do not wait for LDS.
//   rows operand     LDS holds [line][64], 8 pieces of 16 bytes a line, piece p of line l at p ^ (l & 7): the 16 lines of a fragment fall on distinct banks
//   columns operand  LDS holds [64][line]; fragments come out transposed by ds_read_b64_tr_b16 (4 contraction rows x 16 lines a 16-lane group); the 32-byte
//                    piece q of row k sits at q ^ h(k), with h different for the 16 rows that one instruction reads
// Lines and contraction beyond the operand are loaded as zero (an offset outside of the buffer's range).
// 16384 x 4096 x 4096 bf16 with 256 x 256 tiles: y 511 us (1.08 Pflop/s; the library 448), with gelu, residual and act' kept 541; dx 500 (522), dW 442 .. 484 (577).  Four tiles a
// compute unit: what is left is their starts and ends, 15 us each, in which the matrix cores wait; the clock falls with them busy, so less waiting gains less than it
// takes away.  The next lines' residual loaded ahead in the epilogue: 588 us for 577.  4096 x 2048 x 2048 with 128 x 128 tiles: 39, 40, 41 us (36, 38, 50).
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

template <typename T, bool ACOLS, bool BCOLS, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(BM / WM * (BN / WN) * 64, 2) k_product16(Operand<T> A, Operand<T> B, int64_t M, int64_t N, int64_t lines_a, int64_t lines_b, int64_t K, int64_t slice, Epilogue<T> E,
                                                                           Columns<T> C) {
#if defined(__HIP_DEVICE_COMPILE__)          // the host pass has no type for a buffer's descriptor
    constexpr int THREADS = BM / WM * (BN / WN) * 64, TM = WM / 16, TN = WN / 16, PARTS = TM / 4, CLUSTERS = 2 * PARTS;
    // each buffer (A's tile, then B's) is a variable of its own: the compiler then knows which loads a read of LDS has to wait for
    constexpr int BUFFER = (BM + BN) * STEP;
    __shared__ __attribute__((aligned(1024))) short s0[BUFFER], s1[BUFFER];
    const uint32_t tiles_m = (uint32_t)((M + BM - 1) / BM), tiles_n = (uint32_t)((N + BN - 1) / BN);
    if (blockIdx.x >= tiles_m * tiles_n) {
        if (blockIdx.y == 0) join_columns<T>(C, blockIdx.x - tiles_m * tiles_n, (float*)s0);
        return;
    }
    uint32_t ti, tj;
    tile_of(blockIdx.x, tiles_m, tiles_n, ti, tj);
    const int64_t i0 = (int64_t)ti * BM, j0 = (int64_t)tj * BN;
    const int64_t c_begin = (int64_t)blockIdx.y * slice, len = (c_begin + slice < K ? c_begin + slice : K) - c_begin;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave / (BN / WN) * WM, wj = wave % (BN / WN) * WN;
    Feed<ACOLS, BM, THREADS> fa;
    Feed<BCOLS, BN, THREADS> fb;
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
        wait_and_meet<0>();          // the next step's tiles have arrived, and nobody reads this step's any more
        if (++k < steps) read(next, 0);
        if (k + 1 < steps) load(s);
        multiply(CLUSTERS - 1);
    };
    if (steps > 0) load(s0);
    if (steps > 1) load(s1);
    wait_and_meet<0>();
    if (steps > 0) read(s0, 0);
    while (k < steps) {
        step(s0, s1);
        if (k < steps) step(s1, s0);
    }
    // nobody reads or loads tiles any more: the buffers hold the waves' sums
    static_assert(WN == 64 && BUFFER * 2 * 2 == THREADS / 64 * 64 * 64 * 4, "LDS for the sums");
    constexpr int SHARE = THREADS / 64 / 2;
    short* mine = wave < SHARE ? s0 : s1;
    store_wave<T, TM, (TM > 4 ? 1 : 4)>(E, acc, (float*)mine + wave % SHARE * 64 * 64, i0 + wi, j0 + wj, M, N);
#endif
}

// The same product where the tiles do not fill the chip and latency is what counts: one workgroup a compute unit, tiles of BM x 128, four buffers, so that three steps are
// on their way while one is multiplied, and twice the waves: each 64 x 64 of the tile is done by two of them, one for either half of a step, whose sums are added in the end.
// 2048 x 2048 x 2048 bf16: y 20.5 us, dx 23, dW 24 (the library 23, 27, 30); 1000 x 1000 x 1000 fp16 10, 11, 11 (21, 20, 22); 512 x 4096 x 4096 27, 37, 24 (27, 35, 27).
// Every step loads and reads ahead, behind the end too (nothing but zeros comes from there): without branches the compiler sees which loads a read waits for.
template <typename T, bool ACOLS, bool BCOLS, int BM>
__global__ void __launch_bounds__(BM * 4) k_product16_deep(Operand<T> A, Operand<T> B, int64_t M, int64_t N, int64_t lines_a, int64_t lines_b, int64_t K, int64_t slice, Epilogue<T> E, Columns<T> C) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int THREADS = BM * 4, QUARTERS = BM / 32, BUFFER = (BM + TILE) * STEP;
    __shared__ __attribute__((aligned(1024))) short s0[BUFFER], s1[BUFFER], s2[BUFFER], s3[BUFFER];
    const uint32_t tiles_m = (uint32_t)((M + BM - 1) / BM), tiles_n = (uint32_t)((N + TILE - 1) / TILE);
    if (blockIdx.x >= tiles_m * tiles_n) {
        if (blockIdx.y == 0) join_columns<T>(C, blockIdx.x - tiles_m * tiles_n, (float*)s0);
        return;
    }
    uint32_t ti, tj;
    tile_of(blockIdx.x, tiles_m, tiles_n, ti, tj);
    const int64_t i0 = (int64_t)ti * BM, j0 = (int64_t)tj * TILE;
    const int64_t c_begin = (int64_t)blockIdx.y * slice, len = (c_begin + slice < K ? c_begin + slice : K) - c_begin;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int quarter = wave % QUARTERS, half = wave / QUARTERS, wi = (quarter >> 1) * 64, wj = (quarter & 1) * 64;
    Feed<ACOLS, BM, THREADS> fa;
    Feed<BCOLS, TILE, THREADS> fb;
    constexpr int LOADS = Feed<ACOLS, BM, THREADS>::LOADS + Feed<BCOLS, TILE, THREADS>::LOADS;
    fa.init(A.p, A.ld, i0, lines_a, c_begin);
    fb.init(B.p, B.ld, j0, lines_b, c_begin);
    f32x4 acc[4][4] = {};
    s16x8 va[4], vb[4];
    const int steps = (int)((len + STEP - 1) / STEP);
    int64_t left = len;
    const auto load = [&](short* s) __attribute__((always_inline)) {
        fa.load(s, left);
        fb.load(s + BM * STEP, left);
        left -= STEP;
    };
    const auto read = [&](const short* s) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 4; ++u) va[u] = fragment<ACOLS, BM>(s, wi + u * 16, half);
#pragma unroll
        for (int w = 0; w < 4; ++w) vb[w] = fragment<BCOLS, TILE>(s + BM * STEP, wj + w * 16, half);
    };
    const auto step = [&](short* s, short* next) __attribute__((always_inline)) {
        wait_and_meet<2 * LOADS>();          // the next step's tiles have arrived, and nobody reads this step's any more
        s16x8 xa[4], xb[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) xa[u] = va[u], xb[u] = vb[u];
        read(next);
        load(s);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int w = 0; w < 4; ++w) acc[u][w] = mfma<T>(xb[w], xa[u], acc[u][w]);
    };
    load(s0);
    load(s1);
    load(s2);
    load(s3);
    wait_and_meet<3 * LOADS>();
    read(s0);
    int k = 0;
    for (; k + 4 <= steps; k += 4) {
        step(s0, s1);
        step(s1, s2);
        step(s2, s3);
        step(s3, s0);
    }
    if (k < steps) step(s0, s1);
    if (k + 1 < steps) step(s1, s2);
    if (k + 2 < steps) step(s2, s3);
    wait_and_meet<0>();
    // nobody reads or loads tiles any more: one half's sums into LDS, the other's onto them, and each wave takes half of the lines to memory
    constexpr int PER = BUFFER * 2 / (64 * 64 * 4);          // 64 x 64 sums that a buffer holds
    static_assert(QUARTERS <= 2 * PER, "LDS for the sums");
    float* sums = (float*)(quarter < PER ? s0 : s1) + quarter % PER * 64 * 64;
    if (half == 1) put_sums<4>(acc, 0, sums);
    __syncthreads();
    if (half == 0) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                f32x4* at = (f32x4*)(sums + piece_of_sums(u * 16 + (lane & 15), w * 4 + (lane >> 4)));
                const f32x4 other = *at;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[u][w][e] += other[e];
                *at = acc[u][w];
            }
    }
    __syncthreads();
    drain_sums<T, 4>(E, sums, half * 32, half * 32 + 32, i0 + wi, j0 + wj, M, N);
#endif
}

// ---- few rows -------------------------------------------------------------------------------------------------------------------------------------------
// y for at most 32 rows of x (serving): bound by the weight's bytes and by latency.  A workgroup takes 16 NT rows of W, its 8 waves share the contraction out in stretches of
// CHUNK, and fragments come straight from memory: each matrix instruction takes 16 bytes a lane of 16 rows of W, so W is read once, with nothing staged, and the loads of the
// next stretch are on their way while one is multiplied.  16-bit: one instruction a load; fp32: the fp32 matrix instruction four times (its rate does not matter here, and it
// rounds like a chain of fused multiply-adds).  The waves' sums meet in LDS.
// 1 x 4096 x 4096 bf16 9.7 us, 24 rows of 2048 -> 8192 fp16 with bias and silu 10.2: 33.6 MB, 6.5 us of a large copy's rate, and a launch; all of W is asked for at once.
constexpr int ROWS_THREADS = 512, ROWS_WAVES = ROWS_THREADS / 64;
template <typename T, int MT, int NT>
__global__ void __launch_bounds__(ROWS_THREADS) k_rows(const T* x, int64_t ldx, const T* w, int64_t ldw, int64_t M, int64_t N, int64_t K, int64_t slice, Epilogue<T> E) {
    constexpr int V = width<T>(), PER = 4 * V, U = MT * NT == 1 ? 8 : 4, CHUNK = PER * U;          // PER of the contraction a load
    typedef Pack<T, V> Vec;
    __shared__ float sums[ROWS_WAVES][MT * NT][16][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = (lane >> 4) * V;
    const int64_t n0 = (int64_t)blockIdx.x * 16 * NT;
    const int64_t c_begin = (int64_t)blockIdx.y * slice, c_end = c_begin + slice < K ? c_begin + slice : K;
    // lines beyond the end repeat the last one; nobody stores what comes of them
    const T* line[NT + MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t n = n0 + t * 16 + (lane & 15);
        line[t] = w + (n < N ? n : N - 1) * ldw + at;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t m = t * 16 + (lane & 15);
        line[NT + t] = x + (m < M ? m : M - 1) * ldx + at;
    }
    struct Chunk { Vec v[NT + MT][U]; };
    const auto fetch = [&](int64_t c, Chunk& q) __attribute__((always_inline)) {
        if (c + CHUNK <= c_end) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < NT + MT; ++t) q.v[t][u] = *(const Vec*)(line[t] + c + u * PER);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < NT + MT; ++t)
#pragma unroll
                    for (int e = 0; e < V; ++e) q.v[t][u].v[e] = c + u * PER + at + e < c_end ? line[t][c + u * PER + e] : (T)0.f;
        }
    };
    f32x4 acc[NT][MT] = {};
    const auto multiply = [&](const Chunk& q) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const Vec &a = q.v[n][u], &b = q.v[NT + m][u];
                    if constexpr (sizeof(T) == 4) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[n][m] = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], acc[n][m], 0, 0, 0);
                    } else {
                        acc[n][m] = mfma<T>(__builtin_bit_cast(s16x8, a), __builtin_bit_cast(s16x8, b), acc[n][m]);
                    }
                }
    };
    constexpr int64_t ROUND = ROWS_WAVES * CHUNK;
    int64_t c = c_begin + wave * CHUNK;
    Chunk p, q;
    if (c < c_end) fetch(c, p);
    for (; c < c_end; c += 2 * ROUND) {
        if (c + ROUND < c_end) fetch(c + ROUND, q);
        multiply(p);
        if (c + ROUND >= c_end) break;
        if (c + 2 * ROUND < c_end) fetch(c + 2 * ROUND, p);
        multiply(q);
    }
    // a lane holds 4 neighbouring columns (rows of W) of one row of x
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[wave][n * MT + m][lane & 15][(lane >> 4) * 4 + e] = acc[n][m][e];
    __syncthreads();
    for (int k = threadIdx.x; k < MT * NT * 256; k += ROWS_THREADS) {
        const int n = k / (MT * 256), m16 = k / 16 % (16 * MT);
        const int64_t m = m16, j = n0 + n * 16 + (k & 15);
        if (m >= M || j >= N) continue;
        float z[1][1] = {{0.f}};
#pragma unroll
        for (int s = 0; s < ROWS_WAVES; ++s) z[0][0] += sums[s][n * MT + (m16 >> 4)][m16 & 15][k & 15];
        if (E.part) E.part[((int64_t)blockIdx.y * M + m) * N + j] = z[0][0];
        else {
            const float q[1] = {E.bias ? (float)E.bias[j] : 0.f};
            finish<T, 1, 1>(E, m, 0, j, M, N, z, q);
        }
    }
}

// The slices of a contraction joined, then the epilogue.  `groups` lanes of a workgroup share the slices of four outputs in equal stretches, in their order.
template <typename T> __global__ void __launch_bounds__(256) k_join(const float* part, int splits, int groups, int64_t M, int64_t N, Epilogue<T> E, uint32_t blocks, Columns<T> C) {
    constexpr int V = 4;
    __shared__ f32x4 sums[256 + 16];
    if (blockIdx.x >= blocks) return join_columns<T>(C, blockIdx.x - blocks, (float*)sums);
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
    if (!ok) return;
    float q[V] = {};
    if (E.bias) load_some<T, V>(E.bias + j, N - j, q);
    finish<T, V, 1>(E, i, 0, j, M, N, z, q);
}

// What the products read, made in one launch.  Workgroups 0 .. : gz = g act'(z), rounded to the layer's type (the matrix instructions take 16-bit operands, and a
// second part of gz would double both products; the gradients' error is 1.4 times that of unrounded ones), in rows that start on 16 bytes with zeros behind their ends, and its
// column sums (of the unrounded values) by slabs of rows: 16384 x 4096 bf16 77 us, 402 MB at 5.2 TB/s (the code of act' taken apart costs 3 us); 28432 x 6528 260 us, 1.1 GB (one line of a lane at a
// time 300, four 354).  The others repack: operands' rows copied to rows that start on 16 bytes, zeros behind their ends.
constexpr int GZ_LANES = 32, GZ_LINES = 8, GZ_ROUND = 2 * GZ_LINES;
template <typename T> struct Gz {
    const T* g;
    const typename dact_type<T>::type* dact;
    T* gz;                          // null: the sums alone
    float* part;                    // [slabs][N], or null
    int64_t ldg, ldgz, M, N, slab;
    uint32_t across, blocks;
};
template <typename T> struct Pack2 {
    const T* p[2];
    T* out[2];
    int64_t ld[2], ldo[2], rows[2], cols[2];
    uint32_t first, blocks[2];
};
template <typename T> __global__ void __launch_bounds__(256) k_prepare(Gz<T> G, Pack2<T> P) {
    constexpr int V = width<T>();
    __shared__ float sums[GZ_LINES][GZ_LANES * V];
    if (blockIdx.x >= G.blocks) {
        uint32_t block = blockIdx.x - G.blocks;
        const int q = block >= P.blocks[0] ? 1 : 0;
        block -= q ? P.blocks[0] : 0;
        const int64_t vectors = P.ldo[q] / V, at = (int64_t)block * 256 + threadIdx.x;
        if (at >= P.rows[q] * vectors) return;
        const int64_t r = at / vectors, c = at % vectors * V;
        float v[V];
        load_some<T, V>(P.p[q] + r * P.ld[q] + c, P.cols[q] - c, v);
        store_some<T, V>(P.out[q] + r * P.ldo[q] + c, V, v);
        return;
    }
    const int x = threadIdx.x % GZ_LANES, y = threadIdx.x / GZ_LANES;
    const int64_t bx = blockIdx.x % G.across, by = blockIdx.x / G.across;
    const int64_t j = (bx * GZ_LANES + x) * V, in_row = G.N - j;
    const int64_t m0 = by * G.slab, m1 = m0 + G.slab < G.M ? m0 + G.slab : G.M;
    float s[V] = {};
    if (in_row > 0)
        for (int64_t m = m0 + y; m < m1; m += GZ_ROUND) {
            // GZ_ROUND / GZ_LINES lines of a lane are on their way together
            float v[GZ_ROUND / GZ_LINES][V], d[GZ_ROUND / GZ_LINES][V];
#pragma unroll
            for (int q = 0; q < GZ_ROUND / GZ_LINES; ++q) {
                const int64_t l = m + q * GZ_LINES, some = l < m1 ? in_row : 0;
                load_some<T, V>(G.g + l * G.ldg + j, some, v[q]);
                if (G.dact) load_some<typename dact_type<T>::type, V>(G.dact + l * G.N + j, some, d[q]);
            }
#pragma unroll
            for (int q = 0; q < GZ_ROUND / GZ_LINES; ++q) {
                const int64_t l = m + q * GZ_LINES;
                if (G.dact)
#pragma unroll
                    for (int k = 0; k < V; ++k) v[q][k] = gated(v[q][k], d[q][k]);
                if (G.gz && l < m1) store_some<T, V>(G.gz + l * G.ldgz + j, V, v[q]);
#pragma unroll
                for (int k = 0; k < V; ++k) s[k] += v[q][k];
            }
        }
    if (!G.part) return;
#pragma unroll
    for (int k = 0; k < V; ++k) sums[y][x * V + k] = s[k];
    __syncthreads();
    for (int c = threadIdx.x; c < GZ_LANES * V; c += 256) {
        const int64_t at = bx * GZ_LANES * V + c;
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < GZ_LINES; ++q) t += sums[q][c];
        if (at < G.N) G.part[by * G.N + at] = t;
    }
}

template <typename T> __global__ void __launch_bounds__(1024) k_join_columns(Columns<T> C) {
    __shared__ float lds[32 * 33];
    join_columns<T>(C, blockIdx.x, lds);
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------------------
constexpr int CUS = 256;
constexpr int64_t MAX_TILES = (1ll << 32) / 256 - 1;          // a launch has fewer than 2^32 lanes
static int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }
static int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

// How a product is run: the kernel, the slices of its contraction, and what of the workspace it takes.
struct Plan {
    int rows = TILE, cols = TILE;          // of a tile
    bool deep = false;                     // k_product16_deep
    int64_t tiles = 0, splits = 1, slice = 0;
    int64_t at_cols = 0, bytes = 0;          // the slices' sums come first, then their column sums
};
static Plan plan(int es, int columns /* operands that come by columns */, int64_t M, int64_t N, int64_t K, bool column_sums) {
    Plan p;
    if (M == 0 || N == 0) return p;
    const auto tiles = [&](int64_t r, int64_t c) { return gs::cdiv(M, r) * gs::cdiv(N, c); };
    // Tiles and slices by what they cost: rounds of the chip x (steps x us a step + the start and the end of a workgroup), and for slices a second launch that reads and
    // writes their sums at 4 TB/s.  The us a step are measured, for one, two and four workgroups on a compute unit.
    const auto join = [&](int64_t s) { return s > 1 ? 4.0 + 2.0 * s * M * N * 4 / 4e6 : 0.0; };
    double best = 1e30;
    const auto take = [&](int rows, int cols, int64_t t, int64_t s, double cost, bool deep) {
        if (cost < best) best = cost, p.rows = rows, p.cols = cols, p.tiles = t, p.splits = s, p.deep = deep;
    };
    if (es == 4) {
        // 128: 2.8 us a step with two a unit, 2.2 with one, 64: 1.4 with four, 1.1 with two, 0.85 with one -- times 1.2 where one operand comes a column at a time (dx), 1.5 where both do
        // (dW).  131072 x 256 x 256: tiles of 128 / 64 107 / 122 us for y, 113 / 127 for dx, 107 / 147 for dW; 50000 x 256 x 295 with softplus: 82 / 73 for y; 52549 x 4927 x 671
        // 2220 / 2580; 31273 x 418 x 40 45 / 32.  The us are rougher than the differences between the two: over full rounds they favour 64 by up to 14 %, and where the last round
        // tips the balance (110000 x 256 x 256) the choice may be the slower by 4 % (y 117 / 113, dx 125 / 120).
        const int64_t steps = gs::cdiv(K, BK);
        const double slow = columns == 0 ? 1.05 : columns == 1 ? 1.2 : 1.5;
        for (int r = 64; r <= TILE; r += 64) {
            const int64_t t = tiles(r, r), most = r == 64 ? 4 : 2;
            if (r == 64 && t >= MAX_TILES) continue;
            for (int64_t a_unit = 0; a_unit <= most; a_unit = a_unit ? 2 * a_unit : 1) {
                int64_t s = a_unit ? a_unit * CUS / t : 1;          // as many slices as fill the chip with a_unit workgroups each, or one
                if (a_unit && s > steps / 2) s = steps / 2;          // (steps / 4 costs small training steps 2 %, steps / 8 7 %)
                if (s < 1 || s > 256) continue;
                const auto round = [&](int64_t wg) {          // of as many workgroups
                    const int64_t on = gs::cdiv(wg, CUS);
                    return wg == 0 ? 0.0 : gs::cdiv(steps, s) * (r == 64 ? (on == 1 ? 0.85 : on == 2 ? 1.1 : 1.4) * slow : (on == 1 ? 2.2 : 2.8)) + (r == 64 ? 5.0 : 11.0);
                };
                const int64_t wg = t * s, full = most * CUS;
                take(r, r, t, s, (wg / full) * round(full) + round(wg % full) + join(s), false);
            }
        }
    } else if (tiles(256, 256) >= 192) {
        // With tiles of 256 / 128, K 2048: 3584 x 3584 (196 tiles of 256) y 57 / 67 us, 4096 x 4096 (256) 61 / 77, 4096 x 4352 (272, a second round for 16 of them) 103 / 95; below
        // them 4096 x 2048 over 4096 (128 tiles) 101 / 75.  A few columns leave most of such a tile outside of the output, which the rule does not
        // look at: 131072 x 64 x 64 21 / 12, 83195 x 62 -> 103 27 / 16.
        p.rows = p.cols = 256, p.tiles = tiles(256, 256);
    } else if (tiles(TILE, TILE) > CUS) {
        p.tiles = tiles(TILE, TILE);
    } else {
        // 0.5 us a step for 128 rows (2048 x 2048 x 2048: 22 us), 0.37 us for 64 (512 x 4096 x 4096: 27 us)
        const int64_t steps = gs::cdiv(K, STEP);
        for (int r = 64; r <= TILE; r += 64) {
            const int64_t t = tiles(r, TILE);
            if (t > CUS) continue;
            int64_t full = CUS / t;
            if (full > steps / 4) full = steps / 4;
            for (const int64_t s : {(int64_t)1, full / 2, full})
                if (s >= 1) take(r, TILE, t, s, gs::cdiv(steps, s) * (r == 64 ? 0.37 : 0.5) + join(s), true);
        }
    }
    p.slice = p.splits > 1 ? gs::cdiv(gs::cdiv(K, p.splits), 64) * 64 : K;
    p.splits = p.splits > 1 ? gs::cdiv(K, p.slice) : 1;
    p.at_cols = p.splits > 1 ? align256(p.splits * M * N * 4) : 0;
    p.bytes = p.at_cols + (column_sums && p.splits > 1 ? align256(p.splits * M * 4) : 0);
    return p;
}

// An operand: the 16-bit kernels read its rows 16 bytes at a time, by 31-bit offsets within a tile; rows that do not start on 16 bytes, or end inside of them, are
// repacked first.
struct Line {
    const void* p;
    int64_t ld, cols;          // row stride, elements of a row that are read
    bool zeros;                // rows have zeros up to a multiple of 8 behind their ends
};
static bool direct(const Line& a) { return ((uintptr_t)a.p & 15) == 0 && a.ld % 8 == 0 && (a.cols % 8 == 0 || a.zeros) && a.ld < (1 << 21); }
static int64_t packed_bytes(int es, const Line& a, int64_t rows) { return es == 2 && !direct(a) ? align256(rows * up8(a.cols) * es) : 0; }

// One more operand for the repacking launch, where it needs it.
template <typename T> int64_t repack(Pack2<T>& P, int q, Line& a, int64_t rows, char* to) {
    const int64_t bytes = packed_bytes(sizeof(T), a, rows);
    if (!bytes) return 0;
    P.p[q] = (const T*)a.p, P.ld[q] = a.ld, P.rows[q] = rows, P.cols[q] = a.cols, P.out[q] = (T*)to, P.ldo[q] = up8(a.cols);
    P.blocks[q] = (uint32_t)gs::cdiv(rows * (P.ldo[q] / width<T>()), 256);
    a = {to, P.ldo[q], a.cols, true};
    return bytes;
}
template <typename T> int prepare(const Gz<T>& G, const Pack2<T>& P, hipStream_t stream) {
    const uint64_t blocks = (uint64_t)G.blocks + P.blocks[0] + P.blocks[1];
    GS_REQUIRE(blocks <= (uint64_t)MAX_TILES, "gs_linear: operands too large for one launch");
    if (blocks) hipLaunchKernelGGL(k_prepare<T>, dim3((unsigned)blocks), dim3(256), 0, stream, G, P);
    return 0;
}

static unsigned join_blocks(int64_t M, int64_t N, int64_t splits, int& groups) {
    groups = splits >= 32 ? 16 : splits >= 8 ? 4 : 1;
    return (unsigned)gs::cdiv(M * gs::cdiv(N, 4), 256 / groups);
}
// C [M,N] over a contraction of K; operands that the kernels can read as they are.  fp32: A times `gate` (row stride ldgate), where there is one, and A's sums to db (dW only).
// columns: sums that are joined beside the product; its `blocks` is set to zero once that is launched.
template <typename T, bool ACOLS, bool BCOLS>
int product(const Line& a, const Line& b, int64_t M, int64_t N, int64_t K, Epilogue<T> E, char* ws, int64_t ws_bytes, hipStream_t stream, const float* gate, int64_t ldgate, T* db,
            Columns<T>& columns) {
    if (M == 0 || N == 0) return 0;
    const Plan p = plan(sizeof(T), ACOLS + BCOLS, M, N, K, db != nullptr);
    GS_REQUIRE(ws_bytes >= p.bytes, "gs_linear: workspace too small");
    GS_REQUIRE(p.tiles + (int64_t)columns.blocks <= (p.rows == 256 || p.deep ? MAX_TILES / 2 : MAX_TILES), "gs_linear: too many tiles for one launch");
    Epilogue<T> first = E;
    first.part = p.splits > 1 ? (float*)ws : nullptr;
    Columns<T> none{}, beside = none;
    if constexpr (sizeof(T) == 4) {
        const dim3 grid((unsigned)p.tiles, (unsigned)p.splits);
        const Operand<float> A{(const float*)a.p, a.ld}, B{(const float*)b.p, b.ld};
        float* cols = db ? (p.splits > 1 ? (float*)(ws + p.at_cols) : db) : nullptr;
        const auto kernel = p.rows == 64 ? (gate ? k_product32<ACOLS, BCOLS, true, 64> : k_product32<ACOLS, BCOLS, false, 64>)
                                         : (gate ? k_product32<ACOLS, BCOLS, true, 128> : k_product32<ACOLS, BCOLS, false, 128>);
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, A, gate, ldgate, B, M, N, K, p.slice, first, cols);
        if (db && p.splits > 1) beside = Columns<T>{cols, db, M, (int)p.splits, (uint32_t)gs::cdiv(M, 32)};
    } else {
        const dim3 grid((unsigned)(p.tiles + columns.blocks), (unsigned)p.splits);
        const int64_t lines_a = ACOLS && a.zeros ? up8(M) : M, lines_b = BCOLS && b.zeros ? up8(N) : N;
        const Operand<T> A{(const T*)a.p, a.ld}, B{(const T*)b.p, b.ld};
        if (p.rows == 256)
            hipLaunchKernelGGL((k_product16<T, ACOLS, BCOLS, 256, 256, 128, 64>), grid, dim3(512), 0, stream, A, B, M, N, lines_a, lines_b, K, p.slice, first, columns);
        else if (!p.deep)
            hipLaunchKernelGGL((k_product16<T, ACOLS, BCOLS, 128, 128, 64, 64>), grid, dim3(256), 0, stream, A, B, M, N, lines_a, lines_b, K, p.slice, first, columns);
        else if (p.rows == 128)
            hipLaunchKernelGGL((k_product16_deep<T, ACOLS, BCOLS, 128>), grid, dim3(512), 0, stream, A, B, M, N, lines_a, lines_b, K, p.slice, first, columns);
        else
            hipLaunchKernelGGL((k_product16_deep<T, ACOLS, BCOLS, 64>), grid, dim3(256), 0, stream, A, B, M, N, lines_a, lines_b, K, p.slice, first, columns);
        columns.blocks = 0;
    }
    if (p.splits > 1) {
        int groups;
        const uint32_t blocks = join_blocks(M, N, p.splits, groups);
        hipLaunchKernelGGL(k_join<T>, dim3(blocks + beside.blocks), dim3(256), 0, stream, (const float*)ws, (int)p.splits, groups, M, N, E, blocks, beside);
    }
    GS_LAUNCH_CHECK();
    return 0;
}

// k_rows: at most 32 rows, and where its workgroups of 16 columns do not fill the chip slices of the contraction, each of one round of the waves or more
static bool few_rows(int64_t M, int64_t N) { return M <= 32 && N <= MAX_TILES * 8; }
static Plan rows_plan(int64_t M, int64_t N, int64_t K) {
    Plan p;
    p.cols = gs::cdiv(N, 32) >= CUS ? 32 : 16;          // x is read by every workgroup: twice the columns where that leaves a workgroup for each compute unit
    p.tiles = gs::cdiv(N, p.cols);
    if (p.tiles < CUS / 2 && K >= 4096) {
        p.splits = CUS / p.tiles < K / 2048 ? CUS / p.tiles : K / 2048;
        p.slice = gs::cdiv(gs::cdiv(K, p.splits), 1024) * 1024;
        p.splits = gs::cdiv(K, p.slice);
    }
    if (p.splits == 1) p.slice = K;
    p.bytes = p.splits > 1 ? align256(p.splits * M * N * 4) : 0;
    return p;
}
template <typename T>
int product_rows(const Line& x, const Line& w, int64_t M, int64_t N, int64_t K, Epilogue<T> E, char* ws, hipStream_t stream) {
    const Plan p = rows_plan(M, N, K);
    Epilogue<T> first = E;
    first.part = p.splits > 1 ? (float*)ws : nullptr;
    const dim3 grid((unsigned)p.tiles, (unsigned)p.splits);
    const auto kernel = p.cols == 32 ? (M <= 16 ? k_rows<T, 1, 2> : k_rows<T, 2, 2>) : (M <= 16 ? k_rows<T, 1, 1> : k_rows<T, 2, 1>);
    hipLaunchKernelGGL(kernel, grid, dim3(ROWS_THREADS), 0, stream, (const T*)x.p, x.ld, (const T*)w.p, w.ld, M, N, K, p.slice, first);
    if (p.splits > 1) {
        int groups;
        const unsigned blocks = join_blocks(M, N, p.splits, groups);
        hipLaunchKernelGGL(k_join<T>, dim3(blocks), dim3(256), 0, stream, (const float*)ws, (int)p.splits, groups, M, N, E, blocks, Columns<T>{});
    }
    GS_LAUNCH_CHECK();
    return 0;
}

static int64_t forward_bytes(int es, const Line& x, const Line& w, int64_t M, int64_t N, int64_t K) {
    if (few_rows(M, N)) return rows_plan(M, N, K).bytes;
    return packed_bytes(es, x, M) + packed_bytes(es, w, N) + plan(es, 0, M, N, K, false).bytes;
}

static Beta beta_of(float beta) {
    const double c = (double)beta * 1.4426950408889634;
    return {(float)c, (float)(c - (double)(float)c), 2.f / beta};
}

template <typename T>
int linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* res, int64_t ldr, int64_t M, int64_t N, int64_t K, int act,
               float beta, void* y, int64_t ldy, void* dact, void* ws, int64_t ws_bytes, hipStream_t stream) {
    Line lx{x, ldx, K, false}, lw{w, ldw, K, false};
    const int64_t need = forward_bytes(sizeof(T), lx, lw, M, N, K);
    GS_REQUIRE(ws_bytes >= need && (ws || need == 0), "gs_linear_fwd: workspace too small");
    GS_REQUIRE(((uintptr_t)ws & 15) == 0, "gs_linear_fwd: the workspace must start on 16 bytes");
    char* at = (char*)ws;
    Epilogue<T> E{(const T*)bias, (const T*)res, (T*)y, (typename dact_type<T>::type*)dact, nullptr, ldr, ldy, act, beta_of(act == ACT_SOFTPLUS ? beta : 1.f)};
    if (few_rows(M, N)) return product_rows<T>(lx, lw, M, N, K, E, at, stream);
    Pack2<T> P{};
    at += repack<T>(P, 0, lx, M, at);
    at += repack<T>(P, 1, lw, N, at);
    if (const int rc = prepare<T>(Gz<T>{}, P, stream)) return rc;
    Columns<T> none{};
    return product<T, false, false>(lx, lw, M, N, K, E, at, (char*)ws + ws_bytes - at, stream, nullptr, 0, nullptr, none);
}

struct BackwardPlan {
    bool gz_made, pass, sums_with_w;          // gz has a place of its own; a pass over g is made; db comes with dW
    int64_t ldgz, slab, slabs, across;
    int64_t cols, packs, prod, total;          // byte offsets (gz comes first): the column sums' slabs, the repacked operands, the products' workspace
};
static BackwardPlan backward_plan(const Line& g, bool has_dact, const Line& x, const Line& w, int64_t M, int64_t N, int64_t K, int es, bool want_x, bool want_w, bool want_b) {
    BackwardPlan p;
    // fp32 products take the gate as they load g, and the sums with dW; 16-bit ones read gz from memory
    p.gz_made = es == 2 && (want_x || want_w) && (has_dact || !direct(g));
    p.sums_with_w = es == 4 && want_w && want_b && K > 0;
    p.pass = p.gz_made || (want_b && !p.sums_with_w);
    p.ldgz = p.gz_made ? up8(N) : g.ld;
    p.across = gs::cdiv(N, GZ_LANES * 16 / es);
    p.slab = gs::cdiv(gs::cdiv(M * p.across, 2048), GZ_LINES) * GZ_LINES;
    if (p.slab < 64) p.slab = 64;
    p.slabs = gs::cdiv(M, p.slab);
    p.cols = p.gz_made ? align256(M * p.ldgz * es) : 0;
    p.packs = p.cols + (p.pass && want_b ? align256(p.slabs * N * 4) : 0);
    p.prod = p.packs + (want_x ? packed_bytes(es, w, N) : 0) + (want_w ? packed_bytes(es, x, M) : 0);
    int64_t b = 0;
    if (want_x) b = plan(es, 1, M, K, N, false).bytes;
    if (want_w) {
        const int64_t c = plan(es, 2, N, K, M, p.sums_with_w).bytes;
        if (c > b) b = c;
    }
    p.total = p.prod + b;
    return p;
}

template <typename T>
int linear_bwd(const void* g, int64_t ldg, const void* dact, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, void* dx,
               void* dw, void* db, void* ws, int64_t ws_bytes, hipStream_t stream) {
    Line gz{g, ldg, N, false}, lx{x, ldx, K, false}, lw{w, ldw, K, false};
    const BackwardPlan p = backward_plan(gz, dact != nullptr, lx, lw, M, N, K, sizeof(T), dx != nullptr, dw != nullptr, db != nullptr);
    GS_REQUIRE(ws_bytes >= p.total && (ws || p.total == 0), "gs_linear_bwd: workspace too small");
    GS_REQUIRE(((uintptr_t)ws & 15) == 0, "gs_linear_bwd: the workspace must start on 16 bytes");
    if (N == 0 && K == 0) return 0;
    char* base = (char*)ws;
    Gz<T> G{};
    Pack2<T> P{};
    Columns<T> columns{};
    if (N > 0 && p.pass) {
        const bool sums = db && !p.sums_with_w;
        G = Gz<T>{(const T*)g, (const typename dact_type<T>::type*)dact, p.gz_made ? (T*)base : nullptr, sums ? (float*)(base + p.cols) : nullptr, ldg, p.ldgz, M, N, p.slab,
                  (uint32_t)p.across, (uint32_t)(p.across * p.slabs)};
        GS_REQUIRE(p.across * p.slabs < (1ll << 31), "gs_linear_bwd: gradient too large for one launch");
        if (sums) columns = Columns<T>{(const float*)(base + p.cols), (T*)db, N, (int)p.slabs, (uint32_t)gs::cdiv(N, 32)};
        if (p.gz_made) gz = {base, p.ldgz, N, true};
    }
    int64_t at = p.packs;
    if (dx) at += repack<T>(P, 0, lw, N, base + at);
    if (dw) at += repack<T>(P, 1, lx, M, base + at);
    if (const int rc = prepare<T>(G, P, stream)) return rc;
    Epilogue<T> E{};
    const float* gate = sizeof(T) == 4 ? (const float*)dact : nullptr;
    E.ldo = K;
    if (dx) {
        E.out = (T*)dx;
        if (const int rc = product<T, false, true>(gz, lw, M, K, N, E, base + p.prod, ws_bytes - p.prod, stream, gate, N, nullptr, columns)) return rc;
    }
    if (dw) {
        E.out = (T*)dw;
        if (const int rc = product<T, true, true>(gz, lx, N, K, M, E, base + p.prod, ws_bytes - p.prod, stream, gate, N, p.sums_with_w ? (T*)db : nullptr, columns)) return rc;
    }
    if (columns.blocks) hipLaunchKernelGGL(k_join_columns<T>, dim3(columns.blocks), dim3(1024), 0, stream, columns);          // no 16-bit product was there to do it beside
    GS_LAUNCH_CHECK();
    return 0;
}

// 16-bit tiles are addressed by 31-bit offsets: 256 rows of 2^21 elements fit
static bool sizes_ok(int64_t M, int64_t N, int64_t K, int dtype) {
    const int64_t top = 1ll << 31, wide = dtype == DT_F32 ? top : 1ll << 21;
    return M >= 0 && N >= 0 && K >= 0 && M < top && N < wide && K < wide;
}

}  // namespace

extern "C" int64_t gs_linear_fwd_workspace_bytes(const void* x, int64_t ldx, const void* weight, int64_t ldw, int64_t M, int64_t N, int64_t K, int dtype) {
    if (dtype < 0 || dtype > 2 || !sizes_ok(M, N, K, dtype)) return -1;
    return M == 0 || N == 0 ? 0 : forward_bytes(dtype == DT_F32 ? 4 : 2, {x, ldx, K, false}, {weight, ldw, K, false}, M, N, K);
}

extern "C" int gs_linear_fwd(const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* bias, const void* residual, int64_t ldr, int64_t M, int64_t N,
                             int64_t K, int dtype, int act, float beta, void* y, int64_t ldy, void* dact, void* workspace, int64_t workspace_bytes, gs_stream_t stream) {
    GS_REQUIRE(dtype >= 0 && dtype <= 2, "gs_linear_fwd: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    GS_REQUIRE(sizes_ok(M, N, K, dtype), "gs_linear_fwd: sizes are 0 .. 2^31 - 1, of 16-bit rows 0 .. 2^21 - 1");
    GS_REQUIRE(act >= 0 && act <= 4, "gs_linear_fwd: unknown activation");
    GS_REQUIRE(act != ACT_SOFTPLUS || (beta > 0.f && beta < 1e30f), "gs_linear_fwd: softplus needs a positive finite beta");
    if (M == 0 || N == 0) return 0;
    GS_REQUIRE(y && ldy >= N && (!residual || ldr >= 0), "gs_linear_fwd: null output or row stride smaller than a row");
    GS_REQUIRE(K == 0 || (x && weight && ldx >= 0 && ldw >= 0), "gs_linear_fwd: null operand or negative row stride");
    const auto run = dtype == DT_F32 ? linear_fwd<float> : dtype == DT_BF16 ? linear_fwd<bf16> : linear_fwd<f16>;
    return run(x, ldx, weight, ldw, bias, residual, ldr, M, N, K, act, beta, y, ldy, dact, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int64_t gs_linear_bwd_workspace_bytes(const void* g, int64_t ldg, int has_dact, const void* x, int64_t ldx, const void* weight, int64_t ldw, int64_t M, int64_t N,
                                                 int64_t K, int dtype, int want_x, int want_w, int want_b) {
    if (dtype < 0 || dtype > 2 || !sizes_ok(M, N, K, dtype)) return -1;
    return backward_plan({g, ldg, N, false}, has_dact, {x, ldx, K, false}, {weight, ldw, K, false}, M, N, K, dtype == DT_F32 ? 4 : 2, want_x, want_w, want_b).total;
}

extern "C" int gs_linear_bwd(const void* g, int64_t ldg, const void* dact, const void* x, int64_t ldx, const void* weight, int64_t ldw, int64_t M, int64_t N, int64_t K,
                             int dtype, void* dx, void* dw, void* db, void* workspace, int64_t workspace_bytes, gs_stream_t stream) {
    GS_REQUIRE(dtype >= 0 && dtype <= 2, "gs_linear_bwd: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    GS_REQUIRE(sizes_ok(M, N, K, dtype), "gs_linear_bwd: sizes are 0 .. 2^31 - 1, of 16-bit rows 0 .. 2^21 - 1");
    GS_REQUIRE(M == 0 || N == 0 || (g && ldg >= 0), "gs_linear_bwd: null gradient");
    GS_REQUIRE(M == 0 || N == 0 || K == 0 || ((!dx || (weight && ldw >= 0)) && (!dw || (x && ldx >= 0))), "gs_linear_bwd: null operand or negative row stride");
    const auto run = dtype == DT_F32 ? linear_bwd<float> : dtype == DT_BF16 ? linear_bwd<bf16> : linear_bwd<f16>;
    return run(g, ldg, dact, x, ldx, weight, ldw, M, N, K, dx, dw, db, workspace, workspace_bytes, (hipStream_t)stream);
}

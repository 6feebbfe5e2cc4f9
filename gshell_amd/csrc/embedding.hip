// GS_CXXFLAGS: -Xclang -target-feature -Xclang -packed-fp32-ops
// Table lookup with scaling, and its gradient by sorted row numbers (gfx950).
//
//     y_t = s W[id_t]                      dW_v = s sum_{t: id_t = v} g_t   (rows that no id names: zero)
//
// The gradient's sums are 32-bit, in an order that does not depend on how the launch is scheduled, nor on where g lies.  Tables of few, narrow rows: partial tables in LDS, added up in their order
// (k_sum_few).  Others: the tokens are sorted by row
// (a stable radix sort of our own), then every CHUNK neighbours of the sorted list are summed by one group of lanes.  A run of equal rows inside a chunk is written at once;
// one that crosses chunks leaves a part in each and is joined in a second launch, so that a row that holds most of the tokens is spread over the chip as well.
// No atomics, no pass over the table but the one that writes it.
// An id outside of [0, V) (which the host cannot see without waiting for the GPU) reads nothing: its output row is NaN and it has no gradient.
#include <hip/hip_runtime.h>

#include "../../include/gshell_hip.h"
#include "common.hpp"

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;

constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr int MAX_BITS = 9, MAX_BINS = 1 << MAX_BITS;
constexpr int SORT_BLOCKS = 64;              // tiles of the sort: few enough that every tile adds up all tiles' counts by itself
constexpr int SMALL_T = 2048, SMALL_BITS = 8;          // tokens that one workgroup sorts in LDS, in one launch
constexpr int CHUNK = 32;

template <typename I> __device__ __forceinline__ uint32_t key_of(I id, int64_t V, int64_t padding) {
    const int64_t v = (int64_t)id;
    return v < 0 || v >= V || v == padding ? (uint32_t)V : (uint32_t)v;          // V: sorted behind every row, summed into none
}

// Exclusive prefix sums of one value a thread, and their total.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* tmp, uint32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(s, d);
        if (lane >= d) s += o;
    }
    if (lane == 63) tmp[wave] = s;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
    for (int w = 0; w < SORT_WAVES; ++w) {
        if (w < wave) before += tmp[w];
        total += tmp[w];
    }
    __syncthreads();
    return before + s - v;
}

// Lanes of this wave that hold the same digit (among the active ones)
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool active) {
    uint64_t m = __ballot(active);
    for (int b = 0; b < bits; ++b) {
        const uint64_t one = __ballot((digit >> b) & 1);
        m &= (digit >> b) & 1 ? one : ~one;
    }
    return m;
}

// Each wave counts the digits of its own stretch [w0, w1) of the list; counts[wave][bin]
template <typename F> __device__ __forceinline__ void wave_counts(F key, int64_t w0, int64_t w1, int shift, int bits, uint32_t* counts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bins = 1 << bits;
    for (int b = threadIdx.x; b < SORT_WAVES * bins; b += SORT_THREADS) counts[b] = 0;
    __syncthreads();
    for (int64_t i = w0; i < w1; i += 64) {
        const bool ok = i + lane < w1;
        if (ok) atomicAdd(&counts[wave * bins + ((key(i + lane) >> shift) & (bins - 1))], 1u);
    }
    __syncthreads();
}

// Stable scatter of the wave's stretch; counts[wave][bin] holds the first free place of (wave, bin) and moves on
template <typename F, typename G> __device__ __forceinline__ void wave_scatter(F key, G put, int64_t w0, int64_t w1, int shift, int bits, uint32_t* counts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bins = 1 << bits;
    for (int64_t i = w0; i < w1; i += 64) {
        const bool ok = i + lane < w1;
        const uint32_t k = ok ? key(i + lane) : 0, digit = (k >> shift) & (bins - 1);
        const uint64_t same = same_digit(digit, bits, ok);
        if (ok) {
            uint32_t* c = &counts[wave * bins + digit];
            const uint32_t at = *c + __popcll(same & ((1ull << lane) - 1));
            put(i + lane, k, at);
            // every lane of a digit has read its counter before the last of them moves it: they run in step, and the wave is the counter's only user
            __builtin_amdgcn_wave_barrier();
            if ((same >> lane) == 1) *c = at + 1;
        }
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

template <typename I>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_count(const I* ids, const uint32_t* keys, int64_t T, int64_t V, int64_t padding, int64_t tile, int shift, int bits, uint32_t* hist) {
    __shared__ uint32_t counts[MAX_BINS];
    const int bins = 1 << bits;
    for (int b = threadIdx.x; b < bins; b += SORT_THREADS) counts[b] = 0;
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * tile, t1 = t0 + tile < T ? t0 + tile : T;
    for (int64_t i = t0 + threadIdx.x; i < t1; i += SORT_THREADS) {
        const uint32_t k = ids ? key_of(ids[i], V, padding) : keys[i];
        atomicAdd(&counts[(k >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += SORT_THREADS) hist[blockIdx.x * MAX_BINS + b] = counts[b];
}

template <typename I>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_scatter(const I* ids, const uint32_t* keys, const uint32_t* pos, int64_t T, int64_t V, int64_t padding, int64_t tile,
                                                              int shift, int bits, const uint32_t* hist, uint32_t* keys_out, uint32_t* pos_out) {
    __shared__ uint32_t counts[SORT_WAVES * MAX_BINS], tmp[SORT_WAVES], part[2][SORT_THREADS];
    const int bins = 1 << bits, wave = threadIdx.x >> 6;
    const int64_t t0 = (int64_t)blockIdx.x * tile, t1 = t0 + tile < T ? t0 + tile : T;
    const int64_t stretch = (tile / SORT_WAVES + 63) / 64 * 64;
    const int64_t w0 = t0 + wave * stretch < t1 ? t0 + wave * stretch : t1, w1 = w0 + stretch < t1 ? w0 + stretch : t1;
    const auto key = [&](int64_t i) { return ids ? key_of(ids[i], V, padding) : keys[i]; };
    wave_counts(key, w0, w1, shift, bits, counts);
    // tokens of each bin in earlier tiles and in all tiles: SORT_THREADS / bins threads share a bin's tiles, eight loads at a time
    const int shares = SORT_THREADS >> bits, share = threadIdx.x >> bits, bin = threadIdx.x & (bins - 1);
    uint32_t before = 0, all = 0;
    for (int b = share; b < (int)gridDim.x; b += 8 * shares) {
        uint32_t c[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) c[k] = b + k * shares < (int)gridDim.x ? hist[(b + k * shares) * MAX_BINS + bin] : 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            before += b + k * shares < (int)blockIdx.x ? c[k] : 0;
            all += c[k];
        }
    }
    part[0][threadIdx.x] = before, part[1][threadIdx.x] = all;
    __syncthreads();
    before = all = 0;
    if ((int)threadIdx.x < bins)
        for (int q = 0; q < shares; ++q) before += part[0][q * bins + threadIdx.x], all += part[1][q * bins + threadIdx.x];
    uint32_t total;
    uint32_t at = block_scan(all, tmp, total) + before;
    if ((int)threadIdx.x < bins)
        for (int w = 0; w < SORT_WAVES; ++w) {
            const uint32_t c = counts[w * bins + threadIdx.x];
            counts[w * bins + threadIdx.x] = at;
            at += c;
        }
    __syncthreads();
    wave_scatter(key, [&](int64_t i, uint32_t k, uint32_t to) { keys_out[to] = k; pos_out[to] = ids ? (uint32_t)i : pos[i]; }, w0, w1, shift, bits, counts);
}

// the whole sort of a short list by one workgroup
template <typename I>
__global__ void __launch_bounds__(SORT_THREADS) k_sort_small(const I* ids, int T, int64_t V, int64_t padding, int total_bits, uint32_t* keys_out, uint32_t* pos_out) {
    __shared__ uint32_t keys[2][SMALL_T], counts[SORT_WAVES << SMALL_BITS], tmp[SORT_WAVES];
    __shared__ uint16_t pos[2][SMALL_T];
    for (int i = threadIdx.x; i < T; i += SORT_THREADS) keys[0][i] = key_of(ids[i], V, padding), pos[0][i] = (uint16_t)i;
    __syncthreads();
    const int wave = threadIdx.x >> 6;
    const int stretch = ((T + SORT_WAVES - 1) / SORT_WAVES + 63) / 64 * 64;
    const int w0 = wave * stretch < T ? wave * stretch : T, w1 = w0 + stretch < T ? w0 + stretch : T;
    int from = 0;
    for (int shift = 0; shift < total_bits; shift += SMALL_BITS) {
        const int bits = total_bits - shift < SMALL_BITS ? total_bits - shift : SMALL_BITS, bins = 1 << bits;
        const uint32_t* kin = keys[from];
        const uint16_t* pin = pos[from];
        uint32_t* kout = keys[from ^ 1];
        uint16_t* pout = pos[from ^ 1];
        const auto key = [&](int64_t i) { return kin[i]; };
        wave_counts(key, w0, w1, shift, bits, counts);
        uint32_t all = 0, total;
        if ((int)threadIdx.x < bins)
            for (int w = 0; w < SORT_WAVES; ++w) all += counts[w * bins + threadIdx.x];
        uint32_t at = block_scan(all, tmp, total);
        if ((int)threadIdx.x < bins)
            for (int w = 0; w < SORT_WAVES; ++w) {
                const uint32_t c = counts[w * bins + threadIdx.x];
                counts[w * bins + threadIdx.x] = at;
                at += c;
            }
        __syncthreads();
        wave_scatter(key, [&](int64_t i, uint32_t k, uint32_t to) { kout[to] = k; pout[to] = pin[i]; }, w0, w1, shift, bits, counts);
        __syncthreads();
        from ^= 1;
    }
    for (int i = threadIdx.x; i < T; i += SORT_THREADS) keys_out[i] = keys[from][i], pos_out[i] = pos[from][i];
}

// VEC neighbouring values of a row (rows may start at any element; the hardware loads unaligned vectors)
template <typename T, int VEC> struct __attribute__((packed)) Pack { T v[VEC]; };

template <typename T, int VEC, typename U> __device__ __forceinline__ void load_row(const T* p, int64_t left, U (&out)[VEC]) {
    if (left >= VEC) {
        const Pack<T, VEC> q = *(const Pack<T, VEC>*)p;
#pragma unroll
        for (int k = 0; k < VEC; ++k) out[k] = (U)q.v[k];
    } else if (left > 0) {          // what is behind the row's end repeats its last value in the load: one branch and one wait
        const int n = (int)left;
#pragma unroll
        for (int k = 0; k < VEC; ++k) out[k] = (U)p[k < n ? k : n - 1];
#pragma unroll
        for (int k = 0; k < VEC; ++k) out[k] = k < n ? out[k] : (U)0.f;
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) out[k] = (U)0.f;
    }
}
template <typename T, int VEC, typename U> __device__ __forceinline__ void store_row(T* p, int64_t left, const U (&in)[VEC]) {
    if (left >= VEC) {
        Pack<T, VEC> q;
#pragma unroll
        for (int k = 0; k < VEC; ++k) q.v[k] = (T)in[k];
        *(Pack<T, VEC>*)p = q;
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (k < left) p[k] = (T)in[k];
    }
}

// Forward: the output is one stretch of memory, written 16 aligned bytes a lane and piece; LOOKUPS pieces a lane are on their way together.  A piece inside a row is one load (at
// whatever address the row has it), one that runs over a row's end is gathered.  The place of a lane's next piece comes without a division: step_rows, step_cols are
// what a workgroup's pieces of one round cover.
// Bound by memory: 65536 rows of 1024 bf16 out of 50000 44 us (134 MB written, 32 MB of different rows read), 262144 of 32 fp32 10 us; 8 rows of 4096 3.2 us, a launch.  One piece a
// lane 47, 9.8 and 2.7 us, four 46, 9.9 and 3.4, eight 57, 10.7 and 5.0.
constexpr int LOOKUPS = 2;
template <typename T, typename I>
__global__ void __launch_bounds__(256) k_lookup(const I* ids, const T* w, int64_t ldw, int64_t tokens, int64_t V, int64_t D, int64_t step_rows, int64_t step_cols, float scale, T* y) {
    constexpr int VEC = 16 / sizeof(T);
    const int64_t total = tokens * D;
    int64_t at = ((int64_t)blockIdx.x * 256 * LOOKUPS + threadIdx.x) * VEC;
    int64_t t = at / D, c = at - t * D;
    float v[LOOKUPS][VEC];
    int64_t place[LOOKUPS];
#pragma unroll
    for (int u = 0; u < LOOKUPS; ++u) {
        place[u] = at;
        if (at < total) {
            const int64_t id = (int64_t)ids[t];
            const bool ok = id >= 0 && id < V;
            if (c + VEC <= D) {
                if (ok) load_row<T, VEC>(w + id * ldw + c, VEC, v[u]);
                else
#pragma unroll
                    for (int k = 0; k < VEC; ++k) v[u][k] = __builtin_nanf("");
            } else if (D >= VEC && V > 0) {          // two rows; what has no value to read reads the table's first
                const int64_t next = t + 1 < tokens ? (int64_t)ids[t + 1] : -1;
                const bool ok1 = next >= 0 && next < V;
                const T *a = ok ? w + id * ldw + c : w, *b = ok1 ? w + next * ldw : w;
                const int here = (int)(D - c), da = ok ? 1 : 0, db = ok1 ? 1 : 0;
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[u][k] = (float)a[(k < here ? k : 0) * da];
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const float q = (float)b[k < here ? 0 : (k - here) * db];
                    v[u][k] = k < here ? (ok ? v[u][k] : __builtin_nanf("")) : ok1 ? q : __builtin_nanf("");
                }
            } else {
                int64_t r = t, q = c, row = ok ? id : -1;
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    if (q == D) {
                        ++r, q = 0;
                        const int64_t next = at + k < total ? (int64_t)ids[r] : -1;
                        row = next >= 0 && next < V ? next : -1;
                    }
                    v[u][k] = at + k < total ? (row >= 0 ? (float)w[row * ldw + q] : __builtin_nanf("")) : 0.f;
                    ++q;
                }
            }
        }
        at += 256 * VEC;
        t += step_rows, c += step_cols;
        if (c >= D) c -= D, ++t;
    }
#pragma unroll
    for (int u = 0; u < LOOKUPS; ++u) {
        if (place[u] >= total) return;
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[u][k] *= scale;
        store_row<T, VEC>(y + place[u], total - place[u], v[u]);
    }
}

__device__ __forceinline__ int64_t lower_bound(const uint32_t* keys, int64_t n, uint32_t key) {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

constexpr int BVEC = 4;          // columns of a lane in the sums of narrow rows

// Rows of the table that no token names: `rows` of them a wave from v0 on, 64 at most, 2^group_log lanes a row
// (6 tokens of 3389 fp32 over 1801 rows: 15 us with one row a wave, 80 with 64)
template <typename T> __device__ __forceinline__ void clear_rows(const uint32_t* keys, int64_t tokens, int64_t V, int64_t D, int64_t v0, int rows, int group_log, T* dw) {
    constexpr int VEC = 16 / sizeof(T);
    const int lane = threadIdx.x & 63, group = 1 << group_log;
    const int64_t v = v0 + lane;
    if (v0 >= V) return;
    bool empty = false;
    if (lane < rows && v < V) {
        const int64_t at = lower_bound(keys, tokens, (uint32_t)v);
        empty = at >= tokens || keys[at] != (uint32_t)v;
    }
    const uint64_t which = __ballot(empty);
    const float zero[VEC] = {};
    for (int r = lane >> group_log; r < rows; r += 64 >> group_log)
        if (which >> r & 1)
            for (int64_t c = (lane & (group - 1)) * VEC; c < D; c += group * VEC) store_row<T, VEC>(dw + (v0 + r) * D + c, D - c, zero);
}
// 64 rows a wave, fewer where the waves would be fewer than those of four workgroups a compute unit
static int rows_a_wave(int64_t V) { return V >= 64 * 4096 ? 64 : V >= 16 * 4096 ? 16 : V >= 4 * 4096 ? 4 : 1; }

// Rows of more than 256 bytes: a wave takes one (chunk, stretch of columns), and its lanes hold the chunk's rows and numbers, so that every choice is a scalar one and
// eight rows are on their way at a time.  A run of up to CHUNK tokens is summed as a whole by the chunk where it begins; a longer one leaves a part in each of its chunks.
// Bound by memory: 65536 tokens of 1024 bf16, their numbers spread like 1 / n over 50000 rows: 75 us for 134 MB of gradient, 102 MB of table and the long runs' parts
// (3.2 TB/s).
template <typename T, int VEC>
__global__ void __launch_bounds__(256) k_sum_wide(const uint32_t* keys, const uint32_t* pos, const T* g, int64_t ldg, int64_t tokens, int64_t V, int64_t D, int64_t stretches,
                                                  int64_t chunks, int64_t sum_blocks, int rows, int clear_log, float scale, T* dw, float* first, float* last) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((int64_t)blockIdx.x >= sum_blocks) return clear_rows<T>(keys, tokens, V, D, (((int64_t)blockIdx.x - sum_blocks) * 4 + wave) * rows, rows, clear_log, dw);
    const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
    if (unit >= chunks * stretches) return;
    const int64_t chunk = unit / stretches, c = (unit % stretches * 64 + lane) * VEC, e0 = chunk * CHUNK;
    const uint32_t none = (uint32_t)V;
    // this chunk and the next one; the one before in the lower lanes of `past`
    static_assert(CHUNK == 32, "two chunks a wave");
    const uint32_t key = e0 + lane < tokens ? keys[e0 + lane] : none, past = lane < 32 && e0 > 0 ? keys[e0 - 32 + lane] : none;
    const uint32_t row_of = e0 + lane < tokens ? pos[e0 + lane] : 0;
    const uint32_t key0 = __builtin_amdgcn_readlane(key, 0);
    if (key0 == none) return;
    const uint32_t after = __shfl_down(key, 1);
    const uint64_t ends = __ballot(lane == 63 || key != after);          // lanes where a run ends
    // the run that the chunk begins with: its tokens in the chunk before (32 at most) and from here on
    const uint32_t behind = (uint32_t)__ballot(lane < 32 && e0 > 0 && past == key0);
    const int back = behind == 0xffffffffu ? 32 : __clz((int)~behind), ahead = __builtin_ctzll(ends) + 1;
    const bool long_head = back > 0 && back + ahead > CHUNK;
    const int begin = back > 0 && !long_head ? ahead : 0;
    if (begin >= CHUNK) return;
    // the last run that begins (or goes on) in this chunk
    const uint64_t upto = ends & ((1ull << (CHUNK - 1)) - 1);          // runs that end before the chunk's last token
    const int tail = upto ? 64 - __builtin_clzll(upto) : 0;              // where the run of that last token begins (0: with the chunk)
    const int tail_end = __builtin_ctzll(ends >> (CHUNK - 1)) + CHUNK;          // one behind its last token, 64 at most
    const bool tail_is_head = tail == 0 && back > 0, long_tail = tail_is_head ? long_head : tail_end - tail > CHUNK;
    int end = long_tail ? (tail_end < CHUNK ? tail_end : CHUNK) : tail_end;
    const uint64_t empty = __ballot(key == none);
    if (empty && __builtin_ctzll(empty) < end) end = __builtin_ctzll(empty);
    float acc[VEC] = {};
    const T* base = g + c;
    for (int j = begin; j < end; j += 8) {
        float v[8][VEC];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (j + k < end) load_row<T, VEC>(base + (int64_t)(uint32_t)__builtin_amdgcn_readlane(row_of, j + k) * ldg, D - c, v[k]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (j + k >= end) break;
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] += v[k][q];
            if (!(ends >> (j + k) & 1) && j + k + 1 < end) continue;
            if (long_head && j + k < ahead) {
                store_row<float, VEC>(first + chunk * D + c, D - c, acc);
            } else if (long_tail && j + k >= tail) {
                store_row<float, VEC>(last + chunk * D + c, D - c, acc);
            } else {
#pragma unroll
                for (int q = 0; q < VEC; ++q) acc[q] *= scale;
                store_row<T, VEC>(dw + (int64_t)(uint32_t)__builtin_amdgcn_readlane(key, j + k) * D + c, D - c, acc);
            }
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
        }
    }
}

// Narrower rows: several groups of lanes a wave, a chunk each, 25 us for 262144 tokens of 64 bf16 over 160 rows; every run that crosses chunks leaves its parts.  Blocks below `sum_blocks` sum chunks, the others write the rows that no token names.
template <typename T>
__global__ void __launch_bounds__(256) k_sum_chunks(const uint32_t* keys, const uint32_t* pos, const T* g, int64_t ldg, int64_t tokens, int64_t V, int64_t D, int group_log,
                                                    int64_t stretches, int64_t chunks, int64_t sum_blocks, int rows, int clear_log, float scale, T* dw, float* first, float* last) {
    if ((int64_t)blockIdx.x >= sum_blocks) return clear_rows<T>(keys, tokens, V, D, (((int64_t)blockIdx.x - sum_blocks) * 4 + (threadIdx.x >> 6)) * rows, rows, clear_log, dw);
    const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> group_log;
    if (unit >= chunks * stretches) return;
    const int64_t chunk = unit / stretches, c = ((unit % stretches) << group_log) * BVEC + (threadIdx.x & ((1 << group_log) - 1)) * BVEC;
    if (c >= D) return;
    const int64_t e0 = chunk * CHUNK, e1 = e0 + CHUNK < tokens ? e0 + CHUNK : tokens;
    const uint32_t none = (uint32_t)V;
    const uint32_t before = e0 > 0 ? keys[e0 - 1] : none, after = e1 < tokens ? keys[e1] : none;
    uint32_t run = keys[e0];
    bool head = true;          // the run began with the chunk
    float acc[BVEC] = {};
    const auto flush = [&](bool end) {
        if (run == none) return;
        if (head && run == before) store_row<float, BVEC>(first + chunk * D + c, D - c, acc);
        else if (end && run == after) store_row<float, BVEC>(last + chunk * D + c, D - c, acc);
        else {
            float out[BVEC];
#pragma unroll
            for (int k = 0; k < BVEC; ++k) out[k] = acc[k] * scale;
            store_row<T, BVEC>(dw + (int64_t)run * D + c, D - c, out);
        }
    };
    // the next tokens' rows and numbers are on their way while these are summed; what is behind the end repeats the last one
    uint32_t next[8], place[8];
    const auto fetch = [&](int64_t e) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t at = e + k < e1 ? e + k : e1 - 1;
            next[k] = keys[at], place[k] = pos[at];
        }
    };
    fetch(e0);
    for (int64_t e = e0; e < e1; e += 8) {
        uint32_t key[8];
        float v[8][BVEC];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            key[k] = e + k < e1 ? next[k] : none;
            if (key[k] != none) load_row<T, BVEC>(g + (int64_t)place[k] * ldg + c, D - c, v[k]);
        }
        if (e + 8 < e1) fetch(e + 8);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (e + k >= e1) break;
            if (key[k] != run) {
                flush(false);
                run = key[k], head = false;
#pragma unroll
                for (int q = 0; q < BVEC; ++q) acc[q] = 0.f;
            }
            if (key[k] != none)
#pragma unroll
                for (int q = 0; q < BVEC; ++q) acc[q] += v[k][q];
        }
    }
    flush(true);
}

// Runs that left parts, in the order of their chunks: the chunk where a run begins joins it, a workgroup each, whose groups of lanes share the parts out in equal
// stretches.  `shortest`: runs of fewer tokens left none.
template <typename T>
__global__ void __launch_bounds__(1024) k_join_chunks(const uint32_t* keys, int64_t tokens, int64_t V, int64_t D, int group_log, int64_t stretches, int shortest, float scale,
                                                      const float* first, const float* last, T* dw) {
    __shared__ float part[1024 * BVEC];
    const int64_t chunk = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, e1 = (chunk + 1) * CHUNK;
    if (e1 >= tokens) return;
    // one look at this chunk's keys (every wave has them all), the one before it, and the first keys of the 64 chunks that follow
    const int lane = threadIdx.x & 63;
    const uint32_t key = keys[chunk * CHUNK + (lane & (CHUNK - 1))], before = chunk > 0 ? keys[chunk * CHUNK - 1] : (uint32_t)V;
    const int64_t follow = (chunk + 1 + lane) * CHUNK;
    const uint32_t next = follow < tokens ? keys[follow] : (uint32_t)V;
    const uint32_t run = __builtin_amdgcn_readlane(key, CHUNK - 1);
    const uint64_t reach = __ballot(next == run);
    if (run == (uint32_t)V || !(reach & 1)) return;
    const int inside = __popcll(__ballot(key == run && lane < CHUNK));          // its tokens in this chunk
    if (inside == CHUNK && before == run) return;          // it began earlier
    int64_t more = ~reach ? __builtin_ctzll(~reach) : 0;          // chunks behind this one that hold a part
    if (!~reach) more = (lower_bound(keys, tokens, run + 1) - 1) / CHUNK - chunk;
    if (shortest > 1 && more == 1) {          // two chunks: whether it is long enough shows where its last token would be
        const int64_t last_at = e1 - inside + shortest - 1;
        if (last_at >= tokens || keys[last_at] != run) return;
    }
    const int groups = blockDim.x >> group_log, group = threadIdx.x >> group_log, x = threadIdx.x & ((1 << group_log) - 1);
    const int64_t share = (more + groups - 1) / groups, k0 = group * share, k1 = k0 + share < more ? k0 + share : more;
    for (int64_t s = 0; s < stretches; ++s) {
        const int64_t c = ((s << group_log) + x) * BVEC;
        float acc[BVEC] = {};
        if (c < D)
            for (int64_t q = k0; q < k1; q += 8) {
                float v[8][BVEC];
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (q + u < k1) load_row<float, BVEC>(first + (chunk + 1 + q + u) * D + c, D - c, v[u]);
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (q + u < k1)
#pragma unroll
                        for (int e = 0; e < BVEC; ++e) acc[e] += v[u][e];
            }
#pragma unroll
        for (int e = 0; e < BVEC; ++e) part[threadIdx.x * BVEC + e] = acc[e];
        __syncthreads();
        if (group == 0 && c < D) {
            float sum[BVEC];
            load_row<float, BVEC>(last + chunk * D + c, D - c, sum);
            for (int q = 0; q < groups; ++q)
#pragma unroll
                for (int e = 0; e < BVEC; ++e) sum[e] += part[((q << group_log) + x) * BVEC + e];
#pragma unroll
            for (int e = 0; e < BVEC; ++e) sum[e] *= scale;
            store_row<T, BVEC>(dw + (int64_t)run * D + c, D - c, sum);
        }
        __syncthreads();
    }
}

// Tables of few and narrow rows: no sort.  Each group of lanes (as many as a row has columns) keeps a table of its own in LDS and adds every groups-th token of the workgroup's
// stretch to it, a lane a column; tokens without a row go to one more behind the last.  A place belongs to one lane, which reads, adds and writes it in the tokens' order: the
// sums are the same every time (LDS's float atomics need twice the time of these).  The tables are added up in their order, the workgroups' sums in a second launch
// (`part`; null: there is one workgroup, which writes dw).  Bound by the chain through LDS, a token at a time for each of a compute unit's 16 .. 512 groups.
constexpr int FEW_FLOATS = 40960, FEW_AHEAD = 8;          // all of a compute unit's LDS; tokens of a group that are on their way together
template <typename T, typename I>
__global__ void __launch_bounds__(512) k_sum_few(const I* ids, const T* g, int64_t ldg, int64_t tokens, int64_t per, int V, int D, int64_t padding, int group_log, float scale, T* dw, float* part) {
    __shared__ float tables[FEW_FLOATS];
    const int size = V * D, whole = size + D, groups = blockDim.x >> group_log, group = threadIdx.x >> group_log, lane = threadIdx.x & ((1 << group_log) - 1);
    for (int e = threadIdx.x; e < whole * groups; e += blockDim.x) tables[e] = 0.f;
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * per, t1 = t0 + per < tokens ? t0 + per : tokens;
    if (lane < D) {
        float* mine = tables + group * whole + lane;
        const T* column = g + lane;
        int64_t t = t0 + group;
        for (; t + (FEW_AHEAD - 1) * groups < t1; t += FEW_AHEAD * groups) {
            I id[FEW_AHEAD];
            T v[FEW_AHEAD];
#pragma unroll
            for (int k = 0; k < FEW_AHEAD; ++k) id[k] = ids[t + k * groups], v[k] = column[(t + k * groups) * ldg];
#pragma unroll
            for (int k = 0; k < FEW_AHEAD; ++k) mine[(int)key_of(id[k], V, padding) * D] += (float)v[k];
        }
        for (; t < t1; t += groups) mine[(int)key_of(ids[t], V, padding) * D] += (float)column[t * ldg];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < size; e += blockDim.x) {
        float s = 0.f;
        for (int q = 0; q < groups; ++q) s += tables[q * whole + e];
        if (part) part[(int64_t)blockIdx.x * size + e] = s;
        else dw[e] = (T)(s * scale);
    }
}
// 32 elements a workgroup, the parts in eight stretches side by side
template <typename T> __global__ void __launch_bounds__(256) k_join_few(const float* part, int parts, int size, float scale, T* dw) {
    __shared__ float sums[8][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, e = blockIdx.x * 32 + x, share = (parts + 7) / 8, k0 = y * share, k1 = k0 + share < parts ? k0 + share : parts;
    float s = 0.f;
    if (e < size)
        for (int k = k0; k < k1; k += 8) {
            float q[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) q[u] = k + u < k1 ? part[(int64_t)(k + u) * size + e] : 0.f;
#pragma unroll
            for (int u = 0; u < 8; ++u) s += q[u];
        }
    sums[y][x] = s;
    __syncthreads();
    if (y > 0 || e >= size) return;
    for (int q = 1; q < 8; ++q) s += sums[q][x];
    dw[e] = (T)(s * scale);
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------------------
static int group_log_of(int64_t vectors) {          // lanes, as a power of two, of a group that takes a row or a stretch of one
    int l = 0;
    while (l < 6 && (1ll << l) < vectors) ++l;
    return l;
}

// Whether a table counts as one of few, narrow rows: at most 64 columns, and the tables of 256 lanes' groups fit in LDS; then twice the lanes where theirs do, and workgroups for
// the chip.  fp32, lookup and gradient: 262144 tokens over 72 x 32 26 us, sorted 54; over 140 x 64 54, sorted 59; 2 million over 150 x 8 49, sorted 181; 256 over 72 x 32 13,
// sorted 25.  With more than 64 columns, in stretches of 64: 262144 over 14 x 200 117, sorted 153, but over 70 x 130 132, sorted 116, and over 9 x 1024 689, sorted 584.
constexpr int ONE_BLOCK = 8;
struct FewPlan {
    int threads = 0, group_log = 0;          // no threads: it does not
    int64_t blocks = 0, per = 0, bytes = 0;
};
static FewPlan few_plan(int64_t T, int64_t V, int64_t D) {
    FewPlan p;
    if (T == 0 || V > FEW_FLOATS || D > 64) return p;
    p.group_log = group_log_of(D);
    if ((V + 1) * D * (256 >> p.group_log) > FEW_FLOATS) return p;
    p.threads = (V + 1) * D * (512 >> p.group_log) > FEW_FLOATS ? 256 : 512;
    const int64_t round = (int64_t)(p.threads >> p.group_log) * FEW_AHEAD, rounds = gs::cdiv(T, round);
    // A few rounds by one workgroup, without the second launch: 1000 tokens over 72 x 32 fp32 13 us of GPU time with the lookup, as by 8 workgroups, and 35 us of the host's for 39;
    // 2000 would take 17 us for 13.
    p.per = gs::cdiv(rounds, rounds <= ONE_BLOCK ? 1 : rounds < 256 ? rounds : 256) * round;
    p.blocks = gs::cdiv(T, p.per);
    p.bytes = p.blocks > 1 ? p.blocks * V * D * 4 : 0;
    return p;
}

struct SortPlan {
    int64_t keys[2], pos[2], hist, first, last, total, chunks;
};
static int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }
static SortPlan sort_plan(int64_t T, int64_t D) {
    SortPlan p;
    int64_t at = 0;
    for (int k = 0; k < 2; ++k) {
        p.keys[k] = at, at += align256(T * 4);
        p.pos[k] = at, at += align256(T * 4);
    }
    p.hist = at, at += MAX_BINS * SORT_BLOCKS * 4;
    p.chunks = gs::cdiv(T, CHUNK);
    p.first = at, at += align256(p.chunks * D * 4);
    p.last = at, at += align256(p.chunks * D * 4);
    p.total = at;
    return p;
}

// Elements of a lane's vector.  16 bytes where every row starts on 16; otherwise the hardware takes 16 bytes at any address, but slower than 8 on 8.
static int vector_of(int es, int64_t D, int64_t ld, const void* p, const void* q) {
    const uintptr_t a = (uintptr_t)p | (uintptr_t)q | (uintptr_t)(D * es) | (uintptr_t)(ld * es);
    return (a & 15) == 0 ? 16 / es : 8 / es;
}

template <typename T, typename I>
int lookup(const void* ids, const void* w, int64_t ldw, int64_t tokens, int64_t V, int64_t D, float scale, void* y, hipStream_t stream) {
    constexpr int VEC = 16 / sizeof(T);
    const int64_t blocks = gs::cdiv(tokens * D, 256 * VEC * LOOKUPS), step = 256 * VEC;
    GS_REQUIRE(blocks < (1ll << 24), "gs_embedding_fwd: too large for one launch");
    hipLaunchKernelGGL((k_lookup<T, I>), dim3((unsigned)blocks), dim3(256), 0, stream, (const I*)ids, (const T*)w, ldw, tokens, V, D, step / D, step % D, scale, (T*)y);
    GS_LAUNCH_CHECK();
    return 0;
}

template <typename I> int sort_tokens(const void* ids, int64_t T, int64_t V, int64_t padding, const SortPlan& p, char* base, uint32_t*& keys, uint32_t*& pos, hipStream_t stream) {
    int bits = 1;
    while ((1ll << bits) <= V) ++bits;
    keys = (uint32_t*)(base + p.keys[0]), pos = (uint32_t*)(base + p.pos[0]);
    if (T <= SMALL_T) {
        hipLaunchKernelGGL(k_sort_small<I>, dim3(1), dim3(SORT_THREADS), 0, stream, (const I*)ids, (int)T, V, padding, bits, keys, pos);
        GS_LAUNCH_CHECK();
        return 0;
    }
    uint32_t* hist = (uint32_t*)(base + p.hist);
    const int passes = (bits + MAX_BITS - 1) / MAX_BITS, each = (bits + passes - 1) / passes;
    int64_t tile = gs::cdiv(T, SORT_BLOCKS);
    if (tile < SORT_THREADS) tile = SORT_THREADS;
    tile = (tile + SORT_THREADS - 1) / SORT_THREADS * SORT_THREADS;          // whole rounds of the workgroup: its waves' stretches cover the tile
    const unsigned blocks = (unsigned)gs::cdiv(T, tile);
    const I* in = (const I*)ids;
    const uint32_t *kin = nullptr, *pin = nullptr;
    for (int q = 0, shift = 0; q < passes; ++q, shift += each) {
        const int b = bits - shift < each ? bits - shift : each;
        keys = (uint32_t*)(base + p.keys[q & 1]), pos = (uint32_t*)(base + p.pos[q & 1]);
        hipLaunchKernelGGL(k_sort_count<I>, dim3(blocks), dim3(SORT_THREADS), 0, stream, in, kin, T, V, padding, tile, shift, b, hist);
        hipLaunchKernelGGL(k_sort_scatter<I>, dim3(blocks), dim3(SORT_THREADS), 0, stream, in, kin, pin, T, V, padding, tile, shift, b, (const uint32_t*)hist, keys, pos);
        in = nullptr, kin = keys, pin = pos;
    }
    GS_LAUNCH_CHECK();
    return 0;
}

template <typename T, typename I>
int gradient(const void* ids, const void* g, int64_t ldg, int64_t tokens, int64_t V, int64_t D, int64_t padding, float scale, void* dw, char* base, hipStream_t stream) {
    if (const FewPlan f = few_plan(tokens, V, D); f.threads) {
        float* part = f.blocks > 1 ? (float*)base : nullptr;
        hipLaunchKernelGGL((k_sum_few<T, I>), dim3((unsigned)f.blocks), dim3(f.threads), 0, stream, (const I*)ids, (const T*)g, ldg, tokens, f.per, (int)V, (int)D, padding, f.group_log, scale, (T*)dw, part);
        if (part) hipLaunchKernelGGL(k_join_few<T>, dim3((unsigned)gs::cdiv(V * D, 32)), dim3(256), 0, stream, (const float*)part, (int)f.blocks, (int)(V * D), scale, (T*)dw);
        GS_LAUNCH_CHECK();
        return 0;
    }
    const SortPlan p = sort_plan(tokens, D);
    uint32_t *keys = nullptr, *pos = nullptr;
    if (tokens > 0)
        if (const int rc = sort_tokens<I>(ids, tokens, V, padding, p, base, keys, pos, stream)) return rc;
    float *first = (float*)(base + p.first), *last = (float*)(base + p.last);
    // The gradient stays in the caches for its next reader.  Written past them it is alone 2 .. 30 % faster (82 MB 92 us for 109, 164 MB 104 for 132), but 2 .. 6 % slower with the
    // clipping behind it (149 for 146, 203 for 195), and with clipping and HipAdam (355 for 349, 513 for 504).
    const int rows = rows_a_wave(V), clear_log = group_log_of(gs::cdiv(D, 16 / sizeof(T)));
    const int64_t zero_blocks = gs::cdiv(V, 4 * rows);
    constexpr int V16 = 16 / sizeof(T), V8 = 8 / sizeof(T);
    // Which sums: by the row's size alone, not by where g lies (they add the tokens of a long run in different orders).  Rows of 256 .. 512 bytes, 65536 tokens of 128 fp32 over 50000
    // rows: k_sum_wide with 8 bytes a lane 46 us, k_sum_chunks 49; 262144 of 256 bf16 89 and 102.
    const int64_t row = D * (int64_t)sizeof(T);
    const bool wide = row > 256;
    const int vec = row <= 512 ? V8 : vector_of(sizeof(T), D, ldg, g, dw);
    const int64_t vectors = gs::cdiv(D, BVEC);
    const int gl = group_log_of(vectors);
    const int64_t stretches = gs::cdiv(vectors, 1ll << gl);          // of the narrow sums
    if (wide) {
        const int64_t across = gs::cdiv(gs::cdiv(D, vec), 64), sum_blocks = gs::cdiv(p.chunks * across, 4);
        GS_REQUIRE(sum_blocks + zero_blocks < (1ll << 24), "gs_embedding_bwd: too large for one launch");
        const auto kernel = vec == V16 ? k_sum_wide<T, V16> : k_sum_wide<T, V8>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(sum_blocks + zero_blocks)), dim3(256), 0, stream, (const uint32_t*)keys, (const uint32_t*)pos, (const T*)g, ldg, tokens, V, D,
                           across, p.chunks, sum_blocks, rows, clear_log, scale, (T*)dw, first, last);
    } else {
        const int64_t sum_blocks = gs::cdiv((p.chunks * stretches) << gl, 256);
        GS_REQUIRE(sum_blocks + zero_blocks < (1ll << 24), "gs_embedding_bwd: too large for one launch");
        hipLaunchKernelGGL(k_sum_chunks<T>, dim3((unsigned)(sum_blocks + zero_blocks)), dim3(256), 0, stream, (const uint32_t*)keys, (const uint32_t*)pos, (const T*)g, ldg, tokens, V, D,
                           gl, stretches, p.chunks, sum_blocks, rows, clear_log, scale, (T*)dw, first, last);
    }
    if (p.chunks > 1) {
        // groups cover a whole row; a run may hold most of the tokens: a large workgroup where rows are used a thousand times and more
        const int threads = wide ? (tokens > V * 1000 ? 1024 : 512) : 256;
        int jl = 0;
        while (jl < 8 && (1ll << jl) < vectors) ++jl;
        const int64_t gx = p.chunks < (1 << 20) ? p.chunks : 1 << 20;          // a launch has fewer than 2^32 lanes either way of its grid
        hipLaunchKernelGGL(k_join_chunks<T>, dim3((unsigned)gx, (unsigned)gs::cdiv(p.chunks, gx)), dim3(threads), 0, stream, (const uint32_t*)keys, tokens, V, D, jl, gs::cdiv(vectors, 1ll << jl),
                           wide ? CHUNK + 1 : 1, scale, (const float*)first, (const float*)last, (T*)dw);
    }
    GS_LAUNCH_CHECK();
    return 0;
}

static bool sizes_ok(int64_t T, int64_t V, int64_t D) {
    const int64_t top = (1ll << 31) - 1;
    return T >= 0 && V >= 0 && D >= 0 && T < top && V < top && D < top;
}

static int64_t bytes_of(int64_t T, int64_t V, int64_t D) {
    const FewPlan f = few_plan(T, V, D);
    return f.threads ? align256(f.bytes + 1) : sort_plan(T, D).total;
}

}  // namespace

extern "C" int gs_embedding_fwd(const void* ids, int ids64, const void* weight, int64_t ldw, int64_t T, int64_t V, int64_t D, int dtype, float scale, void* y, gs_stream_t stream) {
    GS_REQUIRE(sizes_ok(T, V, D), "gs_embedding_fwd: sizes are 0 .. 2^31 - 2");
    GS_REQUIRE(dtype >= 0 && dtype <= 2, "gs_embedding_fwd: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (T == 0 || D == 0) return 0;
    GS_REQUIRE(ids && y && (weight || V == 0) && ldw >= 0, "gs_embedding_fwd: null argument");
    const auto run = dtype == 0 ? (ids64 ? lookup<float, int64_t> : lookup<float, int32_t>) : dtype == 1 ? (ids64 ? lookup<bf16, int64_t> : lookup<bf16, int32_t>)
                                                                                            : (ids64 ? lookup<f16, int64_t> : lookup<f16, int32_t>);
    return run(ids, weight, ldw, T, V, D, scale, y, (hipStream_t)stream);
}

extern "C" int64_t gs_embedding_bwd_workspace_bytes(int64_t T, int64_t V, int64_t D) { return sizes_ok(T, V, D) ? bytes_of(T, V, D) : -1; }

extern "C" int gs_embedding_bwd(const void* ids, int ids64, const void* g, int64_t ldg, int64_t T, int64_t V, int64_t D, int64_t padding_idx, int dtype, float scale, void* dw,
                                void* workspace, int64_t workspace_bytes, gs_stream_t stream) {
    GS_REQUIRE(sizes_ok(T, V, D), "gs_embedding_bwd: sizes are 0 .. 2^31 - 2");
    GS_REQUIRE(dtype >= 0 && dtype <= 2, "gs_embedding_bwd: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
    if (V == 0 || D == 0) return 0;
    GS_REQUIRE(dw && (T == 0 || (ids && g && ldg >= 0)), "gs_embedding_bwd: null argument");
    GS_REQUIRE(workspace && workspace_bytes >= bytes_of(T, V, D), "gs_embedding_bwd: workspace too small");
    GS_REQUIRE(((uintptr_t)workspace & 15) == 0, "gs_embedding_bwd: the workspace must start on 16 bytes");
    const auto run = dtype == 0 ? (ids64 ? gradient<float, int64_t> : gradient<float, int32_t>) : dtype == 1 ? (ids64 ? gradient<bf16, int64_t> : gradient<bf16, int32_t>)
                                                                                             : (ids64 ? gradient<f16, int64_t> : gradient<f16, int32_t>);
    return run(ids, g, ldg, T, V, D, padding_idx, scale, dw, (char*)workspace, (hipStream_t)stream);
}

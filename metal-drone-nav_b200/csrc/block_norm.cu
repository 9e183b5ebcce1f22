// The norms around a block with its gate and residual scale, and their
// gradients:
//   h = x + scale * act(gate) * (branch / rms(branch) * branch_weight)
//   y = h / rms(h) * norm_weight
// Bound by memory: every array goes through the chip once, a row's values stay
// in registers between its sums and its outputs. Rows that fill no more than a
// warp's registers belong to one warp (sums by shuffles, no barrier), longer
// ones to one block. 131,072 rows of 480 in bf16 with a gate: 118 us, 5.3 TB/s
// of the 6.55 TB/s that a copy reaches.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "host_common.h"

namespace mdn {
namespace {

using bf16 = __nv_bfloat16;

// 1 / (1 + e^-z) with the hardware's exponential and quotient: off by a few
// units in the last place where it is not small, by 2 + |z| of e^-z where it is.
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

// A thread's share of a row: N values, in vectors of eight consecutive ones
// (V = 8: every row on a 16-byte boundary) or single ones (V = 1), dealt to
// the row's `threads` threads in turn.
template <int V>
__device__ __forceinline__ uint32_t place(uint32_t e, uint32_t tid, uint32_t threads) {
    return V == 8 ? ((e >> 3) * threads + tid) * 8 + (e & 7) : e * threads + tid;
}

// What a thread fetches of a row, as it lies in memory. Fetching and unpacking
// are apart so that all of a row's loads are under way before the first is
// waited for (no branch between them); a place past the row's end fetches its
// last values and unpacks to zeros.
template <class T, int V>
struct Word;
template <>
struct Word<float, 1> {
    float x;
    __device__ void load(const float* p) { x = __ldcs(p); }
    __device__ void unpack(float* y) const { y[0] = x; }
};
template <>
struct Word<bf16, 1> {
    unsigned short x;
    __device__ void load(const bf16* p) { x = __ldcs(reinterpret_cast<const unsigned short*>(p)); }
    __device__ void unpack(float* y) const { y[0] = __uint_as_float(uint32_t(x) << 16); }
};
template <>
struct Word<float, 8> {
    float4 a, b;
    __device__ void load(const float* p) {
        a = __ldcs(reinterpret_cast<const float4*>(p));
        b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ void unpack(float* y) const {
        y[0] = a.x, y[1] = a.y, y[2] = a.z, y[3] = a.w, y[4] = b.x, y[5] = b.y, y[6] = b.z, y[7] = b.w;
    }
};
template <>
struct Word<bf16, 8> {
    uint4 a;
    __device__ void load(const bf16* p) { a = __ldcs(reinterpret_cast<const uint4*>(p)); }
    __device__ void unpack(float* y) const {
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            y[2 * i] = __uint_as_float(w[i] << 16);
            y[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};

__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
    __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(x[4], x[5], x[6], x[7]));
}
__device__ __forceinline__ void store8(bf16* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
}
__device__ __forceinline__ void put(float* p, float x) { __stcs(p, x); }
__device__ __forceinline__ void put(bf16* p, float x) {
    __stcs(reinterpret_cast<unsigned short*>(p), __bfloat16_as_ushort(__float2bfloat16_rn(x)));
}

// FULL: the first values of a thread's N that lie inside every row this variant
// is used for; their addresses need no care.
template <int FULL, class T, int V, int N>
__device__ __forceinline__ void fetch_row(Word<T, V> (&w)[N], const mdn_matrix& m, uint64_t row, uint32_t dim,
                                          uint32_t tid, uint32_t threads) {
    if (!m.data) return;
    const T* p = static_cast<const T*>(m.data) + int64_t(row) * m.row;
#pragma unroll
    for (int e = 0; e < N; e++)
        w[e].load(p + (e * V < FULL ? place<V>(e * V, tid, threads) : min(place<V>(e * V, tid, threads), dim - V)));
}
// Zeros where there is no matrix or the row has ended.
template <int FULL, class T, int V, int N>
__device__ __forceinline__ void unpack_row(float (&x)[N * V], const Word<T, V> (&w)[N], const mdn_matrix& m,
                                           uint32_t dim, uint32_t tid, uint32_t threads) {
#pragma unroll
    for (int e = 0; e < N; e++) {
        float y[V];
        w[e].unpack(y);
        const bool in = m.data && (e * V < FULL || place<V>(e * V, tid, threads) < dim);
#pragma unroll
        for (int k = 0; k < V; k++) x[e * V + k] = in ? y[k] : 0.0f;
    }
}
template <int FULL, class T, int V, int N>
__device__ __forceinline__ void store_row(const float (&x)[N], const mdn_matrix& m, uint64_t row, uint32_t dim,
                                          uint32_t tid, uint32_t threads) {
    if (!m.data) return;
    T* p = static_cast<T*>(m.data) + int64_t(row) * m.row;
#pragma unroll
    for (int e = 0; e < N; e += V) {
        const uint32_t i = place<V>(e, tid, threads);
        if (e >= FULL && i >= dim) continue;
        if constexpr (V == 8) {
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; k++) y[k] = x[e + k];
            store8(p + i, y);
        } else {
            put(p + i, x[e]);
        }
    }
}

// A weight's values beside a thread's share of a row; ones where there is none.
template <int FULL, int V, int N>
__device__ __forceinline__ void load_weight(float (&x)[N], const float* w, uint32_t dim, uint32_t tid,
                                            uint32_t threads) {
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = 1.0f;
    if (!w) return;
#pragma unroll
    for (int e = 0; e < N; e += V) {  // past the end: any of its values
        const uint32_t i = e < FULL ? place<V>(e, tid, threads) : min(place<V>(e, tid, threads), dim - V);
        if constexpr (V == 8) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(w + i)), b = __ldg(reinterpret_cast<const float4*>(w + i) + 1);
            x[e] = a.x, x[e + 1] = a.y, x[e + 2] = a.z, x[e + 3] = a.w;
            x[e + 4] = b.x, x[e + 5] = b.y, x[e + 6] = b.z, x[e + 7] = b.w;
        } else {
            x[e] = __ldg(w + i);
        }
    }
}

// Sums over the threads of a row: a warp, or the block (`turn` picks one of
// two sets of shared slots, so that one barrier a sum is enough).
template <bool WARP, int N>
__device__ __forceinline__ void row_sums(float (&x)[N], float (&slots)[2][N][32], uint32_t turn, uint32_t threads) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
        for (int n = 0; n < N; n++) x[n] += __shfl_xor_sync(~0u, x[n], o);
    if constexpr (!WARP) {
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int n = 0; n < N; n++) slots[turn][n][threadIdx.x >> 5] = x[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; n++) x[n] = 0.0f;
        for (uint32_t w = 0; w < threads / 32; w++)
#pragma unroll
            for (int n = 0; n < N; n++) x[n] += slots[turn][n][w];
    }
}

__device__ __forceinline__ float rms_factor(float squares, float inv, const mdn_block_norm& c) {
    const float x = squares * inv + c.eps, r = rsqrtf(x);
    return x > 0.0f && r > 0.0f ? r * fmaf(-0.5f * x * r, r, 1.5f) : r;  // a Newton step on the estimate
}

// WARP: a row belongs to a warp, four rows to a block; otherwise to the block.
template <class TS, class T, int V, int N, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 512) k_block_norm_forward(const __grid_constant__ mdn_block_norm c) {
    __shared__ float slots[2][1][32];
    const uint32_t threads = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    const uint64_t row = WARP ? uint64_t(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= c.rows) return;  // whole warps, where rows are warps
    constexpr int FULL = !WARP ? 0 : V == 8 ? N - 8 : N - 4;
    const float inv = 1.0f / float(c.dim);
    float h[N], sum[1];
    Word<TS, V> xw[N / V];
    Word<T, V> mw[N / V], zw[N / V];
    fetch_row<FULL>(mw, c.branch, row, c.dim, tid, threads);
    fetch_row<FULL>(zw, c.gate, row, c.dim, tid, threads);
    fetch_row<FULL>(xw, c.x, row, c.dim, tid, threads);
    unpack_row<FULL>(h, xw, c.x, c.dim, tid, threads);
    if (c.branch.data) {
        float m[N], z[N];
        unpack_row<FULL>(m, mw, c.branch, c.dim, tid, threads);
        unpack_row<FULL>(z, zw, c.gate, c.dim, tid, threads);
        sum[0] = 0.0f;
#pragma unroll
        for (int e = 0; e < N; e++) sum[0] = fmaf(m[e], m[e], sum[0]);
        row_sums<WARP, 1>(sum, slots, 0, threads);
        const float rb = rms_factor(sum[0], inv, c);
        if (c.gate.data) {
            const bool silu = c.gate_act == MDN_GATE_SILU;
#pragma unroll
            for (int e = 0; e < N; e++) m[e] *= sigmoid(z[e]) * (silu ? z[e] : 1.0f);
        }
        load_weight<FULL, V, N>(z, c.branch_weight, c.dim, tid, threads);
#pragma unroll
        for (int e = 0; e < N; e++) m[e] *= rb * z[e];
        load_weight<FULL, V, N>(z, c.residual_scale, c.dim, tid, threads);
#pragma unroll
        for (int e = 0; e < N; e++) h[e] = fmaf(m[e], z[e], h[e]);
        store_row<FULL, TS, V, N>(h, c.h, row, c.dim, tid, threads);
    }
    if (!c.y.data) return;
    sum[0] = 0.0f;
#pragma unroll
    for (int e = 0; e < N; e++) sum[0] = fmaf(h[e], h[e], sum[0]);
    row_sums<WARP, 1>(sum, slots, 1, threads);
    const float rh = rms_factor(sum[0], inv, c);
    float w[N];
    load_weight<FULL, V, N>(w, c.norm_weight, c.dim, tid, threads);
#pragma unroll
    for (int e = 0; e < N; e++) h[e] *= rh * w[e];
    store_row<FULL, T, V, N>(h, c.y, row, c.dim, tid, threads);
}

// The gradient of row * r, r = 1 / rms(row): of one value `unit` = row[i] r, from the gradient d of that value and
// mean = mean over the row of gradient * unit: r (d - unit mean). A row of one value has the slope eps r^3, where the
// difference would cancel to noise: there keep = eps r^2 and mean = 0, elsewhere keep = 1.
__device__ __forceinline__ float norm_slope(float r, float keep, float d, float unit, float mean) {
    return r * fmaf(-unit, mean, d * keep);
}

// Blocks of the gradient kernel, each with its own sums for the weights: what
// an SM holds at about 16 warps.
// A row has the fewest threads that hold it in eight values each, or in up to
// twelve where they are single: more rows on an SM hide more of the memory's
// latency than more values a thread do.
uint32_t row_threads(uint32_t dim, uint32_t most) {
    uint32_t threads = 32;
    while (threads < 1024 && threads * (threads < 512 ? most : 8) < dim) threads *= 2;
    return threads;
}
constexpr uint32_t sm_blocks(uint32_t threads) { return threads == 32 ? 4 : threads >= 512 ? 1 : 512 / threads; }

// Each block takes every gridDim-th row (or four rows) and keeps the sums for
// the weights' gradients of its columns in registers. 32,768 rows of 515 (no row
// on a 16-byte boundary), bf16 beside a 32-bit stream: 102 us, and 168 us with
// the forward pass and the weights' last sums. There the instructions count:
// about 100 a value, most of them for single values' loads and stores; values
// whose place is known to lie inside every row cost a third less than guarded
// ones (274 us before), and one sum for both weights of the branch saves another.
template <class TS, class T, int V, int N, int THREADS>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS, sm_blocks(THREADS)) k_block_norm_backward(const __grid_constant__ mdn_block_norm c,
                                                              const __grid_constant__ mdn_block_norm_grads g) {
    constexpr bool WARP = THREADS == 32;
    constexpr int FULL = V == 8 ? 0 : N - 2;
    constexpr uint32_t threads = THREADS;
    __shared__ float slots3[2][3][32], slots1[2][1][32];
    const uint32_t tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    const uint64_t first = WARP ? uint64_t(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
    const uint64_t step = WARP ? uint64_t(gridDim.x) * 4 : gridDim.x;
    const mdn_matrix hm = c.branch.data ? c.h : c.x;
    const float inv = 1.0f / float(c.dim);
    // sums over rows of dy h / rms(h), and of dh act branch / rms(branch): times residual_scale the gradient of
    // branch_weight, times branch_weight that of residual_scale
    float wn[N], wa[N];
#pragma unroll
    for (int e = 0; e < N; e++) wn[e] = wa[e] = 0.0f;
    uint32_t turn = 0;
    for (uint64_t row = first; row < c.rows; row += step, turn ^= 1) {
        float h[N], dy[N], dh[N], m[N], z[N];
        Word<TS, V> hw[N / V], dhw[N / V];
        Word<T, V> dyw[N / V], mw[N / V], zw[N / V];
        fetch_row<FULL>(hw, hm, row, c.dim, tid, threads);
        fetch_row<FULL>(dyw, g.dy, row, c.dim, tid, threads);
        fetch_row<FULL>(mw, c.branch, row, c.dim, tid, threads);
        fetch_row<FULL>(dhw, g.dh, row, c.dim, tid, threads);
        fetch_row<FULL>(zw, c.gate, row, c.dim, tid, threads);
        unpack_row<FULL>(h, hw, hm, c.dim, tid, threads);
        unpack_row<FULL>(dy, dyw, g.dy, c.dim, tid, threads);
        unpack_row<FULL>(m, mw, c.branch, c.dim, tid, threads);
        unpack_row<FULL>(dh, dhw, g.dh, c.dim, tid, threads);
        unpack_row<FULL>(z, zw, c.gate, c.dim, tid, threads);
        float w[N], r[N], sum[3] = {0.0f, 0.0f, 0.0f};
        load_weight<FULL, V, N>(w, c.norm_weight, c.dim, tid, threads);
#pragma unroll
        for (int e = 0; e < N; e++) {
            sum[0] = fmaf(h[e], h[e], sum[0]);
            sum[1] = fmaf(dy[e] * w[e], h[e], sum[1]);
            if (c.branch.data) sum[2] = fmaf(m[e], m[e], sum[2]);
        }
        row_sums<WARP, 3>(sum, slots3, turn, threads);
        const bool single = c.dim == 1;
        const float rh = rms_factor(sum[0], inv, c), mean = single ? 0.0f : sum[1] * rh * inv;
        const float keep = single ? c.eps * rh * rh : 1.0f;
#pragma unroll
        for (int e = 0; e < N; e++) {  // zeros past the end of the row
            const float hat = h[e] * rh;
            wn[e] = fmaf(dy[e], hat, wn[e]);
            if (g.dy.data) dh[e] += norm_slope(rh, keep, dy[e] * w[e], hat, mean);
        }
        store_row<FULL, TS, V, N>(dh, g.dx, row, c.dim, tid, threads);
        if (!c.branch.data) continue;
        const float rb = rms_factor(sum[2], inv, c);
        float total[1] = {0.0f};
        load_weight<FULL, V, N>(w, c.branch_weight, c.dim, tid, threads);
        load_weight<FULL, V, N>(r, c.residual_scale, c.dim, tid, threads);
        const bool silu = c.gate_act == MDN_GATE_SILU;
#pragma unroll
        for (int e = 0; e < N; e++) {  // m: its unit value, h: the gradient of that, z: the gate's gradient
            float act = 1.0f, slope = 0.0f;
            if (c.gate.data) {  // z p or p, p (1 - p) z + p or p (1 - p)
                const float p = sigmoid(z[e]), zz = silu ? z[e] : 1.0f;
                act = p * zz;
                slope = fmaf(p * (1.0f - p), zz, silu ? p : 0.0f);
            }
            m[e] *= rb;
            const float both = w[e] * r[e], da = dh[e] * act;
            wa[e] = fmaf(da, m[e], wa[e]);
            z[e] = dh[e] * both * (m[e] * slope);
            h[e] = da * both;
            total[0] = fmaf(h[e], m[e], total[0]);
        }
        store_row<FULL, T, V, N>(z, g.dgate, row, c.dim, tid, threads);
        row_sums<WARP, 1>(total, slots1, turn, threads);
        total[0] = single ? 0.0f : total[0] * inv;
        const float keep_b = single ? c.eps * rb * rb : 1.0f;
#pragma unroll
        for (int e = 0; e < N; e++) h[e] = norm_slope(rb, keep_b, h[e], m[e], total[0]);
        store_row<FULL, T, V, N>(h, g.dbranch, row, c.dim, tid, threads);
    }
    if constexpr (WARP) {  // the four warps' sums together, in order
        __shared__ float joined[2][32 * N];
        for (uint32_t w = 0; w < 4; w++) {
            __syncthreads();
            if (threadIdx.x >> 5 != w) continue;
#pragma unroll
            for (int e = 0; e < N; e++) {
                const uint32_t i = place<V>(e, tid, threads);
                joined[0][i] = w ? joined[0][i] + wn[e] : wn[e];
                joined[1][i] = w ? joined[1][i] + wa[e] : wa[e];
            }
        }
        __syncthreads();
        float* part = static_cast<float*>(g.workspace) + size_t(blockIdx.x) * 2 * c.dim;
        for (uint32_t k = 0; k < 2; k++)
            for (uint32_t i = threadIdx.x; i < c.dim; i += 128) part[k * c.dim + i] = joined[k][i];
    } else {
        float* part = static_cast<float*>(g.workspace) + size_t(blockIdx.x) * 2 * c.dim;
#pragma unroll
        for (int e = 0; e < N; e++) {
            const uint32_t i = place<V>(e, tid, threads);
            if (i < c.dim) part[i] = wn[e], part[c.dim + i] = wa[e];
        }
    }
}

// The blocks' sums of 32 columns: 32 warps take every 32nd block, joined in
// order.
__global__ void __launch_bounds__(1024) k_block_norm_weights(const __grid_constant__ mdn_block_norm c,
                                                            const __grid_constant__ mdn_block_norm_grads g,
                                                            uint32_t blocks) {
    __shared__ float sums[32][32];
    const uint32_t i = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5, kind = blockIdx.y;
    const float* part = static_cast<const float*>(g.workspace) + size_t(kind) * c.dim + i;
    float sum = 0.0f;
    if (i < c.dim) {
#pragma unroll 8
        for (uint32_t b = slice; b < blocks; b += 32) sum += part[size_t(b) * 2 * c.dim];
    }
    sums[slice][threadIdx.x & 31] = sum;
    __syncthreads();
    if (slice || i >= c.dim) return;
    for (int w = 1; w < 32; w++) sum += sums[w][threadIdx.x];
    // a gradient whose input was absent is not written, except that no rows leave zeros in all
    const bool branch = c.branch.data || c.rows == 0;
    if (kind == 0) {
        if (g.dnorm_weight && (c.norm_weight || c.rows == 0)) g.dnorm_weight[i] = sum;
    } else if (branch) {
        if (g.dbranch_weight && (c.branch_weight || c.rows == 0))
            g.dbranch_weight[i] = sum * (c.residual_scale ? c.residual_scale[i] : 1.0f);
        if (g.dresidual_scale && (c.residual_scale || c.rows == 0))
            g.dresidual_scale[i] = sum * (c.branch_weight ? c.branch_weight[i] : 1.0f);
    }
}

bool even_weights(const mdn_block_norm& c) {
    return (reinterpret_cast<uintptr_t>(c.branch_weight) | reinterpret_cast<uintptr_t>(c.residual_scale) |
            reinterpret_cast<uintptr_t>(c.norm_weight)) % 16 == 0;
}
// Whether every row starts on a 16-byte boundary (eight bf16 or four floats).
bool even_rows(const mdn_matrix& m, uint32_t dtype) {
    const int64_t per = dtype == MDN_F32 ? 4 : 8;
    return reinterpret_cast<uintptr_t>(m.data) % 16 == 0 && m.row % per == 0;
}

constexpr uint32_t kWarpDim = 768;  // the longest rows that one warp takes forward

// Calls f with the fewest values a lane (in steps of 4, or of 8) that hold a row.
template <class F>
void by_share(uint32_t dim, int v, F&& f) {
    const uint32_t n = (dim + 31) / 32;
    if (n <= 4 && v == 1) f(std::integral_constant<int, 4>());
    else if (n <= 8) f(std::integral_constant<int, 8>());
    else if (n <= 12 && v == 1) f(std::integral_constant<int, 12>());
    else if (n <= 16) f(std::integral_constant<int, 16>());
    else if (n <= 20 && v == 1) f(std::integral_constant<int, 20>());
    else f(std::integral_constant<int, 24>());
}

template <class TS, class T, int V>
void forward(const mdn_block_norm& c, cudaStream_t s) {
    if (c.dim <= kWarpDim)
        by_share(c.dim, V, [&](auto n) {
            constexpr int N = decltype(n)::value;
            if constexpr (N % V == 0)
                k_block_norm_forward<TS, T, V, N, true><<<unsigned((c.rows + 3) / 4), 128, 0, s>>>(c);
        });
    else k_block_norm_forward<TS, T, V, 16, false><<<unsigned(c.rows), (c.dim + 511) / 512 * 32, 0, s>>>(c);
}
template <class TS, class T>
void forward(const mdn_block_norm& c, cudaStream_t s) {
    const bool even = c.dim % 8 == 0 && even_weights(c) && even_rows(c.x, c.stream_dtype) && even_rows(c.branch, c.dtype) &&
                      even_rows(c.gate, c.dtype) && even_rows(c.h, c.stream_dtype) && even_rows(c.y, c.dtype);
    if (even) forward<TS, T, 8>(c, s);
    else forward<TS, T, 1>(c, s);
}
void forward(const mdn_block_norm& c, cudaStream_t s) {
    if (c.stream_dtype == MDN_F32) return c.dtype == MDN_F32 ? forward<float, float>(c, s) : forward<float, bf16>(c, s);
    return c.dtype == MDN_F32 ? forward<bf16, float>(c, s) : forward<bf16, bf16>(c, s);
}

template <class TS, class T, int V, int N, int THREADS>
unsigned backward_rows(const mdn_block_norm& c, const mdn_block_norm_grads& g, cudaStream_t s) {
    const uint64_t needed = THREADS == 32 ? (c.rows + 3) / 4 : c.rows;
    const unsigned blocks = unsigned(std::min<uint64_t>(needed, 148 * sm_blocks(THREADS)));
    if (blocks) k_block_norm_backward<TS, T, V, N, THREADS><<<blocks, std::max(THREADS, THREADS == 32 ? 128 : 0), 0, s>>>(c, g);
    return blocks;
}
template <class TS, class T>
unsigned backward_vectors(const mdn_block_norm& c, const mdn_block_norm_grads& g, cudaStream_t s) {
    switch (row_threads(c.dim, 8)) {
        case 32: return backward_rows<TS, T, 8, 8, 32>(c, g, s);
        case 64: return backward_rows<TS, T, 8, 8, 64>(c, g, s);
        case 128: return backward_rows<TS, T, 8, 8, 128>(c, g, s);
        case 256: return backward_rows<TS, T, 8, 8, 256>(c, g, s);
        case 512: return backward_rows<TS, T, 8, 8, 512>(c, g, s);
        default: return backward_rows<TS, T, 8, 8, 1024>(c, g, s);
    }
}
// Single values: the fewest a thread, in steps of two.
template <class TS, class T, int THREADS>
unsigned backward_singles(const mdn_block_norm& c, const mdn_block_norm_grads& g, cudaStream_t s) {
    const uint32_t n = (c.dim + THREADS - 1) / THREADS;
    if constexpr (THREADS == 32) {
        if (n <= 2) return backward_rows<TS, T, 1, 2, THREADS>(c, g, s);
        if (n <= 4) return backward_rows<TS, T, 1, 4, THREADS>(c, g, s);
    }
    if constexpr (THREADS == 32 || THREADS == 1024)
        if (n <= 6) return backward_rows<TS, T, 1, 6, THREADS>(c, g, s);
    if (n <= 8 || THREADS >= 512) return backward_rows<TS, T, 1, 8, THREADS>(c, g, s);
    if constexpr (THREADS < 512) {
        if (n <= 10) return backward_rows<TS, T, 1, 10, THREADS>(c, g, s);
        return backward_rows<TS, T, 1, 12, THREADS>(c, g, s);
    }
    return 0;
}
template <class TS, class T>
unsigned backward_singles(const mdn_block_norm& c, const mdn_block_norm_grads& g, cudaStream_t s) {
    switch (row_threads(c.dim, 12)) {
        case 32: return backward_singles<TS, T, 32>(c, g, s);
        case 64: return backward_singles<TS, T, 64>(c, g, s);
        case 128: return backward_singles<TS, T, 128>(c, g, s);
        case 256: return backward_singles<TS, T, 256>(c, g, s);
        case 512: return backward_singles<TS, T, 512>(c, g, s);
        default: return backward_singles<TS, T, 1024>(c, g, s);
    }
}
template <class TS, class T>
unsigned backward(const mdn_block_norm& c, const mdn_block_norm_grads& g, cudaStream_t s) {
    const bool even = c.dim % 8 == 0 && even_weights(c) && even_rows(c.branch.data ? c.h : c.x, c.stream_dtype) &&
                      even_rows(c.branch, c.dtype) && even_rows(c.gate, c.dtype) && even_rows(g.dh, c.stream_dtype) &&
                      even_rows(g.dy, c.dtype) && even_rows(g.dx, c.stream_dtype) && even_rows(g.dbranch, c.dtype) &&
                      even_rows(g.dgate, c.dtype);
    return even ? backward_vectors<TS, T>(c, g, s) : backward_singles<TS, T>(c, g, s);
}
unsigned backward(const mdn_block_norm& c, const mdn_block_norm_grads& g, cudaStream_t s) {
    if (c.stream_dtype == MDN_F32)
        return c.dtype == MDN_F32 ? backward<float, float>(c, g, s) : backward<float, bf16>(c, g, s);
    return c.dtype == MDN_F32 ? backward<bf16, float>(c, g, s) : backward<bf16, bf16>(c, g, s);
}

void check_call(const mdn_block_norm* c, const char* who) {
    const std::string at = std::string(who) + ": ";
    require(c, MDN_ERR_INVALID, at + "null call");
    require(c->dim >= 1 && c->dim <= MDN_NORM_MAX_DIM, MDN_ERR_INVALID, at + "dim must be 1..8192");
    require(c->rows <= 0x7fffffffu, MDN_ERR_INVALID, at + "rows exceeds 2^31 - 1");
    require(c->dtype <= MDN_BF16 && c->stream_dtype <= MDN_BF16, MDN_ERR_INVALID,
            at + "dtypes must be MDN_F32 or MDN_BF16");
    require(c->gate_act <= MDN_GATE_SILU, MDN_ERR_INVALID, at + "unknown gate activation");
    require(std::isfinite(c->eps) && c->eps >= 0.0f, MDN_ERR_INVALID, at + "eps must be finite and not negative");
}
void check_matrix(const mdn_matrix& m, uint32_t dtype, bool needed, const char* who, const char* name) {
    require(m.data || !needed, MDN_ERR_INVALID, std::string(who) + ": " + name + " is null");
    require(reinterpret_cast<uintptr_t>(m.data) % (dtype == MDN_F32 ? 4 : 2) == 0, MDN_ERR_INVALID,
            std::string(who) + ": " + name + " is not aligned to its type");
}

}  // namespace
}  // namespace mdn

extern "C" size_t mdn_block_norm_workspace_bytes(const mdn_block_norm* call) {
    using namespace mdn;
    size_t n = 0;
    guarded([&] {
        check_call(call, "mdn_block_norm_workspace_bytes");
        n = size_t(148) * 8 * 2 * call->dim * sizeof(float);  // of the most blocks that any variant has
    });
    return n;
}

extern "C" int mdn_block_norm_forward(const mdn_block_norm* call, void* stream) {
    using namespace mdn;
    return guarded([&] {
        const char* who = "mdn_block_norm_forward";
        check_call(call, who);
        const mdn_block_norm& c = *call;
        if (c.rows == 0) return;
        check_matrix(c.x, c.stream_dtype, true, who, "x");
        check_matrix(c.branch, c.dtype, false, who, "branch");
        check_matrix(c.gate, c.dtype, false, who, "gate");
        check_matrix(c.h, c.stream_dtype, false, who, "h");
        check_matrix(c.y, c.dtype, false, who, "y");
        require(c.branch.data || !c.gate.data, MDN_ERR_INVALID, "mdn_block_norm_forward: a gate without a branch");
        require((c.branch.data && c.h.data) || c.y.data, MDN_ERR_INVALID, "mdn_block_norm_forward: no output");
        forward(c, static_cast<cudaStream_t>(stream));
        cuda_check(cudaGetLastError(), who);
    });
}

extern "C" int mdn_block_norm_backward(const mdn_block_norm* call, const mdn_block_norm_grads* grads, void* stream) {
    using namespace mdn;
    return guarded([&] {
        const char* who = "mdn_block_norm_backward";
        check_call(call, who);
        require(grads, MDN_ERR_INVALID, "mdn_block_norm_backward: null grads");
        const mdn_block_norm& c = *call;
        const mdn_block_norm_grads& g = *grads;
        require(g.workspace && reinterpret_cast<uintptr_t>(g.workspace) % 16 == 0, MDN_ERR_INVALID,
                "mdn_block_norm_backward: workspace is null or not 16-byte aligned");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (c.rows) {
            check_matrix(c.branch, c.dtype, false, who, "branch");
            check_matrix(c.gate, c.dtype, false, who, "gate");
            if (c.branch.data) check_matrix(c.h, c.stream_dtype, true, who, "h");
            else check_matrix(c.x, c.stream_dtype, true, who, "x");
            check_matrix(g.dh, c.stream_dtype, false, who, "dh");
            check_matrix(g.dy, c.dtype, false, who, "dy");
            check_matrix(g.dx, c.stream_dtype, false, who, "dx");
            check_matrix(g.dbranch, c.dtype, false, who, "dbranch");
            check_matrix(g.dgate, c.dtype, false, who, "dgate");
            require(c.branch.data || !c.gate.data, MDN_ERR_INVALID, "mdn_block_norm_backward: a gate without a branch");
        }
        const unsigned blocks = backward(c, g, s);
        cuda_check(cudaGetLastError(), who);
        k_block_norm_weights<<<dim3((c.dim + 31) / 32, 2), 1024, 0, s>>>(c, g, blocks);
        cuda_check(cudaGetLastError(), "mdn_block_norm_backward: weights");
    });
}

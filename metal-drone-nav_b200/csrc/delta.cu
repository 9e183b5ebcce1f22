// The gated delta rule on sm_100a: a policy's recurrent memory over a rollout
// (any number of steps, one included) and its gradients.
//
//   S <- a_t S,  u_t = b_t (v_t - S^T k_t),  S <- S + k_t u_t^T,  o_t = s S^T q_t
//
// with a_t = exp(log_decay_t) and S [key][value] per environment and head.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "host_common.h"

namespace mdn {
namespace {

constexpr int kCell = 16;  // steps between two saved states

using bf16 = __nv_bfloat16;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void store(float* p, float x) { *p = x; }
__device__ __forceinline__ void store(bf16* p, float x) { *p = __float2bfloat16_rn(x); }

__host__ __device__ __forceinline__ uint32_t padded_key(uint32_t dk) { return dk <= 32 ? 32 : dk <= 64 ? 64 : 128; }

template <class T>
__device__ __forceinline__ T* row_ptr(const mdn_rows& r, uint32_t t, uint32_t env, uint32_t head) {
    return static_cast<T*>(r.data) + int64_t(t) * r.step + int64_t(env) * r.env + int64_t(head) * r.head;
}

__device__ __forceinline__ uint32_t live_steps(const mdn_delta& c, uint32_t env) {
    if (!c.lengths) return c.steps;
    const int32_t n = c.lengths[env];
    return n <= 0 ? 0u : min(uint32_t(n), c.steps);
}

// 1 / sqrt(x), the hardware's estimate with a Newton step.
__device__ __forceinline__ float unit_factor(float x) {
    const float r = rsqrtf(x);
    return x > 0.0f && r > 0.0f ? r * fmaf(-0.5f * x * r, r, 1.5f) : r;
}

// ------------------------------------------------------------------ tick
// One step (the policy tick): the state is read once, held in registers, and
// written once. Bound by those bytes. Both products with the state are taken
// in the one pass, with o = s (a S)^T q + s (q.k) u in place of a second pass
// over the new state. A group of GT threads holds one state, 32 values a
// thread: column units of V values (V = 4: 16-byte accesses) across lanes, and
// NI = 32 / V consecutive rows for each of the GT / CP row groups. GT = 32
// keeps all sums inside a warp; larger states join their warps' sums in shared
// memory. 65,536 environments x 4 heads of 32 x 32: 423 us, 5.3 TB/s; 8,192 x 4
// of 64 x 64: 204 us, 5.4 TB/s, of 6.55 TB/s that a copy reaches. Six blocks of
// 128 an SM hide more latency than five (230 us), at the price of a few spills;
// GT = 32 is best left to the compiler's 93 registers.
template <class T, int V, int GT>
__global__ void __launch_bounds__(GT < 128 ? 128 : GT, V == 4 && GT >= 128 ? 768 / GT : 0) k_delta_tick(const __grid_constant__ mdn_delta c, int log_cp) {
    constexpr int NI = 32 / V, kWarps = GT / 32, kGroups = GT < 128 ? 128 / GT : 1;
    constexpr int kWide = 128;  // the widest axis
    __shared__ float sums[kWarps > 1 ? kWarps : 1][2][kWarps > 1 ? kWide : 1];
    __shared__ __align__(16) float keys[kGroups][2][kWide];  // k, q; zeros past the last
    const uint32_t item = blockIdx.x * kGroups + threadIdx.x / GT, tid = threadIdx.x % GT, lane = threadIdx.x & 31;
    if (item >= c.envs * c.heads) return;  // only whole groups leave, and only where groups are warps
    const uint32_t env = item / c.heads, head = item % c.heads, qh = head / (c.heads / c.qk_heads);
    const uint32_t dk = c.key_dim, dv = c.value_dim;
    const uint32_t col = (tid & ((1u << log_cp) - 1)) * V, r0 = (tid >> log_cp) * NI;
    const bool mine = col < dv;
    const size_t state = size_t(item) * dk * dv;
    const bool live = live_steps(c, env) != 0;
    const bool fresh = live && c.starts && c.starts[int64_t(env) * c.starts_env];
    float S[NI][V];
    const float* p = c.state_in + state + size_t(r0) * dv + col;
    const bool read = mine && c.state_in && !fresh;
#pragma unroll
    for (int i = 0; i < NI; i++, p += dv) {
#pragma unroll
        for (int e = 0; e < V; e++) S[i][e] = 0.0f;
        if (read && r0 + i < dk) {
            if constexpr (V == 4) {
                const float4 x = __ldcs(reinterpret_cast<const float4*>(p));
                S[i][0] = x.x, S[i][1] = x.y, S[i][2] = x.z, S[i][3] = x.w;
            } else {
                S[i][0] = __ldcs(p);
            }
        }
    }
    if (live) {
        float(&keyq)[2][kWide] = keys[threadIdx.x / GT];
        const T* qp = row_ptr<T>(c.q, 0, env, qh);
        const T* kp = row_ptr<T>(c.k, 0, env, qh);
        for (uint32_t i = tid; i < kWide; i += GT) {
            keyq[0][i] = i < dk ? to_float(kp[i]) : 0.0f;
            keyq[1][i] = i < dk ? to_float(qp[i]) : 0.0f;
        }
        const float a = expf(*row_ptr<float>(c.log_decay, 0, env, head));
        const float b = *row_ptr<float>(c.beta, 0, env, head);
        float v[V];
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = mine ? to_float(row_ptr<T>(c.v, 0, env, head)[col + e]) : 0.0f;
        if constexpr (kWarps > 1) __syncthreads();
        else __syncwarp();
        float qq = 0.0f, kk = 0.0f, qk = 0.0f;
        for (uint32_t i = lane; i < dk; i += 32) {
            const float x = keyq[1][i], y = keyq[0][i];
            qq = fmaf(x, x, qq), kk = fmaf(y, y, kk), qk = fmaf(x, y, qk);
        }
        for (int o = 16; o; o >>= 1) {
            qq += __shfl_xor_sync(~0u, qq, o);
            kk += __shfl_xor_sync(~0u, kk, o);
            qk += __shfl_xor_sync(~0u, qk, o);
        }
        float rq = 1.0f, rk = 1.0f;
        if (c.flags & MDN_DELTA_NORMALIZE) rq = unit_factor(qq + c.norm_eps), rk = unit_factor(kk + c.norm_eps);
        float ks[V] = {}, qs[V] = {}, k[NI];
#pragma unroll
        for (int i = 0; i < NI; i += 4) {
            float4 kr = make_float4(0.0f, 0.0f, 0.0f, 0.0f), qr = kr;
            if (r0 + i < kWide) {
                kr = *reinterpret_cast<const float4*>(&keyq[0][r0 + i]);
                qr = *reinterpret_cast<const float4*>(&keyq[1][r0 + i]);
            }
            const float q[4] = {qr.x, qr.y, qr.z, qr.w};
            k[i] = kr.x, k[i + 1] = kr.y, k[i + 2] = kr.z, k[i + 3] = kr.w;
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int e = 0; e < V; e++) {
                    S[i + n][e] *= a;
                    ks[e] = fmaf(k[i + n], S[i + n][e], ks[e]);
                    qs[e] = fmaf(q[n], S[i + n][e], qs[e]);
                }
        }
        for (int o = 16; o >= (1 << log_cp); o >>= 1) {
#pragma unroll
            for (int e = 0; e < V; e++) {
                ks[e] += __shfl_xor_sync(~0u, ks[e], o);
                qs[e] += __shfl_xor_sync(~0u, qs[e], o);
            }
        }
        if constexpr (kWarps > 1) {
            // Columns of one warp: all of them (CP <= 32), or the warp's own stretch of a wider axis.
            const uint32_t warp = tid >> 5;
            if (mine && (lane >> min(log_cp, 5)) == 0) {
#pragma unroll
                for (int e = 0; e < V; e++) sums[warp][0][col + e] = ks[e], sums[warp][1][col + e] = qs[e];
            }
            __syncthreads();
            const uint32_t stride = log_cp > 5 ? 1u << (log_cp - 5) : 1u;  // warps that share these columns
#pragma unroll
            for (int e = 0; e < V; e++) ks[e] = qs[e] = 0.0f;
            if (mine)
                for (uint32_t w = warp % stride; w < kWarps; w += stride) {
#pragma unroll
                    for (int e = 0; e < V; e++) ks[e] += sums[w][0][col + e], qs[e] += sums[w][1][col + e];
                }
        }
        float u[V];
#pragma unroll
        for (int e = 0; e < V; e++) {
            u[e] = b * (v[e] - rk * ks[e]);
            const float o = c.scale * rq * fmaf(qk * rk, u[e], qs[e]);
            if (mine && r0 == 0) store(row_ptr<T>(c.out, 0, env, head) + col + e, o);
            u[e] *= rk;
        }
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int e = 0; e < V; e++) S[i][e] = fmaf(k[i], u[e], S[i][e]);
    } else if (mine && r0 == 0) {
#pragma unroll
        for (int e = 0; e < V; e++) store(row_ptr<T>(c.out, 0, env, head) + col + e, 0.0f);
    }
    if (!c.state_out || !mine) return;
    float* d = c.state_out + state + size_t(r0) * dv + col;
#pragma unroll
    for (int i = 0; i < NI; i++, d += dv) {
        if (r0 + i >= dk) break;
        if constexpr (V == 4) __stcs(reinterpret_cast<float4*>(d), make_float4(S[i][0], S[i][1], S[i][2], S[i][3]));
        else __stcs(d, S[i][0]);
    }
}

// ---------------------------------------------------------------- chunks
// A rollout goes in chunks of up to 16 steps that cross no episode start.
// With G_ij = prod_{l=j+1..i} a_l and g_i = prod_{l<=i} a_l, a chunk that
// begins with the state S is a linear system for w_t = v_t - (a_t S_{t-1})^T k_t:
//   X = V - g K S,  A_ij = G_ij (k_i.k_j) b_j below the diagonal,
//   W = (I + A)^-1 X,
//   O_i = s g_i q_i S + sum_{j<=i} s G_ij (q_i.k_j) b_j w_j,
//   S' = g_C S + sum_j G_Cj b_j k_j w_j^T,
// all products of at least 16 x 16 x 16: tensor-core work. The decay products
// G are built by multiplication, so full forgetting (a = 0) needs no care.
//
// Precision: the tensor cores multiply bf16. A 32-bit value is cut into three
// bf16 parts of 8 significant bits each, which hold it exactly, and products
// of parts i and j are taken where i + j <= 2: what is left out is about 2^-25
// of the product. bf16 inputs are one exact part.
//
// A warp holds 16 value columns of the state, S^T as the accumulator layout of
// m16n8k16: rows = value columns, so that it is the A operand of the next
// chunk's products without leaving the registers. m16n8k16 rather than
// tcgen05: a 16-step chunk needs 3 d^2 + 64 d products a step where the
// 128-row tcgen05 tile (chunks of 64 or more steps) needs 3 d^2 + 320 d, and the
// 32-bit state would go through tensor memory and shared memory for its three
// parts every chunk, on the chain that bounds the rollout.

constexpr int kMatRow = 48;     // bytes of a 16-value bf16 row of a 16 x 16 matrix: 8 rows, 8 bank groups
constexpr int kScratchRow = 20;  // floats of a 16-value row in the producer's scratch
constexpr int kFactorRow = 36;   // the same with room for what lies past the triangle

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x and y to the nearest bf16 as a packed pair.
__device__ __forceinline__ uint32_t round_pair(float x, float y) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}
// The same, and x and y become what is left: three times over holds them
// exactly. Rounded rather than cut off, so that what a product leaves out has
// no common sign.
__device__ __forceinline__ uint32_t cut(float& x, float& y) {
    const uint32_t r = round_pair(x, y);
    x -= __uint_as_float(r << 16);
    y -= __uint_as_float(r & 0xffff0000u);
    return r;
}
// Two accumulator tiles (16 rows x 16 columns) as the N parts of an A operand.
template <int N>
__device__ __forceinline__ void cut_tiles(const float (&t0)[4], const float (&t1)[4], uint32_t (&p)[N][4]) {
    float x[8] = {t0[0], t0[1], t0[2], t0[3], t1[0], t1[1], t1[2], t1[3]};
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) p[n][r] = cut(x[2 * r], x[2 * r + 1]);
}
// d0, d1 += A B over one k step of 16, for the products of orders `from` down
// to `to`, smallest first.
template <int NA, int NB>
__device__ __forceinline__ void mma_orders(float (&d0)[4], float (&d1)[4], const uint32_t (&a)[NA][4],
                                           const uint32_t (&b)[NB][4], int from, int to) {
#pragma unroll
    for (int order = from; order >= to; order--)
#pragma unroll
        for (int i = 0; i < NA; i++) {
            const int j = order - i;
            if (j < 0 || j >= NB) continue;
            mma(d0, a[i], b[j][0], b[j][1]);
            mma(d1, a[i], b[j][2], b[j][3]);
        }
}
template <int NA, int NB>
__device__ __forceinline__ void mma_parts(float (&d0)[4], float (&d1)[4], const uint32_t (&a)[NA][4],
                                          const uint32_t (&b)[NB][4]) {
    mma_orders(d0, d1, a, b, 2, 0);
}
// The same with the small products (order 1 and 2) in accumulators of their
// own: the tensor cores round every accumulation toward zero, which over
// several k steps costs bits where large and small products share a sum.
template <int NA, int NB>
__device__ __forceinline__ void mma_parts(float (&d0)[4], float (&d1)[4], float (&e0)[4], float (&e1)[4],
                                          const uint32_t (&a)[NA][4], const uint32_t (&b)[NB][4]) {
    mma_orders(e0, e1, a, b, 2, 1);
    mma_orders(d0, d1, a, b, 0, 0);
}

// For a result that is stored as bf16 the operands have two parts and the
// product of both second parts is left out: 2^-18 where the store rounds at 2^-9;
// with three parts all products count.
template <int NA, int NB>
__device__ __forceinline__ void mma_out(float (&d0)[4], float (&d1)[4], const uint32_t (&a)[NA][4],
                                        const uint32_t (&b)[NB][4]) {
    mma_orders(d0, d1, a, b, NA == 2 || NB == 2 ? 1 : 2, 0);
}

// Lane offsets of the 8 x 8 blocks that ldmatrix.x4 fetches from rows of `row`
// bytes: block order by rows of the pair first, or by columns first.
__device__ __forceinline__ uint32_t lane_rows_first(uint32_t lane, uint32_t row) {
    return (((lane >> 3) & 1) * 8 + (lane & 7)) * row + (lane >> 4) * 16;
}
__device__ __forceinline__ uint32_t lane_cols_first(uint32_t lane, uint32_t row) {
    return ((lane >> 4) * 8 + (lane & 7)) * row + ((lane >> 3) & 1) * 16;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A piece of work in the stream that a CTA goes through: a chunk of an item
// (the value columns of one block of one environment and head).
struct ChunkMeta {
    uint32_t t, n;   // first step, steps (0: an item without any)
    uint32_t flags;
    uint32_t bh;     // environment x heads + head
    uint32_t env, head, qh, v0;
};
// An episode starts at t; the item's first, last chunk; the end of the stream;
// an item of the segment's map. From bit 8 on: the segment.
constexpr uint32_t kFresh = 1, kFirst = 2, kLast = 4, kDone = 8, kMap = 16;

// A long rollout of few environments is cut into segments of `cells` cells that
// run at once. A chunk is linear in the state it begins with, so a segment is
// S -> M S + b: pass kJoin runs every segment but the last from zeros (its last
// state is b) and, on no values, from the unit matrix (its last state is M, as
// columns of a memory of key_dim values); k_delta_carry goes through them for
// the state that each segment begins with; pass kRun computes the outputs.
// Twice to three times the work, over so many more SMs.
enum Pass : uint32_t { kRun = 0, kJoin = 1 };
struct Segments {
    uint32_t count, cells;
    Pass pass;
    // The state that each segment begins with, [count][envs x heads][key][value] (the first one's is a copy, as the last
    // segment may write over it), and the maps of all but the last, [count - 1][envs x heads][key][key].
    float *carry, *map;
};

__host__ __device__ inline uint32_t value_blocks(const mdn_delta& c) { return (c.value_dim + 63) / 64; }

// Walks the chunks of items first, first + stride, ... in order: cells of 16
// steps, cut at episode starts. One warp holds it; the next cell's start flags
// are fetched a cell ahead.
struct ChunkWalk {
    const uint8_t* starts;
    uint32_t item, items, stride, live, cell_t, pos, mask, next_flag;
    uint32_t bh, env, head, qh, v0, kind;
    bool open;  // inside an item
    __device__ void begin(uint32_t first, uint32_t items_, uint32_t stride_) {
        item = first, items = items_, stride = stride_, open = false;
    }
    __device__ uint32_t flag(const mdn_delta& c, uint32_t t, uint32_t lane) const {
        return starts && lane < kCell && t + lane < live ? starts[int64_t(t + lane) * c.starts_step] : 0u;
    }
    template <bool SPLIT>
    __device__ ChunkMeta next(const mdn_delta& c, const Segments& g, uint32_t lane) {
        uint32_t first = 0;
        if (!open) {
            if (item >= items) return ChunkMeta{0, 0, kDone};
            const uint32_t values = value_blocks(c);
            const uint32_t blocks = SPLIT && g.pass == kJoin ? values + (c.key_dim + 63) / 64 : values;
            uint32_t rest = item;
            kind = cell_t = 0;
            if constexpr (SPLIT) {
                const uint32_t all = c.envs * c.heads * blocks, segment = item / all;
                rest -= segment * all;
                kind = segment << 8;
                cell_t = segment * g.cells * kCell;
            }
            bh = rest / blocks, env = bh / c.heads, head = bh - env * c.heads;
            qh = head / (c.heads / c.qk_heads), v0 = rest - bh * blocks;
            live = live_steps(c, env);
            if constexpr (SPLIT) {
                if (v0 >= values) kind |= kMap, v0 -= values;
                if ((kind >> 8) + 1 < g.count) live = min(live, cell_t + g.cells * kCell);
            }
            v0 *= 64;
            starts = c.starts ? c.starts + int64_t(env) * c.starts_env : nullptr;
            pos = 0;
            const uint32_t now = flag(c, cell_t, lane);
            next_flag = flag(c, cell_t + kCell, lane);
            mask = __ballot_sync(~0u, now);
            open = true;
            first = kFirst;
        }
        ChunkMeta m{cell_t + pos, 0, kind | first, bh, env, head, qh, v0};
        if (cell_t + pos < live) {
            const uint32_t later = mask & ~((2u << pos) - 1);
            uint32_t end = later ? __ffs(later) - 1 : kCell;
            end = min(end, live - cell_t);
            m.n = end - pos;
            if ((mask >> pos) & 1) m.flags |= kFresh;
            pos = end;
            if (pos == kCell) {
                pos = 0;
                cell_t += kCell;
                mask = __ballot_sync(~0u, next_flag);
                next_flag = flag(c, cell_t + kCell, lane);
            }
        }
        if (cell_t + pos >= live) {
            m.flags |= kLast;
            open = false;
            item = items - item > stride ? item + stride : items;
        }
        return m;
    }
};

// Rows off 16-byte boundaries, value by value; out of line, as the instructions
// that an SM has at hand are what the rollout kernel runs short of.
template <class T>
__device__ __noinline__ void fetch_singles(const T* base, int64_t step, uint32_t dim, uint32_t n, char* dst,
                                           uint32_t width, uint32_t row, uint32_t lane) {
    for (uint32_t e = lane; e < kCell * width; e += 32) {
        const uint32_t r = e / width, col = e % width;
        T x = T(0.0f);
        if (r < n && col < dim) x = base[int64_t(r) * step + col];
        *reinterpret_cast<T*>(dst + r * row + col * sizeof(T)) = x;
    }
}

// n <= 16 rows of `dim` values from `base` on into shared rows of ROW bytes,
// WIDTH values wide; what lies past `dim` or past the rows is zeros.
template <class T, int WIDTH, int ROW>
__device__ __forceinline__ void fetch_rows(const T* base, int64_t step, bool vec, uint32_t dim, uint32_t n, char* dst,
                                           uint32_t lane) {
    if (vec) {
        constexpr uint32_t per = 16 / sizeof(T), granules = WIDTH / per, rows = 32 / granules;
        const uint32_t r0 = lane / granules, col = lane % granules * per;
        const uint32_t bytes = col < dim ? min(per, dim - col) * uint32_t(sizeof(T)) : 0u;
        const T* p = bytes ? base + int64_t(r0) * step + col : base;
        const int64_t jump = rows * step;
        const uint32_t d = smem_addr(dst) + r0 * ROW + lane % granules * 16;
#pragma unroll
        for (uint32_t r = 0; r < kCell; r += rows) {
            const uint32_t got = r0 + r < n ? bytes : 0u;
            cp_async16(d + r * ROW, got ? p : base, got);
            p += jump;
        }
    } else {
        fetch_singles(base, step, dim, n, dst, WIDTH, ROW, lane);
    }
}

// log_decay and beta of a chunk's steps into shared memory; zeros past n.
// `p`: of the lane's own array (lanes 0..15: log_decay) at the first step.
__device__ __forceinline__ void fetch_scalars(const float* p, int64_t step, uint32_t n, float* dst, uint32_t lane) {
    const uint32_t r = lane & (kCell - 1);
    cp_async4(smem_addr(dst + lane), r < n ? p + int64_t(r) * step : p, r < n ? 4 : 0);
}

// Where an environment and head's rows begin.
template <class T>
struct Bases {
    const T *q, *k, *v;
    const float* scalars;  // log_decay in lanes 0..15, beta in lanes 16..31
    int64_t scalars_step;
    __device__ __forceinline__ void set(const mdn_delta& c, uint32_t env, uint32_t head, uint32_t qh, uint32_t v0,
                                        uint32_t lane) {
        q = row_ptr<T>(c.q, 0, env, qh);
        k = row_ptr<T>(c.k, 0, env, qh);
        v = row_ptr<T>(c.v, 0, env, head) + v0;
        scalars = row_ptr<float>(lane < kCell ? c.log_decay : c.beta, 0, env, head);
        scalars_step = lane < kCell ? c.log_decay.step : c.beta.step;
    }
};

// 16 rows of DK values (of type T, rows of raw_row bytes) as bf16 parts.
template <int DK, int ROW>
__device__ __forceinline__ void cut_rows(const char* raw, uint32_t raw_row, char* parts, uint32_t lane) {
#pragma unroll 4
    for (uint32_t e = lane; e < kCell * DK / 4; e += 32) {
        const uint32_t r = e / (DK / 4), col = e % (DK / 4) * 4;
        float4 x = *reinterpret_cast<const float4*>(raw + r * raw_row + col * 4);
#pragma unroll
        for (int p = 0; p < 3; p++) {
            uint2 y;
            y.x = cut(x.x, x.y);
            y.y = cut(x.z, x.w);
            *reinterpret_cast<uint2*>(parts + p * kCell * ROW + r * ROW + col * 2) = y;
        }
    }
}

// Sum of squares of the 32-bit row that two lanes share (lane / 2), in both.
template <int DK>
__device__ __forceinline__ float row_squares(const char* raw, uint32_t raw_row, uint32_t lane) {
    const float* p = reinterpret_cast<const float*>(raw + (lane >> 1) * raw_row) + (lane & 1) * (DK / 2);
    float sum[4] = {};
#pragma unroll
    for (int i = 0; i < DK / 2; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(p + i);
        sum[0] = fmaf(x.x, x.x, sum[0]), sum[1] = fmaf(x.y, x.y, sum[1]);
        sum[2] = fmaf(x.z, x.z, sum[2]), sum[3] = fmaf(x.w, x.w, sum[3]);
    }
    const float s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    return s + __shfl_xor_sync(~0u, s, 1);
}

__device__ __forceinline__ void load16(float (&x)[16], const float* p) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        const float4 y = *reinterpret_cast<const float4*>(p + i);
        x[i] = y.x, x[i + 1] = y.y, x[i + 2] = y.z, x[i + 3] = y.w;
    }
}

// k_j.k_i and k_j.q_i of a chunk's steps as [j][i], and |q_j|^2 where the
// inputs are single bf16 parts (`squares`).
template <int NP, int DK, int ROW>
__device__ __forceinline__ void key_products(const char* keys, const char* queries, float* kk, float* kq,
                                             float* squares, uint32_t lane) {
    const uint32_t g = lane >> 2, t = lane & 3, qp = smem_addr(queries), kp = smem_addr(keys);
    float dk0[4] = {}, dk1[4] = {}, dq0[4] = {}, dq1[4] = {}, qq0[4] = {}, qq1[4] = {};
#pragma unroll 1
    for (int kb = 0; kb < DK / 16; kb++) {
        uint32_t ak[NP][4], bk[NP][4], bq[NP][4];
#pragma unroll
        for (int p = 0; p < NP; p++) {
            ldsm4(ak[p], kp + p * kCell * ROW + kb * 32 + lane_rows_first(lane, ROW));
            ldsm4(bq[p], qp + p * kCell * ROW + kb * 32 + lane_cols_first(lane, ROW));
            // the same blocks in the other order
            bk[p][0] = ak[p][0], bk[p][1] = ak[p][2], bk[p][2] = ak[p][1], bk[p][3] = ak[p][3];
        }
        mma_parts<NP, NP>(dk0, dk1, ak, bk);
        mma_parts<NP, NP>(dq0, dq1, ak, bq);
        if constexpr (NP == 1) {
            const uint32_t aq[1][4] = {{bq[0][0], bq[0][2], bq[0][1], bq[0][3]}};
            mma_parts<1, 1>(qq0, qq1, aq, bq);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t at = (g + 8 * h) * kScratchRow + 2 * t;
        *reinterpret_cast<float2*>(kk + at) = make_float2(dk0[2 * h], dk0[2 * h + 1]);
        *reinterpret_cast<float2*>(kk + at + 8) = make_float2(dk1[2 * h], dk1[2 * h + 1]);
        *reinterpret_cast<float2*>(kq + at) = make_float2(dq0[2 * h], dq0[2 * h + 1]);
        *reinterpret_cast<float2*>(kq + at + 8) = make_float2(dq1[2 * h], dq1[2 * h + 1]);
    }
    if constexpr (NP == 1) {
        if (t == g >> 1) {
            squares[g] = g & 1 ? qq0[1] : qq0[0];
            squares[8 + g] = g & 1 ? qq1[3] : qq1[2];
        }
    }
}

// Column j of (I + A)^-1 by forward substitution, each step's value subtracted
// from all later ones. `cols`: A as [j][i].
__device__ __forceinline__ void substitute(float (&col)[16], const float* cols, uint32_t j) {
#pragma unroll
    for (int i = 0; i < kCell; i++) col[i] = i == int(j) ? 1.0f : 0.0f;
#pragma unroll
    for (int l = 0; l < kCell - 1; l++) {
        float al[16];
        load16(al, cols + l * kScratchRow);
#pragma unroll
        for (int i = l + 1; i < kCell; i++) col[i] = fmaf(-al[i], col[l], col[i]);
    }
}

// A column as a row of the three parts of a matrix kept as [j][i].
__device__ __forceinline__ void store_parts(float (&col)[16], char* dst) {
#pragma unroll
    for (int p = 0; p < 3; p++) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = cut(col[2 * i], col[2 * i + 1]);
        *reinterpret_cast<uint4*>(dst + p * kCell * kMatRow) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(dst + p * kCell * kMatRow + 16) = make_uint4(w[4], w[5], w[6], w[7]);
    }
}

// The forward kernel's stages, each on a chunk of its own while four warps
// compute chunk i: one warp fetches chunk i + kLead and finishes the matrices of
// chunk i + 1, one starts those of chunk i + 2. Rows live in rings of slots. i is the step that reads, j the step that wrote: c (I + A)^-1 is
// kept as [j][i], P (I + A)^-1 as [i][j].
template <class T, int DK>
struct Forward {
    static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
    // 32-bit rows are twice as long and have parts beside them: one chunk less in flight leaves room for two blocks.
    static constexpr int kPending = kParts == 1 ? 1 : 0, kLead = 3 + kPending, kRing = kLead + 1;
    static constexpr int kKeyRing = kParts == 1 ? kRing : 2;    // raw queries and keys go once their parts are there
    static constexpr int kRow = DK * 2 + 16;                    // a bf16 part's row
    static constexpr int kRawRow = DK * int(sizeof(T)) + 16;
    static constexpr int kRawV = 64 * int(sizeof(T)) + 16;
    static constexpr int kKeys = 2 * kCell * kRawRow;           // queries, keys
    static constexpr int kSlotS = kCell * kRawV, kSlot = kSlotS + 128 + 32;  // values, 16 log-decays and betas, ChunkMeta
    static constexpr int kStageK = kParts == 3 ? 3 * kCell * kRow : 0;  // after the queries' parts
    static constexpr int kStageT = 2 * kStageK;                 // three parts of c (I + A)^-1, then of P (I + A)^-1
    static constexpr int kStageP = kStageT + 3 * kCell * kMatRow;
    static constexpr int kStageVec = kStageP + 3 * kCell * kMatRow;  // g_k[16], g_q[16], c[16], g_C
    static constexpr int kStage = kStageVec + 3 * 64 + 16;
    // P with its columns reversed; 15 rows for what lies past it, and before the next; -A with both axes reversed; -A
    // as [j][i]; decay[16], zeros[16], 1/|k|[16], scale/|q|[16], and 32 that are read beside them
    static constexpr int kBack = 31 * kFactorRow, kForth = 47 * kFactorRow, kDecay = 63 * kFactorRow;
    static constexpr int kFactors = kDecay + 96;
    // shared memory
    static constexpr int kSlots = kKeyRing * kKeys, kStages = kSlots + kRing * kSlot, kFactor = kStages + 3 * kStage;
    static constexpr int kScratch = kFactor + 2 * kFactors * 4;  // k.k, k.q, |q|^2[16]
    static constexpr size_t kSmem = size_t(kScratch) + 2 * kCell * kScratchRow * 4 + 64;

    char* smem;

    __device__ explicit Forward(char* base) : smem(base) {}
    __device__ char* rows(uint32_t i) const { return smem + i % kKeyRing * kKeys; }
    __device__ char* slot(uint32_t i) const { return smem + kSlots + i % kRing * kSlot; }
    __device__ char* stage(uint32_t i) const { return smem + kStages + i % 3 * kStage; }
    __device__ float* factors(uint32_t i) const { return reinterpret_cast<float*>(smem + kFactor) + (i & 1) * kFactors; }
    __device__ ChunkMeta* meta(uint32_t i) const { return reinterpret_cast<ChunkMeta*>(slot(i) + kSlotS + 128); }
    // The bf16 parts of chunk i's queries and keys.
    __device__ const char* queries(uint32_t i) const { return kParts == 1 ? rows(i) : stage(i); }
    __device__ const char* keys(uint32_t i) const { return kParts == 1 ? rows(i) + kCell * kRawRow : stage(i) + kStageK; }

    // values: the value columns to fetch
    __device__ void fetch(const mdn_delta& c, uint32_t vec, const ChunkMeta& m, const Bases<T>& at, uint32_t values,
                          uint32_t i, uint32_t lane) const {
        char* dst = slot(i);
        if (lane == 0) *meta(i) = m;
        if (m.n) {
            char* key_rows = rows(i);
            fetch_rows<T, DK, kRawRow>(at.q + int64_t(m.t) * c.q.step, c.q.step, vec & 1, c.key_dim, m.n, key_rows, lane);
            fetch_rows<T, DK, kRawRow>(at.k + int64_t(m.t) * c.k.step, c.k.step, vec & 2, c.key_dim, m.n,
                                       key_rows + kCell * kRawRow, lane);
            fetch_rows<T, 64, kRawV>(at.v + int64_t(m.t) * c.v.step, c.v.step, vec & 4,
                                     values, m.n, dst, lane);
            fetch_scalars(at.scalars + int64_t(m.t) * at.scalars_step, at.scalars_step, m.n,
                          reinterpret_cast<float*>(dst + kSlotS), lane);
        }
        if (m.flags & kFirst && c.state_in && !(m.flags & kFresh) && m.flags < 256) {  // the state, on its way to the L2 cache
            const char* p = reinterpret_cast<const char*>(c.state_in + size_t(m.bh) * c.key_dim * c.value_dim);
            const uint32_t bytes = c.key_dim * c.value_dim * 4;
            for (uint32_t b = lane * 128; b < bytes; b += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + b));
        }
        cp_async_commit();
    }

    // Once, before the first chunk: zeros where nothing is written later.
    __device__ void prepare_first(uint32_t lane) const {
        float* p = factors(0);
        for (uint32_t i = lane; i < 2 * kFactors; i += 32) p[i] = 0.0f;
        __syncwarp();
    }

    // Chunk `index`'s products of keys and queries and its decays: -A, P and the factors.
    __device__ void start(const mdn_delta& c, uint32_t index, uint32_t lane) const {
        const uint32_t n = meta(index)->n;
        char* st = stage(index);
        float* kk = reinterpret_cast<float*>(smem + kScratch);
        float *kq = kk + kCell * kScratchRow, *squares = kq + kCell * kScratchRow;
        float *pr = factors(index), *back = pr + kBack, *forth = pr + kForth, *a = pr + kDecay;
        float* fac = reinterpret_cast<float*>(st + kStageVec);
        const float x = reinterpret_cast<const float*>(slot(index) + kSlotS)[lane];  // log_decay, beta
        const float decay = expf(x), beta = __shfl_sync(~0u, x, 16 + (lane & 15));
        if (lane < kCell) a[lane] = decay;
        if constexpr (kParts == 3) {
            cut_rows<DK, kRow>(rows(index) + kCell * kRawRow, kRawRow, st + kStageK, lane);
            const float sum = row_squares<DK>(rows(index), kRawRow, lane);
            if (!(lane & 1)) squares[lane >> 1] = sum;
            asm volatile("bar.sync 2, 64;" ::: "memory");  // the other warp cuts the queries
        }
        key_products<kParts, DK, kRow>(keys(index), queries(index), kk, kq, squares, lane);
        // g_j = prod_{l<=j} a_l in lanes j, and G_Cj = prod_{l>j} a_l (steps past the chunk's have a = 1)
        const uint32_t j = lane & 15;
        const bool low = lane < 16;
        float lead = __shfl_sync(~0u, decay, j), tail = __shfl_down_sync(~0u, lead, 1, 16);
        if (j == 15) tail = 1.0f;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            const float up = __shfl_up_sync(~0u, lead, o, 16), down = __shfl_down_sync(~0u, tail, o, 16);
            if (j >= uint32_t(o)) lead *= up;
            if (j + o < 16) tail *= down;
        }
        __syncwarp();
        float r = 1.0f;
        if (c.flags & MDN_DELTA_NORMALIZE) r = unit_factor((low ? kk[j * (kScratchRow + 1)] : squares[j]) + c.norm_eps);
        a[32 + lane] = low ? r : c.scale * r;
        const float rk = __shfl_sync(~0u, r, j);
        __syncwarp();
        const bool in = j < n;
        if (low) {
            fac[j] = in ? lead * r : 0.0f;
            fac[32 + j] = in ? tail * (rk * beta) : 0.0f;
            if (j + 1 == n) fac[48] = lead;
        } else {
            fac[16 + j] = in ? lead * (c.scale * r) : 0.0f;
        }
        // Lanes 0..15: column j of -A below the diagonal; lanes 16..31: of P. Step by step down from the diagonal
        // with the decays' product, so that a lane's elements are its own; past the last row the product is 0.
        {
            const float* dec = a + j;
            const float* left = a + (low ? 32 : 48) + j;
            const float* dot = (low ? kk : kq) + j * (kScratchRow + 1);
            const float bk = low ? -(rk * beta) : rk * beta;
            float run = 1.0f, y[16];
#pragma unroll
            for (int d = 0; d < kCell; d++) {  // all reads before the first write
                if (d) run *= dec[d];
                y[d] = run * left[d] * (bk * dot[d]);
            }
            // No branches: what lies past the triangle goes to rows and columns that nobody reads.
            float* out = low ? forth + j * (kFactorRow + 1) : pr + j * kFactorRow + (15 - j);
            float* rev = low ? back + (15 - j) * kFactorRow + (15 - j) : out;
            const int next = low ? 1 : kFactorRow, prev = low ? -kFactorRow : kFactorRow;
#pragma unroll
            for (int d = 0; d < kCell; d++) {
                *out = y[d];
                *rev = y[d];
                out += next;
                rev += prev;
            }
        }
    }

    // What is left of chunk `index`'s matrices.
    __device__ void finish(uint32_t index, uint32_t lane) const {
        char* st = stage(index);
        const float *pr = factors(index), *back = pr + kBack, *forth = pr + kForth;
        const uint32_t j = lane & 15;
        const bool low = lane < 16;
        // Lanes 0..15: column j of (I + A)^-1 by forward substitution. Lanes 16..31: row j of P (I + A)^-1 from its
        // last value to its first, the same steps on the reversed matrix. Each value goes to all later ones.
        float col[16];
        if (low) {
#pragma unroll
            for (int i = 0; i < kCell; i++) col[i] = i == int(j) ? 1.0f : 0.0f;
        } else {
            load16(col, pr + j * kFactorRow);
        }
        const float* step = low ? forth : back;
#pragma unroll
        for (int l = 0; l < kCell - 1; l++) {
            float row[16];
            load16(row, step + l * kFactorRow);
#pragma unroll
            for (int i = l + 1; i < kCell; i++) col[i] = fmaf(row[i], col[l], col[i]);
        }
        if (low) {
            float cs[16];
            load16(cs, reinterpret_cast<const float*>(st + kStageVec) + 32);
#pragma unroll
            for (int i = 0; i < kCell; i++) col[i] *= cs[i];
        } else {
#pragma unroll
            for (int i = 0; i < kCell / 2; i++) {
                const float y = col[i];
                col[i] = col[15 - i];
                col[15 - i] = y;
            }
        }
        store_parts(col, st + (low ? kStageT : kStageP) + j * kMatRow);
    }
};

// Values of two value columns (col, col + 1) of one step; apart where rows are
// not on pairs' boundaries, or have no second.
template <class T>
__device__ __forceinline__ void store_apart(T* p, uint32_t col, uint32_t cols, float x, float y) {
    if (col < cols) store(p + col, x);
    if (col + 1 < cols) store(p + col + 1, y);
}
template <class T>
__device__ __forceinline__ void store_two(T* p, bool pair, uint32_t col, uint32_t cols, float x, float y) {
    if (pair) {
        if (col >= cols) return;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p + col) = make_float2(x, y);
        else *reinterpret_cast<uint32_t*>(p + col) = round_pair(x, y);
    } else {
        store_apart(p, col, cols, x, y);
    }
}

// A CTA takes 64 value columns of one environment and head after the other; a
// warp for each 16 of them. 128 steps of 1,024 environments x 4 heads of 64 x 64
// in bf16: 315 us, six times the time of its bytes. Twelve warps an SM issue in
// 40% of the cycles: each chunk is a chain of products and cuts of some 2,800
// cycles in a warp, and the roles' code (about 30 KB) passes the instruction
// caches, so what is rarely reached is kept out of line. Two blocks an SM with
// 168 registers a thread; 112 registers allow no third (four warps a scheduler),
// and 96, which do, gave 338 us.
template <class T, int DK, bool SPLIT>
__global__ void __maxnreg__(168) k_delta_rollout(const __grid_constant__ mdn_delta c, uint32_t vec,
                                                                 uint32_t items, const __grid_constant__ Segments seg) {
    using F = Forward<T, DK>;
    constexpr int NP = F::kParts, NT = DK / 8;
    extern __shared__ __align__(16) char smem_raw[];
    const bool join = SPLIT && seg.pass == kJoin;
    const F f(smem_raw);
    const uint32_t warps = blockDim.x / 32 - 2, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == warps + 1) {
        ChunkWalk walk;
        walk.begin(blockIdx.x, items, gridDim.x);
        Bases<T> at;
        for (int i = -F::kLead;; i++) {
            if (i >= 0 && f.meta(i)->flags & kDone) break;
            if constexpr (NP == 3) {
                if (i + 2 >= 0 && f.meta(i + 2)->n) {
                    cut_rows<DK, F::kRow>(f.rows(i + 2), F::kRawRow, f.stage(i + 2), lane);
                    asm volatile("bar.sync 2, 64;" ::: "memory");
                }
            }
            const ChunkMeta m = walk.template next<SPLIT>(c, seg, lane);
            if (m.flags & kFirst) at.set(c, m.env, m.head, m.qh, SPLIT && m.flags & kMap ? 0 : m.v0, lane);
            f.fetch(c, vec, m, at, SPLIT && m.flags & kMap ? 0u : min(64u, c.value_dim - m.v0), i + F::kLead, lane);
            if (i + 1 >= 0 && f.meta(i + 1)->n) f.finish(i + 1, lane);
            cp_async_wait<F::kPending>();
            __syncthreads();
        }
        cp_async_wait<0>();
        return;
    }
    if (warp == warps) {
        f.prepare_first(lane);
        for (int i = -F::kLead;; i++) {
            if (i >= 0 && f.meta(i)->flags & kDone) break;
            if (i + 2 >= 0 && f.meta(i + 2)->n) f.start(c, i + 2, lane);
            __syncthreads();
        }
        return;
    }
    for (int i = -F::kLead; i < 0; i++) __syncthreads();
    // Row g of a warp's tile is value column 2 g, row g + 8 is 2 g + 1: a lane
    // then holds neighbours, and reads and writes them as pairs.
    const uint32_t g = lane >> 2, t4 = lane & 3, colw = warp * 16 + 2 * g, dv = c.value_dim;
    const uint32_t dvp = (dv + 15) / 16 * 16;
    float S[NT][4];
    for (uint32_t i = 0;; i++) {
        const ChunkMeta m = *f.meta(i);
        if (m.flags & kDone) break;
        const uint32_t col = m.v0 + colw;
        const size_t state = size_t(m.bh) * c.key_dim * dv;
        const uint32_t segment = SPLIT ? m.flags >> 8 : 0;
        const size_t all = size_t(c.envs) * c.heads * c.key_dim;  // rows of a segment's states
        if (m.flags & (kFirst | kFresh)) {
            const bool unit = SPLIT && m.flags & kMap && !(m.flags & kFresh);
            const float* from = join || m.flags & kFresh ? nullptr : SPLIT ? seg.carry + segment * all * dv : c.state_in;
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t r = 8 * j + 2 * t4 + e;
                    const float* p = from + state + size_t(r) * dv + col;
                    const bool in = from && r < c.key_dim;
                    float2 x = make_float2(0.0f, 0.0f);
                    if (vec & 128) {
                        if (in && col < dv) x = *reinterpret_cast<const float2*>(p);
                    } else {
                        if (in && col < dv) x.x = p[0];
                        if (in && col + 1 < dv) x.y = p[1];
                    }
                    if (SPLIT && unit) x = make_float2(r == col ? 1.0f : 0.0f, r == col + 1 ? 1.0f : 0.0f);
                    S[j][e] = x.x, S[j][2 + e] = x.y;
                }
        }
        if (m.n) {
            const char* st = f.stage(i);
            const float* fac = reinterpret_cast<const float*>(st + F::kStageVec);
            if (c.saved && !join && m.t % kCell == 0 && col < dvp) {
                float* d = static_cast<float*>(c.saved) +
                           (size_t(m.t / kCell) * c.envs * c.heads + m.bh) * c.key_dim * dvp + col;
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t r = 8 * j + 2 * t4 + e;
                        if (r < c.key_dim)
                            *reinterpret_cast<float2*>(d + size_t(r) * dvp) = make_float2(S[j][e], S[j][2 + e]);
                    }
            }
            const char* slot = f.slot(i);
            const uint32_t kp = smem_addr(f.keys(i)), qp = smem_addr(f.queries(i));
            // S^T K^T and S^T Q^T: [16 value columns x 16 steps] each
            float xk[2][4] = {}, xq[2][4] = {}, ek[2][4] = {}, eq[2][4] = {};
#pragma unroll
            for (int kb = 0; kb < DK / 16; kb++) {
                uint32_t a[3][4], bk[NP][4], bq[NP][4];
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    ldsm4(bk[p], kp + p * kCell * F::kRow + kb * 32 + lane_cols_first(lane, F::kRow));
                    if (!join) ldsm4(bq[p], qp + p * kCell * F::kRow + kb * 32 + lane_cols_first(lane, F::kRow));
                }
                cut_tiles<3>(S[2 * kb], S[2 * kb + 1], a);
                mma_parts<3, NP>(xk[0], xk[1], ek[0], ek[1], a, bk);
                if (!join) mma_parts<3, NP>(xq[0], xq[1], eq[0], eq[1], a, bq);
            }
            // X = V - g K S, and g Q S
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t s = 8 * n + 2 * t4 + e;
                    float v0, v1;
                    if constexpr (sizeof(T) == 2) {
                        const uint32_t x = *reinterpret_cast<const uint32_t*>(slot + s * F::kRawV + colw * 2);
                        v0 = __uint_as_float(x << 16), v1 = __uint_as_float(x & 0xffff0000u);
                    } else {
                        const float2 x = *reinterpret_cast<const float2*>(slot + s * F::kRawV + colw * 4);
                        v0 = x.x, v1 = x.y;
                    }
                    const float gk = fac[s], gq = fac[16 + s];
                    xk[n][e] = fmaf(-gk, xk[n][e] + ek[n][e], v0);
                    xk[n][2 + e] = fmaf(-gk, xk[n][2 + e] + ek[n][2 + e], v1);
                    xq[n][e] = gq * (xq[n][e] + eq[n][e]);
                    xq[n][2 + e] = gq * (xq[n][2 + e] + eq[n][2 + e]);
                }
            // c W and O = g Q S + P W, W = (I + A)^-1 X
            float u[2][4] = {}, o[2][4] = {};
            uint32_t parts[3][4], b[3][4];
            cut_tiles<3>(xk[0], xk[1], parts);
#pragma unroll
            for (int p = 0; p < 3; p++)
                ldsm4t(b[p], smem_addr(st + F::kStageT) + p * kCell * kMatRow + lane_rows_first(lane, kMatRow));
            mma_parts<3, 3>(u[0], u[1], parts, b);
            if (!join) {
#pragma unroll
                for (int p = 0; p < 3; p++)
                    ldsm4(b[p], smem_addr(st + F::kStageP) + p * kCell * kMatRow + lane_cols_first(lane, kMatRow));
                mma_parts<3, 3>(o[0], o[1], parts, b);
                T* out = row_ptr<T>(c.out, m.t, m.env, m.head);
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t s = 8 * n + 2 * t4 + e;
                        if (s < m.n)
                            store_two(out + int64_t(s) * c.out.step, vec & 8, col, dv, o[n][e] + xq[n][e],
                                      o[n][2 + e] + xq[n][2 + e]);
                    }
            }
            // S' = g_C S + (c W)^T K
            cut_tiles<3>(u[0], u[1], parts);
            const float gc = fac[48];
#pragma unroll
            for (int kb = 0; kb < DK / 16; kb++) {
                float d0[4] = {}, d1[4] = {};
                uint32_t bk[NP][4];
#pragma unroll
                for (int p = 0; p < NP; p++)
                    ldsm4t(bk[p], kp + p * kCell * F::kRow + kb * 32 + lane_rows_first(lane, F::kRow));
                mma_parts<3, NP>(d0, d1, parts, bk);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    S[2 * kb][e] = fmaf(gc, S[2 * kb][e], d0[e]);
                    S[2 * kb + 1][e] = fmaf(gc, S[2 * kb + 1][e], d1[e]);
                }
            }
        }
        if (m.flags & kLast) {
            float* to = c.state_out;
            uint32_t width = dv;
            if (join) {
                width = m.flags & kMap ? c.key_dim : dv;
                to = m.flags & kMap ? seg.map + segment * all * width : seg.carry + (segment + 1) * all * width;
            } else {
                const bool last = !SPLIT || segment + 1 == seg.count;
                const uint32_t end = last ? c.steps : (segment + 1) * seg.cells * kCell;
                for (uint32_t t = m.t + m.n + t4; t < end; t += 4)
                    store_two(row_ptr<T>(c.out, t, m.env, m.head), vec & 8, col, dv, 0.0f, 0.0f);
                if (!last) to = nullptr;
            }
            if (to) {
                to += size_t(m.bh) * c.key_dim * width;
                const bool pair = join ? width % 2 == 0 : (vec & 128) != 0;
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t r = 8 * j + 2 * t4 + e;
                        if (r < c.key_dim) store_two(to + size_t(r) * width, pair, col, width, S[j][e], S[j][2 + e]);
                    }
            }
        }
        __syncthreads();
    }
}

// The state that each segment but the first begins with, over its b: 16 value
// columns of one environment and head a block, four of them of one key row a
// thread. A map's zeros take nothing with them: what is not finite before a
// start stays there.
__global__ void __launch_bounds__(512) k_delta_carry(const __grid_constant__ mdn_delta c,
                                                     const __grid_constant__ Segments seg) {
    __shared__ __align__(16) float now[2][128][16];
    const uint32_t dk = c.key_dim, dv = c.value_dim, r = threadIdx.x >> 2, e0 = (threadIdx.x & 3) * 4;
    const uint32_t col = blockIdx.y * 16 + e0, env = blockIdx.x / c.heads, cols = col < dv ? min(4u, dv - col) : 0u;
    const size_t rows = size_t(c.envs) * c.heads * dk, row = size_t(blockIdx.x) * dk + r;
    const bool fresh = live_steps(c, env) && c.starts && c.starts[int64_t(env) * c.starts_env];
    if (r < dk)
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
            const float x = c.state_in && !fresh && e < cols ? c.state_in[row * dv + col + e] : 0.0f;
            now[0][r][e0 + e] = x;
            if (e < cols) seg.carry[row * dv + col + e] = x;
        }
    for (uint32_t s = 0; s + 1 < seg.count; s++) {
        const float(*from)[16] = now[s & 1];
        float* carry = seg.carry + ((s + 1) * rows + row) * dv + col;
        const float* map = seg.map + (s * rows + row) * dk;
        __syncthreads();
        if (r < dk) {
            float x[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) x[e] = e < cols ? carry[e] : 0.0f;
            auto add = [&](float y, uint32_t k) {
                const uint4 z = *reinterpret_cast<const uint4*>(&from[k][e0]);
                const uint32_t keep = y != 0.0f ? ~0u : 0u;  // no branch, so that the loads run ahead
                x[0] = fmaf(y, __uint_as_float(z.x & keep), x[0]);
                x[1] = fmaf(y, __uint_as_float(z.y & keep), x[1]);
                x[2] = fmaf(y, __uint_as_float(z.z & keep), x[2]);
                x[3] = fmaf(y, __uint_as_float(z.w & keep), x[3]);
            };
            if (dk % 4 == 0) {
#pragma unroll 8
                for (uint32_t k = 0; k < dk; k += 4) {
                    const float4 y = __ldg(reinterpret_cast<const float4*>(map + k));
                    add(y.x, k), add(y.y, k + 1), add(y.z, k + 2), add(y.w, k + 3);
                }
            } else {
                for (uint32_t k = 0; k < dk; k++) add(__ldg(map + k), k);
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                now[(s + 1) & 1][r][e0 + e] = x[e];
                if (e < cols) carry[e] = x[e];
            }
        }
    }
}

// -------------------------------------------------------------- gradients
// A chunk's gradients from the state S it began with, the gradient D of the
// state it ended with and do (w, dx, du: value vectors of a step):
//   dU_j = sum_{i>=j} P_ij do_i + c_j D^T k_j,       P without b here,
//   dUt = (I + A)^-T dU with A_ij = b_i G_ij (k_i.k_j),   dx_j = dv_j = b_j dUt_j,
//   F_ij = s G_ij b_j (do_i.w_j)  (i >= j),    E_ij = -G_ij b_j (dx_i.w_j)  (i > j),
//   dq_i = s g_i S do_i + sum_j F_ij k_j,
//   dk_i = -g_i S dx_i + c_i b_i D w_i + sum_l F_li q_l + sum_j (E + E^T)_ij k_j,
//   D' = g_C D + sum_i s g_i q_i do_i^T - sum_i g_i k_i dx_i^T,
//   dbeta_j = w_j.dUt_j.
// The decay's gradient needs no sum over states: scaling S before step t by
// (1 + h) changes the loss by h dlog_decay_t, and the outputs and the last
// state are linear in (S, v) together, so
//   dlog_decay_t = <D, S_C> + sum_{r >= t in the chunk} (do_r.o_r - dv_r.v_r).
// q_i.dq_i and k_i.dk_i, which a normalised row's gradient takes out, follow
// from the same sums over value columns, in 32 bits whatever dq and dk are
// stored in.
//
// Four warps. First each takes 16 value columns (its part of S^T and D^T in
// registers), then, with D, w and dx in shared memory, 16 of every 64 key
// columns of dq and dk. A fifth warp prepares the matrices of the next chunk,
// a sixth fetches the one after. 128 steps of 1,024 environments x 4 heads of
// 64 x 64 in bf16: 1.2 ms, after 0.42 ms for the forward pass that saves the
// states; 512 environments in 32 bits: 1.4 ms, where the parts of q, k and do
// leave room for one block an SM. Bound as the forward kernel is, by latency:
// issue in 32% of the cycles, the tensor cores 22% busy.

template <int N>
__device__ __forceinline__ void cut_pair(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
    for (int n = 0; n < N; n++) p[n] = cut(x, y);
}

// A rollout's chunks from the last to the first.
struct ChunkWalkBack {
    const uint8_t* starts;
    int64_t starts_step;
    uint32_t live, cell_t, pos, mask, next_flag;
    bool done;
    __device__ void begin(const mdn_delta& c, uint32_t env, uint32_t live_steps_, uint32_t lane) {
        starts = c.starts ? c.starts + int64_t(env) * c.starts_env : nullptr;
        starts_step = c.starts_step;
        live = live_steps_;
        done = live == 0;
        cell_t = done ? 0 : (live - 1) / kCell * kCell;
        pos = live - cell_t;
        mask = __ballot_sync(~0u, flag(cell_t, lane));
        next_flag = cell_t ? flag(cell_t - kCell, lane) : 0u;
    }
    __device__ uint32_t flag(uint32_t t, uint32_t lane) const {
        return starts && lane < kCell && t + lane < live ? starts[int64_t(t + lane) * starts_step] : 0u;
    }
    __device__ ChunkMeta next(uint32_t lane) {
        if (done) return ChunkMeta{0, 0, kDone};
        const uint32_t earlier = mask & ((1u << pos) - 1);
        const uint32_t first = earlier ? 31 - __clz(earlier) : 0;
        const ChunkMeta m{cell_t + first, pos - first, (mask >> first) & 1 ? kFresh : 0u};
        pos = first;
        if (pos == 0) {
            done = cell_t == 0;
            cell_t -= done ? 0 : kCell;
            pos = kCell;
            mask = __ballot_sync(~0u, next_flag);
            next_flag = cell_t ? flag(cell_t - kCell, lane) : 0u;
        }
        return m;
    }
};

template <class T, int DK>
struct Backward {
    static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;      // of q, k and do
    static constexpr int kOut = sizeof(T) == 4 ? 3 : 2;        // of what only dq and dk are made of
    // One stage and two slots where two and three do not fit in shared memory.
    static constexpr bool kAhead = !(sizeof(T) == 4 && DK == 128);
    static constexpr int kSlots = kAhead ? 3 : 2, kStages = kAhead ? 2 : 1;
    static constexpr int kRow = DK * 2 + 16, kRowV = 64 * 2 + 16;
    static constexpr int kRawRow = DK * int(sizeof(T)) + 16, kRawV = 64 * int(sizeof(T)) + 16;
    static constexpr int kSlotK = kCell * kRawRow, kSlotV = 2 * kSlotK, kSlotO = kSlotV + kCell * kRawV;
    static constexpr int kSlotS = kSlotO + kCell * kRawV, kSlot = kSlotS + 128 + 32;
    static constexpr int kMat = 3 * kCell * kMatRow;            // three parts of a 16 x 16 matrix
    static constexpr int kSquare = kCell * kScratchRow * 4;     // a 16 x 16 matrix of floats
    static constexpr int kStageK = kParts == 3 ? 3 * kCell * kRow : 0;
    static constexpr int kStageO = 2 * kStageK;
    static constexpr int kStageW = kStageO + (kParts == 3 ? 3 * kCell * kRowV : 0);  // (I + A')^-1, as [j][i]
    static constexpr int kStageU = kStageW + kMat;              // (I + A)^-1
    static constexpr int kStageP = kStageU + kMat;
    static constexpr int kStageF = kStageP + kMat;              // factors of F^T and E^T, k.q and k.k
    static constexpr int kStageVec = kStageF + 4 * kSquare;
    static constexpr int kStage = kStageVec + 8 * 64;
    // after slots and stages
    static constexpr int kD = kSlots * kSlot + kStages * kStage;   // parts of D: [part][value][key]
    static constexpr int kW = kD + kOut * 64 * kRow;               // parts of w: [part][value][step]
    static constexpr int kX = kW + 3 * 64 * kMatRow;               // parts of dx
    static constexpr int kEF = kX + kOut * 64 * kMatRow;           // each warp's F^T and E^T
    static constexpr int kFE = kEF + 4 * 2 * kSquare;              // parts of F^T and E + E^T
    static constexpr int kSums = kFE + 2 * kOut * kCell * kMatRow;  // [warp][5][16], then rows' sums[16], <D, S>[4], S filled[4]
    static constexpr int kScratch = kSums + 4 * 5 * 64 + 64 + 32;
    static constexpr size_t kSmem = size_t(kScratch) + 2 * kSquare + 5 * 64;

    char* smem;

    __device__ explicit Backward(char* base) : smem(base) {}
    __device__ char* slot(uint32_t i) const { return smem + i % kSlots * kSlot; }
    __device__ char* stage(uint32_t i) const { return smem + kSlots * kSlot + i % kStages * kStage; }
    __device__ ChunkMeta* meta(uint32_t i) const { return reinterpret_cast<ChunkMeta*>(slot(i) + kSlotS + 128); }
    __device__ const char* queries(uint32_t i) const { return kParts == 1 ? slot(i) : stage(i); }
    __device__ const char* keys(uint32_t i) const { return kParts == 1 ? slot(i) + kSlotK : stage(i) + kStageK; }
    __device__ const char* douts(uint32_t i) const { return kParts == 1 ? slot(i) + kSlotO : stage(i) + kStageO; }

    __device__ void fetch(const mdn_delta& c, const mdn_delta_grads& d, uint32_t vec, const ChunkMeta& m, uint32_t i,
                          const Bases<T>& at, const T* dout, uint32_t dv, uint32_t lane) const {
        char* dst = slot(i);
        if (lane == 0) *meta(i) = m;
        if (m.n) {
            fetch_rows<T, DK, kRawRow>(at.q + int64_t(m.t) * c.q.step, c.q.step, vec & 1, c.key_dim, m.n, dst, lane);
            fetch_rows<T, DK, kRawRow>(at.k + int64_t(m.t) * c.k.step, c.k.step, vec & 2, c.key_dim, m.n, dst + kSlotK, lane);
            fetch_rows<T, 64, kRawV>(at.v + int64_t(m.t) * c.v.step, c.v.step, vec & 4, dv, m.n, dst + kSlotV, lane);
            fetch_rows<T, 64, kRawV>(dout + int64_t(m.t) * d.dout.step, d.dout.step, vec & 16, dv, m.n, dst + kSlotO, lane);
            fetch_scalars(at.scalars + int64_t(m.t) * at.scalars_step, at.scalars_step, m.n,
                          reinterpret_cast<float*>(dst + kSlotS), lane);
        }
        cp_async_commit();
    }

    // One warp: chunk i's matrices and factors.
    __device__ void prepare(const mdn_delta& c, uint32_t index, uint32_t lane) const {
        const uint32_t n = meta(index)->n;
        if (!n) return;
        char* st = stage(index);
        // g_k, g_q, c_k, beta, decay, 1/|k|, 1/|q|, {g_C}: 16 each
        float* vec = reinterpret_cast<float*>(st + kStageVec);
        const char* rows = slot(index);
        float* fe = reinterpret_cast<float*>(st + kStageF);  // F^T factors, E^T factors, k.q, k.k as [j][i]
        float *kq = fe + 2 * kCell * kScratchRow, *kk = kq + kCell * kScratchRow;
        float* cols = reinterpret_cast<float*>(smem + kScratch);
        float* a = cols + 2 * kCell * kScratchRow;  // |q|^2[16]
        const float x = reinterpret_cast<const float*>(rows + kSlotS)[lane];
        vec[lane < kCell ? 64 + lane : 32 + lane] = lane < kCell ? expf(x) : x;
        if constexpr (kParts == 3) {
            cut_rows<DK, kRow>(rows, kRawRow, st, lane);
            cut_rows<DK, kRow>(rows + kSlotK, kRawRow, st + kStageK, lane);
            cut_rows<64, kRowV>(rows + kSlotO, kRawV, st + kStageO, lane);
            const float squares = row_squares<DK>(rows, kRawRow, lane);
            if (!(lane & 1)) a[lane >> 1] = squares;
            __syncwarp();
        }
        key_products<kParts, DK, kRow>(keys(index), queries(index), kk, kq, a, lane);
        __syncwarp();
        const uint32_t j = lane & 15;
        const bool low = lane < 16;
        float r = 1.0f;
        if (c.flags & MDN_DELTA_NORMALIZE) r = unit_factor((low ? kk[j * (kScratchRow + 1)] : a[j]) + c.norm_eps);
        vec[80 + lane] = r;
        __syncwarp();
        // Lanes 0..15: column j of A' (and of F's factor); lanes 16..31: of A (and of E's factor).
        float col[16], decay[16], rk[16], other[16];
        load16(col, kk + j * kScratchRow);
        load16(decay, vec + 64);
        load16(rk, vec + 80);
        load16(other, vec + (low ? 96 : 48));  // 1/|q| or beta
        const float rkj = vec[80 + j], bj = vec[48 + j], own = low ? bj : 1.0f;
        float run = 0.0f, lead = 1.0f, tail = 0.0f;
        float fac[16];
#pragma unroll
        for (int i = 0; i < kCell; i++) {
            run = i == int(j) ? 1.0f : run * decay[i];
            if (i <= int(j)) lead *= decay[i];
            if (i + 1 == int(n)) tail = run;
            const bool below = i < int(n) && i > int(j);
            const float pair = run * rk[i] * rkj;
            col[i] = below ? pair * col[i] * (low ? own : other[i]) : 0.0f;
            fac[i] = low ? (i < int(n) && i >= int(j) ? c.scale * run * other[i] * rkj * bj : 0.0f)
                         : (below ? -pair * bj : 0.0f);
        }
#pragma unroll
        for (int i = 0; i < kCell; i += 4) {
            float* d = (low ? fe : fe + kCell * kScratchRow) + j * kScratchRow + i;
            *reinterpret_cast<float4*>(d) = make_float4(fac[i], fac[i + 1], fac[i + 2], fac[i + 3]);
            d = (low ? cols : cols + kCell * kScratchRow) + j * kScratchRow + i;
            *reinterpret_cast<float4*>(d) = make_float4(col[i], col[i + 1], col[i + 2], col[i + 3]);
        }
        const bool in = j < n;
        if (low) {
            vec[j] = in ? lead * rkj : 0.0f;
            vec[32 + j] = in ? tail * rkj : 0.0f;
            if (j + 1 == n) vec[112] = lead;
        } else {
            vec[16 + j] = in ? c.scale * lead * r : 0.0f;
        }
        __syncwarp();
        substitute(col, (low ? cols : cols + kCell * kScratchRow), j);
        store_parts(col, st + (low ? kStageW : kStageU) + j * kMatRow);
        // P = scale G (k.q) / |q| / |k|: half a column a lane
        run = 0.0f;
        load16(other, vec + 96);
        load16(col, kq + j * kScratchRow);
#pragma unroll
        for (int i = 0; i < kCell; i++) {
            run = i == int(j) ? 1.0f : run * decay[i];
            col[i] = i < int(n) && i >= int(j) ? c.scale * run * other[i] * rkj * col[i] : 0.0f;
        }
#pragma unroll
        for (int p = 0; p < 3; p++) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float y0 = low ? col[2 * i] : col[8 + 2 * i], y1 = low ? col[2 * i + 1] : col[9 + 2 * i];
                w[i] = cut(y0, y1);
                (low ? col[2 * i] : col[8 + 2 * i]) = y0;
                (low ? col[2 * i + 1] : col[9 + 2 * i]) = y1;
            }
            *reinterpret_cast<uint4*>(st + kStageP + p * kCell * kMatRow + j * kMatRow + (low ? 0 : 16)) =
                make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
};

// The sums over the eight lanes g of 8 values each: value i ends in lane g = i.
__device__ __forceinline__ float sum_over_rows(const float (&x)[8], uint32_t lane) {
    float y[4], z[2];
    const bool b4 = lane & 16, b2 = lane & 8, b1 = lane & 4;
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = (b4 ? x[4 + i] : x[i]) + __shfl_xor_sync(~0u, b4 ? x[i] : x[4 + i], 16);
#pragma unroll
    for (int i = 0; i < 2; i++) z[i] = (b2 ? y[2 + i] : y[i]) + __shfl_xor_sync(~0u, b2 ? y[i] : y[2 + i], 8);
    return (b1 ? z[1] : z[0]) + __shfl_xor_sync(~0u, b1 ? z[0] : z[1], 4);
}

// Where a value block's share of dq, dk, dlog_decay and dbeta goes when other
// value blocks or heads have shares too: parts are [steps][envs][heads][blocks].
struct Shares {
    float *dq, *dk, *dlog_decay, *dbeta;  // dlog_decay, dbeta only with several value blocks
};
__host__ __device__ inline bool rows_shared(const mdn_delta& c) { return c.heads != c.qk_heads || value_blocks(c) > 1; }
__host__ __device__ inline Shares shares_of(const mdn_delta& c, void* workspace) {
    const size_t parts = size_t(c.steps) * c.envs * c.heads * value_blocks(c);
    float* w = static_cast<float*>(workspace);
    return Shares{w, w + parts * c.key_dim, w + 2 * parts * c.key_dim, w + 2 * parts * c.key_dim + parts};
}

template <class T, int DK>
__global__ void __maxnreg__(168) k_delta_gradients(const __grid_constant__ mdn_delta c,
                                                   const __grid_constant__ mdn_delta_grads d, uint32_t vec) {
    using F = Backward<T, DK>;
    constexpr int NP = F::kParts, NO = F::kOut, NT = DK / 8, NS = DK / 64 ? DK / 64 : 1;
    extern __shared__ __align__(16) char smem_raw[];
    const F f(smem_raw);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t env = blockIdx.x / c.heads, head = blockIdx.x % c.heads, qh = head / (c.heads / c.qk_heads);
    const uint32_t v0 = blockIdx.y * 64, live = live_steps(c, env), dk = c.key_dim, dv = c.value_dim;
    if (warp == 5) {
        ChunkWalkBack walk;
        walk.begin(c, env, live, lane);
        Bases<T> at;
        at.set(c, env, head, qh, v0, lane);
        const T* dout = row_ptr<T>(d.dout, 0, env, head) + v0;
        const uint32_t cols = min(64u, dv - v0);
        if constexpr (F::kAhead) {
            f.fetch(c, d, vec, walk.next(lane), 0, at, dout, cols, lane);
            f.fetch(c, d, vec, walk.next(lane), 1, at, dout, cols, lane);
            cp_async_wait<0>();
            __syncthreads();
            __syncthreads();
            for (uint32_t i = 0; f.meta(i)->n; i++) {
                f.fetch(c, d, vec, walk.next(lane), i + 2, at, dout, cols, lane);
                cp_async_wait<0>();
                __syncthreads();
            }
        } else {
            f.fetch(c, d, vec, walk.next(lane), 0, at, dout, cols, lane);
            cp_async_wait<0>();
            __syncthreads();
            for (uint32_t i = 0; f.meta(i)->n; i++) {
                f.fetch(c, d, vec, walk.next(lane), i + 1, at, dout, cols, lane);
                __syncthreads();
                cp_async_wait<0>();
                __syncthreads();
            }
        }
        return;
    }
    if (warp == 4) {
        __syncthreads();
        if constexpr (F::kAhead) {
            f.prepare(c, 0, lane);
            __syncthreads();
            for (uint32_t i = 0; f.meta(i)->n; i++) {
                f.prepare(c, i + 1, lane);
                __syncthreads();
            }
        } else {
            for (uint32_t i = 0; f.meta(i)->n; i++) {
                f.prepare(c, i, lane);
                __syncthreads();
                __syncthreads();
            }
        }
        return;
    }
    // Row g of a warp's tile is value column 2 g, row g + 8 is 2 g + 1: a lane
    // then holds neighbours, and reads and writes them as pairs.
    const uint32_t g = lane >> 2, t4 = lane & 3, colw = warp * 16 + 2 * g, col = v0 + colw;
    const size_t state = size_t(blockIdx.x) * dk * dv;
    const bool shared_rows = rows_shared(c), wide = value_blocks(c) > 1;
    const Shares shares = shares_of(c, d.workspace);
    float D[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t r = 8 * j + 2 * t4 + (e & 1), cc = col + (e >> 1);
            D[j][e] = d.dstate_out && r < dk && cc < dv ? d.dstate_out[state + size_t(r) * dv + cc] : 0.0f;
        }
    for (uint32_t t = live; t < c.steps; t++) {
        const size_t part = ((size_t(t) * c.envs + env) * c.heads + head) * value_blocks(c) + blockIdx.y;
        if (t4 == 0) store_two(row_ptr<T>(d.dv, t, env, head), vec & 8, col, dv, 0.0f, 0.0f);
        for (uint32_t i = threadIdx.x; i < dk; i += 128) {
            if (shared_rows) shares.dq[part * dk + i] = shares.dk[part * dk + i] = 0.0f;
            else store(row_ptr<T>(d.dq, t, env, qh) + i, 0.0f), store(row_ptr<T>(d.dk, t, env, qh) + i, 0.0f);
        }
        if (threadIdx.x == 0) {
            *(wide ? shares.dlog_decay + part : row_ptr<float>(d.dlog_decay, t, env, head)) = 0.0f;
            *(wide ? shares.dbeta + part : row_ptr<float>(d.dbeta, t, env, head)) = 0.0f;
        }
    }
    const uint32_t dvp = (dv + 15) / 16 * 16;
    float* sums = reinterpret_cast<float*>(f.smem + F::kSums);
    float* row_sums = sums + 4 * 5 * 16;
    float* frob = row_sums + 16;
    __syncthreads();
    if constexpr (F::kAhead) __syncthreads();
    // The states before the chunks: zeros after a start inside a cell. The next
    // chunk's is on its way while this one is finished.
    auto saved_at = [&](const ChunkMeta& m) {
        return static_cast<const float*>(c.saved) + (size_t(m.t / kCell) * c.envs * c.heads + blockIdx.x) * dk * dvp;
    };
    float S[NT][4];
    auto load_state = [&](const ChunkMeta& m) {
        const float* p = saved_at(m) + size_t(2 * t4) * dvp + col;
        const bool in = m.n && m.t % kCell == 0 && col < dvp;
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float2 x = make_float2(0.0f, 0.0f);
                if (in && 8 * j + 2 * t4 + e < dk) x = *reinterpret_cast<const float2*>(p + (8 * j + e) * dvp);
                S[j][e] = x.x, S[j][2 + e] = x.y;
            }
    };
    if constexpr (F::kAhead) load_state(*f.meta(0));
    for (uint32_t i = 0;; i++) {
        const ChunkMeta m = *f.meta(i);
        if (!m.n) break;
        const bool cell = m.t % kCell == 0;
        const float* saved = saved_at(m);
        if constexpr (!F::kAhead) {
            load_state(m);
            __syncthreads();
        }
        const char* st = f.stage(i);
        const char* slot = f.slot(i);
        const float* fac = reinterpret_cast<const float*>(st + F::kStageVec);
        const uint32_t kp = smem_addr(f.keys(i)), qp = smem_addr(f.queries(i)), op = smem_addr(f.douts(i));
        const float gc = fac[112];

        // ---- value columns
        float ks[2][4] = {}, qs[2][4] = {}, dsk[2][4] = {}, frobenius = 0.0f;
        uint32_t bits = 0;  // whether the state before the chunk is anything but zeros
        {
            float ek[2][4] = {}, eq[2][4] = {}, ed[2][4] = {};
#pragma unroll
            for (int kb = 0; kb < DK / 16; kb++) {
                uint32_t a[3][4], bk[NP][4], bq[NP][4];
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    ldsm4(bk[p], kp + p * kCell * F::kRow + kb * 32 + lane_cols_first(lane, F::kRow));
                    ldsm4(bq[p], qp + p * kCell * F::kRow + kb * 32 + lane_cols_first(lane, F::kRow));
                }
                cut_tiles<3>(S[2 * kb], S[2 * kb + 1], a);
                mma_parts<3, NP>(ks[0], ks[1], ek[0], ek[1], a, bk);
                mma_parts<3, NP>(qs[0], qs[1], eq[0], eq[1], a, bq);
                cut_tiles<3>(D[2 * kb], D[2 * kb + 1], a);
                mma_parts<3, NP>(dsk[0], dsk[1], ed[0], ed[1], a, bk);
                // D's parts for the other warps
                char* dst = f.smem + F::kD + colw * F::kRow + kb * 32 + 4 * t4;
#pragma unroll
                for (int p = 0; p < NO; p++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        *reinterpret_cast<uint32_t*>(dst + p * 64 * F::kRow + (r & 1) * F::kRow + (r >> 1) * 16) = a[p][r];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    frobenius = fmaf(D[2 * kb][e], S[2 * kb][e], frobenius);
                    frobenius = fmaf(D[2 * kb + 1][e], S[2 * kb + 1][e], frobenius);
                    bits |= (__float_as_uint(S[2 * kb][e]) | __float_as_uint(S[2 * kb + 1][e])) << 1;
                }
            }
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) ks[n][e] += ek[n][e], qs[n][e] += eq[n][e], dsk[n][e] += ed[n][e];
        }
        // v and do of this lane's two columns and four steps 8 n + 2 t4 + (e & 1): element [n][2 * column + e]
        float v[2][4], o[2][4];
        uint32_t oa[NP][4];  // do^T as an A operand
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int n = 0; n < 2; n++) {
                uint32_t w[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t s = 8 * n + 2 * t4 + e;
                    const uint32_t x = *reinterpret_cast<const uint32_t*>(slot + F::kSlotV + s * F::kRawV + colw * 2);
                    w[e] = *reinterpret_cast<const uint32_t*>(slot + F::kSlotO + s * F::kRawV + colw * 2);
                    v[n][e] = __uint_as_float(x << 16), v[n][2 + e] = __uint_as_float(x & 0xffff0000u);
                    o[n][e] = __uint_as_float(w[e] << 16), o[n][2 + e] = __uint_as_float(w[e] & 0xffff0000u);
                }
                oa[0][2 * n] = __byte_perm(w[0], w[1], 0x5410);
                oa[0][2 * n + 1] = __byte_perm(w[0], w[1], 0x7632);
            }
        } else {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t s = 8 * n + 2 * t4 + e;
                    const float2 x = *reinterpret_cast<const float2*>(slot + F::kSlotV + s * F::kRawV + colw * 4);
                    const float2 y = *reinterpret_cast<const float2*>(slot + F::kSlotO + s * F::kRawV + colw * 4);
                    v[n][e] = x.x, v[n][2 + e] = x.y, o[n][e] = y.x, o[n][2 + e] = y.y;
                }
            cut_tiles<NP>(o[0], o[1], oa);
        }
        uint32_t a[3][4], b[3][4];
        float w[2][4] = {}, du[2][4] = {}, dut[2][4] = {};
        // w = (I + A')^-1 (v - g S^T k)
        {
            float x[2][4];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    ks[n][e] *= fac[8 * n + 2 * t4 + (e & 1)];
                    x[n][e] = v[n][e] - ks[n][e];
                }
            cut_tiles<3>(x[0], x[1], a);
#pragma unroll
            for (int p = 0; p < 3; p++)
                ldsm4t(b[p], smem_addr(st + F::kStageW) + p * kCell * kMatRow + lane_rows_first(lane, kMatRow));
            mma_parts<3, 3>(w[0], w[1], a, b);
        }
        // dU = P^T do + c D^T k, dUt = (I + A)^-T dU
#pragma unroll
        for (int p = 0; p < 3; p++)
            ldsm4(b[p], smem_addr(st + F::kStageP) + p * kCell * kMatRow + lane_cols_first(lane, kMatRow));
        mma_parts<NP, 3>(du[0], du[1], oa, b);
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                dsk[n][e] *= fac[32 + 8 * n + 2 * t4 + (e & 1)];
                du[n][e] += dsk[n][e];
            }
        cut_tiles<3>(du[0], du[1], a);
#pragma unroll
        for (int p = 0; p < 3; p++)
            ldsm4(b[p], smem_addr(st + F::kStageU) + p * kCell * kMatRow + lane_cols_first(lane, kMatRow));
        mma_parts<3, 3>(dut[0], dut[1], a, b);
        // dx, dv; sums over value columns: dbeta, v.dv, g (S^T k).dx, c b (D^T k).w, g (S^T q).do
        float dx[2][4];
        {
            float s0[8], s1[8], s2[8];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t s = 8 * n + 2 * t4 + e;
                    const float beta = fac[48 + s], gq = fac[16 + s];
                    dx[n][e] = beta * dut[n][e], dx[n][2 + e] = beta * dut[n][2 + e];
                    const int at = 2 * n + e;
                    s0[at] = fmaf(w[n][e], dut[n][e], w[n][2 + e] * dut[n][2 + e]);
                    s0[4 + at] = fmaf(v[n][e], dx[n][e], v[n][2 + e] * dx[n][2 + e]);
                    s1[at] = fmaf(ks[n][e], dx[n][e], ks[n][2 + e] * dx[n][2 + e]);
                    s1[4 + at] = beta * fmaf(dsk[n][e], w[n][e], dsk[n][2 + e] * w[n][2 + e]);
                    s2[at] = gq * fmaf(qs[n][e], o[n][e], qs[n][2 + e] * o[n][2 + e]);
                    s2[4 + at] = 0.0f;
                    if (s < m.n)
                        store_two(row_ptr<T>(d.dv, m.t + s, env, head), vec & 8, col, dv, dx[n][e], dx[n][2 + e]);
                }
            s2[4] = gc * frobenius;
            // lane g ends with sum g: kinds 2 apart, step (g & 3) -> 8 (g >> 1 & 1) + 2 t4 + (g & 1)
            const float r0 = sum_over_rows(s0, lane), r1 = sum_over_rows(s1, lane);
            float r2 = sum_over_rows(s2, lane);
            const uint32_t s = ((g >> 1) & 1) * 8 + 2 * t4 + (g & 1), kind = g >> 2;
            float* dst = sums + warp * 5 * 16;
            dst[kind * 16 + s] = r0;
            dst[(2 + kind) * 16 + s] = r1;
            if (kind == 0) dst[4 * 16 + s] = r2;
            r2 += __shfl_xor_sync(~0u, r2, 1);
            r2 += __shfl_xor_sync(~0u, r2, 2);
            const bool filled = __any_sync(~0u, bits != 0);
            if (lane == 16) frob[warp] = r2, frob[4 + warp] = filled ? 1.0f : 0.0f;
        }
        // parts of w and dx for the key columns
        {
            uint32_t p[3][4];
            cut_tiles<3>(w[0], w[1], p);
            char* dst = f.smem + F::kW + colw * kMatRow + 4 * t4;
#pragma unroll
            for (int q = 0; q < 3; q++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    *reinterpret_cast<uint32_t*>(dst + q * 64 * kMatRow + (r & 1) * kMatRow + (r >> 1) * 16) = p[q][r];
            dst = f.smem + F::kX + colw * kMatRow + 4 * t4;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                uint32_t q[NO];
                cut_pair<NO>(dx[r >> 1][2 * (r & 1)], dx[r >> 1][2 * (r & 1) + 1], q);
#pragma unroll
                for (int n = 0; n < NO; n++)
                    *reinterpret_cast<uint32_t*>(dst + n * 64 * kMatRow + (r & 1) * kMatRow + (r >> 1) * 16) = q[n];
            }
        }
        __syncwarp();
        // this warp's share of F^T and E^T: w_j . do_i and w_j . dx_i over its value columns
        {
            float f0[4] = {}, f1[4] = {}, e0[4] = {}, e1[4] = {};
            uint32_t wa[3][4], ob[NP][4], xb[NO][4];
#pragma unroll
            for (int p = 0; p < 3; p++)
                ldsm4t(wa[p], smem_addr(f.smem + F::kW) + p * 64 * kMatRow + warp * 16 * kMatRow + lane_cols_first(lane, kMatRow));
#pragma unroll
            for (int p = 0; p < NP; p++)
                ldsm4(ob[p], op + p * kCell * F::kRowV + warp * 32 + lane_cols_first(lane, F::kRowV));
#pragma unroll
            for (int p = 0; p < NO; p++)
                ldsm4t(xb[p], smem_addr(f.smem + F::kX) + p * 64 * kMatRow + warp * 16 * kMatRow + lane_rows_first(lane, kMatRow));
            mma_parts<3, NP>(f0, f1, wa, ob);
            mma_out<3, NO>(e0, e1, wa, xb);
            float* dst = reinterpret_cast<float*>(f.smem + F::kEF + warp * 2 * F::kSquare);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float* p = dst + (g + 8 * h) * kScratchRow + 2 * t4;
                *reinterpret_cast<float2*>(p) = make_float2(f0[2 * h], f0[2 * h + 1]);
                *reinterpret_cast<float2*>(p + 8) = make_float2(f1[2 * h], f1[2 * h + 1]);
                p += kCell * kScratchRow;
                *reinterpret_cast<float2*>(p) = make_float2(e0[2 * h], e0[2 * h + 1]);
                *reinterpret_cast<float2*>(p + 8) = make_float2(e1[2 * h], e1[2 * h + 1]);
            }
        }
        // D' = g_C D + (s g do)^T q - (g dx)^T k
        {
            uint32_t pa[3][4], pb[3][4];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t s = 8 * n + 2 * t4 + (e & 1);
                    o[n][e] *= fac[16 + s];
                    dx[n][e] *= -fac[s];
                }
            cut_tiles<3>(o[0], o[1], pa);
            cut_tiles<3>(dx[0], dx[1], pb);
#pragma unroll
            for (int kb = 0; kb < DK / 16; kb++) {
                float d0[4] = {}, d1[4] = {};
                uint32_t bk[NP][4], bq[NP][4];
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    ldsm4t(bk[p], kp + p * kCell * F::kRow + kb * 32 + lane_rows_first(lane, F::kRow));
                    ldsm4t(bq[p], qp + p * kCell * F::kRow + kb * 32 + lane_rows_first(lane, F::kRow));
                }
                mma_parts<3, NP>(d0, d1, pa, bq);
                mma_parts<3, NP>(d0, d1, pb, bk);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    D[2 * kb][e] = m.flags & kFresh ? 0.0f : fmaf(gc, D[2 * kb][e], d0[e]);
                    D[2 * kb + 1][e] = m.flags & kFresh ? 0.0f : fmaf(gc, D[2 * kb + 1][e], d1[e]);
                }
            }
        }
        // this warp's key columns of the state, for after the barrier
        float2 sx[16];
        auto load_keys = [&](uint32_t k0) {
            const float* p = saved + size_t(k0 + g) * dvp + v0 + 2 * t4;
#pragma unroll
            for (int vb = 0; vb < 4; vb++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint32_t key = k0 + g + 8 * (r >> 1), value = v0 + vb * 16 + 2 * t4 + 8 * (r & 1);
                    sx[vb * 4 + r] = make_float2(0.0f, 0.0f);
                    if (cell && key < dk && value < dvp)
                        sx[vb * 4 + r] = *reinterpret_cast<const float2*>(p + (8 * (r >> 1)) * dvp + vb * 16 + 8 * (r & 1));
                }
        };
        load_keys(warp * 16);
        asm volatile("bar.sync 1, 128;" ::: "memory");

        // ---- F and E: the warps' shares together, with their factors
        {
            const uint32_t j = threadIdx.x >> 3, i2 = (threadIdx.x & 7) * 2, at = j * kScratchRow + i2;
            const float* part = reinterpret_cast<const float*>(f.smem + F::kEF);
            const float* fe = reinterpret_cast<const float*>(st + F::kStageF);
            constexpr int sq = kCell * kScratchRow;
            float2 x = make_float2(0.0f, 0.0f), y = x;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const float2 p = *reinterpret_cast<const float2*>(part + 2 * q * sq + at);
                const float2 r = *reinterpret_cast<const float2*>(part + (2 * q + 1) * sq + at);
                x.x += p.x, x.y += p.y, y.x += r.x, y.y += r.y;
            }
            const float2 ff = *reinterpret_cast<const float2*>(fe + at), ef = *reinterpret_cast<const float2*>(fe + sq + at);
            const float2 kq = *reinterpret_cast<const float2*>(fe + 2 * sq + at);
            const float2 kk = *reinterpret_cast<const float2*>(fe + 3 * sq + at);
            // outside the triangle the factor is 0 and the sums belong to no product
            x.x = ff.x != 0.0f ? x.x * ff.x : 0.0f, x.y = ff.y != 0.0f ? x.y * ff.y : 0.0f;
            y.x = ef.x != 0.0f ? y.x * ef.x : 0.0f, y.y = ef.y != 0.0f ? y.y * ef.y : 0.0f;
            float* back = reinterpret_cast<float*>(f.smem + F::kEF);
            const float2 pf = make_float2(x.x * kq.x, x.y * kq.y), pe = make_float2(y.x * kk.x, y.y * kk.y);
            *reinterpret_cast<float2*>(back + at) = pf;
            *reinterpret_cast<float2*>(back + sq + at) = pe;
            float row = (pf.x + pe.x) + (pf.y + pe.y);
            row += __shfl_xor_sync(~0u, row, 1);
            row += __shfl_xor_sync(~0u, row, 2);
            row += __shfl_xor_sync(~0u, row, 4);
            if ((threadIdx.x & 7) == 0) row_sums[j] = row;
            uint32_t p[NO], q[NO];
            cut_pair<NO>(x.x, x.y, p);
            cut_pair<NO>(y.x, y.y, q);
            char* dst = f.smem + F::kFE;
            constexpr int es = NO * kCell * kMatRow;
#pragma unroll
            for (int n = 0; n < NO; n++) {
                char* z = dst + n * kCell * kMatRow;
                *reinterpret_cast<uint32_t*>(z + j * kMatRow + i2 * 2) = p[n];
                // E^T above the diagonal (i > j), E below; the diagonal is 0
                if (i2 >= j) {
                    uint16_t* up = reinterpret_cast<uint16_t*>(z + es + j * kMatRow + i2 * 2);
                    if (i2 > j) up[0] = uint16_t(q[n]);
                    else up[0] = 0;
                    up[1] = uint16_t(q[n] >> 16);
                    if (i2 > j) *reinterpret_cast<uint16_t*>(z + es + i2 * kMatRow + j * 2) = uint16_t(q[n]);
                    *reinterpret_cast<uint16_t*>(z + es + (i2 + 1) * kMatRow + j * 2) = uint16_t(q[n] >> 16);
                } else if (i2 + 1 == j) {
                    *reinterpret_cast<uint16_t*>(z + es + j * kMatRow + j * 2) = 0;
                }
            }
        }
        // ---- key columns: S do, S dx and D w over all value columns
        float aq[NS][2][4] = {}, ax[NS][2][4] = {}, aw[NS][2][4] = {};
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const uint32_t k0 = (s * 4 + warp) * 16;
            if (k0 >= DK) break;
            if (s) load_keys(k0);
#pragma unroll
            for (int vb = 0; vb < 4; vb++) {
                uint32_t oa2[NP][4], xa[NO][4], wa[NO][4], sb[NO][4], db[NO][4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    uint32_t p[NO];
                    cut_pair<NO>(sx[vb * 4 + r].x, sx[vb * 4 + r].y, p);
#pragma unroll
                    for (int n = 0; n < NO; n++) sb[n][r] = p[n];
                }
#pragma unroll
                for (int p = 0; p < NP; p++)
                    ldsm4(oa2[p], op + p * kCell * F::kRowV + vb * 32 + lane_rows_first(lane, F::kRowV));
#pragma unroll
                for (int p = 0; p < NO; p++) {
                    ldsm4t(xa[p], smem_addr(f.smem + F::kX) + p * 64 * kMatRow + vb * 16 * kMatRow + lane_cols_first(lane, kMatRow));
                    ldsm4t(wa[p], smem_addr(f.smem + F::kW) + p * 64 * kMatRow + vb * 16 * kMatRow + lane_cols_first(lane, kMatRow));
                    ldsm4t(db[p], smem_addr(f.smem + F::kD) + p * 64 * F::kRow + vb * 16 * F::kRow + k0 * 2 + lane_rows_first(lane, F::kRow));
                }
                mma_out<NP, NO>(aq[s][0], aq[s][1], oa2, sb);
                mma_out<NO, NO>(ax[s][0], ax[s][1], xa, sb);
                mma_out<NO, NO>(aw[s][0], aw[s][1], wa, db);
            }
        }
        if constexpr (F::kAhead) load_state(*f.meta(i + 1));
        asm volatile("bar.sync 1, 128;" ::: "memory");

        // q.dq and k.dk of step lane & 15: column sums of F (k.q) or E (k.k), rows' sums, sums over value columns
        float qd, kd;
        {
            const float* p = reinterpret_cast<const float*>(f.smem + F::kEF) + (lane < 16 ? 0 : kCell * kScratchRow) + (lane & 15);
            float x = 0.0f;
#pragma unroll
            for (int j = 0; j < kCell; j++) x += p[j * kScratchRow];
            const uint32_t s = lane & 15;
            float t = 0.0f, u = 0.0f;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const float* r = sums + q * 5 * 16 + s;
                if (lane < 16) t += r[4 * 16];
                else t += r[3 * 16], u += r[2 * 16];
            }
            x = lane < 16 ? x + t : x + row_sums[s] + (t - u);
            const float y = __shfl_xor_sync(~0u, x, 16);
            qd = lane < 16 ? x : y;
            kd = lane < 16 ? y : x;
        }
        if (warp == 0) {  // dlog_decay and dbeta
            const uint32_t s = lane & 15;
            float db = 0.0f, vd = 0.0f, end = 0.0f;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const float* r = sums + q * 5 * 16 + s;
                db += r[0], vd += r[16], end += r[3 * 16];
            }
            for (int q = 8; q; q >>= 1) end += __shfl_xor_sync(~0u, end, q);
            end += (frob[0] + frob[1]) + (frob[2] + frob[3]);
            float dg = s < m.n ? qd - vd : 0.0f;
#pragma unroll
            for (int q = 1; q < 16; q <<= 1) {
                const float x = __shfl_down_sync(~0u, dg, q, 16);
                if (s + q < 16) dg += x;
            }
            dg += end;
            // exactly 0 where the state before the step counts for nothing
            const bool filled = frob[4] + frob[5] + frob[6] + frob[7] != 0.0f;
            if (fac[64 + s] == 0.0f || (s == 0 && !filled)) dg = 0.0f;
            if (lane < m.n) {
                const size_t part = ((size_t(m.t + s) * c.envs + env) * c.heads + head) * value_blocks(c) + blockIdx.y;
                *(wide ? shares.dlog_decay + part : row_ptr<float>(d.dlog_decay, m.t + s, env, head)) = dg;
                *(wide ? shares.dbeta + part : row_ptr<float>(d.dbeta, m.t + s, env, head)) = db;
            }
        }
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const uint32_t k0 = (s * 4 + warp) * 16;
            if (k0 >= DK) break;
            uint32_t kb[NP][4], qb[NP][4], fa[NO][4], ft[NO][4], ea[NO][4];
#pragma unroll
            for (int p = 0; p < NP; p++) {
                ldsm4t(kb[p], kp + p * kCell * F::kRow + k0 * 2 + lane_rows_first(lane, F::kRow));
                ldsm4t(qb[p], qp + p * kCell * F::kRow + k0 * 2 + lane_rows_first(lane, F::kRow));
            }
#pragma unroll
            for (int p = 0; p < NO; p++) {
                const uint32_t fe = smem_addr(f.smem + F::kFE) + p * kCell * kMatRow;
                ldsm4t(fa[p], fe + lane_cols_first(lane, kMatRow));
                ldsm4(ft[p], fe + lane_rows_first(lane, kMatRow));
                ldsm4(ea[p], fe + NO * kCell * kMatRow + lane_rows_first(lane, kMatRow));
            }
            float rq[2][4] = {}, rk[2][4] = {};
            mma_out<NO, NP>(rq[0], rq[1], fa, kb);
            mma_out<NO, NP>(rk[0], rk[1], ft, qb);
            mma_out<NO, NP>(rk[0], rk[1], ea, kb);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t step = g + 8 * h;
                const float gq = fac[16 + step], gk = fac[step], cb = fac[32 + step] * fac[48 + step];
                const float fq = fac[96 + step] * fac[96 + step], fk = fac[80 + step] * fac[80 + step];
                const float qdot = __shfl_sync(~0u, qd, step), kdot = __shfl_sync(~0u, kd, step);
                const size_t part = ((size_t(m.t + step) * c.envs + env) * c.heads + head) * value_blocks(c) + blockIdx.y;
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const uint32_t key = k0 + 8 * n + 2 * t4;
                    float yq[2], yk[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int at = 2 * h + e;
                        yq[e] = fmaf(gq, aq[s][n][at], rq[n][at]);
                        yk[e] = fmaf(-gk, ax[s][n][at], fmaf(cb, aw[s][n][at], rk[n][at]));
                    }
                    if (c.flags & MDN_DELTA_NORMALIZE) {
                        const T* qr = reinterpret_cast<const T*>(slot + step * F::kRawRow) + key;
                        const T* kr = reinterpret_cast<const T*>(slot + F::kSlotK + step * F::kRawRow) + key;
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            // One key value: x / sqrt(x^2 + eps) has the slope eps r^3; the difference would
                            // cancel to noise.
                            yq[e] = dk == 1 ? yq[e] * (c.norm_eps * fq) : fmaf(-fq * qdot, to_float(qr[e]), yq[e]);
                            yk[e] = dk == 1 ? yk[e] * (c.norm_eps * fk) : fmaf(-fk * kdot, to_float(kr[e]), yk[e]);
                        }
                    }
                    if (step >= m.n) continue;
                    if (shared_rows) {
                        store_two(shares.dq + part * dk, dk % 2 == 0, key, dk, yq[0], yq[1]);
                        store_two(shares.dk + part * dk, dk % 2 == 0, key, dk, yk[0], yk[1]);
                    } else {
                        store_two(row_ptr<T>(d.dq, m.t + step, env, qh), vec & 32, key, dk, yq[0], yq[1]);
                        store_two(row_ptr<T>(d.dk, m.t + step, env, qh), vec & 64, key, dk, yk[0], yk[1]);
                    }
                }
            }
        }
        __syncthreads();
    }
    if (d.dstate_in) {
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t r = 8 * j + 2 * t4 + (e & 1), cc = col + (e >> 1);
                if (r < dk && cc < dv) d.dstate_in[state + size_t(r) * dv + cc] = D[j][e];
            }
    }
}

// dq and dk of a query/key head, dlog_decay and dbeta: the sums of the shares
// of its value heads and their value blocks, in order.
template <class T>
__global__ void k_delta_join(const __grid_constant__ mdn_delta c, const __grid_constant__ mdn_delta_grads d) {
    const uint32_t dk = c.key_dim, blocks = value_blocks(c), group = c.heads / c.qk_heads * blocks;
    const size_t rows = size_t(c.steps) * c.envs * c.qk_heads, total = rows * dk;
    const Shares s = shares_of(c, d.workspace);
    const size_t first = size_t(blockIdx.x) * blockDim.x + threadIdx.x, stride = size_t(gridDim.x) * blockDim.x;
    for (size_t i = first; i < total; i += stride) {
        const uint32_t e = uint32_t(i % dk);
        const size_t row = i / dk, te = row / c.qk_heads;
        const uint32_t qh = uint32_t(row % c.qk_heads), env = uint32_t(te % c.envs), t = uint32_t(te / c.envs);
        float sq = 0.0f, sk = 0.0f;
        for (uint32_t h = 0; h < group; h++) {
            const size_t at = (row * group + h) * dk + e;
            sq += s.dq[at];
            sk += s.dk[at];
        }
        store(row_ptr<T>(d.dq, t, env, qh) + e, sq);
        store(row_ptr<T>(d.dk, t, env, qh) + e, sk);
    }
    if (blocks == 1) return;
    const size_t scalars = size_t(c.steps) * c.envs * c.heads;
    for (size_t i = first; i < scalars; i += stride) {
        const uint32_t head = uint32_t(i % c.heads), env = uint32_t(i / c.heads % c.envs), t = uint32_t(i / c.heads / c.envs);
        float dg = 0.0f, db = 0.0f;
        for (uint32_t b = 0; b < blocks; b++) dg += s.dlog_decay[i * blocks + b], db += s.dbeta[i * blocks + b];
        *row_ptr<float>(d.dlog_decay, t, env, head) = dg;
        *row_ptr<float>(d.dbeta, t, env, head) = db;
    }
}

size_t saved_bytes(const mdn_delta& c) {
    const size_t cells = (size_t(c.steps) + kCell - 1) / kCell;
    return cells * c.envs * c.heads * c.key_dim * ((c.value_dim + 15) / 16 * 16) * sizeof(float);
}
size_t workspace_bytes(const mdn_delta& c) {
    if (!rows_shared(c)) return 0;
    return size_t(c.steps) * c.envs * c.heads * value_blocks(c) * (2 * c.key_dim + 2) * sizeof(float);
}

void check_shape(const mdn_delta* c, const char* who) {
    const std::string at = std::string(who) + ": ";
    require(c, MDN_ERR_INVALID, at + "null call");
    require(c->heads >= 1 && c->qk_heads >= 1 && c->heads % c->qk_heads == 0, MDN_ERR_INVALID,
            at + "heads must be a multiple of qk_heads, both at least 1");
    require(c->key_dim >= 1 && c->key_dim <= MDN_DELTA_MAX_DIM && c->value_dim >= 1 &&
                c->value_dim <= MDN_DELTA_MAX_DIM,
            MDN_ERR_INVALID, at + "key_dim and value_dim must be 1..128");
    require(c->dtype == MDN_F32 || c->dtype == MDN_BF16, MDN_ERR_INVALID, at + "dtype must be MDN_F32 or MDN_BF16");
    require((c->flags & ~MDN_DELTA_NORMALIZE) == 0, MDN_ERR_INVALID, at + "unknown flags");
    require(uint64_t(c->envs) * c->heads <= 0x7fffffffu, MDN_ERR_INVALID, at + "envs x heads exceeds 2^31 - 1");
    require(c->steps <= 0x7fffffffu, MDN_ERR_INVALID, at + "steps exceeds 2^31 - 1");
}

void check_rows(const mdn_rows& r, uint32_t bytes, const char* who, const char* name) {
    require(r.data, MDN_ERR_INVALID, std::string(who) + ": " + name + " is null");
    require(reinterpret_cast<uintptr_t>(r.data) % bytes == 0, MDN_ERR_INVALID,
            std::string(who) + ": " + name + " is not aligned to its type");
}

void check_inputs(const mdn_delta* c, const char* who) {
    const uint32_t e = c->dtype == MDN_F32 ? 4 : 2;
    check_rows(c->q, e, who, "q");
    check_rows(c->k, e, who, "k");
    check_rows(c->v, e, who, "v");
    check_rows(c->log_decay, 4, who, "log_decay");
    check_rows(c->beta, 4, who, "beta");
    require(std::isfinite(c->scale) && std::isfinite(c->norm_eps) && c->norm_eps >= 0.0f, MDN_ERR_INVALID,
            std::string(who) + ": scale and norm_eps must be finite, norm_eps not negative");
    require(reinterpret_cast<uintptr_t>(c->saved) % 16 == 0, MDN_ERR_INVALID,
            std::string(who) + ": saved is not 16-byte aligned");
}

// Lets a kernel use `bytes` of shared memory, and how many of its blocks the
// device holds at once: asked once per device.
template <auto Kernel>
uint32_t resident_blocks(size_t bytes, int threads) {
    constexpr int kDevices = 64;
    static std::atomic<uint32_t> known[kDevices];
    int dev = 0;
    cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
    if (dev < kDevices)
        if (const uint32_t blocks = known[dev].load(std::memory_order_relaxed)) return blocks;
    int per_sm = 0, sms = 0;
    cuda_check(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)), "shared memory");
    cuda_check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, Kernel, threads, bytes), "occupancy");
    cuda_check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "SM count");
    const uint32_t blocks = uint32_t(std::max(1, per_sm * sms));
    if (dev < kDevices) known[dev].store(blocks, std::memory_order_relaxed);
    return blocks;
}

// Whether rows start on `bytes`-byte boundaries whatever the step, environment and head.
bool aligned_rows(const mdn_rows& r, uint32_t elem, uint32_t bytes) {
    const int64_t m = bytes / elem;
    return reinterpret_cast<uintptr_t>(r.data) % bytes == 0 && r.step % m == 0 && r.env % m == 0 && r.head % m == 0;
}

template <class T, int V, int GT>
void launch_tick(const mdn_delta& c, int log_cp, cudaStream_t s) {
    constexpr uint32_t groups = GT < 128 ? 128 / GT : 1;
    const uint32_t items = c.envs * c.heads;
    k_delta_tick<T, V, GT><<<(items + groups - 1) / groups, GT * groups, 0, s>>>(c, log_cp);
}

template <class T, int V>
void tick(const mdn_delta& c, cudaStream_t s) {
    int log_cp = 0;
    while ((V << log_cp) < int(c.value_dim)) log_cp++;
    // threads that hold the state at 32 values each
    const uint32_t need = (c.key_dim << log_cp) / (32 / V) + ((c.key_dim << log_cp) % (32 / V) != 0);
    if (need <= 32 && log_cp <= 5) launch_tick<T, V, 32>(c, log_cp, s);
    else if (need <= 128) launch_tick<T, V, 128>(c, log_cp, s);
    else if (need <= 256) launch_tick<T, V, 256>(c, log_cp, s);
    else launch_tick<T, V, 512>(c, log_cp, s);
}

template <class T>
void tick(const mdn_delta& c, cudaStream_t s) {
    const uintptr_t states = reinterpret_cast<uintptr_t>(c.state_in) | reinterpret_cast<uintptr_t>(c.state_out);
    if (c.value_dim % 4 == 0 && states % 16 == 0) tick<T, 4>(c, s);
    else tick<T, 1>(c, s);
}

// Segments for a rollout of few environments; one where they fill the device
// anyway or the axis is short. Both passes take as long as a segment does as
// long as the joining pass, the larger one, fits on the device at once: 2
// environments x 8 heads, 4,096 steps of 128 keys and values take 530 us whole,
// 356 us in five segments, 374 us in nine (the joining pass in two waves). A segment has at
// least eight cells, over which the pipeline's start and the carried state's
// load are spread.
Segments segments_of(const mdn_delta& c) {
    const uint32_t cells = (c.steps + kCell - 1) / kCell;
    const uint64_t joined = uint64_t(c.envs) * c.heads * (value_blocks(c) + (c.key_dim + 63) / 64);
    const uint64_t room = 148 * 2;
    Segments g{1, cells, kRun, nullptr, nullptr};
    if (!joined || joined * 3 > room || cells < 32) return g;  // two and three segments gain nothing
    const uint32_t count = uint32_t(std::min(std::min(room / joined + 1, uint64_t(cells / 8)), uint64_t(32)));
    g.cells = (cells + count - 1) / count;
    g.count = (cells + g.cells - 1) / g.cells;
    return g;
}
size_t forward_bytes(const mdn_delta& c) {
    const size_t count = segments_of(c).count, rows = size_t(c.envs) * c.heads * c.key_dim;
    return count < 2 ? 0 : (count * rows * c.value_dim + 3) / 4 * 16 + (count - 1) * rows * c.key_dim * sizeof(float);
}

template <class T, int DK, bool SPLIT>
void launch_rollout(const mdn_delta& c, uint32_t vec, uint32_t items, uint32_t columns, const Segments& g, cudaStream_t s) {
    static_assert(Forward<T, DK>::kSmem <= 227 * 1024, "shared memory");
    const uint32_t threads = ((std::min(columns, 64u) + 15) / 16 + 2) * 32;
    const uint32_t blocks = resident_blocks<k_delta_rollout<T, DK, SPLIT>>(Forward<T, DK>::kSmem, 192);
    k_delta_rollout<T, DK, SPLIT><<<std::min(items, blocks), threads, Forward<T, DK>::kSmem, s>>>(c, vec, items, g);
}

template <class T, int DK>
void rollout(const mdn_delta& c, void* workspace, cudaStream_t s) {
    constexpr uint32_t e = sizeof(T);
    uint32_t vec = 0;
    if (aligned_rows(c.q, e, 16)) vec |= 1;
    if (aligned_rows(c.k, e, 16)) vec |= 2;
    if (aligned_rows(c.v, e, 16)) vec |= 4;
    if (aligned_rows(c.out, e, 2 * e) && c.value_dim % 2 == 0) vec |= 8;
    const uintptr_t states = reinterpret_cast<uintptr_t>(c.state_in) | reinterpret_cast<uintptr_t>(c.state_out);
    if (states % 8 == 0 && c.value_dim % 2 == 0) vec |= 128;
    const uint32_t rows = c.envs * c.heads;
    Segments g = segments_of(c);
    if (!workspace) g = Segments{1, (c.steps + kCell - 1) / kCell, kRun, nullptr, nullptr};
    if (g.count > 1) {
        g.carry = static_cast<float*>(workspace);
        g.map = g.carry + (size_t(g.count) * rows * c.key_dim * c.value_dim + 3) / 4 * 4;
        g.pass = kJoin;
        launch_rollout<T, DK, true>(c, vec, (g.count - 1) * rows * (value_blocks(c) + (c.key_dim + 63) / 64),
                              std::max(c.key_dim, c.value_dim), g, s);
        cuda_check(cudaGetLastError(), "mdn_delta_forward: segments");
        k_delta_carry<<<dim3(rows, (c.value_dim + 15) / 16), 512, 0, s>>>(c, g);
        cuda_check(cudaGetLastError(), "mdn_delta_forward: carried states");
        g.pass = kRun;
        launch_rollout<T, DK, true>(c, vec, g.count * rows * value_blocks(c), c.value_dim, g, s);
    } else {
        launch_rollout<T, DK, false>(c, vec, rows * value_blocks(c), c.value_dim, g, s);
    }
}

template <class T, int DK>
void gradients(const mdn_delta& c, const mdn_delta_grads& d, cudaStream_t s) {
    constexpr uint32_t e = sizeof(T);
    uint32_t vec = 0;
    if (aligned_rows(c.q, e, 16)) vec |= 1;
    if (aligned_rows(c.k, e, 16)) vec |= 2;
    if (aligned_rows(c.v, e, 16)) vec |= 4;
    if (aligned_rows(d.dv, e, 2 * e) && c.value_dim % 2 == 0) vec |= 8;
    if (aligned_rows(d.dout, e, 16)) vec |= 16;
    if (aligned_rows(d.dq, e, 2 * e) && c.key_dim % 2 == 0) vec |= 32;
    if (aligned_rows(d.dk, e, 2 * e) && c.key_dim % 2 == 0) vec |= 64;
    static_assert(Backward<T, DK>::kSmem <= 227 * 1024, "shared memory");
    resident_blocks<k_delta_gradients<T, DK>>(Backward<T, DK>::kSmem, 192);
    k_delta_gradients<T, DK><<<dim3(c.envs * c.heads, value_blocks(c)), 192, Backward<T, DK>::kSmem, s>>>(c, d, vec);
}

template <class T>
void backward(const mdn_delta& c, const mdn_delta_grads& d, cudaStream_t s) {
    switch (padded_key(c.key_dim)) {
        case 32: gradients<T, 32>(c, d, s); break;
        case 64: gradients<T, 64>(c, d, s); break;
        default: gradients<T, 128>(c, d, s);
    }
    cuda_check(cudaGetLastError(), "mdn_delta_backward");
    if (!c.steps || !rows_shared(c)) return;
    const size_t total = size_t(c.steps) * c.envs * c.qk_heads * c.key_dim;
    k_delta_join<T><<<unsigned(std::min<size_t>((total + 255) / 256, 148 * 16)), 256, 0, s>>>(c, d);
    cuda_check(cudaGetLastError(), "mdn_delta_backward: shares");
}

template <class T>
void forward(const mdn_delta& c, void* workspace, cudaStream_t s) {
    if (c.steps == 1 && !c.saved) return tick<T>(c, s);
    switch (padded_key(c.key_dim)) {
        case 32: return rollout<T, 32>(c, workspace, s);
        case 64: return rollout<T, 64>(c, workspace, s);
        default: return rollout<T, 128>(c, workspace, s);
    }
}

}  // namespace
}  // namespace mdn

extern "C" size_t mdn_delta_saved_bytes(const mdn_delta* call) {
    using namespace mdn;
    size_t n = 0;
    guarded([&] { check_shape(call, "mdn_delta_saved_bytes"), n = saved_bytes(*call); });
    return n;
}

extern "C" size_t mdn_delta_workspace_bytes(const mdn_delta* call) {
    using namespace mdn;
    size_t n = 0;
    guarded([&] { check_shape(call, "mdn_delta_workspace_bytes"), n = workspace_bytes(*call); });
    return n;
}

extern "C" size_t mdn_delta_forward_bytes(const mdn_delta* call) {
    using namespace mdn;
    size_t n = 0;
    guarded([&] { check_shape(call, "mdn_delta_forward_bytes"), n = forward_bytes(*call); });
    return n;
}

extern "C" int mdn_delta_forward(const mdn_delta* call, void* stream) {
    return mdn_delta_forward_with(call, nullptr, stream);
}

extern "C" int mdn_delta_forward_with(const mdn_delta* call, void* workspace, void* stream) {
    using namespace mdn;
    return guarded([&] {
        const char* who = "mdn_delta_forward";
        check_shape(call, who);
        const mdn_delta& c = *call;
        if (c.envs == 0) return;
        if (c.steps) {
            check_inputs(call, who);
            check_rows(c.out, c.dtype == MDN_F32 ? 4 : 2, who, "out");
        }
        require(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, MDN_ERR_INVALID,
                "mdn_delta_forward: workspace is not 16-byte aligned");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (c.dtype == MDN_F32) forward<float>(c, workspace, s);
        else forward<bf16>(c, workspace, s);
        cuda_check(cudaGetLastError(), who);
    });
}

extern "C" int mdn_delta_backward(const mdn_delta* call, const mdn_delta_grads* grads, void* stream) {
    using namespace mdn;
    return guarded([&] {
        const char* who = "mdn_delta_backward";
        check_shape(call, who);
        require(grads, MDN_ERR_INVALID, "mdn_delta_backward: null grads");
        const mdn_delta& c = *call;
        const mdn_delta_grads& g = *grads;
        if (c.envs == 0) return;
        if (c.steps) {
            const uint32_t e = c.dtype == MDN_F32 ? 4 : 2;
            check_inputs(call, who);
            require(c.saved, MDN_ERR_INVALID, "mdn_delta_backward: saved is null");
            check_rows(g.dout, e, who, "dout");
            check_rows(g.dq, e, who, "dq");
            check_rows(g.dk, e, who, "dk");
            check_rows(g.dv, e, who, "dv");
            check_rows(g.dlog_decay, 4, who, "dlog_decay");
            check_rows(g.dbeta, 4, who, "dbeta");
            require(!workspace_bytes(c) || g.workspace, MDN_ERR_INVALID, "mdn_delta_backward: workspace is null");
            require(reinterpret_cast<uintptr_t>(g.workspace) % 16 == 0, MDN_ERR_INVALID,
                    "mdn_delta_backward: workspace is not 16-byte aligned");
        }
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (c.dtype == MDN_F32) backward<float>(c, g, s);
        else backward<bf16>(c, g, s);
    });
}

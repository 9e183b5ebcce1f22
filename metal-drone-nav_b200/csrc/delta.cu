// The gated delta rule on sm_100a: a policy's recurrent memory over a rollout
// (any number of steps, one included) and its gradients.
//
//   S <- a_t S,  u_t = b_t (v_t - S^T k_t),  S <- S + k_t u_t^T,  o_t = s S^T q_t
//
// with a_t = exp(log_decay_t) and S [key][value] per environment and head.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <string>

#include "host_common.h"

namespace mdn {
namespace {

constexpr int kCell = 16;  // steps between two saved states
constexpr int kThreads = 128;

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

__device__ __forceinline__ float block_sum(float x, float* scratch) {
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    float sum = 0.0f;
    for (int w = 0; w < kThreads / 32; w++) sum += scratch[w];
    return sum;
}

__device__ __forceinline__ uint32_t live_steps(const mdn_delta& c, uint32_t env) {
    if (!c.lengths) return c.steps;
    const int32_t n = c.lengths[env];
    return n <= 0 ? 0u : min(uint32_t(n), c.steps);
}

// One step's key or query row into shared memory, divided by its length when
// the call asks for it; returns the factor.
template <class T>
__device__ __forceinline__ float load_row(const mdn_delta& c, const mdn_rows& rows, uint32_t t, uint32_t env,
                                          uint32_t head, float* dst, float* scratch) {
    const T* p = row_ptr<T>(rows, t, env, head);
    const float x = threadIdx.x < c.key_dim ? to_float(p[threadIdx.x]) : 0.0f;
    float r = 1.0f;
    if (c.flags & MDN_DELTA_NORMALIZE) r = 1.0f / sqrtf(block_sum(x * x, scratch) + c.norm_eps);
    __syncthreads();
    if (threadIdx.x < c.key_dim) dst[threadIdx.x] = x * r;
    __syncthreads();
    return r;
}

// ------------------------------------------------------------------ tick
// One step (the policy tick): the state is read once, held in registers, and
// written once. Bound by those bytes. Both products with the state are taken
// in the one pass, with o = s (a S)^T q + s (q.k) u in place of a second pass
// over the new state. A group of GT threads holds one state, 32 values a
// thread: column units of V values (V = 4: 16-byte accesses) across lanes, the
// rows dealt to the RG = GT / CP row groups. GT = 32 keeps all sums inside a
// warp; larger states join their warps' sums in shared memory.
template <class T, int V, int GT>
__global__ void __launch_bounds__(GT < 128 ? 128 : GT) k_delta_tick(const __grid_constant__ mdn_delta c, int log_cp) {
    constexpr int NI = 32 / V, kWarps = GT / 32, kGroups = GT < 128 ? 128 / GT : 1;
    constexpr int kRow = 128;  // widest column axis
    __shared__ float sums[kWarps > 1 ? kWarps : 1][2][kWarps > 1 ? kRow : 1];
    const uint32_t item = blockIdx.x * kGroups + threadIdx.x / GT, tid = threadIdx.x % GT, lane = threadIdx.x & 31;
    if (item >= c.envs * c.heads) return;  // only whole groups leave, and only where groups are warps
    const uint32_t env = item / c.heads, head = item % c.heads, qh = head / (c.heads / c.qk_heads);
    const uint32_t dk = c.key_dim, dv = c.value_dim;
    const uint32_t col = (tid & ((1u << log_cp) - 1)) * V, rg = tid >> log_cp, nrg = GT >> log_cp;
    const bool mine = col < dv;
    const size_t state = size_t(item) * dk * dv;
    const bool live = live_steps(c, env) != 0;
    const bool fresh = live && c.starts && c.starts[int64_t(env) * c.starts_env];
    float S[NI][V];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const uint32_t r = rg + i * nrg;
#pragma unroll
        for (int e = 0; e < V; e++) S[i][e] = 0.0f;
        if (mine && r < dk && c.state_in && !fresh) {
            const float* p = c.state_in + state + size_t(r) * dv + col;
            if constexpr (V == 4) {
                const float4 x = __ldcs(reinterpret_cast<const float4*>(p));
                S[i][0] = x.x, S[i][1] = x.y, S[i][2] = x.z, S[i][3] = x.w;
            } else {
                S[i][0] = *p;
            }
        }
    }
    if (live) {
        const T* qp = row_ptr<T>(c.q, 0, env, qh);
        const T* kp = row_ptr<T>(c.k, 0, env, qh);
        const float a = expf(*row_ptr<float>(c.log_decay, 0, env, head));
        const float b = *row_ptr<float>(c.beta, 0, env, head);
        float v[V];
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = mine ? to_float(row_ptr<T>(c.v, 0, env, head)[col + e]) : 0.0f;
        float qq = 0.0f, kk = 0.0f, qk = 0.0f;
        for (uint32_t i = lane; i < dk; i += 32) {
            const float x = to_float(qp[i]), y = to_float(kp[i]);
            qq = fmaf(x, x, qq), kk = fmaf(y, y, kk), qk = fmaf(x, y, qk);
        }
        for (int o = 16; o; o >>= 1) {
            qq += __shfl_xor_sync(~0u, qq, o);
            kk += __shfl_xor_sync(~0u, kk, o);
            qk += __shfl_xor_sync(~0u, qk, o);
        }
        float rq = 1.0f, rk = 1.0f;
        if (c.flags & MDN_DELTA_NORMALIZE) rq = 1.0f / sqrtf(qq + c.norm_eps), rk = 1.0f / sqrtf(kk + c.norm_eps);
        float ks[V] = {}, qs[V] = {};
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const uint32_t r = rg + i * nrg;
            const float kr = r < dk ? to_float(kp[r]) : 0.0f, qr = r < dk ? to_float(qp[r]) : 0.0f;
#pragma unroll
            for (int e = 0; e < V; e++) {
                S[i][e] *= a;
                ks[e] = fmaf(kr, S[i][e], ks[e]);
                qs[e] = fmaf(qr, S[i][e], qs[e]);
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
            if (mine && rg == 0) store(row_ptr<T>(c.out, 0, env, head) + col + e, o);
            u[e] *= rk;
        }
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const uint32_t r = rg + i * nrg;
            const float kr = r < dk ? to_float(kp[r]) : 0.0f;
#pragma unroll
            for (int e = 0; e < V; e++) S[i][e] = fmaf(kr, u[e], S[i][e]);
        }
    } else if (mine && rg == 0) {
#pragma unroll
        for (int e = 0; e < V; e++) store(row_ptr<T>(c.out, 0, env, head) + col + e, 0.0f);
    }
    if (!c.state_out) return;
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const uint32_t r = rg + i * nrg;
        if (!mine || r >= dk) continue;
        float* p = c.state_out + state + size_t(r) * dv + col;
        if constexpr (V == 4) __stcs(reinterpret_cast<float4*>(p), make_float4(S[i][0], S[i][1], S[i][2], S[i][3]));
        else *p = S[i][0];
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
// of parts i and j are taken where i + j <= 2: what is left out is below 2^-24
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
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The next 8 significant bits of x and y as a packed bf16 pair, cut off x and y.
__device__ __forceinline__ uint32_t cut(float& x, float& y) {
    const uint32_t xi = __float_as_uint(x), yi = __float_as_uint(y);
    x -= __uint_as_float(xi & 0xffff0000u);
    y -= __uint_as_float(yi & 0xffff0000u);
    return __byte_perm(xi, yi, 0x7632);
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
// d0, d1 += A B over one k step of 16, smallest parts first.
template <int NA, int NB>
__device__ __forceinline__ void mma_parts(float (&d0)[4], float (&d1)[4], const uint32_t (&a)[NA][4],
                                          const uint32_t (&b)[NB][4]) {
#pragma unroll
    for (int order = 2; order >= 0; order--)
#pragma unroll
        for (int i = 0; i < NA; i++) {
            const int j = order - i;
            if (j < 0 || j >= NB) continue;
            mma(d0, a[i], b[j][0], b[j][1]);
            mma(d1, a[i], b[j][2], b[j][3]);
        }
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

struct ChunkMeta {
    uint32_t t, n;      // first step, steps (0: the rollout is done)
    uint32_t fresh;     // an episode starts at t
    uint32_t slot;      // where its rows are
};

// Walks a rollout's chunks in order: cells of 16 steps, cut at episode starts.
// One warp holds it; the next cell's start flags are fetched a cell ahead.
struct ChunkWalk {
    const uint8_t* starts;
    int64_t starts_step;
    uint32_t live, cell_t, pos, mask, next_flag;
    __device__ void begin(const mdn_delta& c, uint32_t env, uint32_t live_steps_, uint32_t lane) {
        starts = c.starts ? c.starts + int64_t(env) * c.starts_env : nullptr;
        starts_step = c.starts_step;
        live = live_steps_;
        cell_t = pos = 0;
        next_flag = flag(0, lane);
        mask = __ballot_sync(~0u, next_flag);
        next_flag = flag(kCell, lane);
    }
    __device__ uint32_t flag(uint32_t t, uint32_t lane) const {
        return starts && lane < kCell && t + lane < live ? starts[int64_t(t + lane) * starts_step] : 0u;
    }
    __device__ ChunkMeta next(uint32_t lane) {
        ChunkMeta m{cell_t + pos, 0, 0, 0};
        if (cell_t + pos >= live) return m;
        const uint32_t later = mask & ~((2u << pos) - 1);
        uint32_t end = later ? __ffs(later) - 1 : kCell;
        end = min(end, live - cell_t);
        m.n = end - pos;
        m.fresh = (mask >> pos) & 1;
        pos = end;
        if (pos == kCell) {
            pos = 0;
            cell_t += kCell;
            mask = __ballot_sync(~0u, next_flag);
            next_flag = flag(cell_t + kCell, lane);
        }
        return m;
    }
};

// `count` rows of `dim` values from step t on into shared rows of `row`
// bytes, `width` values wide; what lies past `dim` or past the rows is zeros.
template <class T>
__device__ __forceinline__ void fetch_rows(const mdn_rows& src, bool vec, uint32_t t, uint32_t env, uint32_t head,
                                           uint32_t first, uint32_t dim, uint32_t n, char* dst, uint32_t row,
                                           uint32_t width, uint32_t lane) {
    const T* base = row_ptr<T>(src, t, env, head) + first;
    constexpr uint32_t per = 16 / sizeof(T);
    if (vec) {
        const uint32_t granules = width / per;  // a power of two
        const uint32_t shift = 31 - __clz(granules);
        for (uint32_t e = lane; e < kCell * granules; e += 32) {
            const uint32_t r = e >> shift, col = (e & (granules - 1)) * per;
            const uint32_t values = r < n && col < dim ? min(per, dim - col) : 0;
            cp_async16(smem_addr(dst + r * row + col * sizeof(T)), values ? base + int64_t(r) * src.step + col : base,
                       values * sizeof(T));
        }
    } else {
        for (uint32_t e = lane; e < kCell * width; e += 32) {
            const uint32_t r = e / width, col = e % width;
            T x = T(0.0f);
            if (r < n && col < dim) x = base[int64_t(r) * src.step + col];
            *reinterpret_cast<T*>(dst + r * row + col * sizeof(T)) = x;
        }
    }
}

// log_decay and beta of a chunk's steps into shared memory; zeros past n.
__device__ __forceinline__ void fetch_scalars(const mdn_delta& c, uint32_t t, uint32_t env, uint32_t head, uint32_t n,
                                              float* dst, uint32_t lane) {
    const mdn_rows& src = lane < kCell ? c.log_decay : c.beta;
    const uint32_t r = lane & (kCell - 1);
    const float* p = row_ptr<float>(src, t, env, head);
    cp_async4(smem_addr(dst + lane), r < n ? p + int64_t(r) * src.step : p, r < n ? 4 : 0);
}

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

// Sum of squares of the row that two lanes share (lane / 2), in both.
template <class T, int DK>
__device__ __forceinline__ float row_squares(const char* raw, uint32_t raw_row, uint32_t lane) {
    const T* p = reinterpret_cast<const T*>(raw + (lane >> 1) * raw_row) + (lane & 1) * (DK / 2);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < DK / 2; i += 16 / int(sizeof(T))) {
        const uint4 w = *reinterpret_cast<const uint4*>(p + i);
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (sizeof(T) == 4) {
                const float v = __uint_as_float(x[e]);
                sum = fmaf(v, v, sum);
            } else {
                const float lo = __uint_as_float(x[e] << 16), hi = __uint_as_float(x[e] & 0xffff0000u);
                sum = fmaf(lo, lo, sum);
                sum = fmaf(hi, hi, sum);
            }
        }
    }
    return sum + __shfl_xor_sync(~0u, sum, 1);
}

template <class T, int DK>
struct Forward {
    static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
    static constexpr int kSlots = sizeof(T) == 4 ? 3 : 4;
    static constexpr int kRow = DK * 2 + 16;                   // a bf16 part's row
    static constexpr int kRawRow = DK * int(sizeof(T)) + 16;
    static constexpr int kRawV = 64 * int(sizeof(T)) + 16;
    static constexpr int kSlotK = kCell * kRawRow, kSlotV = 2 * kSlotK, kSlotS = kSlotV + kCell * kRawV;
    static constexpr int kSlot = kSlotS + 128;                  // q, k, v rows, then 16 log-decays and 16 betas
    static constexpr int kStageQ = 0;
    static constexpr int kStageK = kParts == 3 ? 3 * kCell * kRow : 0;
    static constexpr int kStageT = 2 * kStageK;                // three parts of (I + A)^-1
    static constexpr int kStageP = kStageT + 3 * kCell * kMatRow;
    static constexpr int kStageVec = kStageP + 3 * kCell * kMatRow;  // g_k[16], g_q[16], c[16], g_C, ChunkMeta
    static constexpr int kStage = kStageVec + 3 * 64 + 32;
    static constexpr int kScratch = 2 * kCell * kScratchRow * 4 + 5 * 64;
    static constexpr size_t kSmem = size_t(kSlots) * kSlot + 2 * kStage + kScratch;

    char *slots, *stages, *scratch;

    __device__ explicit Forward(char* smem)
        : slots(smem), stages(smem + kSlots * kSlot), scratch(smem + kSlots * kSlot + 2 * kStage) {}

    // The bf16 parts of a chunk's keys or queries, in the slot or the stage.
    __device__ const char* parts(uint32_t slot, uint32_t stage, bool key) const {
        return kParts == 1 ? slots + slot * kSlot + (key ? kSlotK : 0)
                           : stages + stage * kStage + (key ? kStageK : kStageQ);
    }

    __device__ void fetch(const mdn_delta& c, uint32_t vec, const ChunkMeta& m, uint32_t env, uint32_t head,
                          uint32_t qh, uint32_t v0, uint32_t lane) const {
        char* slot = slots + m.slot * kSlot;
        if (m.n) {
            fetch_rows<T>(c.q, vec & 1, m.t, env, qh, 0, c.key_dim, m.n, slot, kRawRow, DK, lane);
            fetch_rows<T>(c.k, vec & 2, m.t, env, qh, 0, c.key_dim, m.n, slot + kSlotK, kRawRow, DK, lane);
            fetch_rows<T>(c.v, vec & 4, m.t, env, head, v0, min(64u, c.value_dim - v0), m.n, slot + kSlotV, kRawV, 64,
                          lane);
            fetch_scalars(c, m.t, env, head, m.n, reinterpret_cast<float*>(slot + kSlotS), lane);
        }
        cp_async_commit();
    }

    // One warp: a chunk's matrices and factors, from its rows.
    __device__ void prepare(const mdn_delta& c, const ChunkMeta& m, uint32_t stage, uint32_t lane) const {
        char* st = stages + stage * kStage;
        float* vec = reinterpret_cast<float*>(st + kStageVec);
        if (lane == 0) *reinterpret_cast<ChunkMeta*>(vec + 52) = m;
        if (!m.n) return;
        const char* slot = slots + m.slot * kSlot;
        if constexpr (kParts == 3) {
            cut_rows<DK, kRow>(slot, kRawRow, st + kStageQ, lane);
            cut_rows<DK, kRow>(slot + kSlotK, kRawRow, st + kStageK, lane);
        }
        float* kk = reinterpret_cast<float*>(scratch);
        float* qk = kk + kCell * kScratchRow;
        float* a = qk + kCell * kScratchRow;  // a[16], beta[16], 1/|k|[16], 1/|q|[16]
        float rk = 1.0f, rq = 1.0f;
        if (c.flags & MDN_DELTA_NORMALIZE) {
            rq = 1.0f / sqrtf(row_squares<T, DK>(slot, kRawRow, lane) + c.norm_eps);
            rk = 1.0f / sqrtf(row_squares<T, DK>(slot + kSlotK, kRawRow, lane) + c.norm_eps);
        }
        const float x = reinterpret_cast<const float*>(slot + kSlotS)[lane];
        a[lane] = lane < kCell ? expf(x) : x;
        if (!(lane & 1)) a[32 + (lane >> 1)] = rk, a[48 + (lane >> 1)] = rq;
        __syncwarp();
        const char *qp = parts(m.slot, stage, false), *kp = parts(m.slot, stage, true);
        float dk0[4] = {}, dk1[4] = {}, dq0[4] = {}, dq1[4] = {};
#pragma unroll
        for (int kb = 0; kb < DK / 16; kb++) {
            uint32_t ak[kParts][4], aq[kParts][4], b[kParts][4];
#pragma unroll
            for (int p = 0; p < kParts; p++) {
                ldsm4(b[p], smem_addr(kp) + p * kCell * kRow + kb * 32 + lane_cols_first(lane, kRow));
                ldsm4(ak[p], smem_addr(kp) + p * kCell * kRow + kb * 32 + lane_rows_first(lane, kRow));
                ldsm4(aq[p], smem_addr(qp) + p * kCell * kRow + kb * 32 + lane_rows_first(lane, kRow));
            }
            mma_parts<kParts, kParts>(dk0, dk1, ak, b);
            mma_parts<kParts, kParts>(dq0, dq1, aq, b);
        }
        const uint32_t g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float* d = kk + (g + 8 * h) * kScratchRow + 2 * t;
            d[0] = dk0[2 * h], d[1] = dk0[2 * h + 1], d[8] = dk1[2 * h], d[9] = dk1[2 * h + 1];
            d += kCell * kScratchRow;
            d[0] = dq0[2 * h], d[1] = dq0[2 * h + 1], d[8] = dq1[2 * h], d[9] = dq1[2 * h + 1];
        }
        __syncwarp();
        // Lanes 0..15 scale column j of A, lanes 16..31 that of P; decay products down the column.
        const uint32_t j = lane & 15;
        const bool low = lane < 16;
        const float bj = a[16 + j], rkj = a[32 + j];
        float run = 0.0f, lead = 1.0f, tail = 0.0f;  // G_ij, g_j, G_Cj
        float col[16];
#pragma unroll
        for (int i = 0; i < kCell; i++) {
            const float ai = a[i];
            run = i == int(j) ? 1.0f : run * ai;
            if (i <= int(j)) lead *= ai;
            if (i + 1 == int(m.n)) tail = run;
            const float other = low ? a[32 + i] : c.scale * a[48 + i];
            const bool in = i < int(m.n) && (low ? i > int(j) : i >= int(j));
            const float y = (low ? kk : qk)[i * kScratchRow + j];
            col[i] = in ? run * other * rkj * bj * y : 0.0f;
        }
        if (lane < kCell) {
            const bool in = j < m.n;
            vec[j] = in ? lead * rkj : 0.0f;
            vec[16 + j] = in ? c.scale * lead * a[48 + j] : 0.0f;
            vec[32 + j] = in ? tail * rkj * bj : 0.0f;
            if (j + 1 == m.n) vec[48] = lead;
        }
        __syncwarp();
        if (low) {
#pragma unroll
            for (int i = 0; i < kCell; i++) kk[i * kScratchRow + j] = col[i];
        }
        __syncwarp();
        if (low) {  // column j of (I + A)^-1 by forward substitution
#pragma unroll
            for (int i = 0; i < kCell; i++) {
                float sum = 0.0f;
#pragma unroll
                for (int l = 0; l < i; l++) sum = fmaf(kk[i * kScratchRow + l], col[l], sum);
                col[i] = i == int(j) ? 1.0f : -sum;
            }
        }
        char* dst = st + (low ? kStageT : kStageP) + j * 2;
#pragma unroll
        for (int i = 0; i < kCell; i += 2) {
            float y0 = col[i], y1 = col[i + 1];
#pragma unroll
            for (int p = 0; p < 3; p++) {
                const uint32_t w = cut(y0, y1);
                char* d = dst + p * kCell * kMatRow + i * kMatRow;
                *reinterpret_cast<uint16_t*>(d) = uint16_t(w);
                *reinterpret_cast<uint16_t*>(d + kMatRow) = uint16_t(w >> 16);
            }
        }
    }
};

// Values of two accumulator columns (steps) and rows (value columns) to `out`
// rows of steps t0 + 2 t, + 1. Two lanes swap so that each stores a pair.
template <class T>
__device__ __forceinline__ void store_pairs(const mdn_rows& out, bool pairs, uint32_t t0, uint32_t n, uint32_t env,
                                            uint32_t head, uint32_t col0, uint32_t cols, const float (&d)[4],
                                            uint32_t step, uint32_t lane) {
    const uint32_t g = lane >> 2;
    if constexpr (sizeof(T) == 2) {
        if (pairs) {
            const bool odd = g & 1;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float got = __shfl_xor_sync(~0u, odd ? d[2 * h] : d[2 * h + 1], 4);
                const uint32_t col = col0 + 8 * h + (g & ~1u), s = step + odd;
                const __nv_bfloat162 w = odd ? __floats2bfloat162_rn(got, d[2 * h + 1])
                                             : __floats2bfloat162_rn(d[2 * h], got);
                if (s < n && col < cols)
                    *reinterpret_cast<__nv_bfloat162*>(row_ptr<T>(out, t0 + s, env, head) + col) = w;
            }
            return;
        }
    }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t col = col0 + 8 * h + g, s = step + e;
            if (s < n && col < cols) store(row_ptr<T>(out, t0 + s, env, head) + col, d[2 * h + e]);
        }
}

// One CTA: 64 value columns of one environment and head; a warp for each 16 of
// them and one warp that fetches the next chunks and prepares their matrices.
template <class T, int DK>
__global__ void __launch_bounds__(160) k_delta_rollout(const __grid_constant__ mdn_delta c, uint32_t vec) {
    using F = Forward<T, DK>;
    constexpr int NP = F::kParts, NT = DK / 8;
    extern __shared__ __align__(16) char smem_raw[];
    const F f(smem_raw);
    const uint32_t warps = blockDim.x / 32 - 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t env = blockIdx.x / c.heads, head = blockIdx.x % c.heads, qh = head / (c.heads / c.qk_heads);
    const uint32_t v0 = blockIdx.y * 64, live = live_steps(c, env);
    if (warp == warps) {
        ChunkWalk walk;
        walk.begin(c, env, live, lane);
        ChunkMeta ring[F::kSlots];
#pragma unroll
        for (int i = 0; i < F::kSlots - 1; i++) {
            ring[i] = walk.next(lane);
            ring[i].slot = i;
            f.fetch(c, vec, ring[i], env, head, qh, v0, lane);
        }
        cp_async_wait<F::kSlots - 2>();
        __syncwarp();
        f.prepare(c, ring[0], 0, lane);
        __syncthreads();
        uint32_t slot = F::kSlots - 1;
        for (uint32_t i = 0; ring[0].n; i++) {
            ChunkMeta m = walk.next(lane);
            m.slot = slot;
            slot = slot + 1 == F::kSlots ? 0 : slot + 1;
            f.fetch(c, vec, m, env, head, qh, v0, lane);
            cp_async_wait<F::kSlots - 2>();
            __syncwarp();
            f.prepare(c, ring[1], (i + 1) & 1, lane);
#pragma unroll
            for (int r = 0; r < F::kSlots - 2; r++) ring[r] = ring[r + 1];
            ring[F::kSlots - 2] = m;
            __syncthreads();
        }
        cp_async_wait<0>();
        return;
    }
    const uint32_t g = lane >> 2, t4 = lane & 3, col0 = v0 + warp * 16, dv = c.value_dim;
    const size_t state = size_t(blockIdx.x) * c.key_dim * dv;
    float S[NT][4];
    const bool use_in = c.state_in && !(live && c.starts && c.starts[int64_t(env) * c.starts_env]);
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t r = 8 * j + 2 * t4 + (e & 1), col = col0 + g + 8 * (e >> 1);
            S[j][e] = use_in && r < c.key_dim && col < dv ? c.state_in[state + size_t(r) * dv + col] : 0.0f;
        }
    const bool pairs = vec & 8;
    const uint32_t tiles = (dv + 15) / 16;
    __syncthreads();
    for (uint32_t i = 0;; i++) {
        const uint32_t stage = i & 1;
        const char* st = f.stages + stage * F::kStage;
        const float* fac = reinterpret_cast<const float*>(st + F::kStageVec);
        const ChunkMeta m = *reinterpret_cast<const ChunkMeta*>(fac + 52);
        if (!m.n) break;
        if (m.fresh) {
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) S[j][e] = 0.0f;
        }
        if (c.saved && m.t % kCell == 0 && col0 < dv) {
            float4* d = static_cast<float4*>(c.saved) +
                        (((size_t(m.t / kCell) * c.envs * c.heads + blockIdx.x) * tiles + col0 / 16) * NT) * 32 + lane;
#pragma unroll
            for (int j = 0; j < NT; j++) d[j * 32] = make_float4(S[j][0], S[j][1], S[j][2], S[j][3]);
        }
        const char* slot = f.slots + m.slot * F::kSlot;
        const uint32_t kp = smem_addr(f.parts(m.slot, stage, true)), qp = smem_addr(f.parts(m.slot, stage, false));
        // S^T K^T and S^T Q^T: [16 value columns x 16 steps] each
        float xk[2][4] = {}, xq[2][4] = {};
#pragma unroll
        for (int kb = 0; kb < DK / 16; kb++) {
            uint32_t a[3][4], bk[NP][4], bq[NP][4];
#pragma unroll
            for (int p = 0; p < NP; p++) {
                ldsm4(bk[p], kp + p * kCell * F::kRow + kb * 32 + lane_cols_first(lane, F::kRow));
                ldsm4(bq[p], qp + p * kCell * F::kRow + kb * 32 + lane_cols_first(lane, F::kRow));
            }
            cut_tiles<3>(S[2 * kb], S[2 * kb + 1], a);
            mma_parts<3, NP>(xk[0], xk[1], a, bk);
            mma_parts<3, NP>(xq[0], xq[1], a, bq);
        }
        // X = V - g K S
        if constexpr (sizeof(T) == 2) {
            uint32_t v[4];
            ldsm4t(v, smem_addr(slot + F::kSlotV + warp * 32) + lane_cols_first(lane, F::kRawV));
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const float g0 = fac[8 * n + 2 * t4], g1 = fac[8 * n + 2 * t4 + 1];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    xk[n][2 * h] = __uint_as_float(v[2 * n + h] << 16) - g0 * xk[n][2 * h];
                    xk[n][2 * h + 1] = __uint_as_float(v[2 * n + h] & 0xffff0000u) - g1 * xk[n][2 * h + 1];
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t s = 8 * n + 2 * t4 + (e & 1);
                    const float v = reinterpret_cast<const float*>(slot + F::kSlotV + s * F::kRawV)[warp * 16 + g + 8 * (e >> 1)];
                    xk[n][e] = v - fac[s] * xk[n][e];
                }
        }
        // W = (I + A)^-1 X
        float w[2][4] = {};
        uint32_t parts[3][4], b[3][4];
        cut_tiles<3>(xk[0], xk[1], parts);
#pragma unroll
        for (int p = 0; p < 3; p++)
            ldsm4(b[p], smem_addr(st + F::kStageT) + p * kCell * kMatRow + lane_cols_first(lane, kMatRow));
        mma_parts<3, 3>(w[0], w[1], parts, b);
        // S' = g_C S + (c W)^T K
        float u0[4], u1[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            u0[e] = w[0][e] * fac[32 + 2 * t4 + (e & 1)];
            u1[e] = w[1][e] * fac[40 + 2 * t4 + (e & 1)];
        }
        cut_tiles<3>(u0, u1, parts);
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
        // O = g Q S + P W
#pragma unroll
        for (int e = 0; e < 4; e++) {
            xq[0][e] *= fac[16 + 2 * t4 + (e & 1)];
            xq[1][e] *= fac[24 + 2 * t4 + (e & 1)];
        }
        cut_tiles<3>(w[0], w[1], parts);
#pragma unroll
        for (int p = 0; p < 3; p++)
            ldsm4(b[p], smem_addr(st + F::kStageP) + p * kCell * kMatRow + lane_cols_first(lane, kMatRow));
        mma_parts<3, 3>(xq[0], xq[1], parts, b);
#pragma unroll
        for (int n = 0; n < 2; n++)
            store_pairs<T>(c.out, pairs, m.t, m.n, env, head, col0, dv, xq[n], 8 * n + 2 * t4, lane);
        __syncthreads();
    }
    for (uint32_t t = live; t < c.steps; t++)
        if (lane < 16 && col0 + lane < dv) store(row_ptr<T>(c.out, t, env, head) + col0 + lane, 0.0f);
    if (c.state_out) {
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t r = 8 * j + 2 * t4 + (e & 1), col = col0 + g + 8 * (e >> 1);
                if (r < c.key_dim && col < dv) c.state_out[state + size_t(r) * dv + col] = S[j][e];
            }
    }
}

// Steps back through the rollout; the state before each step is replayed from
// the saved state of its cell.
template <class T>
__global__ void __launch_bounds__(kThreads) k_delta_backward(const __grid_constant__ mdn_delta c,
                                                             const __grid_constant__ mdn_delta_grads g) {
    extern __shared__ float smem[];
    const uint32_t dk = c.key_dim, dv = c.value_dim;
    float* S = smem;
    float* dS = S + dk * dv;
    float* q = dS + dk * dv;
    float* k = q + dk;
    float* u = k + dk;
    float* dx = u + dv;
    float* dout = dx + dv;
    float* scratch = dout + dv;
    const uint32_t env = blockIdx.x / c.heads, head = blockIdx.x % c.heads, group = c.heads / c.qk_heads;
    const uint32_t qh = head / group, j = threadIdx.x, live = live_steps(c, env);
    const size_t state = size_t(blockIdx.x) * dk * dv;
    const float* saved = static_cast<const float*>(c.saved);
    float* part = static_cast<float*>(g.workspace);  // [2][steps][envs][heads][dk] when heads are shared
    const size_t part_k = size_t(c.steps) * c.envs * c.heads * dk;
    for (uint32_t i = j; i < dk * dv; i += kThreads) dS[i] = g.dstate_out ? g.dstate_out[state + i] : 0.0f;
    auto put = [&](uint32_t t, float dq_j, float dk_j) {
        if (j >= dk) return;
        if (group > 1) {
            const size_t at = ((size_t(t) * c.envs + env) * c.heads + head) * dk + j;
            part[at] = dq_j;
            part[part_k + at] = dk_j;
        } else {
            store(row_ptr<T>(g.dq, t, env, qh) + j, dq_j);
            store(row_ptr<T>(g.dk, t, env, qh) + j, dk_j);
        }
    };
    for (uint32_t t = c.steps; t-- > live;) {
        if (j < dv) store(row_ptr<T>(g.dv, t, env, head) + j, 0.0f);
        put(t, 0.0f, 0.0f);
        if (j == 0) *row_ptr<float>(g.dlog_decay, t, env, head) = 0.0f, *row_ptr<float>(g.dbeta, t, env, head) = 0.0f;
    }
    for (uint32_t t = live; t-- > 0;) {
        const uint32_t cell = t / kCell;
        __syncthreads();
        for (uint32_t i = j; i < dk * dv; i += kThreads) {
            const uint32_t r = i / dv, col = i % dv, lane = (col & 7) * 4 + ((r & 7) >> 1), e = (r & 1) + ((col >> 3) & 1) * 2;
            S[i] = saved[((((size_t(cell) * c.envs * c.heads + blockIdx.x) * ((dv + 15) / 16) + col / 16) *
                               (padded_key(dk) / 8) + r / 8) * 32 + lane) * 4 + e];
        }
        __syncthreads();
        float a = 0.0f, b = 0.0f, rk = 0.0f, ks = 0.0f, v = 0.0f;
        bool reset = false;
        for (uint32_t r = cell * kCell; r <= t; r++) {
            reset = c.starts && c.starts[int64_t(r) * c.starts_step + int64_t(env) * c.starts_env];
            rk = load_row<T>(c, c.k, r, env, qh, k, scratch);
            a = expf(*row_ptr<float>(c.log_decay, r, env, head));
            b = *row_ptr<float>(c.beta, r, env, head);
            if (j < dv) {
                ks = 0.0f;
                for (uint32_t i = 0; i < dk; i++) {
                    const float s = reset ? 0.0f : a * S[i * dv + j];
                    S[i * dv + j] = s;
                    ks = fmaf(k[i], s, ks);
                }
                v = to_float(row_ptr<T>(c.v, r, env, head)[j]);
                if (r < t)
                    for (uint32_t i = 0; i < dk; i++) S[i * dv + j] = fmaf(k[i], b * (v - ks), S[i * dv + j]);
            }
            __syncthreads();
        }
        const float rq = load_row<T>(c, c.q, t, env, qh, q, scratch);
        float db = 0.0f;
        if (j < dv) {  // S holds a S_{t-1}; the step's own k u^T is added where it is needed
            const float d = to_float(row_ptr<T>(g.dout, t, env, head)[j]);
            float du = 0.0f;
            for (uint32_t i = 0; i < dk; i++) {
                dS[i * dv + j] = fmaf(c.scale * q[i], d, dS[i * dv + j]);
                du = fmaf(dS[i * dv + j], k[i], du);
            }
            u[j] = b * (v - ks);
            dx[j] = b * du;
            dout[j] = d;
            db = du * (v - ks);
            store(row_ptr<T>(g.dv, t, env, head) + j, b * du);
        }
        db = block_sum(db, scratch);
        float dqj = 0.0f, dkj = 0.0f, dg = 0.0f;
        if (j < dk)
            for (uint32_t e = 0; e < dv; e++) {
                dqj = fmaf(fmaf(k[j], u[e], S[j * dv + e]), dout[e], dqj);
                dkj = fmaf(dS[j * dv + e], u[e], dkj);
                dkj = fmaf(-S[j * dv + e], dx[e], dkj);
            }
        dqj *= c.scale;
        __syncthreads();
        if (j < dv)
            for (uint32_t i = 0; i < dk; i++) {
                const float d = fmaf(-k[i], dx[j], dS[i * dv + j]);
                dg = fmaf(d, S[i * dv + j], dg);
                dS[i * dv + j] = reset ? 0.0f : a * d;
            }
        dg = block_sum(dg, scratch);
        if (c.flags & MDN_DELTA_NORMALIZE) {
            const float qd = block_sum(j < dk ? dqj * q[j] : 0.0f, scratch);
            const float kd = block_sum(j < dk ? dkj * k[j] : 0.0f, scratch);
            // One key value: x / sqrt(x^2 + eps) has the slope eps r^3; the difference below would cancel to noise.
            if (dk == 1) dqj *= rq * rq * rq * c.norm_eps, dkj *= rk * rk * rk * c.norm_eps;
            else if (j < dk) dqj = rq * (dqj - q[j] * qd), dkj = rk * (dkj - k[j] * kd);
        }
        put(t, dqj, dkj);
        if (j == 0) *row_ptr<float>(g.dlog_decay, t, env, head) = dg, *row_ptr<float>(g.dbeta, t, env, head) = db;
    }
    __syncthreads();
    if (g.dstate_in)
        for (uint32_t i = j; i < dk * dv; i += kThreads) g.dstate_in[state + i] = dS[i];
}

// dq and dk of shared heads: the sum of the group's parts, in head order.
template <class T>
__global__ void k_delta_group_sum(const __grid_constant__ mdn_delta c, const __grid_constant__ mdn_delta_grads g) {
    const uint32_t dk = c.key_dim, group = c.heads / c.qk_heads;
    const size_t rows = size_t(c.steps) * c.envs * c.qk_heads, total = rows * dk;
    const float* part = static_cast<const float*>(g.workspace);
    const size_t part_k = size_t(c.steps) * c.envs * c.heads * dk;
    for (size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += size_t(gridDim.x) * blockDim.x) {
        const uint32_t d = uint32_t(i % dk);
        const size_t row = i / dk;
        const uint32_t qh = uint32_t(row % c.qk_heads);
        const size_t te = row / c.qk_heads;
        const uint32_t env = uint32_t(te % c.envs), t = uint32_t(te / c.envs);
        float sq = 0.0f, sk = 0.0f;
        for (uint32_t h = 0; h < group; h++) {
            const size_t at = (te * c.heads + qh * group + h) * dk + d;
            sq += part[at];
            sk += part[part_k + at];
        }
        store(row_ptr<T>(g.dq, t, env, qh) + d, sq);
        store(row_ptr<T>(g.dk, t, env, qh) + d, sk);
    }
}

size_t saved_bytes(const mdn_delta& c) {
    const size_t cells = (size_t(c.steps) + kCell - 1) / kCell;
    return cells * c.envs * c.heads * padded_key(c.key_dim) * ((c.value_dim + 15) / 16 * 16) * sizeof(float);
}
size_t workspace_bytes(const mdn_delta& c) {
    return c.heads == c.qk_heads ? 0 : 2 * size_t(c.steps) * c.envs * c.heads * c.key_dim * sizeof(float);
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

// Lets a kernel use `bytes` of shared memory, once per device.
template <auto Kernel>
void allow_smem(size_t bytes) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return;
    cuda_check(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)), "shared memory");
    done.fetch_or(bit, std::memory_order_relaxed);
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

template <class T, int DK>
void rollout(const mdn_delta& c, cudaStream_t s) {
    constexpr uint32_t e = sizeof(T);
    uint32_t vec = 0;
    if (aligned_rows(c.q, e, 16)) vec |= 1;
    if (aligned_rows(c.k, e, 16)) vec |= 2;
    if (aligned_rows(c.v, e, 16)) vec |= 4;
    if (aligned_rows(c.out, e, 4) && c.value_dim % 2 == 0) vec |= 8;
    allow_smem<k_delta_rollout<T, DK>>(Forward<T, DK>::kSmem);
    const uint32_t warps = (std::min(c.value_dim, 64u) + 15) / 16 + 1;
    const dim3 grid(c.envs * c.heads, (c.value_dim + 63) / 64);
    k_delta_rollout<T, DK><<<grid, warps * 32, Forward<T, DK>::kSmem, s>>>(c, vec);
}

template <class T>
void forward(const mdn_delta& c, cudaStream_t s) {
    if (c.steps == 1 && !c.saved) return tick<T>(c, s);
    switch (padded_key(c.key_dim)) {
        case 32: return rollout<T, 32>(c, s);
        case 64: return rollout<T, 64>(c, s);
        default: return rollout<T, 128>(c, s);
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

extern "C" int mdn_delta_forward(const mdn_delta* call, void* stream) {
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
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (c.dtype == MDN_F32) forward<float>(c, s);
        else forward<bf16>(c, s);
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
        const size_t smem = (2 * size_t(c.key_dim) * c.value_dim + 2 * c.key_dim + 3 * c.value_dim + 32) * sizeof(float);
        auto kernel = c.dtype == MDN_F32 ? k_delta_backward<float> : k_delta_backward<bf16>;
        if (c.dtype == MDN_F32) allow_smem<k_delta_backward<float>>(227 * 1024);
        else allow_smem<k_delta_backward<bf16>>(227 * 1024);
        kernel<<<c.envs * c.heads, kThreads, smem, s>>>(c, g);
        cuda_check(cudaGetLastError(), who);
        if (c.heads != c.qk_heads && c.steps) {
            auto sum = c.dtype == MDN_F32 ? k_delta_group_sum<float> : k_delta_group_sum<bf16>;
            const size_t total = size_t(c.steps) * c.envs * c.qk_heads * c.key_dim;
            sum<<<unsigned(std::min<size_t>((total + 255) / 256, 148 * 16)), 256, 0, s>>>(c, g);
            cuda_check(cudaGetLastError(), "mdn_delta_backward: shared heads");
        }
    });
}

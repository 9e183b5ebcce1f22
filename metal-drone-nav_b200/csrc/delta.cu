// The gated delta rule on sm_100a: a policy's recurrent memory over a rollout
// (any number of steps, one included) and its gradients.
//
//   S <- a_t S,  u_t = b_t (v_t - S^T k_t),  S <- S + k_t u_t^T,  o_t = s S^T q_t
//
// with a_t = exp(log_decay_t) and S [key][value] per environment and head.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

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

// One thread per value column (value_dim <= 128 = kThreads), the state in
// shared memory: the recurrence as it is written.
template <class T>
__global__ void __launch_bounds__(kThreads) k_delta_forward(const __grid_constant__ mdn_delta c) {
    extern __shared__ float smem[];
    const uint32_t dk = c.key_dim, dv = c.value_dim;
    float* S = smem;
    float* q = S + dk * dv;
    float* k = q + dk;
    float* scratch = k + dk;
    const uint32_t env = blockIdx.x / c.heads, head = blockIdx.x % c.heads, qh = head / (c.heads / c.qk_heads);
    const uint32_t j = threadIdx.x, live = live_steps(c, env);
    const size_t state = size_t(blockIdx.x) * dk * dv;
    const bool fresh = live && c.starts && c.starts[int64_t(env) * c.starts_env];
    for (uint32_t i = j; i < dk * dv; i += kThreads) S[i] = c.state_in && !fresh ? c.state_in[state + i] : 0.0f;
    __syncthreads();
    float* saved = static_cast<float*>(c.saved);
    const size_t cell_stride = size_t(c.envs) * c.heads * dk * dv;
    for (uint32_t t = 0; t < live; t++) {
        const bool reset = c.starts && c.starts[int64_t(t) * c.starts_step + int64_t(env) * c.starts_env];
        if (saved && t % kCell == 0)
            for (uint32_t i = j; i < dk * dv; i += kThreads) saved[t / kCell * cell_stride + state + i] = S[i];
        load_row<T>(c, c.k, t, env, qh, k, scratch);
        load_row<T>(c, c.q, t, env, qh, q, scratch);
        const float a = expf(*row_ptr<float>(c.log_decay, t, env, head));
        const float b = *row_ptr<float>(c.beta, t, env, head);
        if (j < dv) {
            float ks = 0.0f;
            for (uint32_t i = 0; i < dk; i++) {
                const float s = reset ? 0.0f : a * S[i * dv + j];
                S[i * dv + j] = s;
                ks = fmaf(k[i], s, ks);
            }
            const float u = b * (to_float(row_ptr<T>(c.v, t, env, head)[j]) - ks);
            float o = 0.0f;
            for (uint32_t i = 0; i < dk; i++) {
                const float s = fmaf(k[i], u, S[i * dv + j]);
                S[i * dv + j] = s;
                o = fmaf(q[i], s, o);
            }
            store(row_ptr<T>(c.out, t, env, head) + j, c.scale * o);
        }
        __syncthreads();
    }
    for (uint32_t t = live; t < c.steps; t++)
        if (j < dv) store(row_ptr<T>(c.out, t, env, head) + j, 0.0f);
    if (c.state_out)
        for (uint32_t i = j; i < dk * dv; i += kThreads) c.state_out[state + i] = S[i];
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
    const size_t state = size_t(blockIdx.x) * dk * dv, cell_stride = size_t(c.envs) * c.heads * dk * dv;
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
        for (uint32_t i = j; i < dk * dv; i += kThreads) S[i] = saved[cell * cell_stride + state + i];
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
    return cells * c.envs * c.heads * c.key_dim * c.value_dim * sizeof(float);
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

template <class K>
void allow_smem(K kernel, size_t bytes) {
    cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)), "shared memory");
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
        const size_t smem = (size_t(c.key_dim) * c.value_dim + 2 * c.key_dim + 32) * sizeof(float);
        auto kernel = c.dtype == MDN_F32 ? k_delta_forward<float> : k_delta_forward<bf16>;
        allow_smem(kernel, smem);
        kernel<<<c.envs * c.heads, kThreads, smem, static_cast<cudaStream_t>(stream)>>>(c);
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
        allow_smem(kernel, smem);
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

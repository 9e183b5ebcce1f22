// The norms around a block with its gate and residual scale, and their
// gradients:
//   h = x + scale * act(gate) * (branch / rms(branch) * branch_weight)
//   y = h / rms(h) * norm_weight
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <string>

#include "host_common.h"

namespace mdn {
namespace {

using bf16 = __nv_bfloat16;
constexpr int kThreads = 256;
constexpr int kPartBlocks = 296;  // blocks that each sum the weight gradients of their rows

__device__ __forceinline__ float get(const mdn_matrix& m, uint32_t dtype, uint64_t row, uint32_t i) {
    const int64_t at = int64_t(row) * m.row + i;
    return dtype == MDN_F32 ? static_cast<const float*>(m.data)[at]
                            : __bfloat162float(static_cast<const bf16*>(m.data)[at]);
}
__device__ __forceinline__ void put(const mdn_matrix& m, uint32_t dtype, uint64_t row, uint32_t i, float x) {
    const int64_t at = int64_t(row) * m.row + i;
    if (dtype == MDN_F32) static_cast<float*>(m.data)[at] = x;
    else static_cast<bf16*>(m.data)[at] = __float2bfloat16_rn(x);
}
__device__ __forceinline__ float weight(const float* w, uint32_t i) { return w ? w[i] : 1.0f; }

__device__ __forceinline__ float sigmoid(float z) { return 1.0f / (1.0f + expf(-z)); }
__device__ __forceinline__ float gate_value(uint32_t act, float z) {
    return act == MDN_GATE_SIGMOID ? sigmoid(z) : z * sigmoid(z);
}
__device__ __forceinline__ float gate_slope(uint32_t act, float z) {
    const float p = sigmoid(z);
    return act == MDN_GATE_SIGMOID ? p * (1.0f - p) : p * (1.0f + z * (1.0f - p));
}

__device__ __forceinline__ float block_sum(float x) {
    __shared__ float scratch[kThreads / 32];
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
    __syncthreads();
    float sum = 0.0f;
    for (int w = 0; w < kThreads / 32; w++) sum += scratch[w];
    return sum;
}

__device__ __forceinline__ float rms_factor(float squares, const mdn_block_norm& c) {
    return 1.0f / sqrtf(squares / float(c.dim) + c.eps);
}

// The gradient of row * r, r = 1 / rms(row): of one value `unit` = row[i] r, from the gradient d of that value and
// mean = mean over the row of gradient * unit. A row of one value has the slope eps r^3: there the difference would
// cancel to noise.
__device__ __forceinline__ float norm_slope(const mdn_block_norm& c, float r, float d, float unit, float mean) {
    return c.dim == 1 ? d * (c.eps * r * r * r) : r * (d - unit * mean);
}

__device__ __forceinline__ float h_value(const mdn_block_norm& c, uint64_t row, uint32_t i, float rb) {
    const float x = get(c.x, c.stream_dtype, row, i);
    if (!c.branch.data) return x;
    const float act = c.gate.data ? gate_value(c.gate_act, get(c.gate, c.dtype, row, i)) : 1.0f;
    const float n = get(c.branch, c.dtype, row, i) * rb * weight(c.branch_weight, i);
    return fmaf(weight(c.residual_scale, i) * act, n, x);
}

__global__ void __launch_bounds__(kThreads) k_block_norm_forward(const __grid_constant__ mdn_block_norm c) {
    for (uint64_t row = blockIdx.x; row < c.rows; row += gridDim.x) {
        float rb = 0.0f, sum = 0.0f;
        if (c.branch.data) {
            for (uint32_t i = threadIdx.x; i < c.dim; i += kThreads) {
                const float m = get(c.branch, c.dtype, row, i);
                sum = fmaf(m, m, sum);
            }
            rb = rms_factor(block_sum(sum), c);
            sum = 0.0f;
        }
        for (uint32_t i = threadIdx.x; i < c.dim; i += kThreads) {
            const float h = h_value(c, row, i, rb);
            sum = fmaf(h, h, sum);
        }
        const float rh = rms_factor(block_sum(sum), c);
        for (uint32_t i = threadIdx.x; i < c.dim; i += kThreads) {
            const float h = h_value(c, row, i, rb);
            if (c.branch.data && c.h.data) put(c.h, c.stream_dtype, row, i, h);
            if (c.y.data) put(c.y, c.dtype, row, i, h * rh * weight(c.norm_weight, i));
        }
    }
}

__global__ void __launch_bounds__(kThreads) k_block_norm_backward(const __grid_constant__ mdn_block_norm c,
                                                                  const __grid_constant__ mdn_block_norm_grads g) {
    float* part = static_cast<float*>(g.workspace) + size_t(blockIdx.x) * 3 * c.dim;
    for (uint32_t i = threadIdx.x; i < 3 * c.dim; i += kThreads) part[i] = 0.0f;
    const mdn_matrix hm = c.branch.data ? c.h : c.x;
    for (uint64_t row = blockIdx.x; row < c.rows; row += gridDim.x) {
        float sh = 0.0f, shd = 0.0f, sb = 0.0f, sbd = 0.0f, rh = 0.0f, rb = 0.0f;
        for (uint32_t i = threadIdx.x; i < c.dim; i += kThreads) {
            const float h = get(hm, c.stream_dtype, row, i);
            const float dy = g.dy.data ? get(g.dy, c.dtype, row, i) : 0.0f;
            sh = fmaf(h, h, sh);
            shd = fmaf(dy * weight(c.norm_weight, i), h, shd);
            if (c.branch.data) {
                const float m = get(c.branch, c.dtype, row, i);
                sb = fmaf(m, m, sb);
            }
        }
        rh = rms_factor(block_sum(sh), c);
        shd = block_sum(shd) * rh / float(c.dim);
        if (c.branch.data) rb = rms_factor(block_sum(sb), c);
        auto dh_value = [&](uint32_t i) {
            const float dh = g.dh.data ? get(g.dh, c.stream_dtype, row, i) : 0.0f;
            if (!g.dy.data) return dh;
            const float hat = get(hm, c.stream_dtype, row, i) * rh;
            return dh + norm_slope(c, rh, get(g.dy, c.dtype, row, i) * weight(c.norm_weight, i), hat, shd);
        };
        if (c.branch.data) {
            for (uint32_t i = threadIdx.x; i < c.dim; i += kThreads) {
                const float act = c.gate.data ? gate_value(c.gate_act, get(c.gate, c.dtype, row, i)) : 1.0f;
                const float n = get(c.branch, c.dtype, row, i) * rb;
                sbd = fmaf(dh_value(i) * weight(c.residual_scale, i) * act * weight(c.branch_weight, i), n, sbd);
            }
            sbd = block_sum(sbd) / float(c.dim);
        }
        for (uint32_t i = threadIdx.x; i < c.dim; i += kThreads) {
            const float dh = dh_value(i);
            if (g.dy.data) part[i] = fmaf(get(g.dy, c.dtype, row, i), get(hm, c.stream_dtype, row, i) * rh, part[i]);
            if (g.dx.data) put(g.dx, c.stream_dtype, row, i, dh);
            if (!c.branch.data) continue;
            const float z = c.gate.data ? get(c.gate, c.dtype, row, i) : 0.0f;
            const float act = c.gate.data ? gate_value(c.gate_act, z) : 1.0f;
            const float n = get(c.branch, c.dtype, row, i) * rb, w = weight(c.branch_weight, i);
            const float r = weight(c.residual_scale, i), dn = dh * r * act;
            part[c.dim + i] = fmaf(dn, n, part[c.dim + i]);
            part[2 * c.dim + i] = fmaf(dh * act, n * w, part[2 * c.dim + i]);
            if (g.dbranch.data) put(g.dbranch, c.dtype, row, i, norm_slope(c, rb, dn * w, n, sbd));
            if (g.dgate.data && c.gate.data) put(g.dgate, c.dtype, row, i, dh * r * n * w * gate_slope(c.gate_act, z));
        }
    }
}

__global__ void k_block_norm_weights(const __grid_constant__ mdn_block_norm c,
                                     const __grid_constant__ mdn_block_norm_grads g, uint32_t blocks) {
    const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= 3 * c.dim) return;
    float* out = i < c.dim ? g.dnorm_weight : i < 2 * c.dim ? g.dbranch_weight : g.dresidual_scale;
    const bool known = i < c.dim ? c.norm_weight != nullptr
                                 : c.branch.data && (i < 2 * c.dim ? c.branch_weight : c.residual_scale) != nullptr;
    if (!out || !(known || c.rows == 0)) return;
    float sum = 0.0f;
    for (uint32_t b = 0; b < blocks; b++) sum += static_cast<const float*>(g.workspace)[size_t(b) * 3 * c.dim + i];
    out[i % c.dim] = sum;
}

void check_call(const mdn_block_norm* c, const char* who) {
    const std::string at = std::string(who) + ": ";
    require(c, MDN_ERR_INVALID, at + "null call");
    require(c->dim >= 1 && c->dim <= MDN_NORM_MAX_DIM, MDN_ERR_INVALID, at + "dim must be 1..8192");
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
        n = size_t(kPartBlocks) * 3 * call->dim * sizeof(float);
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
        const unsigned blocks = unsigned(std::min<uint64_t>(c.rows, 148 * 8));
        k_block_norm_forward<<<blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(c);
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
        const unsigned blocks = unsigned(std::min<uint64_t>(c.rows, kPartBlocks));
        if (blocks) k_block_norm_backward<<<blocks, kThreads, 0, s>>>(c, g);
        cuda_check(cudaGetLastError(), who);
        k_block_norm_weights<<<(3 * c.dim + 255) / 256, 256, 0, s>>>(c, g, blocks);
        cuda_check(cudaGetLastError(), "mdn_block_norm_backward: weights");
    });
}

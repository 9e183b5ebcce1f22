"""The memory block: operators of a policy with a recurrent memory, on torch CUDA tensors.

`delta_rule` (a rollout), `delta_rule_backward` (its gradients) and `delta_step` (one policy tick) run the gated
delta rule; `block_norm` and `block_norm_backward` the norms around a block with its gate and residual scale
(mdn_delta_*, mdn_block_norm_* in include/mdn.h; no reference counterpart). `delta_rule_train` and
`block_norm_train` are the same under torch autograd.

Rollout arrays are time-major, [steps][envs][heads][dim], like the simulator's buffers; any strides are taken as
long as the last axis is contiguous. Work is queued on the current stream of the tensors' device and nothing is
synchronised; a tensor made on another stream is the caller's to order, as for any torch operator. Bad arguments
raise MdnError.
"""
import ctypes
import struct

import torch

from .capi import ERR, MdnError, check, lib

_Tensor = torch.Tensor
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_GATES = {"sigmoid": 0, "silu": 1}
_NORMALIZE = 1
MAX_DIM = 128  # MDN_DELTA_MAX_DIM
_LONG = 32 * 16 - 15  # no shorter rollout is cut into segments (mdn_delta_forward_bytes)
MAX_NORM_DIM = 8192  # MDN_NORM_MAX_DIM

# mdn_delta, mdn_delta_grads, mdn_block_norm, mdn_block_norm_grads
_DELTA = struct.Struct("8I2f" + "P3q" * 5 + "P2q" + "3P" + "P3q" + "P")
_DELTA_GRADS = struct.Struct("P3q" + "P" + "P3q" * 5 + "2P")
_NORM = struct.Struct("Q4If4x" + "Pq" * 3 + "3P" + "Pq" * 2)
_NORM_GRADS = struct.Struct("Pq" * 5 + "4P")
_NO_ROWS = (0, 0, 0, 0)
_NO_MATRIX = (0, 0)


def _fail(message):
    raise MdnError(ERR["INVALID"], message)


def _tensor(x, name, shape, dtype, device):
    if not isinstance(x, _Tensor) or x.device != device:
        _fail(f"{name} must be a tensor on {device}")
    if x.dtype != dtype:
        _fail(f"{name} must be {dtype}, not {x.dtype}")
    if x.shape != shape:
        _fail(f"{name} must have the shape {tuple(shape)}, not {tuple(x.shape)}")


def _rows(x, name, shape, dtype, device):
    """A [steps, envs, heads, dim] tensor as an mdn_rows: address and strides."""
    _tensor(x, name, shape, dtype, device)
    a, b, c, d = x.stride()
    if d != 1 and shape[3] > 1:
        _fail(f"{name} must be contiguous in its last axis")
    return x.data_ptr(), a, b, c


def _scalars(x, name, shape, device):
    """A [steps, envs, heads] float tensor as an mdn_rows."""
    _tensor(x, name, shape, torch.float32, device)
    return x.data_ptr(), *x.stride()


def _plain(x, name, shape, dtype, device):
    """A contiguous tensor's address; 0 for None."""
    if x is None:
        return 0
    _tensor(x, name, shape, dtype, device)
    if not x.is_contiguous():
        _fail(f"{name} must be contiguous")
    return x.data_ptr()


def _device(x, name):
    if not isinstance(x, torch.Tensor) or x.device.type != "cuda":
        _fail(f"{name} must be a CUDA tensor")
    if x.dtype not in _DTYPES:
        _fail(f"{name} must be float32 or bfloat16, not {x.dtype}")
    return x.device


# the current stream's handle, without a Stream object around it (3 us a call)
_raw_stream = torch._C._cuda_getCurrentRawStream


def _launch(device, fn, *args):
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(index))
    else:
        status = fn(*args, _raw_stream(index))
    if status:
        check(status)


class DeltaSaved:
    """What the gradients of one `delta_rule` call need. It keeps that call's input tensors (which must not change
    until the gradients are taken) and the states that the call saved."""

    __slots__ = ("call", "shape", "dtype", "device", "tensors")


def _delta_call(q, k, v, log_decay, beta, state, starts, lengths, scale, normalize, norm_eps, state_out, out, saved):
    """The packed mdn_delta of checked arguments, all [steps, ...]."""
    device = q.device
    steps, envs, qk, dk = q.shape
    heads, dv = v.shape[2], v.shape[3]
    dtype = q.dtype
    lead = (steps, envs, heads)
    begin = (0, 0, 0)
    if starts is not None:
        if starts.dtype == torch.bool:
            starts = starts.view(torch.uint8)
        _tensor(starts, "starts", (steps, envs), torch.uint8, device)
        begin = (starts.data_ptr(), *starts.stride())
    return _DELTA.pack(
        steps, envs, heads, qk, dk, dv, _DTYPES[dtype], _NORMALIZE if normalize else 0,
        dk ** -0.5 if scale is None else scale, norm_eps,
        *_rows(q, "q", (steps, envs, qk, dk), dtype, device), *_rows(k, "k", (steps, envs, qk, dk), dtype, device),
        *_rows(v, "v", (steps, envs, heads, dv), dtype, device), *_scalars(log_decay, "log_decay", lead, device),
        *_scalars(beta, "beta", lead, device), *begin, _plain(lengths, "lengths", (envs,), torch.int32, device),
        _plain(state, "state", (envs, heads, dk, dv), torch.float32, device),
        _plain(state_out, "state_out", (envs, heads, dk, dv), torch.float32, device),
        *_rows(out, "out", (steps, envs, heads, dv), dtype, device), saved)


def _check_delta_shape(q, v, ndim):
    device = _device(q, "q")
    if q.dim() != ndim or not isinstance(v, torch.Tensor) or v.dim() != ndim:
        _fail(f"q and v must have {ndim} axes")
    qk, dk = q.shape[-2], q.shape[-1]
    heads, dv = v.shape[-2], v.shape[-1]
    if qk < 1 or heads < 1 or heads % qk:
        _fail(f"the heads of v ({heads}) must be a multiple of those of q and k ({qk}), both at least 1")
    if not (1 <= dk <= MAX_DIM and 1 <= dv <= MAX_DIM):
        _fail(f"key and value sizes must be 1..{MAX_DIM}, not {dk} and {dv}")
    return device


def delta_rule(q, k, v, log_decay, beta, state=None, *, starts=None, lengths=None, scale=None, normalize=True,
               norm_eps=1e-6, save=False):
    """The gated delta rule over a rollout. Per environment and head, with a memory S [key, value]:

        S <- exp(log_decay_t) S        (S <- 0 first where starts_t is set)
        u_t = beta_t (v_t - S^T k_t),  S <- S + k_t u_t^T,  out_t = scale S^T q_t

    q, k: [steps, envs, qk_heads, key]; v: [steps, envs, heads, value], heads a multiple of qk_heads (head h uses
    q/k head h // (heads // qk_heads)), all float32 or all bfloat16. log_decay, beta: [steps, envs, heads] float32.
    state: [envs, heads, key, value] float32 or None for zeros. starts: [steps, envs] uint8 or bool, where an episode
    begins; what the memory held before, NaN and infinities too, is then gone. lengths: [envs] int32, steps from
    lengths[env] on are not read, give zeros and leave the state. scale: key ** -0.5 unless given. normalize: q and
    k rows are divided by sqrt(|x|^2 + norm_eps).

    Returns (out, state), and with save=True (out, state, saved) for `delta_rule_backward`."""
    device = _check_delta_shape(q, v, 4)
    steps, envs = q.shape[:2]
    heads, dk, dv = v.shape[2], q.shape[3], v.shape[3]
    out = q.new_empty((steps, envs, heads, dv))
    state_out = q.new_empty((envs, heads, dk, dv), dtype=torch.float32)
    kept = None
    args = (q, k, v, log_decay, beta, state, starts, lengths, scale, normalize, norm_eps, state_out, out)
    if save:
        call = _delta_call(*args, 0)
        kept = q.new_empty(lib().mdn_delta_saved_bytes(call), dtype=torch.uint8)
    call = _delta_call(*args, 0 if kept is None else kept.data_ptr())
    size = lib().mdn_delta_forward_bytes(call) if steps >= _LONG else 0
    if size:  # few environments, a long axis
        work = q.new_empty(size, dtype=torch.uint8)
        _launch(device, lib().mdn_delta_forward_with, call, work.data_ptr())
    else:
        _launch(device, lib().mdn_delta_forward, call)
    if not save:
        return out, state_out
    saved = DeltaSaved()
    saved.call, saved.shape, saved.dtype, saved.device = call, (steps, envs, q.shape[2], heads, dk, dv), q.dtype, device
    saved.tensors = (q, k, v, log_decay, beta, state, starts, lengths, kept)
    return out, state_out, saved


def delta_rule_backward(saved, dout, dstate=None):
    """Gradients of a `delta_rule(..., save=True)` call, from those of its out and (None: zeros) its state. Returns
    (dq, dk, dv, dlog_decay, dbeta, dstate) in the shapes and types of q, k, v, log_decay, beta and state."""
    steps, envs, qk, heads, dk, dv = saved.shape
    device, dtype = saved.device, saved.dtype
    like = saved.tensors[0]
    dq, dkey = like.new_empty((steps, envs, qk, dk)), like.new_empty((steps, envs, qk, dk))
    dvalue = like.new_empty((steps, envs, heads, dv))
    dlog_decay = like.new_empty((steps, envs, heads), dtype=torch.float32)
    dbeta = like.new_empty((steps, envs, heads), dtype=torch.float32)
    dstate_in = like.new_empty((envs, heads, dk, dv), dtype=torch.float32)
    size = lib().mdn_delta_workspace_bytes(saved.call)
    work = like.new_empty(size, dtype=torch.uint8) if size else None
    grads = _DELTA_GRADS.pack(
        *_rows(dout, "dout", (steps, envs, heads, dv), dtype, device),
        _plain(dstate, "dstate", (envs, heads, dk, dv), torch.float32, device),
        dq.data_ptr(), *dq.stride()[:3], dkey.data_ptr(), *dkey.stride()[:3], dvalue.data_ptr(), *dvalue.stride()[:3],
        dlog_decay.data_ptr(), *dlog_decay.stride(), dbeta.data_ptr(), *dbeta.stride(), dstate_in.data_ptr(),
        0 if work is None else work.data_ptr())
    _launch(device, lib().mdn_delta_backward, saved.call, grads)
    return dq, dkey, dvalue, dlog_decay, dbeta, dstate_in


def delta_step(q, k, v, log_decay, beta, state, *, starts=None, scale=None, normalize=True, norm_eps=1e-6, out=None,
               state_out=None):
    """One policy tick of `delta_rule`: q, k: [envs, qk_heads, key]; v: [envs, heads, value]; log_decay, beta:
    [envs, heads]; starts: [envs]. The state is updated in place unless state_out is given. Returns (out, state)."""
    device = _check_delta_shape(q, v, 3)
    if state is None:
        _fail("delta_step needs a state")
    if out is None:
        out = q.new_empty(v.shape)
    if state_out is None:
        state_out = state
    envs, qk, dk = q.shape
    heads, dv = v.shape[1:]
    dtype = q.dtype
    begin = (0, 0, 0)
    if starts is not None:
        if starts.dtype == torch.bool:
            starts = starts.view(torch.uint8)
        _tensor(starts, "starts", (envs,), torch.uint8, device)
        begin = (starts.data_ptr(), 0, starts.stride(0))
    one = (1, envs, heads, dv)
    call = _DELTA.pack(
        1, envs, heads, qk, dk, dv, _DTYPES[dtype], _NORMALIZE if normalize else 0,
        dk ** -0.5 if scale is None else scale, norm_eps,
        *_tick_rows(q, "q", (envs, qk, dk), dtype, device), *_tick_rows(k, "k", (envs, qk, dk), dtype, device),
        *_tick_rows(v, "v", one[1:], dtype, device), *_tick_scalars(log_decay, "log_decay", (envs, heads), device),
        *_tick_scalars(beta, "beta", (envs, heads), device), *begin, 0,
        _plain(state, "state", (envs, heads, dk, dv), torch.float32, device),
        _plain(state_out, "state_out", (envs, heads, dk, dv), torch.float32, device),
        *_tick_rows(out, "out", one[1:], dtype, device), 0)
    _launch(device, lib().mdn_delta_forward, call)
    return out, state_out


def _tick_rows(x, name, shape, dtype, device):
    _tensor(x, name, shape, dtype, device)
    b, c, d = x.stride()
    if d != 1 and shape[2] > 1:
        _fail(f"{name} must be contiguous in its last axis")
    return x.data_ptr(), 0, b, c


def _tick_scalars(x, name, shape, device):
    _tensor(x, name, shape, torch.float32, device)
    return x.data_ptr(), 0, *x.stride()


# ------------------------------------------------------------ block norms

def _matrix(x, name, shape, dtype, device):
    """A [rows, dim] tensor as an mdn_matrix; zeros for None."""
    if x is None:
        return _NO_MATRIX
    _tensor(x, name, shape, dtype, device)
    if shape[1] > 1 and x.stride(1) != 1:
        _fail(f"{name} must be contiguous in its last axis")
    return x.data_ptr(), x.stride(0)


def _norm_args(x, branch, gate, gate_act):
    device = _device(x, "x")
    if x.dim() != 2:
        _fail("rows are [rows, dim] tensors")
    if not 1 <= x.shape[1] <= MAX_NORM_DIM:
        _fail(f"dim must be 1..{MAX_NORM_DIM}, not {x.shape[1]}")
    if gate_act not in _GATES:
        _fail(f"gate_act must be one of {sorted(_GATES)}, not {gate_act!r}")
    if branch is None and gate is not None:
        _fail("a gate without a branch")
    if branch is not None:
        _device(branch, "branch")
    return device


def block_norm(x, branch=None, gate=None, branch_weight=None, residual_scale=None, norm_weight=None, *,
               gate_act="sigmoid", eps=1e-6, dtype=None, next_norm=True):
    """The norm after a block with its gate and residual scale, and the norm before the next block, in one pass:

        h = x + residual_scale * act(gate) * (branch / rms(branch) * branch_weight)
        y = h / rms(h) * norm_weight,      rms(r) = sqrt(mean r^2 + eps)

    x: [rows, dim] (the residual stream); branch (the block's output) and gate: [rows, dim] of one type; float32 or
    bfloat16 each. Weights and scale: [dim] float32, None for ones. Without a branch h is x itself: the norm before
    the first block. y has `dtype` (with a branch, its type; else x's unless given). next_norm=False: only h.
    Returns (h, y)."""
    device = _norm_args(x, branch, gate, gate_act)
    shape = x.shape
    kind = branch.dtype if branch is not None else (dtype or x.dtype)
    if kind not in _DTYPES or (dtype is not None and dtype != kind):
        _fail("y has the type of the branch, float32 or bfloat16")
    if branch is None and not next_norm:
        _fail("without a branch there is only y to compute")
    h = x if branch is None else x.new_empty(shape)
    y = x.new_empty(shape, dtype=kind) if next_norm else None
    _launch(device, lib().mdn_block_norm_forward,
            _pack_norm(x, branch, gate, branch_weight, residual_scale, norm_weight, h if branch is not None else None, y,
                       gate_act, eps, kind, device))
    return h, y


def _pack_norm(x, branch, gate, branch_weight, residual_scale, norm_weight, h, y, gate_act, eps, kind, device):
    ref = x if x is not None else h
    shape = ref.shape
    dim = (shape[1],)
    f32 = torch.float32
    return _NORM.pack(
        shape[0], shape[1], _DTYPES[kind], _DTYPES[ref.dtype], _GATES[gate_act], eps,
        *_matrix(x, "x", shape, ref.dtype, device), *_matrix(branch, "branch", shape, kind, device),
        *_matrix(gate, "gate", shape, kind, device), _plain(branch_weight, "branch_weight", dim, f32, device),
        _plain(residual_scale, "residual_scale", dim, f32, device), _plain(norm_weight, "norm_weight", dim, f32, device),
        *_matrix(h, "h", shape, ref.dtype, device), *_matrix(y, "y", shape, kind, device))


def block_norm_backward(h, branch=None, gate=None, branch_weight=None, residual_scale=None, norm_weight=None, dh=None,
                        dy=None, *, gate_act="sigmoid", eps=1e-6):
    """Gradients of `block_norm` from its h (x where there was no branch) and the gradients of h and y (None: zeros).
    Returns (dx, dbranch, dgate, dbranch_weight, dresidual_scale, dnorm_weight), None for inputs that were None."""
    device = _norm_args(h, branch, gate, gate_act)
    if dh is None and dy is None:
        _fail("block_norm_backward needs dh or dy")
    shape = h.shape
    kind = branch.dtype if branch is not None else dy.dtype if dy is not None else h.dtype
    if kind not in _DTYPES:
        _fail("dy must be float32 or bfloat16")
    call = _pack_norm(h if branch is None else None, branch, gate, branch_weight, residual_scale, norm_weight,
                      h if branch is not None else None, None, gate_act, eps, kind, device)
    dx = h.new_empty(shape)
    dbranch = None if branch is None else branch.new_empty(shape)
    dgate = None if gate is None else gate.new_empty(shape)
    rows = h.new_empty((3, shape[1]), dtype=torch.float32).unbind()
    weights = [row if w is not None and has else None
               for row, w, has in ((rows[0], branch_weight, branch is not None),
                                   (rows[1], residual_scale, branch is not None), (rows[2], norm_weight, True))]
    work = h.new_empty(lib().mdn_block_norm_workspace_bytes(call), dtype=torch.uint8)
    grads = _NORM_GRADS.pack(
        *_matrix(dh, "dh", shape, h.dtype, device), *_matrix(dy, "dy", shape, kind, device), dx.data_ptr(), dx.stride(0),
        *((0, 0) if dbranch is None else (dbranch.data_ptr(), dbranch.stride(0))),
        *((0, 0) if dgate is None else (dgate.data_ptr(), dgate.stride(0))),
        *(0 if w is None else w.data_ptr() for w in weights), work.data_ptr())
    _launch(device, lib().mdn_block_norm_backward, call, grads)
    return dx, dbranch, dgate, *weights


# --------------------------------------------------------------- autograd

class _DeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, beta, state, options):
        out, state_out, ctx.delta = delta_rule(q, k, v, log_decay, beta, state, save=True, **options)
        return out, state_out

    @staticmethod
    def backward(ctx, dout, dstate):
        grads = delta_rule_backward(ctx.delta, dout.contiguous(), dstate.contiguous())
        return (*grads[:5], grads[5] if ctx.needs_input_grad[5] else None, None)


def delta_rule_train(q, k, v, log_decay, beta, state=None, **options):
    """`delta_rule` under torch autograd: (out, state) with gradients to every tensor."""
    return _DeltaRule.apply(q, k, v, log_decay, beta, state, options)


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gate, branch_weight, residual_scale, norm_weight, options):
        h, y = block_norm(x, branch, gate, branch_weight, residual_scale, norm_weight, **options)
        ctx.save_for_backward(h, branch, gate, branch_weight, residual_scale, norm_weight)
        ctx.options = {n: options[n] for n in ("gate_act", "eps") if n in options}
        # without a branch the residual stream goes on as it came
        return (x.view_as(x) if branch is None else h), y

    @staticmethod
    def backward(ctx, dh, dy):
        return (*block_norm_backward(*ctx.saved_tensors, dh.contiguous(), dy.contiguous(), **ctx.options), None)


def block_norm_train(x, branch=None, gate=None, branch_weight=None, residual_scale=None, norm_weight=None, **options):
    """`block_norm` under torch autograd: (h, y) with gradients to every tensor."""
    return _BlockNorm.apply(x, branch, gate, branch_weight, residual_scale, norm_weight, options)

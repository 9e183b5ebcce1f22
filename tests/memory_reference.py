"""64-bit restatement of the memory-block operators from their formulas, step by step, for the tests of
mdn_delta_* and mdn_block_norm_*: torch on the CPU, gradients by autograd. Time-major arrays."""
import torch


def delta(q, k, v, log_decay, beta, state, starts=None, lengths=None, scale=None, normalize=True, eps=1e-6):
    steps, envs, qk, dk = q.shape
    heads = v.shape[2]
    scale = dk ** -0.5 if scale is None else scale
    if normalize:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + eps)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + eps)
    q, k = (x.repeat_interleave(heads // qk, 2) for x in (q, k))
    out = []
    for t in range(steps):
        old = state
        if starts is not None:
            old = torch.where(starts[t].bool()[:, None, None, None], torch.zeros_like(old), old)
        old = old * torch.exp(log_decay[t])[..., None, None]
        u = beta[t][..., None] * (v[t] - torch.einsum("bhd,bhde->bhe", k[t], old))
        new = old + k[t][..., :, None] * u[..., None, :]
        o = scale * torch.einsum("bhd,bhde->bhe", q[t], new)
        if lengths is not None:
            live = t < lengths
            new = torch.where(live[:, None, None, None], new, state)
            o = torch.where(live[:, None, None], o, torch.zeros_like(o))
        out.append(o)
        state = new
    return (torch.stack(out) if out else torch.zeros_like(v)), state


def rms(x, eps):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)


def block(x, branch, gate, branch_weight, residual_scale, norm_weight, act="sigmoid", eps=1e-6):
    """(h, y) of the block norm; None for what is absent."""
    h = x
    if branch is not None:
        n = rms(branch, eps)
        n = n if branch_weight is None else n * branch_weight
        if gate is not None:
            p = torch.sigmoid(gate)
            n = n * (p if act == "sigmoid" else gate * p)
        h = x + (n if residual_scale is None else residual_scale * n)
    return h, next_norm(h, norm_weight, eps)


def next_norm(h, norm_weight, eps=1e-6):
    y = rms(h, eps)
    return y if norm_weight is None else y * norm_weight

"""Cases of the memory-block operators: the gated delta rule (a policy's recurrent memory: a whole rollout, its
gradients, and one tick) and the block norms (the norm after a block with its gate and residual scale, fused with
the norm before the next one, and its gradients).

`run` computes them in plain torch operations in 32 bits, or, where `own` is true, through the package's entry
points. Every array of a rollout is time-major, [steps][envs], as the simulator's buffers are."""
import importlib
import math

import torch

own = False

F32, BF16 = "f32", "bf16"
DTYPES = {F32: torch.float32, BF16: torch.bfloat16}
EPS = 1e-6


def _package():
    return importlib.import_module("metal-drone-nav_b200")


# ------------------------------------------------------------------ cases

def _rollout(name, grad, dtype, steps, envs, heads, qk_heads, dk, dv, resets, ragged, normalize):
    return dict(name=name, op="delta", grad=grad, dtype=dtype, steps=steps, envs=envs, heads=heads, qk_heads=qk_heads,
                dk=dk, dv=dv, resets=resets, ragged=ragged, normalize=normalize)


def _tick(name, dtype, envs, heads, qk_heads, dk, dv):
    return dict(name=name, op="tick", dtype=dtype, envs=envs, heads=heads, qk_heads=qk_heads, dk=dk, dv=dv)


def _norm(name, grad, dtype, stream, rows, dim, block, gate):
    return dict(name=name, op="norm", grad=grad, dtype=dtype, stream=stream, rows=rows, dim=dim, block=block, gate=gate)


def listed():
    return [
        # one drone in flight: the 20 Hz policy tick of a deployed policy, where only latency counts
        _tick("tick-1-f32", F32, 1, 4, 4, 64, 64),
        # a policy tick of the headline simulator, 65,536 environments, small heads
        _tick("tick-65536-bf16", BF16, 65536, 4, 4, 32, 32),
        # a policy tick of an 8,192-environment shard, two memories for each key head
        _tick("tick-8192-f32", F32, 8192, 4, 2, 64, 64),
        # values of a 128-step rollout of 1,024 environments, episodes ending inside it
        _rollout("rollout-128x1024-bf16", False, BF16, 128, 1024, 4, 4, 64, 64, 0.01, False, True),
        # a short evaluation of unequal episodes, odd head sizes, keys already of unit length
        _rollout("ragged-100x333-f32", False, F32, 100, 333, 4, 2, 48, 40, 0.02, True, False),
        # two long recorded flights replayed: few rows, a long axis, wide heads
        _rollout("long-4096x2-bf16", False, BF16, 4096, 2, 8, 8, 128, 128, 0.0, False, True),
        # one PPO minibatch through the memory and back, in the framework's own 32 bits
        _rollout("train-128x512-f32", True, F32, 128, 512, 4, 4, 64, 64, 0.01, False, True),
        # the same in bf16, a larger shard
        _rollout("train-128x1024-bf16", True, BF16, 128, 1024, 4, 4, 64, 64, 0.01, False, True),
        # a truncated window of an odd length, shared keys, odd heads, unequal episodes
        _rollout("train-65x37-bf16", True, BF16, 65, 37, 3, 1, 40, 72, 0.03, True, True),
        # one observation row of a deployed policy into its first block: latency alone
        _norm("norm-1x184-f32", False, F32, F32, 1, 184, False, "none"),
        # a rollout's rows out of one block and into the next: a 480-unit policy, 8,192 environments x 16 steps
        _norm("norm-131072x480-bf16", False, BF16, BF16, 131072, 480, True, "silu"),
        # the same block trained, residual stream in 32 bits, an odd width
        _norm("norm-train-32768x515-mixed", True, BF16, F32, 32768, 515, True, "sigmoid"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tick", "rollout", "train", "norm", "norm-train"])
    dtype = rng.choice([F32, BF16])
    if kind.startswith("norm"):
        dim = _log_int(rng, 1, 8192)
        rows = _log_int(rng, 1, max(2, min(131072, 50_000_000 // dim)))
        block = kind == "norm-train" or rng.random() < 0.7
        gate = rng.choice(["none", "sigmoid", "silu"]) if block else "none"
        case = _norm("", kind == "norm-train", dtype, rng.choice([dtype, F32]), rows, dim, block, gate)
    else:
        dk = rng.choice([16, 32, 64, 64, 128, rng.randint(1, 128)])
        dv = rng.choice([dk, dk, 64, 128, rng.randint(1, 128)])
        qk_heads = rng.choice([1, 2, 4])
        heads = qk_heads * rng.choice([1, 1, 2, 3])
        state = heads * dk * dv  # values of one environment's memory
        if kind == "tick":
            envs = _log_int(rng, 1, max(2, min(65536, 200_000_000 // state)))
            case = _tick("", dtype, envs, heads, qk_heads, dk, dv)
        else:
            steps = _log_int(rng, 1, 2048)
            most = (400_000_000 if kind == "train" else 1_500_000_000) // (state * steps)
            envs = _log_int(rng, 1, max(2, min(8192, most)))
            case = _rollout("", kind == "train", dtype, steps, envs, heads, qk_heads, dk, dv,
                            rng.choice([0.0, 0.01, 0.1]), rng.random() < 0.4, rng.random() < 0.7)
    del case["name"]
    return case


# ----------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    s = dict(case=case)
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        stream = DTYPES[case["stream"]]
        s["x"] = normal(rows, dim, dtype=stream)
        s["norm_weight"] = 1.0 + normal(dim, std=0.1)
        if case["block"]:
            s["branch"] = normal(rows, dim, std=0.7, dtype=dt)
            s["gate"] = normal(rows, dim, dtype=dt) if case["gate"] != "none" else None
            s["branch_weight"] = 1.0 + normal(dim, std=0.1)
            s["residual_scale"] = 0.3 + normal(dim, std=0.05)
        if case["grad"]:
            s["dh"] = normal(rows, dim, dtype=stream)
            s["dy"] = normal(rows, dim, dtype=dt)
        return s
    heads, qk, dk, dv, envs = case["heads"], case["qk_heads"], case["dk"], case["dv"], case["envs"]
    lead = (envs,) if case["op"] == "tick" else (case["steps"], envs)
    # projections of normed observations: about unit values, decays of a memory of some tens of steps
    s["q"] = normal(*lead, qk, dk, dtype=dt)
    s["k"] = normal(*lead, qk, dk, dtype=dt)
    s["v"] = normal(*lead, heads, dv, dtype=dt)
    s["log_decay"] = -torch.exp(normal(*lead, heads) - 3.0)
    s["beta"] = torch.sigmoid(normal(*lead, heads))
    s["state"] = normal(envs, heads, dk, dv, std=0.3)
    if case["op"] == "tick":
        s["starts"] = (uniform(envs) < 0.01).to(torch.uint8)
        s["out"] = torch.empty(envs, heads, dv, dtype=dt, device="cuda")
        s["state_out"] = torch.empty_like(s["state"])
        return s
    if not case["normalize"]:  # the caller's keys and queries have unit length
        for name in ("q", "k"):
            x = s[name].float()
            s[name] = (x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)).to(dt)
    s["starts"] = (uniform(*lead) < case["resets"]).to(torch.uint8) if case["resets"] else None
    s["lengths"] = torch.floor(uniform(envs) * (case["steps"] + 1)).to(torch.int32) if case["ragged"] else None
    if case["grad"]:
        s["dout"] = normal(*lead, heads, dv, dtype=dt)
        s["dstate"] = normal(envs, heads, dk, dv, std=0.1)
    return s


# ------------------------------------------------------------ plain forms

def _unit(x):
    r = torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)
    return x * r, r


def _unit_backward(grad, unit, r):
    return r * (grad - unit * (grad * unit).sum(-1, keepdim=True))


def _row(vector, matrix):  # vector^T matrix over the key axis
    return torch.matmul(vector.unsqueeze(-2), matrix).squeeze(-2)


def _column(matrix, vector):  # matrix vector over the value axis
    return torch.matmul(matrix, vector.unsqueeze(-1)).squeeze(-1)


def _group_sum(x, qk):
    return x.reshape(*x.shape[:-2], qk, x.shape[-2] // qk, x.shape[-1]).sum(-2)


def _plain_tick(s):
    c, dt = s["case"], s["q"].dtype
    group = c["heads"] // c["qk_heads"]
    q = _unit(s["q"].float())[0].repeat_interleave(group, -2)
    k = _unit(s["k"].float())[0].repeat_interleave(group, -2)
    old = torch.where((s["starts"] != 0)[:, None, None, None], 0.0, s["state"])
    old = old * torch.exp(s["log_decay"])[..., None, None]
    u = s["beta"][..., None] * (s["v"].float() - _row(k, old))
    new = old + k[..., :, None] * u[..., None, :]
    return dict(out=(_row(q, new) * c["dk"] ** -0.5).to(dt), state=new)


def _plain_rollout(s):
    c, dt = s["case"], s["q"].dtype
    qk, group, steps, scale = c["qk_heads"], c["heads"] // c["qk_heads"], c["steps"], c["dk"] ** -0.5
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if c["normalize"]:
        (q, rq), (k, rk) = _unit(q), _unit(k)
    q, k = q.repeat_interleave(group, -2), k.repeat_interleave(group, -2)
    decay, beta = torch.exp(s["log_decay"]), s["beta"][..., None]
    fresh = None if s["starts"] is None else (s["starts"] != 0)[..., None, None, None]
    live = None
    if s["lengths"] is not None:
        live = (torch.arange(steps, device="cuda")[:, None] < s["lengths"])[..., None, None]
    state = s["state"].float()
    out, olds, us, errs = torch.zeros_like(v), [], [], []
    for t in range(steps):
        old = state if fresh is None else torch.where(fresh[t], 0.0, state)
        old = old * decay[t][..., None, None]
        err = v[t] - _row(k[t], old)
        u = beta[t] * err
        new = old + k[t][..., :, None] * u[..., None, :]
        o = _row(q[t], new) * scale
        if live is not None:
            new, o = torch.where(live[t][..., None], new, state), torch.where(live[t], o, 0.0)
        out[t] = o
        state = new
        if c["grad"]:
            olds.append(old)
            us.append(u)
            errs.append(err)
    result = dict(out=out.to(dt), state=state)
    if not c["grad"]:
        return result
    dout, ds = s["dout"].float(), s["dstate"].float()
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dg, db = torch.zeros_like(s["log_decay"]), torch.zeros_like(s["beta"])
    for t in reversed(range(steps)):
        old, u = olds[t], us[t]
        new = old + k[t][..., :, None] * u[..., None, :]
        dnew = ds + (scale * q[t])[..., :, None] * dout[t][..., None, :]
        du = _row(k[t], dnew)
        dx = beta[t] * du
        dold = dnew - k[t][..., :, None] * dx[..., None, :]
        grads = [scale * _column(new, dout[t]), _column(dnew, u) - _column(old, dx), dx, (dold * old).sum((-1, -2)),
                 (du * errs[t]).sum(-1)]
        back = dold * decay[t][..., None, None]
        if fresh is not None:
            back = torch.where(fresh[t], 0.0, back)
        if live is not None:
            grads = [torch.where(live[t] if x.dim() == 3 else live[t][..., 0], x, 0.0) for x in grads]
            back = torch.where(live[t][..., None], back, ds)
        dq[t], dk[t], dv[t], dg[t], db[t] = grads
        ds = back
    dq, dk = _group_sum(dq, qk), _group_sum(dk, qk)
    if c["normalize"]:
        dq = _unit_backward(dq, q[..., ::group, :], rq)
        dk = _unit_backward(dk, k[..., ::group, :], rk)
    result.update(dq=dq.to(dt), dk=dk.to(dt), dv=dv.to(dt), dlog_decay=dg, dbeta=db, dstate=ds)
    return result


def _activation(z, kind):
    return torch.sigmoid(z) if kind == "sigmoid" else z * torch.sigmoid(z)


def _activation_slope(z, kind):
    p = torch.sigmoid(z)
    return p * (1.0 - p) if kind == "sigmoid" else p * (1.0 + z * (1.0 - p))


def _rms(x):
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r, r


def _rms_backward(grad, unit, r):
    return r * (grad - unit * (grad * unit).mean(-1, keepdim=True))


def _plain_norm(s):
    c = s["case"]
    stream, dt = DTYPES[c["stream"]], DTYPES[c["dtype"]]
    h = s["x"].float()
    if c["block"]:
        unit, r = _rms(s["branch"].float())
        normed = unit * s["branch_weight"]
        act = 1.0 if s["gate"] is None else _activation(s["gate"].float(), c["gate"])
        h = h + s["residual_scale"] * act * normed
    result = dict(y=(_rms(h)[0] * s["norm_weight"]).to(dt))
    if c["block"]:
        result["h"] = h.to(stream)
    if not c["grad"]:
        return result
    saved = h.to(stream).float()  # a trainer keeps the residual stream in its own type
    hat, rh = _rms(saved)
    dy = s["dy"].float()
    dh = s["dh"].float() + _rms_backward(dy * s["norm_weight"], hat, rh)
    dnormed = dh * s["residual_scale"] * act
    result.update(dx=dh.to(stream), dnorm_weight=(dy * hat).sum(0), dresidual_scale=(dh * act * normed).sum(0),
                  dbranch_weight=(dnormed * unit).sum(0),
                  dbranch=_rms_backward(dnormed * s["branch_weight"], unit, r).to(dt))
    if s["gate"] is not None:
        slope = _activation_slope(s["gate"].float(), c["gate"])
        result["dgate"] = (dh * s["residual_scale"] * normed * slope).to(dt)
    return result


# ------------------------------------------------------ the package's own

def _own_tick(s):
    out, state = _package().delta_step(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["state"],
                                       starts=s["starts"], normalize=True, norm_eps=EPS, out=s["out"],
                                       state_out=s["state_out"])
    return dict(out=out, state=state)


def _own_rollout(s):
    c, mdn = s["case"], _package()
    got = mdn.delta_rule(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["state"], starts=s["starts"],
                         lengths=s["lengths"], normalize=c["normalize"], norm_eps=EPS, save=c["grad"])
    result = dict(out=got[0], state=got[1])
    if c["grad"]:
        names = ("dq", "dk", "dv", "dlog_decay", "dbeta", "dstate")
        result.update(zip(names, mdn.delta_rule_backward(got[2], s["dout"], s["dstate"])))
    return result


def _own_norm(s):
    c, mdn = s["case"], _package()
    if not c["block"]:
        return dict(y=mdn.block_norm(s["x"], norm_weight=s["norm_weight"], eps=EPS, dtype=DTYPES[c["dtype"]])[1])
    kind = c["gate"] if s["gate"] is not None else "sigmoid"
    h, y = mdn.block_norm(s["x"], s["branch"], s["gate"], s["branch_weight"], s["residual_scale"], s["norm_weight"],
                          gate_act=kind, eps=EPS)
    result = dict(h=h, y=y)
    if c["grad"]:
        names = ("dx", "dbranch", "dgate", "dbranch_weight", "dresidual_scale", "dnorm_weight")
        grads = mdn.block_norm_backward(h, s["branch"], s["gate"], s["branch_weight"], s["residual_scale"],
                                        s["norm_weight"], s["dh"], s["dy"], gate_act=kind, eps=EPS)
        result.update((n, g) for n, g in zip(names, grads) if g is not None)
    return result


def run(state):
    op = state["case"]["op"]
    if own:
        return {"tick": _own_tick, "delta": _own_rollout, "norm": _own_norm}[op](state)
    return {"tick": _plain_tick, "delta": _plain_rollout, "norm": _plain_norm}[op](state)


# ------------------------------------------------------------------- work

def work(case):
    b = {F32: 4, BF16: 2}
    e = b[case["dtype"]]
    if case["op"] == "norm":
        n, dim, st = case["rows"] * case["dim"], case["dim"], b[case["stream"]]
        gated = case["gate"] != "none"
        if not case["block"]:
            return dict(bytes=n * (st + e) + 4 * dim, flops=4 * n)
        # x, branch, gate in; h, y out; three weights
        size, flops = n * (2 * st + 2 * e + gated * e) + 12 * dim, 14 * n
        if case["grad"]:
            # h, branch, gate, dh, dy in; dx, dbranch, dgate out; three weights' gradients
            size += n * (3 * st + 3 * e + 2 * gated * e) + 24 * dim
            flops += 40 * n
        return dict(bytes=size, flops=flops)
    heads, qk, dk, dv, envs = case["heads"], case["qk_heads"], case["dk"], case["dv"], case["envs"]
    tokens = envs * case.get("steps", 1)
    per_token = e * (2 * qk * dk + 2 * heads * dv) + 8 * heads
    size = tokens * per_token + 2 * 4 * envs * heads * dk * dv
    flops = 7 * tokens * heads * dk * dv  # decay, k S, rank-1 update, q S
    if case["op"] == "delta" and case["grad"]:
        # q, k, v, dout, decays, betas and both states in; six gradients out
        size += tokens * (e * (4 * qk * dk + 3 * heads * dv) + 16 * heads) + 3 * 4 * envs * heads * dk * dv
        flops += 15 * tokens * heads * dk * dv  # S do, k dS, dS u, S dx, two rank-1 updates, decay, <dS, S>
    return dict(bytes=size, flops=flops)


# ------------------------------------------------------------------ exact

def _exact_chunk(q, k, v, g, beta, seg, state):
    """One chunk of the delta rule in 64 bits as a linear system: w = v - (decayed state)^T k over the chunk's
    steps. seg: the number of resets up to each step. Arrays [envs, heads, chunk, ...]."""
    n = g.shape[-1]
    total = torch.cumsum(g, -1)
    same = (seg[..., :, None] == seg[..., None, :]) & torch.tril(torch.ones(n, n, dtype=torch.bool, device=g.device))
    # g is finite: a reset is a change of segment, not an infinite decay
    pair = torch.where(same, torch.exp(torch.where(same, total[..., :, None] - total[..., None, :], 0.0)), 0.0)
    first = torch.where(seg == 0, torch.exp(total), 0.0)
    kk = torch.einsum("bhid,bhjd->bhij", k, k)
    system = torch.eye(n, dtype=g.dtype, device=g.device) + torch.tril(pair * kk, -1) * beta[..., None, :]
    rhs = v - first[..., None] * torch.einsum("bhid,bhde->bhie", k, state)
    w = torch.linalg.solve_triangular(system, rhs, upper=False)
    u = beta[..., None] * w
    o = first[..., None] * torch.einsum("bhid,bhde->bhie", q, state)
    o = o + torch.einsum("bhij,bhje->bhie", pair * torch.einsum("bhid,bhjd->bhij", q, k), u)
    state = first[..., -1, None, None] * state + torch.einsum("bhi,bhid,bhie->bhde", pair[..., -1, :], k, u)
    return o, state


def _exact_rollout(case, s):
    steps, envs, heads, qk = case["steps"], case["envs"], case["heads"], case["qk_heads"]
    dk, dv, chunk = case["dk"], case["dv"], 32
    bytes_64 = 8 * envs * heads * (6 * steps * (dk + dv) + (1 + steps // chunk) * 6 * (dk * dv + 4 * chunk * chunk))
    if bytes_64 * (3 if case["grad"] else 1) > 60e9:
        return None
    names = ["q", "k", "v", "log_decay", "beta", "state"]
    leaf = {n: s[n].double().requires_grad_(case["grad"]) for n in names}
    q, k = leaf["q"], leaf["k"]
    if case["normalize"]:
        q, k = (x / torch.sqrt((x ** 2).sum(-1, keepdim=True) + EPS) for x in (q, k))
    live = torch.ones(steps, envs, dtype=torch.float64, device="cuda")
    if s["lengths"] is not None:  # steps past an environment's end write nothing and forget nothing
        live = (torch.arange(steps, device="cuda")[:, None] < s["lengths"]).double()
    starts = torch.zeros(steps, envs, device="cuda") if s["starts"] is None else (s["starts"] != 0).double()
    starts = starts * live

    def heads_first(x):  # [steps, envs, heads, ...] -> [envs, heads, steps, ...]
        return x.movedim(0, 2)

    q, k = (heads_first(torch.repeat_interleave(x, heads // qk, 2)) for x in (q, k))
    v = heads_first(leaf["v"])
    g = heads_first(leaf["log_decay"] * live[..., None])
    beta = heads_first(leaf["beta"] * live[..., None])
    seg = starts.movedim(0, 1)[:, None]
    state, outs = leaf["state"], []
    for a in range(0, steps, chunk):
        part = slice(a, min(a + chunk, steps))
        o, state = _exact_chunk(q[:, :, part], k[:, :, part], v[:, :, part], g[:, :, part], beta[:, :, part],
                                torch.cumsum(seg[..., part], -1), state)
        outs.append(o)
    out = torch.cat(outs, 2).movedim(2, 0) * live[..., None, None] / math.sqrt(dk)
    result = dict(out=out.detach(), state=state.detach())
    if case["grad"]:
        loss = (out * s["dout"].double()).sum() + (state * s["dstate"].double()).sum()
        grads = torch.autograd.grad(loss, [leaf[n] for n in names])
        result.update(zip(("dq", "dk", "dv", "dlog_decay", "dbeta", "dstate"), grads))
    return result


def _exact_tick(case, s):
    heads, qk = case["heads"], case["qk_heads"]
    q, k = (s[n].double() for n in ("q", "k"))
    q, k = (torch.repeat_interleave(x / torch.sqrt((x ** 2).sum(-1, keepdim=True) + EPS), heads // qk, 1)
            for x in (q, k))
    keep = torch.exp(s["log_decay"].double()) * (s["starts"] == 0).double()[:, None]
    state = s["state"].double() * keep[..., None, None]
    u = s["beta"].double()[..., None] * (s["v"].double() - torch.einsum("bhd,bhde->bhe", k, state))
    state = state + torch.einsum("bhd,bhe->bhde", k, u)
    return dict(out=torch.einsum("bhd,bhde->bhe", q, state) / math.sqrt(case["dk"]), state=state)


def _exact_norm(case, s):
    def norm(x):
        return x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + EPS)

    gated = case["block"] and s["gate"] is not None
    names = ["branch", "branch_weight", "residual_scale"] * case["block"] + ["gate"] * gated
    leaf = {n: s[n].double().requires_grad_(case["grad"]) for n in names}
    weight = s["norm_weight"].double().requires_grad_(case["grad"])

    def branch():
        a = 1.0
        if gated:
            a = 1.0 / (1.0 + torch.exp(-leaf["gate"]))
            a = a * leaf["gate"] if case["gate"] == "silu" else a
        return leaf["residual_scale"] * a * (norm(leaf["branch"]) * leaf["branch_weight"])

    h = s["x"].double()
    if case["block"]:
        h = h + branch()
    result = dict(y=(norm(h) * weight).detach())
    if not case["block"]:
        return result
    result["h"] = h.detach()
    if case["grad"]:
        # the gradient's input is the residual stream as it was kept: rounded from 32 bits to its own type
        stream = DTYPES[case["stream"]]
        kept = h.detach().float().to(stream).double().requires_grad_(True)
        dhat, result["dnorm_weight"] = torch.autograd.grad((norm(kept) * weight * s["dy"].double()).sum(),
                                                           [kept, weight])
        dh = s["dh"].double() + dhat
        result["dx"] = dh
        grads = torch.autograd.grad((branch() * dh).sum(), [leaf[n] for n in names])
        result.update(("d" + n, x) for n, x in zip(names, grads))
    return result


def exact(case, seed):
    s = prepare(case, seed)
    return {"tick": _exact_tick, "delta": _exact_rollout, "norm": _exact_norm}[case["op"]](case, s)

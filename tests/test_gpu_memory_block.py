"""The memory-block operators (delta_rule, delta_step, block_norm and their gradients) against the 64-bit
restatement of their formulas, at the sizes, masks, layouts and streams where such kernels go wrong.

Tolerances, fixed before the kernels first ran. u = 2^-24 is the unit roundoff of 32 bits. A value of the delta rule
is a sum over a key axis of at most 128 products with a state that remembers some tens of steps, each step with a
relative error of the order of u sqrt(128): together about u sqrt(128 * 30) = 62 u = 4e-6 of the array's rms, with
random signs; F32_NORM holds the 2-norm to that and F32_MAX one value to ten times it. A norm's row sums give
u sqrt(dim) at most 5e-6 of a value, weight gradients the same over rows. A bf16 output adds its own rounding: bf16 has
8 significant bits, so half an ulp is up to 2^-8 of the value.
"""

import numpy as np
import pytest

from conftest import load_package
from memory_reference import block, delta, next_norm

pytestmark = pytest.mark.gpu

F32_NORM, F32_MAX, BF16_ROUND = 4e-6, 4e-5, 2.0 ** -8


@pytest.fixture(scope="module")
def torch():
    import torch
    torch.manual_seed(5)
    return torch


@pytest.fixture(scope="module")
def mdn():
    return load_package()


def close(got, want, name, scale=1.0):
    """got (32 bits or bf16) against want (64 bits)."""
    bf16 = "bfloat16" in str(got.dtype)
    g, w = got.detach().double().cpu().numpy(), want.detach().double().cpu().numpy()
    assert g.shape == w.shape, (name, g.shape, w.shape)
    if not w.size:
        return
    assert np.isfinite(g).all(), f"{name}: not finite"
    rms = np.sqrt(np.mean(w * w))
    err = np.abs(g - w)
    allowed = F32_MAX * scale * np.maximum(rms, np.abs(w)) + (BF16_ROUND * np.abs(w) if bf16 else 0.0) + 1e-30
    assert (err <= allowed).all(), f"{name}: {(err / allowed).max():.3g} times what one value may be off"
    if not bf16:
        assert np.linalg.norm(g - w) <= F32_NORM * scale * np.linalg.norm(w) + 1e-30, \
            f"{name}: 2-norm off by {np.linalg.norm(g - w) / np.linalg.norm(w):.3g}"


class Rollout:
    """Inputs of one rollout on the GPU and, in 64 bits, on the CPU."""

    def __init__(self, torch, dtype, steps, envs, qk, heads, dk, dv, resets=0.0, ragged=False, state=True, seed=1):
        gen = torch.Generator().manual_seed(seed * 7919 + steps * 31 + envs * 17 + dk * 5 + dv)
        dt = dict(f32=torch.float32, bf16=torch.bfloat16)[dtype]

        def rand(*shape, kind=torch.float32, std=1.0):
            return (torch.randn(*shape, generator=gen) * std).to(kind)
        self.torch, self.dt = torch, dt
        self.q, self.k = rand(steps, envs, qk, dk, kind=dt), rand(steps, envs, qk, dk, kind=dt)
        self.v = rand(steps, envs, heads, dv, kind=dt)
        self.log_decay = -torch.exp(rand(steps, envs, heads) - 2.5)
        self.beta = torch.sigmoid(rand(steps, envs, heads))
        self.state = rand(envs, heads, dk, dv, std=0.3) if state else None
        self.starts = (torch.rand(steps, envs, generator=gen) < resets).to(torch.uint8) if resets else None
        self.lengths = torch.randint(0, steps + 1, (envs,), generator=gen, dtype=torch.int32) if ragged else None
        if ragged and envs > 1:
            self.lengths[0], self.lengths[-1] = 0, steps
        self.dout, self.dstate = rand(steps, envs, heads, dv, kind=dt), rand(envs, heads, dk, dv, std=0.1)

    NAMES = ("q", "k", "v", "log_decay", "beta", "state")

    def gpu(self, *names):
        return [None if getattr(self, n) is None else getattr(self, n).cuda() for n in names]

    def exact(self, normalize=True, scale=None, grad=False):
        torch = self.torch
        leaf = [getattr(self, n) for n in self.NAMES]
        shape = (self.v.shape[1], self.v.shape[2], self.q.shape[3], self.v.shape[3])
        leaf[5] = torch.zeros(shape) if leaf[5] is None else leaf[5]
        leaf = [x.double().requires_grad_(grad) for x in leaf]
        out, state = delta(*leaf, self.starts, self.lengths, scale, normalize)
        if not grad:
            return out, state
        loss = (out * self.dout.double()).sum() + (state * self.dstate.double()).sum()
        grads = torch.autograd.grad(loss, leaf, allow_unused=True)
        return out, state, [torch.zeros_like(x) if g is None else g for x, g in zip(leaf, grads)]


SHAPES = [  # steps, envs, qk heads, heads, key, value
    (1, 1, 1, 1, 1, 1), (1, 5, 2, 4, 64, 64), (2, 3, 1, 1, 8, 16), (15, 2, 1, 2, 16, 33), (16, 3, 2, 2, 32, 32),
    (17, 2, 1, 1, 64, 64), (33, 4, 1, 3, 40, 72), (50, 2, 2, 2, 128, 128), (64, 1, 1, 1, 100, 65), (100, 2, 1, 2, 64, 128),
    (47, 3, 1, 1, 33, 1), (31, 2, 1, 1, 1, 64), (130, 1, 1, 1, 128, 17), (3, 1, 1, 1, 65, 100),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("resets,ragged,normalize", [(0.0, False, True), (0.1, True, True), (0.4, False, False)])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_rollout_and_gradients(torch, mdn, shape, resets, ragged, normalize, dtype):
    r = Rollout(torch, dtype, *shape, resets=resets, ragged=ragged)
    if not normalize:  # keys of about unit length, as a caller without normalize has them
        r.q, r.k = ((x.float() * x.shape[-1] ** -0.5).to(r.dt) for x in (r.q, r.k))
    want_out, want_state, want = r.exact(normalize, grad=True)
    args = r.gpu(*Rollout.NAMES)
    starts, lengths, dout, dstate = r.gpu("starts", "lengths", "dout", "dstate")
    out, state, saved = mdn.delta_rule(*args, starts=starts, lengths=lengths, normalize=normalize, save=True)
    close(out, want_out, "out")
    close(state, want_state, "state")
    got = mdn.delta_rule_backward(saved, dout, dstate)
    for name, g, w in zip(Rollout.NAMES, got, want):
        close(g, w, "d" + name)
    plain = mdn.delta_rule(*args, starts=starts, lengths=lengths, normalize=normalize)
    close(plain[0], want_out, "out without save")
    close(plain[1], want_state, "state without save")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("steps", [0, 1, 40])
def test_rollout_without_state_scale_and_gradient_of_state(torch, mdn, steps, dtype):
    r = Rollout(torch, dtype, steps, 3, 1, 2, 24, 48, state=False)
    q, k, v, g, b, _ = r.gpu(*Rollout.NAMES)
    out, state, saved = mdn.delta_rule(q, k, v, g, b, scale=0.7, save=True)
    r.dstate = torch.zeros_like(r.dstate)
    want_out, want_state, want = r.exact(scale=0.7, grad=True)
    close(out, want_out, "out")
    close(state, want_state, "state")
    for name, got, w in zip(Rollout.NAMES, mdn.delta_rule_backward(saved, r.dout.cuda()), want):
        close(got, w, "d" + name)


def test_no_environments(torch, mdn):
    z = dict(device="cuda")
    q, v = torch.zeros(4, 0, 2, 8, **z), torch.zeros(4, 0, 2, 8, **z)
    g, s = torch.zeros(4, 0, 2, **z), torch.zeros(0, 2, 8, 8, **z)
    out, state, saved = mdn.delta_rule(q, q, v, g, g, s, save=True)
    assert out.shape == v.shape and state.shape == s.shape
    assert mdn.delta_rule_backward(saved, v, s)[0].shape == q.shape


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradients_against_differences(torch, mdn, dtype):
    """Directional derivatives of the 64-bit formulas by central differences (step 1e-5, error about 1e-9)."""
    r = Rollout(torch, dtype, 37, 2, 1, 2, 48, 40, resets=0.06, ragged=True, seed=3)
    args = r.gpu(*Rollout.NAMES)
    starts, lengths, dout, dstate = r.gpu("starts", "lengths", "dout", "dstate")
    *_, saved = mdn.delta_rule(*args, starts=starts, lengths=lengths, save=True)
    grads = mdn.delta_rule_backward(saved, dout, dstate)
    base = [getattr(r, n).double() for n in Rollout.NAMES]

    def loss(xs):
        out, state = delta(*xs, r.starts, r.lengths)
        return float((out * r.dout.double()).sum() + (state * r.dstate.double()).sum())
    for i, name in enumerate(Rollout.NAMES):
        direction = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(i)).double()
        at = [[x + s * 1e-5 * direction if j == i else x for j, x in enumerate(base)] for s in (1, -1)]
        want = (loss(at[0]) - loss(at[1])) / 2e-5
        got = float((grads[i].double().cpu() * direction).sum())
        size = float(grads[i].double().norm())  # a random direction's product has about this spread
        tolerance = (2.0 ** -8 if grads[i].dtype == torch.bfloat16 else F32_NORM) * 4 * size + 1e-6 * (1 + abs(want))
        assert abs(got - want) <= tolerance, (name, got, want, tolerance)


@pytest.mark.parametrize("steps,at", [(40, 0), (40, 5), (40, 16), (40, 23)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_an_episode_does_not_see_the_one_before(torch, mdn, steps, at, bad):
    """What is not finite before a start, in the state or in an earlier episode, stays there."""
    r = Rollout(torch, "f32", steps, 3, 1, 2, 32, 48)
    r.starts = torch.zeros(steps, 3, dtype=torch.uint8)
    r.starts[at, 1] = 1
    args = r.gpu(*Rollout.NAMES)
    starts, dout, dstate = r.gpu("starts", "dout", "dstate")

    def both(xs, d):
        out, state, saved = mdn.delta_rule(*xs, starts=starts, save=True)
        return (out, state), mdn.delta_rule_backward(saved, d, dstate)
    clean, clean_grads = both(args, dout)
    dirty = [x.clone() for x in args]
    d = dout.clone()
    dirty[5][1] = bad
    if at:
        for x in dirty[:3]:
            x[:at, 1] = bad
        d[:at, 1] = bad
    got, grads = both(dirty, d)
    assert torch.equal(got[0][at:, 1], clean[0][at:, 1]) and torch.equal(got[1][1], clean[1][1])
    for g, c in zip(grads[:5], clean_grads[:5]):
        assert torch.equal(g[at:, 1], c[at:, 1])
    for env in (0, 2):
        assert torch.equal(got[0][:, env], clean[0][:, env]) and torch.equal(got[1][env], clean[1][env])
        for g, c in zip(grads[:5], clean_grads[:5]):
            assert torch.equal(g[:, env], c[:, env])
    if at == 0:  # the state of that environment was not read and gets no gradient
        assert not grads[5][1].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_steps_past_the_length_are_not_read(torch, mdn, dtype):
    r = Rollout(torch, dtype, 39, 4, 1, 2, 40, 24, resets=0.05)
    r.lengths = torch.tensor([0, 39, 20, -3], dtype=torch.int32)
    args = r.gpu(*Rollout.NAMES)
    starts, lengths, dout, dstate = r.gpu("starts", "lengths", "dout", "dstate")
    for x in args[:5] + [dout]:
        for env, n in ((0, 0), (2, 20), (3, 0)):
            x[n:, env] = float("nan")
    want_out, want_state, want = r.exact(grad=True)
    out, state, saved = mdn.delta_rule(*args, starts=starts, lengths=lengths, save=True)
    close(out, want_out, "out")
    close(state, want_state, "state")
    assert not out[:, 0].any() and not out[20:, 2].any() and torch.equal(state[0], args[5][0])
    for name, g, w in zip(Rollout.NAMES, mdn.delta_rule_backward(saved, dout, dstate), want):
        close(g, w, "d" + name)


def test_full_forgetting_and_strong_decays(torch, mdn):
    """A log-decay of -inf clears the memory like a start; large decays underflow quietly."""
    r = Rollout(torch, "f32", 36, 2, 1, 2, 32, 32)
    r.log_decay[5], r.log_decay[20] = float("-inf"), float("-inf")
    r.log_decay[9:12], r.log_decay[30] = -90.0, -200.0
    r.log_decay[25:27] = 0.0
    args = r.gpu(*Rollout.NAMES)
    out, state, saved = mdn.delta_rule(*args, save=True)
    grads = mdn.delta_rule_backward(saved, *r.gpu("dout", "dstate"))
    want_out, want_state, want = r.exact(grad=True)
    want[3][5] = want[3][20] = 0.0  # autograd's own 0 * inf there
    close(out, want_out, "out")
    close(state, want_state, "state")
    for name, g, w in zip(Rollout.NAMES, grads, want):
        close(g, w, "d" + name)


def test_betas_of_zero_and_zero_keys(torch, mdn):
    r = Rollout(torch, "f32", 20, 2, 1, 1, 16, 16)
    r.beta[3:6], r.beta[10] = 0.0, 1.0
    r.k[7], r.q[8] = 0.0, 0.0
    args = r.gpu(*Rollout.NAMES)
    out, state, saved = mdn.delta_rule(*args, save=True)
    want_out, want_state, want = r.exact(grad=True)
    close(out, want_out, "out")
    close(state, want_state, "state")
    for name, g, w in zip(Rollout.NAMES, mdn.delta_rule_backward(saved, *r.gpu("dout", "dstate")), want):
        close(g, w, "d" + name)


def layouts_of(torch, r):
    """The same values in other layouts: slices of one fused projection, environment-major, one element off any
    16-byte boundary."""
    def odd(x):
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:]
        flat.copy_(x.reshape(-1))
        return flat.view(x.shape)

    args = r.gpu(*Rollout.NAMES)
    q, k, v, g, b, s = args
    steps, envs = q.shape[:2]
    sizes = [x[0, 0].numel() for x in (q, k, v)]
    fused = torch.cat([x.reshape(steps, envs, -1) for x in (q, k, v)], -1)
    parts = [p.unflatten(-1, x.shape[2:]) for p, x in zip(fused.split(sizes, -1), (q, k, v))]
    decays = torch.stack([g, b], -1)
    major = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, g, b)]
    headed = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, g, b)]
    return dict(fused=[*parts, decays[..., 0], decays[..., 1], s], env_major=major + [s], head_major=headed + [s],
                unaligned=[odd(x) for x in args])


@pytest.mark.parametrize("layout", ["fused", "env_major", "head_major", "unaligned"])
@pytest.mark.parametrize("dtype,shape", [("f32", (35, 3, 2, 4, 32, 64)), ("bf16", (35, 3, 1, 2, 64, 32)),
                                         ("bf16", (19, 2, 1, 1, 37, 21)), ("bf16", (1, 6, 1, 2, 64, 64)),
                                         ("f32", (1, 6, 2, 2, 36, 20))])
def test_layouts(torch, mdn, layout, dtype, shape):
    r = Rollout(torch, dtype, *shape, resets=0.05)
    want_out, want_state, want = r.exact(grad=True)
    args = layouts_of(torch, r)[layout]
    starts, dout, dstate = r.gpu("starts", "dout", "dstate")
    starts = starts.t().contiguous().t()
    dout = dout.transpose(0, 2).contiguous().transpose(0, 2)
    out, state, saved = mdn.delta_rule(*args, starts=starts.bool(), save=True)
    close(out, want_out, "out")
    close(state, want_state, "state")
    for name, g, w in zip(Rollout.NAMES, mdn.delta_rule_backward(saved, dout, dstate), want):
        close(g, w, "d" + name)


def test_broadcast_inputs(torch, mdn):
    """One decay for all heads, one query for all environments: strides of zero."""
    r = Rollout(torch, "f32", 30, 3, 2, 2, 32, 32)
    r.log_decay = r.log_decay[:, :, :1].expand(-1, -1, 2)
    r.q = r.q[:, :1].expand(-1, 3, -1, -1)
    want_out, want_state, want = r.exact(grad=True)
    q, k, v, g, b, s = r.gpu(*Rollout.NAMES)
    g = g[:, :, :1].expand(-1, -1, 2)
    q = q[:, :1].expand(-1, 3, -1, -1)
    out, state, saved = mdn.delta_rule(q, k, v, g, b, s, save=True)
    close(out, want_out, "out")
    for name, got, w in zip(Rollout.NAMES, mdn.delta_rule_backward(saved, *r.gpu("dout", "dstate")), want):
        close(got, w, "d" + name)


def test_long_offsets(torch, mdn):
    """Rows more than 2^32 bytes and 2^31 elements apart."""
    steps, envs, dk, dv = 18, 2, 64, 64
    r = Rollout(torch, "bf16", steps, envs, 1, 1, dk, dv)
    far = 1_200_000_128  # elements between the environments, times two steps' worth of rows
    buffer = torch.empty(2 * far, dtype=torch.bfloat16, device="cuda")

    def spread(x, at):
        view = buffer[at:].as_strided(x.shape, (x.shape[2] * x.shape[3], far, x.shape[3], 1))
        view.copy_(x.cuda())
        return view
    q, k, v = spread(r.q, 0), spread(r.k, 1 << 16), spread(r.v, 1 << 17)
    _, _, _, g, b, s = r.gpu(*Rollout.NAMES)
    out, state, saved = mdn.delta_rule(q, k, v, g, b, s, save=True)
    want_out, want_state, want = r.exact(grad=True)
    close(out, want_out, "out")
    close(state, want_state, "state")
    for name, got, w in zip(Rollout.NAMES, mdn.delta_rule_backward(saved, *r.gpu("dout", "dstate")), want):
        close(got, w, "d" + name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 64, 64), (37, 2, 4, 32, 32), (5, 1, 3, 128, 128), (9, 1, 1, 50, 70),
                                   (3, 1, 2, 7, 3), (300, 1, 1, 16, 128)])
def test_tick(torch, mdn, shape, dtype):
    envs, qk, heads, dk, dv = shape
    r = Rollout(torch, dtype, 3, envs, qk, heads, dk, dv, resets=0.2)
    want_out, want_state = r.exact()
    q, k, v, g, b, s = r.gpu(*Rollout.NAMES)
    starts = r.starts.cuda()
    state = s.clone()
    state[starts[0] != 0] = float("nan")  # never read
    for t in range(3):
        out, got = mdn.delta_step(q[t], k[t], v[t], g[t], b[t], state, starts=starts[t])
        assert got is state
        close(out, want_out[t], f"out {t}")
    close(state, want_state, "state")
    other, target = torch.empty_like(out), torch.empty_like(s)
    before = s.clone()
    got = mdn.delta_step(q[0], k[0], v[0], g[0], b[0], s, out=other, state_out=target, normalize=True)
    assert got[0] is other and got[1] is target and torch.equal(s, before)


def test_rollout_in_pieces(torch, mdn):
    """A rollout cut anywhere and continued from its state gives the same values as one call."""
    r = Rollout(torch, "f32", 75, 2, 1, 2, 64, 48, resets=0.03)
    q, k, v, g, b, s = r.gpu(*Rollout.NAMES)
    starts = r.starts.cuda()
    want_out, want_state = r.exact()
    outs, state = [], s
    for a, e in ((0, 1), (1, 20), (20, 20), (20, 52), (52, 75)):
        o, state = mdn.delta_rule(q[a:e], k[a:e], v[a:e], g[a:e], b[a:e], state, starts=starts[a:e])
        outs.append(o)
    close(torch.cat(outs), want_out, "out")
    close(state, want_state, "state")


@pytest.mark.parametrize("steps", [2048, 5000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_axis(torch, mdn, steps, dtype):
    """Few environments, a long axis."""
    r = Rollout(torch, dtype, steps, 1, 1, 2, 64, 64, resets=0.0005)
    want_out, want_state, want = r.exact(grad=True)
    args = r.gpu(*Rollout.NAMES)
    starts, dout, dstate = r.gpu("starts", "dout", "dstate")
    out, state, saved = mdn.delta_rule(*args, starts=starts, save=True)
    close(out, want_out, "out")
    close(state, want_state, "state")
    for name, g, w in zip(Rollout.NAMES, mdn.delta_rule_backward(saved, dout, dstate), want):
        close(g, w, "d" + name)


def test_deterministic_streams_and_graph(torch, mdn):
    """The same bits again, on another stream, and from a replayed graph with new inputs."""
    r = Rollout(torch, "bf16", 70, 9, 1, 3, 64, 64, resets=0.03)
    args = r.gpu(*Rollout.NAMES)
    starts, dout, dstate = r.gpu("starts", "dout", "dstate")

    def go():
        out, state, saved = mdn.delta_rule(*args, starts=starts, save=True)
        return (out, state, *mdn.delta_rule_backward(saved, dout, dstate))
    first = go()
    for a, b in zip(first, go()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = go()
    side.synchronize()
    for a, b in zip(first, again):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = go()
    args[2].mul_(-1.0)
    args[5].mul_(-1.0)  # linear in values and state: outputs change sign
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured[0], -first[0]) and torch.equal(captured[1], -first[1])


def test_autograd(torch, mdn):
    r = Rollout(torch, "f32", 21, 2, 1, 2, 32, 32)
    args = [x.requires_grad_() for x in r.gpu(*Rollout.NAMES)]
    out, state = mdn.delta_rule_train(*args)
    ((out * r.dout.cuda()).sum() + (state * r.dstate.cuda()).sum()).backward()
    for name, x, w in zip(Rollout.NAMES, args, r.exact(grad=True)[2]):
        close(x.grad, w, "d" + name)
    q, k, v, g, b, _ = r.gpu(*Rollout.NAMES)
    v.requires_grad_()
    mdn.delta_rule_train(q, k, v, g, b)[0].sum().backward()
    assert v.grad is not None


def test_delta_refusals(torch, mdn):
    r = Rollout(torch, "f32", 4, 2, 1, 2, 16, 16)
    q, k, v, g, b, s = r.gpu(*Rollout.NAMES)

    def refused(fn, *args, **kw):
        with pytest.raises(mdn.MdnError) as e:
            fn(*args, **kw)
        assert e.value.code == 1
    refused(mdn.delta_rule, q.cpu(), k, v, g, b, s)
    refused(mdn.delta_rule, q, k.bfloat16(), v, g, b, s)
    refused(mdn.delta_rule, q.double(), k, v, g, b, s)
    refused(mdn.delta_rule, q, k, v, g.double(), b, s)
    refused(mdn.delta_rule, q, k, v, g, b[:2], s)
    refused(mdn.delta_rule, q, k, v, g, b, s[:1])
    refused(mdn.delta_rule, q, k, v, g, b, s.transpose(2, 3))
    refused(mdn.delta_rule, q, k, v[:, :, :1].expand(-1, -1, 3, -1)[..., ::2], g, b, s)
    refused(mdn.delta_rule, q.transpose(0, 3), k, v, g, b, s)
    refused(mdn.delta_rule, q, k, v, g, b, s, starts=torch.zeros(4, 2, device="cuda"))
    refused(mdn.delta_rule, q, k, v, g, b, s, lengths=torch.zeros(2, device="cuda"))
    refused(mdn.delta_rule, q, k, v, g, b, s, norm_eps=-1.0)
    refused(mdn.delta_rule, q, k, v, g, b, s, scale=float("nan"))
    wide = torch.zeros(4, 2, 1, 129, device="cuda")
    refused(mdn.delta_rule, wide, wide, v, g, b)
    two = torch.zeros(4, 2, 2, 16, device="cuda")
    three = torch.zeros(4, 2, 3, 16, device="cuda")
    refused(mdn.delta_rule, two, two, three, g, b)
    refused(mdn.delta_step, q[0], k[0], v[0], g[0], b[0], None)
    refused(mdn.delta_step, q, k, v, g, b, s)
    *_, saved = mdn.delta_rule(q, k, v, g, b, s, save=True)
    refused(mdn.delta_rule_backward, saved, v.bfloat16())
    refused(mdn.delta_rule_backward, saved, v, s[:1])


# ------------------------------------------------------------ block norms

def norm_inputs(torch, rows, dim, dtype, stream, branch, gate, weights, seed=0):
    gen = torch.Generator().manual_seed(seed + rows * 13 + dim)
    types = dict(f32=torch.float32, bf16=torch.bfloat16)

    def rand(*shape, kind="f32", std=1.0, mean=0.0):
        return (mean + std * torch.randn(*shape, generator=gen)).to(types[kind])
    return dict(x=rand(rows, dim, kind=stream), branch=rand(rows, dim, kind=dtype, std=0.7) if branch else None,
                gate=rand(rows, dim, kind=dtype, std=2.0) if gate else None,
                branch_weight=rand(dim, mean=1.0, std=0.1) if branch and weights else None,
                residual_scale=rand(dim, mean=0.3, std=0.1) if branch and weights else None,
                norm_weight=rand(dim, mean=1.0, std=0.1) if weights else None,
                dh=rand(rows, dim, kind=stream), dy=rand(rows, dim, kind=dtype))


NORM_SHAPES = [(1, 1), (3, 2), (1, 184), (5, 31), (700, 33), (64, 480), (33, 515), (9, 1024), (300, 64), (4, 5120),
               (3, 8191), (2, 8192), (1500, 7)]


def check_norm(torch, mdn, i, act, eps=1e-6, gpu=None, dh=True, dy=True):
    order = ("x", "branch", "gate", "branch_weight", "residual_scale", "norm_weight")
    leaf = {n: None if i[n] is None else i[n].double().requires_grad_() for n in order}
    want_h, want_y = block(*leaf.values(), act, eps)
    c = gpu or {n: None if t is None else t.cuda() for n, t in i.items()}
    kind = {} if i["branch"] is not None else dict(dtype=i["dy"].dtype)
    h, y = mdn.block_norm(*(c[n] for n in order), gate_act=act, eps=eps, **kind)
    close(h, want_h, "h")
    close(y, want_y, "y")
    # gradients from the h that was kept
    kept = (h if i["branch"] is not None else c["x"]).double().cpu().requires_grad_()
    weight = leaf["norm_weight"]
    dhat = torch.zeros_like(kept)
    dweight = None if weight is None else torch.zeros_like(weight)
    if dy:
        loss = (next_norm(kept, weight, eps) * i["dy"].double()).sum()
        got = torch.autograd.grad(loss, [kept] if weight is None else [kept, weight])
        dhat, dweight = got[0], dweight if weight is None else got[1]
    total = dhat + (i["dh"].double() if dh else 0.0)
    want = dict(dx=total, dnorm_weight=dweight)
    if i["branch"] is not None:
        names = [n for n in order[1:5] if leaf[n] is not None]
        zero = torch.zeros_like(leaf["x"])
        grads = torch.autograd.grad((block(zero, *list(leaf.values())[1:], act, eps)[0] * total).sum(),
                                    [leaf[n] for n in names])
        want.update(("d" + n, g) for n, g in zip(names, grads))
    grads = mdn.block_norm_backward(h, *(c[n] for n in order[1:]), c["dh"] if dh else None, c["dy"] if dy else None,
                                    gate_act=act, eps=eps)
    for name, g in zip(["d" + n for n in order], grads):
        if want.get(name) is None:
            assert g is None, name
        else:
            close(g, want[name], name)


@pytest.mark.parametrize("dtype,stream", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("branch,gate,act,weights", [(True, True, "sigmoid", True), (True, True, "silu", True),
                                                     (True, False, "silu", False), (False, False, "sigmoid", True)])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_block_norm(torch, mdn, shape, branch, gate, act, weights, dtype, stream):
    check_norm(torch, mdn, norm_inputs(torch, *shape, dtype, stream, branch, gate, weights), act)


@pytest.mark.parametrize("dh,dy", [(True, False), (False, True)])
def test_block_norm_one_gradient(torch, mdn, dh, dy):
    check_norm(torch, mdn, norm_inputs(torch, 40, 96, "f32", "f32", True, True, True), "silu", dh=dh, dy=dy)


@pytest.mark.parametrize("dim", [64, 100, 480])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_block_norm_layouts(torch, mdn, dtype, dim):
    """Rows that are slices of wider ones, and buffers off any 16-byte boundary."""
    i = norm_inputs(torch, 50, dim, dtype, dtype, True, True, True, seed=4)
    wide = {n: None if t is None or t.dim() == 1 else torch.zeros(50, dim + 37, dtype=t.dtype) for n, t in i.items()}
    gpu = {}
    for n, t in i.items():
        if t.dim() == 1:
            gpu[n] = torch.cat([t[:1], t]).cuda()[1:]
        else:
            wide[n][:, 3:3 + dim] = t
            gpu[n] = wide[n].cuda()[:, 3:3 + dim]
    check_norm(torch, mdn, i, "sigmoid", gpu=gpu)


def test_block_norm_zero_rows_and_no_rows(torch, mdn):
    i = norm_inputs(torch, 12, 48, "f32", "f32", True, True, True)
    i["branch"][3], i["x"][5], i["branch"][5] = 0.0, 0.0, 0.0
    i["gate"][7], i["gate"][8] = -200.0, 200.0
    check_norm(torch, mdn, i, "silu")
    empty = {n: t[:0] if t.dim() == 2 else t for n, t in i.items()}
    c = {n: t.cuda() for n, t in empty.items()}
    names = ("x", "branch", "gate", "branch_weight", "residual_scale", "norm_weight")
    h, y = mdn.block_norm(*(c[n] for n in names))
    assert h.shape == y.shape == (0, 48)
    grads = mdn.block_norm_backward(h, *(c[n] for n in names[1:]), c["dh"], c["dy"])
    assert grads[0].shape == (0, 48) and all(not g.any() for g in grads[3:])


def test_block_norm_rows_stay_apart(torch, mdn):
    """NaN and infinities in one row change no other row."""
    i = norm_inputs(torch, 30, 96, "bf16", "f32", True, True, True)
    c = {n: t.cuda() for n, t in i.items()}
    names = ("x", "branch", "gate", "branch_weight", "residual_scale", "norm_weight")
    clean = mdn.block_norm(*(c[n] for n in names))
    clean_grads = mdn.block_norm_backward(clean[0], *(c[n] for n in names[1:]), c["dh"], c["dy"])
    bad = {n: t.clone() for n, t in c.items()}
    bad["x"][4], bad["branch"][11], bad["gate"][17, 5] = float("nan"), float("inf"), float("nan")
    got = mdn.block_norm(*(bad[n] for n in names))
    grads = mdn.block_norm_backward(got[0], *(bad[n] for n in names[1:]), c["dh"], c["dy"])
    fine = [r for r in range(30) if r not in (4, 11, 17)]
    for a, b in zip(clean + clean_grads[:3], got + grads[:3]):
        assert torch.equal(a[fine], b[fine])


def test_block_norm_deterministic_streams_and_graph(torch, mdn):
    i = {n: t.cuda() for n, t in norm_inputs(torch, 5000, 480, "bf16", "f32", True, True, True).items()}
    names = ("x", "branch", "gate", "branch_weight", "residual_scale", "norm_weight")

    def go():
        h, y = mdn.block_norm(*(i[n] for n in names), gate_act="silu")
        return (h, y, *mdn.block_norm_backward(h, *(i[n] for n in names[1:]), i["dh"], i["dy"], gate_act="silu"))
    first = go()
    for a, b in zip(first, go()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = go()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = go()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, captured))


def test_block_norm_long_offsets(torch, mdn):
    """Rows whose offsets pass 2^32 bytes and 2^31 elements."""
    far, dim = 1_100_000_000, 65
    i = norm_inputs(torch, 3, dim, "bf16", "bf16", True, False, True)
    buffer = torch.empty(2 * far + 4096, dtype=torch.bfloat16, device="cuda")
    gpu = {n: None if t is None else t.cuda() for n, t in i.items()}
    for at, n in enumerate(("x", "branch")):
        view = buffer[at * 512:].as_strided((3, dim), (far, 1))
        view.copy_(gpu[n])
        gpu[n] = view
    check_norm(torch, mdn, i, "sigmoid", gpu=gpu)


def test_block_norm_autograd(torch, mdn):
    i = norm_inputs(torch, 10, 40, "f32", "f32", True, True, True)
    names = ("x", "branch", "gate", "branch_weight", "residual_scale", "norm_weight")
    leaf = [i[n].double().requires_grad_() for n in names]
    h, y = block(*leaf, "silu")
    want = torch.autograd.grad((h * i["dh"].double()).sum() + (y * i["dy"].double()).sum(), leaf)
    args = [i[n].cuda().requires_grad_() for n in names]
    h, y = mdn.block_norm_train(*args, gate_act="silu")
    ((h * i["dh"].cuda()).sum() + (y * i["dy"].cuda()).sum()).backward()
    for n, a, w in zip(names, args, want):
        close(a.grad, w, "d" + n)
    x, w = i["x"].cuda().requires_grad_(), i["norm_weight"].cuda().requires_grad_()
    h, y = mdn.block_norm_train(x, norm_weight=w)
    ((h * i["dh"].cuda()).sum() + (y * i["dy"].cuda()).sum()).backward()
    xr, wr = i["x"].double().requires_grad_(), i["norm_weight"].double().requires_grad_()
    dx, dw = torch.autograd.grad((xr * i["dh"].double()).sum() + (next_norm(xr, wr) * i["dy"].double()).sum(), [xr, wr])
    close(x.grad, dx, "dx")
    close(w.grad, dw, "dnorm_weight")


def test_block_norm_refusals(torch, mdn):
    i = {n: t.cuda() for n, t in norm_inputs(torch, 4, 16, "f32", "f32", True, True, True).items()}

    def refused(fn, *args, **kw):
        with pytest.raises(mdn.MdnError) as e:
            fn(*args, **kw)
        assert e.value.code == 1
    refused(mdn.block_norm, i["x"].cpu())
    refused(mdn.block_norm, i["x"].double())
    refused(mdn.block_norm, i["x"][None])
    refused(mdn.block_norm, i["x"], None, i["gate"])
    refused(mdn.block_norm, i["x"], i["branch"][:2])
    refused(mdn.block_norm, i["x"], i["branch"], i["gate"].bfloat16())
    refused(mdn.block_norm, i["x"], i["branch"], gate_act="relu")
    refused(mdn.block_norm, i["x"], i["branch"], branch_weight=i["branch_weight"][:3])
    refused(mdn.block_norm, i["x"], i["branch"], norm_weight=i["norm_weight"].bfloat16())
    refused(mdn.block_norm, i["x"], next_norm=False)
    refused(mdn.block_norm, i["x"], i["branch"], dtype=torch.bfloat16)
    refused(mdn.block_norm, i["x"].t().contiguous().t())
    refused(mdn.block_norm, torch.zeros(1, 8193, device="cuda"))
    refused(mdn.block_norm, i["x"], eps=-1.0)
    refused(mdn.block_norm_backward, i["x"])
    refused(mdn.block_norm_backward, i["x"], i["branch"], dh=i["dh"].bfloat16())


def test_library_refuses_null_call(mdn):
    lib = mdn.lib()
    assert lib.mdn_delta_forward(None, None) == 1 and b"null call" in lib.mdn_last_error()
    assert lib.mdn_block_norm_forward(None, None) == 1
    assert lib.mdn_delta_saved_bytes(None) == 0


def test_example_learns_and_ticks_agree():
    """The example end to end: the loss falls, and ticks give what the rollout gave. Two runs of the same layers in
    32 bits, one by rows of a rollout and one by ticks: each within F32_NORM of the exact values, through products that
    torch may sum in another order (u sqrt(184) = 1e-6 of a value)."""
    import importlib.util

    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("memory_policy", ROOT / "examples" / "memory_policy.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, off = example.run(envs=96, horizon=24, rollouts=5, report=lambda line: None)
    assert losses[-1] < 0.7 * losses[0], losses
    assert max(off) <= 4 * F32_NORM, off


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(20, 700, 1, 1, 16, 16), (18, 400, 1, 2, 24, 72), (7, 500, 1, 1, 100, 40)])
def test_more_environments_than_fit_at_once(torch, mdn, shape, dtype):
    """Blocks that go through several environments, some of them without any step."""
    r = Rollout(torch, dtype, *shape, resets=0.05, ragged=True)
    want_out, want_state, want = r.exact(grad=True)
    args = r.gpu(*Rollout.NAMES)
    starts, lengths, dout, dstate = r.gpu("starts", "lengths", "dout", "dstate")
    out, state, saved = mdn.delta_rule(*args, starts=starts, lengths=lengths, save=True)
    close(out, want_out, "out")
    close(state, want_state, "state")
    for name, g, w in zip(Rollout.NAMES, mdn.delta_rule_backward(saved, dout, dstate), want):
        close(g, w, "d" + name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape,resets,ragged", [
    ((497, 1, 1, 1, 64, 64), 0.0, False), ((512, 3, 1, 2, 32, 48), 0.01, True), ((1030, 2, 2, 2, 40, 72), 0.002, True),
    ((700, 1, 1, 1, 128, 17), 0.0, False), ((2100, 1, 1, 1, 33, 128), 0.001, False)])
def test_segments_of_a_long_axis(torch, mdn, shape, resets, ragged, dtype):
    """Long rollouts of few environments, cut into segments and joined; gradients from the states that were saved."""
    r = Rollout(torch, dtype, *shape, resets=resets, ragged=ragged, seed=9)
    want_out, want_state, want = r.exact(grad=True)
    args = r.gpu(*Rollout.NAMES)
    starts, lengths, dout, dstate = r.gpu("starts", "lengths", "dout", "dstate")
    out, state, saved = mdn.delta_rule(*args, starts=starts, lengths=lengths, save=True)
    close(out, want_out, "out")
    close(state, want_state, "state")
    for name, g, w in zip(Rollout.NAMES, mdn.delta_rule_backward(saved, dout, dstate), want):
        close(g, w, "d" + name)


@pytest.mark.parametrize("at", [0, 100, 530])
def test_segments_keep_episodes_apart(torch, mdn, at):
    """What is not finite before a start, in the state or the inputs, does not pass a segment's border."""
    r = Rollout(torch, "f32", 900, 1, 1, 1, 32, 32)
    r.starts = torch.zeros(900, 1, dtype=torch.uint8)
    r.starts[at, 0] = 1
    args = r.gpu(*Rollout.NAMES)
    clean = mdn.delta_rule(*args, starts=r.starts.cuda())
    dirty = [x.clone() for x in args]
    dirty[5][:] = float("nan")
    for x in dirty[:3]:
        x[:at] = float("inf")
    got = mdn.delta_rule(*dirty, starts=r.starts.cuda())
    assert torch.equal(got[0][at:], clean[0][at:]) and torch.equal(got[1], clean[1])


def test_segments_with_the_state_in_place(torch, mdn):
    """state_out may be state_in for a rollout in segments too: the first segment's state is read before the last one
    writes."""
    import sys
    memory = sys.modules[mdn.delta_rule.__module__]
    r = Rollout(torch, "f32", 1200, 2, 1, 2, 64, 64)
    q, k, v, g, b, s = r.gpu(*Rollout.NAMES)
    out, state = mdn.delta_rule(q, k, v, g, b, s)
    for _ in range(5):
        place, got = s.clone(), torch.empty_like(out)
        call = memory._delta_call(q, k, v, g, b, place, None, None, None, True, 1e-6, place, got, 0)
        size = mdn.lib().mdn_delta_forward_bytes(call)
        assert size > 0
        work = torch.empty(size, dtype=torch.uint8, device="cuda")
        mdn.capi.check(mdn.lib().mdn_delta_forward_with(call, work.data_ptr(), torch.cuda.current_stream().cuda_stream))
        assert torch.equal(got, out) and torch.equal(place, state)

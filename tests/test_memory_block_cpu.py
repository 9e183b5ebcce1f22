"""The memory-block entry points' host side: struct layouts of the Python veneer against include/mdn.h, and refusals
that need no GPU (every argument is checked before the first CUDA call)."""
import ctypes
import importlib
import subprocess
import sys

import pytest

from conftest import ROOT, load_package


@pytest.fixture(scope="module")
def pkg():
    return load_package()


@pytest.fixture(scope="module")
def memory(pkg):
    pkg.delta_rule  # loads the module
    return sys.modules[pkg.__name__ + ".memory"]


def test_struct_layouts(memory, tmp_path):
    """Sizes and the offset of every struct's last member, from the compiler."""
    src = tmp_path / "sizes.c"
    src.write_text('#include "mdn.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void) {\n'
                   'printf("%zu %zu %zu %zu %zu %zu %zu %zu\\n", sizeof(mdn_delta), offsetof(mdn_delta, saved),\n'
                   'sizeof(mdn_delta_grads), offsetof(mdn_delta_grads, workspace), sizeof(mdn_block_norm),\n'
                   'offsetof(mdn_block_norm, y), sizeof(mdn_block_norm_grads),\n'
                   'offsetof(mdn_block_norm_grads, workspace));\nreturn 0;\n}\n')
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True).stdout.split()]
    sizes = [s.size for s in (memory._DELTA, memory._DELTA_GRADS, memory._NORM, memory._NORM_GRADS)]
    assert got[0::2] == sizes
    assert got[1::2] == [sizes[0] - 8, sizes[1] - 8, sizes[2] - 16, sizes[3] - 8]


def delta_call(memory, steps=4, envs=2, heads=2, qk=1, dk=16, dv=16, dtype=0, flags=0, scale=1.0, eps=0.0, q=64,
               saved=0, starts=(0, 0, 0)):
    rows = (64, 16, 16, 16)
    return memory._DELTA.pack(steps, envs, heads, qk, dk, dv, dtype, flags, scale, eps, q, 1, 1, 1, *rows, *rows, *rows,
                              *rows, *starts, 0, 0, 0, *rows, saved)


@pytest.mark.parametrize("bad,message", [
    (dict(heads=3, qk=2), b"multiple of qk_heads"), (dict(heads=0), b"multiple of qk_heads"),
    (dict(qk=0), b"multiple of qk_heads"), (dict(dk=0), b"1..128"), (dict(dk=129), b"1..128"),
    (dict(dv=0), b"1..128"), (dict(dv=129), b"1..128"), (dict(dtype=2), b"dtype"), (dict(flags=4), b"unknown flags"),
    (dict(q=0), b"q is null"), (dict(q=66), b"q is not aligned"), (dict(scale=float("inf")), b"finite"),
    (dict(eps=-1.0), b"finite"), (dict(saved=8), b"saved is not 16-byte aligned"),
    (dict(envs=1 << 31), b"2^31"), (dict(steps=1 << 31), b"2^31")])
def test_delta_refusals(pkg, memory, bad, message):
    lib = pkg.lib()
    call = delta_call(memory, **bad)
    assert lib.mdn_delta_forward(call, None) == 1
    assert message in lib.mdn_last_error()


def test_delta_backward_refusals(pkg, memory):
    lib = pkg.lib()
    rows = (64, 16, 16, 16)

    def grads(**kw):
        f = dict(dout=rows, dq=rows, work=64)
        f.update(kw)
        return memory._DELTA_GRADS.pack(*f["dout"], 0, *f["dq"], *rows, *rows, *rows, *rows, 0, f["work"])
    assert lib.mdn_delta_backward(delta_call(memory, saved=64), None, None) == 1
    for call, g, message in ((delta_call(memory), grads(), b"saved is null"),
                             (delta_call(memory, saved=64), grads(dout=(0, 0, 0, 0)), b"dout is null"),
                             (delta_call(memory, saved=64), grads(dq=(65, 0, 0, 0)), b"dq is not aligned"),
                             (delta_call(memory, saved=64), grads(work=0), b"workspace is null"),
                             (delta_call(memory, saved=64), grads(work=24), b"workspace is not 16-byte aligned")):
        assert lib.mdn_delta_backward(call, g, None) == 1
        assert message in lib.mdn_last_error()


def test_sizes(pkg, memory):
    lib = pkg.lib()
    assert lib.mdn_delta_saved_bytes(delta_call(memory, steps=0)) == 0
    assert lib.mdn_delta_saved_bytes(delta_call(memory, steps=33)) > 0
    assert lib.mdn_delta_workspace_bytes(delta_call(memory)) > 0  # shared heads
    assert lib.mdn_delta_saved_bytes(delta_call(memory, dk=200)) == 0


def norm_call(memory, rows=4, dim=16, dtype=0, stream=0, act=0, eps=1e-6, x=64, branch=64, gate=64, h=64, y=64):
    return memory._NORM.pack(rows, dim, dtype, stream, act, eps, x, 16, branch, 16, gate, 16, 0, 0, 0, h, 16, y, 16)


@pytest.mark.parametrize("bad,message", [
    (dict(dim=0), b"1..8192"), (dict(dim=8193), b"1..8192"), (dict(dtype=3), b"dtypes"), (dict(stream=2), b"dtypes"),
    (dict(act=2), b"activation"), (dict(eps=float("nan")), b"eps"), (dict(eps=-1.0), b"eps"), (dict(x=0), b"x is null"),
    (dict(x=62), b"x is not aligned"), (dict(branch=0), b"gate without a branch"), (dict(h=0, y=0), b"no output")])
def test_block_norm_refusals(pkg, memory, bad, message):
    lib = pkg.lib()
    assert lib.mdn_block_norm_forward(norm_call(memory, **bad), None) == 1
    assert message in lib.mdn_last_error()


def test_block_norm_backward_refusals(pkg, memory):
    lib = pkg.lib()
    assert lib.mdn_block_norm_backward(norm_call(memory), None, None) == 1

    def grads(dx=64, work=64):
        return memory._NORM_GRADS.pack(64, 16, 64, 16, dx, 16, 64, 16, 64, 16, 0, 0, 0, work)
    for call, g, message in ((norm_call(memory), grads(work=0), b"workspace"),
                             (norm_call(memory), grads(work=8), b"workspace"),
                             (norm_call(memory, h=0), grads(), b"h is null"),
                             (norm_call(memory), grads(dx=2), b"dx is not aligned")):
        assert lib.mdn_block_norm_backward(call, g, None) == 1
        assert message in lib.mdn_last_error()


def test_tensors_on_the_cpu_are_refused(pkg):
    torch = importlib.import_module("torch")
    x = torch.zeros(2, 1, 1, 4)
    for call in (lambda: pkg.delta_rule(x, x, x, x[..., 0], x[..., 0]),
                 lambda: pkg.delta_step(x[0], x[0], x[0], x[0, ..., 0], x[0, ..., 0], torch.zeros(1, 1, 4, 4)),
                 lambda: pkg.block_norm(torch.zeros(2, 4)), lambda: pkg.block_norm_backward(torch.zeros(2, 4))):
        with pytest.raises(pkg.MdnError) as e:
            call()
        assert e.value.code == pkg.capi.ERR["INVALID"]
    assert not hasattr(pkg, "no_such_operator")
    assert ctypes.sizeof(ctypes.c_void_p) == 8

"""A simulator made in device memory that was used before starts as one in fresh memory does: unused obstacle slots
are zeros, not what an earlier tensor left there."""
import pytest

from conftest import load_oracle_module, load_package

pytestmark = pytest.mark.gpu


def test_reset_in_used_memory():
    import torch

    pkg, om = load_package(), load_oracle_module()
    dev = pkg.Device(0)
    cfg = pkg.layouts.default_config(n=300, family=12, speed=1.0, distance=3.0, seed=5)
    used = [torch.full((size,), 0xfd, dtype=torch.uint8, device="cuda") for size in (1 << 16, 1 << 18, 1 << 20) * 24]
    torch.cuda.synchronize()
    del used
    torch.cuda.empty_cache()
    sim = pkg.Sim(dev, cfg, 4)
    try:
        ora = om.OracleSim(pkg.layouts, cfg, 4, sim.raptor)
        for name in ("states", "runs", "worlds", "sensors"):
            assert sim.download(name).tobytes() == ora.buf(name).tobytes(), name
    finally:
        sim.close()
        dev.close()

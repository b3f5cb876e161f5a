"""block.add_rms_moe_fp8 on tensors of another device than the current one."""

from __future__ import annotations

import pytest
import torch

from oracle import moe_oracle as orc
from tests.helpers import BF16
from tests.test_gpu_block_fp8 import EPS, _fp8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 40])
def test_block_fp8_launches_on_its_tensors_device(pkg, dev, monkeypatch, T):
    """With some other device said to be the current one, every call into the library is made inside a
    switch to the tensors' device (one device is enough for that)."""
    import __graft_entry__

    mlp = _fp8(pkg, __graft_entry__._mlp_from_weights(orc.make_weights(256, 16, 96, 160, seed=3), dev))
    g = torch.Generator().manual_seed(T)
    x, h = (torch.randn(T, 256, generator=g).to(BF16).to(dev) for _ in range(2))
    w = torch.zeros(256, dtype=BF16, device=dev)
    want = pkg.block.add_rms_moe_fp8(x, h, w, EPS, mlp, 4)

    inside, calls, lib, switch = [], [], pkg._lib.load(), torch.cuda.device

    class Device(switch):
        def __enter__(self):
            inside.append(self.idx)
            return super().__enter__()

        def __exit__(self, *args):
            inside.pop()
            return super().__exit__(*args)

    class Call:
        """The library's function, noted when it is called."""

        def __init__(self, name):
            self.name = name

        def __call__(self, *args):
            calls.append((self.name, inside[-1:]))
            return getattr(lib, self.name)(*args)

    class Library:
        def __getattr__(self, name):
            return Call(name)

    monkeypatch.setattr(pkg._lib, "_lib", Library())
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: dev.index + 1)
    got = pkg.block.add_rms_moe_fp8(x, h, w, EPS, mlp, 4)
    monkeypatch.undo()
    launches = [c for c in calls if not c[0].endswith("_bytes")]
    assert len(launches) >= 7 and all(at == [dev.index] for _, at in launches), calls
    assert torch.equal(got, want)

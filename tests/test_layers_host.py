"""The host's part of the layer operators: loading, binding, and what is refused there (no GPU needed)."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

ROOT = Path(__file__).resolve().parent.parent


def test_the_package_imports_where_torch_has_no_gpu_backend(lib_built):
    """A torch build without one lacks the functions that ask for the current device and stream."""
    code = ("import torch\n"
            "for name in ('_cuda_getDevice', '_cuda_getCurrentRawStream'):\n"
            "    if hasattr(torch._C, name): delattr(torch._C, name)\n"
            "torch.cuda.device_count = lambda: 0\n"
            "from vmc_pde_amd import layers\n"
            "try:\n"
            "    layers.dense(torch.zeros(3, 4), torch.zeros(4, 5))\n"
            "except ValueError as refused:\n"
            "    assert 'device' in str(refused)\n"
            "else:\n"
            "    raise SystemExit(1)\n")
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, timeout=300)


def test_forward_mode_tangents_are_refused_on_the_host():
    from vmc_pde_amd import layers
    x, kernel, stats = torch.zeros(3, 4), torch.zeros(4, 5), torch.zeros(3)
    with forward_ad.dual_level(), torch.no_grad():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: layers.dense(dual(x), kernel), lambda: layers.dense(x, dual(kernel)), lambda: layers.layer_norm(dual(x)), lambda: layers.layer_norm(x, dual(x[0])),
                     lambda: layers.layer_norm_backward(x, x, dual(stats), stats), lambda: layers.global_norm([x, dual(x)]), lambda: layers.clip_by_global_norm(dual(x), 1.0),
                     lambda: layers.clip_by_global_norm(x, 1.0, out=dual(x.clone()))):
            with pytest.raises(ValueError, match="autograd"):
                call()


def test_every_lane_of_a_row_holds_the_same_sum():
    """The lane exchanges of layers.hpp's group_sum, replayed: partners exchange, so both add the same two numbers and addition's order is no matter."""
    import re

    import numpy as np
    text = (ROOT / "vmc_pde_amd" / "csrc" / "layers.hpp").read_text()
    body = text[text.index("A group_sum(A v)"):text.index("// elements of a 16-byte vector")]
    steps = [int(v, 16) for v in re.findall(r"dpp_move<(0x[0-9a-f]+)>", body)]
    assert len(steps) == 4

    def source(control, lane):
        row, i = lane & ~15, lane & 15
        if control < 0x100:                                    # quad_perm
            return row | (i & ~3) | (control >> 2 * (i & 3) & 3)
        if 0x121 <= control <= 0x12f:                          # row_ror
            return row | (i - (control & 15)) % 16
        return row | {0x140: 15 - i, 0x141: (i & 8) | 7 - (i & 7)}[control]
    v = np.random.default_rng(1).standard_normal((1000, 64)).astype(np.float32)
    for control in steps:
        v = v + v[:, [source(control, lane) for lane in range(64)]]
    rows = v.reshape(1000, 4, 16)
    assert (rows == rows[:, :, :1]).all()

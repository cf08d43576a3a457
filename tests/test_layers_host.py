"""The host's part of the layer operators: loading, binding, and what is refused there (no GPU needed)."""
import subprocess
import sys
import threading
import warnings
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture()
def nat(lib_built):
    from vmc_pde_amd import _native
    _native.lib()
    return _native


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


@pytest.mark.parametrize("case", ["another torch", "no library at all"])
def test_a_stale_native_module_is_left_out(nat, monkeypatch, tmp_path, case):
    """The Python code is the whole operator: a module that was built for another torch, or does not load, is left out with a warning."""
    monkeypatch.setattr(torch.cuda, "device_count", lambda: 1)
    monkeypatch.setattr(nat, "_calls", None)
    if case == "another torch":
        monkeypatch.setattr(torch, "__version__", "0.0.0")
    else:
        (tmp_path / "_lib").mkdir()
        (tmp_path / "_lib" / "vmcpde_layer_calls.so").write_bytes(b"not a library")
        monkeypatch.setattr(nat, "_HERE", tmp_path)
    with pytest.warns(RuntimeWarning, match="vmcpde_layer_calls"):
        assert nat.layer_calls() is None
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert nat.layer_calls() is None           # said once


def test_the_native_module_loads(nat, monkeypatch):
    monkeypatch.setattr(torch.cuda, "device_count", lambda: 1)
    monkeypatch.setattr(nat, "_calls", None)
    assert nat.layer_calls() is not None


def test_the_native_module_is_built_again_for_another_torch(monkeypatch, tmp_path):
    from vmc_pde_amd import build
    commands = []
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **_: commands.append(cmd))
    monkeypatch.setattr(build, "_stale", lambda target, deps: False)
    monkeypatch.setattr(build, "CALLS_LIB", tmp_path / "vmcpde_layer_calls.so")
    for version, built in (("0.0.0", 1), ("0.0.0", 1), ("0.0.1", 2), ("0.0.1", 2)):
        monkeypatch.setattr(torch, "__version__", version)
        build.build_calls()
        assert len(commands) == built


def test_entry_points_bound_by_two_threads(nat, monkeypatch):
    """A thread that calls while another one binds the entry points finds all of them or binds them itself, never some."""
    from vmc_pde_amd import layers
    real, first, go_on = nat.lib(), threading.Event(), threading.Event()
    binder = threading.Thread(target=lambda: layers._entries())

    class Slow:
        def __getitem__(self, name):
            if threading.current_thread() is binder:
                if first.is_set():
                    go_on.wait(30)
                first.set()
            return real[name]
    monkeypatch.setattr(layers, "_entry", {})
    monkeypatch.setattr(nat, "lib", Slow)
    binder.start()
    assert first.wait(30)
    try:
        assert layers._workspace("vmcpde_global_norm_workspace_bytes", "cpu", None, 0) == (None, 0)       # (no tensors: nothing is read)
    finally:
        go_on.set()
        binder.join()
    assert len(layers._entry) == 8


@pytest.mark.parametrize("dtype, rows, n_in, n_out, backward, fits", [
    (1, 1 << 29, 8, 128, 0, False), (1, (1 << 29) - 64, 8, 128, 0, True), (0, 1 << 29, 100, 8, 1, False), (0, 1 << 29, 8, 64, 0, True), (3, 1 << 29, 8, 128, 0, True),
    (3, (1 << 30) - 1, 8, 64, 0, False), (2, (1 << 30) - 1, 8, 32, 0, True)])
def test_dense_refuses_more_tiles_than_a_launch_takes(nat, dtype, rows, n_in, n_out, backward, fits):
    """2^24 tiles of 256 lanes: on the host, before the first of the call's launches."""
    here = 4096      # stands for an address
    a = nat.DenseArgs(dtype=dtype, activation=0, kernel_t=0, rows=rows, n_in=n_in, n_out=n_out, x=here, ldx=n_in, kernel=here, ldk=n_out, scale=1.0, y=here, ldy=n_out,
                      dy=here, ldd=n_out, dx=here, dkernel=None, dbias=None)
    need = nat.lib().vmcpde_dense_workspace_bytes(a, backward)
    assert (need >= 0) == fits
    if not fits:
        run = nat.lib().vmcpde_dense_backward if backward else nat.lib().vmcpde_dense
        assert run(a, here, 1 << 60, None) == -1 and b"tiles" in nat.lib().vmcpde_last_error()


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

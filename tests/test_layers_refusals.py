"""The layer operators refuse what they cannot do, on the host and before anything is launched (no GPU needed: the pointers are never followed)."""
import ctypes as C

import numpy as np
import pytest
import torch

F64, F32, F16, BF16 = 0, 1, 2, 3
HERE = 4096   # stands for an address


@pytest.fixture(scope="module")
def nat(lib_built):
    from vmc_pde_amd import _native
    _native.lib()
    return _native


def dense_args(nat, **changed):
    v = dict(dtype=F32, activation=1, kernel_t=0, rows=4, n_in=5, n_out=6, x=HERE, ldx=5, kernel=HERE, ldk=6, bias=None, residual=None, ldr=0, scale=1.0, y=HERE,
             ldy=6, slope=None, dy=HERE, ldd=6, dx=HERE, dkernel=HERE, dbias=HERE)
    v.update(changed)
    return nat.DenseArgs(**v)


def norm_args(nat, **changed):
    v = dict(dtype=BF16, weight_dtype=F32, rows=4, cols=5, x=HERE, ldx=5, weight=HERE, bias=HERE, eps=1e-6, y=HERE, ldy=5, mean=HERE, rstd=HERE, dy=HERE, ldd=5, dx=HERE,
             dweight=HERE, dbias=HERE)
    v.update(changed)
    return nat.NormArgs(**v)


@pytest.mark.parametrize("changed, backward", [
    (dict(dtype=4), 0), (dict(dtype=-1), 1), (dict(activation=9), 0), (dict(rows=-1), 0), (dict(n_in=0), 0), (dict(n_out=0), 1), (dict(n_in=1 << 30), 0),
    (dict(x=None), 0), (dict(ldx=4), 0), (dict(kernel=None), 0), (dict(ldk=5), 0), (dict(kernel_t=1, ldk=4), 0), (dict(y=None), 0), (dict(ldy=5), 0),
    (dict(residual=HERE, ldr=5), 0), (dict(scale=float("nan")), 0), (dict(dy=None), 1), (dict(ldd=5), 1), (dict(x=None), 1), (dict(kernel=None), 1)])
def test_dense_refuses(nat, changed, backward):
    a = dense_args(nat, **changed)
    L = nat.lib()
    assert L.vmcpde_dense_workspace_bytes(a, backward) == -1
    rc = (L.vmcpde_dense_backward if backward else L.vmcpde_dense)(a, HERE, 1 << 40, None)
    assert rc == -1 and b"dense" in L.vmcpde_last_error()


def test_dense_refuses_a_short_workspace(nat):
    L = nat.lib()
    a = dense_args(nat, rows=4, n_in=100000, ldx=100000)
    need = L.vmcpde_dense_workspace_bytes(a, 0)
    assert need > 0
    assert L.vmcpde_dense(a, HERE, need - 1, None) == -1 and b"workspace" in L.vmcpde_last_error()
    assert L.vmcpde_dense(a, None, need, None) == -1
    assert L.vmcpde_dense(a, HERE + 8, need, None) == -1 and b"aligned" in L.vmcpde_last_error()
    assert L.vmcpde_dense_workspace_bytes(a, 1) == 0   # dz is dy itself, and four rows' column sums take no partials
    a = dense_args(nat, rows=4, n_in=100000, ldx=100000, slope=HERE)
    need = L.vmcpde_dense_workspace_bytes(a, 1)
    assert need > 0 and L.vmcpde_dense_backward(a, HERE, need - 1, None) == -1
    assert L.vmcpde_dense(None, None, 0, None) == -1 and L.vmcpde_dense_workspace_bytes(None, 0) == -1


def test_dense_without_rows_launches_nothing(nat):
    L = nat.lib()
    for dtype in (F64, F32, F16, BF16):
        assert L.vmcpde_dense_workspace_bytes(dense_args(nat, rows=0, x=None, y=None, dtype=dtype), 0) == 0
        assert L.vmcpde_dense_workspace_bytes(dense_args(nat, rows=0, x=None, y=None, dy=None, dtype=dtype), 1) >= 0
    assert L.vmcpde_dense(dense_args(nat, rows=0, x=None, y=None), None, 0, None) == 0
    assert L.vmcpde_layer_norm(norm_args(nat, rows=0, x=None, y=None), None) == 0


@pytest.mark.parametrize("changed", [dict(dtype=7), dict(weight_dtype=F64), dict(dtype=F32, weight_dtype=BF16), dict(dtype=F64, weight_dtype=F32), dict(weight_dtype=F16),
                                     dict(rows=-1), dict(rows=1 << 31), dict(cols=0), dict(x=None), dict(ldx=4), dict(cols=1 << 27, ldx=1 << 27),
                                     dict(rows=1 << 22, cols=16385, ldx=16385), dict(rows=1 << 22, dtype=F64, weight_dtype=F64, cols=4097, ldx=4097)])
def test_layer_norm_refuses(nat, changed):
    L, a = nat.lib(), norm_args(nat, **changed)
    assert L.vmcpde_layer_norm(a, None) == -1 and b"layer norm" in L.vmcpde_last_error()
    assert L.vmcpde_layer_norm_backward_workspace_bytes(a) == -1
    assert L.vmcpde_layer_norm_backward(a, HERE, 1 << 40, None) == -1


def test_layer_norm_refuses_by_direction(nat):
    L = nat.lib()
    for changed in (dict(eps=-1.0), dict(eps=float("nan")), dict(mean=None), dict(rstd=None), dict(y=None), dict(ldy=4)):
        assert L.vmcpde_layer_norm(norm_args(nat, **changed), None) == -1, changed
    for changed in (dict(dy=None), dict(ldd=4), dict(mean=None), dict(rstd=None)):
        assert L.vmcpde_layer_norm_backward(norm_args(nat, **changed), HERE, 1 << 40, None) == -1, changed
    a = norm_args(nat)
    need = L.vmcpde_layer_norm_backward_workspace_bytes(a)
    assert need > 0 and L.vmcpde_layer_norm_backward(a, HERE, need - 1, None) == -1 and b"workspace" in L.vmcpde_last_error()


def table(*rows):
    t = np.array(rows, dtype=np.int64)
    return t, t.ctypes.data, len(rows)


@pytest.mark.parametrize("rows, clip, max_norm", [
    ([(HERE, HERE, 10, 4)], 0, 0.0), ([(HERE, HERE, -1, F32)], 0, 0.0), ([(0, 0, 3, F32)], 0, 0.0), ([(HERE, 0, 3, F32)], 1, 1.0), ([(HERE + 2, HERE, 3, F32)], 0, 0.0),
    ([(HERE, HERE + 1, 3, F16)], 1, 1.0), ([(HERE, HERE, 3, F32)], 1, -1.0), ([(HERE, HERE, 3, F32)], 1, float("nan"))])
def test_global_norm_refuses(nat, rows, clip, max_norm):
    L = nat.lib()
    keep, address, count = table(*rows)
    assert L.vmcpde_global_norm(address, count, clip, max_norm, HERE, HERE, 1 << 40, None) == -1 and b"norm" in L.vmcpde_last_error()


@pytest.mark.parametrize("rows", [
    [(HERE, HERE, 10, F32), (HERE, HERE, 10, F32)],                                   # the same tensor twice, in place
    [(HERE, HERE, 10, F32), (HERE + 36, HERE + 36, 10, F32)],                         # the last element of one is the first of the other
    [(HERE, 2 * HERE, 10, F32), (HERE + 400, 2 * HERE + 4, 10, F32)],                 # two outputs
    [(HERE, HERE + 4, 10, F32)],                                                      # an output into its own input, moved
    [(HERE, 2 * HERE, 10, F32), (2 * HERE + 8, 3 * HERE, 10, F64)]])                  # an output into another input
def test_clipping_refuses_what_overlaps(nat, rows):
    L = nat.lib()
    keep, address, count = table(*rows)
    assert L.vmcpde_global_norm(address, count, 1, 1.0, HERE * 9, HERE * 10, 1 << 40, None) == -1 and b"overlaps" in L.vmcpde_last_error()


def test_global_norm_refuses_a_short_workspace(nat):
    L = nat.lib()
    keep, address, count = table((HERE, HERE, 1 << 20, F32))
    need = L.vmcpde_global_norm_workspace_bytes(address, count)
    assert need > 0 and L.vmcpde_global_norm(address, count, 0, 0.0, HERE, HERE, 64, None) == -1 and b"workspace" in L.vmcpde_last_error()
    assert L.vmcpde_global_norm(address, count, 0, 0.0, None, HERE, need, None) == -1
    assert L.vmcpde_global_norm(None, 1, 0, 0.0, HERE, HERE, need, None) == -1


def test_python_side_refuses_types_gradients_and_host_tensors(lib_built):
    from vmc_pde_amd import layers
    x, k = torch.zeros(3, 4), torch.zeros(4, 5)
    for call in (lambda: layers.dense(x, k), lambda: layers.layer_norm(x), lambda: layers.global_norm(x), lambda: layers.clip_by_global_norm([x], 1.0)):
        with pytest.raises(ValueError, match="device"):
            call()
    for call in (lambda: layers.dense(x, k.double()), lambda: layers.dense(x.int(), k.int()), lambda: layers.dense(x, None or [1]), lambda: layers.dense("x", k),
                 lambda: layers.layer_norm(x.int()), lambda: layers.global_norm("x"), lambda: layers.global_norm([x, 3]),
                 lambda: layers.clip_by_global_norm(x, 1.0, out=3)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: layers.dense(x.clone().requires_grad_(), k), lambda: layers.dense(x, k.clone().requires_grad_()),
                 lambda: layers.layer_norm(x.clone().requires_grad_())):
        with pytest.raises(ValueError, match="autograd"):
            call()
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            layers.clip_by_global_norm(x, bad)
    with pytest.raises(ValueError, match="no tensors"):
        layers.global_norm([])

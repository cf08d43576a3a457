"""Layer operators of a fit: the dense layer with its epilogue, layer norm, and the global gradient norm.

The conditioners of the coupling flow are chains of dense layers (reference: vmc_fluids/net.py:53-61) that `csrc/flow.hip` evaluates whole,
per sample, with their weights in LDS.  These are the same layers as operators over a batch, of any width, in fp64, fp32, fp16 and bf16, with
what a training step of a wide network needs around them.  Like the rest of this package they are explicit: every operator has its gradient as
a function of its own, and takes no part in torch's automatic differentiation (tensors that require it are refused while it is recording).

All run on the current HIP stream, allocate through torch, never synchronise with the host, and can be captured into a graph.  Sums, statistics
and epilogues are held in fp32 for fp32 and 16-bit elements, in fp64 for fp64.  None uses atomics: the same call gives the same bits.
"""
from __future__ import annotations

import contextlib

import numpy as np
import torch

from . import _native as nat

DTYPE = {torch.float64: 0, torch.float32: 1, torch.float16: 2, torch.bfloat16: 3}
ACTIVATION = {"none": 0, "tanh": 1, "gelu": 2, "silu": 3}
_HALF = (torch.float16, torch.bfloat16)
SLOPE = {torch.float64: torch.float64, torch.float32: torch.float32, torch.float16: torch.float32, torch.bfloat16: torch.float16}


def _on(device):
    return contextlib.nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _check(first, **others):
    """Element type and device of `first`, which every other tensor must share."""
    if not isinstance(first, torch.Tensor):
        raise TypeError(f"a tensor is needed, not {type(first).__name__}")
    if first.dtype not in DTYPE:
        raise TypeError(f"element type {first.dtype}: fp64, fp32, fp16 and bf16 are supported")
    recording = torch.is_grad_enabled()
    if recording and first.requires_grad:
        raise ValueError("the layer operators are no autograd functions: call them under torch.no_grad() and use their *_backward")
    for name, t in others.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: a tensor is needed, not {type(t).__name__}")
        if t.dtype != first.dtype:
            raise TypeError(f"{name} has type {t.dtype} beside {first.dtype}")
        if t.device != first.device:
            raise ValueError(f"{name} is on {t.device}, not on {first.device}")
        if recording and t.requires_grad:
            raise ValueError("the layer operators are no autograd functions: call them under torch.no_grad() and use their *_backward")
    if not first.is_cuda:
        raise ValueError("the layer operators run on device (HBM) tensors only")


def _rows(t, cols, name):
    """(tensor, row pitch) of t as a matrix of `cols` columns whose rows' elements lie behind each other; copied only where no such view exists."""
    if t.dim() == 0 or t.shape[-1] != cols:
        raise ValueError(f"{name} has shape {tuple(t.shape)}: its last axis should have {cols}")
    if t.is_contiguous():
        return t, cols
    m = t.reshape(-1, cols)
    if cols > 1 and m.stride(1) != 1 or m.shape[0] > 1 and m.stride(0) < cols:
        return m.contiguous(), cols
    return m, m.stride(0) if m.shape[0] > 1 else cols


def _same_shape(t, shape, name):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}: {tuple(shape)} is needed")


def _vector(t, n, name):
    if t is None:
        return None
    _same_shape(t, (n,), name)
    return t.contiguous()


def _address(t):
    return None if t is None else t.data_ptr()


def _workspace(nbytes, device):
    if nbytes < 0:
        nat.check(-1, "layers")
    return (None, 0) if nbytes == 0 else (torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes)


def _kernel_layout(kernel):
    """(tensor, row pitch, whether it is stored (n_out, n_in)) of a kernel of shape (n_in, n_out)."""
    if kernel.dim() != 2 or 0 in kernel.shape:
        raise ValueError(f"kernel has shape {tuple(kernel.shape)}: (n_in, n_out), neither of them 0, is needed")
    n_in, n_out = kernel.shape
    s0, s1 = kernel.stride()
    if (s1 == 1 or n_out == 1) and (s0 >= n_out or n_in == 1):
        return kernel, max(s0, n_out), 0
    if (s0 == 1 or n_in == 1) and (s1 >= n_in or n_out == 1):
        return kernel, max(s1, n_in), 1
    return kernel.contiguous(), n_out, 0


def dense(x, kernel, bias=None, *, activation="none", scale=1.0, residual=None, want_slope=False):
    """y = scale * act(x @ kernel + bias) + residual, in one pass over x and the kernel.

    x (..., n_in); kernel (n_in, n_out), the layout of the flat parameter vector's leaves, or a transposed view of an (n_out, n_in) one; bias
    (n_out,); residual of y's shape.  activation: "none", "tanh", "gelu" (z Phi(z)), "silu".  `scale` is the output factor of the reference's
    conditioners (net.py:50, 61: 10 * tanh).  Widths and row pitches are below 2^22 (2^21 in fp64).  With `want_slope` returns (y, slope): act'(z), which `dense_backward` takes (None for "none");
    of the type SLOPE[x.dtype] (fp16 for bf16, fp32 for fp16, else the element type)."""
    _check(x, kernel=kernel, bias=bias, residual=residual)
    if activation not in ACTIVATION:
        raise ValueError(f"activation {activation!r}: one of {sorted(ACTIVATION)} is needed")
    kernel, ldk, kernel_t = _kernel_layout(kernel)
    n_in, n_out = kernel.shape
    shape = (*x.shape[:-1], n_out)
    x, ldx = _rows(x, n_in, "x")
    bias = _vector(bias, n_out, "bias")
    ldr = 0
    if residual is not None:
        _same_shape(residual, shape, "residual")
        residual, ldr = _rows(residual, n_out, "residual")
    device = x.device
    with _on(device):
        y = torch.empty(shape, dtype=x.dtype, device=device)
        slope = None
        if want_slope and activation != "none":
            slope = torch.empty(shape, dtype=SLOPE[x.dtype], device=device)
        a = nat.DenseArgs(DTYPE[x.dtype], ACTIVATION[activation], kernel_t, 0, x.numel() // n_in, n_in, n_out, x.data_ptr(), ldx, kernel.data_ptr(), ldk,
                          _address(bias), _address(residual), ldr, float(scale), y.data_ptr(), n_out, _address(slope))
        ws, nbytes = _workspace(nat.lib().vmcpde_dense_workspace_bytes(a, 0), device)
        nat.call("vmcpde_dense", a, _address(ws), nbytes, nat.stream())
    return (y, slope) if want_slope else y


def dense_backward(dy, x, kernel, slope=None, *, scale=1.0, want_x=True, want_kernel=True, want_bias=True):
    """(dx, dkernel, dbias) of `dense` for the gradient dy of y, None where not wanted: with dz = scale * slope * dy, dx = dz @ kernel^T,
    dkernel = x^T @ dz (n_in, n_out), dbias = the sum of dz over the rows.  `slope` and `scale` as the forward call had them; the residual's
    gradient is dy itself.  dz is rounded to the element type, in which the matrix pipe takes it."""
    _check(dy, x=x, kernel=kernel)
    kernel, ldk, kernel_t = _kernel_layout(kernel)
    n_in, n_out = kernel.shape
    _same_shape(dy, (*x.shape[:-1], n_out), "dy")
    x_shape = x.shape
    x, ldx = _rows(x, n_in, "x")
    dy, ldd = _rows(dy, n_out, "dy")
    if slope is not None:
        want = SLOPE[x.dtype]
        if slope.dtype != want or slope.device != x.device:
            raise TypeError(f"slope is {slope.dtype} on {slope.device}: {want} on {x.device} is needed, as dense(..., want_slope=True) returns it")
        _same_shape(slope, (*x_shape[:-1], n_out), "slope")
        slope = slope.contiguous()
    device = x.device
    with _on(device):
        dx = torch.empty(x_shape, dtype=x.dtype, device=device) if want_x else None
        dkernel = torch.empty((n_in, n_out), dtype=x.dtype, device=device) if want_kernel else None
        dbias = torch.empty(n_out, dtype=x.dtype, device=device) if want_bias else None
        a = nat.DenseArgs(DTYPE[x.dtype], 0, kernel_t, 0, x.numel() // n_in, n_in, n_out, x.data_ptr(), ldx, kernel.data_ptr(), ldk, None, None, 0,
                          float(scale), None, 0, _address(slope), dy.data_ptr(), ldd, _address(dx), _address(dkernel), _address(dbias))
        ws, nbytes = _workspace(nat.lib().vmcpde_dense_workspace_bytes(a, 1), device)
        nat.call("vmcpde_dense_backward", a, _address(ws), nbytes, nat.stream())
    return dx, dkernel, dbias


def _norm_weights(x, weight, bias):
    """The weights' element type: x's, or fp32 beside 16-bit elements."""
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dtype != x.dtype and not (x.dtype in _HALF and t.dtype == torch.float32):
            raise TypeError(f"{name} has type {t.dtype} beside {x.dtype}: the same, or fp32 beside 16-bit elements")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, not on {x.device}")
        if torch.is_grad_enabled() and t.requires_grad:
            raise ValueError("the layer operators are no autograd functions: call them under torch.no_grad() and use their *_backward")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight has type {weight.dtype} and bias {bias.dtype}")
    first = weight if weight is not None else bias
    return x.dtype if first is None else first.dtype


def layer_norm(x, weight=None, bias=None, *, eps=1e-6, want_stats=False):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last axis (the variance is the mean of the squared deviations).

    weight, bias (cols,): x's element type, or fp32 beside 16-bit elements.  With `want_stats` returns (y, mean, rstd), which
    `layer_norm_backward` takes: of the leading shape, fp32 (fp64 for fp64)."""
    _check(x)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x has shape {tuple(x.shape)}: a last axis of one or more is needed")
    if not eps >= 0:
        raise ValueError(f"eps = {eps}")
    weights = _norm_weights(x, weight, bias)
    shape, cols = x.shape, x.shape[-1]
    weight, bias = _vector(weight, cols, "weight"), _vector(bias, cols, "bias")
    x, ldx = _rows(x, cols, "x")
    device = x.device
    with _on(device):
        y = torch.empty(shape, dtype=x.dtype, device=device)
        mean = rstd = None
        if want_stats:
            wide = torch.float64 if x.dtype == torch.float64 else torch.float32
            mean, rstd = torch.empty(shape[:-1], dtype=wide, device=device), torch.empty(shape[:-1], dtype=wide, device=device)
        a = nat.NormArgs(DTYPE[x.dtype], DTYPE[weights], x.numel() // cols, cols, x.data_ptr(), ldx, _address(weight), _address(bias), float(eps),
                         y.data_ptr(), cols, _address(mean), _address(rstd))
        nat.call("vmcpde_layer_norm", a, nat.stream())
    return (y, mean, rstd) if want_stats else y


def layer_norm_backward(dy, x, mean, rstd, weight=None, *, want_x=True, want_weight=True, want_bias=True, weight_dtype=None):
    """(dx, dweight, dbias) of `layer_norm` for the gradient dy of y, None where not wanted; mean, rstd from `layer_norm(..., want_stats=True)`.
    dweight and dbias have the weight's type (without a weight `weight_dtype`, else x's)."""
    _check(dy, x=x)
    weights = _norm_weights(x, weight, None)
    if weight is None and weight_dtype is not None:
        if weight_dtype != x.dtype and not (x.dtype in _HALF and weight_dtype == torch.float32):
            raise TypeError(f"weight_dtype {weight_dtype} beside {x.dtype}: the same, or fp32 beside 16-bit elements")
        weights = weight_dtype
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x has shape {tuple(x.shape)}: a last axis of one or more is needed")
    shape, cols = x.shape, x.shape[-1]
    _same_shape(dy, shape, "dy")
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    for name, t in (("mean", mean), ("rstd", rstd)):
        _same_shape(t, shape[:-1], name)
        if t.dtype != wide or t.device != x.device:
            raise TypeError(f"{name} is {t.dtype} on {t.device}: {wide} on {x.device} is needed")
    weight = _vector(weight, cols, "weight")
    x, ldx = _rows(x, cols, "x")
    dy, ldd = _rows(dy, cols, "dy")
    mean, rstd = mean.contiguous(), rstd.contiguous()
    device = x.device
    with _on(device):
        dx = torch.empty(shape, dtype=x.dtype, device=device) if want_x else None
        dweight = torch.empty(cols, dtype=weights, device=device) if want_weight else None
        dbias = torch.empty(cols, dtype=weights, device=device) if want_bias else None
        a = nat.NormArgs(DTYPE[x.dtype], DTYPE[weights], x.numel() // cols, cols, x.data_ptr(), ldx, _address(weight), None, 0.0, None, 0, mean.data_ptr(),
                         rstd.data_ptr(), dy.data_ptr(), ldd, _address(dx), _address(dweight), _address(dbias))
        ws, nbytes = (None, 0)
        if want_weight or want_bias:
            ws, nbytes = _workspace(nat.lib().vmcpde_layer_norm_backward_workspace_bytes(a), device)
        nat.call("vmcpde_layer_norm_backward", a, _address(ws), nbytes, nat.stream())
    return dx, dweight, dbias


def _leaves(tree, out):
    if isinstance(tree, torch.Tensor):
        out.append(tree)
    elif isinstance(tree, dict):
        for key in sorted(tree):               # the parameter trees' order, and the same one for a dict and the dict it is written to
            _leaves(tree[key], out)
    elif isinstance(tree, (list, tuple)):
        for v in tree:
            _leaves(v, out)
    else:
        raise TypeError(f"a tensor, or a list or (nested) dict of tensors is needed, not {type(tree).__name__}")
    return out


def _fills_memory(t):
    """Whether t's elements, in whatever order, lie behind each other."""
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _global_norm(tensors, max_norm, out):
    leaves = _leaves(tensors, [])
    if not leaves:
        raise ValueError("no tensors")
    device = leaves[0].device
    if not leaves[0].is_cuda:
        raise ValueError("the layer operators run on device (HBM) tensors only")
    for t in leaves:
        if t.device != device:
            raise ValueError(f"tensors on {device} and {t.device}")
        if t.dtype not in DTYPE:
            raise TypeError(f"element type {t.dtype}: fp64, fp32, fp16 and bf16 are supported")
        if not (t.is_contiguous() or t.numel() == 0 or _fills_memory(t)):
            raise ValueError(f"a tensor of shape {tuple(t.shape)} and strides {t.stride()} does not fill its memory: pass a contiguous one")
    targets = leaves
    if out is not None:
        targets = _leaves(out, [])
        if len(targets) != len(leaves):
            raise ValueError(f"{len(leaves)} tensors and {len(targets)} to write them to")
        for t, o in zip(leaves, targets):
            if o.shape != t.shape or o.dtype != t.dtype or o.device != device or o.stride() != t.stride():
                raise ValueError(f"out: shape {tuple(o.shape)}, strides {o.stride()}, {o.dtype} on {o.device} beside {tuple(t.shape)}, {t.stride()}, {t.dtype} on {device}")
    if max_norm is not None and torch.is_grad_enabled() and any(t.requires_grad for t in targets):
        raise ValueError("clipping writes into tensors that automatic differentiation records: call it under torch.no_grad()")
    table = np.array([(t.data_ptr(), o.data_ptr(), t.numel(), DTYPE[t.dtype]) for t, o in zip(leaves, targets)], dtype=np.int64)   # vmcpde_tensor
    address, count = table.ctypes.data, len(leaves)
    with _on(device):
        norm = torch.empty((), dtype=torch.float64, device=device)
        ws, nbytes = _workspace(nat.lib().vmcpde_global_norm_workspace_bytes(address, count), device)
        nat.call("vmcpde_global_norm", address, count, 0 if max_norm is None else 1, 0.0 if max_norm is None else max_norm, norm.data_ptr(), _address(ws), nbytes,
                 nat.stream())
    return norm


def global_norm(tensors):
    """2-norm over all elements of a tensor, or of a list or (nested) dict of them (`VarState.params`), as an fp64 scalar on the device.
    Element types may differ.  Squares are summed in fp64; no finite norm overflows or vanishes on its way."""
    return _global_norm(tensors, None, None)


def clip_by_global_norm(tensors, max_norm, out=None):
    """Multiplies every tensor by max_norm / norm where their `global_norm` exceeds max_norm, in place or into `out` (tensors of the same shapes,
    strides and types).  Returns the norm before clipping; nothing is read back to the host.  A NaN norm leaves the elements as they are, an
    infinite one makes finite elements zero.  Tensors that overlap each other are refused: they would be scaled twice."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm = {max_norm}")
    if out is not None and not isinstance(out, (torch.Tensor, list, tuple, dict)):
        raise TypeError("out: a tensor, or a list or (nested) dict of tensors")
    return _global_norm(tensors, max_norm, out)

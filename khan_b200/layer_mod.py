"""Operators of normalised layers of the atomic networks, on torch tensors: layer norm with its gradients, and activations
whose input is kept in 8 bits for the backward pass.

Rows are atoms.  With ``acs`` (host counts of the four elements, as in :mod:`khan_b200.ani_mod`) they are in element order,
``gain`` and ``bias`` are lists of four vectors, one per element, and every sum over rows has a leading dimension of four
(zeros for an element without atoms); without ``acs`` all rows share one ``gain`` and ``bias`` and the sums have no such
dimension.  One launch covers all elements (two where sums over many rows are formed), on torch's current stream.  Results
are bit-reproducible, nothing is kept from one call for the next, and a call can be captured into a CUDA graph.

The functions are not recorded by autograd, but for :func:`layer_norm_autograd`; networks with checkpoints are differentiated
by :class:`khan_b200.model.nn.MoleculeNN`.  A backward pass is captured while no eager graph of the same parameters is alive:
torch ties a parameter's gradient to the stream of the graph that it was first part of, and gives up in the capture.

Rows may be strided (a slice of a wider tensor); other layouts are copied.  Widths go from 1 to 4096.  Layer norm takes
float32 and float64, checkpoints float32.  There is no CPU path.
"""
from __future__ import annotations

import numpy as np
import torch

from . import _lib
from .ani_mod import host_counts
from .model import activations

MAX_WIDTH = 4096
CHECKPOINT_BLOCK = 128      # columns that share a base and a step


_ACTIVATION_IDS = {**activations.KERNEL_ID, **{name: activations.KERNEL_ID[activations.get_fn_by_name(name)]
                                               for name in activations.get_all_fn_names()}}


def _activation_id(activation) -> int:
    """The kernels' number of an activation function of the networks, or of its name."""
    try:
        return _ACTIVATION_IDS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"no kernel for the activation {activation!r}: one of {activations.get_all_fn_names()}") from None


def _rows(t, name: str, like=None):
    """``t`` as rows that the kernels take: two dimensions, CUDA, values of a row next to each other."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError(f"{name} must be a tensor [rows, width]")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (khan_b200 has no CPU path)")
    if like is not None and t.dtype != like.dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {like.dtype}")
    if not 1 <= t.shape[1] <= MAX_WIDTH:
        raise ValueError(f"{name} has {t.shape[1]} columns: 1 to {MAX_WIDTH} are supported")
    regular = (t.shape[1] == 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1])
    return t if regular else t.contiguous()


def _counts(acs, n: int):
    if acs is None:
        return None
    acs = host_counts(acs)
    if (acs < 0).any() or int(acs.sum(dtype=np.int64)) != n:
        raise ValueError(f"acs counts {acs.tolist()} atoms of four elements, there are {n} rows")
    return acs


def _vectors(v, name: str, acs, x):
    """One vector per element (a list of four with ``acs``), of x's type and width, contiguous."""
    if acs is not None and (not isinstance(v, (list, tuple)) or len(v) != 4):
        raise ValueError(f"{name}: rows grouped by element take a list of four vectors")
    if acs is None and not isinstance(v, torch.Tensor):
        raise ValueError(f"{name} must be a tensor (a list of four goes with acs)")
    out = []
    for t in v if acs is not None else [v]:
        if not isinstance(t, torch.Tensor) or t.numel() != x.shape[1]:
            raise ValueError(f"{name} must hold {x.shape[1]} values, one per column")
        if t.dtype != x.dtype:
            raise TypeError(f"{name} is {t.dtype}, expected {x.dtype}")
        out.append(t.detach().reshape(-1).contiguous())
    _lib.same_device(x.device, *out, where=name)
    return out if acs is not None else out[0]


def _per_row(t, name: str, x):
    if not isinstance(t, torch.Tensor) or t.numel() != x.shape[0] or t.dtype != x.dtype:
        raise ValueError(f"{name} must hold {x.shape[0]} values of {x.dtype}, one per row")
    _lib.same_device(x.device, t, where=name)
    return t.reshape(-1).contiguous()


def _done(where: str, out):
    if type(out) is int:
        _lib.check(out, where)
    if out is None:
        raise ValueError(f"{where}: the arguments do not fit each other")
    return out


def layer_norm(x, gain, bias, acs=None, eps: float = 1e-5):
    """``y = gain * (x - mean) * rstd + bias`` row by row; returns ``(y, mean, rstd)`` with
    ``rstd = 1 / sqrt(variance + eps)``, the variance divided by the width."""
    out = _lib.torch_ops().layer_norm(x, gain, bias, acs, eps)
    if out is None:
        x = _rows(x, "x")
        if x.dtype not in (torch.float32, torch.float64):
            raise TypeError(f"layer_norm supports float32 and float64, got {x.dtype}")
        acs = _counts(acs, x.shape[0])
        out = _lib.torch_ops().layer_norm(x, _vectors(gain, "gain", acs, x), _vectors(bias, "bias", acs, x), acs, eps)
    return _done("ani_layer_norm", out)


def layer_norm_grad(grad_y, x, gain, mean, rstd, acs=None):
    """Gradients of :func:`layer_norm`: ``(grad_x, grad_gain, grad_bias)`` from the gradient of y, x and what the forward
    pass returned."""
    out = _lib.torch_ops().layer_norm_grad(grad_y, x, gain, mean, rstd, acs)
    if out is None:
        x = _rows(x, "x")
        if x.dtype not in (torch.float32, torch.float64):
            raise TypeError(f"layer_norm_grad supports float32 and float64, got {x.dtype}")
        grad_y = _rows(grad_y, "grad_y", x)
        if grad_y.shape != x.shape:
            raise ValueError(f"grad_y is {tuple(grad_y.shape)}, x {tuple(x.shape)}")
        _lib.same_device(x.device, grad_y, where="layer_norm_grad")
        acs = _counts(acs, x.shape[0])
        out = _lib.torch_ops().layer_norm_grad(grad_y, x, _vectors(gain, "gain", acs, x), _per_row(mean, "mean", x),
                                               _per_row(rstd, "rstd", x), acs)
    return _done("ani_layer_norm_grad", out)


class ActivationCheckpoint:
    """What :func:`checkpoint_activation` keeps of the input of an activation: ``codes`` (uint8, a row of
    ``ceil(width / 16) * 16`` bytes per atom), ``blocks`` (float32 ``[n, ceil(width / 128), 2]``: base and step of every 128
    columns; a code stands for ``base + code * step``), and with a norm ``mean`` and ``rstd`` of the rows.  One made by
    :func:`checkpoint_activation` has them in one buffer, one made from its parts refers to those."""

    __slots__ = ("_parts", "width", "activation", "_rows", "_normed")

    def __init__(self, codes, blocks, width: int, activation, mean=None, rstd=None):
        self._parts, self.width, self._rows = (codes, blocks, mean, rstd), int(width), codes.shape[0]
        self._normed = mean is not None
        self.activation = _activation_id(activation)

    @classmethod
    def _of_buffer(cls, buffer, rows, width, activation, normed):      # activation: its number
        kept = cls.__new__(cls)
        kept._parts, kept._rows, kept.width, kept.activation, kept._normed = (buffer, None, None, None), rows, width, activation, normed
        return kept

    def _part(self, which: int):
        if self._parts[1] is not None:
            return self._parts[which]
        n, row, blocks = self._rows, -(-self.width // 16) * 16, -(-self.width // CHECKPOINT_BLOCK)
        if which >= 2 and not self._normed:
            return None
        start = (0, n * row, n * (row + 8 * blocks), n * (row + 8 * blocks + 4))[which]
        shape = ((n, row), (n, blocks, 2), (n,), (n,))[which]
        raw = self._parts[0][start:start + int(np.prod(shape, dtype=np.int64)) * (4 if which else 1)]
        return (raw.view(torch.float32) if which else raw).view(shape)

    codes = property(lambda self: self._part(0))
    blocks = property(lambda self: self._part(1))
    mean = property(lambda self: self._part(2))
    rstd = property(lambda self: self._part(3))

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self._parts if t is not None)

    def _check(self, where: str, norm: bool):
        codes, blocks, mean, rstd = (self._part(k) for k in range(4))
        n = self._rows
        if (codes.dtype != torch.uint8 or tuple(codes.shape) != (n, -(-self.width // 16) * 16)
                or blocks.dtype != torch.float32 or tuple(blocks.shape) != (n, -(-self.width // CHECKPOINT_BLOCK), 2)
                or not codes.is_contiguous() or not blocks.is_contiguous()):
            raise ValueError(f"{where}: not a checkpoint of {n} rows of {self.width} values")
        if not codes.is_cuda:
            raise ValueError(f"{where}: the checkpoint must be on a CUDA device (khan_b200 has no CPU path)")
        if norm != (mean is not None) or norm != (rstd is not None):
            raise ValueError(f"{where}: gain and bias go with the checkpoint of a normalised layer, and only with that")
        for t in (mean, rstd) if norm else ():
            _per_row(t, "mean and rstd", torch.empty((n, 0), dtype=torch.float32, device=codes.device))
            if not t.is_contiguous():
                raise ValueError(f"{where}: mean and rstd must be contiguous")
        _lib.same_device(codes.device, blocks, where=where)


def _params(gain, bias, acs, x, where: str):
    if (gain is None) != (bias is None):
        raise ValueError(f"{where}: gain and bias are given together or not at all")
    if gain is None:
        return None, None
    return _vectors(gain, "gain", acs, x), _vectors(bias, "bias", acs, x)


def checkpoint_activation(z, activation, gain=None, bias=None, acs=None, eps: float = 1e-5):
    """``(a, checkpoint)``: ``a = act(z)``, or ``act(layer_norm(z))`` with ``gain`` and ``bias``, and an
    :class:`ActivationCheckpoint` of ``z`` (``a`` itself is exact, only the backward pass sees the 8 bits).
    ``activation``: one of :mod:`khan_b200.model.activations`, or its name."""
    act = _activation_id(activation)
    out = _lib.torch_ops().checkpoint_activation(z, act, gain, bias, acs, eps)
    if out is None:
        z = _rows(z, "z")
        if z.dtype != torch.float32:
            raise TypeError(f"checkpoints are of float32 layers, got {z.dtype}")
        acs = _counts(acs, z.shape[0])
        gain, bias = _params(gain, bias, acs, z, "checkpoint_activation")
        out = _lib.torch_ops().checkpoint_activation(z, act, gain, bias, acs, eps)
    a, buffer = _done("ani_checkpoint_activation_f32", out)
    return a, ActivationCheckpoint._of_buffer(buffer, *z.shape, act, gain is not None)


def _grad_arguments(kept, grad, width, gain, bias, acs, where):
    kept._check(where, gain is not None)
    grad = _rows(grad, "the gradient")
    if grad.dtype != torch.float32:
        raise TypeError(f"{where}: the gradient is {grad.dtype}, expected torch.float32")
    if grad.shape[0] != kept._rows or (width is not None and grad.shape[1] != width):
        raise ValueError(f"{where}: a gradient {tuple(grad.shape)} does not fit the checkpoint of "
                         f"{kept._rows} rows of {kept.width} values")
    _lib.same_device(kept._parts[0].device, grad, where=where)
    acs = _counts(acs, grad.shape[0])
    like = torch.empty((0, kept.width), dtype=torch.float32, device=grad.device)
    gain, bias = _params(gain, bias, acs, like, where)
    return grad, gain, bias, acs


def checkpoint_activation_grad(kept, grad_a, gain=None, bias=None, acs=None):
    """Backward pass of :func:`checkpoint_activation` from its checkpoint: ``(grad_z, grad_sum, grad_gain, grad_bias)``,
    ``grad_sum`` the column sums of ``grad_z`` (the gradient of the bias of the dense layer in front), the last two None
    without a norm."""
    call = _lib.torch_ops().checkpoint_activation_grad
    out = call(*kept._parts, kept._rows, kept._normed, kept.width, kept.activation, grad_a, gain, bias, acs)
    if out is None:
        grad_a, gain, bias, acs = _grad_arguments(kept, grad_a, kept.width, gain, bias, acs, "checkpoint_activation_grad")
        out = call(*kept._parts, kept._rows, kept._normed, kept.width, kept.activation, grad_a, gain, bias, acs)
    return _done("ani_checkpoint_activation_grad_f32", out)


def checkpoint_weight_grad(kept, grad_z, gain=None, bias=None, acs=None):
    """Weight gradient of the dense layer behind a checkpointed activation, ``act(...)^T grad_z`` summed over the rows (of
    each element), ``[width, out]`` or ``[4, width, out]``; the activations are recomputed from the checkpoint."""
    call = _lib.torch_ops().checkpoint_weight_grad
    out = call(*kept._parts, kept._rows, kept._normed, kept.width, kept.activation, grad_z, gain, bias, acs)
    if out is None:
        grad_z, gain, bias, acs = _grad_arguments(kept, grad_z, None, gain, bias, acs, "checkpoint_weight_grad")
        out = call(*kept._parts, kept._rows, kept._normed, kept.width, kept.activation, grad_z, gain, bias, acs)
    return _done("ani_checkpoint_weight_grad_f32", out)


# ---------------------------------------------------------------- autograd
def dense_layer_norm(x, gain, bias, eps: float):
    """Layer norm of one group of rows in plain differentiable torch ops."""
    d = x - x.mean(1, keepdim=True)
    return d * torch.rsqrt((d * d).mean(1, keepdim=True) + eps) * gain + bias


class _LayerNorm(torch.autograd.Function):
    """Layer norm on the kernels.  When its backward pass itself has to be differentiated (force training,
    ``create_graph=True``) that pass is evaluated in dense differentiable torch ops instead."""

    @staticmethod
    def forward(ctx, x, acs, eps, *params):
        groups = len(params) // 2
        gain, bias = (list(params[:4]), list(params[4:])) if acs is not None else params
        y, mean, rstd = layer_norm(x, gain, bias, acs, eps)
        ctx.save_for_backward(x, mean, rstd, *params)
        ctx.acs, ctx.eps, ctx.groups = acs, eps, groups
        return y

    @staticmethod
    def backward(ctx, grad_y):
        x, mean, rstd, *params = ctx.saved_tensors
        acs, groups = ctx.acs, ctx.groups
        if torch.is_grad_enabled():
            # With respect to views of the inputs, one for each place: a tensor that serves several elements, or that x was
            # made from, gets at each place that place's part alone (autograd adds them up and goes on behind x itself).
            with torch.enable_grad():
                inputs = [t.view_as(t) for t in (x, *params)]
                ends = np.cumsum(acs if acs is not None else [x.shape[0]]).tolist()
                y = torch.cat([dense_layer_norm(inputs[0][a:b], inputs[1 + t].reshape(-1), inputs[1 + groups + t].reshape(-1), ctx.eps)
                               for t, (a, b) in enumerate(zip([0] + ends[:-1], ends))])
                need = [ctx.needs_input_grad[0]] + list(ctx.needs_input_grad[3:])
                wanted = [k for k, wants in enumerate(need) if wants]
                got = torch.autograd.grad(y, [inputs[k] for k in wanted], grad_y, create_graph=True, allow_unused=True)
            out = [None] * len(inputs)
            for k, g in zip(wanted, got):
                out[k] = g
            return (out[0], None, None, *out[1:])
        gain = list(params[:4]) if acs is not None else params[0]
        dx, dgain, dbias = layer_norm_grad(grad_y, x, gain, mean, rstd, acs)
        per_group = [*dgain, *dbias] if acs is not None else [dgain, dbias]
        return (dx, None, None, *(g.view(p.shape) for g, p in zip(per_group, params)))


def layer_norm_autograd(x, gain, bias, acs=None, eps: float = 1e-5):
    """:func:`layer_norm` (``y`` alone) that torch.autograd can differentiate, twice where that is asked for."""
    if acs is not None:
        gain, bias = tuple(gain), tuple(bias)
        for v, name in ((gain, "gain"), (bias, "bias")):
            if len(v) != 4:      # eight in all would do for what follows: the fifth gain would be the first bias
                raise ValueError(f"{name}: rows grouped by element take a list of four vectors, not of {len(v)}")
        # the counts as they are now: the caller's array may be filled with another batch's before the backward pass
        return _LayerNorm.apply(x, _counts(acs, x.shape[0]).copy(), eps, *gain, *bias)
    return _LayerNorm.apply(x, None, eps, gain, bias)

"""Atomic and molecular networks: the model side of khan (``khan/model/nn.py`` of the reference).

``AtomNN`` is one dense stack per element, ``A = act(A W + b)`` with a linear last layer of width
one; ``MoleculeNN`` holds one ``AtomNN`` per element, evaluates each on the feature rows of its
element and brings the atomic energies back to atom order with ``gather_idxs``
(``khan/model/nn.py:39-67,165-172``).  Parameters keep the reference's shapes and names
(``W`` is ``(in, out)``, names like ``near_W_H_384x128_l1``) so that its ``.npz`` checkpoints map
one to one.

For float32 and the architecture 384-128-128-64-1 the forward pass of all four networks is one
fused tensor-core kernel (``ani_mlp_forward_f32``); its backward pass and every other
architecture or precision use torch's dense GEMMs on the GPU.

Two options go beyond the reference, for networks that are deeper or wider than its own.  ``layer_norm``:
every hidden layer is ``A = act(norm(A W + b))`` with a gain and a shift per column.
``activation_checkpoints``: training keeps the input of every activation in 8 bits between the forward and
the backward pass, instead of that input and the activation in 32 (:mod:`khan_b200.layer_mod`).
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from .. import _lib, layer_mod
from . import activations

FUSED_LAYERS = (384, 128, 128, 64, 1)
TYPE_MAP = ["H", "C", "N", "O"]


class AtomNN:
    """Dense stack for the atoms of one element."""

    def __init__(self, layer_sizes, precision=torch.float32, activation_fn=activations.celu,
                 atom_type: str = "", prefix: str = "", device="cuda", generator=None,
                 init: str = "reference", layer_norm: bool = False, norm_eps: float = 1e-5):
        assert precision in (torch.float32, torch.float64)
        assert layer_sizes[-1] == 1
        self.layer_sizes = tuple(int(v) for v in layer_sizes)
        self.precision = precision
        self.activation_fn = activation_fn
        self.atom_type = atom_type
        self.layer_norm, self.norm_eps = bool(layer_norm), float(norm_eps)
        self.Ws, self.bs, self.names = [], [], []
        self.gains, self.shifts, self.norm_names = [], [], []      # of the hidden layers' norms
        for idx in range(1, len(layer_sizes)):
            x, y = layer_sizes[idx - 1], layer_sizes[idx]
            # reference: N(0, sqrt(2 / (x + y))), khan/model/nn.py:45-59; "he": N(0, sqrt(2 / x))
            std = (2.0 / (x + y)) ** 0.5 if init == "reference" else (2.0 / x) ** 0.5
            w = torch.randn((x, y), dtype=torch.float64, generator=generator) * std
            name = "_" + atom_type + "_" + str(x) + "x" + str(y) + "_l" + str(idx)
            self.Ws.append(w.to(precision).to(device).requires_grad_(True))
            self.bs.append(torch.zeros(y, dtype=precision, device=device, requires_grad=True))
            self.names.append((prefix + "W" + name, prefix + "b" + name))
            if self.layer_norm and idx < len(layer_sizes) - 1:
                name = "_" + atom_type + "_" + str(y) + "_l" + str(idx)
                self.gains.append(torch.ones(y, dtype=precision, device=device, requires_grad=True))
                self.shifts.append(torch.zeros(y, dtype=precision, device=device, requires_grad=True))
                self.norm_names.append((prefix + "gain" + name, prefix + "shift" + name))

    def get_parameters(self):
        return self.Ws + self.bs + self.gains + self.shifts

    def named_parameters(self):
        out = {}
        for names, first, second in ((self.names, self.Ws, self.bs), (self.norm_names, self.gains, self.shifts)):
            for (fn, sn), f, s in zip(names, first, second):
                out[fn + ":0"] = f
                out[sn + ":0"] = s
        return out

    def atom_energies(self, features: torch.Tensor) -> torch.Tensor:
        """Energies ``(n,)`` of the feature rows ``(n, layer_sizes[0])`` (dense torch path)."""
        a = features
        last = len(self.Ws) - 1
        for k, (w, b) in enumerate(zip(self.Ws, self.bs)):
            a = a @ w + b
            if k != last:
                if self.layer_norm:
                    norm = layer_mod.layer_norm_autograd if a.is_cuda else layer_mod.dense_layer_norm
                    a = norm(a, self.gains[k], self.shifts[k], eps=self.norm_eps)
                a = self.activation_fn(a)
        return a.reshape(-1)


def _dense_energies(features, acs, act_fn, params):
    """The four networks in plain differentiable torch ops (element-sorted rows in and out)."""
    starts = np.concatenate([[0], np.cumsum(acs)])
    parts = []
    for t in range(4):
        a = features[int(starts[t]):int(starts[t + 1])]
        w1, b1, w2, b2, w3, b3, w4, b4 = params[8 * t: 8 * t + 8]
        a = act_fn(a @ w1 + b1)
        a = act_fn(a @ w2 + b2)
        a = act_fn(a @ w3 + b3)
        parts.append((a @ w4 + b4).reshape(-1))
    return torch.cat(parts)


class _FusedMlp(torch.autograd.Function):
    """The four atomic networks on the tensor-core kernels: one launch forward
    (``ani_mlp_forward_f32``), one launch for the backward pass along the activations
    (``ani_mlp_backward_f32``: dz1, dz2, dz3 and the feature gradient); the weight gradients are
    the plain products ``A_{l-1}^T dz_l`` over the atoms of each element.  When the backward pass
    itself has to be differentiated (force training, ``create_graph=True``) it is evaluated in
    dense differentiable torch ops instead."""

    @staticmethod
    def forward(ctx, features, acs, act_id, split, act_and_packed, *params):
        act_fn, packed = act_and_packed
        # params: for each of the 4 elements W1,b1,W2,b2,W3,b3,W4,b4 (reference shapes, W = (in, out))
        n = features.shape[0]
        dev = features.device
        _lib.same_device(dev, *params, packed, where="atomic networks (forward)")
        starts = np.concatenate([[0], np.cumsum(acs)])
        f32 = dict(dtype=torch.float32, device=dev)
        energy = torch.empty(n, **f32)
        acts = [torch.empty((n, 128), **f32), torch.empty((n, 128), **f32), torch.empty((n, 64), **f32)]
        dacts = [torch.empty((n, 128), **f32), torch.empty((n, 128), **f32), torch.empty((n, 64), **f32)]
        args = _lib.MlpArgs()
        keep = []
        for t in range(4):
            w1, b1, w2, b2, w3, b3, w4, b4 = params[8 * t: 8 * t + 8]
            tr = [w1.detach().contiguous(), w2.detach().contiguous(), w3.detach().contiguous(),
                  w4.detach().reshape(-1).contiguous()]      # no copies: the kernel reads [in][out]
            keep.extend(tr)
            s = int(starts[t])
            cnt = int(acs[t])

            def ptr(tensor, offset=0, live=cnt > 0):
                return ctypes.c_void_p(tensor.data_ptr() + offset * tensor.element_size()) if live else None

            args.features[t] = ptr(features, s * 384)
            args.w1[t], args.w2[t], args.w3[t], args.w4[t] = (ptr(x) for x in tr)
            args.b1[t], args.b2[t], args.b3[t], args.b4[t] = (ptr(b.detach()) for b in (b1, b2, b3, b4))
            args.energy[t] = ptr(energy, s)
            args.act1[t], args.act2[t], args.act3[t] = (ptr(a, s * a.shape[1]) for a in acts)
            args.dact1[t], args.dact2[t], args.dact3[t] = (ptr(d, s * d.shape[1]) for d in dacts)
            args.packed[t] = ptr(packed[t]) if packed is not None else None
        acs_arr = np.ascontiguousarray(np.asarray(acs, dtype=np.int32))
        stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().ani_mlp_forward_f32(ctypes.byref(args), acs_arr.ctypes.data_as(_lib.c_int_p),
                                                      int(act_id), int(split) & 1, stream),
                       "ani_mlp_forward_f32")
        ctx.save_for_backward(features, *acts, *dacts, *params)
        ctx.acs, ctx.act_fn, ctx.split, ctx.accumulate = acs_arr, act_fn, bool(int(split) & 1), bool(int(split) & 2)
        ctx.packed = packed      # the weights do not change between this pass and its backward pass
        return energy

    @staticmethod
    def backward(ctx, grad_energy):
        features, a1, a2, a3, d1, d2, d3, *params = ctx.saved_tensors
        acs, act_fn = ctx.acs, ctx.act_fn
        if torch.is_grad_enabled():
            # double backward: everything from differentiable ops so that the second derivative
            # through the activation is kept
            with torch.enable_grad():
                inputs = [features] + list(params)
                wanted = [k for k, need in enumerate([ctx.needs_input_grad[0]] + list(ctx.needs_input_grad[5:])) if need]
                energy = _dense_energies(features, acs, act_fn, params)
                got = torch.autograd.grad(energy, [inputs[k] for k in wanted], grad_energy, create_graph=True,
                                          allow_unused=True)
            out = [None] * len(inputs)
            for k, g in zip(wanted, got):
                out[k] = g
            return (out[0], None, None, None, None, *out[1:])
        n = features.shape[0]
        dev = features.device
        starts = np.concatenate([[0], np.cumsum(acs)])
        f32 = dict(dtype=torch.float32, device=dev)
        dz1, dz2, dz3 = torch.empty((n, 128), **f32), torch.empty((n, 128), **f32), torch.empty((n, 64), **f32)
        grad_feat = torch.empty_like(features) if ctx.needs_input_grad[0] else None
        g = grad_energy.contiguous()
        args = _lib.MlpBackwardArgs()
        keep = []
        for t in range(4):
            s, cnt = int(starts[t]), int(acs[t])
            w1, _, w2, _, w3, _, w4, _ = params[8 * t: 8 * t + 8]
            ws = [w1.detach().contiguous(), w2.detach().contiguous(), w3.detach().contiguous(),
                  w4.detach().reshape(-1).contiguous()]
            keep.extend(ws)

            def ptr(tensor, offset=0, live=cnt > 0):
                return ctypes.c_void_p(tensor.data_ptr() + offset * tensor.element_size()) if live else None

            args.grad_energy[t] = ptr(g, s)
            args.w1[t], args.w2[t], args.w3[t], args.w4[t] = (ptr(x) for x in ws)
            args.dact1[t], args.dact2[t], args.dact3[t] = ptr(d1, s * 128), ptr(d2, s * 128), ptr(d3, s * 64)
            args.dz1[t], args.dz2[t], args.dz3[t] = ptr(dz1, s * 128), ptr(dz2, s * 128), ptr(dz3, s * 64)
            args.grad_features[t] = ptr(grad_feat, s * 384) if grad_feat is not None else None
            args.packed[t] = ptr(ctx.packed[t]) if ctx.packed is not None else None
        stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().ani_mlp_backward_f32(ctypes.byref(args), acs.ctypes.data_as(_lib.c_int_p),
                                                       int(ctx.split), stream), "ani_mlp_backward_f32")
        # weight and bias gradients: one more launch.  With `accumulate_into_grad` set on the model
        # (only valid when gradients are obtained with .backward(), as the trainer does) and a
        # gradient buffer on every parameter (the flat optimiser provides them) the kernel adds
        # into those buffers directly and None is returned, which is what autograd's own
        # accumulation would do with 32 separate additions; otherwise the gradients are slices
        # of one zero-filled buffer and are returned.
        sizes = [384 * 128, 128, 128 * 128, 128, 128 * 64, 64, 64, 4]   # the last slot holds b4 (1 value): keeps every slice 16-byte aligned
        per_elem = sum(sizes)
        direct = ctx.accumulate and all(p.grad is not None and p.grad.is_contiguous() and p.grad.dtype == torch.float32
                     and p.grad.data_ptr() % 16 == 0 for p in params)
        wbuf = None if direct else torch.zeros(4 * per_elem, **f32)
        wargs = _lib.MlpWeightGradArgs()
        grads = [None] * len(params)
        for t in range(4):
            s, e = int(starts[t]), int(starts[t + 1])
            cnt = e - s

            def ptr(tensor, offset=0, live=cnt > 0):
                return ctypes.c_void_p(tensor.data_ptr() + offset * tensor.element_size()) if live else None

            wargs.features[t], wargs.act1[t], wargs.act2[t] = ptr(features, s * 384), ptr(a1, s * 128), ptr(a2, s * 128)
            wargs.act3[t], wargs.grad_energy[t] = ptr(a3, s * 64), ptr(g, s)
            wargs.dz1[t], wargs.dz2[t], wargs.dz3[t] = ptr(dz1, s * 128), ptr(dz2, s * 128), ptr(dz3, s * 64)
            if direct:
                outs = [ptr(p.grad) for p in params[8 * t: 8 * t + 8]]
            else:
                offs = np.concatenate([[0], np.cumsum(sizes)]) + t * per_elem
                outs = [ptr(wbuf, int(o)) for o in offs[:8]]
                if cnt > 0:
                    grads[8 * t: 8 * t + 8] = [
                        wbuf[int(offs[k]):int(offs[k]) + params[8 * t + k].numel()].view(params[8 * t + k].shape)
                        for k in range(8)]
            (wargs.dw1[t], wargs.db1[t], wargs.dw2[t], wargs.db2[t], wargs.dw3[t], wargs.db3[t],
             wargs.dw4[t], wargs.db4[t]) = outs
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().ani_mlp_weight_grad_f32(ctypes.byref(wargs), acs.ctypes.data_as(_lib.c_int_p),
                                                          int(ctx.split), stream), "ani_mlp_weight_grad_f32")
        return (grad_feat, None, None, None, None, *grads)


class _CheckpointedStacks(torch.autograd.Function):
    """The four atomic networks with 8-bit activation checkpoints: dense products by torch, activations, norms and the
    weight gradients behind them by :mod:`khan_b200.layer_mod`.  Between the passes there are one byte and a little per
    hidden activation, and the features.  Gradients are those of the weights; they see the checkpoints (half a step of
    1/255 of a row's spread over 128 columns), the energies do not."""

    @staticmethod
    def forward(ctx, features, acs, act_id, eps, layers, normed, *params):
        # params, layer by layer: four W, four b, and for a normalised hidden layer four gains, four shifts
        ends = np.cumsum(acs).tolist()
        ranges = list(zip([0] + ends[:-1], ends))
        per_layer = _CheckpointedStacks._by_layer(params, layers, normed)
        a, kept = features, []
        for k, (ws, bs, gains, shifts) in enumerate(per_layer):
            z = torch.empty((features.shape[0], ws[0].shape[1]), dtype=torch.float32, device=features.device)
            for (s, e), w, b in zip(ranges, ws, bs):
                if e > s:
                    torch.addmm(b, a[s:e], w, out=z[s:e])
            if k == layers - 1:
                break
            a, checkpoint = layer_mod.checkpoint_activation(z, act_id, gains, shifts, acs, eps)
            kept.append(checkpoint)
        # the checkpoints with the tensors: the backward pass lets go of them, however long the energies are kept
        ctx.save_for_backward(features, *params, *(c._parts[0] for c in kept))
        ctx.ranges, ctx.acs, ctx.layers, ctx.normed, ctx.activation = ranges, acs, layers, normed, kept[0].activation
        return z.reshape(-1)

    @staticmethod
    def _by_layer(params, layers, normed):
        out, at = [], 0
        for k in range(layers):
            with_norm = normed and k < layers - 1
            group = [list(params[at + 4 * i: at + 4 * i + 4]) for i in range(4 if with_norm else 2)]
            out.append((*group, *(() if with_norm else (None, None))))
            at += 4 * len(group)
        return out

    @staticmethod
    def backward(ctx, grad_energy):
        if torch.is_grad_enabled():
            raise RuntimeError("a pass with activation checkpoints can be differentiated once: its activations are kept in "
                               "8 bits (build the network without activation_checkpoints for higher derivatives)")
        features, *saved = ctx.saved_tensors
        acs, ranges, layers = ctx.acs, ctx.ranges, ctx.layers
        params, buffers = saved[:-(layers - 1)], saved[-(layers - 1):]
        per_layer = _CheckpointedStacks._by_layer(params, layers, ctx.normed)
        kept = [layer_mod.ActivationCheckpoint._of_buffer(b, features.shape[0], layer[0][0].shape[1], ctx.activation, ctx.normed)
                for b, layer in zip(buffers, per_layer)]
        grads = [None] * layers
        dz = grad_energy.reshape(-1, 1)
        dsum = torch.stack([dz[s:e].sum(0) for s, e in ranges])
        norm_grads = ()
        for k in range(layers - 1, -1, -1):
            ws = per_layer[k][0]
            if k == 0:
                dws = [features[s:e].t() @ dz[s:e] for s, e in ranges]
            else:
                gains, shifts = per_layer[k - 1][2:]
                dws = layer_mod.checkpoint_weight_grad(kept[k - 1], dz, gains, shifts, acs)
            grads[k] = [*dws, *dsum, *(g for four in norm_grads for g in four)]
            if k == 0:
                break
            da = torch.empty((features.shape[0], ws[0].shape[0]), dtype=torch.float32, device=features.device)
            for (s, e), w in zip(ranges, ws):
                if e > s:
                    torch.mm(dz[s:e], w.t(), out=da[s:e])
            dz, dsum, *norm_grads = layer_mod.checkpoint_activation_grad(kept[k - 1], da, gains, shifts, acs)
            norm_grads = norm_grads if ctx.normed else ()
        return (None,) * 6 + tuple(g for layer in grads for g in layer)


class _GatherRows(torch.autograd.Function):
    """``x[idx]`` whose backward is one scatter-add (torch's own index backward sorts the
    indices first: five launches instead of two)."""

    @staticmethod
    def forward(ctx, x, idx):
        ctx.save_for_backward(idx)
        ctx.n = x.shape[0]
        return x[idx]

    @staticmethod
    def backward(ctx, grad):
        (idx,) = ctx.saved_tensors
        out = torch.zeros((ctx.n,) + tuple(grad.shape[1:]), dtype=grad.dtype, device=grad.device)
        return out.index_add_(0, idx, grad), None


class MoleculeNN:
    """One :class:`AtomNN` per element plus the gather back to atom order."""

    def __init__(self, type_map=TYPE_MAP, layer_sizes=FUSED_LAYERS, precision=torch.float32,
                 activation_fn=activations.celu, prefix: str = "near_", device="cuda", seed=None,
                 init: str = "reference", split_precision: bool = True, layer_norm: bool = False,
                 norm_eps: float = 1e-5, activation_checkpoints: bool = False):
        if activation_checkpoints and (precision != torch.float32 or activation_fn not in activations.KERNEL_ID
                                       or len(type_map) != 4 or len(layer_sizes) < 3):
            raise ValueError("activation checkpoints are for float32 networks of four elements with a hidden layer and one "
                             f"of the activations {activations.get_all_fn_names()}")
        if (layer_norm or activation_checkpoints) and max(layer_sizes[1:]) > layer_mod.MAX_WIDTH:
            raise ValueError(f"layers of normalised or checkpointed networks have at most {layer_mod.MAX_WIDTH} columns")
        gen = torch.Generator().manual_seed(seed) if seed is not None else None
        self.type_map = list(type_map)
        self.layer_sizes = tuple(layer_sizes)
        self.precision = precision
        self.activation_fn = activation_fn
        self.split_precision = split_precision
        self.layer_norm, self.norm_eps = bool(layer_norm), float(norm_eps)
        self.activation_checkpoints = bool(activation_checkpoints)
        self.accumulate_into_grad = False   # see _FusedMlp.backward; set by trainers that call .backward()
        self.anns = [AtomNN(layer_sizes, precision, activation_fn, atom_type=t, prefix=prefix,
                            device=device, generator=gen, init=init, layer_norm=layer_norm, norm_eps=norm_eps)
                     for t in self.type_map]

    def get_parameters(self):
        out = []
        for a in self.anns:
            out.extend(a.get_parameters())
        return out

    def named_parameters(self):
        out = {}
        for a in self.anns:
            out.update(a.named_parameters())
        return out

    def pack_weights(self, stream=None):
        """Refreshes the pre-packed copy of W1, W2, W3 of the four networks (``ani_mlp_pack_weights_f32``:
        one small launch) and returns it, ``[4, ani_mlp_packed_bytes()]`` bytes on the parameters' device.
        The tensor-core kernels that are given it fetch their weight chunks with one bulk copy each;
        it has to be refreshed whenever the weights changed, so the callers do it once per pass."""
        dev = self.anns[0].Ws[0].device
        if getattr(self, "_packed", None) is None or self._packed.device != dev:
            self._packed = torch.empty((4, int(_lib.lib().ani_mlp_packed_bytes())), dtype=torch.uint8, device=dev)
        args = _lib.MlpPackArgs()
        for t, ann in enumerate(self.anns):
            w1, w2, w3 = (w.detach() for w in ann.Ws[:3])
            if not (w1.is_contiguous() and w2.is_contiguous() and w3.is_contiguous()):
                return None
            args.w1[t], args.w2[t], args.w3[t] = w1.data_ptr(), w2.data_ptr(), w3.data_ptr()
            args.packed[t] = self._packed[t].data_ptr()
        if stream is None:
            stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().ani_mlp_pack_weights_f32(ctypes.byref(args), stream), "ani_mlp_pack_weights_f32")
        return self._packed

    def packed_weights(self):
        """The pre-packed copy as ``pack_weights`` last wrote it (None before the first call)."""
        return getattr(self, "_packed", None)

    @property
    def has_kernels(self) -> bool:
        """The architecture of the hand-written network kernels: in float32 all of them, in float64 the one
        that evaluates energies and their gradient (``ani_energy_pass_f64``)."""
        return (self.layer_sizes == FUSED_LAYERS and len(self.anns) == 4
                and self.activation_fn in activations.KERNEL_ID and not self.layer_norm)

    @property
    def fused(self) -> bool:
        return self.precision == torch.float32 and self.has_kernels

    def atom_energies_sorted(self, features: torch.Tensor, acs) -> torch.Tensor:
        """Energies in element-sorted order from the ``[n_atoms, F]`` feature buffer laid out H
        rows, C rows, N rows, O rows."""
        acs = np.asarray(acs, dtype=np.int64)
        if self.activation_checkpoints and features.is_cuda and torch.is_grad_enabled() and not features.requires_grad:
            return self._checkpointed_energies(features, acs)
        if self.fused and features.is_cuda:
            params = []
            for a in self.anns:
                for w, b in zip(a.Ws, a.bs):
                    params.extend([w, b])
            flags = (1 if self.split_precision else 0) | (2 if self.accumulate_into_grad else 0)
            _lib.same_device(features.device, self.anns[0].Ws[0], where="MoleculeNN.atom_energies_sorted")
            packed = self.pack_weights()
            return _FusedMlp.apply(features, acs, activations.KERNEL_ID[self.activation_fn],
                                   flags, (self.activation_fn, packed), *params)
        starts = np.concatenate([[0], np.cumsum(acs)])
        if self.layer_norm and len(self.anns) == 4 and features.is_cuda:
            return self._normed_energies(features, acs, starts)
        parts = [ann.atom_energies(features[int(starts[t]):int(starts[t + 1])])
                 for t, ann in enumerate(self.anns)]
        return torch.cat(parts)

    def _normed_energies(self, features, acs, starts):
        """Dense products per element, every norm of the four elements as one operator."""
        acs = acs.astype(np.int32)
        a = features
        for k in range(len(self.layer_sizes) - 1):
            a = torch.cat([a[int(starts[t]):int(starts[t + 1])] @ ann.Ws[k] + ann.bs[k] for t, ann in enumerate(self.anns)])
            if k < len(self.layer_sizes) - 2:
                a = self.activation_fn(layer_mod.layer_norm_autograd(
                    a, [ann.gains[k] for ann in self.anns], [ann.shifts[k] for ann in self.anns], acs, self.norm_eps))
        return a.reshape(-1)

    def _checkpointed_energies(self, features, acs):
        """Training: the exact energies, and gradients of the weights from 8-bit checkpoints.  Gradients with respect to the
        features (forces) are never formed this way: they would lose digits that a user sees."""
        _lib.same_device(features.device, self.anns[0].Ws[0], where="MoleculeNN.atom_energies_sorted")
        params = []
        layers = len(self.layer_sizes) - 1
        for k in range(layers):
            lists = ["Ws", "bs"] + (["gains", "shifts"] if self.layer_norm and k < layers - 1 else [])
            params.extend(getattr(ann, name)[k] for name in lists for ann in self.anns)
        return _CheckpointedStacks.apply(features, acs.astype(np.int32), self.activation_fn, self.norm_eps, layers,
                                         self.layer_norm, *params)

    def atom_outputs(self, features: torch.Tensor, acs, gather_idxs: torch.Tensor) -> torch.Tensor:
        """Atomic energies in atom order (``tf.gather(tf.concat(...), gather_idxs)``,
        khan/model/nn.py:171-172)."""
        return _GatherRows.apply(self.atom_energies_sorted(features, acs), gather_idxs.long())

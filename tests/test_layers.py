"""Normalised layers and activation checkpoints: what can be checked without a GPU (argument checks of the C entry points,
refusals of the Python ones, the reference implementation of the GPU tests)."""
import ctypes

import numpy as np
import pytest
import torch

import layer_reference as ref
from khan_b200 import _lib, layer_mod

P = ctypes.c_void_p


@pytest.fixture(scope="module")
def handle():
    _lib.build()
    return _lib.lib()


def four(*addresses):
    return (ctypes.c_void_p * 4)(*(list(addresses) + [None] * (4 - len(addresses))))


def test_sizes(handle):
    assert [handle.ani_checkpoint_row_bytes(w) for w in (1, 16, 17, 128, 4096)] == [16, 16, 32, 128, 4096]
    assert [handle.ani_checkpoint_blocks(w) for w in (1, 128, 129, 4096)] == [1, 1, 2, 32]
    assert handle.ani_checkpoint_row_bytes(0) == handle.ani_checkpoint_blocks(4097) == -2
    one, many = (ctypes.c_int * 4)(3, 0, 0, 2), (ctypes.c_int * 4)(100000, 0, 50000, 1)
    assert handle.ani_layer_sums_workspace_bytes(128, one, 3, 4) == 0
    small, large = (handle.ani_layer_sums_workspace_bytes(128, many, 3, s) for s in (4, 8))
    assert small > 0 and large == 2 * small and small % (3 * 128 * 4) == 0
    assert handle.ani_checkpoint_weight_grad_workspace_bytes(128, 64, one) == 0
    assert handle.ani_checkpoint_weight_grad_workspace_bytes(128, 64, many) % (128 * 64 * 4) == 0
    assert handle.ani_checkpoint_weight_grad_workspace_bytes(1, 1, many) % (32 * 32 * 4) == 0
    assert handle.ani_layer_sums_workspace_bytes(0, many, 3, 4) == handle.ani_checkpoint_weight_grad_workspace_bytes(1, 5000, many) == 0


def test_layer_norm_checks_need_no_gpu(handle):
    acs, bad, none = (ctypes.c_int * 4)(5, 0, 0, 2), (ctypes.c_int * 4)(5, -1, 0, 0), (ctypes.c_int * 4)()
    v, x, y = four(0x10000, None, None, 0x20000), 0x30000, 0x40000
    for fwd, grad in ((handle.ani_layer_norm_f32, handle.ani_layer_norm_grad_f32), (handle.ani_layer_norm_f64, handle.ani_layer_norm_grad_f64)):
        assert fwd(None, 128, None, None, 128, 1e-5, none, None, None, None, None) == 0
        assert fwd(x, 128, v, v, 128, 1e-5, None, y, y, y, None) == -1
        assert fwd(None, 128, v, v, 128, 1e-5, acs, y, y, y, None) == fwd(x, 128, None, v, 128, 1e-5, acs, y, y, y, None) == -1
        assert fwd(x, 128, four(0x10000), v, 128, 1e-5, acs, y, y, y, None) == fwd(x, 128, v, v, 128, 1e-5, acs, y, None, y, None) == -1
        for width, stride, eps, counts in ((0, 128, 1e-5, acs), (4097, 5000, 1e-5, acs), (128, 127, 1e-5, acs), (128, 128, -1.0, acs),
                                           (128, 128, float("nan"), acs), (128, 128, float("inf"), acs), (128, 128, 1e-5, bad)):
            assert fwd(x, stride, v, v, width, eps, counts, y, y, y, None) == -2
        assert grad(x, 127, x, 128, v, x, x, 128, acs, y, v, v, None, None) == grad(x, 128, x, 127, v, x, x, 128, acs, y, v, v, None, None) == -2
        assert grad(x, 128, x, 128, v, x, x, 128, acs, y, None, v, None, None) == grad(x, 128, x, 128, v, x, x, 128, acs, None, v, v, None, None) == -1
        # many rows need a workspace, 16-byte aligned
        assert grad(x, 128, x, 128, four(x), x, x, 128, (ctypes.c_int * 4)(100000), y, four(y), four(y), None, None) == -1
        assert grad(x, 128, x, 128, four(x), x, x, 128, (ctypes.c_int * 4)(100000), y, four(y), four(y), y + 8, None) == -9


def test_checkpoint_checks_need_no_gpu(handle):
    acs, none, many = (ctypes.c_int * 4)(5), (ctypes.c_int * 4)(), (ctypes.c_int * 4)(100000)
    v, x = four(0x10000), 0x30000
    fwd, grad, wgrad = handle.ani_checkpoint_activation_f32, handle.ani_checkpoint_activation_grad_f32, handle.ani_checkpoint_weight_grad_f32
    assert fwd(None, 64, None, None, 64, 0.0, 0, none, None, None, None, None, None, None) == 0
    for act in (-1, 4):
        assert fwd(x, 64, None, None, 64, 0.0, act, acs, x, x, x, None, None, None) == -2
        assert grad(x, x, None, None, x, 64, None, None, 64, act, acs, x, v, None, None, None, None) == -2
        assert wgrad(x, x, None, None, None, None, 64, act, x, 8, 8, acs, v, None, None) == -2
    assert fwd(x, 63, None, None, 64, 0.0, 0, acs, x, x, x, None, None, None) == -2
    assert fwd(x, 64, v, v, 64, -1.0, 0, acs, x, x, x, x, x, None) == -2
    # a gain without a bias, a norm without a place for the statistics, codes and blocks that are not aligned
    assert fwd(x, 64, v, None, 64, 0.0, 0, acs, x, x, x, x, x, None) == fwd(x, 64, v, v, 64, 0.0, 0, acs, x, x, x, None, x, None) == -1
    assert fwd(x, 64, None, None, 64, 0.0, 0, acs, x, x + 8, x, None, None, None) == fwd(x, 64, None, None, 64, 0.0, 0, acs, x, x, x + 4, None, None, None) == -9
    assert grad(x, x, None, None, x, 63, None, None, 64, 0, acs, x, v, None, None, None, None) == -2
    assert grad(x, x, None, None, x, 64, None, None, 64, 0, acs, x, None, None, None, None, None) == -1
    assert grad(x, x, x, x, x, 64, v, v, 64, 0, acs, x, v, v, None, None, None) == grad(x, x, None, x, x, 64, v, v, 64, 0, acs, x, v, v, v, None, None) == -1
    assert grad(x + 1, x, None, None, x, 64, None, None, 64, 0, acs, x, v, None, None, None, None) == -9
    assert grad(x, x, None, None, x, 64, None, None, 64, 0, many, x, v, None, None, None, None) == -1
    for width, out, stride in ((0, 8, 8), (4097, 8, 8), (64, 0, 8), (64, 4097, 5000), (64, 8, 7)):
        assert wgrad(x, x, None, None, None, None, width, 0, x, stride, out, acs, v, None, None) == -2
    assert wgrad(x, x, None, None, None, None, 64, 0, x, 8, 8, acs, None, None, None) == wgrad(x, x, None, None, v, None, 64, 0, x, 8, 8, acs, v, None, None) == -1
    assert wgrad(x, x + 4, None, None, None, None, 64, 0, x, 8, 8, acs, v, None, None) == -9
    assert wgrad(x, x, None, None, None, None, 64, 0, x, 8, 8, many, v, None, None) == -1
    assert wgrad(x, x, None, None, None, None, 64, 0, x, 8, 8, many, v, x + 8, None) == -9
    assert grad(x, x, None, None, x, 64, None, None, 64, 0, many, x, v, None, None, x + 4, None) == -9


def test_there_is_no_cpu_path():
    x, g = torch.zeros(3, 4), torch.ones(4)
    for call in (lambda: layer_mod.layer_norm(x, g, g), lambda: layer_mod.layer_norm_grad(x, x, g, x[:, 0], x[:, 0]),
                 lambda: layer_mod.checkpoint_activation(x, "celu")):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    kept = layer_mod.ActivationCheckpoint(torch.zeros((3, 16), dtype=torch.uint8), torch.zeros((3, 1, 2)), 4, "celu")
    for call in (layer_mod.checkpoint_activation_grad, layer_mod.checkpoint_weight_grad):
        with pytest.raises(ValueError, match="no CPU path"):
            call(kept, x)
    with pytest.raises(ValueError, match="activation"):
        layer_mod.ActivationCheckpoint(kept.codes, kept.blocks, 4, "relu")


def test_reference_norm_agrees_with_torch_in_double():
    rng = np.random.default_rng(0)
    x, up = rng.standard_normal((9, 13)), rng.standard_normal((9, 13))
    gain, bias = [list(rng.standard_normal((4, 13))) for _ in range(2)]
    acs = np.array([4, 0, 3, 2])
    (y, mean, rstd), _ = ref.norm(x, gain, bias, acs, 1e-3)
    (dx, dg, db), _ = ref.norm_grad(up, x, gain, mean.astype(float), rstd.astype(float), acs)
    for t, rows in enumerate(ref.element_rows(acs)):
        xt, g, b = (torch.from_numpy(np.asarray(v)).requires_grad_(True) for v in (x[rows], gain[t], bias[t]))
        out = torch.nn.functional.layer_norm(xt, (13,), g, b, 1e-3)
        out.backward(torch.from_numpy(up[rows]))
        for got, want in ((y[rows], out.detach()), (dx[rows], xt.grad), (dg[t], g.grad), (db[t], b.grad)):
            assert np.allclose(got.astype(float), want.numpy(), rtol=0, atol=1e-12)


def test_reference_activations_agree_with_the_framework_in_double():
    from khan_b200.model import activations
    u = torch.linspace(-6, 6, 2001, dtype=torch.float64, requires_grad=True)
    for name in activations.get_all_fn_names():
        a = activations.get_fn_by_name(name)(u)
        (d,) = torch.autograd.grad(a.sum(), u)
        value, slope, second = ref.act(name, u.detach().numpy().astype(ref.LD))
        assert np.abs(value - a.detach().numpy()).max() < 1e-14 and np.abs(slope - d.numpy()).max() < 1e-14
        assert np.abs(np.diff(slope)).max() <= second * 0.006 * (1 + 1e-9)


def test_reference_codes_stand_for_the_values():
    rng = np.random.default_rng(1)
    z = (rng.standard_normal((30, 300)) * 5 + 100).astype(np.float32)
    codes, blocks = ref.encode(z)
    step = blocks[:, np.arange(300) // 128, 1]
    assert (np.abs(ref.decode(codes, blocks) - z) <= step * (0.5 + 1e-4)).all() and codes.max() == 255 and codes.min() == 0


def test_networks_refuse_what_checkpoints_cannot_do():
    from khan_b200.model.nn import MoleculeNN
    for kw in (dict(precision=torch.float64), dict(activation_fn=torch.tanh), dict(type_map=["H", "C"]), dict(layer_sizes=(384, 1))):
        with pytest.raises(ValueError, match="activation checkpoints"):
            MoleculeNN(device="cpu", activation_checkpoints=True, **kw)
    with pytest.raises(ValueError, match="4096"):
        MoleculeNN(device="cpu", layer_norm=True, layer_sizes=(384, 4097, 1))


def test_normed_networks_have_named_gains_and_shifts():
    from khan_b200.model.nn import MoleculeNN
    net = MoleculeNN(device="cpu", layer_norm=True, layer_sizes=(384, 32, 16, 1), seed=1)
    names = net.named_parameters()
    assert names["near_gain_H_32_l1:0"] is net.anns[0].gains[0] and names["near_shift_O_16_l2:0"] is net.anns[3].shifts[1]
    assert sorted(map(id, names.values())) == sorted(map(id, net.get_parameters()))
    plain = MoleculeNN(device="cpu", layer_sizes=(384, 32, 16, 1), seed=1)
    assert sorted(plain.named_parameters()) == sorted(n for n in names if "gain" not in n and "shift" not in n)
    x = torch.rand((5, 384))
    u = x @ net.anns[0].Ws[0] + net.anns[0].bs[0]
    a = torch.nn.functional.layer_norm(u, (32,), net.anns[0].gains[0], net.anns[0].shifts[0], 1e-5)
    a = net.activation_fn(a) @ net.anns[0].Ws[1] + net.anns[0].bs[1]
    a = torch.nn.functional.layer_norm(a, (16,), net.anns[0].gains[1], net.anns[0].shifts[1], 1e-5)
    want = (net.activation_fn(a) @ net.anns[0].Ws[2] + net.anns[0].bs[2]).reshape(-1)
    assert torch.allclose(net.atom_energies_sorted(x, [5, 0, 0, 0]), want, atol=1e-5)


@pytest.fixture
def norm_on_the_host(monkeypatch):
    """layer_norm and layer_norm_grad in torch's operations on the host, so that what autograd makes of them needs no GPU."""
    def norm(x, gain, bias, acs=None, eps=1e-5):
        mean = x.detach().mean(1)
        rstd = ((x.detach() - mean[:, None]).square().mean(1) + eps).rsqrt()
        gain, bias = ([gain], [bias]) if acs is None else (gain, bias)
        y = [(x.detach()[r] - mean[r, None]) * rstd[r, None] * gain[t].detach().reshape(-1) + bias[t].detach().reshape(-1)
             for t, r in enumerate(ref.element_rows([len(x)] if acs is None else acs))]
        return torch.cat(y), mean, rstd

    def norm_grad(grad_y, x, gain, mean, rstd, acs=None):
        xhat, dx, sums = (x - mean[:, None]) * rstd[:, None], [], []
        for g, r in zip([gain] if acs is None else gain, ref.element_rows([len(x)] if acs is None else acs)):
            up = g.reshape(-1) * grad_y[r]
            dx.append(rstd[r, None] * (up - up.mean(1, keepdim=True) - xhat[r] * (up * xhat[r]).mean(1, keepdim=True)))
            sums.append(((grad_y[r] * xhat[r]).sum(0), grad_y[r].sum(0)))
        dg, db = (torch.stack(s) for s in zip(*sums))
        return (torch.cat(dx), dg, db) if acs is not None else (torch.cat(dx), dg[0], db[0])

    monkeypatch.setattr(layer_mod, "layer_norm", norm)
    monkeypatch.setattr(layer_mod, "layer_norm_grad", norm_grad)


def shared_norms(device="cpu"):
    """Layer norms whose parameters and rows are not independent of each other, each as (name, output, inputs)."""
    gen = torch.Generator().manual_seed(5)

    def new(*shape):
        return torch.randn(shape, generator=gen, dtype=torch.float64).to(device).requires_grad_(True)

    acs = np.array([3, 0, 2, 4], np.int32)
    x, g, b, h = new(9, 6), new(6), new(6), new(6)
    yield "one gain and bias for all elements", layer_mod.layer_norm_autograd(x, [g] * 4, [b] * 4, acs, 1e-3), (x, g, b)
    yield "gains in pairs", layer_mod.layer_norm_autograd(x, [g, h, h, g], [b, g, b, h], acs, 1e-3), (x, g, b, h)
    yield "bias = gain", layer_mod.layer_norm_autograd(x, g, g, None, 1e-3), (x, g)
    first = torch.tanh(layer_mod.layer_norm_autograd(x, g, b, None, 1e-3) * 1.5)
    yield "one gain in two norms", layer_mod.layer_norm_autograd(first, g, b, None, 1e-3), (x, g, b)
    yield "rows made of the gain", layer_mod.layer_norm_autograd(x * g, g, b, None, 1e-3), (x, g, b)


def check_shared_norms(device):
    """The first derivatives do not depend on whether a second one may follow, and the second ones are those of the formula."""
    plain = layer_mod.dense_layer_norm
    for name, y, inputs in shared_norms(device):
        up = torch.randn(y.shape, generator=torch.Generator().manual_seed(6), dtype=torch.float64).to(device)
        once = torch.autograd.grad(y, inputs, up, retain_graph=True)
        twice = torch.autograd.grad(y, inputs, up, create_graph=True)
        for p, q in zip(once, twice):
            # sums of at most 54 terms of size below 40 in double precision, formed in another order
            assert float((p - q.detach()).abs().max()) < 54 * 40 * 2.0 ** -52, name
        second = torch.autograd.grad(sum((t * t).sum() for t in twice), inputs, materialize_grads=True)
        x, g, b, *rest = [t.detach().clone().requires_grad_(True) for t in inputs] + ([] if len(inputs) > 2 else [None])
        rows = ref.element_rows([3, 0, 2, 4])
        grouped = lambda gs, bs: torch.cat([plain(x[r], p, q, 1e-3) for r, p, q in zip(rows, gs, bs)])  # noqa: E731
        want = {"one gain and bias for all elements": lambda: grouped([g] * 4, [b] * 4),
                "gains in pairs": lambda: grouped([g, rest[0], rest[0], g], [b, g, b, rest[0]]),
                "bias = gain": lambda: plain(x, g, g, 1e-3),
                "one gain in two norms": lambda: plain(torch.tanh(plain(x, g, b, 1e-3) * 1.5), g, b, 1e-3),
                "rows made of the gain": lambda: plain(x * g, g, b, 1e-3)}[name]()
        leaves = [t for t in (x, g, b, *rest) if t is not None]
        first = torch.autograd.grad(want, leaves, up, create_graph=True)
        for p, q in zip(twice, first):
            assert torch.allclose(p, q, rtol=1e-10, atol=1e-10), name
        for p, q in zip(second, torch.autograd.grad(sum((t * t).sum() for t in first), leaves, materialize_grads=True)):
            assert torch.allclose(p, q, rtol=1e-9, atol=1e-9 * float(q.abs().max())), name


def test_second_derivatives_of_norms_that_share_parameters(norm_on_the_host):
    check_shared_norms("cpu")


def test_lists_of_gains_and_biases_are_of_four(norm_on_the_host):
    """Eight vectors in all are not enough: the fifth gain would serve as the first bias."""
    x, v, acs = torch.ones((5, 3)), torch.ones(3), np.array([2, 1, 1, 1], np.int32)
    for gains, biases in ((5, 3), (3, 5), (4, 3), (5, 5), (8, 0), (0, 8)):
        with pytest.raises(ValueError, match="list of four"):
            layer_mod.layer_norm_autograd(x, [v] * gains, [v] * biases, acs)
    for gain, bias in ((v, v), ([v] * 4, v), (v, [v] * 4)):
        with pytest.raises(ValueError, match="list of four"):
            layer_mod.layer_norm_autograd(x, gain, bias, acs)
    for four in ([v] * 4, (v,) * 4, torch.ones(4, 3)):
        assert layer_mod.layer_norm_autograd(x, four, [v] * 4, acs).shape == layer_mod.layer_norm_autograd(x, [v] * 4, four, acs).shape == (5, 3)


@pytest.mark.parametrize("shape", [(6,), (1, 6), (6, 1), (2, 3)])
@pytest.mark.parametrize("grouped", [False, True])
def test_gains_and_biases_of_any_shape_with_a_value_per_column(norm_on_the_host, shape, grouped):
    """Their gradients have their shape, and the values of the vector's, whether a second derivative follows or not."""
    gen = torch.Generator().manual_seed(7)
    x, g, b, up = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((6, 6), 6, 6, (6, 6)))      # as many rows as columns
    acs = np.array([2, 0, 3, 1], np.int32) if grouped else None
    results = []
    for s in ((6,), shape):
        p, q = (t.reshape(s).clone().requires_grad_(True) for t in (g, b))
        leaf = x.clone().requires_grad_(True)
        y = layer_mod.layer_norm_autograd(leaf, [p] * 4 if grouped else p, [q] * 4 if grouped else q, acs)
        once = torch.autograd.grad(y, (leaf, p, q), up, retain_graph=True)
        twice = torch.autograd.grad(y, (leaf, p, q), up, create_graph=True)
        second = torch.autograd.grad((twice[0] ** 2).sum() + (twice[1] ** 2).sum(), (leaf, p))
        assert once[1].shape == twice[1].shape == once[2].shape == twice[2].shape == second[1].shape == torch.Size(s)
        results.append([t.detach().reshape(-1) for t in (*once, *twice, *second)])
    for got, want in zip(results[1], results[0]):
        assert torch.equal(got, want)


def test_counts_may_change_behind_the_forward_pass(norm_on_the_host):
    """A batch's counts are often the place of the next batch's: the backward pass goes by those of its forward pass."""
    gen = torch.Generator().manual_seed(8)
    x, up = (torch.randn((9, 4), generator=gen, dtype=torch.float64) for _ in range(2))
    gains, biases = ([torch.randn(4, generator=gen, dtype=torch.float64).requires_grad_(True) for _ in range(4)] for _ in range(2))
    results = []
    for counts in (np.array([3, 1, 4, 1], np.int32), torch.tensor([3, 1, 4, 1], dtype=torch.int32)):
        for twice in (False, True):
            for change in (False, True):
                acs = counts.clone() if isinstance(counts, torch.Tensor) else counts.copy()
                leaf = x.clone().requires_grad_(True)
                y = layer_mod.layer_norm_autograd(leaf, gains, biases, acs)
                if change:
                    acs[:] = acs[[1, 0, 3, 2]]
                results.append(torch.autograd.grad(y, (leaf, *gains, *biases), up, create_graph=twice))
    for got in results[1:]:
        for p, q in zip(got, results[0]):
            assert torch.allclose(p, q, rtol=1e-10, atol=1e-10)

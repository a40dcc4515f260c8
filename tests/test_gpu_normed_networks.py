"""Networks with layer norms and with 8-bit activation checkpoints: MoleculeNN and the trainer on the operators of
khan_b200.layer_mod, together."""
import numpy as np
import pytest

import layer_reference as ref

pytestmark = pytest.mark.gpu

LAYERS = (384, 96, 130, 33, 1)
ACS = [np.array([70, 50, 20, 13], np.int32), np.array([0, 41, 0, 7], np.int32)]


def network(precision="float32", layers=LAYERS, act="celu", seed=3, **kw):
    import torch
    from khan_b200.model import activations
    from khan_b200.model.nn import MoleculeNN
    net = MoleculeNN(layer_sizes=layers, precision=getattr(torch, precision), activation_fn=activations.get_fn_by_name(act),
                     device="cuda:0", seed=seed, **kw)
    gen = torch.Generator().manual_seed(seed + 1)
    with torch.no_grad():
        for ann in net.anns:
            for p in ann.bs + ann.gains + ann.shifts:
                p.add_(0.2 * torch.randn(p.shape, generator=gen, dtype=torch.float64).to(p))
    return net


def rows(acs, precision="float32", seed=0):
    import torch
    gen = torch.Generator().manual_seed(seed)
    n = int(acs.sum())
    return (torch.rand((n, 384), generator=gen, dtype=torch.float64).to(getattr(torch, precision)).cuda(),
            torch.randn(n, generator=gen, dtype=torch.float64).to(getattr(torch, precision)).cuda() * 1e-2)


def plain_energies(net, features, acs, params):
    """The networks in double precision, in torch's elementary operations; params: {id of a parameter: its double}."""
    import torch
    out = []
    for ann, r in zip(net.anns, ref.element_rows(acs)):
        a = features[r]
        for k, (w, b) in enumerate(zip(ann.Ws, ann.bs)):
            a = a @ params[id(w)] + params[id(b)]
            if k < len(ann.Ws) - 1:
                if net.layer_norm:
                    d = a - a.mean(1, keepdim=True)
                    a = d / torch.sqrt((d * d).mean(1, keepdim=True) + net.norm_eps) * params[id(ann.gains[k])] + params[id(ann.shifts[k])]
                a = net.activation_fn(a)
        out.append(a.reshape(-1))
    return torch.cat(out)


def doubles(net):
    return {id(p): p.detach().double().requires_grad_(True) for p in net.get_parameters()}


def off(a, b):
    a, b = a.detach().double(), b.detach()
    return float((a - b).norm() / b.norm().clamp_min(1e-300))


@pytest.mark.parametrize("precision,tol", [("float32", 5e-6), ("float64", 1e-13)])
@pytest.mark.parametrize("acs", ACS)
def test_normed_networks_and_their_gradients(acs, precision, tol):
    """Energies, gradients of weights and of the features, and second derivatives, against double precision."""
    import torch
    net = network(precision, layer_norm=True)
    assert not net.fused and len(net.named_parameters()) == len(net.get_parameters()) == 4 * (2 * 4 + 2 * 3)
    features, up = rows(acs, precision)
    features.requires_grad_(True)
    params = doubles(net)
    f64 = features.detach().double().requires_grad_(True)
    energy, want = net.atom_energies_sorted(features, acs), plain_energies(net, f64, acs, params)
    assert off(energy, want) < tol
    (energy * up).sum().backward(retain_graph=True)
    (want * up.double()).sum().backward(retain_graph=True)
    assert off(features.grad, f64.grad) < 4 * tol
    for p in net.get_parameters():
        other = params[id(p)].grad
        if not other.any():
            assert not p.grad.any()
        else:
            assert off(p.grad, other) < 8 * tol
    # through the gradient: what force training differentiates
    (g,) = torch.autograd.grad(energy.sum(), features, create_graph=True)
    (h,) = torch.autograd.grad(want.sum(), f64, create_graph=True)
    got = torch.autograd.grad((g * g).sum(), [net.anns[1].Ws[0], net.anns[1].gains[1], net.anns[3].Ws[2]])
    other = torch.autograd.grad((h * h).sum(), [params[id(p)] for p in (net.anns[1].Ws[0], net.anns[1].gains[1], net.anns[3].Ws[2])])
    for p, q in zip(got, other):
        assert off(p, q) < 100 * tol


@pytest.mark.parametrize("act", ["celu", "gaussian", "softplus"])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("acs", ACS)
def test_gradients_from_checkpoints(acs, normed, act, monkeypatch):
    """The whole stack: the energies are exact; the weight gradients are those of the formula with every activation at the
    point that its checkpoint stands for, in extended precision."""
    from khan_b200 import layer_mod
    net = network(layer_norm=normed, act=act, activation_checkpoints=True)
    features, up = rows(acs)
    kept, keep = [], layer_mod.checkpoint_activation
    monkeypatch.setattr(layer_mod, "checkpoint_activation", lambda *a, **k: [kept.append(out[1]) or out for out in [keep(*a, **k)]][0])
    energy = net.atom_energies_sorted(features, acs)
    (energy * up).sum().backward()
    assert len(kept) == 3
    assert off(energy, plain_energies(net, features.double(), acs, doubles(net)).detach()) < 5e-6
    host = lambda t: t.detach().cpu().numpy()  # noqa: E731
    wide = lambda t: host(t).astype(ref.LD)  # noqa: E731
    da = wide(up)[:, None] * np.concatenate([np.broadcast_to(wide(ann.Ws[3])[:, 0], (int(c), 33)) for ann, c in zip(net.anns, acs)])
    dz = host(up)[:, None]
    for k in (2, 1, 0):
        w = net.layer_sizes[k + 1]
        gain = [host(a.gains[k]) for a in net.anns] if normed else None
        bias = [host(a.shifts[k]) for a in net.anns] if normed else None
        stats = (host(kept[k].mean), host(kept[k].rstd)) if normed else (None, None)
        args = (host(kept[k].codes)[:, :w], host(kept[k].blocks), *stats, act)
        dw, _ = ref.weight_grad(*args, dz, gain, bias, acs)
        # the gradients come from longer chains of float32 products: their relative error in the 2-norm, not a bound
        for t, ann in enumerate(net.anns):
            if acs[t] == 0:
                assert not ann.Ws[k + 1].grad.any() and not ann.bs[k + 1].grad.any()
                continue
            assert np.linalg.norm((host(ann.Ws[k + 1].grad) - dw[t]).astype(float)) < 2e-5 * np.linalg.norm(dw[t].astype(float))
            assert np.allclose(host(ann.bs[k + 1].grad), dz[ref.element_rows(acs)[t]].sum(0).astype(float), rtol=1e-4, atol=1e-7)
        (dz, _, *rest), _ = ref.activation_grad(*args, da, gain, bias, acs)
        for name, want in zip(("gains", "shifts"), rest):
            for t, ann in enumerate(net.anns):
                got = host(getattr(ann, name)[k].grad)
                assert np.linalg.norm((got - want[t]).astype(float)) <= 2e-5 * np.linalg.norm(want[t].astype(float))
        if k:
            da = np.concatenate([dz[r] @ wide(ann.Ws[k]).T for ann, r in zip(net.anns, ref.element_rows(acs))])
    for t, (ann, r) in enumerate(zip(net.anns, ref.element_rows(acs))):
        want = (wide(features)[r].T @ dz[r]).astype(float)
        assert np.linalg.norm(host(ann.Ws[0].grad) - want) <= 2e-5 * np.linalg.norm(want)
    # the checkpoints are a quarter of the activations' inputs and a little, and half a step costs the gradient little
    assert sum(c.nbytes for c in kept) < 0.4 * 4 * len(features) * sum(net.layer_sizes[1:-1])
    exact = network(layer_norm=normed, act=act)
    (exact.atom_energies_sorted(features, acs) * up).sum().backward()
    for p, q in zip(net.get_parameters(), exact.get_parameters()):
        if q.grad.any():
            assert off(p.grad, q.grad.double()) < 0.05


def test_where_checkpoints_are_not_used():
    """Evaluation and gradients with respect to the features are exact, on whatever path; a second derivative is refused."""
    import torch
    acs = ACS[0]
    features, up = rows(acs)
    for layers, normed in ((LAYERS, True), (LAYERS, False), ((384, 128, 128, 64, 1), False)):
        net, plain = network(layers=layers, layer_norm=normed, activation_checkpoints=True), network(layers=layers, layer_norm=normed)
        with torch.no_grad():
            assert torch.equal(net.atom_energies_sorted(features, acs), plain.atom_energies_sorted(features, acs))
        grads = []
        for m in (net, plain):
            x = features.clone().requires_grad_(True)
            grads.append(torch.autograd.grad(m.atom_energies_sorted(x, acs).sum(), x)[0])
        assert torch.equal(*grads)
    energy = net.atom_energies_sorted(features, acs)
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(energy.sum(), net.anns[0].Ws[0], create_graph=True)


def test_a_pass_differentiated_twice_over_and_captured():
    """Two backward passes of one forward pass agree; a captured forward and backward pass gives on replay, with other features
    in the same place, what the eager one gives."""
    import torch
    acs = np.array([400, 300, 90, 60], np.int32)
    features, up = rows(acs)
    other, _ = rows(acs, seed=4)
    net = network(layer_norm=True, activation_checkpoints=True)
    params = net.get_parameters()

    def grads(x, **kw):
        return torch.autograd.grad((net.atom_energies_sorted(x, acs) * up).sum(), params, **kw)

    energy = (net.atom_energies_sorted(features, acs) * up).sum()
    first = torch.autograd.grad(energy, params, retain_graph=True)
    for p, q in zip(first, torch.autograd.grad(energy, params)):
        assert torch.equal(p, q)
    del energy
    want = grads(other)
    place = features.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(place)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = grads(place)
    for source, expected in ((features, first), (other, want), (features, first)):
        place.copy_(source)
        graph.replay()
        for p, q in zip(out, expected):
            # a product that the library forms in another order in a captured pass may move one of 220,000 codes by a step
            assert off(p, q.double()) < 1e-3 or not q.any()


def test_no_atoms():
    import torch
    none = np.zeros(4, np.int32)
    for kw in (dict(layer_norm=True), dict(activation_checkpoints=True), dict(layer_norm=True, activation_checkpoints=True)):
        net = network(**kw)
        energy = net.atom_energies_sorted(torch.zeros((0, 384), device="cuda:0"), none)
        energy.sum().backward()
        assert energy.shape == (0,) and all(not p.grad.any() for p in net.get_parameters())


def trainer(seed=3, layers=(64, 48, 1), **kw):
    import torch
    from khan_b200 import TrainerMultiTower
    return TrainerMultiTower(None, [torch.device("cuda", 0)], layer_sizes=layers, seed=seed, **kw)


def data(n=40):
    from khan_b200 import RawDataset
    from khan_b200.data import synthetic as syn
    b = syn.config1(n_mols=n)
    mols = b.molecules()
    rng = np.random.default_rng(2)
    return RawDataset(mols, [0.01 * len(m) for m in mols], [1e-2 * rng.standard_normal((len(m), 3)) for m in mols])


@pytest.mark.parametrize("kw", [dict(layer_norm=True), dict(activation_checkpoints=True), dict(layer_norm=True, activation_checkpoints=True),
                                dict(layer_norm=True, precision="float64"), dict(layers=(128, 128, 64, 1), activation_checkpoints=True)])
def test_training_saving_and_serving(kw, tmp_path):
    """A training pass with the trainer, its checkpoint file, forces, and force training of the same networks."""
    import torch
    ds, tr = data(), trainer(**kw)
    before = [p.detach().clone() for p in tr.parameters]
    losses = [r[1] for r in tr.feed_dataset(ds, True, [tr.train_op, tr.tower_exp_loss], 16, before_hooks=tr.max_norm_ops)]
    assert len(losses) == 3 and np.isfinite(losses).all()
    assert all(torch.isfinite(p).all() for p in tr.parameters) and not any(torch.equal(p, q) for p, q in zip(before, tr.parameters))
    file = str(tmp_path / "save_file.npz")
    tr.save_numpy(file)
    other = trainer(seed=8, **kw)
    other.load_numpy(file)
    assert all(torch.equal(p, q) for p, q in zip(tr.parameters, other.parameters))
    # atom by atom (the sums over a molecule that predict returns are formed in any order)
    features = rows(ACS[0], kw.get("precision", "float32"))[0]
    with torch.no_grad():
        assert torch.equal(tr.model.atom_energies_sorted(features, ACS[0]), other.model.atom_energies_sorted(features, ACS[0]))
    assert np.isfinite(other.predict(ds)).all()
    # forces against differences of the energy, in double precision
    if kw.get("precision") == "float64":
        X = ds.all_Xs[0].copy()
        _, grad = tr.energy_and_gradient(X)
        for i, c in ((0, 1), (2, 3)):
            e = []
            for h in (1e-4, -1e-4):
                Y = X.copy()
                Y[i, c] += h
                e.append(tr.energy_and_gradient(Y)[0])
            assert abs((e[0] - e[1]) / 2e-4 - grad[i, c - 1]) < 1e-6 * max(1, np.abs(grad).max())
    assert all(np.isfinite(r[1]).all() for r in tr.feed_dataset(ds, False, [tr.train_op_forces, tr.tower_force_rmses], 16))
    assert all(torch.isfinite(p).all() for p in tr.parameters)


def test_files_of_networks_with_and_without_norms_are_told_apart(tmp_path):
    normed, plain = trainer(layer_norm=True), trainer()
    files = [str(tmp_path / f) for f in ("normed.npz", "plain.npz")]
    normed.save_numpy(files[0])
    plain.save_numpy(files[1])
    with pytest.raises(ValueError, match="with layer norms"):
        plain.load_numpy(files[0])
    with pytest.raises(ValueError, match="without layer norms"):
        normed.load_numpy(files[1])


@pytest.mark.parametrize("normed", [False, True])
def test_the_energy_server_reads_both_kinds_of_files(normed, tmp_path, monkeypatch):
    from khan_b200 import energy_server
    tr = trainer(layers=(128, 128, 64, 1), layer_norm=normed, precision="float64")
    tr.save_numpy(str(tmp_path / "save_file.npz"))
    served = []
    monkeypatch.setattr(energy_server, "serve", lambda evaluator, *a, **k: served.append(evaluator))
    energy_server.main(["--save-dir", str(tmp_path)])
    X = data().all_Xs[1]
    want, got = tr.energy_and_gradient(X), served[0].energy_and_gradient(X)
    assert served[0].model.layer_norm == normed
    assert abs(want[0] - got[0]) < 1e-12 * max(1, abs(want[0])) and np.allclose(want[1], got[1], rtol=0, atol=1e-12 * max(1, np.abs(want[1]).max()))


def test_training_step_is_reproducible():
    """The same batches, twice from the same weights: the operators' sums have one order.  (Torch's products and scatter sums
    of the energies are as reproducible as torch makes them: one batch of one molecule each.)"""
    import torch
    acs = np.array([900, 800, 200, 100], np.int32)
    features, up = rows(acs)
    grads = []
    for _ in range(3):
        net = network(layer_norm=True, activation_checkpoints=True)
        (net.atom_energies_sorted(features, acs) * up).sum().backward()
        grads.append([p.grad.clone() for p in net.get_parameters()])
    for other in grads[1:]:
        for p, q in zip(grads[0], other):
            assert torch.equal(p, q)


@pytest.mark.parametrize("normed", [False, True])
def test_the_backward_pass_lets_go_of_the_checkpoints(normed, monkeypatch):
    """As of every tensor that autograd keeps: gone when the graph has been used, though the energies are still there; kept
    with retain_graph; and not to be written to in between."""
    import torch
    from khan_b200 import layer_mod
    acs = np.array([4000, 3000, 900, 600], np.int32)
    net = network(layer_norm=normed, activation_checkpoints=True)
    features, up = rows(acs)
    sizes, keep, last = [], layer_mod.checkpoint_activation, []

    def watched(*args, **kw):
        a, kept = keep(*args, **kw)
        sizes.append(kept.nbytes)
        last[:] = [kept] if watch else []
        return a, kept

    monkeypatch.setattr(layer_mod, "checkpoint_activation", watched)
    watch = False

    def held(retain):
        for p in net.get_parameters():
            p.grad = None
        sizes.clear()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        energy = net.atom_energies_sorted(features, acs)
        forward = torch.cuda.memory_allocated() - before
        grads = torch.autograd.grad((energy * up).sum(), net.get_parameters(), retain_graph=retain)
        assert len(grads) == len(net.get_parameters())
        del grads
        torch.cuda.synchronize()
        return energy, forward, torch.cuda.memory_allocated() - before

    held(False)      # the libraries' workspaces
    energy, forward, after = held(False)
    assert len(sizes) == 3 and forward >= sum(sizes) > 2_000_000
    assert after < 500_000      # the energies, 34 kB, and what the allocator rounds up
    with pytest.raises(RuntimeError, match="second time"):
        energy.sum().backward()
    del energy
    energy, _, after = held(True)
    assert after >= sum(sizes)
    del energy
    watch = True
    energy = net.atom_energies_sorted(features, acs)
    last[0].codes.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        energy.sum().backward()

"""Layer norm, activations kept in 8 bits and the weight gradient from such a checkpoint, against plain implementations in
extended precision (tests/layer_reference.py, where the tolerances are derived)."""
import ctypes

import numpy as np
import pytest
import torch

import layer_reference as ref
from khan_b200 import _lib, layer_mod

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
EPS = 1e-5
ACTS = ["celu", "gaussian", "normal", "softplus"]
# rows, width: every team size and number of column groups, both sides of their borders, one row, one column, odd widths
SHAPES = [(1, 1), (3, 2), (5, 7), (33, 31), (40, 32), (17, 33), (9, 64), (7, 65), (20, 128), (300, 97), (40, 129), (25, 256),
          (13, 257), (13, 384), (11, 500), (6, 513), (5, 1000), (4, 1024), (3, 1025), (3, 2048), (3, 2050), (2, 4095), (2, 4096)]
# many rows: several ranges per element, so that sums are joined by a second launch
MANY = [(2400, 24), (9001, 128), (5000, 300), (1200, 1030)]


def elements(n, kind):
    """Counts of four elements: all of them, some without rows, everything in one."""
    if kind == "mixed":
        c = [n - 3 * (n // 4), n // 4, n // 4, n // 4]
    elif kind == "gaps":
        c = [0, n - n // 3, 0, n // 3]
    else:
        c = [0, 0, n, 0]
    return np.array(c, dtype=np.int32)


def rng_of(*key):
    return np.random.default_rng([int.from_bytes(str(k).encode(), "little") % (1 << 31) for k in key])


def make(n, w, dtype, kind="mixed", seed=0):
    rng = rng_of(n, w, seed)
    x = (rng.standard_normal((n, w)) * (0.3 + rng.random(w)) + rng.standard_normal(w)).astype(dtype)
    gain = [(1 + 0.3 * rng.standard_normal(w)).astype(dtype) for _ in range(4)]
    bias = [(0.3 * rng.standard_normal(w)).astype(dtype) for _ in range(4)]
    up = (rng.standard_normal((n, w)) * 1e-2).astype(dtype)
    return x, gain, bias, up, elements(n, kind)


def dev(a):
    return [torch.from_numpy(v).to(DEV) for v in a] if isinstance(a, list) else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def near(got, want, err, what=""):
    got = got.detach().cpu().numpy()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = np.abs(got.astype(ref.LD) - want)
    bad = ~(off <= err)
    assert not bad.any(), (what, int(bad.sum()), float(off[bad].max()), float(np.broadcast_to(err, off.shape)[bad].min()))


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("n,w", SHAPES + MANY)
def test_layer_norm(n, w, dtype):
    for kind in ("mixed", "gaps"):
        x, gain, bias, _, acs = make(n, w, dtype, kind)
        got = layer_mod.layer_norm(dev(x), dev(gain), dev(bias), acs, EPS)
        want, err = ref.norm(x, gain, bias, acs, EPS)
        for name, g, v, e in zip(("y", "mean", "rstd"), got, want, err):
            near(g, v, e, name)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("n,w", SHAPES + MANY)
def test_layer_norm_gradients(n, w, dtype):
    for kind in ("mixed", "gaps"):
        x, gain, bias, up, acs = make(n, w, dtype, kind)
        _, mean, rstd = layer_mod.layer_norm(dev(x), dev(gain), dev(bias), acs, EPS)
        got = layer_mod.layer_norm_grad(dev(up), dev(x), dev(gain), mean, rstd, acs)
        want, err = ref.norm_grad(up, x, gain, mean.cpu().numpy(), rstd.cpu().numpy(), acs)
        for name, g, v, e in zip(("dx", "dgain", "dbias"), got, want, err):
            near(g, v, e, name)


def test_layer_norm_of_rows_far_from_zero_and_of_constant_rows():
    x, gain, bias, up, acs = make(64, 128, np.float32)
    x = (x + 4096.0).astype(np.float32)
    x[5] = 7.25
    x[6] = 0.0
    got = layer_mod.layer_norm(dev(x), dev(gain), dev(bias), acs, EPS)
    want, err = ref.norm(x, gain, bias, acs, EPS)
    for g, v, e in zip(got, want, err):
        near(g, v, e)
    y, _, rstd = got
    assert torch.equal(y[5:7], dev(bias)[0][None].expand(2, -1))
    near(rstd[5:7], 1 / np.sqrt(np.full(2, EPS, ref.LD)), 1e-6 / np.sqrt(EPS))


def test_layer_norm_keeps_bad_rows_to_themselves():
    x, gain, bias, up, acs = make(40, 200, np.float32)
    clean = [t.cpu() for t in layer_mod.layer_norm(dev(x), dev(gain), dev(bias), acs, EPS)]
    x[3, 7], x[11, 199], x[20, 0] = np.nan, np.inf, -np.inf
    y, mean, rstd = (t.cpu() for t in layer_mod.layer_norm(dev(x), dev(gain), dev(bias), acs, EPS))
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[3, 11, 20]] = True
    assert torch.isnan(y[bad]).all() and not torch.isnan(y[~bad]).any()
    for a, b in zip((y, mean, rstd), clean):
        assert torch.equal(a[~bad], b[~bad])


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("layout", ["slice", "odd_offset", "odd_stride", "transposed", "one_row_for_all", "misaligned_gain"])
def test_layouts_of_rows(dtype, layout):
    x, gain, bias, up, acs = make(60, 128, dtype)
    gd, bd = dev(gain), dev(bias)
    xd, ud = dev(x), dev(up)
    if layout == "slice":
        xd = torch.cat([xd, xd, xd], 1)[:, 128:256]
        ud = torch.cat([ud, ud], 1)[:, 128:]
    elif layout == "odd_offset":
        xd = torch.cat([xd[:, :1], xd, xd[:, :3]], 1)[:, 1:129]
        ud = torch.cat([ud[:, :1], ud, ud[:, :3]], 1)[:, 1:129]
    elif layout == "odd_stride":
        xd = torch.cat([xd, xd[:, :1]], 1)[:, :128]
        ud = torch.cat([ud, ud[:, :1]], 1)[:, :128]
    elif layout == "transposed":
        xd, ud = xd.t().contiguous().t(), ud.t().contiguous().t()
    elif layout == "one_row_for_all":
        xd, x = xd[:1].expand(60, 128), np.repeat(x[:1], 60, 0)
        ud, up = ud[:1].expand(60, 128), np.repeat(up[:1], 60, 0)
    else:
        gd = [torch.cat([g[:1], g])[1:] for g in gd]
    y, mean, rstd = layer_mod.layer_norm(xd, gd, bd, acs, EPS)
    want, err = ref.norm(x, gain, bias, acs, EPS)
    near(y, want[0], err[0])
    got = layer_mod.layer_norm_grad(ud, xd, gd, mean, rstd, acs)
    want, err = ref.norm_grad(up, x, gain, mean.cpu().numpy(), rstd.cpu().numpy(), acs)
    for g, v, e in zip(got, want, err):
        near(g, v, e)
    if dtype == np.float32:
        for g, b in ((None, None), (gd, bd)):
            a, kept = layer_mod.checkpoint_activation(xd, "celu", g, b, acs, EPS)
            same_a, same = layer_mod.checkpoint_activation(dev(x), "celu", g and dev(gain), g and dev(bias), acs, EPS)
            assert torch.equal(a, same_a) and torch.equal(kept.codes[:, :128], same.codes[:, :128]) and torch.equal(kept.blocks, same.blocks)
            for p, q in zip(layer_mod.checkpoint_activation_grad(kept, ud, g, b, acs),
                            layer_mod.checkpoint_activation_grad(same, dev(up), g and dev(gain), g and dev(bias), acs)):
                assert p is q is None or torch.equal(p, q)
            assert torch.equal(layer_mod.checkpoint_weight_grad(kept, ud, g, b, acs),
                               layer_mod.checkpoint_weight_grad(same, dev(up), g and dev(gain), g and dev(bias), acs))


def test_one_group_is_the_first_element_alone():
    x, gain, bias, up, _ = make(77, 96, np.float32)
    acs = np.array([77, 0, 0, 0], dtype=np.int32)
    xd, ud, g, b = dev(x), dev(up), dev(gain), dev(bias)
    alone, four = layer_mod.layer_norm(xd, g[0], b[0]), layer_mod.layer_norm(xd, g, b, acs)
    for p, q in zip(alone, four):
        assert torch.equal(p, q)
    one, all4 = layer_mod.layer_norm_grad(ud, xd, g[0], *alone[1:]), layer_mod.layer_norm_grad(ud, xd, g, *alone[1:], acs)
    assert torch.equal(one[0], all4[0])
    for p, q in zip(one[1:], all4[1:]):
        assert p.shape == (96,) and torch.equal(p, q[0]) and not q[1:].any()
    _, kept = layer_mod.checkpoint_activation(xd, "softplus", g[0], b[0])
    single = layer_mod.checkpoint_activation_grad(kept, ud, g[0], b[0])
    grouped = layer_mod.checkpoint_activation_grad(kept, ud, g, b, acs)
    assert torch.equal(single[0], grouped[0])
    for p, q in zip(single[1:], grouped[1:]):
        assert torch.equal(p, q[0]) and not q[1:].any()
    dw, dw4 = layer_mod.checkpoint_weight_grad(kept, ud, g[0], b[0]), layer_mod.checkpoint_weight_grad(kept, ud, g, b, acs)
    assert dw.shape == (96, 96) and torch.equal(dw, dw4[0]) and not dw4[1:].any()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("n,w", [(1, 1), (5, 7), (33, 31), (9, 64), (20, 128), (40, 129), (25, 256), (11, 500), (5, 1000), (3, 2050), (2, 4096)])
def test_activation_and_its_checkpoint(n, w, norm, act):
    x, gain, bias, up, acs = make(n, w, np.float32, "gaps", seed=act)
    gain, bias = (gain, bias) if norm else (None, None)
    a, kept = layer_mod.checkpoint_activation(dev(x), act, gain and dev(gain), bias and dev(bias), acs, EPS)
    codes, blocks = ref.encode(x)
    assert np.array_equal(kept.codes.cpu().numpy()[:, :w], codes) and np.array_equal(kept.blocks.cpu().numpy(), blocks)
    want, err, stats, stats_err = ref.activation(x, act, gain, bias, acs, EPS)
    near(a, want, err, "a")
    mean = rstd = None
    if norm:
        near(kept.mean, stats[0], stats_err[0], "mean")
        near(kept.rstd, stats[1], stats_err[1], "rstd")
        mean, rstd = kept.mean.cpu().numpy(), kept.rstd.cpu().numpy()
    got = layer_mod.checkpoint_activation_grad(kept, dev(up), gain and dev(gain), bias and dev(bias), acs)
    want, err = ref.activation_grad(codes, blocks, mean, rstd, act, up, gain, bias, acs)
    assert norm or got[2] is got[3] is None
    for name, g, v, e in zip(("dz", "dsum", "dgain", "dbias"), got, want, err):
        near(g, v, e, name)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("n,w", MANY)
def test_activation_of_many_rows(n, w, norm):
    x, gain, bias, up, acs = make(n, w, np.float32)
    gain, bias = (gain, bias) if norm else (None, None)
    a, kept = layer_mod.checkpoint_activation(dev(x), "celu", gain and dev(gain), bias and dev(bias), acs, EPS)
    codes, blocks = ref.encode(x)
    assert np.array_equal(kept.codes.cpu().numpy()[:, :w], codes) and np.array_equal(kept.blocks.cpu().numpy(), blocks)
    near(a, *ref.activation(x, "celu", gain, bias, acs, EPS)[:2])
    stats = (kept.mean.cpu().numpy(), kept.rstd.cpu().numpy()) if norm else (None, None)
    got = layer_mod.checkpoint_activation_grad(kept, dev(up), gain and dev(gain), bias and dev(bias), acs)
    want, err = ref.activation_grad(codes, blocks, *stats, "celu", up, gain, bias, acs)
    for name, g, v, e in zip(("dz", "dsum", "dgain", "dbias"), got, want, err):
        near(g, v, e, name)


def test_a_checkpoint_is_half_a_step_off_at_most():
    """And a block far from zero has all of its steps; a block of one value is that value."""
    x, *_ = make(50, 300, np.float32)
    x[:, 128:256] += 3e4
    x[4, :128] = -2.5
    _, kept = layer_mod.checkpoint_activation(dev(x), "celu")
    blocks = kept.blocks.cpu().numpy()
    back = ref.decode(kept.codes.cpu().numpy()[:, :300], blocks)
    step = blocks[:, np.arange(300) // 128, 1].astype(ref.LD)
    # code - (z - base) / step: the two roundings of the product with 1 / step, 255 steps at most, then half a step
    assert (np.abs(back - x) <= step * (0.5 + 256 * 4 * ref.U(np.float32))).all()
    assert (blocks[4, 0] == [-2.5, 0.0]).all() and (back[4, :128] == -2.5).all()
    assert (kept.codes.cpu().numpy()[:, 128:256].max(1) == 255).all()


def test_what_is_not_finite_stays_in_its_block():
    x, gain, bias, up, acs = make(12, 384, np.float32)
    x[2, 130], x[5, 0], x[7, 383], x[8, 140], x[8, 141] = np.nan, np.inf, -np.inf, 3e38, -3e38
    a, kept = layer_mod.checkpoint_activation(dev(x), "softplus")
    codes, blocks = ref.encode(x)
    assert np.array_equal(kept.blocks.cpu().numpy(), blocks, equal_nan=True)
    bad = np.isnan(blocks[:, :, 0])
    assert bad.sum() == 4 and bad[2, 1] and bad[5, 0] and bad[7, 2] and bad[8, 1]
    dz = layer_mod.checkpoint_activation_grad(kept, dev(up))[0].cpu().numpy()
    columns = np.repeat(bad, 128, 1)
    assert np.isnan(dz[columns]).all() and np.isfinite(dz[~columns]).all()
    assert np.isnan(a.cpu().numpy()[2, 130]) and np.isfinite(a.cpu().numpy()[8, 140])
    # with a norm the row is lost, as its output is, and no other row is
    a, kept = layer_mod.checkpoint_activation(dev(x), "softplus", dev(gain), dev(bias), acs)
    dz = layer_mod.checkpoint_activation_grad(kept, dev(up), dev(gain), dev(bias), acs)[0].cpu().numpy()
    assert np.isnan(dz[[2, 5, 7, 8]]).all() and np.isfinite(np.delete(dz, [2, 5, 7, 8], 0)).all()


def test_tiny_and_huge_values():
    x = np.zeros((6, 128), np.float32)
    x[0] = np.linspace(-1e-38, 1e-38, 128)
    x[1] = np.linspace(0, 1e-27, 128)
    x[2] = np.linspace(-1e38, 1e38, 128)
    x[3, ::2] = 1e-40
    x[4] = np.linspace(1e30, 1.0000001e30, 128)
    _, kept = layer_mod.checkpoint_activation(dev(x), "gaussian")
    codes, blocks = ref.encode(x)
    assert np.array_equal(kept.codes.cpu().numpy(), codes) and np.array_equal(kept.blocks.cpu().numpy(), blocks)
    assert (blocks[[0, 3, 5], 0, 1] == 0).all() and codes[1].max() == 255 and codes[2].max() == 255


WGRAD = [(1, 1, 1), (3, 2, 5), (17, 7, 1), (40, 33, 19), (64, 128, 128), (130, 97, 64), (257, 130, 129), (100, 384, 128),
         (33, 260, 300), (700, 64, 8), (2000, 128, 64), (5003, 200, 33), (31, 1000, 17), (40, 17, 1001), (9, 4096, 3), (9, 3, 4096)]


@pytest.mark.parametrize("norm,act", [(False, "celu"), (True, "celu"), (True, "gaussian"), (False, "normal"), (True, "softplus")])
@pytest.mark.parametrize("n,w,out", WGRAD)
def test_weight_gradient(n, w, out, norm, act):
    for kind in ("mixed", "gaps"):
        x, gain, bias, _, acs = make(n, w, np.float32, kind, seed=out)
        dz = (rng_of(n, w, out, "dz").standard_normal((n, out)) * 1e-2).astype(np.float32)
        gain, bias = (gain, bias) if norm else (None, None)
        _, kept = layer_mod.checkpoint_activation(dev(x), act, gain and dev(gain), bias and dev(bias), acs, EPS)
        kept.codes[:, w:] = 255      # bytes behind the width mean nothing
        stats = (kept.mean.cpu().numpy(), kept.rstd.cpu().numpy()) if norm else (None, None)
        dw = layer_mod.checkpoint_weight_grad(kept, dev(dz), gain and dev(gain), bias and dev(bias), acs)
        want, err = ref.weight_grad(kept.codes.cpu().numpy()[:, :w], kept.blocks.cpu().numpy(), *stats, act, dz, gain, bias, acs)
        near(dw, want, err, "dw")


def test_weight_gradient_is_as_exact_as_float32_products():
    """Relative error in the 2-norm: a plain float32 product of 20,000 rows is off by about 5e-7, tf32 products by 3e-4."""
    x, gain, bias, _, acs = make(20000, 256, np.float32)
    dz = (rng_of("exact").standard_normal((20000, 192)) * 1e-2).astype(np.float32)
    _, kept = layer_mod.checkpoint_activation(dev(x), "celu", dev(gain), dev(bias), acs, EPS)
    dw = layer_mod.checkpoint_weight_grad(kept, dev(dz), dev(gain), dev(bias), acs).double()
    z = kept.blocks.double()[:, torch.arange(256) // 128, 0] + kept.codes.double() * kept.blocks.double()[:, torch.arange(256) // 128, 1]
    xhat = (z - kept.mean.double()[:, None]) * kept.rstd.double()[:, None]
    for t, rows in enumerate(ref.element_rows(acs)):
        u = xhat[rows] * dev(gain)[t].double() + dev(bias)[t].double()
        a = torch.where(u >= 0, u, 0.1 * torch.expm1(10 * u.clamp(max=0)))
        want = a.T @ dev(dz)[rows].double()
        assert float((dw[t] - want).norm() / want.norm()) < 2e-6


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_weight_gradient_shows_what_is_not_finite(bad):
    x, _, _, up, acs = make(50, 64, np.float32)
    _, kept = layer_mod.checkpoint_activation(dev(x), "celu", acs=acs)
    up[acs[0] + 2, 5] = bad
    dw = layer_mod.checkpoint_weight_grad(kept, dev(up), acs=acs).cpu().numpy()
    assert not np.isfinite(dw[1, :, 5]).any() and np.isfinite(np.delete(dw[1], 5, 1)).all() and np.isfinite(dw[[0, 2, 3]]).all()


def test_no_rows():
    g = [torch.ones(24, device=DEV)] * 4
    none, acs = torch.zeros((0, 24), device=DEV), np.zeros(4, np.int32)
    y, mean, rstd = layer_mod.layer_norm(none, g, g, acs)
    assert y.shape == (0, 24) and mean.shape == rstd.shape == (0,)
    dx, dg, db = layer_mod.layer_norm_grad(none, none, g, mean, rstd, acs)
    assert dx.shape == (0, 24) and not dg.any() and not db.any()
    a, kept = layer_mod.checkpoint_activation(none, "celu", g, g, acs)
    dz, *s = layer_mod.checkpoint_activation_grad(kept, none, g, g, acs)
    assert dz.shape == (0, 24) and all(t.shape == (4, 24) and not t.any() for t in s)
    dw = layer_mod.checkpoint_weight_grad(kept, torch.zeros((0, 5), device=DEV), g, g, acs)
    assert dw.shape == (4, 24, 5) and not dw.any()
    assert not layer_mod.checkpoint_weight_grad(kept, torch.zeros((0, 5), device=DEV), g[0], g[0]).any()


def everything(x, up, dz, gain, bias, acs):
    y, mean, rstd = layer_mod.layer_norm(x, gain, bias, acs, EPS)
    a, kept = layer_mod.checkpoint_activation(x, "celu", gain, bias, acs, EPS)
    b, flat = layer_mod.checkpoint_activation(x, "normal")
    return [y, mean, rstd, *layer_mod.layer_norm_grad(up, x, gain, mean, rstd, acs), a, kept.blocks, b,
            *layer_mod.checkpoint_activation_grad(kept, up, gain, bias, acs), layer_mod.checkpoint_activation_grad(flat, up)[0],
            layer_mod.checkpoint_weight_grad(kept, dz, gain, bias, acs), layer_mod.checkpoint_weight_grad(flat, dz)]


def inputs(n, w, out, seed):
    x, gain, bias, up, acs = make(n, w, np.float32, seed=seed)
    return [dev(x), dev(up), dev(rng_of(seed, "dz").standard_normal((n, out)).astype(np.float32)), dev(gain), dev(bias), acs]


@pytest.mark.parametrize("n,w,out", [(40, 128, 64), (6000, 128, 128), (3000, 600, 140)])
def test_results_do_not_change_from_run_to_run(n, w, out):
    args = inputs(n, w, out, 1)
    first = everything(*args)
    for _ in range(3):
        for p, q in zip(first, everything(*args)):
            assert torch.equal(p, q)


def test_captured_graphs_replay_on_new_inputs():
    """Two graphs of different sizes, replayed in turns with inputs that change between the replays; then the eager calls
    once more."""
    cases = [inputs(5000, 128, 64, 2), inputs(3000, 300, 130, 3)]
    new = [inputs(5000, 128, 64, 4), inputs(3000, 300, 130, 5)]
    eager = [[everything(*a), everything(*b)] for a, b in zip(cases, new)]
    graphs, outs = [], []
    for a in cases:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(everything(*a))
        graphs.append(g)
    for turn in range(2):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for k in range(2):
            for p, q in zip(outs[k], eager[k][turn]):
                assert torch.equal(p, q)
            for p, q in zip(cases[k][:3], new[k][:3]):
                p.copy_(q)
            for p, q in zip(cases[k][3] + cases[k][4], new[k][3] + new[k][4]):
                p.copy_(q)
    for k in range(2):
        for p, q in zip(everything(*new[k]), eager[k][1]):
            assert torch.equal(p, q)


def test_calls_on_several_streams():
    cases = [inputs(4000 + 500 * k, 128, 64, 10 + k) for k in range(4)]
    want = [everything(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [None] * 4
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = everything(*cases[k])
    torch.cuda.synchronize()
    for p, q in zip(want, got):
        for a, b in zip(p, q):
            assert torch.equal(a, b)


def test_nothing_behind_the_rows_is_written():
    """The C entry points with outputs inside larger buffers."""
    lib, n, w, out = _lib.lib(), 77, 100, 30
    x, gain, bias, up, acs = make(n, w, np.float32)
    xd, ud, g, b = dev(x), dev(up), dev(gain), dev(bias)
    dz = torch.randn((n, out), device=DEV)
    four = lambda ts: (ctypes.c_void_p * 4)(*[t.data_ptr() for t in ts])  # noqa: E731
    counts = acs.ctypes.data_as(_lib.c_int_p)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    guarded = []

    def room(*shape, dtype=torch.float32):
        size = int(np.prod(shape))
        t = torch.full((size + 256,), 77, dtype=dtype, device=DEV)
        guarded.append((t, size))
        return t

    y, mean, rstd, dx = room(n, w), room(n), room(n), room(n, w)
    assert lib.ani_layer_norm_f32(xd.data_ptr(), w, four(g), four(b), w, EPS, counts, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), stream) == 0
    sums = [[room(w) for _ in range(4)] for _ in range(5)]
    ws = room(max(4, lib.ani_layer_sums_workspace_bytes(w, counts, 3, 4)) // 4)
    assert lib.ani_layer_norm_grad_f32(ud.data_ptr(), w, xd.data_ptr(), w, four(g), mean.data_ptr(), rstd.data_ptr(), w, counts,
                                       dx.data_ptr(), four(sums[0]), four(sums[1]), ws.data_ptr(), stream) == 0
    a, codes, blocks = room(n, w), room(n, lib.ani_checkpoint_row_bytes(w), dtype=torch.uint8), room(n, lib.ani_checkpoint_blocks(w), 2)
    m2, r2 = room(n), room(n)
    assert lib.ani_checkpoint_activation_f32(xd.data_ptr(), w, four(g), four(b), w, EPS, 0, counts, a.data_ptr(), codes.data_ptr(),
                                             blocks.data_ptr(), m2.data_ptr(), r2.data_ptr(), stream) == 0
    dzz = room(n, w)
    assert lib.ani_checkpoint_activation_grad_f32(codes.data_ptr(), blocks.data_ptr(), m2.data_ptr(), r2.data_ptr(), ud.data_ptr(), w,
                                                  four(g), four(b), w, 0, counts, dzz.data_ptr(), four(sums[2]), four(sums[3]),
                                                  four(sums[4]), ws.data_ptr(), stream) == 0
    dw = [room(w, out) for _ in range(4)]
    ww = room(max(4, lib.ani_checkpoint_weight_grad_workspace_bytes(w, out, counts)) // 4)
    assert lib.ani_checkpoint_weight_grad_f32(codes.data_ptr(), blocks.data_ptr(), m2.data_ptr(), r2.data_ptr(), four(g), four(b), w, 0,
                                              dz.data_ptr(), out, out, counts, four(dw), ww.data_ptr(), stream) == 0
    torch.cuda.synchronize()
    for t, size in guarded:
        assert (t[size:] == 77).all()


def test_offsets_beyond_31_bits():
    """More than 2^31 values: the last rows of every output, against a call on those rows alone; the sums over rows, whose
    other rows are zero but for the last."""
    n, w, out, tail = 530_000, 4096, 8, 40
    assert n * w > 2 ** 31
    small = rng_of("offsets").standard_normal((tail, w)).astype(np.float32)
    gain, bias = torch.rand(w, device=DEV) + 0.5, torch.rand(w, device=DEV) - 0.5
    x = torch.zeros((n, w), device=DEV)
    x[-tail:] = dev(small)
    y, mean, rstd = layer_mod.layer_norm(x, gain, bias)
    for got, want in zip((y, mean, rstd), layer_mod.layer_norm(dev(small), gain, bias)):
        assert torch.equal(got[-tail:], want)
    up = torch.zeros((n, w), device=DEV)
    up[-tail:] = dev(small) * 1e-2
    small_up = up[-tail:].clone()
    dx, dgain, dbias = layer_mod.layer_norm_grad(up, x, gain, mean, rstd)
    want = layer_mod.layer_norm_grad(small_up, dev(small), gain, mean[-tail:].clone(), rstd[-tail:].clone())
    assert torch.equal(dx[-tail:], want[0])
    # the same forty terms in another order: 40 roundings of their sum of magnitudes
    terms = small_up.abs().sum(0) * 40 * 6e-8
    assert ((dbias - want[2]).abs() <= terms).all() and ((dgain - want[1]).abs() <= terms * 8).all()
    del y, dx
    a, kept = layer_mod.checkpoint_activation(x, "celu", gain, bias)
    small_a, small_kept = layer_mod.checkpoint_activation(dev(small), "celu", gain, bias)
    assert torch.equal(a[-tail:], small_a) and torch.equal(kept.codes[-tail:], small_kept.codes) and torch.equal(kept.blocks[-tail:], small_kept.blocks)
    del a, x
    dz, dsum, _, _ = layer_mod.checkpoint_activation_grad(kept, up, gain, bias)
    small_dz, small_dsum, _, _ = layer_mod.checkpoint_activation_grad(small_kept, small_up, gain, bias)
    assert torch.equal(dz[-tail:], small_dz) and ((dsum - small_dsum).abs() <= small_dz.abs().sum(0) * 40 * 6e-8).all()
    dz_out = torch.zeros((n, out), device=DEV)
    dz_out[-tail:] = small_up[:, :out]
    dw = layer_mod.checkpoint_weight_grad(kept, dz_out, gain, bias)
    want = layer_mod.checkpoint_weight_grad(small_kept, small_up[:, :out].contiguous(), gain, bias)
    # |activations| <= 6: xhat is below 5 and the bias below 1; two products of forty rows, each 2^-21 and 40 roundings off
    assert ((dw - want).abs() <= 2 * (2.0 ** -21 + 80 * 6e-8) * 10 * small_up[:, :out].abs().sum(0)).all()


def test_elements_that_share_their_gain():
    """The same tensor for all elements: the gradient is the sum over all rows."""
    torch.manual_seed(5)
    x = torch.randn((50, 20), dtype=torch.float64, device=DEV, requires_grad=True)
    g, b = (torch.randn(20, dtype=torch.float64, device=DEV, requires_grad=True) for _ in range(2))
    up = torch.randn((50, 20), dtype=torch.float64, device=DEV)
    y = layer_mod.layer_norm_autograd(x, [g] * 4, [b] * 4, np.array([20, 10, 0, 20], np.int32))
    grouped = torch.autograd.grad(y, (x, g, b), up)
    alone = torch.autograd.grad(layer_mod.layer_norm_autograd(x, g, b), (x, g, b), up)
    assert torch.equal(grouped[0], alone[0])
    for p, q in zip(grouped[1:], alone[1:]):
        assert torch.allclose(p, q, rtol=0, atol=1e-13 * float(up.abs().sum()))


@pytest.mark.parametrize("norm", [False, True])
def test_a_checkpoint_made_of_its_parts(norm):
    x, gain, bias, up, acs = make(70, 150, np.float32)
    g, b = (dev(gain), dev(bias)) if norm else (None, None)
    _, kept = layer_mod.checkpoint_activation(dev(x), layer_mod.activations.softplus, g, b, acs)
    parts = layer_mod.ActivationCheckpoint(kept.codes.clone(), kept.blocks.clone(), 150, "softplus", *([kept.mean.clone(), kept.rstd.clone()] if norm else []))
    assert kept.nbytes == parts.nbytes == 70 * (160 + 2 * 8 + (8 if norm else 0)) and (kept.mean is None) != norm
    for p, q in zip(layer_mod.checkpoint_activation_grad(kept, dev(up), g, b, acs), layer_mod.checkpoint_activation_grad(parts, dev(up), g, b, acs)):
        assert p is q is None or torch.equal(p, q)
    dz = dev(up)[:, :33]
    assert torch.equal(layer_mod.checkpoint_weight_grad(kept, dz, g, b, acs), layer_mod.checkpoint_weight_grad(parts, dz, g, b, acs))


def test_counts_in_other_forms():
    x, gain, bias, up, acs = make(30, 24, np.float32)
    want = layer_mod.layer_norm(dev(x), dev(gain), dev(bias), acs)
    for form in (acs.tolist(), acs.astype(np.int64), torch.from_numpy(acs).to(DEV), tuple(dev(gain)) and acs[::1].copy()):
        for p, q in zip(want, layer_mod.layer_norm(dev(x), tuple(dev(gain)), dev(bias), form)):
            assert torch.equal(p, q)


# ---------------------------------------------------------------- autograd
def test_layer_norm_autograd_against_differences():
    torch.manual_seed(3)
    acs = np.array([3, 0, 2, 1], np.int32)
    x = torch.randn((6, 5), dtype=torch.float64, device=DEV, requires_grad=True)
    params = [torch.randn(5, dtype=torch.float64, device=DEV, requires_grad=True) for _ in range(8)]
    fn = lambda x, *p: layer_mod.layer_norm_autograd(x, list(p[:4]), list(p[4:]), acs, 1e-3)  # noqa: E731
    assert torch.autograd.gradcheck(fn, (x, *params))
    assert torch.autograd.gradgradcheck(fn, (x, *params))
    alone = lambda x, g, b: layer_mod.layer_norm_autograd(x, g, b, eps=1e-3)  # noqa: E731
    assert torch.autograd.gradcheck(alone, (x, params[0], params[1]))


def test_activation_gradient_against_differences():
    """The gradient is that of the activation at the point that the checkpoint stands for: differences of the plain formula
    there, in float64."""
    x, gain, bias, up, acs = make(7, 40, np.float32)
    for act in ACTS:
        _, kept = layer_mod.checkpoint_activation(dev(x), act, acs=acs)
        dz = layer_mod.checkpoint_activation_grad(kept, dev(up), acs=acs)[0].cpu().numpy()
        z = ref.decode(kept.codes.cpu().numpy()[:, :40], kept.blocks.cpu().numpy())
        h = ref.LD(1e-7)
        slope = (ref.act(act, z + h)[0] - ref.act(act, z - h)[0]) / (2 * h)
        # a difference over the kink of celu's slope is off by 10 h at most, elsewhere by h^2 times the third derivative
        near(torch.from_numpy(dz), up * slope, np.abs(up) * (20 * h + 40 * ref.U(np.float32)) + 1e-12)


# ---------------------------------------------------------------- refusals
def test_refusals():
    x, gain, bias, up, acs = make(10, 16, np.float32)
    xd, ud, g, b = dev(x), dev(up), dev(gain), dev(bias)
    with pytest.raises(ValueError, match="acs counts"):
        layer_mod.layer_norm(xd, g, b, np.array([1, 1, 1, 1], np.int32))
    with pytest.raises(ValueError, match="list of four"):
        layer_mod.layer_norm(xd, g[0], b[0], acs)
    with pytest.raises(ValueError, match="a list of four goes with acs"):
        layer_mod.layer_norm(xd, g, b)
    with pytest.raises(ValueError, match="one per column"):
        layer_mod.layer_norm(xd, g[0][:5], b[0])
    with pytest.raises(TypeError, match="gain is torch.float64"):
        layer_mod.layer_norm(xd, g[0].double(), b[0])
    with pytest.raises(TypeError, match="float32 and float64"):
        layer_mod.layer_norm(xd.half(), g[0].half(), b[0].half())
    with pytest.raises(ValueError, match="4096"):
        layer_mod.layer_norm(torch.zeros((2, 4097), device=DEV), torch.ones(4097, device=DEV), torch.ones(4097, device=DEV))
    with pytest.raises(ValueError):
        layer_mod.layer_norm(xd[0], g[0], b[0])
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(_lib.AniError):
            layer_mod.layer_norm(xd, g[0], b[0], eps=eps)
    _, mean, rstd = layer_mod.layer_norm(xd, g[0], b[0])
    with pytest.raises(ValueError, match="one per row"):
        layer_mod.layer_norm_grad(ud, xd, g[0], mean[:3], rstd)
    with pytest.raises(ValueError, match="grad_y is"):
        layer_mod.layer_norm_grad(ud[:4], xd, g[0], mean, rstd)
    with pytest.raises(TypeError):
        layer_mod.checkpoint_activation(xd.double(), "celu")
    with pytest.raises(ValueError, match="activation"):
        layer_mod.checkpoint_activation(xd, "relu")
    with pytest.raises(ValueError, match="together"):
        layer_mod.checkpoint_activation(xd, "celu", g[0])
    _, kept = layer_mod.checkpoint_activation(xd, "celu")
    _, normed = layer_mod.checkpoint_activation(xd, "celu", g[0], b[0])
    with pytest.raises(ValueError, match="gain and bias go with"):
        layer_mod.checkpoint_activation_grad(kept, ud, g[0], b[0])
    with pytest.raises(ValueError, match="gain and bias go with"):
        layer_mod.checkpoint_weight_grad(normed, ud)
    with pytest.raises(ValueError, match="does not fit"):
        layer_mod.checkpoint_activation_grad(kept, ud[:, :8])
    with pytest.raises(ValueError, match="does not fit"):
        layer_mod.checkpoint_weight_grad(kept, ud[:4])
    with pytest.raises(ValueError, match="not a checkpoint"):
        layer_mod.checkpoint_weight_grad(layer_mod.ActivationCheckpoint(kept.codes, kept.blocks, 40, "celu"), ud)
    with pytest.raises(ValueError, match="CUDA"):
        layer_mod.checkpoint_weight_grad(layer_mod.ActivationCheckpoint(kept.codes.cpu(), kept.blocks.cpu(), 16, "celu"), ud)
    with pytest.raises(ValueError, match="CUDA"):
        layer_mod.checkpoint_activation_grad(kept, ud.cpu())


def test_second_derivatives_of_norms_that_share_parameters():
    from test_layers import check_shared_norms
    check_shared_norms(DEV)


def test_second_derivatives_against_differences_with_a_shared_gain():
    torch.manual_seed(4)
    acs = np.array([3, 0, 2, 1], np.int32)
    x = torch.randn((6, 5), dtype=torch.float64, device=DEV, requires_grad=True)
    g, b = (torch.randn(5, dtype=torch.float64, device=DEV, requires_grad=True) for _ in range(2))
    fn = lambda x, g, b: layer_mod.layer_norm_autograd(torch.tanh(layer_mod.layer_norm_autograd(x, g, b, eps=1e-3)), [g] * 4, [b, b, g, b], acs, 1e-3)  # noqa: E731
    assert torch.autograd.gradcheck(fn, (x, g, b))
    assert torch.autograd.gradgradcheck(fn, (x, g, b))


@pytest.mark.parametrize("w,kept_rows,normed,given_rows", [(16, 4, False, 3), (16, 3, True, 4), (7, 40, False, 30), (128, 18, False, 17), (200, 28, True, 29)])
def test_a_checkpoint_of_other_rows_is_refused(w, kept_rows, normed, given_rows):
    """As many bytes as one of given_rows rows with a norm where it has none, or without one where it has: told apart by what
    the checkpoint is, not by its size."""
    size = lambda n, norm: n * (-(-w // 16) * 16 + 8 * -(-w // 128) + (8 if norm else 0))  # noqa: E731
    x, gain, bias, up, _ = make(kept_rows, w, np.float32)
    g = (dev(gain[0]), dev(bias[0]))
    _, kept = layer_mod.checkpoint_activation(dev(x), "celu", *(g if normed else ()))
    assert kept.nbytes == size(kept_rows, normed) == size(given_rows, not normed)
    for params in (g, ()):
        for rows in (given_rows, kept_rows, kept_rows + 1):
            if rows == kept_rows and normed == bool(params):
                continue
            grad = torch.ones((rows, w), device=DEV)
            for call in (layer_mod.checkpoint_activation_grad, layer_mod.checkpoint_weight_grad):
                with pytest.raises(ValueError, match="gain and bias go with" if normed != bool(params) else "does not fit"):
                    call(kept, grad, *params)


@pytest.mark.parametrize("act", ["celu", "gaussian"])
@pytest.mark.parametrize("n,w", [(5, 16), (3, 5), (40, 32), (9, 97), (6, 128), (11, 260), (5, 513), (3, 1024), (2, 2050)])
def test_columns_and_rows_that_are_not_there_add_nothing(n, w, act):
    """Rows of one large value, whose mean times 1 / sqrt(eps) is beyond float32: zero minus that mean is not a column's xhat,
    neither behind the width nor behind the last row.  Every column's own xhat is 0, so all is as for rows of zeros."""
    x, gain, bias, up, acs = make(n, w, np.float32, "gaps", seed=act)
    g, b = dev(gain), dev(bias)
    codes = torch.zeros((n, -(-w // 16) * 16), dtype=torch.uint8, device=DEV)
    blocks = torch.zeros((n, -(-w // 128), 2), device=DEV)
    mean, rstd = torch.zeros(n, device=DEV), torch.full((n,), EPS ** -0.5, device=DEV)
    want = layer_mod.checkpoint_activation_grad(layer_mod.ActivationCheckpoint(codes, blocks, w, act, mean, rstd), dev(up), g, b, acs)
    assert all(torch.isfinite(t).all() for t in want)
    value = 2.0 ** 123
    blocks, mean = blocks.clone(), torch.full((n,), value, device=DEV)
    blocks[:, :, 0] = value
    got = layer_mod.checkpoint_activation_grad(layer_mod.ActivationCheckpoint(codes, blocks, w, act, mean, rstd), dev(up), g, b, acs)
    for p, q in zip(got, want):
        assert torch.equal(p, q)
    # bytes behind the width mean nothing, whatever their step
    codes, blocks = codes.clone(), blocks.clone()
    codes[:, w:] = 255
    blocks[:, :, 0], blocks[:, :, 1], mean = 0.0, 2.0 ** 119, torch.zeros(n, device=DEV)
    got = layer_mod.checkpoint_activation_grad(layer_mod.ActivationCheckpoint(codes, blocks, w, act, mean, rstd), dev(up), g, b, acs)
    for p, q in zip(got, want):
        assert torch.equal(p, q)


def test_activation_of_constant_rows_of_a_large_value():
    """The same from the forward pass on: a constant row is its bias, and its gradient that of a row of zeros."""
    x, gain, bias, up, acs = make(5, 16, np.float32)
    results = []
    for value in (2.0 ** 123, 0.0):
        a, kept = layer_mod.checkpoint_activation(torch.full((5, 16), value, device=DEV), "softplus", dev(gain), dev(bias), acs, EPS)
        results.append((a, *layer_mod.checkpoint_activation_grad(kept, dev(up), dev(gain), dev(bias), acs)))
    for p, q in zip(*results):
        assert torch.isfinite(q).all() and torch.equal(p, q)


# rows, width, out, norm, activation: ranges of a few hundred rows; widths whose rows are copied value by value; one column;
# so many tiles that an element of 5,000 rows is one range, with one accumulator for all of its small products
EXACT = [(20000, 256, 192, True, "celu"), (20000, 256, 192, False, "softplus"), (20000, 256, 97, True, "softplus"), (13750, 64, 1, False, "celu"),
         (13750, 128, 128, True, "gaussian"), (20000, 1700, 1700, True, "celu"), (20000, 1700, 1601, False, "softplus")]


@pytest.mark.parametrize("n,w,out,norm,act", EXACT)
def test_weight_gradient_over_long_sums(n, w, out, norm, act):
    """Relative error in the 2-norm, below 7e-7.  What is expected of it:
      the tensor core cuts a sum off at its last place, by half a place in the mean: 2^-24 / m of a sum with mantissa m, 4.3e-8
      over the mantissas.  A chain of 128 rows is 16 such sums; the i-th is i / 16 of the last, seen along it (terms of either
      sign): 8.5 * 4.3e-8 = 3.7e-7, always towards zero.  (A chain over a range of 544 rows: 1.5e-6; over 5,000: 1.4e-5.)
      The small products have one chain for a range, but are 2^-11 of the sum: 5,000 rows 1e-8.
      What the parts leave out, low times low and the low parts' own last places: 1e-7.
      Activations: an exponential of 2^-22, a reciprocal and up to ten roundings, 2e-7 of their root mean square at most.
    Together (square root of the sum of squares) 4.3e-7."""
    x, gain, bias, _, acs = make(n, w, np.float32, seed=out)
    dz = dev((rng_of("long", n, w, out).standard_normal((n, out)) * 1e-2).astype(np.float32))
    g, b = (dev(gain), dev(bias)) if norm else (None, None)
    _, kept = layer_mod.checkpoint_activation(dev(x), act, g, b, acs)
    dw = layer_mod.checkpoint_weight_grad(kept, dz, g, b, acs).double()
    blocks = kept.blocks.double()[:, torch.arange(w) // 128]
    z = blocks[:, :, 0] + kept.codes[:, :w].double() * blocks[:, :, 1]
    for t, rows in enumerate(ref.element_rows(acs)):
        u = z[rows]
        if norm:
            u = (u - kept.mean.double()[rows, None]) * kept.rstd.double()[rows, None] * g[t].double() + b[t].double()
        if act == "celu":
            a = torch.where(u >= 0, u, 0.1 * torch.expm1(10 * u.clamp(max=0)))
        elif act == "gaussian":
            a = torch.exp(-u * u)
        else:
            a = u.clamp(min=0) + torch.log1p(torch.exp(-u.abs())) - 0.69314718056
        want = a.T @ dz[rows].double()
        off = float((dw[t] - want).norm() / want.norm())
        assert off < 7e-7

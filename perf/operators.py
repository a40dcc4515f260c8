"""Operators of normalised layers of the atomic networks: layer norm with its gradients, activations whose input is kept in
8 bits for the backward pass, and the weight gradient of the next layer from such a checkpoint.

Rows are atoms sorted by element (H, C, N, O), ``acs`` counts them, every element has its own gain, bias and weights.

  norm         y = gain (x - mean) / sqrt(var + eps) + bias, and the row's mean and 1 / sqrt(var + eps)
  norm_grad    dx, dgain, dbias from dy, x, mean and 1 / sqrt(var + eps)
  activation   a = act(z) or act(norm(z)), with z kept as one byte a value (and a base and a step for each row and block of 128
               columns), then dz, its column sums (and dgain, dbias) from da and what was kept
  weight_grad  dW = sum over an element's atoms of act(...)^T dz, the activations recomputed from the bytes

The bytes are defined by float32 operations: base = min, step = (max - min) * (1 / 255), byte = rint((z - base) * (1 / step));
a block whose step is below 1e-30 is its base.
"""
import numpy as np
import torch

own = False

EPS = 1e-5
BLOCK = 128
ACTIVATIONS = ("celu", "gaussian", "normal", "softplus")


def _counts(n):
    """Atoms per element of organic molecules: about half hydrogen; small batches lack elements."""
    o, nit = n // 13, n // 9
    c = (n - o - nit) * 2 // 5
    return [n - o - nit - c, c, nit, o]


def listed():
    # 1024 molecules of the training set are 13,750 atoms, 8192 are 110,000; hidden layers are 128 and 64 wide, features 384
    return [
        # one molecule, as the energy server evaluates it: latency
        dict(name="norm one molecule", kind="norm", n=20, w=128, f64=False),
        # the features of a training batch
        dict(name="norm batch", kind="norm", n=13750, w=384, f64=False),
        # a network in double precision, an odd width
        dict(name="norm double odd", kind="norm", n=5003, w=97, f64=True),
        # a hidden layer of a training batch
        dict(name="norm grad batch", kind="norm_grad", n=13750, w=128, f64=False),
        # the largest batch, wide layer
        dict(name="norm grad large", kind="norm_grad", n=110000, w=512, f64=False),
        # training in double precision
        dict(name="norm grad double", kind="norm_grad", n=13750, w=128, f64=True),
        # a few molecules, normalised layer: latency of a small training step
        dict(name="activation small", kind="activation", n=150, w=128, act="celu", norm=True),
        # a hidden layer of a training batch, not normalised
        dict(name="activation batch", kind="activation", n=13750, w=128, act="celu", norm=False),
        # a wide normalised layer of the largest batch
        dict(name="activation large", kind="activation", n=110000, w=512, act="softplus", norm=True),
        # the output layer: one column
        dict(name="weights output layer", kind="weight_grad", n=13750, w=64, out=1, act="celu", norm=False),
        # a hidden layer of a training batch
        dict(name="weights batch", kind="weight_grad", n=13750, w=128, out=128, act="celu", norm=True),
        # a wide layer of the largest batch
        dict(name="weights large", kind="weight_grad", n=110000, w=512, out=512, act="celu", norm=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(float(np.exp(rng.uniform(np.log(lo), np.log(hi))))))


def draw(rng):
    kind = rng.choice(("norm", "norm_grad", "activation", "weight_grad"))
    norm = kind in ("norm", "norm_grad") or rng.random() < 0.5
    # a norm over a handful of columns has a gradient that is almost nothing but rounding: networks have wider layers
    w = _log_uniform(rng, 8 if norm else 1, 1500)
    most = 25_000_000 // w
    case = dict(kind=kind, w=w)
    if kind in ("norm", "norm_grad"):
        case["f64"] = rng.random() < 0.4
    else:
        case["act"], case["norm"] = rng.choice(ACTIVATIONS), norm
    if kind == "weight_grad":
        case["out"] = _log_uniform(rng, 1, 1000)
        most = min(most, 25_000_000_000 // (w * case["out"]), 25_000_000 // case["out"])
    case["n"] = _log_uniform(rng, 1, min(110_000, most))
    return case


def _ranges(acs):
    ends = np.cumsum(acs)
    return [(int(e - c), int(e)) for e, c in zip(ends, acs)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1009 + 17)
    n, w, kind = case["n"], case["w"], case["kind"]
    dt = torch.float64 if case.get("f64") else torch.float32

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    # rows as a dense layer leaves them: columns of different spread around different offsets
    x = normal(n, w) * (0.4 + normal(w).abs()) + 0.5 * normal(w)
    state = dict(case=case, acs=np.array(_counts(n), dtype=np.int32), x=x,
                 gains=[1.0 + 0.2 * normal(w) for _ in range(4)], biases=[0.2 * normal(w) for _ in range(4)])
    if kind == "norm_grad":
        state["grad"] = normal(n, w) * 1e-2
        x64 = x.double()
        mean = x64.mean(1)
        state["mean"] = mean.to(dt)
        state["rstd"] = ((x64 - mean[:, None]).square().mean(1) + EPS).rsqrt().to(dt)
    if kind == "activation":
        state["grad"] = normal(n, w) * 1e-2
    if kind == "weight_grad":
        state["grad"] = normal(n, case["out"]) * 1e-2
        # what the forward pass kept: bytes in rows of a multiple of 16, (base, step) for each block, the row's statistics
        base, step, codes = _encode(x)
        state["codes"] = torch.zeros((n, -(-w // 16) * 16), dtype=torch.uint8, device="cuda")
        state["codes"][:, :w] = codes.to(torch.uint8)
        state["blocks"] = torch.stack([base, step], dim=2).contiguous()
        x64 = x.double()
        mean = x64.mean(1)
        state["mean"] = mean.float()
        state["rstd"] = ((x64 - mean[:, None]).square().mean(1) + EPS).rsqrt().float()
        del state["x"]
    if not case.get("norm", True):
        for k in ("gains", "biases", "mean", "rstd"):
            state.pop(k, None)
    return state


# ---------------------------------------------------------------- plain forms
def _statistics(x):
    mean = x.mean(1, keepdim=True)
    d = x - mean
    return mean, 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)


def _norm(x, gain, bias):
    mean, rstd = _statistics(x)
    return (x - mean) * rstd * gain + bias, mean[:, 0], rstd[:, 0]


def _norm_grad(grad, xhat, rstd, gain):
    g = grad * gain
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return dx, (grad * xhat).sum(0), grad.sum(0)


def _encode(z):
    """(base, step) of every row and block of columns, and the values' bytes (as float32)."""
    n, w = z.shape
    blocks = -(-w // BLOCK)
    full = torch.cat([z, z[:, -1:].expand(n, blocks * BLOCK - w)], 1).view(n, blocks, BLOCK)
    base = full.amin(2)
    step = (full.amax(2) - base) * (1.0 / 255.0)     # the scalar as float32
    small = step < 1e-30
    inv = torch.where(small, torch.zeros_like(step), torch.reciprocal(step))
    step = torch.where(small, torch.zeros_like(step), step)
    codes = torch.round((full - base[:, :, None]) * inv[:, :, None]).clamp(max=255.0)
    return base, step, codes.view(n, blocks * BLOCK)[:, :w]


def _decode(base, step, codes):
    w = codes.shape[1]
    per_column = [t.repeat_interleave(BLOCK, dim=1)[:, :w] for t in (base, step)]
    return per_column[0] + codes * per_column[1]


def _act(u, act):
    if act == "celu":
        return torch.where(u >= 0, u, 0.1 * (torch.exp(torch.clamp(u, max=0.0) / 0.1) - 1.0))
    if act == "gaussian":
        return torch.exp(-u * u)
    if act == "normal":
        return torch.exp(-0.5 * u * u)
    return torch.clamp(u, min=0.0) + torch.log1p(torch.exp(-u.abs())) - 0.69314718056


def _act_grad(u, act):
    if act == "celu":
        return torch.where(u >= 0, torch.ones_like(u), torch.exp(torch.clamp(u, max=0.0) / 0.1))
    if act == "gaussian":
        return -2.0 * u * torch.exp(-u * u)
    if act == "normal":
        return -u * torch.exp(-0.5 * u * u)
    return 1.0 / (1.0 + torch.exp(-u))


def _plain_activation(z, grad, act, gain, bias):
    base, step, codes = _encode(z)
    kept = _decode(base, step, codes)
    if gain is None:
        dz = grad * _act_grad(kept, act)
        return _act(z, act), dz, dz.sum(0)
    u, mean, rstd = _norm(z, gain, bias)
    xhat = (kept - mean[:, None]) * rstd[:, None]
    dz, dgain, dbias = _norm_grad(grad * _act_grad(xhat * gain + bias, act), xhat, rstd, gain)
    return _act(u, act), dz, dz.sum(0), dgain, dbias


def _plain(s):
    case, rows = s["case"], _ranges(s["acs"])
    kind, norm = case["kind"], case.get("norm", True)
    if kind == "norm":
        y, mean, rstd = zip(*[_norm(s["x"][a:b], s["gains"][t], s["biases"][t]) for t, (a, b) in enumerate(rows)])
        return {"y": torch.cat(y), "mean": torch.cat(mean), "rstd": torch.cat(rstd)}
    if kind == "norm_grad":
        dx, dgain, dbias = zip(*[
            _norm_grad(s["grad"][a:b], (s["x"][a:b] - s["mean"][a:b, None]) * s["rstd"][a:b, None], s["rstd"][a:b],
                       s["gains"][t]) for t, (a, b) in enumerate(rows)])
        return {"dx": torch.cat(dx), "dgain": torch.stack(dgain), "dbias": torch.stack(dbias)}
    if kind == "activation":
        out = list(zip(*[_plain_activation(s["x"][a:b], s["grad"][a:b], case["act"], s["gains"][t] if norm else None,
                                           s["biases"][t] if norm else None) for t, (a, b) in enumerate(rows)]))
        named = {"a": torch.cat(out[0]), "dz": torch.cat(out[1]), "dsum": torch.stack(out[2])}
        return {**named, "dgain": torch.stack(out[3]), "dbias": torch.stack(out[4])} if norm else named
    kept = _decode(s["blocks"][:, :, 0], s["blocks"][:, :, 1], s["codes"][:, :case["w"]].float())
    if norm:
        kept = (kept - s["mean"][:, None]) * s["rstd"][:, None]
    return {"dw": torch.stack([
        _act(kept[a:b] * s["gains"][t] + s["biases"][t] if norm else kept[a:b], case["act"]).T @ s["grad"][a:b]
        for t, (a, b) in enumerate(rows)])}


# ---------------------------------------------------------------- the framework's calls
def run(state):
    if not own:
        return _plain(state)
    from khan_b200 import layer_mod
    s, case = state, state["case"]
    gains, biases = s.get("gains"), s.get("biases")
    if case["kind"] == "norm":
        y, mean, rstd = layer_mod.layer_norm(s["x"], gains, biases, s["acs"], EPS)
        return {"y": y, "mean": mean, "rstd": rstd}
    if case["kind"] == "norm_grad":
        dx, dgain, dbias = layer_mod.layer_norm_grad(s["grad"], s["x"], gains, s["mean"], s["rstd"], s["acs"])
        return {"dx": dx, "dgain": dgain, "dbias": dbias}
    if case["kind"] == "activation":
        a, kept = layer_mod.checkpoint_activation(s["x"], case["act"], gains, biases, s["acs"], EPS)
        dz, dsum, dgain, dbias = layer_mod.checkpoint_activation_grad(kept, s["grad"], gains, biases, s["acs"])
        named = {"a": a, "dz": dz, "dsum": dsum}
        return {**named, "dgain": dgain, "dbias": dbias} if case["norm"] else named
    kept = layer_mod.ActivationCheckpoint(s["codes"], s["blocks"], case["w"], case["act"], s.get("mean"), s.get("rstd"))
    return {"dw": layer_mod.checkpoint_weight_grad(kept, s["grad"], gains, biases, s["acs"])}


def work(case):
    n, w, size = case["n"], case["w"], 8 if case.get("f64") else 4
    rows, stats, params = n * w, 2 * n * size, 4 * w * size
    kept = rows + 8 * n * -(-w // BLOCK)
    norm = case.get("norm", True)
    if case["kind"] == "norm":
        return {"bytes": 2 * rows * size + stats + 2 * params, "flops": 8 * rows}
    if case["kind"] == "norm_grad":
        return {"bytes": 3 * rows * size + stats + 3 * params, "flops": 14 * rows}
    if case["kind"] == "activation":
        # forward: z in, a and the checkpoint out; backward: da and the checkpoint in, dz out
        return {"bytes": 16 * rows + 2 * kept + params + (2 * stats + 4 * params if norm else 0),
                "flops": (50 if norm else 30) * rows}
    out = case["out"]
    return {"bytes": kept + 4 * n * out + 16 * w * out + (stats + 2 * params if norm else 0), "flops": 2 * rows * out}


# ---------------------------------------------------------------- 64 bits
def _exact_kept(codes, base, step):
    """z as the bytes stand for it: base + byte * step, column by column, in float64."""
    block = torch.arange(codes.shape[1], device=codes.device) // BLOCK
    return base.double()[:, block] + codes.double() * step.double()[:, block]


def _exact_encode(z):
    """The bytes by their definition in float32 (they are whole numbers; the float32 operations are part of it)."""
    base, step, codes = [], [], []
    for k in range(0, z.shape[1], BLOCK):
        part = z[:, k:k + BLOCK]
        low, high = part.min(1).values, part.max(1).values
        width = (high - low) * torch.full_like(low, 1.0 / 255.0)
        flat = width < 1e-30
        inverse = torch.ones_like(width) / width.masked_fill(flat, 1.0)
        code = torch.round((part - low[:, None]) * inverse[:, None])
        codes.append(code.masked_fill(flat[:, None], 0.0).clamp_(0.0, 255.0))
        base.append(low)
        step.append(width.masked_fill(flat, 0.0))
    return torch.stack(base, 1), torch.stack(step, 1), torch.cat(codes, 1)


def _exact_act(u, act):
    """The activation and its derivative in float64."""
    if act == "celu":
        e = torch.exp(10.0 * u.clamp(max=0.0))
        return torch.where(u >= 0, u, torch.expm1(10.0 * u.clamp(max=0.0)) / 10.0), torch.where(u >= 0, torch.ones_like(u), e)
    if act in ("gaussian", "normal"):
        k = 1.0 if act == "gaussian" else 0.5
        a = torch.exp(-k * u.square())
        return a, -2.0 * k * u * a
    return torch.logaddexp(u, torch.zeros_like(u)) - 0.69314718056, torch.sigmoid(u)


def exact(case, seed):
    s = prepare(case, seed)
    rows, norm, kind = _ranges(s["acs"]), case.get("norm", True), case["kind"]
    n, w = case["n"], case["w"]
    element = torch.repeat_interleave(torch.arange(4), torch.from_numpy(s["acs"]).long()).to("cuda")

    def per_row(params):
        return torch.stack(params).double()[element]

    def sums(t):
        return torch.zeros((4, t.shape[1]), dtype=torch.float64, device="cuda").index_add_(0, element, t)

    def back(du, xhat, rstd, gain):
        up = du * gain
        dx = (up - up.sum(1, keepdim=True) / w - xhat * ((up * xhat).sum(1, keepdim=True) / w)) * rstd[:, None]
        return dx, sums(du * xhat), sums(du)

    if kind in ("norm", "activation"):
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = torch.rsqrt(var + EPS)
    if kind == "norm":
        y = per_row(s["gains"]) * ((x - mean[:, None]) * rstd[:, None]) + per_row(s["biases"])
        return {"y": y, "mean": mean, "rstd": rstd}
    if kind == "norm_grad":
        mean, rstd = s["mean"].double(), s["rstd"].double()
        dx, dgain, dbias = back(s["grad"].double(), (s["x"].double() - mean[:, None]) * rstd[:, None], rstd, per_row(s["gains"]))
        return {"dx": dx, "dgain": dgain, "dbias": dbias}
    if kind == "activation":
        base, step, codes = _exact_encode(s["x"])
        kept, grad = _exact_kept(codes, base, step), s["grad"].double()
        if not norm:
            dz = grad * _exact_act(kept, case["act"])[1]
            return {"a": _exact_act(x, case["act"])[0], "dz": dz, "dsum": sums(dz)}
        gain, bias = per_row(s["gains"]), per_row(s["biases"])
        a = _exact_act(gain * ((x - mean[:, None]) * rstd[:, None]) + bias, case["act"])[0]
        xhat = (kept - mean[:, None]) * rstd[:, None]
        dz, dgain, dbias = back(grad * _exact_act(gain * xhat + bias, case["act"])[1], xhat, rstd, gain)
        return {"a": a, "dz": dz, "dsum": sums(dz), "dgain": dgain, "dbias": dbias}
    u = _exact_kept(s["codes"][:, :w], s["blocks"][:, :, 0], s["blocks"][:, :, 1])
    if norm:
        u = (u - s["mean"].double()[:, None]) * s["rstd"].double()[:, None]
        u = u * per_row(s["gains"]) + per_row(s["biases"])
    a, grad = _exact_act(u, case["act"])[0], s["grad"].double()
    return {"dw": torch.stack([torch.einsum("ni,nj->ij", a[p:q], grad[p:q]) for p, q in rows])}

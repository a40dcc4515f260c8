"""Plain implementations of the operators of khan_b200.layer_mod in extended precision (numpy's long double), and bounds for
what float arithmetic may add to them.

U(dtype) is half a step relative to a value, the error of one rounding.  A sum over a row of w values is formed in a tree:
at most 16 additions in a thread (4 columns in each of 4 groups), 5 in a warp, 8 over the warps of a CTA: DEPTH = 32 roundings
of partial sums that are no larger than the sum of the magnitudes."""
import numpy as np

LD = np.longdouble
DEPTH = 32
BLOCK = 128


def U(dtype):
    return LD(np.finfo(dtype).eps) / 2


def element_rows(acs):
    ends = np.cumsum(acs)
    return [slice(int(e - c), int(e)) for e, c in zip(ends, acs)]


def per_row(params, acs):
    """The vector of a row's element for each row."""
    return np.concatenate([np.broadcast_to(np.asarray(p, LD), (int(c), len(p))) for p, c in zip(params, acs)])


def sums(t, acs):
    return np.stack([t[r].sum(0) for r in element_rows(acs)])


def sum_depth(n):
    """Roundings of a sum over n rows: a team's share of a range (at least 1 / 8 of 1 / 296 of the rows, 4 at least), the
    teams of a CTA (32), a part of the ranges (300 / 8) and the parts (8), with 32 for what is rounded up."""
    return n // 296 + 4 + 32 + 38 + 8 + 32


def norm(x, gain, bias, acs, eps):
    """y, mean, rstd and a bound of the error of each."""
    u = U(x.dtype)
    x = x.astype(LD)
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1 / np.sqrt((d * d).mean(1) + LD(eps))
    g, h = per_row(gain, acs), per_row(bias, acs)
    xhat = d * rstd[:, None]
    biggest = np.abs(x).max(1)
    mean_err = (DEPTH + 3) * u * biggest
    # sum d^2: its terms are off by 2 |d| (mean_err + u |d|), the mean's part is of second order in the sum (the d's add up
    # to nothing); the division, eps, square root and reciprocal are four roundings more
    rstd_err = rstd * (DEPTH + 10) * u + rstd ** 3 * mean_err ** 2
    y = xhat * g + h
    y_err = np.abs(g) * (rstd[:, None] * (mean_err[:, None] + 2 * u * np.abs(d)) + np.abs(d) * rstd_err[:, None] + 3 * u * np.abs(xhat)) + u * (np.abs(y) + np.abs(h))
    return (y, mean, rstd), (y_err, mean_err, rstd_err)


def norm_back(du, xhat, xhat_err, rstd, g, u):
    """dx and its error from the gradient du behind gain and bias, whose own error is not counted here."""
    up = g * du
    c1, c2 = up.mean(1)[:, None], (up * xhat).mean(1)[:, None]
    m1, m2 = np.abs(up).mean(1)[:, None], np.abs(up * xhat).mean(1)[:, None]
    dx = rstd[:, None] * (up - c1 - xhat * c2)
    c2_err = (DEPTH + 5) * u * m2 + (np.abs(up) * xhat_err).mean(1)[:, None]
    err = rstd[:, None] * (6 * u * np.abs(up) + (DEPTH + 8) * u * m1 + np.abs(xhat) * (c2_err + 6 * u * m2) + xhat_err * m2)
    return dx, err


def norm_grad(dy, x, gain, mean, rstd, acs):
    u = U(x.dtype)
    x, dy, mean, rstd = (t.astype(LD) for t in (x, dy, mean, rstd))
    xhat = (x - mean[:, None]) * rstd[:, None]
    dx, err = norm_back(dy, xhat, 3 * u * np.abs(xhat), rstd, per_row(gain, acs), u)
    depth = sum_depth(len(x)) + 5
    return ((dx, sums(dy * xhat, acs), sums(dy, acs)),
            (err, depth * u * sums(np.abs(dy * xhat), acs), depth * u * sums(np.abs(dy), acs)))


def encode(z):
    """(codes, blocks) by their definition: float32 operations, each rounded once."""
    z = z.astype(np.float32)
    codes, blocks = [], []
    with np.errstate(invalid="ignore", over="ignore"):
        for k in range(0, z.shape[1], BLOCK):
            part = z[:, k:k + BLOCK]
            base, high = part.min(1), part.max(1)
            spread = high - base
            finite = spread < np.inf
            step = spread * np.float32(1.0 / 255.0)
            some = finite & (step >= np.float32(1e-30))
            step = np.where(some, step, np.float32(0))
            inv = np.where(some, np.float32(1) / np.where(some, step, np.float32(1)), np.float32(0))
            code = np.minimum(np.rint((part - base[:, None]) * inv[:, None]), 255)
            codes.append(np.where(some[:, None], code, 0).astype(np.uint8))
            blocks.append(np.stack([np.where(finite, base, np.float32(np.nan)), step], 1))
    return np.concatenate(codes, 1), np.stack(blocks, 1)


def decode(codes, blocks):
    at = np.arange(codes.shape[1]) // BLOCK
    return blocks[:, at, 0].astype(LD) + codes.astype(LD) * blocks[:, at, 1].astype(LD)


def act(name, u):
    """Value, first derivative, and a bound of the second derivative."""
    with np.errstate(over="ignore"):
        if name == "celu":
            e = np.exp(np.minimum(u, 0) * 10)
            return np.where(u >= 0, u, (e - 1) / 10), np.where(u >= 0, LD(1), e), 10
        if name == "gaussian":
            return np.exp(-u * u), -2 * u * np.exp(-u * u), 2
        if name == "normal":
            return np.exp(-u * u / 2), -u * np.exp(-u * u / 2), 1
        # the framework's constant stands for ln 2
        return np.maximum(u, 0) + np.log1p(np.exp(-np.abs(u))) - LD(0.69314718056), 1 / (1 + np.exp(-u)), LD(0.25)


def act_error(u, name, arg, arg_err):
    """Error of an activation and of its derivative for an argument that is off by arg_err: the argument's part, a relative
    error of the exponential of 4 u and of its argument (|arg| <= 10 |u| where it is not flat), and four roundings."""
    a, d, second = act(name, arg)
    return np.abs(d) * arg_err + second * arg_err ** 2 + 24 * u * (1 + np.abs(a)), second * arg_err + 24 * u * (1 + 0 * a)


def activation(z, name, gain, bias, acs, eps):
    u = U(np.float32)
    if gain is None:
        value = z.astype(LD)
        return act(name, value)[0], act_error(u, name, value, 0 * value)[0], None, None
    (y, mean, rstd), (err, mean_err, rstd_err) = norm(z, gain, bias, acs, eps)
    return act(name, y)[0], act_error(u, name, y, err)[0], (mean, rstd), (mean_err, rstd_err)


def kept_input(codes, blocks, mean, rstd, gain, bias, acs):
    """u and xhat as a checkpoint stands for them, and their errors."""
    u = U(np.float32)
    z = decode(codes, blocks)
    z_err = 2 * u * np.abs(z)
    if gain is None:
        return z, z_err, None, None
    mean, rstd = mean.astype(LD)[:, None], rstd.astype(LD)[:, None]
    xhat = (z - mean) * rstd
    xhat_err = rstd * (z_err + 2 * u * (np.abs(z) + np.abs(mean))) + 4 * u * np.abs(xhat)
    g, h = per_row(gain, acs), per_row(bias, acs)
    value = xhat * g + h
    return value, np.abs(g) * xhat_err + 3 * u * (np.abs(xhat * g) + np.abs(h)), xhat, xhat_err


def activation_grad(codes, blocks, mean, rstd, name, da, gain, bias, acs):
    """(dz, dsum[, dgain, dbias]) and their errors."""
    u = U(np.float32)
    value, value_err, xhat, xhat_err = kept_input(codes, blocks, mean, rstd, gain, bias, acs)
    d_err = act_error(u, name, value, value_err)[1]
    da = da.astype(LD)
    du, du_err = da * act(name, value)[1], np.abs(da) * (d_err + u)
    depth = sum_depth(len(da)) + 5
    if gain is None:
        return (du, sums(du, acs)), (du_err, sums(du_err, acs) + depth * u * sums(np.abs(du) + du_err, acs))
    r, g = rstd.astype(LD), per_row(gain, acs)
    dz, err = norm_back(du, xhat, xhat_err, r, g, u)
    up_err = np.abs(g) * du_err
    err = err + r[:, None] * (up_err + up_err.mean(1)[:, None] + np.abs(xhat) * (up_err * np.abs(xhat)).mean(1)[:, None])
    term, term_err = du * xhat, du_err * np.abs(xhat) + np.abs(du) * xhat_err
    return ((dz, sums(dz, acs), sums(term, acs), sums(du, acs)),
            (err, sums(err, acs) + depth * u * sums(np.abs(dz) + err, acs),
             sums(term_err, acs) + depth * u * sums(np.abs(term) + term_err, acs),
             sums(du_err, acs) + depth * u * sums(np.abs(du) + du_err, acs)))


def weight_grad(codes, blocks, mean, rstd, name, dz, gain, bias, acs):
    u = U(np.float32)
    value, value_err, _, _ = kept_input(codes, blocks, mean, rstd, gain, bias, acs)
    a, a_err = act(name, value)[0], act_error(u, name, value, value_err)[0]
    dz = dz.astype(LD)
    # a product in three tf32 parts is off by 2^-21; the sum over a range of rows is cut off (a whole step, 2 u) at every
    # eighth row and rounded at every row where it is not formed by the tensor core, the ranges are added one by one
    depth = 2 * (len(dz) + 300)
    dw = np.stack([a[r].T @ dz[r] for r in element_rows(acs)])
    size = np.stack([np.abs(a[r]).T @ np.abs(dz[r]) for r in element_rows(acs)])
    err = np.stack([a_err[r].T @ np.abs(dz[r]) for r in element_rows(acs)]) + (LD(2) ** -21 + depth * u) * size
    return dw, err

"""Plain 64-bit forms of the row operators, and how far the kernels may be from them.

Error bounds, with u the unit roundoff of the statistics' type (2^-24 for float16 and float32 data, 2^-53 for float64) and
half a step of the result's type for its one rounding.  A sum of k terms added one after the other is off by at most k u times
the sum of their magnitudes; a row's sum is made of at most `depth` additions in a chain."""
import numpy as np


def unit(dt):
    return 2.0 ** -53 if np.dtype(dt) == np.float64 else 2.0 ** -24


def half_step(dt, v):
    """Half a step of type dt at v (its subnormal step at least)."""
    f = np.finfo(dt)
    return np.maximum(np.abs(v) * (f.eps / 2), float(f.smallest_subnormal) / 2)


def depth(n):
    """Additions in a chain for a row of n: at most 64 elements per lane while a row stays in registers, n / 1024 per thread
    beyond; the lanes of a wave and the waves of a block add 6 + 16."""
    return 64 + n / 1024 + 22


def layer_norm(x, w, b, eps):
    x = x.astype("f8")
    mean = x.mean(-1)
    d = x - mean[..., None]
    rstd = 1 / np.sqrt((d * d).mean(-1) + eps)
    h = d * rstd[..., None]
    y = h * (1 if w is None else w.astype("f8")) + (0 if b is None else b.astype("f8"))
    return y, mean, rstd, h


def layer_norm_tolerances(x, w, b, eps):
    dt, u, n = x.dtype, unit(x.dtype), x.shape[-1]
    y, mean, rstd, h = layer_norm(x, w, b, eps)
    k, big = depth(n), np.abs(x.astype("f8")).max(-1)
    t_mean = (k + 2) * u * big  # |sum error| / n <= k u mean|x| <= k u max|x|
    # (x - m): the mean's error and a rounding; the variance of it: k u relative and the square of the mean's error
    rel = (k + 6) * u + ((k + 2) * u * big * rstd) ** 2
    t_rstd = rstd * rel
    aw = 1.0 if w is None else np.abs(w.astype("f8"))
    ab = 0.0 if b is None else np.abs(b.astype("f8"))
    t_h = (t_mean * rstd)[..., None] + np.abs(h) * (rel + 3 * u)[..., None]
    t_y = t_h * aw * 1.01 + 3 * u * (np.abs(h) * aw + ab)
    return t_y + half_step(dt, np.abs(y) + t_y), t_mean, t_rstd


def layer_norm_grad(dy, x, mean, rstd, w):
    dy, x, rstd = dy.astype("f8"), x.astype("f8"), rstd.astype("f8")[..., None]
    h = (x - mean.astype("f8")[..., None]) * rstd
    g = dy if w is None else dy * w.astype("f8")
    dx = rstd * (g - g.mean(-1, keepdims=True) - h * (g * h).mean(-1, keepdims=True))
    rows = tuple(range(x.ndim - 1))
    return dx, (dy * h).sum(rows), dy.sum(rows), h, g


def layer_norm_grad_tolerances(dy, x, mean, rstd, w):
    dt, u, n = x.dtype, unit(x.dtype), x.shape[-1]
    wdt = dt if w is None else w.dtype
    dx, dw, db, h, g = layer_norm_grad(dy, x, mean, rstd, w)
    ag, ah, s = np.abs(g), np.abs(h), np.abs(rstd.astype("f8"))[..., None]
    k = depth(n)
    c1 = (k + 3) * u * ag.mean(-1, keepdims=True)
    c2 = (k + 7) * u * (ag * ah).mean(-1, keepdims=True)
    t = s * (c1 + ah * c2 * 1.01 + 8 * u * (ag + ag.mean(-1, keepdims=True) + ah * (ag * ah).mean(-1, keepdims=True)))
    rows = tuple(range(x.ndim - 1))
    m = int(np.prod(x.shape[:-1]))
    kr = m / 64 + 128  # rows added by one block (a block per CU at least, or one block per row), its groups, the blocks
    ad = np.abs(dy.astype("f8"))
    t_w, t_b = (kr + 4) * u * (ad * ah).sum(rows), kr * u * ad.sum(rows)
    return (t + half_step(dt, np.abs(dx) + t), t_w + half_step(wdt, np.abs(dw) + t_w), t_b + half_step(wdt, np.abs(db) + t_b))


def _softmax(x):
    """(e, largest, sum) of exp(x - largest), with 0 for an empty or all -inf row's exponentials."""
    m = x.max(-1, initial=-np.inf)
    with np.errstate(invalid="ignore"):
        e = np.exp(x - np.where(m > -np.inf, m, 0)[..., None])
    return e, m, e.sum(-1)


def distill(z, t, tok, temp, weights=None):
    """loss, dlogits, and what their bounds are made of.  Two-dimensional arguments."""
    z, t, tok = z.astype("f8"), t.astype("f8"), tok.astype("i8")
    r, v = z.shape
    there = (tok >= 0) & (tok < v)
    at = np.where(there, tok, 0)
    with np.errstate(over="ignore", invalid="ignore"):
        e, m, s = _softmax(z / temp)
    te, tm, ts = _softmax(np.where(there, t, -np.inf) / temp)
    some = ts > 0
    with np.errstate(all="ignore"):
        q = e / s[:, None]
        logq_all = z / temp - m[:, None] - np.log(s)[:, None]
        p = np.where(some[:, None] | np.isnan(ts)[:, None], te / ts[:, None], 0.0)
        logp = t / temp - tm[:, None] - np.log(ts)[:, None]
        logq = np.take_along_axis(logq_all, at, 1)
        term = np.where(p == 0, 0.0, p * (logp - logq))
        loss = temp ** 2 * term.sum(1)
        mass = np.where(some, 1.0, np.where(np.isnan(ts), np.nan, 0.0))
        grad = q * mass[:, None]
        np.subtract.at(grad, (np.arange(r)[:, None], at), p)
        w = np.ones(r) if weights is None else weights.astype("f8")
        grad = grad * (temp * w)[:, None]
        grad[(mass == 0) | (w == 0)] = 0.0
        t_far = np.where(there & np.isfinite(t) & some[:, None], t / temp - tm[:, None], 0.0)
        zm = z / temp - m[:, None]
    return dict(loss=loss, grad=grad, q=q, p=p, at=at, logp=logp, logq=logq, zm=zm, tm=t_far, w=w, s=s)


def distill_tolerances(z, t, tok, temp, weights=None):
    """For finite logits and entries."""
    u, v, k = unit(z.dtype), z.shape[1], t.shape[1]
    d = distill(z, t, tok, temp, weights)
    r = z.shape[0]
    # an exponential: three roundings of its argument, the function itself (2 u)
    de = u * (3 * np.abs(d["zm"]) + 2)
    # a thread's running sum: one addition per element and one rescaling per pack of at most v / 128 in a chain, the joins
    ds = (d["q"] * de).sum(1) + u * (v / 128 + 64)
    dp = u * (3 * np.abs(d["tm"]) + 2)
    dps = (d["p"] * dp).sum(1) + u * (k / 64 + 32)
    with np.errstate(invalid="ignore"):
        lp, lq = np.abs(np.where(d["p"] > 0, d["logp"], 0)), np.abs(np.where(d["p"] > 0, d["logq"], 0))
        # log p and log q: three roundings of the scaled difference, the sum's relative error, the logarithm and a subtraction
        zk = np.abs(np.take_along_axis(d["zm"], d["at"], 1))
        dlp = u * (3 * np.abs(d["tm"]) + 4 * np.abs(lp) + 2 * (lp + np.abs(d["tm"]))) + dps[:, None]
        dlq = u * (3 * zk + 4 * lq + 2 * (lq + zk)) + ds[:, None]
    size = lp + lq
    t_loss = temp ** 2 * (d["p"] * (dlp + dlq) + d["p"] * (dp + dps[:, None] + u * (k / 64 + 32)) * size).sum(1)
    t_loss = t_loss * 1.01 + u * np.abs(d["loss"]) * 4
    sp = np.zeros_like(d["q"])
    np.add.at(sp, (np.arange(r)[:, None], d["at"]), d["p"] * (dp + dps[:, None] + (k + 4) * u))
    t = np.abs(temp * d["w"])[:, None] * ((d["q"] * (de + ds[:, None] + 8 * u)) + sp) * 1.01 + 1e-37
    return t_loss, t + half_step(z.dtype, np.abs(d["grad"]) + t)


def process_logits(z, prompt=None, plen=None, output=None, olen=None, rep=1.0, freq=0.0, pres=0.0, btok=None, bval=None,
                   allowed=None):
    """(result, bound, which logits have to come through unchanged); two-dimensional logits, side arrays with rows."""
    r, v = z.shape
    u = unit(z.dtype)
    seen, said, bias, nb, ab = (np.zeros((r, v)) for _ in range(5))
    for i in range(r):
        for toks, lens, out in ((prompt, plen, False), (output, olen, True)):
            if toks is None:
                continue
            n = toks.shape[1] if lens is None else int(np.clip(lens[i], 0, toks.shape[1]))
            for x in toks[i, :n]:
                if 0 <= x < v:
                    seen[i, x] = 1
                    said[i, x] += out
        if btok is not None:
            for x, b in zip(btok[i], bval[i]):
                if 0 <= x < v:
                    bias[i, x] += np.float64(b)
                    ab[i, x] += abs(np.float64(b))
                    nb[i, x] += 1
    col = lambda p: np.broadcast_to(np.asarray(p, dtype="f8").reshape(-1, 1), (r, 1))  # noqa: E731
    rep, freq, pres = col(rep), col(freq), col(pres)
    x = z.astype("f8")
    with np.errstate(invalid="ignore"):
        y = np.where(seen > 0, np.where(x > 0, x / rep, x * rep), x)
        a = np.abs(y) + np.abs(freq) * said + np.abs(pres) * (said > 0)
        y = y - freq * said - pres * (said > 0) + bias
        tol = 5 * u * a + (nb + 2) * u * ab
        tol = tol + half_step(z.dtype, np.abs(y) + tol)
    same = (seen == 0) & (nb == 0)
    if allowed is not None:
        bits = (allowed.view("u4")[:, np.arange(v) >> 5] >> (np.arange(v) & 31).astype("u4")) & 1
        y = np.where(bits == 0, -np.inf, y)
        same &= bits != 0
    return y, tol, same

"""The row operators at the ends of their ranges: values near the limits of a type, large offsets, calls larger than one
launch, long lists."""
import numpy as np
import pytest

import dpnp_amd.tensor as dpt
from tests import row_operator_references as ref
from tests.helpers import dev, host

pytestmark = pytest.mark.gpu
W = np.longdouble  # its exponents hold differences and products of float64's largest values


def within(got, want, tol, what=""):
    got = host(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    with np.errstate(all="ignore"):
        rounded = want.astype(got.dtype)  # (beyond the type's range: infinite)
        bad = ~(np.abs(got.astype(W) - want) <= tol) & ~(np.isinf(rounded) & (got == rounded))
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(), got[bad][:3], want[bad][:3],
                           np.broadcast_to(tol, want.shape)[bad][:3])


# ---- distillation --------------------------------------------------------------------------------------------------
def distill(z, t, tok, temp, w):
    """(loss, bound, gradient, bound) from the definition, in units of the logits so that nothing overflows.  The bounds count
    the roundings as `distill_tolerances` does: three of an exponential's argument and 2 u of the function, a chain of
    additions and rescalings of v / 128 + 64 at most per sum, and those of the final products."""
    u = W(ref.unit(z.dtype))
    dt, (r, v), k = z.dtype, z.shape, t.shape[1]
    z, t, temp, w = z.astype(W), t.astype(W), W(temp), w.astype(W)
    there = (tok >= 0) & (tok < v)
    at = (np.arange(r)[:, None], np.where(there, tok, 0))
    d = z - z.max(1)[:, None]
    with np.errstate(under="ignore"):
        e = np.exp(d / temp)
    s = e.sum(1)[:, None]
    q = e / s
    some = there.any(1)[:, None]
    top = np.where(there, t, -np.inf).max(1, initial=-np.inf)[:, None]
    td = np.where(there, t - np.where(some, top, 0), 0)
    with np.errstate(under="ignore"):
        te = np.where(there, np.exp(td / temp), 0)
    ts = np.where(some, te.sum(1)[:, None], 1)
    p = te / ts
    zk = d[at]
    loss = np.where(p > 0, temp * p * (td - zk) + temp * temp * p * (np.log(s) - np.log(ts)), 0).sum(1)
    grad = q * some
    np.subtract.at(grad, at, p)
    grad *= (temp * w)[:, None]
    grad[w == 0] = 0
    # bounds
    de, dp = u * (3 * np.abs(d) / temp + 2), u * (3 * np.abs(td) / temp + 2)
    ds = (q * de).sum(1)[:, None] + u * (W(v) / 128 + 64)
    dps = (p * dp).sum(1)[:, None] + u * (W(k) / 64 + 32)
    size = temp * (np.abs(td) + np.abs(zk)) + temp * temp * (np.log(s) + np.log(ts))
    t_loss = (p * (dp + dps + u * (W(k) / 64 + 40)) * size + p * temp * temp * (ds + dps)).sum(1) * W(1.01) + W(1e-37)
    sp = np.zeros_like(q)
    np.add.at(sp, at, p * (dp + dps + (k + 4) * u))
    t = np.abs(temp * w)[:, None] * (q * (de + ds + 8 * u) + sp) * W(1.01) + W(1e-37)
    half = np.maximum((np.abs(grad) + t) * W(np.finfo(dt).eps) / 2, W(np.finfo(dt).smallest_subnormal) / 2)
    return loss, t_loss, grad, t + half


def check_distill(z, t, tok, temp, w=None):
    r, acc = z.shape[0], "f8" if z.dtype == np.float64 else "f4"
    w = np.ones(r, acc) if w is None else w.astype(acc)
    loss, t_loss, grad, t_grad = distill(z, t, tok, temp, w)
    within(dpt.distill_topk(dev(z), dev(t), dev(tok), temperature=temp), loss, t_loss, "loss")
    got, dz = dpt.distill_topk_grad(dev(z), dev(t), dev(tok), dev(w), temperature=temp)
    within(got, loss, t_loss, "loss with gradient")
    within(dz, grad, t_grad, "gradient")


FAR = {"f2": [65504, -65504, 1, 0], "f4": [1e10, -1e10, 1e12, -1e30, 1e38, "max", "min", 0],
       "f8": [1e10, 1e19, -1e19, -1e100, 1e308, "max", "min", 0]}


def far_values(dt):
    return [dict(max=np.finfo(dt).max, min=np.finfo(dt).min).get(x, x) for x in FAR[dt]]


# rows owned by a block (the vocabulary held in registers or read twice) and rows split over blocks
@pytest.mark.parametrize("temp", [0.7, 1.0, 2.0])
@pytest.mark.parametrize("dt,v,least", [("f4", 40, 1), ("f4", 1001, 1), ("f4", 20011, 1), ("f4", 100003, 1), ("f4", 90200, 66),
                                        ("f8", 40, 1), ("f8", 9001, 1), ("f8", 12001, 1), ("f8", 20001, 1),
                                        ("f2", 40, 1), ("f2", 100003, 1)])
def test_distill_of_large_finite_values(dt, v, least, temp):
    rng = np.random.default_rng(v)
    tdt = "f8" if dt == "f8" else "f4"
    zs, ts = far_values(dt), far_values(tdt)
    k, cases = 9, [(a, b) for a in zs + [None] for b in ts + [None]]
    if v > 5000:  # every value on each side, not every pair
        cases = [(a, ts[i % len(ts)]) for i, a in enumerate(zs)] + [(None, b) for b in ts] + [(a, None) for a in zs]
    cases = (cases * (least // len(cases) + 1))[:max(least, len(cases))]
    r = len(cases)
    z, t = np.empty((r, v), dt), np.empty((r, k), tdt)
    tok = np.stack([rng.permutation(v)[:k] for _ in range(r)]).astype("i4")
    tok[::3, 4] = tok[::3, 1]
    tok[1::4, 6:] = -1
    for i, (a, b) in enumerate(cases):
        z[i] = rng.standard_normal(v) if a is None else a
        t[i] = 3 * rng.standard_normal(k) if b is None else b
        if a is not None and i % 2:  # half of the vocabulary so far below that it has no part
            z[i, rng.random(v) < 0.5] = -a if a > 0 else a if a == np.finfo(dt).min else 1.5 * a
        if b is not None and i % 3 == 2:
            t[i, 2] = -b if b > 0 else b
    check_distill(z, t, tok, temp, rng.uniform(0.5, 2, r))


@pytest.mark.parametrize("dt,far,step", [("f4", 1e10, 1024.0), ("f4", -3e12, 2.0 ** 18), ("f8", -1e19, 2048.0), ("f8", 1e40, 2.0 ** 80)])
@pytest.mark.parametrize("v", [300, 33001, 100003])
def test_distill_of_far_offsets_at_high_temperatures(dt, far, step, v):
    """Logits a few steps of their type apart, at temperatures that make something of the steps: on both sides of the limit
    between the two forms of the exponential."""
    rng = np.random.default_rng(v)
    z = (np.dtype(dt).type(far) - step * rng.integers(0, 9, (3, v))).astype(dt)
    t = (np.dtype(dt).type(far) - step * rng.integers(0, 9, (3, 12))).astype(dt)
    tok = np.stack([rng.permutation(v)[:12] for _ in range(3)])
    for temp in (step / 3, step * 2, step * 300):
        check_distill(z, t, tok, temp)


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("v", [60, 100003])
def test_distill_of_masked_teacher_tokens(dt, v):
    """A teacher's token that the student has masked with the lowest value: a large loss, not an infinite one."""
    rng = np.random.default_rng(3)
    z, tok = rng.standard_normal((4, v)).astype(dt), np.stack([rng.permutation(v)[:5] for _ in range(4)]).astype("i4")
    t = rng.standard_normal((4, 5)).astype("f8" if dt == "f8" else "f4")
    z[0, tok[0, 2]] = z[1, tok[1, 0]] = z[1, tok[1, 4]] = np.finfo(dt).min
    z[2] = np.finfo(dt).min
    z[2, tok[2, 3]] = 0
    t[3, 1:] = np.finfo(t.dtype).min
    for temp in (0.7, 1.0, 2.0):
        check_distill(z, t, tok, temp)


@pytest.mark.parametrize("dt", ["f4", "f8"])
def test_distill_at_the_ends_of_the_temperatures(dt):
    rng = np.random.default_rng(5)
    z = rng.standard_normal((3, 50)).astype(dt)
    t, tok = z[:, ::-1].copy(), np.arange(50, dtype="i4")[None].repeat(3, 0)
    for temp in (1e-4, 1e-20, 1e-40) + ((1e-307, 5e-324) if dt == "f8" else ()):
        check_distill(z, t, tok, temp)
    for temp in (1e6, 1e25):  # T^2 is beyond float32: the result may be infinite, but is a number
        loss, dz = dpt.distill_topk_grad(dev(z), dev(t), dev(tok), temperature=temp)
        assert not np.isnan(host(loss)).any() and np.isfinite(host(dz)).all()
    tok = np.arange(10, dtype="i4")[None].repeat(3, 0)
    assert (host(dpt.distill_topk(dev(z), dev(t[:, :10].copy()), dev(tok), temperature=1e25)) > (1e38 if dt == "f4" else 1e49)).all()


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("v", [50, 4097, 100003])
def test_distill_at_low_temperatures(dt, v):
    rng = np.random.default_rng(v)
    tok = np.stack([rng.permutation(v)[:7] for _ in range(3)]).astype("i4")
    for temp in (0.006, 0.0055, 0.004, 1e-3):
        z = (temp * rng.standard_normal((3, v))).astype(dt)
        z[1] = np.clip(z[1], None, 0)
        t = (3 * temp * rng.standard_normal((3, 7))).astype("f8" if dt == "f8" else "f4")
        check_distill(z, t, tok, temp)
        check_distill(z + np.dtype(dt).type(8), t, tok, temp)


@pytest.mark.parametrize("dt,far,temp", [("f2", 1.0, 1e-3), ("f4", 1e30, 1.0), ("f8", 1e300, 1.0)])
@pytest.mark.parametrize("v", [1000, 20011, 100003])
def test_distill_of_far_rows_in_place(dt, far, temp, v):
    rng = np.random.default_rng(v)
    z = np.where(rng.random((3, v)) < 0.5, far, far / 2).astype(dt)
    z[1] = rng.standard_normal(v)
    tok = np.stack([rng.permutation(v)[:7] for _ in range(3)]).astype("i4")
    t = rng.standard_normal((3, 7)).astype("f8" if dt == "f8" else "f4")
    want = [host(a) for a in dpt.distill_topk_grad(dev(z), dev(t), dev(tok), temperature=temp)]
    zd = dev(z)
    got = dpt.distill_topk_grad(zd, dev(t), dev(tok), temperature=temp, out=(None, zd))
    assert np.array_equal(host(got[0]), want[0]) and np.array_equal(host(zd), want[1])
    check_distill(z, t, tok, temp)


# ---- layer norm ----------------------------------------------------------------------------------------------------
def check_layer_norm(x, w, b, eps):
    """The rounded mean m of a row is off by (k + 2) u max|x| at most, k additions in a chain; d = x - m is then as exact as its own
    size, and the mean of d corrects m up to (k + 3) u mean|d|; one of up to 4 u of the root of mean(d^2) need not be applied.  The
    variance, mean(d^2) - mean(d)^2, is off by (k + 5) u times the sum of the two."""
    dt, n = x.dtype, x.shape[-1]
    u, k = W(ref.unit(dt)), W(ref.depth(n))
    xs = x.astype(W)
    near = xs - xs[:, :1]  # (exact in these rows, whose mean would lose digits of its own far from zero)
    mean = xs[:, 0] + near.mean(-1)
    d = near - near.mean(-1)[:, None]
    var = (d * d).mean(-1)
    rstd = 1 / np.sqrt(var + W(eps))
    h = d * rstd[:, None]
    y = h * w.astype(W) + b.astype(W)
    off = (k + 2) * u * np.abs(xs).max(-1)
    centre = (k + 8) * u * (np.sqrt(var) + off)
    rel = (k + 6) * u * (var + 2 * off * off) / (var + W(eps)) + 4 * u
    assert rel.max() < 0.2  # (below, 1 / sqrt(1 + e) is taken as 1 - e / 2 up to its square)
    t_h = (centre * rstd * (1 + rel))[:, None] + np.abs(h) * (rel + 3 * u)[:, None] + 2 * u * off[:, None] * rstd[:, None]
    t_y = t_h * np.abs(w) * W(1.01) + 3 * u * (np.abs(h) * np.abs(w) + np.abs(b))
    half = np.maximum((np.abs(y) + t_y) * W(np.finfo(dt).eps) / 2, W(np.finfo(dt).smallest_subnormal) / 2)
    got = dpt.layer_norm(dev(x), dev(w), dev(b), eps=eps, stats=True)
    within(got[0], y, t_y + half, "y")
    within(got[1], mean, centre + 2 * u * np.abs(mean), "mean")
    within(got[2], rstd, rstd * rel, "rstd")


# rows by lanes of a wave, by a wave, by blocks, with weights out of registers, and longer than the registers
@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("n", [7, 24, 100, 500, 1000, 3001, 9001, 20003, 40000, 70000])
def test_layer_norm_far_from_zero(n, dt):
    rng = np.random.default_rng(n)
    w, b = (1 + 0.1 * rng.standard_normal(n)).astype(dt), (0.1 * rng.standard_normal(n)).astype(dt)
    one = lambda c, s=1.0: (c + s * rng.standard_normal(n)).astype(dt)  # noqa: E731
    if dt == "f2":
        rows = [one(1000.0, 8.0), one(-30000.0, 100.0), one(3.0), one(0.0)]
    else:
        far = 1.0 if dt == "f4" else 1e8
        rows = [one(1e3 * far), one(-1e4 * far), one(1e5 * far), one(1e4 * far, 100.0), one(0.0), one(0.0)]
        rows[4][n // 2] = 1e4  # one large channel in the middle, and as the first element
        rows[5][0] = -1e4
    check_layer_norm(np.stack(rows), w, b, 1e-5)


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("n", [7, 100, 1000, 3000, 20003, 70000])
def test_layer_norm_of_constant_rows(n, dt):
    w, b = np.ones(n, dt), np.zeros(n, dt)
    row = lambda *c: np.repeat(np.array(c, dt)[:, None], n, 1)  # noqa: E731
    check_layer_norm(row(1000.1, 5000.3, -0.1, 0.0, 3.7), w, b, 1e-5)
    check_layer_norm(row(60000.7, -12345.6), w, b, 1e-3)
    if dt != "f2":  # the variance of such rows is a rounding error, of either sign: a number all the same
        y, mean, rstd = (host(a) for a in dpt.layer_norm(dev(row(1e9, -3e12, 1e15 / 3)), stats=True))
        assert np.isfinite(y).all() and np.isfinite(rstd).all() and (np.abs(mean[:, None] / row(1e9, -3e12, 1e15 / 3) - 1) < 1e-6).all()


# ---- more blocks than one launch holds (2^32 threads) --------------------------------------------------------------------
def many(a, times):
    """The rows of `a` over and over: (times, rows, width) without a copy."""
    return dpt.broadcast_to(dev(a), (times,) + a.shape)


def all_equal(got, want):
    got = host(got)
    assert got.shape[1:] == want.shape
    for i in range(0, len(got), 1 << 18):
        assert (got[i:i + (1 << 18)] == want).all(), i


@pytest.mark.parametrize("lists", [False, True])
def test_logits_of_more_rows_than_a_launch(lists):
    rng = np.random.default_rng(1)
    z = rng.standard_normal((13, 8)).astype("f2")
    times = 2 ** 23 // 13 + 1  # 512 threads a row
    allowed = rng.integers(1, 255, (13, 1)).astype("u4")
    tok = rng.integers(0, 8, (13, 3)).astype("i4")
    kw = lambda f: dict(allowed=f(allowed), **(dict(output_tokens=f(tok), presence_penalty=0.5) if lists else {}))  # noqa: E731
    want = host(dpt.process_logits(dev(z), **kw(dev)))
    out = dpt.full((times, 13, 8), 7, dtype="f2")
    dpt.process_logits(many(z, times), out=out, **kw(lambda a: many(a, times)))
    all_equal(out, want)


@pytest.mark.parametrize("grad", [False, True])
def test_distill_of_more_rows_than_a_launch(grad):
    rng = np.random.default_rng(2)
    z, t = rng.standard_normal((13, 4)).astype("f2"), rng.standard_normal((13, 2)).astype("f4")
    tok = np.stack([rng.permutation(4)[:2] for _ in range(13)]).astype("i4")
    times = 2 ** (25 if grad else 24) // 13 + 1  # 128 and 256 threads a row
    want = [host(a) for a in dpt.distill_topk_grad(dev(z), dev(t), dev(tok))]
    loss = dpt.full((times, 13), 7, dtype="f4")
    args = [many(a, times) for a in (z, t, tok)]
    if grad:
        dz = dpt.full((times, 13, 4), 7, dtype="f2")
        dpt.distill_topk_grad(*args, out=(loss, dz))
        all_equal(dz, want[1])
    else:
        want[0] = host(dpt.distill_topk(dev(z), dev(t), dev(tok)))
        dpt.distill_topk(*args, out=loss)
    all_equal(loss, want[0])


def test_layer_norm_grad_of_more_columns_than_a_launch():
    rng = np.random.default_rng(3)
    n = 2 ** 27 + 37  # the fold of the parameters' gradients: 512 threads for 32 columns
    x, dy = (np.resize(rng.standard_normal(65537).astype("f2"), (1, n)) for _ in range(2))
    mean, rstd = np.array([0.25], "f4"), np.array([2.0], "f4")
    out = (None, dpt.full(n, 7, dtype="f2"), dpt.full(n, 7, dtype="f2"))
    dx, dw, db = dpt.layer_norm_grad(dev(dy), dev(x), dev(mean), dev(rstd), dpt.ones(n, dtype="f2"), out=out)
    dw, db = host(dw), host(db)
    assert np.array_equal(db, dy[0])
    for i in range(0, n, 1 << 24):
        at = slice(i, i + (1 << 24))
        # one product of two roundings, rounded to float16 (h is exact but for the rounding of its difference)
        want = (x[0, at].astype("f8") - 0.25) * 2 * dy[0, at]
        tol = 2.0 ** -22 * np.abs(want) + np.maximum(np.abs(want) * 2.0 ** -11 * (1 + 2.0 ** -20), 2.0 ** -25)
        assert (np.abs(dw[at] - want) <= tol).all(), i
    del dw, db
    assert np.isfinite(host(dx[:, -65537:])).all()


# ---- biases of logits ------------------------------------------------------------------------------------------------
def biased(z, tok, val):
    """Each token's biases added up in their order in the type of the sums, then to the logit."""
    acc = "f8" if z.dtype == np.float64 else "f4"
    s = np.zeros(z.shape, acc)
    inside = (tok >= 0) & (tok < z.shape[1])
    np.add.at(s, (np.arange(len(z))[:, None].repeat(tok.shape[1], 1)[inside], tok[inside]), val.astype(acc)[inside])
    return (z.astype(acc) + s).astype(z.dtype)


@pytest.mark.parametrize("dt,itype", [("f2", "i4"), ("f4", "i4"), ("f4", "i8"), ("f8", "i8")])
@pytest.mark.parametrize("rows,v", [(2, 40), (3, 1000), (2, 20011), (600, 1000), (40, 100003)])
@pytest.mark.parametrize("nb", [1, 63, 64, 65, 130, 256, 257, 300, 1000, 4099])
def test_logits_biases_in_their_order(rows, v, nb, dt, itype):
    if rows * nb > 700000:
        rows = 520
    rng = np.random.default_rng(nb)
    z = rng.standard_normal((rows, v)).astype(dt)
    val = rng.uniform(-3, 3, (rows, nb)).astype("f4")
    tok = rng.integers(-2, v + 2, (rows, nb))
    tok[0] = v - 1                                          # one token only
    if rows > 2:
        tok[1] = rng.integers(0, 3, nb) * (v // 3)          # few of them
        tok[2] = np.arange(nb) % v                          # neighbours
    if rows > 4:
        tok[3, ::2] = tok[3, 0] % v                         # one token between others
        tok[4] = np.where(rng.random(nb) < 0.5, -1, tok[4])
    tok = tok.astype(itype)
    got = host(dpt.process_logits(dev(z), bias_tokens=dev(tok), bias_values=dev(val)))
    assert np.array_equal(got, biased(z, tok, val))


def test_logits_biases_beside_everything_else():
    rng = np.random.default_rng(7)
    for rows, v, nb in ((3, 1000, 300), (520, 700, 300), (3, 30000, 5000)):
        z = rng.standard_normal((rows, v)).astype("f4")
        tok, val = rng.integers(-2, v + 2, (rows, nb)).astype("i4"), rng.integers(-40, 41, (rows, nb)).astype("f4") / 4
        said = rng.integers(-2, v + 2, (rows, 200)).astype("i4")
        allowed = rng.integers(0, 2 ** 32, (rows, (v + 31) // 32), dtype="u8").astype("u4")
        want, tol, _ = ref.process_logits(z, prompt=said[:, :100], output=said, rep=1.5, freq=0.25, pres=0.5, btok=tok, bval=val,
                                          allowed=allowed)
        got = host(dpt.process_logits(dev(z), prompt_tokens=dev(said[:, :100].copy()), output_tokens=dev(said), repetition_penalty=1.5,
                                      frequency_penalty=0.25, presence_penalty=0.5, bias_tokens=dev(tok), bias_values=dev(val),
                                      allowed=dev(allowed)))
        masked = want == -np.inf
        assert (got[masked] == -np.inf).all() and (np.abs(got[~masked] - want[~masked]) <= tol[~masked]).all()


def test_logits_time_goes_with_the_number_of_biases():
    import time
    rng = np.random.default_rng(9)
    v = 16000
    z, out = dev(rng.standard_normal((1, v)).astype("f4")), dpt.empty((1, v), dtype="f4")

    def seconds(nb):
        tok, val = dev(rng.integers(0, v, (1, nb)).astype("i4")), dev(rng.standard_normal((1, nb)).astype("f4"))
        best = np.inf
        for _ in range(8):
            start = time.perf_counter()
            dpt.process_logits(z, bias_tokens=tok, bias_values=val, out=out)
            out.sycl_queue.wait()
            best = min(best, time.perf_counter() - start)
        return best

    # 16 times as many: about 6 times the time (a call's fixed costs are part of both); every token through the whole list: 200
    assert seconds(16000) < 50 * seconds(1000)


# ---- a bias without a weight -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt,bdt", [("f2", "f2"), ("f2", "f4"), ("f4", "f4"), ("f8", "f8")])
@pytest.mark.parametrize("rows,n", [(1, 5), (5, 100), (130, 1000), (700, 96), (130, 9001), (40, 40000)])
def test_layer_norm_grad_of_a_bias_alone(rows, n, dt, bdt):
    rng = np.random.default_rng(n)
    x, dy = rng.standard_normal((rows, n)).astype(dt), rng.standard_normal((rows, n)).astype(dt)
    _, mean, rstd = dpt.layer_norm(dev(x), None, dev(np.ones(n, bdt)), stats=True)
    out = dpt.full(n, 7, dtype=bdt)
    dx, dw, db = dpt.layer_norm_grad(dev(dy), dev(x), mean, rstd, out=(None, None, out))
    assert dw is None and db is out
    # dx and dbias as with a weight of ones of that type
    want = dpt.layer_norm_grad(dev(dy), dev(x), mean, rstd, dev(np.ones(n, bdt)))
    assert np.array_equal(host(dx), host(want[0])) and np.array_equal(host(db), host(want[2]))
    tol = ref.layer_norm_grad_tolerances(dy, x, host(mean), host(rstd), np.ones(n, bdt))[2]
    within(db, dy.astype(W).sum(0), tol)
    xd, pair = dev(dy), dpt.full(2 * n, 7, dtype=bdt)  # in place, and into every other element
    dpt.layer_norm_grad(xd, dev(x), mean, rstd, out=(xd, None, pair[::2]))
    assert np.array_equal(host(xd), host(dx)) and np.array_equal(host(pair)[::2], host(db)) and (host(pair)[1::2] == 7).all()
    assert dpt.layer_norm_grad(dev(dy), dev(x), mean, rstd)[1:] == (None, None)


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
def test_layer_norm_mean_of_rows_about_zero(dt):
    """Multiples of 2^-9 up to 4, 4095 of them: every partial sum is exact (2^23 multiples at most), so the mean is off by its last
    two roundings, 3 u of itself, although the differences from it are rounded at their own, far larger size."""
    rng = np.random.default_rng(6)
    x = (np.clip(np.round(rng.standard_normal((200, 4095)) * 512), -2048, 2048) / 512).astype(dt)
    mean = host(dpt.layer_norm(dev(x), stats=True)[1])
    want = x.astype(W).mean(1)
    assert (np.abs(mean - want) <= 3 * W(ref.unit(dt)) * np.abs(want)).all()

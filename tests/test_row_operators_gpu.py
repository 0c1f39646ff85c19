"""layer_norm, layer_norm_grad, distill_topk, distill_topk_grad and process_logits against plain 64-bit forms."""
import numpy as np
import pytest

import dpnp_amd as dpnp
import dpnp_amd.tensor as dpt
from tests import row_operator_references as ref
from tests.helpers import dev, dev_view_like, host

pytestmark = pytest.mark.gpu
TYPES = [("f2", "f2"), ("f2", "f4"), ("f4", "f4"), ("f8", "f8")]


def within(got, want, tol, what=""):
    got = host(got) if not isinstance(got, np.ndarray) else got
    assert got.shape == want.shape, (what, got.shape, want.shape)
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got.astype("f8") - want) <= tol)
    same = (got.astype("f8") == want) | (np.isnan(got) & np.isnan(want))
    bad &= ~same
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(),
                           got[bad][:3], want[bad][:3], np.broadcast_to(tol, want.shape)[bad][:3])


def norm_data(rng, shape, dt, wdt):
    n = shape[-1]
    x = (rng.standard_normal(shape) * np.exp(rng.standard_normal(n) * 0.5) + rng.standard_normal(n)).astype(dt)
    return x, (1 + 0.3 * rng.standard_normal(n)).astype(wdt), rng.standard_normal(n).astype(wdt)


def check_norm(x, w, b, xd=None, eps=1e-5, **kw):
    y, mean, rstd = dpt.layer_norm(dev(x) if xd is None else xd, None if w is None else dev(w), None if b is None else dev(b),
                                   eps=eps, stats=True, **kw)
    wy, wm, wr, _ = ref.layer_norm(x, w, b, eps)
    ty, tm, tr = ref.layer_norm_tolerances(x, w, b, eps)
    assert y.dtype == x.dtype and mean.dtype == rstd.dtype == (np.float64 if x.dtype == np.float64 else np.float32)
    within(y, wy, ty, "y")
    within(mean, wm, tm, "mean")
    within(rstd, wr, tr, "rstd")
    return y, mean, rstd


def check_norm_grad(rng, x, w, mean, rstd, xd=None, dyd=None, dy=None, **kw):
    dy = rng.standard_normal(x.shape).astype(x.dtype) if dy is None else dy
    m, s = host(mean), host(rstd)
    got = dpt.layer_norm_grad(dev(dy) if dyd is None else dyd, dev(x) if xd is None else xd, mean, rstd,
                              None if w is None else dev(w), **kw)
    want, tol = ref.layer_norm_grad(dy, x, m, s, w)[:3], ref.layer_norm_grad_tolerances(dy, x, m, s, w)
    within(got[0], want[0], tol[0], "dx")
    if w is None:
        assert got[1] is None and got[2] is None
    else:
        assert got[1].dtype == got[2].dtype == w.dtype
        within(got[1], want[1], tol[1], "dweight")
        within(got[2], want[2], tol[2], "dbias")
    return got


# every way a row is shared out (lanes of a wave, a wave, blocks, the looped kernels), at and around its limits
LENGTHS = [1, 2, 3, 7, 8, 9, 31, 33, 64, 65, 127, 128, 129, 255, 257, 500, 512, 513, 1000, 1024, 1025, 2047, 2048, 2049, 4096,
           4100, 6143, 8191, 8192, 8193, 12288, 16384, 16385, 20001, 32768, 40003, 65536, 66000]


@pytest.mark.parametrize("dt,wdt", TYPES)
@pytest.mark.parametrize("n", LENGTHS)
def test_layer_norm_lengths(n, dt, wdt):
    rng = np.random.default_rng(n)
    x, w, b = norm_data(rng, (5, n), dt, wdt)
    _, mean, rstd = check_norm(x, w, b)
    check_norm_grad(rng, x, w, mean, rstd)


@pytest.mark.parametrize("dt,wdt", TYPES)
@pytest.mark.parametrize("n", LENGTHS)
def test_layer_norm_grad_of_more_rows(n, dt, wdt):
    # around the number of rows up to which the parameters' gradients need no second launch, and in place, which needs it
    rng = np.random.default_rng(n)
    x, w, b = norm_data(rng, (130, n), dt, wdt)
    _, mean, rstd = dpt.layer_norm(dev(x), dev(w), dev(b), stats=True)
    for r in (127, 128, 129, 130) if n < 600 else (129,):
        check_norm_grad(rng, x[:r], w, mean[:r], rstd[:r])
    dy = rng.standard_normal((3, n)).astype(dt)
    want = dpt.layer_norm_grad(dev(dy), dev(x[:3]), mean[:3], rstd[:3], dev(w))
    for which in (0, 1):
        dyd, xd = dev(dy), dev(x[:3])
        got = check_norm_grad(rng, x[:3], w, mean[:3], rstd[:3], xd=xd, dyd=dyd, dy=dy, out=((dyd, xd)[which], None, None))
        assert got[0] is (dyd, xd)[which] and np.array_equal(host(got[0]), host(want[0]))


@pytest.mark.parametrize("dt,wdt", [("f2", "f4"), ("f4", "f4"), ("f8", "f8")])
@pytest.mark.parametrize("shape", [(1, 1024), (1000, 8), (4097, 24), (2049, 100), (3001, 129), (1030, 1000), (700, 2056), (530, 4104),
                                   (259, 8200), (3, 5, 7, 64), (16, 0), (0, 16), (2, 0, 3)])
def test_layer_norm_rows(shape, dt, wdt):
    rng = np.random.default_rng(sum(shape))
    if shape[-1] == 0:
        x = dpt.empty(shape, dtype=dt)
        with pytest.raises(ValueError, match="no elements"):
            dpt.layer_norm(x)
        return
    x, w, b = norm_data(rng, shape, dt, wdt)
    if 0 in shape:
        y, mean, rstd = dpt.layer_norm(dev(x), dev(w), dev(b), stats=True)
        assert y.shape == shape and mean.shape == shape[:-1]
        dx, dw, db = dpt.layer_norm_grad(dev(x), dev(x), mean, rstd, dev(w))
        assert dx.shape == shape and not host(dw).any() and not host(db).any()
        return
    _, mean, rstd = check_norm(x, w, b)
    check_norm_grad(rng, x, w, mean, rstd)


@pytest.mark.parametrize("dt,n", [("f2", 65537), ("f4", 32769), ("f8", 16385)])
def test_layer_norm_many_long_rows(dt, n):
    # more rows that do not fit a block's registers than blocks run at once
    rng = np.random.default_rng(n)
    few, w, b = norm_data(rng, (13, n), dt, dt)
    xd, want = dpt.broadcast_to(dev(few), (101, 13, n)), [host(a) for a in check_norm(few, w, b)]
    out = dpt.full(xd.shape, 7, dtype=dt)
    stats = [dpt.full(xd.shape[:-1], 7, dtype="f8" if dt == "f8" else "f4") for _ in range(2)]
    dpt.layer_norm(xd, dev(w), dev(b), stats=True, out=(out, *stats))
    for got, one in zip((out, *stats), want):
        got = host(got)
        assert got.shape == (101,) + one.shape and (got == one).all()


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
def test_layer_norm_without_parameters(dt):
    rng = np.random.default_rng(3)
    x, w, b = norm_data(rng, (33, 300), dt, dt)
    check_norm(x, None, None)
    check_norm(x, w, None)
    _, mean, rstd = check_norm(x, None, b, eps=0.0)
    check_norm_grad(rng, x, None, mean, rstd)
    y = dpt.layer_norm(dev(x), dev(w), dev(b))  # without statistics: the same y
    assert np.array_equal(host(y), host(dpt.layer_norm(dev(x), dev(w), dev(b), stats=True)[0]))


def layouts(rng, dt):
    """(name, whole host array, view of it) of arrays whose rows lie in other ways than one after the other"""
    base = rng.standard_normal((6, 9, 80)).astype(dt)
    yield "columns of a wider matrix", base[0], base[0][:, 3:70]
    yield "every other row, reversed", base[0], base[0][::-2]
    yield "rows that do not collapse", base, base[:, 1:8, :65]
    yield "permuted rows", base, base[:, ::3, 5:].transpose(1, 0, 2)
    yield "a strided last axis", base, base[:, :, ::2]
    yield "a transposed matrix", base[0], base[0].T
    yield "a reversed last axis", base, base[:, :, ::-1]
    yield "one row for all", base[0], np.broadcast_to(base[0, :1], (9, 80))
    yield "one vector", base[0, 0], base[0, 0][1:]


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
def test_layer_norm_layouts(dt):
    rng = np.random.default_rng(11)
    for name, whole, x in layouts(rng, dt):
        xd = dev_view_like(x, np.ascontiguousarray(whole))
        w, b = norm_data(rng, x.shape, dt, dt)[1:]
        _, mean, rstd = check_norm(x, w, b, xd=xd)
        check_norm_grad(rng, x, w, mean, rstd, xd=xd)
        # into an array of another layout: every other column of a wider one, the rest of it left as it was
        wide = dpt.full(x.shape[:-1] + (2 * x.shape[-1],), 7, dtype=dt)
        out = wide[..., ::2]
        y = dpt.layer_norm(xd, dev(w), dev(b), out=out)
        assert y is out
        got = host(wide)
        assert np.array_equal(got[..., ::2], host(dpt.layer_norm(xd, dev(w), dev(b)))), name
        assert (got[..., 1::2] == 7).all()
        # and into rows that are part of wider ones (unit stride, odd pitch)
        wide = dpt.full(x.shape[:-1] + (x.shape[-1] + 3,), 7, dtype=dt)
        out = wide[..., 2:2 + x.shape[-1]]
        dpt.layer_norm(xd, dev(w), dev(b), out=out)
        got = host(wide)
        assert np.array_equal(got[..., 2:-1], host(dpt.layer_norm(xd, dev(w), dev(b)))), name
        assert (got[..., :2] == 7).all() and (got[..., -1] == 7).all()


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("n", [5, 100, 1024, 3001, 20003, 70000])
def test_layer_norm_in_place(n, dt):
    rng = np.random.default_rng(n)
    x, w, b = norm_data(rng, (7, n), dt, dt)
    want = host(dpt.layer_norm(dev(x), dev(w), dev(b)))
    xd = dev(x)
    assert dpt.layer_norm(xd, dev(w), dev(b), out=xd) is xd
    assert np.array_equal(host(xd), want)
    xd = dev(x)  # overlapping in another way: computed in a temporary
    dpt.layer_norm(xd[:-1], dev(w), dev(b), out=xd[1:])
    assert np.array_equal(host(xd)[1:], want[:-1]) and np.array_equal(host(xd)[0], x[0])
    _, mean, rstd = dpt.layer_norm(dev(x), dev(w), dev(b), stats=True)
    dy = rng.standard_normal(x.shape).astype(dt)
    want = [host(a) for a in dpt.layer_norm_grad(dev(dy), dev(x), mean, rstd, dev(w))]
    for which in (0, 1):
        d, xx = dev(dy), dev(x)
        got = dpt.layer_norm_grad(d, xx, mean, rstd, dev(w), out=((d, xx)[which], None, None))
        assert got[0] is (d, xx)[which]
        assert all(np.array_equal(host(g), k) for g, k in zip(got, want))


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("n", [24, 700, 5000])
def test_layer_norm_special_values(n, dt):
    """Infinities and NaN stay in their rows; constant rows, large offsets and tiny values are within the bounds."""
    rng = np.random.default_rng(8)
    x, w, b = norm_data(rng, (8, n), dt, dt)
    x[0] = 3
    x[1] = 0
    x[2] = x[2] + 30  # far from zero
    x[3] = x[3] * 1e-3
    x[4, 1] = 1000  # one large channel, the second element
    clean = x.copy()
    x[5, n // 2] = np.nan
    x[6, 0] = np.inf
    x[7, n - 1] = -np.inf
    y, mean, rstd = (host(a) for a in dpt.layer_norm(dev(x), dev(w), dev(b), stats=True))
    wy = ref.layer_norm(clean, w, b, 1e-5)[0]
    ty = ref.layer_norm_tolerances(clean, w, b, 1e-5)[0]
    within(y[:5], wy[:5], ty[:5])
    assert np.isnan(y[5:]).all() and np.isnan(mean[5]) and np.isnan(rstd[5:]).all()
    y0 = host(dpt.layer_norm(dev(x[:1]), dev(w), dev(b), eps=0.0))
    assert np.isnan(y0).all()  # 0 / 0: a constant row without eps


def test_layer_norm_grad_is_the_slope():
    """dx, dweight and dbias against central differences of the forward pass, in float64."""
    rng = np.random.default_rng(4)
    x, w, b = norm_data(rng, (3, 37), "f8", "f8")
    dy = rng.standard_normal(x.shape)
    _, mean, rstd = dpt.layer_norm(dev(x), dev(w), dev(b), stats=True)
    got = [host(a) for a in dpt.layer_norm_grad(dev(dy), dev(x), mean, rstd, dev(w))]
    # step 1e-5: truncation ~ third derivative x 1e-10 / 6, cancellation ~ 1e-16 x |sum| / 1e-5; 1e-7 covers both here
    h = 1e-5
    f = lambda *a: float((host(dpt.layer_norm(*(dev(v) for v in a))) * dy).sum())  # noqa: E731
    for which, arr in enumerate((x, w, b)):
        for at in [tuple(rng.integers(0, s) for s in arr.shape) for _ in range(6)]:
            hi, lo = arr.copy(), arr.copy()
            hi[at] += h
            lo[at] -= h
            args = [x, w, b]
            up, down = args[:], args[:]
            up[which], down[which] = hi, lo
            assert abs((f(*up) - f(*down)) / (2 * h) - got[which][at]) < 1e-7


def test_layer_norm_results_do_not_vary():
    rng = np.random.default_rng(5)
    x, w, b = (dev(a) for a in norm_data(rng, (5000, 777), "f4", "f4"))
    dy = dev(rng.standard_normal((5000, 777)).astype("f4"))
    _, mean, rstd = dpt.layer_norm(x, w, b, stats=True)
    first = [host(a) for a in dpt.layer_norm_grad(dy, x, mean, rstd, w)]
    for _ in range(4):
        assert all(np.array_equal(host(a), k) for a, k in zip(dpt.layer_norm_grad(dy, x, mean, rstd, w), first))


# ---- distillation ----------------------------------------------------------------------------------------------------
def distill_data(rng, r, v, k, dt, tdt=None, itype="i4"):
    z = (1.5 * rng.standard_normal((r, v))).astype(dt)
    tok = np.stack([rng.permutation(v)[:k] if k <= v else rng.integers(0, v, k) for _ in range(r)]).astype(itype)
    t = (6 - np.cumsum(rng.uniform(0, 0.4, (r, k)), 1)).astype(tdt or ("f8" if dt == "f8" else "f4"))
    return z, t, tok


def check_distill(z, t, tok, temp=1.0, weights=None, zd=None, td=None, kd=None, wd=None, tight=True, **kw):
    lead, v = z.shape[:-1], z.shape[-1]
    flat = lambda a: a.reshape(-1, a.shape[-1])  # noqa: E731
    zd, td, kd = dev(z) if zd is None else zd, dev(t) if td is None else td, dev(tok) if kd is None else kd
    wd = None if weights is None else dev(weights) if wd is None else wd
    d = ref.distill(flat(z), flat(t), flat(tok), temp, None if weights is None else weights.reshape(-1))
    tl, tg = ref.distill_tolerances(flat(z), flat(t), flat(tok), temp, None if weights is None else weights.reshape(-1))
    loss = dpt.distill_topk(zd, td, kd, temperature=temp)
    assert loss.dtype == (np.float64 if z.dtype == np.float64 else np.float32)
    within(loss, d["loss"].reshape(lead), tl.reshape(lead), "loss")
    loss2, dz = dpt.distill_topk_grad(zd, td, kd, wd, temperature=temp, **kw)
    within(loss2, d["loss"].reshape(lead), tl.reshape(lead), "loss with gradient")
    assert dz.dtype == z.dtype
    within(dz, d["grad"].reshape(z.shape), tg.reshape(z.shape), "dlogits")
    return loss2, dz


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("v", [1, 2, 3, 7, 8, 9, 255, 1000, 4095, 4096, 8191, 8200, 32768, 50003, 100003, 131072, 140001])
def test_distill_vocabularies(v, dt):
    rng = np.random.default_rng(v)
    z, t, tok = distill_data(rng, 3, v, min(20, v), dt)
    check_distill(z, t, tok)


@pytest.mark.parametrize("dt,tdt,itype,temp", [("f2", "f2", "i4", 1.0), ("f2", "f4", "i8", 2.0), ("f4", "f4", "i8", 0.5), ("f4", "f4", "i4", 4.0),
                                               ("f8", "f8", "i4", 1.7)])
@pytest.mark.parametrize("r,v,k", [(1, 5000, 1), (1, 30000, 256), (2, 300, 257), (5, 1000, 1000), (600, 700, 8), (1100, 1030, 33),
                                   (2, 4000, 2048), (300, 20011, 64), (200, 33001, 5), (2, 90001, 300)])
def test_distill_rows_and_entries(r, v, k, dt, tdt, itype, temp):
    rng = np.random.default_rng(r + v + k)
    z, t, tok = distill_data(rng, r, v, k, dt, tdt, itype)
    w = rng.uniform(-1, 2, r).astype("f8" if dt == "f8" else "f4")
    check_distill(z, t, tok, temp, w)


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("v", [50, 9001])
def test_distill_absent_repeated_and_empty(v, dt):
    rng = np.random.default_rng(6)
    z, t, tok = distill_data(rng, 8, v, 12, dt)
    tok[0, 5:] = -1          # a short list
    tok[1] = -1              # an empty one
    tok[2, ::2] = v          # just outside
    tok[3] = 2 ** 31 - 1
    tok[4, 1:] = tok[4, 0]   # one token twelve times
    tok[5, 6:] = tok[5, :6]  # each twice
    t[6] = -np.inf           # every entry without weight: an empty row
    t[7, 3:] = -np.inf
    loss, dz = check_distill(z, t, tok, 1.5)
    loss, dz = host(loss), host(dz)
    for r in (1, 3, 6):
        assert loss[r] == 0 and not dz[r].any()
    z0, t0, k0 = dev(z), dpt.empty((8, 0), dtype=t.dtype), dpt.empty((8, 0), dtype="i4")
    loss, dz = dpt.distill_topk_grad(z0, t0, k0)
    assert not host(loss).any() and not host(dz).any()


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("v", [600, 40000, 140001])
@pytest.mark.parametrize("k", [63, 65, 257, 2048])
def test_distill_many_entries_some_repeated(v, k, dt):
    rng = np.random.default_rng(k)
    z, t, tok = distill_data(rng, 6, v, k, dt)
    tok[0] = rng.integers(0, v, k)          # as they fall
    tok[1] = rng.integers(0, 5, k) * 64     # few tokens, neighbours in a table of a power of two
    tok[2, k // 2:] = tok[2, :k - k // 2]   # each twice, far apart
    tok[3, 1:] = -1                         # one entry and none else
    tok[4] = np.arange(k) % v               # one after the other
    check_distill(z, t, tok)


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("v", [40, 70000])
def test_distill_special_values(v, dt):
    """What NaN and infinities in the logits, the teacher and the weights come to, row by row."""
    rng = np.random.default_rng(7)
    z, t, tok = distill_data(rng, 9, v, 6, dt)
    w = np.ones(9, "f8" if dt == "f8" else "f4")
    others = np.setdiff1d(np.arange(v), tok[0])
    z[0, others[: v // 2]] = -np.inf  # masked tokens that the teacher does not name
    z[1, tok[1, 2]] = -np.inf         # and one that it does: an infinite loss, a finite gradient
    z[2, 3] = np.nan
    z[3] = -np.inf
    z[4, 5] = np.inf
    t[5, 1] = np.nan
    z[6] = np.nan                     # a padded row: weight 0
    w[6] = 0
    z[7] = np.nan                     # a padded row: no entries
    tok[7] = -1
    z[8] = np.finfo(dt).min           # the type's lowest value everywhere but at the teacher's tokens
    z[8, tok[8]] = 0
    loss, dz = (host(a) for a in dpt.distill_topk_grad(dev(z), dev(t), dev(tok), dev(w)))
    d = ref.distill(z, t, tok, 1.0, w)
    for r in (0, 8):
        tl, tg = ref.distill_tolerances(np.maximum(z, -1000)[r:r + 1], t[r:r + 1], tok[r:r + 1],
                                        1.0)  # (exp(-1000) = 0: the same sums)
        within(loss[r:r + 1], d["loss"][r:r + 1], tl)
        within(dz[r], d["grad"][r], 2 * np.finfo(dt).eps + 1e-5 * (dt != "f8"))
    assert loss[1] == np.inf and np.isfinite(dz[1]).all()
    assert np.allclose(dz[1].astype("f8"), d["grad"][1], atol=2 * np.finfo(dt).eps + 1e-6 * (dt != "f8"))
    for r in (2, 3, 4, 5):
        assert np.isnan(loss[r]) and np.isnan(dz[r]).any()
    assert np.isnan(dz[5]).all() and np.isnan(dz[2]).all()
    assert not dz[6].any() and not dz[7].any() and loss[7] == 0


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("r,v", [(3, 1001), (2, 60001), (2, 90001), (1500, 520), (200, 33001)])
def test_distill_in_place_and_layouts(r, v, dt):
    rng = np.random.default_rng(v)
    z, t, tok = distill_data(rng, r, v, 9, dt)
    tok[0, 4] = tok[0, 2]
    want = [host(a) for a in dpt.distill_topk_grad(dev(z), dev(t), dev(tok), temperature=2.0)]
    zd = dev(z)
    loss, dz = dpt.distill_topk_grad(zd, dev(t), dev(tok), temperature=2.0, out=(None, zd))
    assert dz is zd
    assert np.array_equal(host(zd), want[1]) and np.array_equal(host(loss), want[0])
    # rows of a wider array at an odd place, in place; columns strided; one teacher for every row
    wide = np.full((r, v + 5), 3, dt)
    wide[:, 2:2 + v] = z
    wd = dev(wide)
    view = wd[:, 2:2 + v]
    loss, dz = dpt.distill_topk_grad(view, dev(t), dev(tok), temperature=2.0, out=(None, view))
    got = host(wd)
    # (the order of a row's sum goes by where the row starts: held to the bounds, not to the bits)
    d, (tl, tg) = ref.distill(z, t, tok, 2.0), ref.distill_tolerances(z, t, tok, 2.0)
    within(loss, d["loss"], tl, "loss of a view")
    within(got[:, 2:2 + v], d["grad"], tg, "gradient of a view")
    assert (got[:, :2] == 3).all() and (got[:, -3:] == 3).all()
    wd = dev(wide)  # results at another place of their lines than the logits
    dpt.distill_topk_grad(dev(z), dev(t), dev(tok), temperature=2.0, out=(None, wd[:, 3:3 + v]))
    got = host(wd)
    assert np.array_equal(got[:, 3:3 + v], want[1])
    assert np.array_equal(got[:, :3], wide[:, :3]) and np.array_equal(got[:, -2:], wide[:, -2:])
    twice = np.repeat(z, 2, 1)
    loss, dz = dpt.distill_topk_grad(dev(twice)[:, ::2], dev(np.repeat(t, 3, 1))[:, ::3], dev(tok), temperature=2.0)
    assert np.array_equal(host(dz), want[1]) and np.array_equal(host(loss), want[0])
    one = [host(a) for a in dpt.distill_topk_grad(dev(z), dev(np.repeat(t[:1], r, 0)), dev(np.repeat(tok[:1], r, 0)))]
    got = [host(a) for a in dpt.distill_topk_grad(dev(z), dev(t[:1]), dev(tok[0]), dev(np.ones((), "f8" if dt == "f8" else "f4")))]
    assert np.array_equal(got[0], one[0]) and np.array_equal(got[1], one[1])
    # rows in three dims that do not collapse, and a single row without dims
    if r == 3:
        big = rng.standard_normal((4, 3, v)).astype(dt)
        _, t3, k3 = distill_data(rng, 12, v, 9, dt)
        x = big[::2, ::-1]
        check_distill(x, t3.reshape(4, 3, 9)[::2, ::-1], k3.reshape(4, 3, 9)[::2, ::-1], zd=dev_view_like(x, big))
        loss, dz = dpt.distill_topk_grad(dev(z[0]), dev(t[0]), dev(tok[0]), temperature=2.0)
        assert loss.shape == () and np.array_equal(host(dz), want[1][0])


def test_distill_grad_is_the_slope():
    rng = np.random.default_rng(2)
    z, t, tok = distill_data(rng, 3, 60, 7, "f8")
    tok[1, 3] = tok[1, 0]
    tok[2, 5:] = -1
    w = np.array([0.5, 2.0, -1.0])
    dz = host(dpt.distill_topk_grad(dev(z), dev(t), dev(tok), dev(w), temperature=1.6)[1])
    h = 1e-5  # as for layer_norm: 1e-7 covers truncation and cancellation
    for r in range(3):
        for v in list(tok[r, :3]) + list(rng.integers(0, 60, 5)):
            hi, lo = z.copy(), z.copy()
            hi[r, v] += h
            lo[r, v] -= h
            f = [float((host(dpt.distill_topk(dev(a), dev(t), dev(tok), temperature=1.6)) * w).sum()) for a in (hi, lo)]
            assert abs((f[0] - f[1]) / (2 * h) - dz[r, v]) < 1e-7
    assert np.abs(dz.sum(1)).max() < 1e-14 * 60  # softmax gradients of a row add up to nothing


@pytest.mark.parametrize("r,v", [(4, 3000), (2, 40000), (300, 900)])
@pytest.mark.parametrize("offset", [8192.0, -30000.0])
def test_distill_far_logits(r, v, offset):
    """A common offset of a row's logits costs no accuracy: the bounds know only differences from the largest."""
    rng = np.random.default_rng(9)
    z, t, tok = distill_data(rng, r, v, 10, "f4")
    check_distill((z + np.float32(offset)).astype("f4"), t + np.float32(3 * offset), tok, 1.3)


# ---- logits ------------------------------------------------------------------------------------------------------------
def logits_data(rng, r, v, dt, np_=30, no=20, nb=9, itype="i4"):
    z = (3 * rng.standard_normal((r, v))).astype(dt)
    # crowded tokens, some outside
    toks = lambda n: np.where(rng.random((r, n)) < 0.1, rng.choice([-1, v, v + 7, -5]),  # noqa: E731
                              rng.integers(0, max(1, min(v, 40)), (r, n))).astype(itype)
    d = dict(prompt=toks(np_), output=toks(no), btok=np.where(rng.random((r, nb)) < 0.2, -1, rng.integers(0, v, (r, nb))).astype(itype),
             bval=rng.uniform(-5, 5, (r, nb)).astype("f4"),
             plen=rng.integers(-1, np_ + 3, r).astype("i4"), olen=rng.integers(0, no + 1, r).astype("i4"),
             rep=rng.uniform(0.8, 1.6, r).astype("f4"), freq=rng.uniform(-0.5, 1, r).astype("f4"),
             pres=rng.uniform(-0.5, 1, r).astype("f4"),
             allowed=rng.integers(0, 2 ** 32, (r, (v + 31) // 32), dtype="u8").astype("u4"))
    if nb > 2 and v > 2:
        d["btok"][:, 1] = d["btok"][:, 0]  # a bias given twice
    return z, d


NAMES = dict(prompt="prompt_tokens", output="output_tokens", plen="prompt_lengths", olen="output_lengths", btok="bias_tokens",
             bval="bias_values", rep="repetition_penalty", freq="frequency_penalty", pres="presence_penalty", allowed="allowed")


def call_logits(zd, d, **kw):
    return dpt.process_logits(zd, **{NAMES[k]: (v if np.isscalar(v) else dev(v)) for k, v in d.items()}, **kw)


def check_logits(z, d, zd=None, **kw):
    got = call_logits(dev(z) if zd is None else zd, d, **kw)
    want, tol, same = ref.process_logits(z, **d)
    within(got, want, tol, sorted(d))
    g = host(got)
    assert np.array_equal(g[same], z[same], equal_nan=True)
    return got


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("v", [1, 5, 31, 32, 33, 100, 4095, 4096, 4097, 8192, 20011])
def test_logits_everything(v, dt):
    rng = np.random.default_rng(v)
    z, d = logits_data(rng, 4, v, dt)
    check_logits(z, d)


@pytest.mark.parametrize("itype", ["i4", "i8"])
def test_logits_each_part(itype):
    rng = np.random.default_rng(1)
    z, d = logits_data(rng, 3, 5000, "f4", itype=itype)
    parts = [("prompt", "rep"), ("output", "rep"), ("output", "freq"), ("output", "pres"), ("prompt", "plen", "rep", "freq", "pres"),
             ("btok", "bval"), ("allowed",), ("output", "olen", "freq", "allowed"), ()]
    for p in parts:
        check_logits(z, {k: d[k] for k in p})
    check_logits(z, dict(prompt=d["prompt"], output=d["output"], rep=1.3, freq=np.float32(0.25), pres=2))
    d["allowed"] = d["allowed"].view("i4")
    check_logits(z, {"allowed": d["allowed"]})
    for n in (0, 1):  # lists without entries, and of one
        check_logits(z, dict(d, prompt=d["prompt"][:, :n], output=d["output"][:, :n], btok=d["btok"][:, :n], bval=d["bval"][:, :n],
                             plen=np.minimum(d["plen"], n), olen=np.minimum(d["olen"], n)))


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
def test_logits_long_history_and_many_rows(dt):
    rng = np.random.default_rng(2)
    z, d = logits_data(rng, 2, 9001, dt, np_=5003, no=40000, nb=700)
    d["plen"][:] = [5003, 17]
    d["olen"][:] = [40000, 39999]
    check_logits(z, d)
    z, d = logits_data(rng, 300, 260, dt, nb=700)  # more biases in a block's part of the vocabulary than it lists
    check_logits(z, d)
    for r, v in ((600, 260), (400, 20011), (70, 70003)):  # many rows: blocks that go through several parts of a row
        z, d = logits_data(rng, r, v, dt, 50, 30, nb=20)
        d["prompt"][:, 20:] = np.where(d["prompt"][:, 20:] >= 0, rng.integers(0, v, (r, 30)), -1)
        check_logits(z, d)
    check_logits(z, {"allowed": d["allowed"]})  # ... and without lists
    z, d = logits_data(rng, 1, 131072, dt, 700, 300)
    check_logits(z, d)


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
@pytest.mark.parametrize("parts", ["all", "no mask"])
def test_logits_in_place_and_layouts(dt, parts):
    rng = np.random.default_rng(3)
    z, d = logits_data(rng, 4, 6007, dt)
    if parts == "no mask":
        del d["allowed"]
    want = host(call_logits(dev(z), d))
    zd = dev(z)
    assert call_logits(zd, d, out=zd) is zd
    assert np.array_equal(host(zd), want)
    wide = np.full((4, 6007 + 4), 2, dt)
    wide[:, 1:-3] = z
    wd = dev(wide)
    call_logits(wd[:, 1:-3], d, out=wd[:, 1:-3])
    got = host(wd)
    assert np.array_equal(got[:, 1:-3], want) and (got[:, :1] == 2).all() and (got[:, -3:] == 2).all()
    wd = dev(np.full((4, 6007 + 4), 2, dt))
    call_logits(dev(z), d, out=wd[:, 3:-1])  # results at another place of their lines than the logits
    got = host(wd)
    assert np.array_equal(got[:, 3:-1], want) and (got[:, :3] == 2).all() and (got[:, -1:] == 2).all()
    zd = dev(z)
    call_logits(zd[:-1], {k: a[:-1] for k, a in d.items()}, out=zd[1:])  # rows one further down: through a temporary
    assert np.array_equal(host(zd)[1:], want[:-1])
    assert np.array_equal(host(call_logits(dev(np.repeat(z, 2, 1))[:, ::2], d)), want)
    rev = dev(z)[::-1]
    assert np.array_equal(host(call_logits(rev, {k: np.ascontiguousarray(a[::-1]) for k, a in d.items()})), want[::-1])
    z3 = dev(z.reshape(2, 2, -1))
    d3 = {k: a.reshape((2, 2) + a.shape[1:]) for k, a in d.items()}
    assert np.array_equal(host(call_logits(z3, d3)).reshape(4, -1), want)
    # side arrays of one row serve every row; a single row without dims
    d1 = {k: np.asarray(a[0]) for k, a in d.items()}
    every = {k: np.repeat(a[:1], 4, 0) for k, a in d.items()}
    assert np.array_equal(host(call_logits(dev(z), d1)), host(call_logits(dev(z), every)))
    assert np.array_equal(host(call_logits(dev(z[0]), d1)), want[0])


@pytest.mark.parametrize("dt", ["f2", "f4", "f8"])
def test_logits_special_values(dt):
    rng = np.random.default_rng(4)
    z, d = logits_data(rng, 4, 100, dt)
    z[0, ::3] = np.nan
    z[1, ::3] = -np.inf
    z[2, ::3] = np.inf
    z[3, ::3] = np.finfo(dt).min
    d["rep"][:] = 1.5
    d["allowed"][2] = 0  # nothing allowed
    got = host(call_logits(dev(z), d))
    with np.errstate(over="ignore"):
        want, tol, same = ref.process_logits(z, **d)
        rounded = want.astype(dt)
    assert (got[2] == -np.inf).all()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(rounded)
    assert np.array_equal(got[inf].astype("f8"), rounded[inf].astype("f8"))  # the lowest value times 1.5 overflows to -inf
    fine = np.isfinite(rounded)
    within(got[fine], want[fine], tol[fine])


def test_row_operators_on_dpnp_arrays():
    """The NumPy-flavoured functions: dpnp arrays in and out, `out` handed back."""
    rng = np.random.default_rng(0)
    x, w, b = norm_data(rng, (6, 50), "f4", "f4")
    X, W, B = dpnp.array(x), dpnp.array(w), dpnp.array(b)
    y, mean, rstd = dpnp.layer_norm(X, W, B, stats=True)
    assert all(isinstance(a, dpnp.ndarray) for a in (y, mean, rstd))
    out = dpnp.empty((6, 50), dtype="f4")
    assert dpnp.layer_norm(X, W, B, out=out) is out and np.array_equal(out.asnumpy(), y.asnumpy())
    outs = (dpnp.empty((6, 50), dtype="f4"), None, dpnp.empty((50,), dtype="f4"))
    got = dpnp.layer_norm_grad(y, X, mean, rstd, W, out=outs)
    assert got[0] is outs[0] and got[2] is outs[2] and isinstance(got[1], dpnp.ndarray)
    assert dpnp.layer_norm_grad(y, X, mean, rstd)[1:] == (None, None)
    z, t, tok = distill_data(rng, 4, 90, 5, "f4")
    Z, T, K = dpnp.array(z), dpnp.array(t), dpnp.array(tok)
    loss = dpnp.distill_topk(Z, T, K)
    l2, dz = dpnp.distill_topk_grad(Z, T, K, dpnp.ones(4, dtype="f4"), out=(None, Z))
    assert dz is Z
    d, (tl, tg) = ref.distill(z, t, tok, 1.0), ref.distill_tolerances(z, t, tok, 1.0)
    within(loss.asnumpy(), d["loss"], tl)
    within(l2.asnumpy(), d["loss"], tl)
    within(Z.asnumpy(), d["grad"], tg)
    z, d = logits_data(rng, 4, 90, "f4")
    r = dpnp.process_logits(dpnp.array(z), prompt_tokens=dpnp.array(d["prompt"]), repetition_penalty=1.25,
                            allowed=dpnp.array(d["allowed"]))
    want, tol, _ = ref.process_logits(z, prompt=d["prompt"], rep=1.25, allowed=d["allowed"])
    within(r.asnumpy(), want, tol)


def test_rows_beyond_32_bit_offsets():
    # six rows of an array of 4.6e9 elements: their offsets pass 2^31 and 2^32
    rng = np.random.default_rng(8)
    n, every = 65600, 14001
    far = lambda: dpt.empty((5 * every + 1, n), dtype="f2")[::every]  # noqa: E731
    x, w, b = norm_data(rng, (6, n), "f2", "f4")
    xd, out = far(), far()
    xd[:, :] = dev(x)
    assert xd.strides[0] * 5 > 2 ** 32
    for m in (n, 4001):  # the looped kernels and those that hold the row
        y, mean, rstd = dpt.layer_norm(xd[:, :m], dev(w[:m]), dev(b[:m]), stats=True, out=(out[:, :m], None, None))
        want = dpt.layer_norm(dev(x[:, :m].copy()), dev(w[:m]), dev(b[:m]), stats=True)
        for got, one in zip((y, mean, rstd), want):
            assert np.array_equal(host(got), host(one))
        got = dpt.layer_norm_grad(y, xd[:, :m], mean, rstd, dev(w[:m]), out=(out[:, :m], None, None))
        one = dpt.layer_norm_grad(want[0], dev(x[:, :m].copy()), mean, rstd, dev(w[:m]))
        for g, o in zip(got, one):
            assert np.array_equal(host(g), host(o))
    t, tok = rng.standard_normal((6, 9)).astype("f4"), rng.permutation(n)[:54].reshape(6, 9).astype("i4")
    check_distill(x, t, tok, zd=xd, out=(None, out))
    tok = dev(tok)
    got = dpt.process_logits(xd, prompt_tokens=tok, output_tokens=tok, repetition_penalty=1.5, presence_penalty=0.25, out=out)
    one = dpt.process_logits(dev(x), prompt_tokens=tok, output_tokens=tok, repetition_penalty=1.5, presence_penalty=0.25)
    assert np.array_equal(host(got), host(one))


def test_results_that_share_memory_are_refused():
    x = dpt.ones((6, 8), dtype="f4")
    pair = dpt.empty(8, dtype="f4")
    for out in ((None, pair[:6], pair[:6]), (None, pair[2:], pair[:6]), (x, x[:, 0], None)):
        with pytest.raises(ValueError, match="overlap"):
            dpt.layer_norm(x, stats=True, out=out)
    w = dpt.ones(8, dtype="f4")
    _, mean, rstd = dpt.layer_norm(x, stats=True)
    with pytest.raises(ValueError, match="overlap"):
        dpt.layer_norm_grad(x, x, mean, rstd, w, out=(None, w, w))
    wide = dpt.empty((6, 16), dtype="f4")
    with pytest.raises(ValueError, match="overlap"):
        dpt.distill_topk_grad(x, x[:, :2], dpt.zeros((6, 2), dtype="i4"), out=(wide[:, 2], wide[:, ::2]))


def test_millions_of_short_rows():
    rng = np.random.default_rng(12)
    x, w, b = norm_data(rng, (2 ** 21 + 3, 5), "f4", "f4")
    _, mean, rstd = check_norm(x, w, b)
    dy = rng.standard_normal(x.shape).astype("f4")
    dx, dw, db = dpt.layer_norm_grad(dev(dy), dev(x), mean, rstd, dev(w))
    want, tol = ref.layer_norm_grad(dy, x, host(mean), host(rstd), w)[:3], ref.layer_norm_grad_tolerances(dy, x, host(mean), host(rstd), w)
    for got, one, t in zip((dx, dw, db), want, tol):
        within(got, one, t)
    z, t, tok = distill_data(rng, 100003, 7, 3, "f4")
    check_distill(z, t, tok)
    z, d = logits_data(rng, 2003, 9, "f4")
    check_logits(z, d)


def test_logits_empty_and_very_long_lists():
    rng = np.random.default_rng(14)
    z = rng.standard_normal((3, 1009)).astype("f4")
    none = dpt.empty((3, 0), dtype="i8")
    out = dpt.process_logits(dev(z), prompt_tokens=none, output_tokens=none, repetition_penalty=2.0, frequency_penalty=1.0,
                             bias_tokens=none, bias_values=dpt.empty((3, 0), dtype="f4"))
    assert np.array_equal(host(out), z)
    tok = rng.integers(-50, 1100, (3, 60001))
    tok[:, ::7] += 2 ** 33  # far outside
    lengths = np.array([60001, 0, 33333], "i4")
    got = host(dpt.process_logits(dev(z), output_tokens=dev(tok), output_lengths=dev(lengths), frequency_penalty=0.5, presence_penalty=0.25))
    for i in range(3):
        here = tok[i, :lengths[i]]
        said = np.bincount(here[(here >= 0) & (here < 1009)], minlength=1009)
        # two products and differences in float32
        tol = 2.0 ** -24 * (4 * 0.5 * said + 2 * np.abs(z[i]) + 1)
        assert (np.abs(got[i] - (z[i].astype("f8") - 0.5 * said - 0.25 * (said > 0))) <= tol).all()
        assert np.array_equal(got[i][said == 0], z[i][said == 0])


def test_calls_from_two_threads():
    import threading
    rng = np.random.default_rng(15)
    sets = []
    for r, n in ((300, 700), (257, 1025)):
        x, w, b = norm_data(rng, (r, n), "f4", "f4")
        a = [dev(v) for v in (x, w, b, rng.standard_normal(x.shape).astype("f4"))]
        z, t, tok = (dev(v) for v in distill_data(rng, 4, 100003, 12, "f4"))

        def call(a=a, z=z, t=t, tok=tok):
            y, mean, rstd = dpt.layer_norm(a[0], a[1], a[2], stats=True)
            return (y, *dpt.layer_norm_grad(a[3], a[0], mean, rstd, a[1]), *dpt.distill_topk_grad(z, t, tok))

        sets.append((call, [host(v) for v in call()]))
    wrong = []

    def many(call, want):
        for _ in range(50):
            wrong.extend(1 for g, k in zip(call(), want) if not np.array_equal(host(g), k))

    threads = [threading.Thread(target=many, args=s) for s in sets]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong

"""The row operators without a GPU: what the C entry points and the Python layer refuse before anything is launched, the
workspace sizes, and the 64-bit forms the GPU tests compare with, checked against differences."""
import ctypes

import numpy as np
import pytest

import dpnp_amd as dpnp
import dpnp_amd._lib as L
import dpnp_amd.tensor as dpt
from dpnp_amd.tensor._usmarray import usm_ndarray
from tests import row_operator_references as ref

lib = L.lib
BASE = 0x7F0000000000  # never dereferenced: every call here is refused, or has nothing to do
_next = [0]


def view(shape, dt=L.FLOAT, strides=None, ptr=None, writable=True):
    shape = list(shape)
    if strides is None:
        strides, acc = [0] * len(shape), 1
        for d in range(len(shape) - 1, -1, -1):
            strides[d] = acc
            acc *= max(shape[d], 1)
    if ptr is None:
        _next[0] += 1
        ptr = BASE + (_next[0] << 34)
    return L.make_view(ptr, shape, strides, dt, L.WRITABLE if writable else 0)


def refused(status, code, match):
    assert status == code, (status, lib.dpx_last_error())
    assert match in lib.dpx_last_error().decode(), lib.dpx_last_error()


def norm(x, w=None, b=None, eps=1e-5, y=None, mean=None, rstd=None):
    return lib.dpx_layer_norm(x, w, b, eps, y, mean, rstd, None)


def test_layer_norm_refusals():
    x, y = view((4, 8)), view((4, 8))
    refused(norm(view((4, 8), L.INT32), y=view((4, 8), L.INT32)), L.ERR_NOT_IMPLEMENTED, "not supported")
    refused(norm(view((4, 8), L.CFLOAT), y=view((4, 8), L.CFLOAT)), L.ERR_NOT_IMPLEMENTED, "not supported")
    refused(norm(view(()), y=view(())), L.ERR_RANK_MISMATCH, "dimension")
    refused(norm(x), L.ERR_BAD_ARGUMENT, "no output")
    refused(norm(x, y=view((4, 9))), L.ERR_SHAPE_MISMATCH, "length 9")
    refused(norm(x, y=view((5, 8))), L.ERR_SHAPE_MISMATCH, "leading")
    refused(norm(x, y=view((4, 2, 4))), L.ERR_RANK_MISMATCH, "dimensions")
    refused(norm(x, y=view((4, 8), L.HALF)), L.ERR_BAD_DTYPE, "float16")
    refused(norm(x, y=view((4, 8), writable=False)), L.ERR_NOT_WRITABLE, "read-only")
    refused(norm(x, y=view((4, 8), strides=(0, 1))), L.ERR_NOT_AMPLE, "ample")
    refused(norm(view((2, 2, 8)), y=view((2, 2, 8), strides=(100, 4, 1))), L.ERR_NOT_AMPLE, "ample")
    refused(norm(x, y=view((4, 8), strides=(16, 2))), L.ERR_NOT_IMPLEMENTED, "unit stride")
    refused(norm(view((4, 8), strides=(1, 4)), y=y), L.ERR_NOT_IMPLEMENTED, "unit stride")
    refused(norm(x, y=view((4, 8), ptr=x.data + 4)), L.ERR_OVERLAP, "overlap")
    refused(norm(x, view((7,)), y=y), L.ERR_SHAPE_MISMATCH, "length 7")
    refused(norm(x, view((1, 8)), y=y), L.ERR_RANK_MISMATCH, "one dimension")
    refused(norm(x, view((8,), strides=(2,)), y=y), L.ERR_NOT_IMPLEMENTED, "unit stride")
    refused(norm(x, view((8,), L.HALF), y=y), L.ERR_NOT_IMPLEMENTED, "float16")
    refused(norm(x, view((8,)), view((8,), L.DOUBLE), y=y), L.ERR_NOT_IMPLEMENTED, "one type")
    refused(norm(x, view((8,), ptr=y.data), y=y), L.ERR_OVERLAP, "overlap")
    refused(norm(x, y=y, mean=view((5,))), L.ERR_SHAPE_MISMATCH, "leading")
    refused(norm(x, y=y, mean=view((4,), L.DOUBLE)), L.ERR_BAD_DTYPE, "float64")
    m = view((4,))
    refused(norm(x, y=y, mean=m, rstd=m), L.ERR_OVERLAP, "overlap")
    for eps in (-1e-6, float("nan"), float("inf")):
        refused(norm(x, y=y, eps=eps), L.ERR_BAD_ARGUMENT, "eps")
    refused(norm(view((4, 0)), y=view((4, 0))), L.ERR_BAD_ARGUMENT, "no elements")
    refused(norm(L.make_view(None, (4, 8), (8, 1), L.FLOAT, 0), y=y), L.ERR_BAD_ARGUMENT, "null")
    assert norm(view((0, 8)), y=view((0, 8))) == L.OK  # nothing to do


def test_layer_norm_grad_refusals():
    # (so many rows that the parameters' gradients need a workspace; few need none)
    R = 400
    x, dy, dx, m, s, w = view((R, 8)), view((R, 8)), view((R, 8)), view((R,)), view((R,)), view((8,))
    dw, db = view((8,)), view((8,))
    ws = ctypes.c_void_p(BASE)
    n = lib.dpx_layer_norm_grad_workspace(x)

    def call(dy=dy, x=x, m=m, s=s, w=w, dx=dx, dw=dw, db=db, ws=ws, n=n):
        return lib.dpx_layer_norm_grad(dy, x, m, s, w, dx, dw, db, ws, n, None)

    assert n > 0 and lib.dpx_layer_norm_grad_workspace(view((0, 8))) == lib.dpx_layer_norm_grad_workspace(view((4, 8))) == 0
    refused(call(n=n - 1), L.ERR_BAD_ARGUMENT, "workspace")
    refused(call(ws=None), L.ERR_BAD_ARGUMENT, "workspace")
    refused(call(ws=ctypes.c_void_p(BASE + 8)), L.ERR_BAD_ARGUMENT, "aligned")
    refused(call(db=None), L.ERR_BAD_ARGUMENT, "together")
    refused(call(dx=None), L.ERR_BAD_ARGUMENT, "needed")
    refused(call(m=None), L.ERR_BAD_ARGUMENT, "needed")
    refused(call(dy=view((R, 8), L.HALF)), L.ERR_NOT_IMPLEMENTED, "float16")
    refused(call(dy=view((3, 8))), L.ERR_SHAPE_MISMATCH, "leading")
    refused(call(m=view((R, 1))), L.ERR_RANK_MISMATCH, "dimensions")
    refused(call(dw=view((8,), L.HALF)), L.ERR_BAD_DTYPE, "type of weight")
    refused(call(dw=view((9,))), L.ERR_SHAPE_MISMATCH, "length 9")
    refused(call(dw=w), L.ERR_OVERLAP, "overlap")
    refused(call(db=dw), L.ERR_OVERLAP, "overlap")
    refused(call(dx=view((R, 8), ptr=w.data)), L.ERR_OVERLAP, "overlap")
    refused(call(dx=view((R, 8), ptr=x.data + 4)), L.ERR_OVERLAP, "overlap")
    refused(call(dw=view((8,), ptr=dy.data)), L.ERR_OVERLAP, "overlap")
    refused(call(w=view((8,), L.DOUBLE), dw=view((8,), L.DOUBLE), db=view((8,), L.DOUBLE)), L.ERR_NOT_IMPLEMENTED, "float64")


def test_distill_refusals():
    # (three long rows: split over blocks, which need a workspace; a block per row needs none)
    V = 200000
    z, t, i, loss, dz = view((3, V)), view((3, 5)), view((3, 5), L.INT32), view((3,)), view((3, V))
    n = lib.dpx_distill_topk_workspace(z, t)
    ws = ctypes.c_void_p(BASE)
    assert n > 0 and lib.dpx_distill_topk_workspace(view((0, V)), t) == 0
    assert lib.dpx_distill_topk_workspace(view((4096, 100)), view((4096, 5))) == 0

    def call(z=z, t=t, i=i, w=None, temp=1.0, loss=loss, dz=dz, ws=ws, n=n):
        return lib.dpx_distill_topk_grad(z, t, i, w, temp, loss, dz, ws, n, None)

    refused(call(n=n - 1), L.ERR_BAD_ARGUMENT, "workspace")
    refused(call(ws=None), L.ERR_BAD_ARGUMENT, "workspace")
    refused(lib.dpx_distill_topk(z, t, i, 1.0, loss, ws, 0, None), L.ERR_BAD_ARGUMENT, "workspace")
    for temp in (0.0, -1.0, float("nan"), float("inf")):
        refused(call(temp=temp), L.ERR_BAD_ARGUMENT, "temperature")
    refused(call(z=view((3, V), L.INT64)), L.ERR_NOT_IMPLEMENTED, "int64")
    refused(call(z=view(())), L.ERR_RANK_MISMATCH, "dimension")
    refused(call(t=view((3, 6))), L.ERR_SHAPE_MISMATCH, "length 5")
    refused(call(t=view((2, 5))), L.ERR_SHAPE_MISMATCH, "leading")
    refused(call(t=view((3, 5), L.HALF)), L.ERR_NOT_IMPLEMENTED, "float16")
    refused(call(i=view((3, 5), L.INT16)), L.ERR_NOT_IMPLEMENTED, "int16")
    refused(call(i=view((3, 5), L.FLOAT)), L.ERR_NOT_IMPLEMENTED, "float32")
    refused(call(w=view((3,), L.DOUBLE)), L.ERR_NOT_IMPLEMENTED, "float64")
    refused(call(w=view((3, 1))), L.ERR_RANK_MISMATCH, "dimensions")
    refused(call(loss=view((3,), L.HALF)), L.ERR_BAD_DTYPE, "float16")
    refused(call(dz=None), L.ERR_BAD_ARGUMENT, "missing")
    refused(call(dz=view((3, V), L.HALF)), L.ERR_BAD_DTYPE, "float16")
    refused(call(dz=view((3, V), ptr=z.data + 4)), L.ERR_OVERLAP, "overlap")
    refused(call(dz=view((3, V), ptr=t.data)), L.ERR_OVERLAP, "overlap")
    refused(call(loss=view((3,), ptr=z.data)), L.ERR_OVERLAP, "overlap")
    refused(call(t=view((3, 2049)), i=view((3, 2049), L.INT32)), L.ERR_BAD_ARGUMENT, "2048")
    refused(call(z=view((3, 0)), dz=view((3, 0))), L.ERR_BAD_ARGUMENT, "no elements")
    refused(call(z=view((1, 1 << 31)), t=view((1, 5)), i=view((1, 5), L.INT32), loss=view((1,)), dz=view((1, 1 << 31))),
            L.ERR_BAD_ARGUMENT, "too long")
    assert call(z=view((0, V)), t=view((0, 5)), i=view((0, 5), L.INT32), loss=view((0,)), dz=view((0, V)), ws=None, n=0) == L.OK


def test_process_logits_refusals():
    z, out = view((3, 100)), view((3, 100))

    def call(z=z, out=out, **kw):
        a = L.LogitsArgs(repetition_value=1.0)
        keep = []
        for k, v in kw.items():
            if isinstance(v, L.ArrayView):
                keep.append(v)
                v = ctypes.pointer(v)
            setattr(a, k, v)
        return lib.dpx_process_logits(z, ctypes.byref(a), out, None)

    i4 = lambda *s: view(s, L.INT32)  # noqa: E731
    refused(lib.dpx_process_logits(z, None, out, None), L.ERR_BAD_ARGUMENT, "missing")
    refused(call(out=None), L.ERR_BAD_ARGUMENT, "missing")
    refused(call(z=view((3, 100), L.INT32)), L.ERR_NOT_IMPLEMENTED, "int32")
    refused(call(out=view((3, 100), L.DOUBLE)), L.ERR_BAD_DTYPE, "float64")
    refused(call(out=view((3, 100), ptr=z.data + 4)), L.ERR_OVERLAP, "overlap")
    refused(call(prompt_tokens=view((3, 7), L.INT16)), L.ERR_NOT_IMPLEMENTED, "int16")
    refused(call(prompt_tokens=i4(2, 7)), L.ERR_SHAPE_MISMATCH, "leading")
    refused(call(prompt_tokens=i4(3, 7), output_tokens=view((3, 7), L.INT64)), L.ERR_BAD_ARGUMENT, "one type")
    refused(call(prompt_lengths=i4(3)), L.ERR_BAD_ARGUMENT, "without tokens")
    refused(call(output_tokens=i4(3, 7), output_lengths=view((3,), L.INT64)), L.ERR_NOT_IMPLEMENTED, "int64")
    refused(call(repetition=view((3,), L.DOUBLE)), L.ERR_NOT_IMPLEMENTED, "float64")
    refused(call(repetition=view((4,))), L.ERR_SHAPE_MISMATCH, "leading")
    for r in (0.0, -1.0, float("nan"), float("inf")):
        refused(call(repetition_value=r), L.ERR_BAD_ARGUMENT, "repetition")
    refused(call(frequency_value=float("nan")), L.ERR_BAD_ARGUMENT, "finite")
    refused(call(presence_value=float("inf")), L.ERR_BAD_ARGUMENT, "finite")
    refused(call(bias_tokens=i4(3, 4)), L.ERR_BAD_ARGUMENT, "together")
    refused(call(bias_tokens=i4(3, 4), bias_values=view((3, 5))), L.ERR_SHAPE_MISMATCH, "length 5")
    refused(call(bias_tokens=i4(3, 4), bias_values=view((3, 4), L.HALF)), L.ERR_NOT_IMPLEMENTED, "float16")
    refused(call(allowed=i4(3, 3)), L.ERR_SHAPE_MISMATCH, "4 is needed")
    refused(call(allowed=view((3, 4), L.INT64)), L.ERR_NOT_IMPLEMENTED, "int64")
    refused(call(prompt_tokens=i4()), L.ERR_RANK_MISMATCH, "last axis")
    refused(call(out=view((3, 100), strides=(200, 2))), L.ERR_NOT_IMPLEMENTED, "unit stride")
    m = i4(3, 4)
    refused(call(allowed=m, out=view((3, 100), ptr=m.data)), L.ERR_OVERLAP, "overlap")
    assert call(z=view((0, 100)), out=view((0, 100))) == L.OK


def fake(shape, dtype="f4"):
    """An array object without memory, for the Python layer's own checks."""
    _next[0] += 1
    at = BASE + (_next[0] << 34)

    class Nothing:
        def numel(self):
            return 1 << 30

        def data_ptr(self):
            return at

    return usm_ndarray(shape, dtype=dtype, buffer=Nothing())


def test_python_layer_refusals():
    x = fake((4, 8))
    with pytest.raises(TypeError, match="usm_ndarray"):
        dpt.layer_norm(np.ones((4, 8), "f4"))
    with pytest.raises(TypeError):
        dpnp.layer_norm(np.ones((4, 8), "f4"))
    with pytest.raises(ValueError, match="does not support"):
        dpt.layer_norm(fake((4, 8), "i4"))
    with pytest.raises(ValueError, match="at least one dimension"):
        dpt.layer_norm(fake(()))
    with pytest.raises(ValueError, match="shape"):
        dpt.layer_norm(x, out=fake((4, 9)))
    with pytest.raises(ValueError, match="type"):
        dpt.layer_norm(x, out=fake((4, 8), "f8"))
    with pytest.raises(ValueError, match="tuple of 3"):
        dpt.layer_norm(x, stats=True, out=fake((4, 8)))
    ro = fake((4, 8))
    ro.flags.writable = False
    with pytest.raises(ValueError, match="read-only"):
        dpt.layer_norm(x, out=ro)
    with pytest.raises(ValueError, match="need weight"):
        dpt.layer_norm_grad(x, x, fake((4,)), fake((4,)), out=(x, fake((8,)), None))
    with pytest.raises(ValueError, match="tuple of 2"):
        dpt.distill_topk_grad(x, x, fake((4, 8), "i4"), out=(x,))
    with pytest.raises(TypeError):
        dpt.distill_topk(x, [1.0], [2])
    with pytest.raises(ValueError):
        dpt.distill_topk(x, fake((3, 8)), fake((4, 8), "i4"))  # rows that do not broadcast
    with pytest.raises(ValueError, match="does not support"):
        dpt.process_logits(fake((4, 8), "i8"))
    with pytest.raises(TypeError):
        dpt.process_logits(x, repetition_penalty="1.0")


def test_reference_gradients_are_slopes():
    """The plain forms against central differences (step 1e-6, cancellation 1e-16 / 1e-6: 1e-8 covers both)."""
    rng = np.random.default_rng(0)
    x, w, b, dy = rng.standard_normal((3, 11)), rng.standard_normal(11), rng.standard_normal(11), rng.standard_normal((3, 11))
    f = lambda x, w, b: (ref.layer_norm(x, w, b, 1e-5)[0] * dy).sum()  # noqa: E731
    _, mean, rstd, _ = ref.layer_norm(x, w, b, 1e-5)
    got = ref.layer_norm_grad(dy, x, mean, rstd, w)[:3]
    for k, a in enumerate((x, w, b)):
        for at in np.ndindex(a.shape):
            hi, lo = [v.copy() for v in (x, w, b)], [v.copy() for v in (x, w, b)]
            hi[k][at] += 1e-6
            lo[k][at] -= 1e-6
            assert abs((f(*hi) - f(*lo)) / 2e-6 - got[k][at]) < 1e-8
    z, t = rng.standard_normal((2, 13)), rng.standard_normal((2, 4))
    tok = np.array([[3, 3, 12, -1], [0, 1, 2, 3]])
    wt = np.array([0.5, 2.0])
    g = ref.distill(z, t, tok, 1.3, wt)["grad"]
    f = lambda z: (ref.distill(z, t, tok, 1.3)["loss"] * wt).sum()  # noqa: E731
    for at in np.ndindex(z.shape):
        hi, lo = z.copy(), z.copy()
        hi[at] += 1e-6
        lo[at] -= 1e-6
        assert abs((f(hi) - f(lo)) / 2e-6 - g[at]) < 1e-8

"""Operators over the last axis as language models use them: layer normalisation and its gradient, distillation from a
teacher's top logits and its gradient, and the processing of logits before a token is chosen.

No counterpart in the reference, where each is a chain of mean, var, logsumexp, where and arithmetic over full-size
temporaries.  The dims before the last one are rows and may have any strides.  Arrays whose last axis is strided are laid out
(copied) first; an `out` that overlaps an operand it may not replace is computed in a temporary, as everywhere in this
package.  Float16, float32 and float64 data; statistics and per-row results are float32, float64 for float64 data.
"""
import numbers

from .. import _lib
from . import _tensor_impl as ti
from ._copy_utils import copy
from ._device import alloc
from ._dtypes import float16, float32, float64
from ._manipulation_functions import broadcast_to
from ._usmarray import usm_ndarray

_ext = _lib.ext
_ext.set_alloc_bytes(alloc)


def _array(a, name):
    if type(a) is not usm_ndarray and not isinstance(a, usm_ndarray):
        raise TypeError(f"Expected `{name}` to be of dpnp.tensor.usm_ndarray type, got {type(a)}")
    return a


def _data(a, fn, name):
    """`a` as data with rows: a floating array whose last axis has unit stride (a copy when it has not)."""
    _array(a, name)
    if a._dtype.kind != "f":
        raise ValueError(f"function '{fn}' does not support input type {a._dtype}")
    if not a._shape:
        raise ValueError(f"function '{fn}': {name} needs at least one dimension")
    return _unit(a)


def _unit(a):
    return a if a._strides[-1] == 1 or a._shape[-1] < 2 else copy(a, order="C")


def _vector(a, name):
    if a is None:
        return None
    _array(a, name)
    return _unit(a) if a._shape else a


def _over_rows(a, lead, name):
    """A side array with a last axis, seen with the rows `lead`: broadcast over them where it lacks them."""
    if a is None:
        return None
    shape = _array(a, name)._shape
    if not shape:
        raise ValueError(f"{name} needs at least one dimension")
    if shape[:-1] != lead:
        a = broadcast_to(a, lead + shape[-1:])
    return a if a._strides[-1] == 1 else _unit(a)


def _per_row(a, lead, name):
    """A side array of one value per row."""
    if a is None:
        return None
    return a if _array(a, name)._shape == lead else broadcast_to(a, lead)


class _Out:
    """A result: the array the kernel writes and the one the caller gets."""

    __slots__ = ("kernel", "user")

    def __init__(self, out, shape, dt, name, operands=(), replaces=()):
        if out is None:
            self.kernel = self.user = usm_ndarray._new_contiguous(shape, dt)
            return
        if not isinstance(out, usm_ndarray):
            raise TypeError(f"output array must be of usm_ndarray type, got {type(out)}")
        if not out._writable:
            raise ValueError("provided `out` array is read-only")
        if out._shape != shape:
            raise ValueError(f"The shape of input and output arrays are inconsistent. Expected {name} of shape {shape}, "
                             f"got {out._shape}")
        if out._dtype != dt:
            raise ValueError(f"Output array of type {dt} is needed for {name}, got {out._dtype}")
        self.user = self.kernel = out
        if not ((not shape or shape[-1] < 2 or out._strides[-1] == 1) and _ext.may_write(out, operands, replaces)):
            self.kernel = usm_ndarray._new_contiguous(shape, dt)

    def done(self):
        if self.kernel is not self.user and self.user.size:
            ti._copy_usm_ndarray_into_usm_ndarray(src=self.kernel, dst=self.user)
        return self.user


def _several(out, n, what):
    if out is None:
        return (None,) * n
    if not isinstance(out, tuple) or len(out) != n:
        raise ValueError(f"`out` must be a tuple of {n} arrays or None: {what}")
    return out


def _apart(*outs):
    """No two results share memory (the kernels' own arrays are checked by the library)."""
    for i, a in enumerate(outs):
        for b in outs[:i]:
            if (a.kernel is not a.user or b.kernel is not b.user) and ti._array_overlap(a.user, b.user):
                raise ValueError("the arrays of two results overlap in memory")


def _acc(dt):
    return float64 if dt == float64 else float32


def layer_norm(x, weight=None, bias=None, /, *, eps=1e-5, stats=False, out=None):
    """(x - mean) * rstd * weight + bias along the last axis, with rstd = 1 / sqrt(variance + eps).

    weight, bias: vectors of the last axis' length, of x's type (or float32 for float16 x); None leaves them out.
    stats: also return the rows' mean and rstd, which `layer_norm_grad` takes.  out: the result's array, (y, mean, rstd) with
    stats; y may be x itself.  Returns y, or (y, mean, rstd).
    """
    x = _data(x, "layer_norm", "x")
    weight, bias = _vector(weight, "weight"), _vector(bias, "bias")
    reads = (x, weight, bias)
    if not stats:
        y = _Out(out, x._shape, x._dtype, "y", reads, (x,))
        _ext.layer_norm(x, weight, bias, float(eps), y.kernel, None, None)
        return y.done()
    oy, om, os = _several(out, 3, "(y, mean, rstd)")
    rows, acc = x._shape[:-1], _acc(x._dtype)
    y = _Out(oy, x._shape, x._dtype, "y", reads, (x,))
    mean, rstd = _Out(om, rows, acc, "mean", reads), _Out(os, rows, acc, "rstd", reads)
    _apart(y, mean, rstd)
    _ext.layer_norm(x, weight, bias, float(eps), y.kernel, mean.kernel, rstd.kernel)
    return y.done(), mean.done(), rstd.done()


def layer_norm_grad(grad, x, mean, rstd, weight=None, /, *, out=None):
    """Gradients of `layer_norm`: (dx, dweight, dbias) for `grad`, the gradient of its result.

    mean, rstd: the statistics that layer_norm(x, ..., stats=True) returned.  dweight and dbias have the type of weight and
    are None without one, but for a dbias array given in `out` (of x's type, or float32 for float16 x): the gradient of a bias
    without a weight beside it.  out: (dx, dweight, dbias) arrays, each may be None; dx may be grad or x itself.
    """
    x = _data(x, "layer_norm_grad", "x")
    grad = _data(grad, "layer_norm_grad", "grad")
    _array(mean, "mean")
    _array(rstd, "rstd")
    weight = _vector(weight, "weight")
    ox, ow, ob = _several(out, 3, "(dx, dweight, dbias)")
    reads = (grad, x, mean, rstd, weight)
    if weight is None and ow is not None:
        raise ValueError("dweight would need weight")
    dx = _Out(ox, x._shape, x._dtype, "dx", reads, (grad, x))
    if weight is None:
        if ob is None:
            _ext.layer_norm_grad(grad, x, mean, rstd, None, dx.kernel, None, None)
            return dx.done(), None, None
        shape, dt = x._shape[-1:], x._dtype
        if dt == float16 and isinstance(ob, usm_ndarray) and ob._dtype == float32:
            dt = float32
        db = _Out(ob, shape, dt, "dbias", reads)
        _apart(dx, db)
        # (the kernels make both sums)
        _ext.layer_norm_grad(grad, x, mean, rstd, None, dx.kernel, usm_ndarray._new_contiguous(shape, dt), db.kernel)
        return dx.done(), None, db.done()
    dw = _Out(ow, weight._shape, weight._dtype, "dweight", reads)
    db = _Out(ob, weight._shape, weight._dtype, "dbias", reads)
    _apart(dx, dw, db)
    _ext.layer_norm_grad(grad, x, mean, rstd, weight, dx.kernel, dw.kernel, db.kernel)
    return dx.done(), dw.done(), db.done()


def distill_topk(logits, teacher_logits, teacher_tokens, /, *, temperature=1.0, out=None):
    """Distillation loss of each row: temperature**2 * KL(p || q), with p the softmax of the teacher's top logits over
    temperature and q the softmax of the row's logits over temperature.

    logits (..., V); teacher_logits (..., K) of logits' type or that of the loss; teacher_tokens (..., K) int32 or int64: which
    token each teacher logit belongs to, any number outside [0, V) marks an absent entry.  K is 2048 at most.  A row without
    entries has loss 0.  out: the array of the losses (...): float32, float64 for float64 logits.
    """
    logits = _data(logits, "distill_topk", "logits")
    lead = logits._shape[:-1]
    t, i = _over_rows(teacher_logits, lead, "teacher_logits"), _over_rows(teacher_tokens, lead, "teacher_tokens")
    loss = _Out(out, lead, _acc(logits._dtype), "loss", (logits, t, i))
    _ext.distill_topk(logits, t, i, None, float(temperature), loss.kernel, None)
    return loss.done()


def distill_topk_grad(logits, teacher_logits, teacher_tokens, weights=None, /, *, temperature=1.0, out=None):
    """(loss, dlogits): the losses of `distill_topk` and the gradient of sum(weights * loss) by the logits.

    weights (...): the loss's type, None for ones; a row of weight 0 (padding) gets a zero gradient whatever its logits are.  Its
    loss is that of `distill_topk`, NaN where its logits make it so: where(weights != 0, loss, 0) before it is added up.
    out: (loss, dlogits) arrays, each may be None; dlogits may be logits itself.
    """
    logits = _data(logits, "distill_topk_grad", "logits")
    lead = logits._shape[:-1]
    t, i = _over_rows(teacher_logits, lead, "teacher_logits"), _over_rows(teacher_tokens, lead, "teacher_tokens")
    w = _per_row(weights, lead, "weights")
    ol, od = _several(out, 2, "(loss, dlogits)")
    reads = (logits, t, i, w)
    loss = _Out(ol, lead, _acc(logits._dtype), "loss", reads)
    dz = _Out(od, logits._shape, logits._dtype, "dlogits", reads, (logits,))
    _apart(loss, dz)
    _ext.distill_topk(logits, t, i, w, float(temperature), loss.kernel, dz.kernel)
    return loss.done(), dz.done()


def _penalty(p, lead, name, none):
    if type(p) is usm_ndarray and p._shape == lead:
        return p
    if p is None:
        return none
    if isinstance(p, numbers.Real):
        return float(p)
    return _per_row(p, lead, name)


def process_logits(logits, /, *, prompt_tokens=None, prompt_lengths=None, output_tokens=None, output_lengths=None,
                   repetition_penalty=None, frequency_penalty=None, presence_penalty=None, bias_tokens=None,
                   bias_values=None, allowed=None, out=None):
    """Logits (..., V) with what is applied before a token is chosen, in this order:

    * a token among the row's prompt or output tokens is divided by `repetition_penalty` where its logit is positive and
      multiplied by it where not;
    * `frequency_penalty` times its number of occurrences in the output and, where there are any, `presence_penalty` are
      subtracted;
    * the row's biases for it are added;
    * a token whose bit in `allowed` is 0 becomes -inf.

    prompt_tokens, output_tokens (..., any) int32 or int64, of one type, of which the first prompt_lengths / output_lengths (...)
    int32 count (None: all); penalties: numbers or float32 arrays (...); bias_tokens (..., any) integers with bias_values
    float32; allowed (..., ceil(V / 32)) int32 or uint32, token v's bit being bit v % 32 of word v // 32.  Entries outside [0, V)
    are ignored; a side array without the rows' dims is used for every row.  out may be logits itself.
    """
    z = _data(logits, "process_logits", "logits")
    lead = z._shape[:-1]
    pt, ot = _over_rows(prompt_tokens, lead, "prompt_tokens"), _over_rows(output_tokens, lead, "output_tokens")
    pl = _per_row(prompt_lengths, lead, "prompt_lengths")
    ol = _per_row(output_lengths, lead, "output_lengths")
    rep = _penalty(repetition_penalty, lead, "repetition_penalty", 1.0)
    freq = _penalty(frequency_penalty, lead, "frequency_penalty", 0.0)
    pres = _penalty(presence_penalty, lead, "presence_penalty", 0.0)
    bt, bv = _over_rows(bias_tokens, lead, "bias_tokens"), _over_rows(bias_values, lead, "bias_values")
    ok = _over_rows(allowed, lead, "allowed")
    res = _Out(out, z._shape, z._dtype, "out", (z, pt, pl, ot, ol, rep, freq, pres, bt, bv, ok), (z,))
    _ext.process_logits(z, pt, pl, ot, ol, rep, freq, pres, bt, bv, ok, res.kernel)
    return res.done()

"""Operators over the last axis as language models use them, on dpnp arrays: layer_norm, layer_norm_grad, distill_topk,
distill_topk_grad, process_logits (no counterpart in the reference; see dpnp_amd/tensor/_row_operators.py for what each
computes)."""
import numbers

from . import tensor as dpt
from .dpnp_array import dpnp_array
from .dpnp_iface import _wrap, get_usm_ndarray

__all__ = ["distill_topk", "distill_topk_grad", "layer_norm", "layer_norm_grad", "process_logits"]


def _usm(a):
    return a._array_obj if type(a) is dpnp_array else None if a is None else get_usm_ndarray(a)


def _usm_or_number(a):
    return a if a is None or isinstance(a, numbers.Real) else _usm(a)


def _outs(out):
    return tuple(_usm(o) for o in out) if isinstance(out, tuple) else out


def _give(res, out):
    """The caller's array where there is one, else the result as a dpnp array."""
    return out if out is not None else None if res is None else _wrap(res)


def _give_all(res, out):
    return tuple(_give(r, o) for r, o in zip(res, out if out is not None else (None,) * len(res)))


def layer_norm(x, weight=None, bias=None, /, *, eps=1e-5, stats=False, out=None):
    if stats:
        return _give_all(dpt.layer_norm(_usm(x), _usm(weight), _usm(bias), eps=eps, stats=True, out=_outs(out)), out)
    return _give(dpt.layer_norm(_usm(x), _usm(weight), _usm(bias), eps=eps, out=_usm(out)), out)


def layer_norm_grad(grad, x, mean, rstd, weight=None, /, *, out=None):
    return _give_all(dpt.layer_norm_grad(_usm(grad), _usm(x), _usm(mean), _usm(rstd), _usm(weight), out=_outs(out)), out)


def distill_topk(logits, teacher_logits, teacher_tokens, /, *, temperature=1.0, out=None):
    return _give(dpt.distill_topk(_usm(logits), _usm(teacher_logits), _usm(teacher_tokens), temperature=temperature,
                                  out=_usm(out)), out)


def distill_topk_grad(logits, teacher_logits, teacher_tokens, weights=None, /, *, temperature=1.0, out=None):
    return _give_all(dpt.distill_topk_grad(_usm(logits), _usm(teacher_logits), _usm(teacher_tokens), _usm(weights),
                                           temperature=temperature, out=_outs(out)), out)


def process_logits(logits, /, *, prompt_tokens=None, prompt_lengths=None, output_tokens=None, output_lengths=None,
                   repetition_penalty=None, frequency_penalty=None, presence_penalty=None, bias_tokens=None,
                   bias_values=None, allowed=None, out=None):
    return _give(dpt.process_logits(
        _usm(logits), prompt_tokens=_usm(prompt_tokens), prompt_lengths=_usm(prompt_lengths),
        output_tokens=_usm(output_tokens), output_lengths=_usm(output_lengths),
        repetition_penalty=_usm_or_number(repetition_penalty), frequency_penalty=_usm_or_number(frequency_penalty),
        presence_penalty=_usm_or_number(presence_penalty), bias_tokens=_usm(bias_tokens), bias_values=_usm(bias_values),
        allowed=_usm(allowed), out=_usm(out)), out)


for _f in __all__:
    globals()[_f].__doc__ = getattr(dpt, _f).__doc__
del _f

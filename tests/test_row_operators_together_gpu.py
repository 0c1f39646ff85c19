"""The row operators together, as the output end of a language model has them: a hidden state is normalised, a small head (the
framework's multiply and sum) gives the logits, the distillation loss and its gradient go back through head and norm, and the
parameters take a step; then the same model answers with processed logits."""
import numpy as np
import pytest

import dpnp_amd as dpnp
from tests import row_operator_references as ref

pytestmark = pytest.mark.gpu


def head(h, w):
    return dpnp.sum(h[:, None, :] * w[None, :, :], axis=2)


def loss_of(p, x, t, tok, wt, temp):
    h = dpnp.layer_norm(x, p["gain"], p["shift"])
    return float(dpnp.sum(dpnp.distill_topk(head(h, p["head"]), t, tok, temperature=temp) * wt))


def gradients(p, x, t, tok, wt, temp):
    h, mean, rstd = dpnp.layer_norm(x, p["gain"], p["shift"], stats=True)
    z = head(h, p["head"])
    loss, dz = dpnp.distill_topk_grad(z, t, tok, wt, temperature=temp, out=(None, z))
    dhead = dpnp.sum(dz[:, :, None] * h[:, None, :], axis=0)
    dh = dpnp.sum(dz[:, :, None] * p["head"][None, :, :], axis=1)
    dx, dgain, dshift = dpnp.layer_norm_grad(dh, x, mean, rstd, p["gain"])
    return float(dpnp.sum(loss * wt)), dict(head=dhead, gain=dgain, shift=dshift, x=dx)


def model(rng, rows, width, vocab, k, dt):
    arr = lambda a: dpnp.array(a.astype(dt))  # noqa: E731
    p = dict(gain=arr(1 + 0.1 * rng.standard_normal(width)), shift=arr(0.1 * rng.standard_normal(width)),
             head=arr(rng.standard_normal((vocab, width)) / np.sqrt(width)))
    x = arr(rng.standard_normal((rows, width)))
    tok = np.stack([rng.permutation(vocab)[:k] for _ in range(rows)]).astype("i4")
    tok[-1] = -1  # a padded row
    wt = np.full(rows, 1.0 / (rows - 1))
    wt[-1] = 0
    return p, x, arr(3 * rng.standard_normal((rows, k))), dpnp.array(tok), arr(wt)


def test_training_step_gradients_are_slopes():
    rng = np.random.default_rng(0)
    p, x, t, tok, wt = model(rng, 5, 24, 37, 6, "f8")
    loss, g = gradients(p, x, t, tok, wt, 1.5)
    assert abs(loss - loss_of(p, x, t, tok, wt, 1.5)) < 1e-14 * 100
    h = 1e-5  # truncation ~ 1e-10, cancellation ~ 1e-16 / 1e-5: 1e-8 covers both for values of order one
    for name in ("head", "gain", "shift", "x"):
        arr = x if name == "x" else p[name]
        a = arr.asnumpy()
        for at in [tuple(rng.integers(0, s) for s in a.shape) for _ in range(5)]:
            vals = []
            for s in (h, -h):
                b = a.copy()
                b[at] += s
                q, xx = (p, dpnp.array(b)) if name == "x" else (dict(p, **{name: dpnp.array(b)}), x)
                vals.append(loss_of(q, xx, t, tok, wt, 1.5))
            assert abs((vals[0] - vals[1]) / (2 * h) - float(g[name][at])) < 1e-8, name
    assert not g["x"].asnumpy()[-1].any()


@pytest.mark.parametrize("dt", ["f4", "f2"])
def test_steps_run_and_the_model_answers(dt):
    rng = np.random.default_rng(1)
    p, x, t, tok, wt = model(rng, 9, 40, 101, 8, dt)
    if dt == "f2":
        t, wt = t.astype("f4"), wt.astype("f4")
    for _ in range(4):
        loss, g = gradients(p, x, t, tok, wt, 1.0)
        assert np.isfinite(loss)
        for name in p:
            assert g[name].dtype == p[name].dtype and np.isfinite(g[name].asnumpy()).all()
            p[name] -= g[name] * 0.5
    # answering, token after token: penalties over what was said, a mask that allows a third of the tokens
    said = np.full((9, 6), -1, "i4")
    allowed = np.zeros((9, 4), "u4")
    for v in range(0, 101, 3):
        allowed[:, v >> 5] |= np.uint32(1 << (v & 31))
    z = head(dpnp.layer_norm(x, p["gain"], p["shift"]), p["head"])
    for step in range(6):
        out = dpnp.process_logits(z, output_tokens=dpnp.array(said), output_lengths=dpnp.array(np.full(9, step, "i4")),
                                  repetition_penalty=1.3, frequency_penalty=0.2, presence_penalty=50.0, allowed=dpnp.array(allowed))
        want, tol, _ = ref.process_logits(z.asnumpy(), output=said, olen=np.full(9, step), rep=1.3, freq=0.2, pres=50.0, allowed=allowed)
        got = out.asnumpy()
        masked = want == -np.inf
        assert (got[masked] == -np.inf).all() and (np.abs(got[~masked].astype("f8") - want[~masked]) <= tol[~masked]).all()
        token = dpnp.argmax(out, axis=1).asnumpy()
        assert (token % 3 == 0).all()
        assert not any(token[r] in said[r, :step] for r in range(9))  # the presence penalty is larger than any difference
        said[:, step] = token

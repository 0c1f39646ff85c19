"""The row operators at the output end of a language model, as they are measured: layer normalisation with its gradient,
distillation from a teacher's top logits with its gradient, and the processing of logits before a token is chosen.

`run` computes a case in elementary torch operations, or, where `own` is true, through dpnp_amd's entry points on the same
memory."""
import math
import os

import torch

own = False

EPS = 1e-5
DTYPES = {"f2": torch.float16, "f4": torch.float32, "f8": torch.float64}
SIZE = {"f2": 2, "f4": 4, "f8": 8}


# ---- the cases -----------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of a few sequences: a handful of rows, all latency
        dict(name="norm decode 4x4096 f2", op="norm", rows=4, n=4096, dtype="f2", wdtype="f2", stats=False),
        # a training step's tokens in mixed precision: float16 activations, float32 parameters, statistics kept
        dict(name="norm train 16384x4096 f2", op="norm", rows=16384, n=4096, dtype="f2", wdtype="f4", stats=True),
        # odd width: rows off every boundary, float32
        dict(name="norm odd 20011x1001 f4", op="norm", rows=20011, n=1001, dtype="f4", wdtype="f4", stats=True),
        # its backward pass: mixed precision, and float32 of an odd width and a ragged number of tokens
        dict(name="norm_grad train 16384x4096 f2", op="norm_grad", rows=16384, n=4096, dtype="f2", wdtype="f4"),
        dict(name="norm_grad odd 2049x10007 f4", op="norm_grad", rows=2049, n=10007, dtype="f4", wdtype="f4"),
        # loss only, as an evaluation runs it: a few rows, and many over a large vocabulary
        dict(name="distill small 8x32768 f4", op="distill", rows=8, v=32768, k=16, dtype="f4", temperature=2.0),
        dict(name="distill eval 2048x131072 f2", op="distill", rows=2048, v=131072, k=64, dtype="f2", temperature=1.0),
        # loss and gradient of a training step: many rows; float32 with an odd vocabulary; few rows, long ones
        dict(name="distill_grad train 2048x65536 f2", op="distill_grad", rows=2048, v=65536, k=64, dtype="f2", temperature=1.0),
        dict(name="distill_grad odd 513x100003 f4", op="distill_grad", rows=513, v=100003, k=100, dtype="f4", temperature=2.0),
        dict(name="distill_grad few 16x131072 f4", op="distill_grad", rows=16, v=131072, k=32, dtype="f4", temperature=1.0),
        # answering: one sequence with its history; a full batch of an odd vocabulary with biases and grammar masks
        dict(name="logits decode 1x131072 f4", op="logits", rows=1, v=131072, prompt=700, output=300, biases=0, mask=False,
             dtype="f4"),
        dict(name="logits batch 256x100003 f2", op="logits", rows=256, v=100003, prompt=1800, output=700, biases=50, mask=True,
             dtype="f2"),
    ]


def draw(rng):
    def between(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(["norm", "norm_grad", "distill", "distill_grad", "logits"])
    dtype = rng.choice(["f2", "f2", "f4", "f4", "f8"])
    if op in ("norm", "norm_grad"):
        n = between(64, 16384)
        rows = between(1, max(1, (1 << 26) // (n * SIZE[dtype] // 2)))
        case = dict(op=op, rows=rows, n=n, dtype=dtype, wdtype=rng.choice([dtype, "f4"]) if dtype == "f2" else dtype)
        if op == "norm":
            case["stats"] = rng.random() < 0.5
        return case
    v = between(1000, 160000)
    if op == "logits":
        return dict(op=op, rows=between(1, 256), v=v, prompt=between(1, 4096), output=between(1, 4096),
                    biases=rng.choice([0, between(1, 300)]), mask=rng.random() < 0.5, dtype=dtype)
    rows = between(1, max(1, (1 << 27) // (v * SIZE[dtype] // 2)))
    return dict(op=op, rows=rows, v=v, k=between(1, 256), dtype=dtype, temperature=rng.choice([1.0, 2.0, 0.7]))


def work(case):
    r, s = case["rows"], SIZE[case["dtype"]]
    if case["op"] in ("norm", "norm_grad"):
        n, ws, acc = case["n"], SIZE[case["wdtype"]], 8 if case["dtype"] == "f8" else 4
        if case["op"] == "norm":
            return {"bytes": 2 * r * n * s + 2 * n * ws + (2 * r * acc if case["stats"] else 0), "flops": 8 * r * n}
        return {"bytes": 3 * r * n * s + 3 * n * ws + 2 * r * acc, "flops": 14 * r * n}
    v, acc = case["v"], 8 if case["dtype"] == "f8" else 4
    if case["op"] == "logits":
        side = r * 4 * (case["prompt"] + case["output"]) + r * (12 + 8) + r * 8 * case["biases"]
        return {"bytes": 2 * r * v * s + side + (r * 4 * ((v + 31) // 32) if case["mask"] else 0), "flops": 2 * r * v}
    side = r * case["k"] * (4 + acc) + r * acc
    if case["op"] == "distill":
        return {"bytes": r * v * s + side, "flops": 5 * r * v}
    return {"bytes": 2 * r * v * s + side + r * acc, "flops": 9 * r * v}


# ---- what a program has in hand before the call ------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    state = {"case": dict(case)}
    state.update(_norm_inputs(case, dt, g) if case["op"].startswith("norm") else
                 _logits_inputs(case, dt, g) if case["op"] == "logits" else _distill_inputs(case, dt, g))
    if own:  # the same memory as the framework's arrays, and the result arrays that a program's loop keeps
        state["arrays"] = _arrays(state)
    return state


def _rand(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _real(case):
    return torch.float64 if case["dtype"] == "f8" else torch.float32


def _norm_inputs(case, dt, g):
    r, n, real = case["rows"], case["n"], _real(case)
    wdt = DTYPES[case["wdtype"]]
    # activations: channels of their own scale and offset, a few of them large, as a trained network's are
    scale = torch.exp(0.5 * _rand(g, n, dtype=real))
    x = _rand(g, r, n, dtype=real).mul_(scale).add_(0.3 * _rand(g, n, dtype=real))
    x = x.to(dt)
    s = {"x": x, "weight": (1 + 0.2 * _rand(g, n)).to(wdt), "bias": (0.2 * _rand(g, n)).to(wdt)}
    if case["op"] == "norm_grad":
        s["dy"] = (_rand(g, r, n, dtype=real) * 0.1).to(dt)
        x = x.to(real)
        s["mean"] = x.mean(-1)
        s["rstd"] = 1 / torch.sqrt((x - s["mean"][:, None]).square_().mean(-1) + EPS)
    return s


def _distill_inputs(case, dt, g):
    r, v, k, real = case["rows"], case["v"], case["k"], _real(case)
    z = _rand(g, r, v, dtype=real).mul_(1.5)
    # the teacher's tokens: all different in a row, its logits falling; the student leans towards them
    step = 1 + torch.randint(0, max(1, v // k - 1), (r, 1), generator=g, device="cuda")
    first = torch.randint(0, v, (r, 1), generator=g, device="cuda")
    tokens = (first + step * torch.arange(k, device="cuda")) % v
    teacher = 8 - torch.cumsum(0.3 * torch.rand(r, k, generator=g, device="cuda", dtype=real), -1)
    z.scatter_(1, tokens, 0.8 * teacher + 0.5 * _rand(g, r, k, dtype=real))
    tokens = tokens.to(torch.int32)
    # ragged lists: some rows have fewer entries, one row in 16 (padding) none and no weight
    keep = torch.randint(1, k + 1, (r, 1), generator=g, device="cuda")
    keep = torch.where(torch.rand(r, 1, generator=g, device="cuda") < 0.75, torch.full_like(keep, k), keep)
    keep = torch.where(torch.arange(r, device="cuda")[:, None] % 16 == 15, torch.zeros_like(keep), keep)
    tokens = torch.where(torch.arange(k, device="cuda") < keep, tokens, torch.full_like(tokens, -1))
    s = {"logits": z.to(dt), "teacher": teacher, "tokens": tokens}
    if case["op"] == "distill_grad":
        s["weights"] = torch.where(keep[:, 0] > 0, 0.5 + torch.rand(r, generator=g, device="cuda"), 0.0).to(real)
    return s


def _logits_inputs(case, dt, g):
    r, v = case["rows"], case["v"]
    z = 2.5 * _rand(g, r, v, dtype=_real(case))
    s = {"logits": z.to(dt)}
    for name in ("prompt", "output"):
        n = case[name]
        # token numbers as text has them: low ones often, so that counts rise
        t = (v * torch.rand(r, n, generator=g, device="cuda") ** 4).to(torch.int32).clamp_(0, v - 1)
        s[name] = t
        s[name + "_lengths"] = torch.randint(n // 2, n + 1, (r,), generator=g, device="cuda").to(torch.int32)
    for name, lo, hi in (("repetition", 1.0, 1.4), ("frequency", 0.0, 0.8), ("presence", 0.0, 0.8)):
        s[name] = lo + (hi - lo) * torch.rand(r, generator=g, device="cuda")
    if case["biases"]:
        s["bias_tokens"] = torch.randint(-1, v, (r, case["biases"]), generator=g, device="cuda").to(torch.int32)
        s["bias_values"] = torch.randint(-40, 41, (r, case["biases"]), generator=g, device="cuda").to(torch.float32) / 4
    if case["mask"]:
        s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (r, (v + 31) // 32), generator=g, device="cuda").to(torch.int32)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    return {"norm": _norm, "norm_grad": _norm_grad, "distill": _distill, "distill_grad": _distill_grad, "logits": _logits}[op](state)


def _norm(s):
    real = _real(s["case"])
    x = s["x"].to(real)
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
    y = (d * rstd * s["weight"].to(real) + s["bias"].to(real)).to(s["x"].dtype)
    return (y, mean[:, 0], rstd[:, 0]) if s["case"]["stats"] else y


def _norm_grad(s):
    real = _real(s["case"])
    dy, rstd = s["dy"].to(real), s["rstd"][:, None]
    h = (s["x"].to(real) - s["mean"][:, None]) * rstd
    g = dy * s["weight"].to(real)
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return dx.to(s["x"].dtype), (dy * h).sum(0).to(s["weight"].dtype), dy.sum(0).to(s["weight"].dtype)


def _distill_parts(s):
    real, temp = _real(s["case"]), s["case"]["temperature"]
    z = s["logits"].to(real) / temp
    z = z - z.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    there = (s["tokens"] >= 0) & (s["tokens"] < z.shape[1])
    at = torch.where(there, s["tokens"], 0).long()
    t = torch.where(there, s["teacher"].to(real) / temp, -math.inf)
    top = t.amax(-1, keepdim=True)
    p = torch.exp(t - torch.where(top > -math.inf, top, 0.0))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    logq = torch.gather(z, 1, at) - torch.log(total)
    term = torch.where(p > 0, p * (torch.log(p) - logq), 0.0)
    return e / total, at, p, temp * temp * term.sum(-1)


def _distill(s):
    return _distill_parts(s)[3]


def _distill_grad(s):
    q, at, p, loss = _distill_parts(s)
    grad = (q * p.sum(-1, keepdim=True)).scatter_add_(1, at, -p)
    return loss, (grad * (s["case"]["temperature"] * s["weights"])[:, None]).to(s["logits"].dtype)


def _logits(s):
    real = _real(s["case"])
    z = s["logits"].to(real)
    r, v = z.shape
    column = lambda name: s[name].to(real)[:, None]  # noqa: E731

    def counts(name):
        t = s[name]
        inside = torch.arange(t.shape[1], device=t.device) < s[name + "_lengths"][:, None]
        at = torch.where(inside & (t >= 0) & (t < v), t, v).long()  # column v takes what does not count
        return torch.zeros(r, v + 1, dtype=torch.int32, device=t.device).scatter_add_(1, at, torch.ones_like(t))[:, :v]

    said = counts("output")
    seen = (counts("prompt") > 0) | (said > 0)
    z = torch.where(seen, torch.where(z > 0, z / column("repetition"), z * column("repetition")), z)
    z = z - column("frequency") * said - column("presence") * (said > 0)
    if "bias_tokens" in s:
        t = s["bias_tokens"]
        at = torch.where((t >= 0) & (t < v), t, v).long()
        z = z + torch.zeros(r, v + 1, dtype=real, device=t.device).scatter_add_(1, at, s["bias_values"].to(real))[:, :v]
    if "allowed" in s:
        n = torch.arange(v, device=z.device)
        z = torch.where((s["allowed"][:, n >> 5] >> (n & 31)) & 1 != 0, z, -math.inf)
    return z.to(s["logits"].dtype)


# ---- the framework's calls -----------------------------------------------------------------------------------------
def _framework():
    os.environ.setdefault("DPNP_AMD_MEMORY", "torch")  # its arrays on torch's memory and stream: shared without a copy
    import dpnp_amd

    return dpnp_amd


def _arrays(state):
    dpnp = _framework()
    case, names = state["case"], {torch.float16: "f2", torch.float32: "f4", torch.float64: "f8", torch.int32: "i4"}

    def array(t):
        return dpnp.ndarray(tuple(t.shape), dtype=names[t.dtype], buffer=t.reshape(-1).view(torch.uint8))

    a = {name: array(t) for name, t in state.items() if isinstance(t, torch.Tensor)}
    real, rows = _real(case), case["rows"]
    big = state["x" if "x" in state else "logits"]
    row = lambda: torch.empty(rows, dtype=real, device="cuda")  # noqa: E731
    if case["op"] == "norm":
        out = (torch.empty_like(big), row(), row()) if case["stats"] else (torch.empty_like(big),)
    elif case["op"] == "norm_grad":
        out = (torch.empty_like(big), torch.empty_like(state["weight"]), torch.empty_like(state["weight"]))
    else:
        out = {"distill": lambda: (row(),), "distill_grad": lambda: (row(), torch.empty_like(big)),
               "logits": lambda: (torch.empty_like(big),)}[case["op"]]()
    a["out"] = tuple(array(t) for t in out)
    a["result"] = out if len(out) > 1 else out[0]
    return a


def _own(state, op):
    dpnp = _framework()
    a, case = state["arrays"], state["case"]
    if op == "norm":
        dpnp.layer_norm(a["x"], a["weight"], a["bias"], eps=EPS, stats=case["stats"], out=a["out"] if case["stats"] else a["out"][0])
    elif op == "norm_grad":
        dpnp.layer_norm_grad(a["dy"], a["x"], a["mean"], a["rstd"], a["weight"], out=a["out"])
    elif op == "distill":
        dpnp.distill_topk(a["logits"], a["teacher"], a["tokens"], temperature=case["temperature"], out=a["out"][0])
    elif op == "distill_grad":
        dpnp.distill_topk_grad(a["logits"], a["teacher"], a["tokens"], a["weights"], temperature=case["temperature"], out=a["out"])
    else:
        dpnp.process_logits(a["logits"], prompt_tokens=a["prompt"], prompt_lengths=a["prompt_lengths"],
                            output_tokens=a["output"], output_lengths=a["output_lengths"], repetition_penalty=a["repetition"],
                            frequency_penalty=a["frequency"], presence_penalty=a["presence"],
                            bias_tokens=a.get("bias_tokens"), bias_values=a.get("bias_values"), allowed=a.get("allowed"),
                            out=a["out"][0])
    return a["result"]


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    rows, width = case["rows"], case.get("n", case.get("v"))
    few = max(1, (1 << 25) // width)
    parts = [{"norm": _exact_norm, "norm_grad": _exact_norm_grad, "distill": _exact_distill, "distill_grad": _exact_distill,
              "logits": _exact_logits}[case["op"]](case, s, slice(i, min(rows, i + few))) for i in range(0, rows, few)]
    if case["op"] == "norm_grad":
        return tuple([torch.cat([p[0] for p in parts]), sum(p[1] for p in parts), sum(p[2] for p in parts)])
    whole = tuple(torch.cat(p) for p in zip(*parts))
    return whole if len(whole) > 1 else whole[0]


def _exact_norm(case, s, at):
    x = s["x"][at].double()
    n = x.shape[1]
    mean = x.sum(1) / n
    x = x.sub_(mean[:, None])
    rstd = (torch.linalg.vecdot(x, x) / n + EPS).pow(-0.5)
    y = torch.addcmul(s["bias"].double(), x.mul_(rstd[:, None]), s["weight"].double())
    return (y, mean, rstd) if case["stats"] else (y,)


def _exact_norm_grad(case, s, at):
    dy, x = s["dy"][at].double(), s["x"][at].double()
    n, rstd = x.shape[1], s["rstd"][at].double()[:, None]
    h = x.sub_(s["mean"][at].double()[:, None]).mul_(rstd)
    # dx is dy's product with the Jacobian: the parts along 1 and along h are taken out of dy w
    g = dy * s["weight"].double()
    along_h = torch.linalg.vecdot(g, h)[:, None] / n
    along_1 = g.sum(1, keepdim=True) / n
    dx = (g - along_1 - along_h * h) * rstd
    return dx, torch.linalg.vecdot(dy, h, dim=0), dy.sum(0)


def _exact_distill(case, s, at):
    temp = case["temperature"]
    z = s["logits"][at].double().div_(temp)
    v = z.shape[1]
    tokens, t = s["tokens"][at].long(), s["teacher"][at].double() / temp
    there = (tokens >= 0) & (tokens < v)
    t = t.masked_fill(~there, -math.inf)
    some = there.any(1, keepdim=True)
    logp = torch.where(some, t - torch.logsumexp(t, 1, keepdim=True), -math.inf)
    p = torch.exp(logp)
    z = z.sub_(torch.logsumexp(z, 1, keepdim=True))  # the logarithm of the student's distribution
    own_k = z.gather(1, tokens.clamp(0, v - 1))
    loss = temp ** 2 * (torch.special.xlogy(p, p) - torch.where(p > 0, p * own_k, 0.0)).sum(1)
    if case["op"] == "distill":
        return (loss,)
    grad = z.exp_().mul_(some.double())
    grad.scatter_add_(1, tokens.clamp(0, v - 1), -p)
    return loss, grad.mul_((temp * s["weights"][at].double())[:, None])


def _exact_logits(case, s, at):
    z = s["logits"][at].double()
    r, v = z.shape
    rows = torch.arange(r, device=z.device)[:, None]

    def entries(name):  # flat positions of the tokens that count
        t, n = s[name][at].long(), s[name + "_lengths"][at].long()
        ok = (torch.arange(t.shape[1], device=z.device) < n[:, None]) & (t >= 0) & (t < v)
        return (rows * v + t)[ok]

    said = torch.bincount(entries("output"), minlength=r * v).reshape(r, v)
    touched = torch.zeros(r * v, dtype=torch.bool, device=z.device)
    touched[entries("prompt")] = True
    touched[entries("output")] = True
    touched = touched.reshape(r, v)
    rep = s["repetition"][at].double()[:, None]
    factor = torch.where(z > 0, 1 / rep, rep)
    z = torch.where(touched, z * factor, z)
    z = z - said * s["frequency"][at].double()[:, None] - said.clamp(max=1) * s["presence"][at].double()[:, None]
    if case["biases"]:
        t = s["bias_tokens"][at].long()
        ok = (t >= 0) & (t < v)
        z = z.reshape(-1).index_add_(0, (rows * v + t)[ok], s["bias_values"][at].double()[ok]).reshape(r, v)
    if case["mask"]:
        bits = (s["allowed"][at][:, :, None] >> torch.arange(32, device=z.device)) & 1
        z = z.masked_fill(bits.reshape(r, -1)[:, :v] == 0, -math.inf)
    return (z,)

"""Run by test_row_operators_torch_gpu.py in a process of its own with DPNP_AMD_MEMORY=torch: the row operators on torch's
memory, under its side streams and captured into its graphs.  Prints OK at the end."""
import os
import sys

os.environ["DPNP_AMD_MEMORY"] = "torch"
sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np  # noqa: E402

import dpnp_amd as dpnp  # noqa: E402
import dpnp_amd._lib as L  # noqa: E402

torch = L.torch
DT = {torch.float16: "f2", torch.float32: "f4", torch.int32: "i4"}


def seen(t):
    return dpnp.ndarray(tuple(t.shape), dtype=DT[t.dtype], buffer=t.reshape(-1).view(torch.uint8))


def inputs(seed, r, n, v, k, dt=torch.float32):
    g = torch.Generator("cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    d = dict(x=rnd(r, n).to(dt), dy=rnd(r, n).to(dt), w=1 + 0.1 * rnd(n), b=rnd(n), z=(2 * rnd(r, v)).to(dt), t=4 * rnd(r, k),
             tok=torch.randint(0, v, (r, k), generator=g, device="cuda").to(torch.int32), wt=rnd(r))
    return d


def run(a, out):
    """Every operator once, in the order a step has them; `out`: the result arrays."""
    dpnp.layer_norm(a["x"], a["w"], a["b"], stats=True, out=(out["y"], out["mean"], out["rstd"]))
    dpnp.layer_norm_grad(a["dy"], a["x"], out["mean"], out["rstd"], a["w"], out=(out["dx"], out["dw"], out["db"]))
    dpnp.distill_topk(a["z"], a["t"], a["tok"], out=out["loss"])
    dpnp.distill_topk_grad(a["z"], a["t"], a["tok"], a["wt"], temperature=2.0, out=(out["loss2"], out["dz"]))
    dpnp.process_logits(a["z"], prompt_tokens=a["tok"], output_tokens=a["tok"], repetition_penalty=1.2, frequency_penalty=0.5,
                        out=out["p"])


def outputs(d):
    r, dt = d["x"].shape[0], d["x"].dtype
    like = lambda t: torch.full_like(t, 7)  # noqa: E731
    row = lambda: torch.full((r,), 7.0, device="cuda")  # noqa: E731
    return dict(y=like(d["x"]), mean=row(), rstd=row(), dx=like(d["x"]), dw=like(d["w"]), db=like(d["w"]), loss=row(), loss2=row(),
                dz=like(d["z"]), p=like(d["z"]))


def arrays(d):
    return {k: seen(t) for k, t in d.items()}


def eager(d):
    o = outputs(d)
    run(arrays(d), arrays(o))
    torch.cuda.synchronize()
    return {k: t.clone() for k, t in o.items()}


def same(o, want, what):
    for k in want:
        assert torch.equal(o[k], want[k]), (what, k)


SHAPES = [(3, 1000, 70001, 20), (400, 5000, 3000, 33), (1200, 96, 520, 7)]

for dt in (torch.float32, torch.float16):
    for shape in SHAPES:
        d = inputs(1, *shape, dt=dt)
        want = eager(d)
        # a side stream, the inputs made on it just before
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            e = {k: t.clone() for k, t in d.items()}
            o = outputs(e)
            run(arrays(e), arrays(o))
            copy = {k: t.clone() for k, t in o.items()}
        side.synchronize()
        same(copy, want, "side stream")
        # two streams at once, each call with its own workspace
        e2 = inputs(2, *shape, dt=dt)
        want2 = eager(e2)
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        o1, o2 = outputs(d), outputs(e2)
        a1, b1, a2, b2 = arrays(d), arrays(o1), arrays(e2), arrays(o2)
        torch.cuda.synchronize()
        for _ in range(5):
            with torch.cuda.stream(s1):
                run(a1, b1)
            with torch.cuda.stream(s2):
                run(a2, b2)
        torch.cuda.synchronize()
        same(o1, want, "first of two streams")
        same(o2, want2, "second of two streams")
        print("streams", dt, shape, flush=True)

# captured graphs: several replays with eager work between, new contents in the same inputs, two graphs replayed at once
for dt, shape in ((torch.float32, SHAPES[0]), (torch.float16, SHAPES[1]), (torch.float32, SHAPES[2])):
    sets = [inputs(s, *shape, dt=dt) for s in (3, 4)]
    outs = [outputs(d) for d in sets]
    A, B = [arrays(d) for d in sets], [arrays(o) for o in outs]
    run(A[0], B[0])  # everything loaded before a capture
    torch.cuda.synchronize()
    graphs = []
    for a, b in zip(A, B):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(a, b)
        graphs.append(g)
    for k in range(5):
        new = [inputs(10 + 2 * k + i, *shape, dt=dt) for i in range(2)]
        want = [eager(d) for d in new]
        for d, n in zip(sets, new):
            for name in d:
                d[name].copy_(n[name])
        for o in outs:
            for t in o.values():
                t.fill_(9)
        torch.cuda.synchronize()
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
        eager(new[0])
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            same(o, w, "replay %d" % k)
    print("graphs", dt, shape, flush=True)
print("OK")

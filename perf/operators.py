"""What the training-step operators are measured on: embedding, residual norm, gradient clipping.

``listed()`` and ``draw()`` give cases, ``prepare()`` a case's inputs on the GPU, ``run()`` one pass: in
plain torch operations where ``own`` is false, through ``opus_b200.ops`` where it is true.  ``exact()`` is
the definition in 64 bits.

Kinds of case (``op``):

- ``embed``: Y = scale * W[tokens] (``embed_fwd``), with its gradient dW (``embed_train``), or the gradient
  alone (``embed_grad``), for token ids drawn Zipf(1.1) as text has them;
- ``norm``: h = r * x + gate o z with z = y or a norm of y, n = norm(h) (``norm_fwd``), with every gradient
  (``norm_train``);
- ``clip``: the global norm of a list of gradients (``clip_norm``), clipping it in place when the norm is
  below the bound (``clip_below``), or into another buffer when it is above (``clip_above``).
"""
import math

import torch

own = False

DEV = "cuda"
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    """The widths, vocabularies and sequence lengths are the selection benchmark's model configurations."""
    return [
        # one token of one sequence looked up and scaled, as a step-by-step evaluation of a sample does: latency
        {"name": "embed_one_token", "op": "embed", "form": "fwd", "tokens": 1, "vocab": 50304, "d": 1600,
         "type": "bf16", "scale": 40.0, "padded": 0.0},
        # every candidate and proxy row of a whole selection round looked up at once: 144 x 1024 tokens
        {"name": "embed_round_1600", "op": "embed", "form": "fwd", "tokens": 147456, "vocab": 50304, "d": 1600,
         "type": "bf16", "scale": 1.0, "padded": 0.0},
        # a float32 model's training pass over a round's 80 rows, vocabulary not rounded up
        {"name": "embed_train_768_f32", "op": "embed", "form": "train", "tokens": 81920, "vocab": 50257, "d": 768,
         "type": "f32", "scale": 1.0, "padded": 0.0},
        # backward of a large vocabulary over 4 sequences of 4096, a fifth of it padding
        {"name": "embed_grad_151936", "op": "embed", "form": "grad", "tokens": 16384, "vocab": 151936, "d": 2048,
         "type": "bf16", "scale": 1.0, "padded": 0.2},
        # one token through a pre-norm block's joint: latency
        {"name": "norm_one_token", "op": "norm", "form": "fwd", "batch": 1, "seq": 1, "d": 2048, "type": "bf16",
         "kind": "rms", "post": False, "gate": "none", "residual": 1.0},
        # forward joints of a capture pass at 32 x 4096 tokens, norms on both sides of the block and a gate
        {"name": "norm_sandwich_2048", "op": "norm", "form": "fwd", "batch": 32, "seq": 4096, "d": 2048,
         "type": "bf16", "kind": "rms", "post": True, "gate": "channel", "residual": 1.0},
        # a training pass of a pre-LayerNorm model, 24 rows of 1024
        {"name": "norm_train_layer_1600", "op": "norm", "form": "train", "batch": 24, "seq": 1024, "d": 1600,
         "type": "bf16", "kind": "layer", "post": False, "gate": "none", "residual": 1.0},
        # the same in float32 with an odd width, odd lengths, a gate of its own for each sequence, scaled residual
        {"name": "norm_train_odd_f32", "op": "norm", "form": "train", "batch": 7, "seq": 511, "d": 771,
         "type": "f32", "kind": "rms", "post": True, "gate": "sample", "residual": 0.5},
        # adapters' gradients, 48 small matrices: latency
        {"name": "clip_adapters", "op": "clip", "form": "above", "tensors": 48, "total": 147456, "type": "f32",
         "out": "f32"},
        # the usual step of a 355M model: the norm is read and stays below the bound
        {"name": "clip_below_355m", "op": "clip", "form": "below", "tensors": 292, "total": 354823168, "type": "f32",
         "out": "f32"},
        # a 124M model's bf16 gradients clipped into the optimizer's float32 ones
        {"name": "clip_above_124m", "op": "clip", "form": "above", "tensors": 148, "total": 124439808, "type": "bf16",
         "out": "f32"},
        # a 1.56G model's bf16 gradients, clipped: the largest
        {"name": "clip_above_1558m", "op": "clip", "form": "above", "tensors": 580, "total": 1557611200,
         "type": "bf16", "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed kinds, sizes spread over their logarithm, odd ones among them."""
    op = rng.choice(["embed", "norm", "clip"])
    t = rng.choice(["bf16", "bf16", "f32", "f16"])
    if op == "embed":
        d = _log(rng, 64, 2048)
        d = d if rng.random() < 0.4 else max(64, d // 8 * 8)
        tokens, vocab = _log(rng, 1, 150000), _log(rng, 1000, 152000)
        return {"op": op, "form": rng.choice(["fwd", "train", "grad"]), "tokens": tokens, "vocab": vocab, "d": d,
                "type": t, "scale": rng.choice([1.0, round(math.sqrt(d), 3)]), "padded": rng.choice([0.0, 0.3])}
    if op == "norm":
        d = _log(rng, 64, 8192)
        d = d if rng.random() < 0.4 else max(64, d // 8 * 8)
        rows = _log(rng, 1, min(150000, 250_000_000 // d))
        batch = rng.randint(1, min(rows, 32))
        return {"op": op, "form": rng.choice(["fwd", "train"]), "batch": batch, "seq": max(1, rows // batch), "d": d,
                "type": t, "kind": rng.choice(["rms", "layer"]), "post": rng.random() < 0.5,
                "gate": rng.choice(["none", "channel", "sample"]), "residual": rng.choice([1.0, 0.5])}
    total = _log(rng, 1000, 400_000_000)
    return {"op": op, "form": rng.choice(["norm", "below", "above"]), "tensors": _log(rng, 1, min(600, total)),
            "total": total, "type": t, "out": rng.choice([t, "f32"])}


# ------------------------------------------------------------------------------------------------ inputs
def _embed_inputs(case, g):
    """Zipf(1.1) token ids (rank = id), a tail of padding (the last id), N(0, 0.02) rows."""
    n, v, d, t = case["tokens"], case["vocab"], case["d"], _TYPES[case["type"]]
    p = torch.arange(1, v + 1, dtype=torch.float64, device=DEV).pow(-1.1)
    u = torch.rand(n, dtype=torch.float64, device=DEV, generator=g)
    tokens = torch.searchsorted(torch.cumsum(p / p.sum(), 0), u).clamp_(max=v - 1)
    if case["padded"]:
        tokens[int(n * (1.0 - case["padded"])):] = v - 1
    s = {"tokens": tokens, "scale": case["scale"], "vocab": v, "padding": v - 1 if case["padded"] else None}
    if case["form"] != "grad":
        s["weight"] = (torch.randn(v, d, device=DEV, generator=g) * 0.02).to(t)
    if case["form"] != "fwd":
        s["dy"] = (torch.randn(n, d, device=DEV, generator=g) * 1e-2).to(t)
    return s


def _norm_inputs(case, g):
    b, n, d, t = case["batch"], case["seq"], case["d"], _TYPES[case["type"]]

    def rand(*shape, scale=1.0, mean=0.0):
        return (torch.randn(*shape, device=DEV, generator=g) * scale + mean).to(t)

    layer = case["kind"] == "layer"
    s = {"x": rand(b, n, d, scale=2.0), "y": rand(b, n, d), "weight": rand(d, scale=0.1, mean=1.0),
         "bias": rand(d, scale=0.1) if layer else None,
         "post_weight": rand(d, scale=0.1, mean=1.0) if case["post"] else None,
         "post_bias": rand(d, scale=0.1) if case["post"] and layer else None,
         "gate": {"none": None, "channel": (d,), "sample": (b, 1, d)}[case["gate"]],
         "kind": case["kind"], "eps": 1e-5, "residual": case["residual"]}
    if s["gate"] is not None:
        s["gate"] = rand(*s["gate"], scale=0.2, mean=0.5)
    if case["form"] == "train":
        s["dn"], s["dh"] = rand(b, n, d, scale=1e-2), rand(b, n, d, scale=1e-2)
    return s


def _clip_sizes(case):
    """Sizes of the list's tensors: half of them vectors or small, the others share the rest in unequal matrices."""
    k, total = case["tensors"], case["total"]
    share = [1.0 / (1.0 + (i * 7) % 11) if i % 2 == 0 else 1e-3 / (1.0 + i % 5) for i in range(k)]
    whole = sum(share)
    sizes = [max(1, int(total * x / whole)) for x in share]
    sizes[0] = max(1, sizes[0] + total - sum(sizes))
    return sizes


def _clip_inputs(case, g):
    """Gradients as views of one buffer, each at a multiple of 128 elements, zeros between them."""
    sizes = _clip_sizes(case)
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += (n + 127) // 128 * 128
    t = _TYPES[case["type"]]
    flat = torch.randn(at, device=DEV, generator=g, dtype=t).mul_(1e-3)
    for b, n, e in zip(starts, sizes, starts[1:] + [at]):
        flat[b + n:e] = 0
    rms = math.sqrt(sum(sizes)) * 1e-3
    s = {"flat": flat, "grads": [flat[b:b + n] for b, n in zip(starts, sizes)], "form": case["form"],
         "max_norm": 4.0 * rms if case["form"] == "below" else 0.25 * rms}
    if case["form"] == "above":
        s["to"] = torch.zeros(at, device=DEV, dtype=_TYPES[case["out"]])
        s["out"] = [s["to"][b:b + n] for b, n in zip(starts, sizes)]
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"embed": _embed_inputs, "norm": _norm_inputs, "clip": _clip_inputs}[case["op"]](case, g)
    s["op"], s["form"] = case["op"], case["form"]
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_embed(s):
    r = {}
    if s["form"] != "grad":
        r["y"] = (s["weight"][s["tokens"]].float() * s["scale"]).to(s["weight"].dtype)
    if s["form"] != "fwd":
        dw = torch.zeros(s["vocab"], s["dy"].shape[1], dtype=torch.float32, device=DEV)
        dw.index_add_(0, s["tokens"], s["dy"].float())
        if s["padding"] is not None:
            dw[s["padding"]] = 0
        r["dw"] = dw.mul_(s["scale"]).to(s["dy"].dtype)
    return r


def _normed(v, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    rstd = torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)
    return v * rstd, rstd


def _norm_back(a, hat, rstd, kind):
    back = a - hat * (a * hat).mean(-1, keepdim=True)
    if kind == "layer":
        back = back - a.mean(-1, keepdim=True)
    return back * rstd


def _plain_norm(s):
    kind, eps, t = s["kind"], s["eps"], s["x"].dtype

    def f(name):
        return None if s[name] is None else s[name].float()

    w, b, pw, pb, gate = (f(k) for k in ("weight", "bias", "post_weight", "post_bias", "gate"))
    x, y = f("x"), f("y")
    z = y
    if pw is not None:
        yhat, yr = _normed(y, kind, eps)
        z = yhat * pw if pb is None else yhat * pw + pb
    h = (s["residual"] * x + (z if gate is None else gate * z)).to(t)  # the residual stream as it is stored
    hat, rstd = _normed(h.float(), kind, eps)
    n = (hat * w if b is None else hat * w + b).to(t)
    r = {"n": n, "h": h}
    if s["form"] == "train":
        dn = f("dn")
        dh = f("dh") + _norm_back(dn * w, hat, rstd, kind)
        dz = dh if gate is None else gate * dh
        r["d_x"] = (s["residual"] * dh).to(t)
        r["d_weight"] = (dn * hat).sum((0, 1)).to(t)
        if b is not None:
            r["d_bias"] = dn.sum((0, 1)).to(t)
        if gate is not None:
            r["d_gate"] = ((dh * z).sum((0, 1)) if gate.dim() == 1 else (dh * z).sum(1, keepdim=True)).to(t)
        if pw is None:
            r["d_y"] = dz.to(t)
        else:
            r["d_post_weight"] = (dz * yhat).sum((0, 1)).to(t)
            if pb is not None:
                r["d_post_bias"] = dz.sum((0, 1)).to(t)
            r["d_y"] = _norm_back(dz * pw, yhat, yr, kind).to(t)
    return r


def _plain_clip(s):
    flat = s["flat"]
    norm = flat.float().square().sum(dtype=torch.float64).sqrt().float()
    if s["form"] == "norm":
        return {"norm": norm}
    c = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    if s["form"] == "below":
        flat.copy_(flat.float() * c)
        return {"norm": norm, "grads": flat}
    s["to"].copy_(flat.float() * c)
    return {"norm": norm, "grads": s["to"]}


# ------------------------------------------------------------------------------------------------ one pass
def _own_embed(s):
    from opus_b200 import ops

    r = {}
    if s["form"] != "grad":
        r["y"] = ops.embedding(s["tokens"], s["weight"], scale=s["scale"])
    if s["form"] != "fwd":
        r["dw"] = ops.embedding_grad(s["dy"], s["tokens"], s["vocab"], scale=s["scale"], padding_idx=s["padding"])
    return r


def _own_norm(s):
    from opus_b200 import ops

    kw = {"weight": s["weight"], "bias": s["bias"], "post_weight": s["post_weight"], "post_bias": s["post_bias"],
          "gate": s["gate"], "residual_scale": s["residual"], "kind": s["kind"], "eps": s["eps"]}
    n, h, stats = ops.residual_norm(s["x"], s["y"], **kw)
    r = {"n": n, "h": h}
    if s["form"] == "train":
        del kw["eps"]
        grads = ops.residual_norm_grad(s["dn"], s["dh"], h, stats, s["y"], **kw)
        r |= {"d_" + name: v for name, v in grads.items()}
    return r


def _own_clip(s):
    from opus_b200 import ops

    if s["form"] == "norm":
        return {"norm": ops.grad_norm(s["grads"])}
    if s["form"] == "below":
        return {"norm": ops.clip_grads(s["grads"], s["max_norm"]), "grads": s["flat"]}
    return {"norm": ops.clip_grads(s["grads"], s["max_norm"], out=s["out"]), "grads": s["to"]}


def run(state):
    if own:
        return {"embed": _own_embed, "norm": _own_norm, "clip": _own_clip}[state["op"]](state)
    return {"embed": _plain_embed, "norm": _plain_norm, "clip": _plain_clip}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    """Bytes: each input read once and each output written once.  Flops: one per multiply or add of the formulas."""
    e = _SIZE[case["type"]]
    if case["op"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["d"]
        used = _distinct(n, v)
        real = n * (1.0 - case["padded"])
        b = f = 0.0
        if case["form"] != "grad":
            b, f = b + 8 * n + used * d * e + n * d * e, f + n * d
        if case["form"] != "fwd":
            b, f = b + 8 * n + real * d * e + v * d * e, f + 2 * real * d
        return {"bytes": b, "flops": f}
    if case["op"] == "norm":
        n, d = case["batch"] * case["seq"], case["d"]
        gates = {"none": 0, "channel": d, "sample": case["batch"] * d}[case["gate"]]
        par = (2 * d if case["kind"] == "layer" else d) * (2 if case["post"] else 1) + gates
        fwd, bwd = 4 * n * d + par, 6 * n * d + 2 * par
        train = case["form"] == "train"
        return {"bytes": float((fwd + bwd if train else fwd) * e),
                "flops": float(n * d * ((8 if not case["post"] else 13) + (0 if not train else 14 if not case["post"] else 26)))}
    n = case["total"]
    eo = {"norm": 0, "below": 0, "above": _SIZE[case["out"]]}[case["form"]]
    return {"bytes": float(n * (e + eo)), "flops": float(n * (2 if case["form"] != "above" else 3))}


def _distinct(n, v):
    """Expected number of distinct ids among n draws of the Zipf(1.1) law over v ids."""
    whole = sum(r ** -1.1 for r in range(1, v + 1))
    return sum(-math.expm1(n * math.log1p(-min(0.999999, r ** -1.1 / whole))) for r in range(1, v + 1))


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The outputs of run() by the operators' definitions in float64, sums over samples and rows one after another."""
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "embed":
        r, ids = {}, s["tokens"]
        if "weight" in s:
            r["y"] = torch.index_select(s["weight"], 0, ids).to(f).mul_(s["scale"])
        if "dy" in s:
            dy = s["dy"].to(f)
            if s["padding"] is not None:
                dy.mul_((ids != s["padding"]).to(f)[:, None])
            # rows in the order of their ids: the sum of a run is the difference of two running sums at its ends
            order = torch.argsort(ids, stable=True)
            ends = torch.searchsorted(ids[order], torch.arange(s["vocab"] + 1, device=DEV))
            if dy.shape[0] * dy.shape[1] > 200_000_000:
                dw = torch.zeros(s["vocab"], dy.shape[1], dtype=f, device=DEV).index_add_(0, ids, dy)
            else:
                run_sum = torch.zeros(dy.shape[0] + 1, dy.shape[1], dtype=f, device=DEV)
                torch.cumsum(dy[order], 0, out=run_sum[1:])
                dw = run_sum[ends[1:]] - run_sum[ends[:-1]]
                dw[ends[1:] == ends[:-1]] = 0.0
            r["dw"] = dw.mul_(s["scale"])
        return r
    if case["op"] == "norm":
        if s["x"].numel() > 300_000_000:
            return None
        return _exact_norm(s, f)
    n2 = torch.zeros((), dtype=f, device=DEV)
    for g in s["grads"]:
        n2 += torch.dot(g.to(f), g.to(f))
    norm = torch.sqrt(n2)
    if case["form"] == "norm":
        return {"norm": norm}
    c = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    return {"norm": norm, "grads": s["flat"].to(f).mul_(c)}


def _exact_norm(s, f):
    """Forward by its definition with autograd for the gradients, sample by sample to bound the memory."""
    names = [k for k in ("weight", "bias", "post_weight", "post_bias") if s[k] is not None]
    par = {k: s[k].to(f).requires_grad_() for k in names}
    layer, eps = s["kind"] == "layer", s["eps"]

    def norm(v, w, b):
        c = v - v.mean(-1, keepdim=True) if layer else v
        c = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
        return c * par[w] + par[b] if b in par else c * par[w]

    r = {k: [] for k in ("n", "h", "d_x", "d_y", "d_gate")}
    for i in range(s["x"].shape[0]):
        x, y = s["x"][i].to(f).requires_grad_(), s["y"][i].to(f).requires_grad_()
        gate = None
        if s["gate"] is not None:
            gate = (s["gate"] if s["gate"].dim() == 1 else s["gate"][i]).to(f).requires_grad_()
        z = norm(y, "post_weight", "post_bias") if "post_weight" in par else y
        h = s["residual"] * x + (z if gate is None else gate * z)
        # the norm is of the stored residual stream; its rounding passes gradients through
        n = norm(h + (h.detach().to(s["x"].dtype).to(f) - h.detach()), "weight", "bias")
        r["n"].append(n.detach())
        r["h"].append(h.detach())
        if s["form"] == "train":
            torch.autograd.backward([n, h], [s["dn"][i].to(f), s["dh"][i].to(f)])
            r["d_x"].append(x.grad)
            r["d_y"].append(y.grad)
            if gate is not None:
                r["d_gate"].append(gate.grad)
    got = {k: torch.stack(v) for k, v in r.items() if v}
    if s["form"] == "train":
        got |= {"d_" + k: p.grad for k, p in par.items()}
        if s["gate"] is not None and s["gate"].dim() == 1:
            got["d_gate"] = got["d_gate"].sum(0)
    return got

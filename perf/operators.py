"""What the block norms and the gradient clipping are measured on: cases, inputs, plain forms, exact values.

`run` computes one pass either in plain torch operations (`own` false) or through the package's entry points (`own` true):
`block_norm` / `residual_block_norm` (the norms before and after a model's block, fused with gate, residual and scales) and
`clip_by_global_norm_` (one norm over all gradients, and their scaling by it).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
DEV = "cuda"


# ------------------------------------------------------------------------------------------------------ cases
def _norms(name, mode, train, dtype, rows, width, kind, post, gate, **kw):
    """mode: "pre" = norm(x); "post" = residual + gate * norm(branch); "pair" = that and the next block's norm of it.
    post: whether the branch itself is normalised (models with sandwich norms) or only added."""
    case = {"name": name, "op": "norms", "mode": mode, "train": train, "dtype": dtype, "rows": rows, "width": width,
            "kind": kind, "post": post, "gate": gate, "residual_scale": 1.0, "branch_scale": 1.0}
    case.update(kw)
    return case


def _clip(name, dtype, act, dict_size, layers, max_norm, p):
    """p: "1", "2" or "inf", the norm's order.  Gradients of a transcoder (act x dict_size; none if dict_size is 0) and of the norms of `layers` blocks."""
    return {"name": name, "op": "clip", "dtype": dtype, "act": act, "dict_size": dict_size,
            "layers": layers, "max_norm": max_norm, "p": p}


def listed():
    return [
        # one token of a generation, in a Gemma-2-2B block: attention's post-norm, residual, and the MLP's pre-norm
        _norms("token", "pair", False, "bf16", 1, 2304, "rms", True, "none"),
        # a batch of prompts (32 x 128 tokens) at the same place
        _norms("prompt", "pair", False, "bf16", 4096, 2304, "rms", True, "none"),
        # harvesting: the transcoder's source (pre-norm of the residual) for one model batch of 512 x 128 tokens
        _norms("harvest", "pre", False, "bf16", 65536, 2304, "rms", False, "none"),
        # GPT-2 XL: residual add and layer norm in fp32, an odd number of tokens
        _norms("add_norm_fp32", "pair", False, "fp32", 1023, 1600, "layer", False, "none"),
        # training a spliced Gemma-2-2B block; the gate keeps some tokens (padding) out of the splice
        _norms("train_2b", "pair", True, "bf16", 4096, 2304, "rms", True, "token"),
        # the largest: Gemma-2-27B's width, a learned gate per channel
        _norms("train_27b", "pair", True, "bf16", 16384, 4608, "rms", True, "channel", residual_scale=0.9),
        # GPT-2 small in fp32, forward and backward
        _norms("train_gpt2_fp32", "pair", True, "fp32", 1024, 768, "layer", False, "none"),
        # a width no vector load divides, layer norm on the branch and a gate per element
        _norms("train_odd", "post", True, "bf16", 517, 1001, "layer", True, "full", branch_scale=0.5),
        # the norms and gates of 12 spliced blocks: many small tensors, a step's latency
        _clip("clip_small", "bf16", 2304, 0, 12, 0.5, "2"),
        # the transcoder at GPT-2 small's width in fp32
        _clip("clip_gpt2_fp32", "fp32", 768, 12288, 0, 1.0, "2"),
        # the transcoder at Gemma-2-2B's width, with one block's norms beside it
        _clip("clip_2b", "bf16", 2304, 36864, 1, 1.0, "2"),
        # the largest: the transcoder at Gemma-2-27B's width
        _clip("clip_27b", "bf16", 4608, 73728, 0, 1.0, "2"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if rng.random() < 0.6:
        train = rng.random() < 0.6
        mode = rng.choice(["pre", "post", "pair", "pair"])
        rows, width = _log_int(rng, 1, 32768), _log_int(rng, 8, 8192)
        if rng.random() < 0.7:
            width = (width + 7) // 8 * 8
        rows = max(1, min(rows, (16384 * 4608 // (2 if dtype == "fp32" else 1)) // width))
        gate = "none" if mode == "pre" else rng.choice(["none", "token", "channel", "full"])
        post = mode == "post" or (mode == "pair" and rng.random() < 0.7)
        return _norms("", mode, train, dtype, rows, width, rng.choice(["rms", "layer"]), post, gate,
                      residual_scale=rng.choice([1.0, 1.0, 0.5, 1.25]), branch_scale=rng.choice([1.0, 1.0, 0.25]))
    act = rng.choice([768, 1024, 1280, 1600, 2304, 3584, 4608, _log_int(rng, 5, 8192)])
    most = 300_000_000 if dtype == "bf16" else 150_000_000
    dict_size = 0 if rng.random() < 0.3 else max(1, min(_log_int(rng, 64, 165888), most // act))
    layers = rng.randint(1, 11) if dict_size == 0 or rng.random() < 0.5 else 0
    return _clip("", dtype, act, dict_size, layers, rng.choice([0.5, 1.0, 1.0, 100000.0]), rng.choice(["2", "2", "2", "1", "inf"]))


# ------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(DEV).manual_seed(int(seed) * 7919 + 17)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _norm_inputs(case, seed):
    """A residual stream: unit-sized entries with a handful of channels some 30 times larger, as trained models have."""
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    rows, width, kind = case["rows"], case["width"], case["kind"]
    outlier = 1.0 + 30.0 * (torch.rand(width, generator=g, device=DEV) < 0.004).float()
    offset = 1.0 if kind == "rms" else 0.0       # Gemma's norms scale by 1 + weight

    def params():
        w = 0.3 * _randn(g, width) + (0.0 if kind == "rms" else 1.0)
        return w.to(dt), (None if kind == "rms" else (0.1 * _randn(g, width)).to(dt))

    t = {"offset": offset, "eps": 1e-6 if kind == "rms" else 1e-5}
    t["x"] = (_randn(g, rows, width) * outlier + 0.2).to(dt)
    t["pre"] = params() if case["mode"] != "post" else None
    t["branch"] = t["post"] = t["gate"] = None
    if case["mode"] != "pre":
        t["branch"] = (2.0 * _randn(g, rows, width) + 0.1).to(dt)
        t["post"] = params() if case["post"] else None
        if case["gate"] == "token":
            t["gate"] = (torch.rand(rows, 1, generator=g, device=DEV) > 0.1).float().mul(0.9).to(dt)
        elif case["gate"] == "channel":
            t["gate"] = (1.0 + 0.2 * _randn(g, width)).to(dt)
        elif case["gate"] == "full":
            t["gate"] = torch.sigmoid(_randn(g, rows, width)).to(dt)
    if case["train"]:
        t["d_hidden"] = (1e-2 * _randn(g, rows, width)).to(dt) if case["mode"] != "pre" else None
        t["d_normed"] = (1e-2 * _randn(g, rows, width)).to(dt) if case["mode"] != "post" else None
    return t


def _grad_inputs(case, seed):
    """Gradients as a step leaves them: W_enc's is a transposed view, many of its features' rows are zero."""
    g, dt, A, D = _gen(seed), DTYPES[case["dtype"]], case["act"], case["dict_size"]
    grads = []
    if D:
        for transposed in (True, False):
            w = torch.randn(D, A, generator=g, device=DEV, dtype=dt)
            w *= (1e-3 * torch.rand(D, 1, generator=g, device=DEV) * (torch.rand(D, 1, generator=g, device=DEV) < 0.8)).to(dt)
            grads.append(w.t() if transposed else w)
        grads.append((1e-3 * _randn(g, D)).to(dt))
        grads.append((1e-2 * _randn(g, A)).to(dt))
    for _ in range(case["layers"]):
        grads += [(1e-2 * _randn(g, A)).to(dt) for _ in range(4)]
        grads.append((1e-1 * _randn(g, 1)).to(dt))                          # a scalar gate
    return grads


def prepare(case, seed):
    if case["op"] != "norms":
        grads = _grad_inputs(case, seed)
        return {"case": case, "grads": grads, "out": [torch.empty_like(x) for x in grads]}
    t = _norm_inputs(case, seed)
    state = {"case": case, "t": t}
    if own:
        from matryoshka_transcoder_amd.block_norm import BlockNorm
        leaves = [t["x"], t["branch"], t["gate"]]
        for which in ("post", "pre"):
            state[which] = None
            if t[which] is not None:
                w, b = t[which]
                m = BlockNorm(case["width"], kind=case["kind"], eps=t["eps"], weight_offset=t["offset"], bias=b is not None,
                              dtype=w.dtype, device=w.device)
                with torch.no_grad():
                    m.weight.copy_(w)
                    if b is not None:
                        m.bias.copy_(b)
                m.requires_grad_(case["train"])
                state[which] = m
                leaves += [m.weight, m.bias]
            else:
                leaves += [None, None]
        if case["train"]:
            for leaf in leaves[:3]:
                if leaf is not None:
                    leaf.requires_grad_(True)
        state["leaves"] = [x for x in leaves if x is not None]
    return state


# ------------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if case["op"] == "norms":
        return _run_norms(case, state) if own else _plain_norms(case, state["t"])
    if own:
        from matryoshka_transcoder_amd.grad_clip import clip_by_global_norm_
        norm = clip_by_global_norm_(state["grads"], case["max_norm"], float(case["p"]), out=state["out"])
        return [norm] + state["out"]
    return _plain_clip(case, state["grads"], state["out"])


def _run_norms(case, state):
    from matryoshka_transcoder_amd.block_norm import residual_block_norm
    t = state["t"]
    if case["mode"] == "pre":
        outs = [state["pre"](t["x"])]
        grads = [t.get("d_normed")]
    else:
        out = residual_block_norm(t["x"], t["branch"], state["post"], gate=t["gate"], residual_scale=case["residual_scale"],
                                  branch_scale=case["branch_scale"], pre=state["pre"])
        outs = list(out) if case["mode"] == "pair" else [out]
        grads = [g for g in (t.get("d_hidden"), t.get("d_normed")) if g is not None]
    if not case["train"]:
        return outs
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, state["leaves"], grads))


# ------------------------------------------------------------------------------------------------------ plain forms
def _plain_norm(x, params, kind, eps, offset):
    mean = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    c = x - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    u = c * rstd
    w = params[0].float() + offset
    y = u * w
    if params[1] is not None:
        y = y + params[1].float()
    return y, u, rstd, w


def _plain_norm_backward(dy, u, rstd, w, kind):
    du = dy * w
    dx = du - u * (du * u).mean(1, keepdim=True)
    if kind == "layer":
        dx = dx - du.mean(1, keepdim=True)
    return dx * rstd


def _plain_norms(case, t):
    kind, mode, dt = case["kind"], case["mode"], DTYPES[case["dtype"]]
    rs, bs = case["residual_scale"], case["branch_scale"]
    gate = None if t["gate"] is None else t["gate"].float()
    hidden, outs, post = t["x"].float(), [], None
    if mode != "pre":
        v = t["branch"].float()
        if t["post"] is not None:
            post = _plain_norm(v, t["post"], kind, t["eps"], t["offset"])
            v = post[0]
        z = v * bs
        hidden = hidden * rs + (z if gate is None else z * gate)
        outs.append(hidden.to(dt))
    if mode != "post":
        pre = _plain_norm(hidden, t["pre"], kind, t["eps"], t["offset"])
        outs.append(pre[0].to(dt))
    if not case["train"]:
        return outs
    d = 0.0 if mode == "pre" else t["d_hidden"].float()
    g_params = []
    if mode != "post":
        dn = t["d_normed"].float()
        d = d + _plain_norm_backward(dn, pre[1], pre[2], pre[3], kind)
        g_params = [(dn * pre[1]).sum(0).to(dt)]
        if t["pre"][1] is not None:
            g_params.append(dn.sum(0).to(dt))
    if mode == "pre":
        return outs + [d.to(dt)] + g_params
    dv = d * bs
    d_gate = None
    if gate is not None:
        d_gate = dv * v
        if case["gate"] == "token":
            d_gate = d_gate.sum(1, keepdim=True)
        elif case["gate"] == "channel":
            d_gate = d_gate.sum(0)
        dv = dv * gate
    g_post = []
    d_branch = dv
    if post is not None:
        g_post = [(dv * post[1]).sum(0).to(dt)]
        if t["post"][1] is not None:
            g_post.append(dv.sum(0).to(dt))
        d_branch = _plain_norm_backward(dv, post[1], post[2], post[3], kind)
    grads = [(d * rs).to(dt), d_branch.to(dt)] + ([] if d_gate is None else [d_gate.to(dt)])
    return outs + grads + g_post + g_params


def _plain_clip(case, grads, out):
    p = float(case["p"])
    total = torch.zeros((), dtype=torch.float64, device=DEV)
    for g in grads:
        a = g.float().abs()
        if p == math.inf:
            total = torch.maximum(total, a.max().double())
        else:
            total = total + (a if p == 1.0 else a * a).sum(dtype=torch.float64)
    norm = (torch.sqrt(total) if p == 2.0 else total).float()
    coef = torch.clamp(case["max_norm"] / (norm + 1e-6), max=1.0)
    for g, o in zip(grads, out):
        o.copy_(g.float() * coef)
    return [norm] + out


# ------------------------------------------------------------------------------------------------------ work
def work(case):
    s = 2 if case["dtype"] == "bf16" else 4
    if case["op"] != "norms":
        n = 2 * case["act"] * case["dict_size"] + (case["dict_size"] + case["act"] if case["dict_size"] else 0)
        n += case["layers"] * (4 * case["act"] + 1)
        return {"bytes": 2 * n * s, "flops": 3 * n}
    n = case["rows"] * case["width"]
    full = 1 if case["gate"] == "full" else 0
    reads, writes, flops = {"pre": (1, 1, 5), "post": (2 + full, 1, 8), "pair": (2 + full, 2, 12)}[case["mode"]]
    if case["train"]:       # each input read once and each output written once over forward and backward together
        reads += 2 if case["mode"] == "pair" else 1
        writes += 1 if case["mode"] == "pre" else 2 + full
        flops *= 3
    return {"bytes": n * s * (reads + writes), "flops": n * flops}


# ------------------------------------------------------------------------------------------------------ exact values
def exact(case, seed):
    if case["op"] != "norms":
        return _exact_clip(case, _grad_inputs(case, seed))
    t = _norm_inputs(case, seed)
    need = case["train"]

    def leaf(x):
        return None if x is None else x.double().requires_grad_(need)

    x, branch, gate = leaf(t["x"]), leaf(t["branch"]), leaf(t["gate"])
    post = None if t["post"] is None else [leaf(p) for p in t["post"]]
    pre = None if t["pre"] is None else [leaf(p) for p in t["pre"]]

    def norm(v, params):
        if case["kind"] == "layer":
            v = v - v.sum(-1, keepdim=True) / v.shape[-1]
        scale = (t["eps"] + torch.sum(v ** 2, -1, keepdim=True) / v.shape[-1]) ** -0.5
        y = v * scale * (t["offset"] + params[0])
        return y if params[1] is None else y + params[1]

    outs, back = [], []
    hidden = x
    if case["mode"] != "pre":
        b = branch if post is None else norm(branch, post)
        b = b if gate is None else gate * b
        hidden = case["residual_scale"] * x + case["branch_scale"] * b
        outs.append(hidden)
        back.append(t.get("d_hidden"))
    if case["mode"] != "post":
        outs.append(norm(hidden, pre))
        back.append(t.get("d_normed"))
    if not need:
        return outs
    leaves = [x, branch, gate] + (post or []) + (pre or [])
    grads = torch.autograd.grad(outs, [v for v in leaves if v is not None], [g.double() for g in back])
    return [o.detach() for o in outs] + list(grads)


def _exact_clip(case, grads):
    p = float(case["p"])
    per = torch.stack([g.double().abs().amax() if p == math.inf else (g.double().abs() ** p).sum() for g in grads])
    norm = per.amax() if p == math.inf else per.sum() if p == 1.0 else per.sum() ** 0.5
    factor = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    return [norm] + [factor * g.double() for g in grads]

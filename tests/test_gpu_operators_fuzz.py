"""Seeded random configurations of the block norms and the clipping against float64 (norm_checks.py)."""
import math
import random

import pytest
import torch

import norm_checks as N
from matryoshka_transcoder_amd.block_norm import BlockNorm, residual_block_norm
from matryoshka_transcoder_amd.grad_clip import clip_by_global_norm_

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _strided(rng, t):
    """t's values in memory of another layout: contiguous, a slice of wider rows, shifted by some elements, or permuted."""
    rows, A = t.shape
    how = rng.choice(["same", "same", "wide", "shift", "gap"])
    if how == "wide":
        w = torch.full((rows, A + rng.choice([1, 8, 24])), 9.0, dtype=t.dtype, device=DEV)
        lo = rng.randrange(0, w.shape[1] - A + 1)
        w[:, lo:lo + A] = t
        return w[:, lo:lo + A]
    if how == "shift":
        k = rng.choice([1, 2, 4, 8])
        b = torch.full((rows * A + k,), 9.0, dtype=t.dtype, device=DEV)
        b[k:] = t.reshape(-1)
        return b[k:].view(rows, A)
    if how == "gap":
        b = torch.full((rows, 2, A), 9.0, dtype=t.dtype, device=DEV)
        b[:, 1] = t
        return b[:, 1]
    return t


@pytest.mark.parametrize("seed", range(60))
def test_norms(seed):
    rng = random.Random(seed)
    g = torch.Generator("cpu").manual_seed(seed)
    dt = rng.choice([torch.bfloat16, torch.float32])
    A = int(round(math.exp(rng.uniform(0, math.log(8192)))))
    if rng.random() < 0.6:
        A = min(8192, (A + 7) // 8 * 8)
    rows = max(1, min(int(round(math.exp(rng.uniform(0, math.log(3000))))), 3_000_000 // A))
    mode = rng.choice(["pre", "post", "pair", "pair"])
    kinds = [rng.choice(["rms", "layer"]) for _ in range(2)]
    rs, bs = rng.choice([1.0, 0.5, -1.0]), rng.choice([1.0, 2.0])
    gate_kind = rng.choice(["none", "scalar", "token", "channel", "full"])

    def rand(*s, scale=1.0):
        return (torch.randn(s, generator=g) * scale).to(dt).to(DEV)

    def norm(kind):
        affine = rng.random() < 0.8
        m = BlockNorm(A, kind=kind, eps=rng.choice([1e-6, 1e-3]), weight_offset=rng.choice([0.0, 1.0]), affine=affine,
                      bias=affine and rng.random() < 0.5, dtype=dt, device=DEV)
        with torch.no_grad():
            for p in m.parameters():
                p.add_(rand(A, scale=0.3))
        return m.requires_grad_(rng.random() < 0.7)

    res = _strided(rng, rand(rows, A, scale=rng.choice([0.1, 1.0, 30.0]))).requires_grad_(True)
    branch = gate = post = None
    if mode != "pre":
        branch = _strided(rng, rand(rows, A)).requires_grad_(rng.random() < 0.8)
        post = norm(kinds[0]) if rng.random() < 0.7 else None
        shape = {"none": None, "scalar": (), "channel": (A,), "token": (rows, 1), "full": (rows, A)}[gate_kind]
        gate = None if shape is None else rand(*shape).requires_grad_(rng.random() < 0.7)
        if gate_kind == "full":
            gate = _strided(rng, gate.detach()).requires_grad_(True)
    pre = norm(kinds[1]) if mode != "post" else None
    dh = _strided(rng, rand(rows, A)) if mode != "pre" else None
    dn = _strided(rng, rand(rows, A)) if mode != "post" else None
    spec = lambda m: None if m is None else dict(w=m.weight, b=m.bias, kind=m.kind, eps=m.eps, off=m.weight_offset)       # noqa: E731
    if gate is not None and gate_kind == "channel" and A == 1:
        pytest.skip("one column: the restatement takes [1] for a channel gate of one")
    want = N.reference(res, branch, gate, spec(post), spec(pre), 1.0 if mode == "pre" else rs, bs, dh, dn)
    if mode == "pre":
        outs, names, gr = [pre(res)], ["normed"], [dn]
    else:
        out = residual_block_norm(res, branch, post, gate=gate, residual_scale=rs, branch_scale=bs, pre=pre)
        outs, names, gr = ([out], ["hidden"], [dh]) if mode == "post" else (list(out), ["hidden", "normed"], [dh, dn])
    leaves = {"residual": res, "branch": branch, "gate": gate, "post_w": post and post.weight, "post_b": post and post.bias,
              "pre_w": pre and pre.weight, "pre_b": pre and pre.bias}
    leaves = {k: v for k, v in leaves.items() if v is not None and v.requires_grad}
    got = dict(zip(names, outs))
    got.update(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gr)))
    for k, v in got.items():
        N.compare(k, v, want[k], dt)


@pytest.mark.parametrize("seed", range(30))
def test_clip(seed):
    rng = random.Random(1000 + seed)
    g = torch.Generator("cpu").manual_seed(seed)
    ts = []
    for _ in range(rng.choice([1, 3, 20, 150])):
        dt = rng.choice([torch.bfloat16, torch.float32])
        n = int(round(math.exp(rng.uniform(0, math.log(60000)))))
        t = (torch.randn(n + 3, generator=g) * 10.0 ** rng.randint(-4, 1)).to(dt).to(DEV)
        t = t[rng.choice([0, 1, 3]):][:n]
        if rng.random() < 0.3 and n % 2 == 0:
            t = t.view(2, n // 2).t()
        ts.append(t)
    p = rng.choice([1.0, 2.0, 2.0, math.inf])
    d = [t.double().abs() for t in ts]
    norm = max(float(t.max()) for t in d) if p == math.inf else float(sum(t.pow(p).sum() for t in d)) ** (1.0 / p)
    limit = norm * rng.choice([0.01, 0.5, 2.0])
    before = [t.clone() for t in ts]
    out = [torch.empty_like(t) for t in ts] if rng.random() < 0.5 else None
    got = float(clip_by_global_norm_(ts, limit, p, out=out))
    assert abs(got - norm) <= 2 ** -24 * 1.01 * norm
    coef = min(1.0, limit / (norm + 1e-6))
    for b, t, o in zip(before, ts, ts if out is None else out):
        exact = coef * b.double()
        assert bool(((o.double() - exact).abs() <= (torch.finfo(b.dtype).eps / 2 + 5 * 2.0 ** -24) * exact.abs() + 1e-44).all())
        assert out is None or torch.equal(t, b)

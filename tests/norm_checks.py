"""float64 restatement of the block norms with, for every output, a bound on what fp32 arithmetic may lose.

Each value comes with a magnitude: the sum of the absolute values of the terms it is made of.  A result computed in fp32
and rounded once to the model dtype then differs from the exact one by at most
    half a step of the dtype * |exact|  +  K * 2^-24 * magnitude,
K counting roundings in sequence: a row sum is 8 adds in a thread, 6 levels in a wave, 4 over the waves, its terms carry up
to 6 more, and at most two row sums feed an output through statistics -> K = 64 covers them with the products around.
A column sum adds ceil(rows / 256) rows in a thread, up to 15 row groups and 16 + 16 partials: K grows by that."""
import torch

K_ROW = 64


def k_cols(rows):
    return K_ROW + (rows + 255) // 256 + 48


def _norm(v, vmag, w, b, kind, eps, off):
    n = v.shape[1]
    mu = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    c = v - mu
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    cmag = vmag + (vmag.mean(1, keepdim=True) if kind == "layer" else 0.0)
    # how much of the row survives the subtraction / cancellation: errors of 1/std scale with it
    ratio = (torch.sqrt((cmag * cmag).mean(1, keepdim=True) + eps) * rstd).clamp_min(1.0)
    u, umag = c * rstd, cmag * rstd * ratio
    we = torch.ones(n, dtype=v.dtype, device=v.device) if w is None else off + w
    wmag = torch.ones_like(we) if w is None else abs(off) + w.abs()
    bb = torch.zeros_like(we) if b is None else b
    return dict(y=u * we + bb, ymag=umag * wmag + bb.abs(), u=u, umag=umag, rstd=rstd * 1.0, ratio=ratio, w=we, wmag=wmag, b=bb)


def _norm_back(g, gmag, nm, kind):
    """gradient through u = (v - mu) rstd for du = g (already multiplied by the weight)"""
    dx = g - nm["u"] * (g * nm["u"]).mean(1, keepdim=True)
    mag = gmag + nm["umag"] * (gmag * nm["umag"]).mean(1, keepdim=True)
    if kind == "layer":
        dx = dx - g.mean(1, keepdim=True)
        mag = mag + gmag.mean(1, keepdim=True)
    return dx * nm["rstd"], mag * nm["rstd"] * nm["ratio"]


def reference(residual, branch, gate, post, pre, rs=1.0, bs=1.0, d_hidden=None, d_normed=None):
    """All tensors 2-D [rows, A] (gate: None, [A], [rows, 1], [rows, A] or 0-dim); post / pre: None or dicts with w, b, kind,
    eps, off.  Returns {name: (value, magnitude, K)}; gradients when d_hidden or d_normed is given."""
    f = lambda t: None if t is None else t.detach().double()          # noqa: E731
    residual, branch, gate, d_hidden, d_normed = f(residual), f(branch), f(gate), f(d_hidden), f(d_normed)
    rows = residual.shape[0]
    kc = k_cols(rows)
    out = {}
    h, hmag = residual, residual.abs()
    pn = None
    if branch is not None:
        if post is not None:
            pn = _norm(branch, branch.abs(), f(post["w"]), f(post["b"]), post["kind"], post["eps"], post["off"])
            v, vmag = pn["y"], pn["ymag"]
        else:
            v, vmag = branch, branch.abs()
        g = torch.ones((), dtype=h.dtype, device=h.device) if gate is None else gate
        z, zmag = bs * v, abs(bs) * vmag
        h, hmag = rs * residual + g * z, abs(rs) * residual.abs() + g.abs() * zmag
        out["hidden"] = (h, hmag, K_ROW)
    if pre is not None:
        qn = _norm(h, hmag, f(pre["w"]), f(pre["b"]), pre["kind"], pre["eps"], pre["off"])
        out["normed"] = (qn["y"], qn["ymag"], K_ROW)
    if d_hidden is None and d_normed is None:
        return out
    D = torch.zeros_like(h) if d_hidden is None else d_hidden
    Dmag = D.abs()
    if pre is not None and d_normed is not None:
        out["pre_w"] = ((d_normed * qn["u"]).sum(0), (d_normed.abs() * qn["umag"]).sum(0), kc)
        out["pre_b"] = (d_normed.sum(0), d_normed.abs().sum(0), kc)
        dx, mag = _norm_back(d_normed * qn["w"], d_normed.abs() * qn["wmag"], qn, pre["kind"])
        D, Dmag = D + dx, Dmag + mag
    out["residual"] = (rs * D, abs(rs) * Dmag, K_ROW)
    if branch is None:
        return out
    if gate is not None:
        dg, dgmag = D * z, Dmag * zmag
        if gate.dim() == 0:
            out["gate"] = (dg.sum(), dgmag.sum(), kc + K_ROW)
        elif gate.dim() == 1:
            out["gate"] = (dg.sum(0), dgmag.sum(0), kc)
        elif gate.shape[1] == 1 and residual.shape[1] != 1:
            out["gate"] = (dg.sum(1, keepdim=True), dgmag.sum(1, keepdim=True), K_ROW)
        else:
            out["gate"] = (dg, dgmag, K_ROW)
    dv, dvmag = bs * g * D, abs(bs) * g.abs() * Dmag
    if pn is not None:
        out["post_w"] = ((dv * pn["u"]).sum(0), (dvmag * pn["umag"]).sum(0), kc)
        out["post_b"] = (dv.sum(0), dvmag.sum(0), kc)
        dv, dvmag = _norm_back(dv * pn["w"], dvmag * pn["wmag"], pn, post["kind"])
    out["branch"] = (dv, dvmag, K_ROW)
    return out


def compare(name, got, want, dtype):
    value, mag, k = want
    got = got.detach().double().reshape(value.shape)
    allowed = torch.finfo(dtype).eps / 2 * value.abs() + k * 2.0 ** -24 * mag + 1e-37
    bad = ~((got - value).abs() <= allowed)
    bad &= ~(torch.isnan(got) & torch.isnan(value))
    bad &= ~(got == value)                      # equal infinities
    if bool(bad.any()):
        i = bad.reshape(-1).nonzero()[0].item()
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off; first at {i}: got {got.reshape(-1)[i].item()}, "
                             f"exact {value.reshape(-1)[i].item()}, allowed {allowed.reshape(-1)[i].item()}")

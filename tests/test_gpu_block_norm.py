"""The block norms on the GPU against a float64 restatement, with tolerances from counted roundings (norm_checks.py)."""
import ctypes as C

import pytest
import torch

import norm_checks as N
from matryoshka_transcoder_amd import _lib
from matryoshka_transcoder_amd.block_norm import BlockNorm, block_norm, residual_block_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float32]


def _rand(g, *shape, scale=1.0):
    return torch.randn(shape, generator=g) * scale


def _norm_module(g, A, kind, dt, offset=None, affine=True, bias=None):
    offset = (1.0 if kind == "rms" else 0.0) if offset is None else offset
    m = BlockNorm(A, kind=kind, eps=1e-6 if kind == "rms" else 1e-5, weight_offset=offset, affine=affine, bias=bias, dtype=dt,
                  device=DEV)
    with torch.no_grad():
        if m.weight is not None:
            m.weight.copy_(_rand(g, A, scale=0.3) + 1.0 - offset)
        if m.bias is not None:
            m.bias.copy_(_rand(g, A, scale=0.2))
    return m


def _spec(m):
    return None if m is None else dict(w=m.weight, b=m.bias, kind=m.kind, eps=m.eps, off=m.weight_offset)


def _gate(g, kind, rows, A, dt):
    if kind == "none":
        return None
    shape = {"scalar": (), "channel": (A,), "token": (rows, 1), "full": (rows, A)}[kind]
    t = _rand(g, *shape, scale=0.5) + 0.8
    if kind == "token" and rows > 1:
        t[::3] = 0.0                                   # tokens kept out of the splice
    return t.to(dt).to(DEV)


def _check(rows, A, dt, mode, post_kind, pre_kind, gate_kind, rs=1.0, bs=1.0, seed=0, edit=None, affine=True, bias=None):
    g = torch.Generator("cpu").manual_seed(seed * 977 + rows * 31 + A)
    residual = (_rand(g, rows, A, scale=2.0) + 0.3).to(dt)
    branch = None if mode == "pre" else (_rand(g, rows, A) - 0.1).to(dt)
    if edit is not None:
        edit(residual, branch)
    residual = residual.to(DEV).requires_grad_(True)
    branch = None if branch is None else branch.to(DEV).requires_grad_(True)
    post = _norm_module(g, A, post_kind, dt, affine=affine, bias=bias) if post_kind and mode != "pre" else None
    pre = _norm_module(g, A, pre_kind, dt, affine=affine, bias=bias) if mode != "post" else None
    gate = None if mode == "pre" else _gate(g, gate_kind, rows, A, dt)
    if gate is not None:
        gate.requires_grad_(True)
    dh = None if mode == "pre" else _rand(g, rows, A).to(dt).to(DEV)
    dn = None if mode == "post" else _rand(g, rows, A).to(dt).to(DEV)
    want = N.reference(residual, branch, gate, _spec(post), _spec(pre), rs, bs, dh, dn)
    if mode == "pre":
        outs, names, grads = [pre(residual)], ["normed"], [dn]
    else:
        out = residual_block_norm(residual, branch, post, gate=gate, residual_scale=rs, branch_scale=bs, pre=pre)
        outs, names, grads = ([out], ["hidden"], [dh]) if mode == "post" else (list(out), ["hidden", "normed"], [dh, dn])
    leaves = {"residual": residual, "branch": branch, "gate": gate, "post_w": post and post.weight, "post_b": post and post.bias,
              "pre_w": pre and pre.weight, "pre_b": pre and pre.bias}
    leaves = {k: v for k, v in leaves.items() if v is not None}
    got = dict(zip(names, outs))
    got.update(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), grads)))
    for k, v in got.items():
        assert v.dtype == dt and v.is_contiguous()
        N.compare(k, v, want[k], dt)
    with torch.no_grad():                              # the path without a graph gives the same bits
        if mode == "pre":
            again = [pre(residual)]
        else:
            out = residual_block_norm(residual, branch, post, gate=gate, residual_scale=rs, branch_scale=bs, pre=pre)
            again = [out] if mode == "post" else list(out)
    for a, b in zip(again, outs):
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,A", [(1030, 1024), (1025, 3584), (9, 1536), (1, 2304), (3, 768), (130, 1600), (257, 2304), (65, 4608), (9, 8192), (1, 8), (70, 64),
                                    (33, 520), (1, 1), (5, 7), (300, 1001), (2, 8191)])
def test_pair_rms(rows, A, dt):
    _check(rows, A, dt, "pair", "rms", "rms", "none")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,A", [(1, 768), (131, 1600), (17, 1283), (40, 4608), (30, 256), (29, 1280), (5, 2304)])
@pytest.mark.parametrize("gate", ["none", "scalar", "token", "channel", "full"])
def test_pair_layer_gates(rows, A, gate, dt):
    _check(rows, A, dt, "pair", "layer", "layer", gate, rs=0.75, bs=1.5)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("mode,post,pre", [("pre", None, "rms"), ("pre", None, "layer"), ("post", "rms", None), ("post", "layer", None),
                                           ("post", None, None), ("pair", None, "layer"), ("pair", None, "rms"), ("pair", "rms", "layer"),
                                           ("pair", "layer", "rms")])
@pytest.mark.parametrize("gate", ["none", "token", "scalar"])
def test_modes(mode, post, pre, gate, dt):
    _check(77, 520, dt, mode, post, pre, gate, rs=1.0 if mode == "pre" else -0.5, bs=0.25)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("affine,bias", [(False, False), (True, False), (True, True)])
def test_parameters_absent(affine, bias, dt):
    for kind in ("rms", "layer"):
        _check(19, 264, dt, "pair", kind, kind, "channel", affine=affine, bias=bias)


@pytest.mark.parametrize("dt", DTYPES)
def test_many_rows(dt):
    _check(5000, 512, dt, "pair", "rms", "layer", "scalar")
    _check(5003, 2304, dt, "pair", "rms", "rms", "token", seed=3)


@pytest.mark.parametrize("dt", DTYPES)
def test_rows_far_from_zero_and_empty(dt):
    def edit(r, b):
        r[0] = 0
        b[0] = 0                                       # a row of zeros: eps alone
        r[1] = 0
        b[2] = 0
        r[3] += 64.0                                   # mean far above the spread
        b[4] -= 64.0
    for kind in ("rms", "layer"):
        _check(6, 776, dt, "pair", kind, kind, "none", edit=edit)
        _check(6, 776, dt, "pair", kind, kind, "token", edit=edit)


def test_non_finite_rows_stay_alone():
    """inf / NaN in a row spoil that row's outputs and the column sums, no other row."""
    g = torch.Generator("cpu").manual_seed(5)
    x = _rand(g, 8, 520).to(DEV)
    x[2, 3], x[5, 100] = float("inf"), float("nan")
    y = _rand(g, 8, 520).to(DEV)
    m = _norm_module(g, 520, "rms", torch.float32)
    hidden, normed = residual_block_norm(x, y, m, pre=m)
    clean = [0, 1, 3, 4, 6, 7]
    h2, n2 = residual_block_norm(x[clean], y[clean], m, pre=m)
    assert torch.equal(hidden[clean], h2) and torch.equal(normed[clean], n2)
    assert bool(torch.isnan(normed[5]).all()) and not bool(torch.isfinite(normed[2]).all())


@pytest.mark.parametrize("dt", DTYPES)
def test_strides_and_alignment(dt):
    """Row slices of a wider cache, permuted and expanded leading dimensions, strided columns, odd base addresses: the values
    of the contiguous call (which path serves them is a matter of alignment, so to within the fp32 sums)."""
    g = torch.Generator("cpu").manual_seed(11)
    b, s, A = 3, 5, 264
    post, pre = _norm_module(g, A, "layer", dt), _norm_module(g, A, "rms", dt)

    def run(res, br, gate=None):
        leaves = [res.detach().requires_grad_(True), br.detach().requires_grad_(True)]
        with torch.enable_grad():
            out = residual_block_norm(leaves[0], leaves[1], post, gate=gate, pre=pre)
            gr = torch.autograd.grad(out, leaves, [torch.ones_like(out[0]), torch.ones_like(out[1])])
        want = N.reference(res.reshape(-1, A), br.reshape(-1, A), None if gate is None else gate.reshape(-1, gate.shape[-1]), _spec(post),
                           _spec(pre), 1.0, 1.0, torch.ones(res.numel() // A, A, device=DEV), torch.ones(res.numel() // A, A, device=DEV))
        for k, v in zip(("hidden", "normed", "residual", "branch"), list(out) + list(gr)):
            assert tuple(v.shape) == tuple(res.shape)
            N.compare(k, v, want[k], dt)

    base, base2 = _rand(g, b, s, A).to(dt).to(DEV), _rand(g, b, s, A).to(dt).to(DEV)
    run(base, base2)
    wide = _rand(g, b, s, A + 24).to(dt).to(DEV)
    run(wide[..., 8:8 + A], base2)                                   # aligned rows at a larger stride
    run(wide[..., 3:3 + A], base2)                                   # rows that no 16-byte access may touch
    run(base.transpose(0, 1), base2.transpose(0, 1))                 # [s, b, A]
    run(base[:1].expand(b, s, A), base2)                             # broadcast residual
    cols = _rand(g, b, s, 2 * A).to(dt).to(DEV)
    run(cols[..., ::2], base2)                                       # strided columns
    odd = torch.empty(b * s * A + 1, dtype=dt, device=DEV)[1:].reshape(b, s, A).copy_(base)
    run(odd, base2)                                                  # base address off by one element
    run(base[0, 0], base2[0, 0])                                     # one token, one dimension
    gate = (torch.rand(b, 1, 1, generator=g) > 0.5).to(dt).to(DEV).expand(b, s, 1)
    run(base, base2, gate)
    run(base, base2, wide[..., 1:1 + A])


def test_expanded_residual_gradient():
    """A residual broadcast over the batch: its gradient is the sum over the copies."""
    g = torch.Generator("cpu").manual_seed(12)
    r = _rand(g, 1, 4, 128).to(DEV).requires_grad_(True)
    y = _rand(g, 3, 4, 128).to(DEV)
    (gr,) = torch.autograd.grad(residual_block_norm(r.expand(3, 4, 128), y, None).sum(), [r])
    assert gr.shape == r.shape and torch.equal(gr, torch.full_like(gr, 3.0))


@pytest.mark.parametrize("dt", DTYPES)
def test_partial_gradients(dt):
    """Only what is asked for: one incoming gradient, frozen norms, a branch without gradient."""
    g = torch.Generator("cpu").manual_seed(13)
    rows, A = 40, 520
    res, br = _rand(g, rows, A).to(dt).to(DEV), _rand(g, rows, A).to(dt).to(DEV)
    post, pre = _norm_module(g, A, "rms", dt), _norm_module(g, A, "layer", dt)
    d = _rand(g, rows, A).to(dt).to(DEV)
    for dh, dn in ((d, None), (None, d)):
        r, b = res.clone().requires_grad_(True), br.clone().requires_grad_(True)
        hidden, normed = residual_block_norm(r, b, post, pre=pre)
        out = hidden if dn is None else normed
        params = [post.weight] + ([] if dn is None else [pre.weight, pre.bias])
        got = torch.autograd.grad(out, [r, b] + params, d)
        want = N.reference(res, br, None, _spec(post), _spec(pre), 1.0, 1.0, dh, dn)
        for k, v in zip(("residual", "branch", "post_w", "pre_w", "pre_b"), got):
            N.compare(k, v, want[k], dt)
    hidden, normed = residual_block_norm(r, br, post, pre=pre)
    hidden.backward(d)                                               # normed unused: the pre norm's parameters get zeros or nothing
    assert pre.weight.grad is None or not bool(pre.weight.grad.any())
    post.requires_grad_(False)
    pre.requires_grad_(False)
    r = res.clone().requires_grad_(True)
    hidden, normed = residual_block_norm(r, br, post, pre=pre)
    (gr,) = torch.autograd.grad([hidden, normed], [r], [d, d])
    N.compare("residual", gr, N.reference(res, br, None, _spec(post), _spec(pre), 1.0, 1.0, d, d)["residual"], dt)


@pytest.mark.parametrize("dt", DTYPES)
def test_frozen_norms_with_bias(dt):
    """Frozen layer norms: their biases still belong to the recomputed sum that the pre norm's gradient is taken at."""
    g = torch.Generator("cpu").manual_seed(17)
    rows, A = 70, 264
    post, pre = _norm_module(g, A, "layer", dt).requires_grad_(False), _norm_module(g, A, "layer", dt).requires_grad_(False)
    for gate_kind in ("none", "channel", "full", "scalar"):
        res, br = _rand(g, rows, A).to(dt).to(DEV).requires_grad_(True), _rand(g, rows, A).to(dt).to(DEV).requires_grad_(True)
        gate, d = _gate(g, gate_kind, rows, A, dt), _rand(g, rows, A).to(dt).to(DEV)
        out = residual_block_norm(res, br, post, gate=gate, pre=pre)
        want = N.reference(res, br, gate, _spec(post), _spec(pre), 1.0, 1.0, d, d)
        for k, v in zip(("residual", "branch"), torch.autograd.grad(out, [res, br], [d, d])):
            N.compare(k, v, want[k], dt)


@pytest.mark.parametrize("dt", DTYPES)
def test_streaming_sizes(dt):
    """Passes over more than the Infinity Cache holds run with non-temporal accesses: the same bits as row blocks within it."""
    g = torch.Generator("cpu").manual_seed(18)
    rows, A = (34000, 2304) if dt == torch.bfloat16 else (17000, 2304)
    gen = torch.Generator(DEV).manual_seed(18)
    res, br, dh, dn = (torch.randn(rows, A, generator=gen, device=DEV).to(dt) for _ in range(4))
    post, pre = _norm_module(g, A, "rms", dt), _norm_module(g, A, "rms", dt)

    def both(lo, hi):
        r, b = res[lo:hi].detach().requires_grad_(True), br[lo:hi].detach().requires_grad_(True)
        out = residual_block_norm(r, b, post, pre=pre)
        return list(out) + list(torch.autograd.grad(out, [r, b, post.weight], [dh[lo:hi], dn[lo:hi]]))

    whole = both(0, rows)
    for lo in range(0, rows, 4000):
        part = both(lo, min(rows, lo + 4000))
        for a, b in zip(whole[:4], part[:4]):
            assert torch.equal(a[lo:lo + 4000], b)
    N.compare("post_w", whole[4], N.reference(res, br, None, _spec(post), _spec(pre), 1.0, 1.0, dh, dn)["post_w"], dt)
    alone = block_norm(res, pre.weight, eps=1e-6, weight_offset=1.0)
    assert torch.equal(alone[1000:2000], block_norm(res[1000:2000], pre.weight, eps=1e-6, weight_offset=1.0))


def test_offsets_beyond_32_bits():
    """More than 2^31 elements, and more rows than one launch has waves for: the far rows equal a call on them alone."""
    for rows, A in (((1 << 31) // 2304 + 1000, 2304), ((1 << 25) + 77, 8)):
        x = torch.zeros(rows, A, dtype=torch.bfloat16, device=DEV)
        gen = torch.Generator(DEV).manual_seed(19)
        x[-300:] = torch.randn(300, A, generator=gen, device=DEV).bfloat16()
        m = BlockNorm(A, kind="layer", dtype=torch.bfloat16, device=DEV)
        with torch.no_grad():
            y = m(x)
            assert torch.equal(y[-300:], m(x[-300:])) and not bool(y[:1000].any())
            h, n = residual_block_norm(x, x, m, pre=m)
            h2, n2 = residual_block_norm(x[-300:], x[-300:], m, pre=m)
            assert torch.equal(h[-300:], h2) and torch.equal(n[-300:], n2)
        del y, h, n
        r = x.requires_grad_(True)
        (g,) = torch.autograd.grad(m(r), [r], x.detach())
        r2 = x[-300:].detach().requires_grad_(True)
        (g2,) = torch.autograd.grad(m(r2), [r2], r2.detach())
        assert torch.equal(g[-300:], g2)
        del x, r, g


def test_gradient_against_differences():
    """<gradient, v> against central differences of the float64 forward along v."""
    g = torch.Generator("cpu").manual_seed(14)
    rows, A, dt = 6, 96, torch.float32
    res, br, gate = _rand(g, rows, A).to(DEV), _rand(g, rows, A).to(DEV), _rand(g, rows, 1).to(DEV)
    post, pre = _norm_module(g, A, "layer", dt), _norm_module(g, A, "rms", dt)
    dh, dn = _rand(g, rows, A).to(DEV), _rand(g, rows, A).to(DEV)
    leaves = [t.requires_grad_(True) for t in (res, br, gate)] + [post.weight, post.bias, pre.weight]
    out = residual_block_norm(res, br, post, gate=gate, residual_scale=0.5, branch_scale=2.0, pre=pre)
    grads = torch.autograd.grad(out, leaves, [dh, dn])
    base = [t.detach().double() for t in leaves]

    def loss(ts):
        o = N.reference(ts[0], ts[1], ts[2], dict(_spec(post), w=ts[3], b=ts[4]), dict(_spec(pre), w=ts[5]), 0.5, 2.0)
        return float((o["hidden"][0] * dh.double()).sum() + (o["normed"][0] * dn.double()).sum())

    for i in range(len(leaves)):
        v = _rand(g, *leaves[i].shape).double().to(DEV)
        e = 1e-5
        plus, minus = list(base), list(base)
        plus[i], minus[i] = base[i] + e * v, base[i] - e * v
        diff = (loss(plus) - loss(minus)) / (2 * e)
        dot = float((grads[i].double() * v).sum())
        # differences: e^2 third derivatives (~1e-9 of the terms) + float64 noise / e (~1e-10); gradient: fp32, K 2^-24 a term
        scale = float((grads[i].double().abs() * v.abs()).sum())
        assert abs(diff - dot) <= 2e-5 * scale, (i, diff, dot, scale)


@pytest.mark.parametrize("dt", DTYPES)
def test_same_bits_twice_and_on_another_stream(dt):
    g = torch.Generator("cpu").manual_seed(15)
    rows, A = 3001, 768
    res, br = _rand(g, rows, A).to(dt).to(DEV).requires_grad_(True), _rand(g, rows, A).to(dt).to(DEV).requires_grad_(True)
    post, pre = _norm_module(g, A, "layer", dt), _norm_module(g, A, "layer", dt)
    gate = _gate(g, "channel", rows, A, dt).requires_grad_(True)
    d = _rand(g, rows, A).to(dt).to(DEV)
    leaves = [res, br, gate] + list(post.parameters()) + list(pre.parameters())

    def once():
        out = residual_block_norm(res, br, post, gate=gate, pre=pre)
        return list(out) + list(torch.autograd.grad(out, leaves, [d, d]))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_captured_and_replayed():
    """Forward and backward recorded into one graph, replayed over new inputs with eager work in between."""
    g = torch.Generator("cpu").manual_seed(16)
    rows, A, dt = 65, 520, torch.bfloat16
    post, pre = _norm_module(g, A, "rms", dt), _norm_module(g, A, "layer", dt)
    leaves = [torch.zeros(rows, A, dtype=dt, device=DEV).requires_grad_(True) for _ in range(2)]
    params = [post.weight, pre.weight, pre.bias]
    d = _rand(g, rows, A).to(dt).to(DEV)

    def step(res, br):
        out = residual_block_norm(res, br, post, pre=pre)
        return list(out) + list(torch.autograd.grad(out, [res, br] + params, [d, d]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*leaves)
    for i in range(3):
        x, y = _rand(g, rows, A).to(dt).to(DEV), _rand(g, rows, A).to(dt).to(DEV)
        with torch.no_grad():
            leaves[0].copy_(x)
            leaves[1].copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        want = step(x.requires_grad_(True), y.requires_grad_(True))
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_c_call_leaves_gaps_and_later_rows_alone():
    """Output rows at a larger stride: the columns between them and the rows behind the last stay as they were."""
    from matryoshka_transcoder_amd.engine import _p, _stream
    lib = _lib.load()
    for A, ld in ((64, 80), (61, 67)):
        rows = 5
        x, y = torch.randn(rows, A, device=DEV), torch.randn(rows, A, device=DEV)
        hidden, normed = torch.full((rows + 2, ld), 7.0, device=DEV), torch.full((rows + 2, ld), 7.0, device=DEV)
        d = _lib.BlockNormDesc(rows=rows, A=A, dtype=_lib.MTC_F32, has_branch=1, pre_kind=_lib.MTC_NORM_RMS, pre_eps=1e-6,
                               residual_scale=1.0, branch_scale=1.0, ld_residual=A, ld_branch=A, ld_hidden=ld, ld_normed=ld)
        _lib.check(lib.mtc_block_norm_fwd(C.byref(d), _p(x), _p(y), None, None, None, None, None, _p(hidden), _p(normed), None,
                                          _stream()))
        torch.cuda.synchronize()
        assert torch.equal(hidden[:rows, :A], x + y)
        for o in (hidden, normed):
            assert bool((o[rows:] == 7.0).all()) and bool((o[:, A:] == 7.0).all())


def test_no_rows():
    m = BlockNorm(64, kind="layer", dtype=torch.float32, device=DEV)
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    y = torch.zeros(0, 64, device=DEV, requires_grad=True)
    h, n = residual_block_norm(x, y, m, pre=m)
    assert h.shape == n.shape == (0, 64)
    (h.sum() + n.sum()).backward()
    assert x.grad.shape == (0, 64) and not bool(m.weight.grad.any()) and not bool(m.bias.grad.any())
    assert block_norm(torch.zeros(2, 0, 64, device=DEV)).shape == (2, 0, 64)


def test_refusals_on_the_gpu():
    x = torch.randn(4, 64, device=DEV)
    with pytest.raises(_lib.MtcError, match="share shape"):
        residual_block_norm(x, x.bfloat16())
    with pytest.raises(_lib.MtcError, match="share shape"):
        residual_block_norm(x, x[:3])
    with pytest.raises(_lib.MtcError, match="width 32"):
        residual_block_norm(x, x, BlockNorm(32, device=DEV))
    with pytest.raises(_lib.MtcError, match="weight"):
        block_norm(x, torch.ones(64, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(_lib.MtcError, match="weight"):
        block_norm(x, torch.ones(64))
    with pytest.raises(_lib.MtcError, match="gate of shape"):
        residual_block_norm(x, x, gate=torch.ones(4, device=DEV))
    with pytest.raises(_lib.MtcError, match="gate must be"):
        residual_block_norm(x, x, gate=torch.ones(64))
    with pytest.raises(_lib.MtcError, match="unsupported model dtype"):
        block_norm(x.half())
    with pytest.raises(_lib.MtcError, match="outside"):
        block_norm(torch.zeros(1, 8200, device=DEV))
    with pytest.raises(_lib.MtcError, match="at least one dimension"):
        block_norm(torch.zeros((), device=DEV))
    with pytest.raises(RuntimeError):                                # second derivatives are refused, not wrong
        r = x.clone().requires_grad_(True)
        (gr,) = torch.autograd.grad(block_norm(r).sum(), [r], create_graph=True)
        gr.sum().backward()


def test_recording_beside_a_live_eager_graph_is_refused():
    """The refusal comes before the engine touches the leaf's accumulation node; once the eager graph is gone, the same
    recording works."""
    x = torch.randn(7, 128, device=DEV).requires_grad_(True)
    norm = BlockNorm(128, device=DEV)
    d = torch.randn(7, 128, device=DEV)
    alive = norm(x)                                                  # keeps the leaves' nodes of the default stream
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(norm(x), [x, norm.weight], d)
    with torch.no_grad():
        want = block_norm(x, norm.weight)
    assert torch.equal(alive, want)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(norm(x), [x, norm.weight], d)
    for _ in range(2):
        with torch.no_grad():
            x.copy_(torch.randn(7, 128, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        y = x.detach().clone().requires_grad_(True)
        for a, b in zip(got, torch.autograd.grad(norm(y), [y, norm.weight], d)):
            assert torch.equal(a, b)


def test_only_the_asked_gradients_are_computed():
    """autograd.grad over a part of the leaves: the same bits as with all of them."""
    g = torch.Generator("cpu").manual_seed(23)
    post, pre = _norm_module(g, 96, "layer", torch.float32), _norm_module(g, 96, "rms", torch.float32)
    r, b, gate = (_rand(g, *s).to(DEV).requires_grad_(True) for s in ((9, 96), (9, 96), (9, 1)))
    leaves = [r, b, gate, post.weight, post.bias, pre.weight]
    d = _rand(g, 9, 96).to(DEV)
    grads = lambda which: torch.autograd.grad(residual_block_norm(r, b, post, gate=gate, pre=pre), which, [d, d])      # noqa: E731
    for leaf, want in zip(leaves, grads(leaves)):
        assert torch.equal(grads([leaf])[0], want)
    for leaf in leaves[:3]:                                          # without a gate the edges behind it move up
        if leaf is not gate:
            assert torch.autograd.grad(residual_block_norm(r, b, post), [leaf], d)[0].shape == leaf.shape
    (dw,) = torch.autograd.grad(residual_block_norm(r, b, post), [post.weight], d)
    (db,) = torch.autograd.grad(residual_block_norm(r, b, post), [post.bias], d)
    all_ = torch.autograd.grad(residual_block_norm(r, b, post), [post.weight, post.bias], d)
    assert torch.equal(dw, all_[0]) and torch.equal(db, all_[1])


def test_forward_mode_is_refused():
    x = torch.randn(4, 64, device=DEV)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(_lib.MtcError, match="forward-mode"):
            block_norm(dual)
        with pytest.raises(_lib.MtcError, match="forward-mode"):
            residual_block_norm(x, x, gate=dual)


@pytest.mark.parametrize("dt,A,branch", [(torch.bfloat16, 4608, False), (torch.bfloat16, 2304, True), (torch.float32, 2304, False),
                                         (torch.float32, 1280, True), (torch.bfloat16, 4608, True), (torch.bfloat16, 1001, True)])
def test_row_sums_lose_what_their_tree_loses(dt, A, branch):
    """One entry that swallows whatever is added to it alone: a row's sum may lose at most 18 half steps (8 adds in a run of columns,
    4 levels over a thread's runs or the row's waves, 6 in a wave), however many columns a thread holds.  The mean is that and
    1 / A and its product: 20.  1/std: half of 18 (the root), 1 / A and the sum with eps (half each), the root, the quotient: 12."""
    from matryoshka_transcoder_amd.engine import _p, _stream
    lib, u = _lib.load(), 2.0 ** -24 * 1.01
    code = _lib.MTC_BF16 if dt == torch.bfloat16 else _lib.MTC_F32
    for kind, small, which, bound in ((_lib.MTC_NORM_RMS, 2.0 ** -12, 1, 12), (_lib.MTC_NORM_LAYER, 2.0 ** -24, 0, 20)):
        x = torch.full((3, A), small, dtype=dt, device=DEV)
        for r, c in enumerate((0, 8, A - 1)):
            x[r, c] = 1.0
        x64 = x.double()
        exact = x64.mean(1) if which == 0 else 1.0 / torch.sqrt((x64 * x64).mean(1) + float(torch.tensor(1e-6, dtype=torch.float32)))
        out, zero = torch.empty_like(x), torch.zeros_like(x)
        stats = torch.empty(3, 4, dtype=torch.float32, device=DEV)
        d = _lib.BlockNormDesc(rows=3, A=A, dtype=code, has_branch=int(branch), residual_scale=1.0, branch_scale=1.0, post_eps=1e-6,
                               pre_eps=1e-6, post_kind=kind if branch else 0, pre_kind=0 if branch else kind, ld_residual=A, ld_branch=A,
                               ld_hidden=A, ld_normed=A)
        _lib.check(lib.mtc_block_norm_fwd(C.byref(d), _p(zero if branch else x), _p(x) if branch else None, None, None, None, None, None,
                                          _p(out) if branch else None, None if branch else _p(out), _p(stats), _stream()))
        got = stats[:, which if branch else 2 + which].double()
        assert bool(((got - exact).abs() <= bound * u * exact).all()), (kind, ((got - exact).abs() / (exact * 2.0 ** -24)).tolist())


@pytest.mark.parametrize("A", [776, 777, 7000])
@pytest.mark.parametrize("mode", ["pre", "pair", "post"])
def test_backward_of_layer_norms_far_from_zero(mode, A):
    """The normalised entries that a layer norm's gradients are made of, rebuilt from the row, its mean and its 1/std: the difference is
    exact for entries near the mean, so only the product rounds (and the difference, further away): two half steps of each entry,
    wherever the row lies.  One row and an incoming gradient of ones: the weight's gradient is these entries."""
    from matryoshka_transcoder_amd.engine import _p, _stream
    lib = _lib.load()
    g = torch.Generator("cpu").manual_seed(21)
    x, y = (_rand(g, 1, A) + 4000.0).to(DEV), _rand(g, 1, A).to(DEV)
    one, w, b = torch.ones(1, A, device=DEV), torch.ones(A, device=DEV), torch.zeros(A, device=DEV)
    branch = {"pre": None, "pair": y, "post": x}[mode]
    res = y if mode == "post" else x
    hidden, normed, stats, dw = torch.empty_like(x), torch.empty_like(x), torch.empty(1, 4, device=DEV), torch.empty_like(w)
    layer, pre, post = _lib.MTC_NORM_LAYER, mode != "post", mode == "post"
    d = _lib.BlockNormDesc(rows=1, A=A, dtype=_lib.MTC_F32, has_branch=int(branch is not None), residual_scale=1.0, branch_scale=1.0,
                           post_eps=1e-5, pre_eps=1e-5, post_kind=layer if post else 0, pre_kind=layer if pre else 0, ld_residual=A,
                           ld_branch=A, ld_hidden=A, ld_normed=A)
    weights = (_p(w if post else None), _p(b if post else None), _p(w if pre else None), _p(b if pre else None))
    _lib.check(lib.mtc_block_norm_fwd(C.byref(d), _p(res), _p(branch), None, *weights, _p(hidden if branch is not None else None),
                                      _p(normed if pre else None), _p(stats), _stream()))
    ws = torch.empty(lib.mtc_block_norm_bwd_workspace_bytes(C.byref(d)), dtype=torch.uint8, device=DEV)
    _lib.check(lib.mtc_block_norm_bwd(C.byref(d), _p(res), _p(branch), None, *weights, _p(stats), _p(one if mode == "post" else None), A,
                                      _p(one if pre else None), A, None, None, None, _p(dw if post else None), None,
                                      _p(dw if pre else None), None, _p(ws), ws.numel(), _stream()))
    v = (x if mode != "pair" else x + y).double()[0]                     # the fp32 sum, as the forward took it
    mu, rstd = (stats[0, 0], stats[0, 1]) if post else (stats[0, 2], stats[0, 3])
    u = (v - mu.double()) * rstd.double()
    bad = (dw.double() - u).abs() > 2 * 2.0 ** -24 * 1.01 * u.abs()
    assert not bool(bad.any()), (int(bad.sum()), float((dw.double() - u).abs().max()))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("A", [8192, 7001])
@pytest.mark.parametrize("kind,gate", [("rms", "none"), ("rms", "channel"), ("rms", "full"), ("layer", "none"), ("layer", "token"),
                                       ("layer", "channel"), ("layer", "full")])
def test_wide_rows_walked_more_than_once(kind, gate, A, dt):
    """Above 6144 columns a row takes the whole workgroup of the backward: several rows each, so that the walk, the alternation
    of the reduction's buffers and the column sums over rows repeat."""
    _check(700 if A == 8192 else 600, A, dt, "pair", kind, kind, gate, rs=0.5 if gate == "token" else 1.0, seed=4)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("mode,post,pre", [("pre", None, "layer"), ("post", "layer", None), ("post", "rms", None), ("pair", None, "layer")])
def test_wide_rows_of_single_modes(mode, post, pre, dt):
    _check(600, 8192, dt, mode, post, pre, "none", seed=5)
    _check(520, 6145, dt, mode, post, pre, "none", seed=6)


@pytest.mark.parametrize("dt", DTYPES)
def test_streaming_with_all_column_sums(dt):
    """Layer norms with biases beyond the Infinity Cache: every weight's and bias's gradient, and the rows as in blocks within it."""
    g = torch.Generator("cpu").manual_seed(28)
    rows, A = (26000, 2304) if dt == torch.bfloat16 else (13000, 2304)
    gen = torch.Generator(DEV).manual_seed(28)
    res, br, dh, dn = (torch.randn(rows, A, generator=gen, device=DEV).to(dt) for _ in range(4))
    post, pre = _norm_module(g, A, "layer", dt), _norm_module(g, A, "layer", dt)
    gate = _gate(g, "channel", rows, A, dt).requires_grad_(True)
    names = ("gate", "post_w", "post_b", "pre_w", "pre_b")
    leaves = [gate, post.weight, post.bias, pre.weight, pre.bias]

    def both(lo, hi):
        r, b = res[lo:hi].detach().requires_grad_(True), br[lo:hi].detach().requires_grad_(True)
        out = residual_block_norm(r, b, post, gate=gate, pre=pre)
        return list(out) + list(torch.autograd.grad(out, [r, b] + leaves, [dh[lo:hi], dn[lo:hi]]))

    whole = both(0, rows)
    for lo in range(0, rows, 4000):
        part = both(lo, min(rows, lo + 4000))
        for a, b in zip(whole[:4], part[:4]):
            assert torch.equal(a[lo:lo + 4000], b)
    want = N.reference(res, br, gate, _spec(post), _spec(pre), 1.0, 1.0, dh, dn)
    for k, v in zip(names, whole[4:]):
        N.compare(k, v, want[k], dt)

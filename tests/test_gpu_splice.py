"""The differentiable reconstruction, and the operators together as they are used: a transcoder spliced into blocks, trained
on a loss behind them with clipped gradients."""
import copy

import pytest
import torch

from matryoshka_transcoder_amd import _lib
from matryoshka_transcoder_amd.block_norm import BlockNorm
from matryoshka_transcoder_amd.grad_clip import clip_grad_norm_
from matryoshka_transcoder_amd.splice import SplicedTranscoder
from matryoshka_transcoder_amd.training import FusedAdam
from matryoshka_transcoder_amd.transcoder import MatryoshkaTranscoder

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _cfg(dt, unit, A=64, **kw):
    return dict(dict(seed=49, prefix_sizes=[32, 96, 224, 512], act_size=A, top_k=8, top_k_aux=32, aux_penalty=1 / 32,
                     n_batches_to_dead=20, l1_coeff=0.0, dtype=dt, device=DEV, input_unit_norm=unit, lr=3e-4, beta1=0.9, beta2=0.99), **kw)


def _transcoder(dt, unit, threshold=0.3, **kw):
    m = MatryoshkaTranscoder(_cfg(dt, unit, **kw))
    g = torch.Generator("cpu").manual_seed(3)
    with torch.no_grad():
        m.b_enc.copy_((torch.randn(512, generator=g) * 0.05).to(dt))
        m.b_dec.copy_((torch.randn(m.target_act_size, generator=g) * 0.1).to(dt))
        m.threshold.fill_(threshold)
    return m.eval()


def _dense(m, x, acts_mask):
    """float64 definition with the given selection; parameters and x are float64 leaves."""
    W_enc, b_enc, W_dec, b_dec = m
    xn, mean, std = x, None, None
    unit, mask = acts_mask
    if unit:
        mean = x.mean(-1, keepdim=True)
        std = (x - mean).std(-1, keepdim=True)
        xn = (x - mean) / (std + 1e-5)
    acts = torch.relu(xn @ W_enc + b_enc) * mask
    out = acts @ W_dec + b_dec
    return out * std + mean if unit else out


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("unit", [False, True])
@pytest.mark.parametrize("train", [False, True])
def test_reconstruct_matches_encode_decode_and_its_gradients(dt, unit, train):
    m = _transcoder(dt, unit)
    g = torch.Generator("cpu").manual_seed(5)
    x = torch.randn(2, 19, 64, generator=g).to(dt).to(DEV)
    with torch.no_grad():
        want = m.decode(m.encode(x).reshape(-1, 512)).reshape(2, 19, 64)
        assert torch.equal(m.reconstruct(x), want)                       # eval mode: bit for bit
    m.train(train)
    thr = m.threshold.clone()
    with torch.no_grad():
        mask = (m.encode(x) > 0).reshape(-1, 512).double()
        m.threshold.copy_(thr)
    cnt = m.num_batches_not_active.clone()
    leaf = x.clone().requires_grad_(True)
    out = m.reconstruct(leaf)
    assert torch.equal(m.num_batches_not_active, cnt)
    G = torch.randn(2, 19, 64, generator=g).to(dt).to(DEV)
    params = [m.W_enc, m.b_enc, m.W_dec, m.b_dec]
    got = torch.autograd.grad(out, [leaf] + params, G)
    ref = [t.detach().double().requires_grad_(True) for t in [x] + params]
    ref_out = _dense(ref[1:], ref[0].reshape(-1, 64), (unit, mask)).reshape(2, 19, 64)
    exact = torch.autograd.grad(ref_out, ref, G.double())
    # fp32: sums of up to 512 terms and two products in a row: 1e-4 of the tensor's size.  bf16: every tensor between the
    # steps is rounded (half a step 2^-9 of its size each, about a dozen of them): 12 * 2^-8 < 5e-2 of the tensor's size.
    rel = 1e-4 if dt == torch.float32 else 5e-2
    for name, a, b in zip(["out", "x", "W_enc", "b_enc", "W_dec", "b_dec"], [out] + list(got), [ref_out] + list(exact)):
        assert a.dtype == dt and a.shape == b.shape
        a, b = a.detach().double(), b.detach()
        assert float((a - b).abs().max()) <= rel * float(b.abs().max()), name


def test_reconstruct_gradient_against_differences():
    """Along random directions, where the selection does not change: (f(x + e v) - f(x - e v)) / 2e in float64 on the
    selected features against <gradient, v>."""
    m = _transcoder(torch.float32, True)
    g = torch.Generator("cpu").manual_seed(6)
    x = torch.randn(7, 64, generator=g).to(DEV).requires_grad_(True)
    G = torch.randn(7, 64, generator=g).to(DEV)
    (dx,) = torch.autograd.grad(m.reconstruct(x), [x], G)
    with torch.no_grad():
        mask = (m.encode(x) > 0).double()
    p = [t.detach().double() for t in (m.W_enc, m.b_enc, m.W_dec, m.b_dec)]
    f = lambda t: float((_dense(p, t, (True, mask)) * G.double()).sum())         # noqa: E731
    for _ in range(3):
        v = torch.randn(7, 64, generator=g).double().to(DEV)
        e = 1e-6
        diff = (f(x.detach().double() + e * v) - f(x.detach().double() - e * v)) / (2 * e)
        dot = float((dx.double() * v).sum())
        assert abs(diff - dot) <= 1e-4 * float((dx.double().abs() * v.abs()).sum())


def test_reconstruct_edges():
    m = _transcoder(torch.float32, False)
    x = torch.randn(5, 64, device=DEV, requires_grad=True)
    m.threshold.fill_(1e9)                                               # nothing selected: the bias, and no gradient but its
    out = m.reconstruct(x)
    assert torch.equal(out, m.b_dec.detach().expand(5, 64))
    grads = torch.autograd.grad(out.sum(), [x, m.W_enc, m.b_enc, m.W_dec, m.b_dec])
    assert all(not bool(t.any()) for t in grads[:4]) and torch.equal(grads[4], torch.full_like(m.b_dec, 5.0))
    assert m.reconstruct(torch.zeros(0, 64, device=DEV)).shape == (0, 64)
    assert m.reconstruct(torch.randn(64, device=DEV)).shape == (64,)     # one token
    m.requires_grad_(False)                                              # frozen transcoder: the gradient passes through
    m.threshold.fill_(0.3)
    x2 = torch.randn(5, 64, device=DEV, requires_grad=True)
    (dx,) = torch.autograd.grad(m.reconstruct(x2).sum(), [x2])
    assert bool(dx.any())
    with pytest.raises(_lib.MtcError, match="width 64"):
        m.reconstruct(torch.randn(5, 32, device=DEV))
    with pytest.raises(_lib.MtcError, match="model dtype"):
        m.reconstruct(torch.randn(5, 64, device=DEV).bfloat16())
    m.active_prefixes = 2
    with pytest.raises(_lib.MtcError, match="active_prefixes"):
        m.reconstruct(x)


def _block(dt, unit, kind, gate, seed, A=64):
    t = _transcoder(dt, unit, A=A)
    g = torch.Generator("cpu").manual_seed(seed)

    def norm():
        n = BlockNorm(A, kind=kind, eps=1e-6, weight_offset=1.0 if kind == "rms" else 0.0, dtype=dt, device=DEV)
        with torch.no_grad():
            for p in n.parameters():
                p.add_((torch.randn(A, generator=g) * 0.2).to(dt).to(DEV))
        return n
    return SplicedTranscoder(t, norm(), norm() if kind == "rms" else None, attn_post=norm() if kind == "rms" else None, gate=gate)


def _norm64(v, n, p):
    c = v - v.mean(-1, keepdim=True) if n.kind == "layer" else v
    u = c / torch.sqrt((c * c).mean(-1, keepdim=True) + n.eps)
    y = u * (n.weight_offset + p["weight"])
    return y + p["bias"] if "bias" in p else y


def _forward64(b, P, h, attn, mask, unit, token_gate):
    """The spliced block in float64 with the selection given; P: {name: float64 leaf}."""
    sub = lambda pre: {k[len(pre) + 1:]: v for k, v in P.items() if k.startswith(pre + ".")}         # noqa: E731
    h = h + (_norm64(attn, b.attn_post, sub("attn_post")) if b.attn_post is not None else attn)
    t = sub("transcoder")
    y = _dense((t["W_enc"], t["b_enc"], t["W_dec"], t["b_dec"]), _norm64(h, b.pre, sub("pre")), (unit, mask))
    y = y if b.post is None else _norm64(y, b.post, sub("post"))
    gate = token_gate if token_gate is not None else P.get("gate", 1.0)
    return h + gate * y


@pytest.mark.parametrize("kind,gate", [("rms", None), ("rms", "channel"), ("layer", "scalar")])
@pytest.mark.parametrize("unit", [False, True])
def test_a_training_step_through_the_splice(kind, gate, unit):
    """Attention's output, residual, norms, transcoder, gate, a loss behind them; gradients of every parameter against float64;
    one clip over all of them; FusedAdam for the transcoder and torch's Adam for the rest."""
    dt = torch.float32
    b = _block(dt, unit, kind, gate, 11)
    g = torch.Generator("cpu").manual_seed(12)
    h, attn = torch.randn(3, 11, 64, generator=g).to(DEV), torch.randn(3, 11, 64, generator=g).to(DEV)
    token_gate = (torch.rand(3, 11, 1, generator=g) > 0.3).float().to(DEV) if gate is None else None
    target = torch.randn(3, 11, 64, generator=g).to(DEV)
    opt_t = FusedAdam(b.transcoder, lr=1e-3)
    rest = [p for n, p in b.named_parameters() if not n.startswith("transcoder.")]
    opt_r = torch.optim.Adam(rest, lr=1e-3)
    for step in range(3):
        # the selection of this step, from the block's own source activation
        with torch.no_grad():
            hid = h + (b.attn_post(attn) if b.attn_post is not None else attn)
            mask = (b.transcoder.encode(b.pre(hid)) > 0).reshape(-1, 512).double()
        lh, la = h.clone().requires_grad_(True), attn.clone().requires_grad_(True)
        out = b(lh, la, token_gate=token_gate)
        loss = ((out - target) ** 2).mean()
        loss.backward()
        P = {n: p.detach().double().requires_grad_(True) for n, p in b.named_parameters()}
        h64, a64 = h.double().requires_grad_(True), attn.double().requires_grad_(True)
        flat = lambda t: None if t is None else t.reshape(-1, t.shape[-1])         # noqa: E731
        out64 = _forward64(b, P, flat(h64), flat(a64), mask, unit, None if token_gate is None else flat(token_gate.double()))
        loss64 = ((out64 - flat(target.double())) ** 2).mean()
        loss64.backward()
        named = {n: p.grad for n, p in b.named_parameters()}
        want = {n: P[n].grad for n in P}
        named.update(h=lh.grad, attn=la.grad)
        want.update(h=h64.grad, attn=a64.grad)
        for n in want:
            scale = float(want[n].abs().max())
            assert float((named[n].double() - want[n]).abs().max()) <= 2e-4 * scale + 1e-12, (step, n)
        total = float(torch.sqrt(sum((p.grad ** 2).sum() for p in P.values())))
        before = {n: p.grad.clone() for n, p in b.named_parameters()}
        norm = clip_grad_norm_(b.parameters(), 0.5 * total)
        assert abs(float(norm) - total) <= 2e-4 * total
        for n, p in b.named_parameters():
            assert torch.allclose(p.grad, before[n] * (0.5 * total / (float(norm) + 1e-6)), rtol=1e-6, atol=0)
        opt_t.step(project=True)
        opt_r.step()
        opt_t.zero_grad()
        opt_r.zero_grad()
    if token_gate is not None:                                           # tokens kept out of the splice pass through unchanged
        with torch.no_grad():
            out = b(h, attn, token_gate=token_gate)
            hid = h + (b.attn_post(attn) if b.attn_post is not None else attn)
        off = (token_gate == 0).squeeze(-1)
        assert float((out[off] - hid[off]).abs().max()) <= 1e-6 * float(hid.abs().max())


def test_single_tokens_equal_the_prompt():
    """Serving: the tokens of a prompt one by one give the rows of the whole prompt (eval mode, bf16)."""
    b = _block(torch.bfloat16, True, "rms", "channel", 13)
    h = torch.randn(1, 9, 64, device=DEV).bfloat16()
    a = torch.randn(1, 9, 64, device=DEV).bfloat16()
    with torch.no_grad():
        whole = b(h, a)
        for i in range(9):
            assert torch.equal(b(h[:, i:i + 1], a[:, i:i + 1]), whole[:, i:i + 1])


def test_splice_refusals():
    t = _transcoder(torch.float32, False)
    n = BlockNorm(64, device=DEV)
    with pytest.raises(_lib.MtcError, match="width 32"):
        SplicedTranscoder(t, BlockNorm(32, device=DEV))
    with pytest.raises(_lib.MtcError, match="gate must be"):
        SplicedTranscoder(t, n, gate="row")
    with pytest.raises(_lib.MtcError, match="in front"):
        SplicedTranscoder(t, None)
    with pytest.raises(_lib.MtcError, match="differ"):
        SplicedTranscoder(MatryoshkaTranscoder(_cfg(torch.float32, False, target_act_size=32)), n)
    x = torch.randn(2, 64, device=DEV)
    with pytest.raises(_lib.MtcError, match="either"):
        SplicedTranscoder(t, n, gate="scalar")(x, token_gate=torch.ones(2, 1, device=DEV))
    with pytest.raises(_lib.MtcError, match="attn_out"):
        SplicedTranscoder(t, n, attn_post=copy.deepcopy(n))(x)


def test_store_harvests_through_the_norm():
    """cfg["source_norm"]: the store's source rows are the norm of the harvested residual rows, pairs stay together."""
    from matryoshka_transcoder_amd.activation_store import TensorPairSource, TranscoderActivationsStore
    n = BlockNorm(64, kind="rms", weight_offset=1.0, dtype=torch.bfloat16, device=DEV)
    res, tgt = torch.randn(48, 64, device=DEV).bfloat16(), torch.arange(48, device=DEV).bfloat16()[:, None].expand(48, 64).contiguous()
    cfg = dict(_cfg(torch.bfloat16, False), batch_size=16, num_batches_in_buffer=1, source_norm=n)
    store = TranscoderActivationsStore(None, cfg, source=TensorPairSource([(res, tgt)]))
    with torch.no_grad():
        want = n(res)
    for _ in range(3):
        s, t = store.next_batch()
        assert torch.equal(s, want[t[:, 0].long()])


@pytest.mark.parametrize("train", [True, False])
def test_two_reconstructions_before_the_backward(train):
    """Gradient accumulation and a block used twice: each call keeps its own selection."""
    m = _transcoder(torch.float32, False).train(train)
    if not train:
        m.threshold.fill_(0.3)
    xs = [torch.randn(n, 64, generator=torch.Generator("cpu").manual_seed(n)).to(DEV).requires_grad_(True) for n in (9, 30)]
    ds = [torch.randn(n, 64, generator=torch.Generator("cpu").manual_seed(n + 1)).to(DEV) for n in (9, 30)]
    leaves = [m.W_enc, m.b_enc, m.W_dec, m.b_dec]
    outs = [m.reconstruct(x) for x in xs]
    both = torch.autograd.grad(outs, xs + leaves, ds, retain_graph=True)
    again = torch.autograd.grad(outs, xs + leaves, ds)                # the graph kept: the same bits
    alone = [torch.autograd.grad(m.reconstruct(x), [x] + leaves, d) for x, d in zip(xs, ds)]
    for a, b in zip(both, again):
        assert torch.equal(a, b)
    assert torch.equal(both[0], alone[0][0]) and torch.equal(both[1], alone[1][0])
    for got, a, b in zip(both[2:], alone[0][1:], alone[1][1:]):
        # one fp32 sum of the same two gradients, in either order
        assert torch.equal(got, a + b)


@pytest.mark.parametrize("train", [True, False])
def test_recording_into_a_graph_is_refused(train):
    """Forward and backward, before anything is launched; afterwards the same calls work as before."""
    m = _transcoder(torch.float32, True).train(train)
    x = torch.randn(5, 64, generator=torch.Generator("cpu").manual_seed(8)).to(DEV).requires_grad_(True)
    b = SplicedTranscoder(m, BlockNorm(64, device=DEV))
    with torch.no_grad():
        want = m.reconstruct(x).clone()
    for call in (m.reconstruct, b):
        with pytest.raises(_lib.MtcError, match="recorded into a HIP graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()), torch.no_grad():
                call(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = m.reconstruct(x)
        g = torch.ones_like(out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    with pytest.raises(_lib.MtcError, match="recorded into a HIP graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            torch.autograd.grad(out, [x], g)
    with torch.no_grad():
        assert torch.equal(m.reconstruct(x), want)


@pytest.mark.parametrize("how", ["step", "step_project", "train_step", "unit_norm"])
def test_a_backward_after_the_parameters_moved_is_refused(how):
    """A graph made before an update must not take the new weights for the old ones (torch's own in-place check)."""
    m = _transcoder(torch.float32, False).train()
    opt = FusedAdam(m, lr=1e-3)
    x = torch.randn(16, 64, generator=torch.Generator("cpu").manual_seed(9)).to(DEV)
    m.reconstruct(x).sum().backward()                                    # gradients for the update
    out = m.reconstruct(x)
    if how == "unit_norm":
        m.make_decoder_weights_and_grad_unit_norm()
    elif how == "train_step":
        opt.train_step(x, x)
    else:
        opt.step(project=how == "step_project")
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    opt.zero_grad()
    m.reconstruct(x).sum().backward()                                    # the next forward and backward are as ever
    assert m.W_dec.grad is not None


def test_the_optimizer_s_limit_is_the_transcoder_s_alone():
    """FusedAdam(max_grad_norm) in a spliced block: the norms and the gate are not in its norm and stay as they are."""
    from matryoshka_transcoder_amd.grad_clip import global_norm
    b = _block(torch.float32, False, "rms", "channel", 31)
    opt = FusedAdam(b.transcoder, max_grad_norm=1e-3)
    x, a = (torch.randn(16, 64, generator=torch.Generator("cpu").manual_seed(s)).to(DEV) for s in (32, 33))
    b(x, a).square().mean().backward()
    own = global_norm([p.grad for p in b.transcoder.parameters()])
    every = global_norm([p.grad for p in b.parameters() if p.grad is not None])
    rest = {n: (p.detach().clone(), p.grad.clone()) for n, p in b.named_parameters() if not n.startswith("transcoder.")}
    opt.step(project=True)
    assert torch.equal(opt.last_grad_norm, own) and float(every) > float(own) > 1e-3
    for n, p in b.named_parameters():
        if n in rest:
            assert torch.equal(p, rest[n][0]) and torch.equal(p.grad, rest[n][1])

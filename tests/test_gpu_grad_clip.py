"""Gradient norm and clipping on the GPU against float64, and inside the optimizer.

Tolerances: the sum is fp64 (an error below 1e-11), so the norm is off by its rounding to fp32, half a step: 2^-24.  The
coefficient adds the rounding of norm + 1e-6 and of the quotient, the product one more in fp32 and one in the dtype:
half a step of the dtype + 5 * 2^-24."""
import math
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from matryoshka_transcoder_amd import _lib
from matryoshka_transcoder_amd.grad_clip import (clip_by_global_norm_, clip_grad_norm_, coef_of_power_sum, global_norm, norm_and_coef,
                                                 power_sum)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = math.inf


def _norm64(ts, p):
    d = [t.detach().double() for t in ts if t.numel()]
    if not d:
        return 0.0
    if p == INF:
        return float(torch.stack([t.abs().max() for t in d]).max())
    total = float(sum(t.abs().pow(p).sum() for t in d))
    return total ** (1.0 / p)


def _close(got, want, rel):
    return got == want or abs(got - want) <= rel * abs(want)


def _check(ts, max_norm, p, out=None):
    before = [t.clone() for t in ts]
    want = _norm64(ts, p)
    got = clip_by_global_norm_(ts, max_norm, p, out=out)
    assert got.dtype == torch.float32 and got.dim() == 0 and got.is_cuda
    assert _close(float(got), want, 2 ** -24 * 1.01), (float(got), want)
    assert _close(float(global_norm(before, p)), want, 2 ** -24 * 1.01)
    coef = min(1.0, max_norm / (want + 1e-6))
    for b, t, o in zip(before, ts, out if out is not None else ts):
        if out is not None:
            assert torch.equal(t, b)
        exact = coef * b.double()
        allowed = (torch.finfo(t.dtype).eps / 2 + 5 * 2.0 ** -24) * exact.abs() + 1e-44
        assert bool(((o.double() - exact).abs() <= allowed).all())
        if coef == 1.0:
            assert torch.equal(o, b)
    return want


def _list(g, sizes, dts):
    return [(torch.randn(s, generator=g) * 0.1).to(dt).to(DEV) for s, dt in zip(sizes, dts)]


SIZES = [(1,), (7,), (8,), (4096,), (16384,), (16385,), (100003,), (64, 33), (3, 5, 7), (0,), (2304, 40)]


@pytest.mark.parametrize("p", [1.0, 2.0, INF])
@pytest.mark.parametrize("dts", ["bf16", "fp32", "mixed"])
@pytest.mark.parametrize("max_norm", [0.05, 1e9, 0.0])
def test_sizes(p, dts, max_norm):
    g = torch.Generator("cpu").manual_seed(1)
    b, f = torch.bfloat16, torch.float32
    kinds = {"bf16": [b] * len(SIZES), "fp32": [f] * len(SIZES), "mixed": [b, f] * len(SIZES)}[dts]
    _check(_list(g, SIZES, kinds), max_norm, p)
    ts = _list(g, SIZES, kinds)
    _check(ts, max_norm, p, out=[torch.full_like(t, 3.0) for t in ts])
    for s, dt in zip(SIZES, kinds):
        _check(_list(g, [s], [dt]), max_norm, p)


@pytest.mark.parametrize("p", [1.0, 2.0, INF])
def test_many_tensors(p):
    """More tensors than one launch takes, empty ones among them."""
    g = torch.Generator("cpu").manual_seed(2)
    sizes = [((i * 37) % 600,) for i in range(700)]
    _check(_list(g, sizes, [torch.bfloat16, torch.float32] * 350), 0.5, p)
    _check(_list(g, [(0,)] * 3, [torch.float32] * 3), 0.5, p)
    _check(_list(g, [(1,)] * 129, [torch.float32] * 129), 0.5, p)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_layouts(dt):
    """Transposed views, odd base addresses, gaps, permuted and broadcast inputs."""
    g = torch.Generator("cpu").manual_seed(3)

    def views():
        base = (torch.randn(40, 70, generator=g) * 0.1).to(dt).to(DEV)
        flat = (torch.randn(30001, generator=g) * 0.1).to(dt).to(DEV)
        cube = (torch.randn(4, 6, 10, generator=g) * 0.1).to(dt).to(DEV)
        return [base.t(), flat[1:], flat.clone()[1:16385], cube.permute(2, 0, 1), base.clone()[:, 3:40], base.clone()[::2],
                cube.clone()[..., ::3]]

    for i in range(7):
        _check([views()[i]], 0.5, 2.0)
    _check(views(), 0.5, 2.0)
    ts = views()
    _check(ts, 0.5, 2.0, out=[torch.empty(t.shape, dtype=dt, device=DEV) for t in ts])         # other layouts than the inputs'
    wide = torch.full((40, 70), 2.0, dtype=dt, device=DEV)
    clip_by_global_norm_([wide[:, 10:20]], 1.0)
    assert bool((wide[:, :10] == 2.0).all()) and bool((wide[:, 20:] == 2.0).all()) and bool((wide[:, 10:20] < 2.0).all())
    row = torch.randn(1, 50, generator=g).to(dt).to(DEV)
    assert _close(float(global_norm([row.expand(9, 50)])), 3.0 * _norm64([row], 2), 1e-6)      # broadcast: each copy counts
    with pytest.raises(_lib.MtcError, match="expanded"):
        clip_by_global_norm_([row.expand(9, 50)], 1.0)
    assert _close(float(global_norm([row, row], 1.0)), 2.0 * _norm64([row], 1), 1e-6)          # twice in a norm: counts twice
    with pytest.raises(_lib.MtcError, match="shares memory"):
        clip_by_global_norm_([row, row], 1.0)


def test_neighbours_untouched():
    """Clipping a slice of a buffer leaves the elements before and behind it."""
    for dt in (torch.bfloat16, torch.float32):
        for lo, hi in ((8, 16392), (1, 16386), (3, 10), (16, 17)):
            buf = torch.ones(40000, dtype=dt, device=DEV)
            clip_by_global_norm_([buf[lo:hi]], 1e-3)
            assert bool((buf[:lo] == 1).all()) and bool((buf[hi:] == 1).all()) and bool((buf[lo:hi] < 1).all())


def test_values_at_the_ends_of_the_range():
    big = torch.full((1000,), 3e38, device=DEV)                        # squares far beyond fp32
    assert float(global_norm([big])) == INF                            # sqrt(1000) * 3e38 is beyond fp32 itself
    big = torch.full((4,), 1e38, device=DEV)
    assert _close(float(global_norm([big])), 2e38, 1e-6)
    assert _close(float(global_norm([torch.full((10 ** 6,), 1e-30, device=DEV)])), 1e-27, 1e-6)
    _check([torch.full((64,), 1e30, device=DEV), torch.full((64,), 1e-30, device=DEV)], 1.0, 2.0)
    z = torch.zeros(100, device=DEV)
    assert float(clip_by_global_norm_([z], 1.0)) == 0.0 and not bool(z.any())


@pytest.mark.parametrize("p", [1.0, 2.0, INF])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_non_finite(p, dt):
    """As torch.nn.utils.clip_grad_norm_ does: NaN spreads to all, an infinity zeroes the finite ones."""
    for bad in (float("nan"), INF, -INF):
        ts = [torch.ones(5000, dtype=dt, device=DEV), torch.ones(33, dtype=dt, device=DEV)]
        ts[1][7] = bad
        ref = [torch.nn.Parameter(t.float().clone()) for t in ts]
        for r, t in zip(ref, ts):
            r.grad = t.float().clone()
        want = torch.nn.utils.clip_grad_norm_(ref, 1.0, norm_type=p)
        with pytest.raises(RuntimeError, match="non-finite"):
            clip_by_global_norm_(ts, 1.0, p, error_if_nonfinite=True)
        assert bool((ts[0] == 1).all())
        got = clip_by_global_norm_(ts, 1.0, p)
        assert str(float(got)) == str(float(want))
        for r, t in zip(ref, ts):
            assert torch.equal(torch.isnan(r.grad), torch.isnan(t)) and torch.equal(torch.nan_to_num(r.grad), torch.nan_to_num(t.float()))


@pytest.mark.parametrize("mb", [100, 130, 300, 600])
def test_large_lists(mb):
    """Either side of the sizes at which the launches change: whole values, in place and into outputs, and a limit that is
    not reached."""
    n = mb * 250_000                                                   # fp32 + bf16 tensors of together mb MB
    g = torch.Generator(DEV).manual_seed(mb)
    ts = [torch.randn(n // 2 + 5, generator=g, device=DEV), torch.randn(n - 3, generator=g, device=DEV).bfloat16(), torch.ones(3, device=DEV)]
    _check(ts, 1e9, 2.0)
    _check(ts, 10.0, 2.0, out=[torch.empty_like(t) for t in ts])
    _check(ts, 10.0, 2.0)


def test_offsets_beyond_32_bits():
    n = (1 << 31) + 16400
    t = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    t[-1], t[1 << 31], t[3] = 3.0, 4.0, 12.0
    assert float(global_norm([t])) == 13.0 and float(global_norm([t], INF)) == 12.0
    assert float(clip_by_global_norm_([t], 6.5)) == 13.0
    assert (float(t[-1]), float(t[1 << 31]), float(t[3])) == (1.5, 2.0, 6.0)
    del t


def test_same_bits_twice_and_on_another_stream():
    g = torch.Generator("cpu").manual_seed(4)
    ts = _list(g, [(1000003,), (777,), (512, 300)], [torch.bfloat16, torch.float32, torch.bfloat16])
    outs = [[torch.empty_like(t) for t in ts] for _ in range(2)]
    a = clip_by_global_norm_(ts, 0.7, out=outs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = clip_by_global_norm_(ts, 0.7, out=outs[1])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(*outs))


def test_captured_and_replayed():
    g = torch.Generator("cpu").manual_seed(5)
    sizes, dts = [(30000,), (129, 65), (5,)], [torch.bfloat16, torch.float32, torch.float32]
    ts = _list(g, sizes, dts)
    clip_by_global_norm_([t.clone() for t in ts], 0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_by_global_norm_(ts, 0.5)
    for i in range(4):
        new = _list(g, sizes, dts)
        if i == 2:
            new = [t * 1e-4 for t in new]                              # within the limit: left alone
        for t, x in zip(ts, new):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = clip_by_global_norm_(new, 0.5)
        assert torch.equal(norm, want) and all(torch.equal(t, x) for t, x in zip(ts, new))


def test_clipping_a_saved_tensor_is_noticed():
    """A tensor that autograd saved and that is clipped afterwards: its version moves, so the backward refuses."""
    a, b = torch.ones(8, device=DEV, requires_grad=True), torch.full((8,), 2.0, device=DEV)
    c = (a * b).sum()
    clip_by_global_norm_([b], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        c.backward()


def test_parameters():
    ps = [torch.nn.Parameter(torch.randn(100, device=DEV)) for _ in range(3)]
    ps[0].grad, ps[2].grad = torch.randn(100, device=DEV), torch.randn(100, device=DEV)
    ref = [p.grad.clone() for p in (ps[0], ps[2])]
    want = _norm64(ref, 2)
    assert _close(float(clip_grad_norm_(ps, 2.0)), want, 1e-6) and ps[1].grad is None
    for p, r in zip((ps[0], ps[2]), ref):
        assert torch.allclose(p.grad, r * (2.0 / (want + 1e-6)), rtol=1e-6, atol=0)
    assert _close(float(clip_grad_norm_(ps[0], 1e9)), _norm64([ps[0].grad], 2), 1e-6)


def test_coefficients():
    t = torch.full((16,), 2.0, device=DEV)
    nc = norm_and_coef([t], 4.0)
    assert nc.tolist() == [8.0, float(torch.tensor(4.0) / (torch.tensor(8.0) + 1e-6))]
    assert torch.equal(nc, coef_of_power_sum(power_sum([t]), 4.0)) and float(power_sum([t])) == 64.0
    assert norm_and_coef([t], INF)[1].item() == 1.0 and norm_and_coef([t], 0.0)[1].item() == 0.0
    assert torch.equal(norm_and_coef([t], 1.0, INF), coef_of_power_sum(power_sum([t], INF), 1.0, INF))
    with pytest.raises(_lib.MtcError, match="float64"):
        coef_of_power_sum(torch.ones((), device=DEV), 1.0)
    with pytest.raises(_lib.MtcError, match="no gradients"):
        power_sum([])


def test_refusals_on_the_gpu():
    t = torch.ones(8, device=DEV)
    with pytest.raises(_lib.MtcError, match="float32 or bfloat16"):
        global_norm([t.half()])
    with pytest.raises(_lib.MtcError, match="no CPU fallback"):
        global_norm([t, torch.ones(8)])
    with pytest.raises(_lib.MtcError, match="outputs"):
        clip_by_global_norm_([t], 1.0, out=[])
    with pytest.raises(_lib.MtcError, match="output 0"):
        clip_by_global_norm_([t], 1.0, out=[torch.ones(9, device=DEV)])
    with pytest.raises(_lib.MtcError, match="output 0"):
        clip_by_global_norm_([t], 1.0, out=[t.bfloat16()])
    with pytest.raises(_lib.MtcError, match="none to clip"):
        clip_by_global_norm_([], 1.0, out=[t])
    with pytest.raises(_lib.MtcError, match="shares memory"):
        clip_by_global_norm_([t[:4], t[4:]], 1.0, out=[t[4:], t[:4]])
    with pytest.raises(_lib.MtcError, match="dense"):
        global_norm([torch.eye(4, device=DEV).to_sparse()])


def test_outputs_that_overlap_through_a_copy_are_refused():
    """Outputs of another layout are written by a copy behind the kernel: also those must not share memory."""
    t = [torch.randn(4, 6, device=DEV) for _ in range(2)]
    buf = torch.zeros(4, 24, device=DEV)
    with pytest.raises(_lib.MtcError, match="span the same memory"):
        clip_by_global_norm_(t, 1.0, out=[buf[:, 0:12:2], buf[:, 2:14:2]])
    with pytest.raises(_lib.MtcError, match="span the same memory"):
        clip_by_global_norm_(t, 1.0, out=[buf[:, :6], buf.view(-1)[:24].view(4, 6)])
    assert not bool(buf.any())
    own = torch.zeros(8, 24, device=DEV)                             # rows with gaps, one block behind the other: apart
    n = clip_by_global_norm_(t, 1e9, out=[own[:4, 2:8], own[4:, 2:8]])
    assert torch.equal(own[:4, 2:8], t[0]) and torch.equal(own[4:, 2:8], t[1]) and float(n) > 0


# ------------------------------------------------------------------------------------------------ in the optimizer
def _cfg(dt, unit=True, **kw):
    return dict(dict(seed=49, prefix_sizes=[128, 384, 896, 2048], act_size=256, top_k=16, top_k_aux=64, aux_penalty=1 / 32,
                     n_batches_to_dead=20, l1_coeff=0.0, dtype=dt, device=DEV, input_unit_norm=unit, lr=3e-4, beta1=0.9,
                     beta2=0.99), **kw)


def _batch(i, dt, B=192):
    g = torch.Generator("cpu").manual_seed(1000 + i)
    return torch.randn(B, 256, generator=g).to(dt).to(DEV), torch.randn(B, 256, generator=g).to(dt).to(DEV)


def _params(m):
    return {k: v.detach().clone() for k, v in m.state_dict().items()}


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("project", [True, False])
def test_step_equals_clipping_first(dt, project):
    """FusedAdam(max_grad_norm) = clip_grad_norm_ on the .grad tensors, then FusedAdam: the same bits, for a limit that
    clips and for one that does not."""
    from matryoshka_transcoder_amd.training import FusedAdam
    from matryoshka_transcoder_amd.transcoder import MatryoshkaTranscoder
    for limit in (1e-3, 1e9):
        a, b = MatryoshkaTranscoder(_cfg(dt)), MatryoshkaTranscoder(_cfg(dt))
        oa, ob = FusedAdam(a, max_grad_norm=limit), FusedAdam(b)
        for i in range(3):
            x, y = _batch(i, dt)
            a(x, y)["loss"].backward()
            b(x, y)["loss"].backward()
            grads = [p.grad.clone() for p in a.parameters()]
            if not project:
                a.make_decoder_weights_and_grad_unit_norm()
                b.make_decoder_weights_and_grad_unit_norm()
                grads = [p.grad.clone() for p in a.parameters()]
            norm = clip_grad_norm_(b.parameters(), limit)
            oa.step(project=project)
            ob.step(project=project)
            assert torch.equal(oa.last_grad_norm, norm) and (float(norm) > limit) == (limit < 1)
            for p, g0 in zip(a.parameters(), grads):
                assert torch.equal(p.grad, g0)                         # the coefficient is applied on the way
            oa.zero_grad()
            ob.zero_grad()
        for k, v in _params(a).items():
            assert torch.equal(v, b.state_dict()[k]), k
        for p, q in zip(a.parameters(), b.parameters()):
            for s in ("exp_avg", "exp_avg_sq"):
                assert torch.equal(oa.state[p][s], ob.state[q][s])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("aux", [False, True])
def test_train_step_equals_the_loop(dt, aux):
    """train_step with a limit = forward, backward, clip, step, bit for bit; an inactive limit = the same without one (to within
    the unclipped fused step's own rule: the same bits)."""
    from matryoshka_transcoder_amd.training import FusedAdam
    from matryoshka_transcoder_amd.transcoder import MatryoshkaTranscoder
    kw = dict(n_batches_to_dead=2) if aux else {}
    models = [MatryoshkaTranscoder(_cfg(dt, **kw)) for _ in range(3)]
    opts = [FusedAdam(models[0], max_grad_norm=1e-3), FusedAdam(models[1]), FusedAdam(models[2], max_grad_norm=1e9)]
    plain = MatryoshkaTranscoder(_cfg(dt, **kw))
    oplain = FusedAdam(plain)
    for i in range(5):
        x, y = _batch(i, dt)
        l0 = opts[0].train_step(x, y)["loss"]
        out = models[1](x, y)
        out["loss"].backward()
        clip_grad_norm_(models[1].parameters(), 1e-3)
        opts[1].step(project=True)
        opts[1].zero_grad()
        assert torch.equal(l0, out["loss"].detach())
        opts[2].train_step(x, y)
        oplain.train_step(x, y)
    for k, v in _params(models[0]).items():
        assert torch.equal(v, models[1].state_dict()[k]), k
    if not aux:
        for k, v in _params(models[2]).items():
            assert torch.equal(v, plain.state_dict()[k]), k
    assert all(p.grad is None for p in models[0].parameters())


def test_train_transcoder_clips_when_asked(tmp_path):
    import json
    from matryoshka_transcoder_amd.activation_store import TranscoderActivationsStore
    from matryoshka_transcoder_amd.training import train_transcoder
    from matryoshka_transcoder_amd.transcoder import MatryoshkaTranscoder
    logs = {}
    for clip in (False, True):
        cfg = _cfg(torch.float32, dict_size=2048, batch_size=64, num_tokens=64 * 4, model_batch_size=16, seq_len=16, max_grad_norm=1e-3,
                   log_freq=1, perf_log_freq=1000, checkpoint_freq=1000, results_root=str(tmp_path / str(clip)), model_name="gpt2-small", layer=8)
        if clip:
            cfg["clip_gradients"] = True
        m = MatryoshkaTranscoder(cfg)
        d = train_transcoder(m, TranscoderActivationsStore(None, cfg), None, cfg)
        recs = [json.loads(x) for x in open(d / "train_log.jsonl")]
        logs[clip] = [r for r in recs if "loss" in r]
    assert all("grad_norm" not in r for r in logs[False]) and all(r["grad_norm"] > 1e-3 for r in logs[True])
    assert logs[False][0]["loss"] == logs[True][0]["loss"]


def test_optimizer_refuses_a_bad_limit():
    from matryoshka_transcoder_amd.training import FusedAdam
    from matryoshka_transcoder_amd.transcoder import MatryoshkaTranscoder
    m = MatryoshkaTranscoder(_cfg(torch.float32))
    for bad in (-1.0, float("nan")):
        with pytest.raises(_lib.MtcError, match="max_grad_norm"):
            FusedAdam(m, max_grad_norm=bad)
    o = FusedAdam(m, max_grad_norm=1.0)
    o.step(project=True)                                               # no gradients yet: nothing happens
    assert o.last_grad_norm is None


def _sharded_worker(rank, world, port, ret):
    try:
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
        torch.cuda.set_device(0)
        dist.init_process_group("gloo", rank=rank, world_size=world)
        from matryoshka_transcoder_amd.sharded import ShardedFusedAdam, ShardedMatryoshkaTranscoder
        m = ShardedMatryoshkaTranscoder(_cfg(torch.float32))
        o = ShardedFusedAdam(m, max_grad_norm=0.01)
        norms = []
        for i in range(3):
            o.train_step(*_batch(i, torch.float32))
            norms.append(float(o.last_grad_norm))
        sd = {k: v.cpu() for k, v in m.state_dict().items()}
        ret[f"norms{rank}"] = norms
        if rank == 0:
            ret["sd"] = sd
        ret[f"ok{rank}"] = True
    finally:
        if dist.is_initialized():
            dist.destroy_process_group()


@pytest.mark.parametrize("world", [1, 2])
def test_sharded_norm_is_the_whole_dictionary_s(world):
    from matryoshka_transcoder_amd.training import FusedAdam
    from matryoshka_transcoder_amd.transcoder import MatryoshkaTranscoder
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    with mp.Manager() as mgr:
        ret = mgr.dict()
        mp.spawn(_sharded_worker, args=(world, port, ret), nprocs=world, join=True)
        ret = dict(ret)
    m = MatryoshkaTranscoder(_cfg(torch.float32))
    o = FusedAdam(m, max_grad_norm=0.01)
    for i in range(3):
        o.train_step(*_batch(i, torch.float32))
        assert all(ret[f"norms{r}"][i] == ret["norms0"][i] for r in range(world))          # one coefficient on every rank
        assert _close(ret["norms0"][i], float(o.last_grad_norm), 1e-4) and float(o.last_grad_norm) > 0.01
    for k, v in ret["sd"].items():
        assert float((v - m.state_dict()[k].cpu()).abs().max()) <= 1e-2 * 3e-4 * 3, k       # the fp32 bar of the sharded step


def test_a_step_without_gradients_leaves_no_old_norm():
    """last_grad_norm is the last step's: nothing was clipped in a step that found no gradients."""
    from matryoshka_transcoder_amd.training import FusedAdam
    from matryoshka_transcoder_amd.transcoder import MatryoshkaTranscoder
    cfg = dict(seed=49, prefix_sizes=[32, 128], act_size=64, top_k=8, top_k_aux=32, aux_penalty=1 / 32, n_batches_to_dead=20, l1_coeff=0.0,
               dtype=torch.float32, device=DEV, input_unit_norm=False, lr=3e-4, beta1=0.9, beta2=0.99)
    tc = MatryoshkaTranscoder(cfg)
    opt = FusedAdam(tc, lr=1e-3, max_grad_norm=0.5)
    for p in tc.parameters():
        p.grad = torch.ones_like(p)
    opt.step()
    assert float(opt.last_grad_norm) > 0
    opt.zero_grad()
    opt.step()
    assert opt.last_grad_norm is None

"""The dense layers over the library's calls: k_dense.gated_ffn and Linear8, the unquantised shared expert of a checkpoint
through exl3_loader and k_overlap.SharedOverlap, and a decode step of all of them (routed experts, shared expert, output head,
drawn token), eager and captured."""
import math

import numpy as np
import pytest

import ckpt_synth
import dense_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
H, I, E, KS = 512, 256, 5, (3, 3, 3)
DENSE = {5: (F16, 384), 6: (BF16, 200)}     # layer: type and intermediate size of its shared expert


@pytest.fixture(scope="module")
def loaded(gpu, tmp_path_factory):
    import exl3_loader
    import k_overlap
    tmp = tmp_path_factory.mktemp("dense_ckpt")
    paths, weights = [], {}
    for L, (dt, Is) in DENSE.items():
        paths += ckpt_synth.write(tmp, [L], E=E, H=H, I=I, Ks_by_layer={L: KS}, shared=False)
        weights[L] = ckpt_synth.write_dense(tmp, L, H, Is, dt)
        paths.append(str(tmp / f"dense-{L:05d}.safetensors"))
    so = k_overlap.SharedOverlap(0)
    return dict(so=so, weights=weights, res=exl3_loader.load(paths, gpu, shared=so))


def _picks(rng, M):
    x = torch.from_numpy((rng.standard_normal((M, H)) * 0.5).astype(np.float16)).cuda()
    sel = torch.from_numpy(np.stack([rng.permutation(E)[:3] for _ in range(M)]).astype(np.int64)).cuda()
    return x, sel, torch.from_numpy(rng.random((M, 3)).astype(np.float32)).cuda()


@pytest.mark.parametrize("L", list(DENSE))
@pytest.mark.parametrize("M", [1, 5, 40])
def test_shared_expert_from_the_checkpoint(gpu, loaded, L, M):
    x, sel, w = _picks(np.random.default_rng(L * 10 + M), M)
    wg, wu, wd = loaded["weights"][L]
    # bf16 weights below 2^-14 are rounded to fp16's step of 2^-24, by at most half of it; the others are exact
    for a, b in zip(loaded["res"][L].dense, (wg, wu, wd)):
        off = (a.cpu().double() - b.double()).abs()
        assert a.dtype == F16 and bool((off <= torch.where(b.double().abs() < 2.0 ** -14, 2.0 ** -25, 0.0)).all())
    routed, both = (torch.empty((M, H), dtype=F32, device="cuda") for _ in range(2))
    gpu.moe_forward(L, x, sel, w, routed)
    before = loaded["so"].summary()
    assert loaded["so"].forward(gpu, L, x, sel, w, both) is both
    after = loaded["so"].summary()
    assert after == dict(before, dense=before["dense"] + 1)
    ref = R.FFN(x, *(t.half().cuda() for t in (wg, wu, wd)), out_dt=F32)
    want = routed.double().cpu() + ref.y
    R.within(both, want, ref.ey + 2.0 ** -24 * (want.abs() + ref.ey), "routed + shared")


def test_a_layer_registered_again(gpu, loaded):
    """The last registration of a layer is the one that runs."""
    import k_overlap
    import synth
    so = k_overlap.SharedOverlap(0)
    x, sel, w = _picks(np.random.default_rng(3), 4)
    shared = synth.SynthLayer(63, 1, H, I, KS)
    routed, a, b = (torch.empty((4, H), dtype=F32, device="cuda") for _ in range(3))
    gpu.moe_forward(5, x, sel, w, routed)
    so.register(5, H, I, shared.Ks, shared.ptr_table, keep=shared)
    so.forward(gpu, 5, x, sel, w, a)
    so.register_dense(5, *loaded["res"][5].dense)
    so.forward(gpu, 5, x, sel, w, b)
    assert so.summary()["dense"] == 1 and not torch.equal(a, b)
    so.register(5, H, I, shared.Ks, shared.ptr_table, keep=shared)
    so.forward(gpu, 5, x, sel, w, b)
    assert so.summary()["dense"] == 1 and torch.equal(a, b)


def _block(M, Hd, Id, dt, seed):
    g = torch.Generator()
    g.manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    return ((r(M, Hd)).to(dt).cuda(), (r(Id, Hd) / math.sqrt(Hd)).to(dt).cuda(), (r(Id, Hd) / math.sqrt(Hd)).to(dt).cuda(),
            (r(Hd, Id) / math.sqrt(Id)).to(dt).cuda(), r(M, Hd).to(dt).cuda())


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("shape", [(6, 1), (6,), (2, 3)])
@pytest.mark.parametrize("L", [0.0, 0.75])
def test_gated_ffn_gradients(gpu, dt, shape, L):
    import k_dense
    *ins, dy = _block(6, 264, 200, dt, 4)
    ref = R.FFN(*ins, L)
    for t in ins:
        t.requires_grad_()
    x = ins[0].reshape(*shape, 264)
    y = k_dense.gated_ffn(x, *ins[1:], act_limit=L)
    assert y.shape == x.shape
    R.within(y.detach().reshape(6, 264), ref.y, ref.ey, "y")
    y.backward(dy.reshape(y.shape))
    for t, (v, e), n in zip(ins, ref.backward(dy), ("dx", "dwg", "dwu", "dwd")):
        R.within(t.grad, v, e, n)


def test_gated_ffn_partial_shared_and_broadcast(gpu):
    """Only some inputs with gradients; one weight for gate and up; a broadcast gradient; two uses before one backward."""
    import _native
    import k_dense
    x, wg, wu, wd, dy = _block(9, 136, 72, F16, 7)
    want = R.FFN(x, wg, wg, wd).backward(torch.ones_like(dy))
    w = wg.clone().requires_grad_()
    y = k_dense.gated_ffn(x, w, w, wd)
    y.sum().backward()
    # the sum of two gradients, each rounded, is rounded again
    v, e = want[1][0] + want[2][0], want[1][1] + want[2][1]
    R.within(w.grad, v, e + R.half_step(F16) * (v.abs() + e) + R.tiny(F16), "dwg + dwu")
    assert x.grad is None and wd.grad is None
    a = x.clone().requires_grad_()
    out = k_dense.gated_ffn(a, wg, wu, wd) + k_dense.gated_ffn(a, wu, wg, wd)
    out.backward(dy)
    one = [_native.ffn_backward(dy, x, *_native.ffn_forward(x, p, q, wd, save=True)[1:], p, q, wd, need=(True, False, False, False))[0]
           for p, q in ((wg, wu), (wu, wg))]
    assert torch.equal(a.grad, one[0] + one[1]) or torch.equal(a.grad, one[1] + one[0])
    with torch.no_grad():
        assert not k_dense.gated_ffn(a, wg, wu, wd).requires_grad
    z = torch.empty((0, 136), dtype=F16, device="cuda", requires_grad=True)
    k_dense.gated_ffn(z, w, w, wd).sum().backward()
    assert z.grad.shape == (0, 136)


def test_gated_ffn_refusals(gpu, monkeypatch):
    import k_dense
    x, wg, wu, wd, dy = _block(3, 64, 40, F16, 8)
    x.requires_grad_()
    y = k_dense.gated_ffn(x, wg, wu, wd)
    with pytest.raises(RuntimeError, match="once_differentiable|once differentiable"):
        d, = torch.autograd.grad(y, x, dy.requires_grad_(), create_graph=True)
        d.sum().backward()
    dy = dy.detach()
    for bad in (dict(act_limit=-1.0), dict(act_limit=math.nan)):
        with pytest.raises(RuntimeError, match="act_limit"):
            k_dense.gated_ffn(x, wg, wu, wd, **bad)
    # a gradient that another call changed its input for
    a = x.detach().clone()
    y = k_dense.gated_ffn(a, wg.requires_grad_(), wu, wd)
    a.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)
    # capture: refused with gradients, whichever half it would take; forward without is captured
    y = k_dense.gated_ffn(x, wg, wu, wd)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="stream capture"):
        k_dense.gated_ffn(x, wg, wu, wd)
    with pytest.raises(RuntimeError, match="stream capture"):
        y.backward(dy)


def _head_ref(h, weight, dt_out=F32):
    """Logits of Linear8's definition: weight and tokens quantised per row, their exact product scaled; and bounds."""
    (q, s), (p, t) = R.quant(weight), R.quant(h)
    want = (p.double() @ q.double().t()) * t.double()[:, None] * s.double()[None, :]
    # the sum's conversion, two products and the two scales round in fp32
    return want, want.abs() * (R.half_step(dt_out) + 6 * 2.0 ** -24) + R.tiny(dt_out)


def test_decode_step(gpu, loaded):
    """Routed experts + shared expert -> output head -> drawn token: each part against its definition on the tensors the part
    before made, then the step captured and replayed on new tokens beside eager steps."""
    import _native
    import k_dense
    L, M, V = 5, 4, 4001
    rng = np.random.default_rng(17)
    g = torch.Generator()
    g.manual_seed(17)
    weight = (torch.randn((V, H), generator=g) / math.sqrt(H)).half().cuda()
    head = k_dense.Linear8(weight)
    x, sel, w = _picks(rng, M)
    u = torch.rand(M, generator=g).cuda()
    kw = dict(temperature=torch.full((M,), 0.8, device="cuda"), top_k=torch.full((M,), 50, dtype=torch.int32, device="cuda"),
              top_p=torch.full((M,), 0.9, device="cuda"), min_p=torch.full((M,), 0.02, device="cuda"))

    def step(y):
        loaded["so"].forward(gpu, L, x, sel, w, y)
        h = (x + y).half()
        logits = head(h, dtype=F32)
        return (h, logits) + tuple(_native.sample(logits, u, **kw))

    y = torch.empty((M, H), dtype=F32, device="cuda")
    h, logits, tok, prob = step(y)
    want, bound = _head_ref(h, weight)
    R.within(logits, want, bound, "logits")
    for b, (t, p, m) in enumerate(R.sample(logits, u, **kw)):
        assert m > 2.0 ** -36 and int(tok[b]) == t
        assert abs(float(prob[b]) - p) <= p * 2.0 ** -23 + V * 2.0 ** -42

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(y)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    yg = torch.empty_like(y)
    with torch.cuda.graph(graph):
        outs = step(yg)
    for _ in range(4):
        for t, new in zip((x, sel, w), _picks(rng, M)):
            t.copy_(new)
        u.copy_(torch.rand(M, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = step(y)
        torch.cuda.synchronize()
        assert torch.equal(yg, y)
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_linear8(gpu, dt):
    import k_dense
    g = torch.Generator()
    g.manual_seed(2)
    weight, x = torch.randn((301, 200), generator=g).to(dt).cuda(), torch.randn((2, 3, 200), generator=g).to(dt).cuda()
    lin = k_dense.Linear8(torch.nn.Parameter(weight))
    want, bound = _head_ref(x.reshape(6, 200), weight, dt)
    y = lin(x)
    assert y.shape == (2, 3, 301) and y.dtype == dt
    R.within(y.reshape(6, 301), want, bound)
    out = torch.empty((2, 3, 301), dtype=F32, device="cuda")
    assert lin(x, out=out) is not None
    want, bound = _head_ref(x.reshape(6, 200), weight, F32)
    R.within(out.reshape(6, 301), want, bound)


@pytest.mark.parametrize("limit", [0.0, 0.05])
def test_the_checkpoints_clamp(gpu, loaded, tmp_path, limit):
    """load(act_limit=...) clamps the unquantised shared experts it registers."""
    import exl3_loader
    import k_overlap
    L, M = 7, 9
    paths = ckpt_synth.write(tmp_path, [L], E=E, H=H, I=I, Ks_by_layer={L: KS}, shared=False)
    weights = [t.cuda() for t in ckpt_synth.write_dense(tmp_path, L, H, 384, F16)]
    paths.append(str(tmp_path / f"dense-{L:05d}.safetensors"))
    so = k_overlap.SharedOverlap(0)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="act_limit"):
            exl3_loader.load(paths, gpu, shared=so, act_limit=bad)
    exl3_loader.load(paths, gpu, shared=so, act_limit=limit)
    x, sel, w = _picks(np.random.default_rng(70), M)
    routed, both = (torch.empty((M, H), dtype=F32, device="cuda") for _ in range(2))
    gpu.moe_forward(L, x, sel, w, routed)
    so.forward(gpu, L, x, sel, w, both)
    ref, off = R.FFN(x, *weights, limit, out_dt=F32), R.FFN(x, *weights, out_dt=F32)
    assert limit == 0 or bool(((ref.y - off.y).abs() > ref.ey + off.ey).any())
    want = routed.double().cpu() + ref.y
    R.within(both, want, ref.ey + 2.0 ** -24 * (want.abs() + ref.ey), "routed + shared")

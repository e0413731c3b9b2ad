"""The dense layers without a GPU: which unquantised shared experts exl3_loader.scan finds, and what it,
SharedOverlap.register_dense and k_dense refuse."""
import pytest
import torch

import ckpt_synth

KS = {1: (3, 3, 3)}


def _scan(tmp_path, H, Is, dtype, shared=False):
    import exl3_loader
    paths = ckpt_synth.write(tmp_path, [1], E=2, H=512, I=256, Ks_by_layer=KS, shared=shared)
    ckpt_synth.write_dense(tmp_path, 1, H, Is, dtype)
    return exl3_loader.scan(paths + [str(tmp_path / "dense-00001.safetensors")])[1]


@pytest.mark.parametrize("dtype,found", [(torch.float16, True), (torch.bfloat16, True), (torch.float32, False)])
def test_scan_finds_the_unquantised_shared_expert(tmp_path, dtype, found):
    sp = _scan(tmp_path, 512, 384, dtype)
    assert not sp.has_shared and sorted(sp.dense) == (["down", "gate", "up"] if found else [])


def test_scan_prefers_the_quantised_one(tmp_path):
    sp = _scan(tmp_path, 512, 384, torch.float16, shared=True)
    assert sp.has_shared and not sp.dense


def test_scan_refuses_weights_of_another_hidden_size(tmp_path):
    with pytest.raises(ValueError, match="do not fit hidden 512"):
        _scan(tmp_path, 520, 384, torch.float16)


def test_bf16_weights_past_fp16(tmp_path):
    import exl3_loader
    from safetensors import safe_open
    from safetensors.torch import save_file
    key, path = "a", str(tmp_path / "w.safetensors")
    for vals, ok in (([1.0, 65280.0, 2.0 ** -20], True), ([-65536.0, 0.0], False), ([3e38], False)):
        t = torch.tensor([vals], dtype=torch.bfloat16)
        save_file({key: t}, path)
        sp = exl3_loader.LayerSpec(layer=1, dense={"gate": (path, key)})
        with safe_open(path, framework="pt", device="cpu") as f:
            if ok:
                assert torch.equal(exl3_loader._dense_weight(1, "gate", sp, {path: f}, "cpu").float(), t.float())
            else:
                with pytest.raises(ValueError, match="past fp16"):
                    exl3_loader._dense_weight(1, "gate", sp, {path: f}, "cpu")


def test_register_dense_refusals():
    import k_overlap
    so = object.__new__(k_overlap.SharedOverlap)     # no context: nothing here reaches the device
    so.device, so._dense = torch.device("cpu"), {}
    w = lambda *s, dt=torch.float16: torch.zeros(s, dtype=dt)
    ok = (w(8, 16), w(8, 16), w(16, 8))
    so.register_dense(0, *ok, act_limit=7.0)
    assert so._dense[0][3] == 7.0
    for bad, word in (((w(8, 16), w(9, 16), w(16, 8)), "must be"), ((w(8, 16), w(8, 16), w(8, 16)), "must be"),
                      ((w(128), w(128), w(128)), "must be"), ((w(8, 16, dt=torch.bfloat16),) + ok[1:], "fp16"),
                      ((w(16, 8).t(),) + ok[1:], "contiguous"), ((w(8, 16).to("meta"),) + ok[1:], "on cpu")):
        with pytest.raises(ValueError, match=word):
            so.register_dense(1, *bad)
    for limit in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="act_limit"):
            so.register_dense(1, *ok, act_limit=limit)
    assert list(so._dense) == [0]


def test_layers_refuse_host_tensors_and_shapes():
    import k_dense
    w = lambda *s: torch.zeros(s, dtype=torch.float16)
    for grad in (False, True):
        with pytest.raises(ValueError, match="device"):
            k_dense.gated_ffn(w(2, 16), w(8, 16).requires_grad_(grad), w(8, 16), w(16, 8))
    for bad in (w(8), w(8, 0), torch.zeros((1, 131072), dtype=torch.float16, device="meta"), w(2, 3, 4)):
        with pytest.raises(ValueError, match="Linear8"):
            k_dense.Linear8(bad)
    with pytest.raises(ValueError, match="device"):
        k_dense.Linear8(w(4, 8))


def _plain_calls(monkeypatch):
    """The layers over plain torch operations instead of the device's calls."""
    import _native

    def ffn_forward(x, wg, wu, wd, act_limit=0.0, save=False, **kw):
        with torch.no_grad():
            g, u = x.float() @ wg.float().t(), x.float() @ wu.float().t()
            y = ((torch.sigmoid(g) * g * u) @ wd.float().t()).to(x.dtype)
        return (y, g, u) if save else y

    monkeypatch.setattr(_native, "ffn_forward", ffn_forward)
    monkeypatch.setattr(_native, "quant_i8", lambda w: (torch.zeros(w.shape, dtype=torch.int8), torch.ones(w.shape[0])))
    monkeypatch.setattr(_native, "linear_i8", lambda x, w, s, out=None, dtype=None: x.new_zeros(x.shape[:-1] + w.shape[:1]))


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", [False, True])
def test_gated_ffn_refuses_forward_mode(monkeypatch, which, grad):
    """A tangent that the block would drop without a word is refused, whichever input holds it."""
    import k_dense
    import torch.autograd.forward_ad as fwd
    _plain_calls(monkeypatch)
    w = lambda *s: torch.randn(s).half()
    args = [w(2, 16), w(8, 16), w(8, 16), w(16, 8)]
    if grad:
        args[3 - which].requires_grad_()
    k_dense.gated_ffn(*args)
    with fwd.dual_level():
        k_dense.gated_ffn(*args)     # no tangent: as outside
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            k_dense.gated_ffn(*args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            k_dense.gated_ffn(*args)


def test_linear8_refuses_gradients(monkeypatch):
    """The 8-bit layer has no gradient: an input that asks for one is refused instead of being cut off."""
    import k_dense
    import torch.autograd.forward_ad as fwd
    _plain_calls(monkeypatch)
    head = k_dense.Linear8(torch.randn(4, 8).half().requires_grad_())    # the weight is taken as it stands
    x = torch.randn(2, 8).half()
    assert not head(x).requires_grad
    y = x.clone().requires_grad_()
    for t in (y, y * 2):
        with pytest.raises(RuntimeError, match="Linear8.*gradient"):
            head(t)
        with torch.no_grad():
            assert not head(t).requires_grad
        assert not head(t.detach()).requires_grad
    with torch.inference_mode():
        head(y)
    with fwd.dual_level(), pytest.raises(RuntimeError, match="Linear8.*forward-mode"):
        head(fwd.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="Linear8.*gradient"):
        head(x, out=torch.zeros(2, 4).requires_grad_())


@pytest.mark.parametrize("have", [("gate",), ("gate", "down"), ("up", "down")])
def test_load_refuses_part_of_a_shared_expert(tmp_path, have):
    """One or two of the three unquantised weights: what is asked to load shared experts says what is missing, before anything
    is copied. scan, and load without shared experts, leave it alone."""
    import exl3_loader
    from safetensors import safe_open
    from safetensors.torch import save_file
    paths = ckpt_synth.write(tmp_path, [1], E=2, H=512, I=256, Ks_by_layer=KS, shared=False)
    ckpt_synth.write_dense(tmp_path, 1, 512, 384, torch.float16)
    with safe_open(str(tmp_path / "dense-00001.safetensors"), framework="pt", device="cpu") as f:
        part = {k: f.get_tensor(k) for k in f.keys() if any(f".{p}_proj." in k for p in have)}
    save_file(part, str(tmp_path / "part.safetensors"))
    paths.append(str(tmp_path / "part.safetensors"))
    assert not exl3_loader.scan(paths)[1].dense
    missing = [p for p in exl3_loader.PROJ if p not in have]
    for layers in (None, [1]):
        with pytest.raises(ValueError, match="layer 1.*" + ".*".join(missing)):
            exl3_loader.load(paths, None, layers=layers, shared=object())


def test_load_takes_other_layers_beside_part_of_a_shared_expert(tmp_path):
    """A layer that is not asked for, or whose shared expert is there in quantised form, is no reason to refuse."""
    import exl3_loader
    paths = ckpt_synth.write(tmp_path, [1, 2], E=2, H=512, I=256, Ks_by_layer={1: (3, 3, 3), 2: (3, 3, 3)}, shared=True)
    ckpt_synth.write_dense(tmp_path, 1, 512, 384, torch.float16)
    from safetensors import safe_open
    from safetensors.torch import save_file
    with safe_open(str(tmp_path / "dense-00001.safetensors"), framework="pt", device="cpu") as f:
        key = sorted(f.keys())[0]
        save_file({key: f.get_tensor(key)}, str(tmp_path / "part.safetensors"))
    specs = exl3_loader.scan(paths + [str(tmp_path / "part.safetensors")])
    exl3_loader._check_dense(specs, [1, 2])


def test_a_shared_expert_of_another_width_is_refused_before_the_routed_call():
    import k_overlap

    class Routed:
        def moe_forward(self, *a):
            raise AssertionError("the routed call ran first, and left its output without the shared expert")

    so = object.__new__(k_overlap.SharedOverlap)
    so.device, so._dense = torch.device("cpu"), {}
    w = lambda *s: torch.zeros(s, dtype=torch.float16)
    so.register_dense(0, w(8, 16), w(8, 16), w(16, 8))
    for x in (w(2, 24), w(2, 16).to("meta")):
        with pytest.raises(ValueError, match="layer 0"):
            so.forward(Routed(), 0, x, None, None, torch.zeros(x.shape))

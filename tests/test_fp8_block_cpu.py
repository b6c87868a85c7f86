"""Block-scaled 8-bit operators on the CPU: the format, the eager arithmetic that the GPU kernels are held to,
and what is refused."""
import math

import pytest
import torch

from lset_b200.ops import fp8_block as fb


def _by_hand(block, e5m2):
    """A block's values after the cast, one by one in Python floats (64 bits)."""
    top = max(abs(v) for v in block)
    if not math.isfinite(top) or any(math.isnan(v) for v in block):
        return [math.nan] * len(block)
    fmax, bits, low = (57344.0, 2, -14) if e5m2 else (448.0, 3, -6)
    e = -126
    while top > fmax * 2.0 ** e:
        e += 1
    if top == 0:
        e = 0
    out = []
    for v in block:
        y = v / 2.0 ** e
        step = 2.0 ** (max(math.frexp(y)[1] - 1, low) - bits)
        out.append(round(y / step) * step * 2.0 ** e)     # Python rounds halves to even
    return out


def _same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


SPECIAL = [0.0, 448.0, 449.0, 450.0, -448.0, 1e-30, 2.0 ** -133, 3.3e38, 2.0 ** -126, 57344.0, 57600.0, 1.75, 1.7578125]


@pytest.mark.parametrize("e5m2", [False, True])
@pytest.mark.parametrize("R,C", [(1, 1), (3, 130), (129, 24), (128, 128), (257, 131)])
def test_values_of_every_kind_of_block(R, C, e5m2):
    g = torch.Generator().manual_seed(R * C)
    x = (torch.randn(R, C, generator=g) * torch.exp(4 * torch.randn(R, C, generator=g))).to(torch.bfloat16)
    for i, v in enumerate(SPECIAL):
        x[(i * 5) % R, (i * 37) % C] = v
    if R > 2:
        x[2] = 0
    xl = x.double().tolist()
    rows = torch.tensor([sum((_by_hand(r[c:c + 128], e5m2) for c in range(0, C, 128)), []) for r in xl])
    cols = torch.tensor([sum((_by_hand(r[c:c + 128], e5m2) for c in range(0, R, 128)), [])
                         for r in x.double().t().tolist()])
    q, q_t = fb.quantize_fp8_block(x, e5m2=e5m2, want_t=True)
    assert q.shape == (R, C) and q_t.shape == (C, R)
    assert _same(q.dequantize(), rows.float()) and _same(q_t.dequantize(), cols.float())
    t, t_t = fb.quantize_fp8_block(x, tile=True, e5m2=e5m2, want_t=True)
    tiles = torch.zeros(R, C)
    for r in range(0, R, 128):
        for c in range(0, C, 128):
            part = x[r:r + 128, c:c + 128].double()
            tiles[r:r + 128, c:c + 128] = torch.tensor(_by_hand(part.flatten().tolist(), e5m2)).view(part.shape)
    assert _same(t.dequantize(), tiles) and _same(t_t.dequantize(), tiles.t())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_block_that_is_not_finite_is_nan_and_no_other(bad):
    x = torch.ones(5, 300, dtype=torch.bfloat16)
    x[1, 140] = bad
    q, q_t = fb.quantize_fp8_block(x, want_t=True)
    want = torch.zeros(5, 300, dtype=torch.bool)
    want[1, 128:256] = True
    assert torch.equal(torch.isnan(q.dequantize()), want)
    want = torch.zeros(300, 5, dtype=torch.bool)
    want[140] = True
    assert torch.equal(torch.isnan(q_t.dequantize()), want)
    t, _ = fb.quantize_fp8_block(x, tile=True)
    assert torch.isnan(t.dequantize()[:, 128:256]).all() and not torch.isnan(t.dequantize()[:, :128]).any()


def test_products_and_accumulation():
    torch.manual_seed(1)
    a, _ = fb.quantize_fp8_block(torch.randn(7, 200))
    b, _ = fb.quantize_fp8_block(torch.randn(24, 200), tile=True, e5m2=True)
    ref = a.dequantize().double() @ b.dequantize().double().t()
    bound = 200 * 2.0 ** -23 * (a.dequantize().abs() @ b.dequantize().abs().t())
    c = fb.matmul_fp8_block(a, b, out_dtype=torch.float32)
    assert ((c - ref).abs() <= bound).all()
    out = torch.ones(7, 24)
    assert fb.matmul_fp8_block(a, b, out=out, accumulate=True) is out
    assert ((out - 1 - ref).abs() <= bound + 2.0 ** -23 * (1 + ref.abs())).all()
    bias = torch.randn(24)
    y = fb.matmul_fp8_block(a, b, bias=bias)
    assert y.dtype == torch.bfloat16
    want = ref + bias.bfloat16().double()
    assert ((y - want).abs() <= 2.0 ** -8 * want.abs() + 2 * bound + 1e-6).all()


def test_linear_gradients_are_products_of_the_cast_operands():
    torch.manual_seed(2)
    x = torch.randn(3, 50, 136, requires_grad=True)
    w, b = torch.randn(72, 136, requires_grad=True), torch.randn(72, requires_grad=True)
    y = fb.linear_fp8_block(x, w, b)
    dy = torch.randn_like(y)
    y.backward(dy)
    x2, d2 = x.detach().view(150, 136), dy.view(150, 72)
    (xq, xt), (wq, _) = fb.quantize_fp8_block(x2, want_t=True), fb.quantize_fp8_block(w.detach(), tile=True)
    dq, dt = fb.quantize_fp8_block(d2, want_t=True)
    close = lambda got, a, c: torch.allclose(got, a @ c, rtol=1e-5, atol=1e-4)  # noqa: E731
    assert y.dtype == torch.float32 and y.shape == (3, 50, 72)
    assert close(y.detach().view(150, 72) - b.detach().bfloat16().float(), xq.dequantize(), wq.dequantize().t())
    assert close(x.grad.view(150, 136), dq.dequantize(), wq.dequantize())
    assert close(w.grad, dt.dequantize(), xt.dequantize().t())
    assert torch.allclose(b.grad, d2.sum(0), atol=1e-4)
    # the same values from a kept weight
    with torch.no_grad():
        assert torch.equal(fb.linear_fp8_block(x, wq, b), y)


def test_refusals():
    x = torch.randn(4, 64)
    w = torch.randn(32, 64)
    wq, _ = fb.quantize_fp8_block(w, tile=True)
    xq, _ = fb.quantize_fp8_block(x)
    with pytest.raises(ValueError, match="2-D"):
        fb.quantize_fp8_block(torch.randn(2, 3, 64))
    with pytest.raises(ValueError, match="floating"):
        fb.quantize_fp8_block(torch.ones(4, 64, dtype=torch.int32))
    with pytest.raises(ValueError, match="contraction"):
        fb.matmul_fp8_block(xq, fb.quantize_fp8_block(torch.randn(32, 128))[0])
    with pytest.raises(ValueError, match="out has to be"):
        fb.matmul_fp8_block(xq, wq, out=torch.empty(4, 31))
    with pytest.raises(ValueError, match="out has to be"):
        fb.matmul_fp8_block(xq, wq, out=torch.empty(32, 4).t())
    with pytest.raises(TypeError, match="bf16 or fp32"):
        fb.matmul_fp8_block(xq, wq, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="accumulate"):
        fb.matmul_fp8_block(xq, wq, accumulate=True)
    with pytest.raises(ValueError, match="accumulate"):
        fb.matmul_fp8_block(xq, wq, out=torch.zeros(4, 32, dtype=torch.bfloat16), accumulate=True)
    with pytest.raises(ValueError, match="bias"):
        fb.matmul_fp8_block(xq, wq, bias=torch.zeros(31))
    with pytest.raises(ValueError, match="features"):
        fb.linear_fp8_block(x, torch.randn(32, 63))
    with pytest.raises(ValueError, match="without gradients"):
        fb.linear_fp8_block(x.requires_grad_(), wq)
    for data, cols, scales in ((wq.data, 640, wq.scales), (wq.data, 64, wq.scales[:, :31]),
                               (wq.data.t(), 32, wq.scales), (wq.data[:, :60], 64, wq.scales),
                               (wq.data, 64, wq.scales.flip(0).transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            fb.Fp8BlockTensor(data, cols, scales)
    with pytest.raises(TypeError):
        fb.Fp8BlockTensor(wq.data.float(), 64, wq.scales)
    with pytest.raises(AttributeError):
        wq.data = wq.data.clone()


def test_empty_matrices():
    e, e_t = fb.quantize_fp8_block(torch.empty(0, 64), want_t=True)
    assert e.shape == (0, 64) and e_t.shape == (64, 0)
    w, _ = fb.quantize_fp8_block(torch.randn(32, 64), tile=True)
    assert fb.matmul_fp8_block(e, w).shape == (0, 32)
    assert not fb.matmul_fp8_block(e_t, e_t).any()


def test_linear_gradient_against_differences():
    """On values that the format holds exactly (small whole numbers) the layer is linear, and so is a difference of
    its outputs: both sides are whole numbers below 2^24, and equal."""
    g = torch.Generator().manual_seed(3)
    whole = lambda *s: torch.randint(-4, 5, s, generator=g).float()  # noqa: E731
    x, w, dy = whole(140, 256).requires_grad_(), whole(16, 256).requires_grad_(), whole(140, 16)
    fb.linear_fp8_block(x, w).backward(dy)
    with torch.no_grad():
        f = lambda a, b: (fb.linear_fp8_block(a, b).double() * dy).sum()  # noqa: E731
        d = whole(140, 256)
        assert f(x + d, w) - f(x, w) == (x.grad.double() * d).sum()
        d = whole(16, 256)
        assert f(x, w + d) - f(x, w) == (w.grad.double() * d).sum()


def _mlp_reference(x, wg, wu, wd, kind, dy):
    """The gated block by its formulas in 64 bits, from the cast values of its operands."""
    r = lambda v, rows, cols: _cast_double(v, rows, cols)  # noqa: E731
    bf = lambda v: v.to(torch.bfloat16).double()  # noqa: E731
    xv, gv, uv, dv = r(x, 1, 128), r(wg, 128, 128), r(wu, 128, 128), r(wd, 128, 128)
    g, u = bf(xv @ gv.t()).requires_grad_(), bf(xv @ uv.t()).requires_grad_()
    act = torch.nn.functional.silu(g) if kind == "swiglu" else torch.nn.functional.gelu(g, approximate="tanh")
    h = act * u
    hb = bf(h.detach())
    y = r(hb, 1, 128) @ dv.t()
    dh = bf(r(dy, 1, 128) @ dv)
    dg, du = (bf(t) for t in torch.autograd.grad(h, (g, u), dh))
    dgu, wgu = torch.cat([dg, du], 1), torch.cat([gv, uv])
    dw = r(dgu, 128, 1).t() @ r(x, 128, 1)
    return y, r(dgu, 1, 128) @ wgu, dw[:g.shape[1]], dw[g.shape[1]:], r(dy, 128, 1).t() @ r(hb, 128, 1)


def _cast_double(v, rows, cols):
    """bf16 values in blocks of 1 x 128 (rows = 1), 128 x 1 or 128 x 128, as the (separately tested) cast has them."""
    v = v.detach().to(torch.bfloat16)
    if rows == 1:
        return fb.quantize_fp8_block(v)[0].dequantize().double()
    if cols == 1:
        return fb.quantize_fp8_block(v, want=False, want_t=True)[1].dequantize().t().double()
    return fb.quantize_fp8_block(v, tile=True)[0].dequantize().double()


def _norm_off(a, b):
    return float((a.double() - b).norm() / b.norm())


@pytest.mark.parametrize("kind", ["swiglu", "geglu"])
@pytest.mark.parametrize("T,H,I", [(1, 64, 128), (37, 136, 256), (130, 72, 384)])
def test_gated_mlp_forward_and_gradients(T, H, I, kind):
    g = torch.Generator().manual_seed(T + I)
    n = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(torch.bfloat16)  # noqa: E731
    x, dy = n(T, H), n(T, H)
    wg, wu, wd = n(I, H, scale=H ** -0.5), n(I, H, scale=H ** -0.5), n(H, I, scale=I ** -0.5)
    want = _mlp_reference(x, wg, wu, wd, kind, dy)
    x.requires_grad_()
    fused, wd = torch.cat([wg, wu]).requires_grad_(), wd.requires_grad_()
    wg, wu = wg.requires_grad_(), wu.requires_grad_()
    y = fb.gated_mlp_fp8_block(x, wg, wu, wd, kind)
    got = [y.detach(), *torch.autograd.grad(y, (x, wg, wu, wd), dy)]
    # outputs are rounded to bf16 (2^-8 of a value at most); a bf16 value in between that falls to the other side of
    # a rounding in 32 bits moves by 2^-7 of itself, and its 8-bit form by up to 2^-3: rare, below 2^-7 of a norm
    for a, b in zip(got, want):
        assert a.dtype == torch.bfloat16 and _norm_off(a, b) < 2.0 ** -6
    y2 = fb.gated_mlp_fp8_block(x, fused, None, wd, kind)
    gf = torch.autograd.grad(y2, (x, fused, wd), dy)
    assert torch.equal(y2, y) and torch.equal(gf[0], got[1])
    assert torch.equal(gf[1], torch.cat([got[2], got[3]])) and torch.equal(gf[2], got[4])
    with torch.no_grad():
        kept = [fb.quantize_fp8_block(w, tile=True)[0] for w in (fused, wd)]
        assert torch.equal(fb.gated_mlp_fp8_block(x, kept[0], None, kept[1], kind), y)


def test_gated_mlp_gradients_of_some_inputs_only():
    g = torch.Generator().manual_seed(5)
    mk = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)  # noqa: E731
    x, wg, wu, wd, dy = mk(2, 9, 64), mk(128, 64), mk(128, 64), mk(64, 128), mk(2, 9, 64)
    leaves = [x, wg, wu, wd]
    for t in leaves:
        t.requires_grad_()
    full = torch.autograd.grad(fb.gated_mlp_fp8_block(*leaves), leaves, dy)
    for i in range(4):
        for t in leaves:
            t.requires_grad_(t is leaves[i])
        (one,) = torch.autograd.grad(fb.gated_mlp_fp8_block(*leaves), (leaves[i],), dy)
        assert one.shape == leaves[i].shape and torch.equal(one, full[i])


def test_gated_mlp_refusals():
    x, wg, wd = torch.randn(3, 64), torch.randn(256, 64), torch.randn(64, 128)
    with pytest.raises(ValueError, match="activation"):
        fb.gated_mlp_fp8_block(x, wg, None, wd, "relu")
    with pytest.raises(ValueError, match="multiple of 128"):
        fb.gated_mlp_fp8_block(x, torch.randn(128, 64), None, torch.randn(64, 64))
    with pytest.raises(ValueError, match="do not fit"):
        fb.gated_mlp_fp8_block(x, wg, wg, wd)
    with pytest.raises(ValueError, match="features"):
        fb.gated_mlp_fp8_block(torch.randn(3, 65), wg, None, wd)
    q = [fb.quantize_fp8_block(w, tile=True)[0] for w in (wg, wd)]
    with pytest.raises(ValueError, match="8-bit weights"):
        fb.gated_mlp_fp8_block(x, q[0], None, wd)
    with pytest.raises(ValueError, match="without gradients"):
        fb.gated_mlp_fp8_block(x.requires_grad_(), q[0], None, q[1])


# ------------------------------------------------------------------------------------------------
# Models
# ------------------------------------------------------------------------------------------------
def _mlp(H, I, fused, recipe="block128"):
    from lset_b200.models.layers import GatedMLP
    from lset_b200.train.quantization.fp8 import apply_fp8_training

    torch.manual_seed(11)
    return apply_fp8_training(GatedMLP(H, I, "swiglu", fused), recipe)


@pytest.fixture
def calls(monkeypatch):
    seen = []
    real = fb.gated_mlp_fp8_block
    monkeypatch.setattr(fb, "gated_mlp_fp8_block", lambda *a: seen.append(a) or real(*a))
    return seen


@pytest.mark.parametrize("fused", [False, True])
def test_gated_mlp_module_runs_as_one_operator(fused, calls):
    mlp = _mlp(64, 256, fused)
    x = torch.randn(5, 64)
    y = mlp(x)
    assert len(calls) == 1
    y.sum().backward()
    assert all(p.grad is not None and p.grad.abs().sum() > 0 for p in mlp.parameters())
    handle = mlp.down_proj.register_forward_hook(lambda *a: None)      # a hook wants the layer's own call
    z = mlp(x)
    assert len(calls) == 1 and torch.allclose(z, y, rtol=2e-2, atol=2e-2 * float(y.abs().max()))
    handle.remove()
    mlp.down_proj.forward = type(mlp.down_proj).forward.__get__(mlp.down_proj)   # and so does a replaced forward
    mlp(x)
    assert len(calls) == 1


@pytest.mark.parametrize("H,I,recipe", [(64, 144, "block128"), (64, 256, "tensorwise")])
def test_gated_mlp_module_of_other_widths_and_recipes_runs_layer_by_layer(H, I, recipe, calls):
    y = _mlp(H, I, True, recipe)(torch.randn(5, H))
    assert y.shape == (5, H) and not calls


def _tiny():
    from lset_b200.models import Qwen3Config, Qwen3Decoder

    torch.manual_seed(12)
    return Qwen3Decoder(Qwen3Config(vocab_size=97, hidden_size=64, intermediate_size=128, num_hidden_layers=2,
                                    num_attention_heads=4, num_key_value_heads=2, head_dim=16)).eval()


def test_inference_model_keeps_8_bit_weights(calls):
    from lset_b200.train.quantization.fp8 import Fp8KeptLinear, apply_fp8_inference

    model, ids = _tiny(), torch.randint(0, 97, (2, 9), generator=torch.Generator().manual_seed(0))
    with torch.no_grad():
        want = model(ids)["hidden_states"]
        apply_fp8_inference(model)
        got = model(ids)["hidden_states"]
    kinds = [type(m) for m in model.modules()]
    assert kinds.count(Fp8KeptLinear) == 2 * 6 and not any(issubclass(k, torch.nn.Linear) for k in kinds)
    assert len(calls) == 2
    # each of the seven products a layer is off by about 2^-4 / sqrt(3) x sqrt(2) relative to its norm at most
    assert float(torch.nn.functional.cosine_similarity(got, want, dim=-1).min()) > 0.98
    state = model.state_dict()
    assert sum(v.dtype == torch.uint8 for v in state.values()) == 2 * 2 * 6
    again = apply_fp8_inference(_tiny())
    again.load_state_dict(state)
    with torch.no_grad():
        assert torch.equal(again(ids)["hidden_states"], got)


def test_layers_of_biased_models_keep_their_bias():
    from lset_b200.train.quantization.fp8 import Fp8KeptLinear, apply_fp8_inference

    torch.manual_seed(13)
    m = torch.nn.Sequential(torch.nn.Linear(64, 32), torch.nn.Linear(32, 20))
    x = torch.randn(7, 64)
    with torch.no_grad():
        q, _ = fb.quantize_fp8_block(m[0].weight, tile=True)
        want = fb.linear_fp8_block(x, q, m[0].bias)
        last = m[1](want)
        apply_fp8_inference(m)
        assert isinstance(m[0], Fp8KeptLinear) and type(m[1]) is torch.nn.Linear     # 20: no multiple of 16
        assert torch.equal(m[0](x), want) and torch.equal(m(x), last)
    with pytest.raises(ValueError, match="without gradients"):
        m[0](x.requires_grad_())


@pytest.mark.parametrize("family", ["qwen3", "llama", "embeddinggemma", "bert"])
def test_every_family_encodes_with_kept_weights(family):
    from lset_b200.models import BertConfig, GemmaConfig, LlamaConfig, get_model_spec
    from lset_b200.models import Qwen3Config
    from lset_b200.train.quantization.fp8 import Fp8KeptLinear, apply_fp8_inference

    dims = dict(vocab_size=97, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4)
    cfg = {"qwen3": lambda: Qwen3Config(**dims, num_key_value_heads=2, head_dim=16),
           "llama": lambda: LlamaConfig(**dims, num_key_value_heads=2, head_dim=16),
           "embeddinggemma": lambda: GemmaConfig(**dims, num_key_value_heads=1, head_dim=16),
           "bert": lambda: BertConfig(**dims)}[family]()
    torch.manual_seed(14)
    model = get_model_spec(family).model_cls(cfg).eval()
    ids, mask = torch.randint(0, 97, (2, 11)), torch.ones(2, 11, dtype=torch.long)
    mask[1, 7:] = 0
    with torch.no_grad():
        want = model(ids, mask)["hidden_states"]
        apply_fp8_inference(model)
        got = model(ids, mask)["hidden_states"]
    assert sum(isinstance(m, Fp8KeptLinear) for m in model.modules()) == 12
    keep = mask.bool()
    assert float(torch.nn.functional.cosine_similarity(got[keep], want[keep], dim=-1).min()) > 0.97


def test_gradients_of_some_inputs_of_a_linear_layer():
    g = torch.Generator().manual_seed(6)
    mk = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)  # noqa: E731
    x, w, b, dy = mk(2, 9, 64), mk(32, 64), mk(32), mk(2, 9, 32)
    leaves = [x, w, b]
    for t in leaves:
        t.requires_grad_()
    full = torch.autograd.grad(fb.linear_fp8_block(*leaves), leaves, dy)
    for i in range(3):
        for t in leaves:
            t.requires_grad_(t is leaves[i])
        (one,) = torch.autograd.grad(fb.linear_fp8_block(*leaves), (leaves[i],), dy)
        assert one.shape == leaves[i].shape and torch.equal(one, full[i])


def test_no_gradient_of_a_gradient():
    x, w = torch.randn(4, 64, requires_grad=True), torch.randn(32, 64, requires_grad=True)
    (dx,) = torch.autograd.grad(fb.linear_fp8_block(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_evaluation_of_a_model_with_the_recipe_keeps_8_bit_weights(monkeypatch):
    import sys
    import types

    from lset_b200.config import LSETConfig
    from lset_b200.eval import mteb_evaluator
    from lset_b200.eval.run import run_eval

    seen = []
    monkeypatch.setitem(sys.modules, "mteb", types.SimpleNamespace(
        get_tasks=lambda tasks: list(tasks), evaluate=lambda *a, **k: types.SimpleNamespace(task_results=[])))
    monkeypatch.setattr(mteb_evaluator.LSETMTEBModel, "from_pretrained",
                        classmethod(lambda cls, path, **kw: seen.append(kw.get("fp8", False))))
    for enabled, recipe in ((True, "block128"), (True, "tensorwise"), (False, "block128")):
        cfg = LSETConfig()
        cfg.fp8.enabled, cfg.fp8.recipe = enabled, recipe
        run_eval(cfg)
    assert seen == [True, False, False]


# ------------------------------------------------------------------------------------------------
# Whose memory a matrix is
# ------------------------------------------------------------------------------------------------
def _copies(q, tmp_path):
    import copy
    import pickle

    torch.save(q, tmp_path / "q.pt")
    return {"deepcopy": copy.deepcopy(q), "pickle": pickle.loads(pickle.dumps(q)),
            "save": torch.load(tmp_path / "q.pt", weights_only=False)}


@pytest.mark.parametrize("rows,cols,e5m2", [(40, 640, False), (1, 136, True), (0, 64, False)])
def test_copies_are_on_memory_of_their_own(rows, cols, e5m2, tmp_path):
    import copy

    q, _ = fb.quantize_fp8_block(torch.randn(rows, cols), e5m2=e5m2)
    values = q.dequantize()
    for name, c in _copies(q, tmp_path).items():
        assert type(c) is fb.Fp8BlockTensor and c.shape == q.shape and c.e5m2 == q.e5m2, name
        assert c._where == (c.data.data_ptr(), q._where[1], c.scales.data_ptr(), q._where[3]), name
        assert rows == 0 or (c._where[0] != q._where[0] and c._where[2] != q._where[2]), name
    same = copy.copy(q)
    assert same.data is q.data and same._where == q._where
    copies = _copies(q, tmp_path)
    q.data.zero_()
    assert all(torch.equal(c.dequantize(), values) for c in copies.values())


def test_parts_of_a_matrix_copy_with_their_strides(tmp_path):
    b, _ = fb.quantize_fp8_block(torch.randn(384, 640), tile=True)
    part = fb.Fp8BlockTensor(b.data[128:256, :512], 512, b.scales[:1, 128:256])
    for c in _copies(part, tmp_path).values():
        assert c._where[1] == c.data.stride(0) and torch.equal(c.dequantize(), part.dequantize())


def test_exchanged_memory_is_looked_at_again():
    q, _ = fb.quantize_fp8_block(torch.randn(40, 640))
    other, _ = fb.quantize_fp8_block(torch.randn(40, 640))
    q.data.data, q.scales.data = other.data, other.scales
    assert q._where == (other.data.data_ptr(), 640, other.scales.data_ptr(), 40)
    q.data.data = torch.zeros(40, 656, dtype=torch.uint8)
    assert q._where == (q.data.data_ptr(), 656, other.scales.data_ptr(), 40)
    q.scales.data = torch.zeros(2, 39, 4, dtype=torch.uint8)      # a row less
    with pytest.raises(ValueError, match="belong together"):
        q._where
    q.scales.data = other.scales
    q.data.data = torch.zeros(656, 40, dtype=torch.uint8).t()
    with pytest.raises(ValueError, match="next to one another"):
        q._where
    q.data.data = other.data
    q.data.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="released"):
        q._where


def test_products_of_more_rows_than_are_counted_are_refused(monkeypatch):
    """The kernels' sizes are ints of 32 bits, which 2^31 rows would pass (0 columns: nothing is stored here)."""
    many = fb.Fp8BlockTensor(torch.empty(1 << 31, 0, dtype=torch.uint8), 0, torch.empty(0, 1 << 31, 4, dtype=torch.uint8))
    few = fb.Fp8BlockTensor(torch.empty(2, 0, dtype=torch.uint8), 0, torch.empty(0, 2, 4, dtype=torch.uint8))
    monkeypatch.setattr(fb.nv, "use_native", lambda *t: True)
    made = []
    monkeypatch.setattr(fb, "_on_device", lambda *t: made.append(t))
    for a, b in ((many, few), (few, many)):
        with pytest.raises(ValueError, match="more rows or columns"):
            fb.matmul_fp8_block(a, b)
    assert not made


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.bfloat16, torch.float64])
def test_results_of_empty_batches_have_the_type_of_others(dtype):
    w, wd = torch.randn(256, 64, requires_grad=True), torch.randn(64, 128, requires_grad=True)
    b = torch.randn(256)
    for fn in (lambda x: fb.linear_fp8_block(x, w, b), lambda x: fb.gated_mlp_fp8_block(x, w, None, wd)):
        empty, some = torch.empty(0, 64, dtype=dtype, requires_grad=True), torch.randn(3, 64).to(dtype)
        y, z = fn(empty), fn(some)
        assert y.dtype == z.dtype == (torch.float32 if dtype is torch.float32 else torch.bfloat16)
        assert y.shape == (0, z.shape[1])
        y.sum().backward()
        assert empty.grad.shape == (0, 64) and empty.grad.dtype == dtype and not w.grad.any()


def test_weights_of_another_type_are_not_loaded_into_bytes():
    from lset_b200.train.quantization.fp8 import apply_fp8_inference

    plain = _tiny().state_dict()
    model = apply_fp8_inference(_tiny())
    before = {k: v.clone() for k, v in model.state_dict().items()}
    for strict in (True, False):      # not strict, missing scales alone would pass
        with pytest.raises(RuntimeError, match="before apply_fp8_inference"):
            model.load_state_dict(plain, strict=strict)
    assert all(torch.equal(v, before[k]) for k, v in model.state_dict().items() if v.dtype is torch.uint8)
    model.load_state_dict(before)


def test_adapters_stay_as_they_are_and_merge_with_the_values_of_kept_weights():
    from lset_b200.train.lora import LoRALinear, apply_lora
    from lset_b200.train.quantization.fp8 import Fp8KeptLinear, apply_fp8_inference

    model, ids = _tiny(), torch.randint(0, 97, (2, 9), generator=torch.Generator().manual_seed(0))
    apply_lora(model, r=16, target_modules=["q_proj", "down_proj"])
    for m in model.modules():
        if isinstance(m, LoRALinear):
            torch.nn.init.normal_(m.lora_B.weight, std=0.05)
    with torch.no_grad():
        want = model(ids)["hidden_states"]
        merged = [m.merged_weight() for m in model.modules() if isinstance(m, LoRALinear)]
        apply_fp8_inference(model)
        got = model(ids)["hidden_states"]
        layers = [m for m in model.modules() if isinstance(m, LoRALinear)]
        assert len(layers) == len(merged) == 4
        for m, w in zip(layers, merged):
            assert isinstance(m.base_linear, Fp8KeptLinear) and type(m.lora_A).__name__ == "Linear"
            assert float((m.merged_weight() - w).norm() / w.norm()) < 2.0 ** -4      # half a step of e4m3 at most
    assert float(torch.nn.functional.cosine_similarity(got, want, dim=-1).min()) > 0.98


def _tp_model():
    from lset_b200.models import Qwen3Config, Qwen3Decoder
    from lset_b200.models.layers import init_normal_
    from lset_b200.train.quantization.fp8 import apply_fp8_training

    torch.manual_seed(15)
    cfg = Qwen3Config(vocab_size=97, hidden_size=64, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=16)
    model = Qwen3Decoder(cfg, fused_projections=False)
    init_normal_(model, 0.05)
    return apply_fp8_training(model, "block128"), cfg, torch.randint(0, 97, (2, 9))


def _tp_worker(rank, world, port, out_dir):
    import os

    import torch.distributed as dist

    from lset_b200.dist.tp import apply_tp
    from lset_b200.models.parallel_plan import decoder_tp_plan

    os.environ.update(RANK=str(rank), WORLD_SIZE=str(world), MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    model, cfg, ids = _tp_model()
    apply_tp(model, dist.group.WORLD, decoder_tp_plan(cfg))
    seen = []
    real = fb.gated_mlp_fp8_block
    fb.gated_mlp_fp8_block = lambda *a: seen.append(a) or real(*a)
    out = model(ids)["hidden_states"]
    out.pow(2).sum().backward()
    if rank == 0:
        torch.save({"out": out.detach(), "grad": model.layers[0].mlp.down_proj.weight.grad, "calls": len(seen)},
                   os.path.join(out_dir, "tp.pt"))
    dist.barrier()
    dist.destroy_process_group()


def test_tensor_parallel_layers_run_one_by_one(tmp_path):
    """Shards of 256 features, which the gated operator would take: its partial sums would miss the all-reduce behind the
    down projection and the one in front of the gate's backward, so the layers' own forwards run. Blocks of 128 lie within
    a shard, and partial sums are what the shards add to in either case, but for where they are rounded."""
    import socket

    import torch.multiprocessing as mp

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_tp_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True)
    got = torch.load(tmp_path / "tp.pt", weights_only=False)
    model, _, ids = _tp_model()
    out = model(ids)["hidden_states"]
    out.pow(2).sum().backward()
    assert got["calls"] == 0
    # o_proj's blocks of 128 inputs become one of 32 a rank, with scales of their own: an 8-bit step, 2^-4 / sqrt(3) of a
    # value in the mean, at some of seven products a layer
    assert _norm_off(got["out"], out.detach()) < 0.1
    assert _norm_off(got["grad"], model.layers[0].mlp.down_proj.weight.grad[:, :256]) < 0.3

"""Block-scaled 8-bit operators on the GPU: the casts' bytes against the eager ones, products against 64-bit
sums of the values that the operands stand for, layers against their definition."""
import pytest
import torch

from lset_b200.ops import _native as nv
from lset_b200.ops import fp8_block as fb

pytestmark = pytest.mark.gpu


def _rand(*shape, seed=0, spread=2.0):
    g = torch.Generator("cuda").manual_seed(seed + sum(shape))
    x = torch.randn(*shape, generator=g, device="cuda")
    return (x * torch.exp(spread * torch.randn(*shape, generator=g, device="cuda"))).to(torch.bfloat16)


def _same_bytes(got, want):
    assert got.shape == want.shape and got.e5m2 == want.e5m2
    assert torch.equal(got.data[:, :got.cols].cpu(), want.data[:, :want.cols])
    assert torch.equal(got.scales.cpu(), want.scales)


def _check_product(c, a, b, bias=None, base=None):
    """Errors of a product: half a step of the output's type, and of the fp32 sums at most 2^-22 of the summed
    magnitudes for each of the K / 32 instructions (a sum cut to 24 bits is off by 2^-23 of itself) and two more
    for the products inside one."""
    A, B = a.dequantize().double(), b.dequantize().double()
    ref = A @ B.t()
    if bias is not None:
        ref = ref + bias.double()
    if base is not None:
        ref = ref + base.double()
    sums = (a.cols // 32 + 3) * 2.0 ** -22 * (A.abs() @ B.abs().t())
    half = 2.0 ** -8 if c.dtype == torch.bfloat16 else 2.0 ** -23
    assert ((c.double() - ref).abs() <= half * ref.abs() + sums).all(), \
        float(((c.double() - ref).abs() - half * ref.abs() - sums).max())


@pytest.mark.parametrize("R,C", [(1, 8), (3, 136), (128, 128), (129, 520), (300, 264), (1000, 1032), (7, 4096)])
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("e5m2", [False, True])
def test_cast_has_the_bytes_of_the_eager_one(R, C, tile, e5m2):
    x = _rand(R, C)
    x[R // 2] = 0
    x[0, 0], x[R - 1, C - 1] = 448.0, 2.0 ** -133
    if R > 2:
        x[1, C // 2], x[2, 1] = float("inf"), float("nan")
    q, q_t = fb.quantize_fp8_block(x, tile=tile, e5m2=e5m2, want_t=True)
    e, e_t = fb.quantize_fp8_block(x.cpu(), tile=tile, e5m2=e5m2, want_t=True)
    _same_bytes(q, e)
    _same_bytes(q_t, e_t)
    only, none = fb.quantize_fp8_block(x, tile=tile, e5m2=e5m2)
    assert none is None and torch.equal(only.data[:, :C], q.data[:, :C])
    none, only = fb.quantize_fp8_block(x, tile=tile, e5m2=e5m2, want=False, want_t=True)
    assert none is None and torch.equal(only.data[:, :R], q_t.data[:, :R])


def test_cast_of_strided_and_unaligned_inputs():
    x = _rand(70, 300)
    for view in (x[:, 4:260], x[3:, :256], x[::2, 8:136], x[:, 1:257], x.t()[:, :64], x[:8].t()[:64].float()):
        q, q_t = fb.quantize_fp8_block(view, want_t=True)
        e, e_t = fb.quantize_fp8_block(view.cpu(), want_t=True)
        _same_bytes(q, e)
        _same_bytes(q_t, e_t)


SHAPES = [(1, 128, 128), (1, 8, 16), (5, 264, 272), (16, 128, 1024), (17, 136, 520), (33, 1000, 640), (64, 256, 4096),
          (65, 512, 2560), (128, 128, 128), (129, 257, 144), (300, 264, 208), (500, 384, 1920), (1, 2560, 9728),
          (12, 4096, 2560), (1000, 1032, 1040),
          # tiles of CTA pairs: one stage, whole and ragged ones, more tiles than pairs, bands of them
          (1030, 2304, 16), (1500, 2056, 256), (2000, 2304, 640), (2561, 1288, 1040), (4097, 4360, 2576),
          (1100, 16392, 2064),
          # last waves in half tiles: of one wave, behind whole ones, with halves that lie outside the matrix
          (4000, 264, 2048), (2300, 1024, 1040), (5000, 4096, 272), (9000, 2056, 640)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("tile", [False, True])
def test_product(M, N, K, tile):
    a, _ = fb.quantize_fp8_block(_rand(M, K))
    b, _ = fb.quantize_fp8_block(_rand(N, K, seed=1), tile=tile)
    for dt in (torch.bfloat16, torch.float32):
        c = fb.matmul_fp8_block(a, b, out_dtype=dt)
        nv.check_status()
        assert c.dtype == dt and c.shape == (M, N)
        _check_product(c, a, b)


@pytest.mark.parametrize("M,N,K", [(5, 264, 272), (200, 384, 1040), (1800, 1800, 640)])
@pytest.mark.parametrize("formats", [(True, False), (False, True), (True, True)])
def test_product_of_either_format(M, N, K, formats):
    a, _ = fb.quantize_fp8_block(_rand(M, K), e5m2=formats[0])
    b, _ = fb.quantize_fp8_block(_rand(N, K, seed=1), e5m2=formats[1])
    _check_product(fb.matmul_fp8_block(a, b, out_dtype=torch.float32), a, b)


@pytest.mark.parametrize("M,N,K", [(3, 136, 640), (150, 256, 272), (700, 520, 1040), (1700, 1800, 1040)])
def test_bias_accumulation_and_outputs_within_a_larger_tensor(M, N, K):
    a, _ = fb.quantize_fp8_block(_rand(M, K))
    b, _ = fb.quantize_fp8_block(_rand(N, K, seed=1), tile=True)
    bias = _rand(N, spread=0.5)
    _check_product(fb.matmul_fp8_block(a, b, bias=bias), a, b, bias)
    _check_product(fb.matmul_fp8_block(a, b, bias=bias, out_dtype=torch.float32), a, b, bias)
    for dt in (torch.bfloat16, torch.float32):
        wide = torch.full((M + 2, N + 24), 7.0, dtype=dt, device="cuda")
        out = wide[1:M + 1, 8:N + 8]
        assert fb.matmul_fp8_block(a, b, out=out) is out
        _check_product(out, a, b)
        kept = wide.clone()
        kept[1:M + 1, 8:N + 8] = 7
        assert (kept == 7).all()                 # nothing around it
    base = torch.randn(M, N, device="cuda")
    out = base.clone()
    fb.matmul_fp8_block(a, b, out=out, accumulate=True)
    _check_product(out, a, b, base=base)


def test_parts_of_a_cast_matrix():
    """Rows of a kept weight (the gate half of a fused one) are a weight of their own."""
    a, _ = fb.quantize_fp8_block(_rand(40, 640))
    b, _ = fb.quantize_fp8_block(_rand(384, 640, seed=1), tile=True)
    for lo, hi in ((0, 128), (128, 384), (200, 201)):
        part = fb.Fp8BlockTensor(b.data[lo:hi], 640, b.scales[:, lo:hi])
        _check_product(fb.matmul_fp8_block(a, part), a, part)


@pytest.mark.parametrize("M,N,K", [(5, 136, 272), (300, 264, 640), (1500, 2056, 640), (2000, 2304, 16)])
def test_bytes_of_blocks_that_are_not_there_are_not_read(M, N, K):
    a, _ = fb.quantize_fp8_block(_rand(M, K))
    b, _ = fb.quantize_fp8_block(_rand(N, K, seed=1), tile=True)
    want = fb.matmul_fp8_block(a, b)
    for q in (a, b):
        words = q.scales.transpose(0, 1).reshape(q.rows, -1).clone()
        words[:, (K + 127) // 128:] = 255          # not a number
        q.scales.copy_(words.view(q.rows, -1, 4).transpose(0, 1))
        q.data[:, K:] = 0x7F
    assert torch.equal(fb.matmul_fp8_block(a, b), want)


def test_values_that_are_not_finite_stay_in_their_rows():
    x = _rand(6, 384)
    x[2, 130], x[4, 0] = float("nan"), float("inf")
    a, _ = fb.quantize_fp8_block(x)
    b, _ = fb.quantize_fp8_block(_rand(128, 384, seed=1), tile=True)
    c = fb.matmul_fp8_block(a, b)
    assert torch.isnan(c[[2, 4]]).all() and torch.isfinite(c[[0, 1, 3, 5]]).all()


def test_scales_over_their_whole_range():
    """Factors from 2^-100 to 2^100 on either side: the product of two scales is what counts."""
    for ea, eb in ((-100, 90), (100, -110), (-60, -50), (50, 40)):
        a, _ = fb.quantize_fp8_block((_rand(9, 256, spread=0.5).float() * 2.0 ** ea).to(torch.bfloat16))
        b, _ = fb.quantize_fp8_block((_rand(136, 256, seed=1, spread=0.5).float() * 2.0 ** eb).to(torch.bfloat16))
        _check_product(fb.matmul_fp8_block(a, b, out_dtype=torch.float32), a, b)


def test_refusals_and_empty_products():
    with pytest.raises(ValueError, match="multiple of 8"):
        fb.quantize_fp8_block(torch.zeros(4, 12, device="cuda"))
    q, _ = fb.quantize_fp8_block(torch.zeros(4, 64, device="cuda"))
    with pytest.raises(ValueError, match="on cuda"):
        fb.matmul_fp8_block(q, q, out=torch.zeros(4, 4))
    with pytest.raises(ValueError, match="16 bytes"):
        fb.matmul_fp8_block(q, fb.Fp8BlockTensor(torch.zeros(4, 72, dtype=torch.uint8, device="cuda")[:, :64], 64, q.scales))
    e, e_t = fb.quantize_fp8_block(torch.empty(0, 64, device="cuda"), want_t=True)
    assert fb.matmul_fp8_block(e, q).shape == (0, 4)
    assert not fb.matmul_fp8_block(e_t, e_t).any()
    bias = torch.arange(64, device="cuda").to(torch.bfloat16)
    assert torch.equal(fb.matmul_fp8_block(e_t, e_t, bias=bias), bias.expand(64, 64))


# ------------------------------------------------------------------------------------------------
# Layers
# ------------------------------------------------------------------------------------------------
def _value(v, rows, cols):
    """What a matrix stands for once it is cast (the cast has tests of its own), in 64 bits."""
    v = v.detach()
    if rows == 1:
        return fb.quantize_fp8_block(v)[0].dequantize().double()
    if cols == 1:
        return fb.quantize_fp8_block(v, want=False, want_t=True)[1].dequantize().t().double()
    return fb.quantize_fp8_block(v, tile=True)[0].dequantize().double()


def _off(a, b):
    return float((a.double() - b).norm() / b.norm().clamp(min=1e-300))


TOKENS = [1, 2, 15, 16, 17, 31, 32, 33, 64, 129, 333, 1000, 2600]


@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("K,N,bias", [(136, 264, True), (1024, 512, False), (640, 72, True), (4104, 256, False)])
def test_linear_forward_and_gradients(T, K, N, bias):
    x, w, dy = _rand(T, K, spread=1.0), _rand(N, K, seed=1, spread=0.5), _rand(T, N, seed=2, spread=1.0)
    b = _rand(N, seed=3, spread=0.5) if bias else None
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = fb.linear_fp8_block(x, w, b)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    nv.check_status()
    wv = _value(w, 128, 128)
    want = [_value(x, 1, 128) @ wv.t() + (0 if b is None else b.detach().double()), _value(dy, 1, 128) @ wv,
            _value(dy, 128, 1).t() @ _value(x, 128, 1)] + ([] if b is None else [dy.double().sum(0)])
    for a, c in zip(got, want):      # bf16 outputs: half a step, 2^-8 of a value, at most
        assert a.dtype == torch.bfloat16 and a.shape == c.shape and _off(a, c) < 2.0 ** -8
    with torch.no_grad():
        q, _ = fb.quantize_fp8_block(w, tile=True)
        assert torch.equal(fb.linear_fp8_block(x, q, b), y)


def test_linear_of_other_types_and_shapes():
    x, w = _rand(2, 3, 5, 128, spread=0.5).float(), _rand(64, 128, spread=0.5).float()
    y = fb.linear_fp8_block(x.requires_grad_(), w.requires_grad_())
    assert y.dtype == torch.float32 and y.shape == (2, 3, 5, 64)
    y.sum().backward()
    assert x.grad.dtype == w.grad.dtype == torch.float32 and x.grad.shape == x.shape
    e = fb.linear_fp8_block(torch.empty(0, 128, device="cuda", dtype=torch.bfloat16), w)
    assert e.shape == (0, 64)


def test_weight_gradients_go_to_the_accumulator():
    x, w, dy = _rand(300, 256, spread=1.0), _rand(384, 256, seed=1, spread=0.5), _rand(300, 384, seed=2, spread=1.0)
    w.requires_grad_()
    w.main_grad = torch.full((384, 256), 3.0, device="cuda")
    fb.linear_fp8_block(x, w).backward(dy)
    want = _value(dy, 128, 1).t() @ _value(x, 128, 1)
    assert w.grad is None and _off(w.main_grad - 3, want) < 1e-5


@pytest.mark.parametrize("kind", ["swiglu", "geglu"])
@pytest.mark.parametrize("T,H,I", [(1, 256, 128), (100, 264, 384), (2049, 2048, 1280), (1500, 4104, 1024)])
def test_gated_mlp_against_the_separate_steps(T, H, I, kind):
    from lset_b200.ops.activation import glu

    x, dy = _rand(T, H, spread=0.5), _rand(T, H, seed=1, spread=1.0)
    w, wd = (_rand(2 * I, H, seed=2, spread=0.3) * H ** -0.5), (_rand(H, I, seed=3, spread=0.3) * I ** -0.5)
    leaves = [t.requires_grad_() for t in (x, w, wd)]
    y = fb.gated_mlp_fp8_block(x, w, None, wd, kind)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    with torch.no_grad():
        (xq, xt), (dq, dt) = fb.quantize_fp8_block(x, want_t=True), fb.quantize_fp8_block(dy, want_t=True)
        (wq, wt), (vq, vt) = (fb.quantize_fp8_block(t, tile=True, want_t=True) for t in (w, wd))
        gu, dh = fb.matmul_fp8_block(xq, wq), fb.matmul_fp8_block(dq, vt)
    gu.requires_grad_()
    h = glu(gu, kind)
    (dgu,) = torch.autograd.grad(h, gu, dh)
    (hq, ht), (d, d_t) = fb.quantize_fp8_block(h, want_t=True), fb.quantize_fp8_block(dgu, want_t=True)
    want = [fb.matmul_fp8_block(hq, vq), fb.matmul_fp8_block(d, wt), fb.matmul_fp8_block(d_t, xt),
            fb.matmul_fp8_block(dt, ht)]
    nv.check_status()
    # The same bytes but for values that two sigmoids 2^-21 apart put on either side of a rounding to bf16 (one in 2^11,
    # by 2^-7 of itself) and, of those, to 3 bits (one in 2^3, by 2^-3): 2^-14 of the values by 2^-3, 2^-10 of a norm,
    # and half a step of bf16 outputs, 2^-8 of a value, for sums that fall to the other side of theirs.
    for a, b in zip(got, want):
        assert _off(a, b.double()) < 2.0 ** -10 + 2.0 ** -8


def _mlp_want(x, wgu, wd, kind, dy):
    bf = lambda v: v.to(torch.bfloat16)  # noqa: E731
    I = wd.shape[1]
    wv, dv = _value(wgu, 128, 128), _value(wd, 128, 128)
    gu = bf(_value(x, 1, 128) @ wv.t()).double().requires_grad_()
    act = torch.nn.functional.silu if kind == "swiglu" else lambda g: torch.nn.functional.gelu(g, approximate="tanh")
    h = act(gu[:, :I]) * gu[:, I:]
    hb, dh = bf(h.detach()), bf(_value(dy, 1, 128) @ dv).double()
    dgu = bf(torch.autograd.grad(h, gu, dh)[0])
    return [_value(hb, 1, 128) @ dv.t(), _value(dgu, 1, 128) @ wv, _value(dgu, 128, 1).t() @ _value(x, 128, 1),
            _value(dy, 128, 1).t() @ _value(hb, 128, 1)]


@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("H,I,kind", [(72, 128, "swiglu"), (264, 384, "geglu"), (1024, 1152, "swiglu")])
def test_gated_mlp_forward_and_gradients(T, H, I, kind):
    x, dy = _rand(T, H, spread=0.5), _rand(T, H, seed=1, spread=1.0)
    w, wd = _rand(2 * I, H, seed=2, spread=0.3), _rand(H, I, seed=3, spread=0.3)
    w, wd = (w.float() * H ** -0.5).to(torch.bfloat16), (wd.float() * I ** -0.5).to(torch.bfloat16)
    want = _mlp_want(x, w, wd, kind, dy)
    leaves = [t.requires_grad_() for t in (x, w, wd)]
    y = fb.gated_mlp_fp8_block(x, w, None, wd, kind)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    nv.check_status()
    # 2^-8 of a value for the bf16 output, and as much of a norm for values in between that fall to the other side
    # of a rounding when sums are taken in another order
    for a, c in zip(got, want):
        assert a.dtype == torch.bfloat16 and a.shape == c.shape and _off(a, c) < 2.0 ** -7
    with torch.no_grad():
        kept = [fb.quantize_fp8_block(t, tile=True)[0] for t in (w, wd)]
        assert torch.equal(fb.gated_mlp_fp8_block(x, kept[0], None, kept[1], kind), y)
    halves = [t.detach().clone().requires_grad_() for t in (w[:I], w[I:])]
    y2 = fb.gated_mlp_fp8_block(x, *halves, wd, kind)
    g2 = torch.autograd.grad(y2, [x, *halves, wd], dy)
    assert torch.equal(y2, y) and torch.equal(g2[0], got[1]) and torch.equal(g2[3], got[3])
    # (a product of half the rows may add its sums in another order: the same bound against the formula, then)
    assert _off(torch.cat([g2[1], g2[2]]), want[2]) < 2.0 ** -7


# ------------------------------------------------------------------------------------------------
# Ways of calling
# ------------------------------------------------------------------------------------------------
def test_gradients_of_some_inputs_only():
    x, w, b, dy = _rand(300, 256, spread=1.0), _rand(520, 256, seed=1, spread=0.5), _rand(520, seed=2), _rand(300, 520, seed=3)
    wg, wu, wd, dz = (_rand(256, 256, seed=4, spread=0.3) * 0.06, _rand(256, 256, seed=5, spread=0.3) * 0.06,
                      _rand(256, 256, seed=6, spread=0.3) * 0.06, _rand(300, 256, seed=7))
    for fn, leaves, grad in ((fb.linear_fp8_block, [x, w, b], dy), (fb.gated_mlp_fp8_block, [x, wg, wu, wd], dz)):
        for t in leaves:
            t.requires_grad_()
        full = torch.autograd.grad(fn(*leaves), leaves, grad)
        for some in range(1, 1 << len(leaves)):
            for i, t in enumerate(leaves):
                t.requires_grad_(bool(some >> i & 1))
            wanted = [t for t in leaves if t.requires_grad]
            got = torch.autograd.grad(fn(*leaves), wanted, grad)
            for t, g in zip(wanted, got):
                want = full[[a is t for a in leaves].index(True)]
                assert torch.equal(g, want), some
    nv.check_status()


def test_kept_weights_in_the_wider_format_and_as_parts():
    x = _rand(50, 512, spread=0.5)
    w, wd = _rand(512, 512, seed=1, spread=0.3) * 0.05, _rand(512, 256, seed=2, spread=0.3) * 0.05
    with torch.no_grad():
        for T in (7, 50):
            for e5m2 in (False, True):
                q, _ = fb.quantize_fp8_block(w, tile=True, e5m2=e5m2)
                d, _ = fb.quantize_fp8_block(wd, tile=True, e5m2=e5m2)
                xq, _ = fb.quantize_fp8_block(x[:T])
                want = xq.dequantize().double() @ q.dequantize().double().t()
                assert _off(fb.linear_fp8_block(x[:T], q), want) < 2.0 ** -8
                part = fb.Fp8BlockTensor(q.data[128:392], 512, q.scales[:, 128:392], e5m2)
                assert _off(fb.linear_fp8_block(x[:T], part), want[:, 128:392]) < 2.0 ** -8
                gu = want.to(torch.bfloat16).double()
                h = (torch.nn.functional.silu(gu[:, :256]) * gu[:, 256:]).to(torch.bfloat16)
                y = fb.gated_mlp_fp8_block(x[:T], q, None, d)
                assert _off(y, _value(h, 1, 128) @ d.dequantize().double().t()) < 2.0 ** -7
    nv.check_status()


@pytest.mark.parametrize("M,N,K", [(5, 136, 272), (300, 264, 640), (1500, 2056, 640)])
def test_outputs_that_start_anywhere(M, N, K):
    a, _ = fb.quantize_fp8_block(_rand(M, K))
    b, _ = fb.quantize_fp8_block(_rand(N, K, seed=1), tile=True)
    for dt in (torch.bfloat16, torch.float32):
        wide = torch.full((M, N + 9), 7.0, dtype=dt, device="cuda")
        out = wide[:, 1:N + 1]
        fb.matmul_fp8_block(a, b, out=out)
        _check_product(out, a, b)
        assert (wide[:, 0] == 7).all() and (wide[:, N + 1:] == 7).all()


def test_gradients_that_are_no_plain_matrices():
    x, w = _rand(130, 256, spread=0.5).requires_grad_(), _rand(136, 256, seed=1, spread=0.3).requires_grad_()
    y = fb.linear_fp8_block(x, w)
    dy = _rand(136, 130, seed=2)
    got = torch.autograd.grad(y, (x, w), dy.t(), retain_graph=True)            # transposed
    want = torch.autograd.grad(y, (x, w), dy.t().contiguous(), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)              # one value, expanded
    want = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_result_depends_on_timing():
    x, w = _rand(3000, 1040, spread=1.0).requires_grad_(), _rand(520, 1040, seed=1, spread=0.5).requires_grad_()
    b, dy = _rand(520, seed=2, spread=0.5).requires_grad_(), _rand(3000, 520, seed=3, spread=1.0)
    first = None
    for _ in range(4):
        out = torch.autograd.grad(fb.linear_fp8_block(x, w, b), (x, w, b), dy)
        torch.cuda.synchronize()
        first = first or out
        assert all(torch.equal(a, c) for a, c in zip(first, out))


def test_on_a_stream_of_its_own_and_from_two_threads():
    import threading

    x, w = _rand(700, 512, spread=1.0), _rand(1024, 512, seed=1, spread=0.5)
    want = fb.linear_fp8_block(x, w)
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s), torch.no_grad():
            for _ in range(10):
                got[i] = fb.linear_fp8_block(x, w)
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("T", [9, 1500])
def test_captured_and_replayed(T):
    x, w, wd = _rand(T, 256, spread=0.5), _rand(2048, 256, seed=1, spread=0.3) * 0.06, _rand(256, 1024, seed=2, spread=0.3) * 0.03
    kept = [fb.quantize_fp8_block(t, tile=True)[0] for t in (w, wd)]
    new = _rand(T, 256, seed=5, spread=0.5)
    with torch.no_grad():
        want = [fb.gated_mlp_fp8_block(v, kept[0], None, kept[1]) for v in (x, new)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            fb.gated_mlp_fp8_block(x, kept[0], None, kept[1])
        torch.cuda.current_stream().wait_stream(s)
        g = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        out = []
        for graph in g:
            with torch.cuda.graph(graph):
                out.append(fb.gated_mlp_fp8_block(x, kept[0], None, kept[1]))
        for graph, o in zip(g, out):
            graph.replay()
            assert torch.equal(o, want[0])
        x.copy_(new)
        for graph in g:
            graph.replay()
        assert torch.equal(out[0], want[1]) and torch.equal(out[1], want[1])


def test_training_step_captured_and_replayed():
    x, w, dy = _rand(300, 256, spread=0.5), _rand(512, 256, seed=1, spread=0.3), _rand(300, 512, seed=2, spread=1.0)
    x.requires_grad_(), w.requires_grad_()
    step = lambda: torch.autograd.grad(fb.linear_fp8_block(x, w), (x, w), dy)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    nv.check_status()


def test_rows_behind_the_last_do_not_matter():
    """A batch padded to a longer one: its own rows are what they are without the padding."""
    x, w = _rand(200, 512, spread=1.0), _rand(256, 512, seed=1, spread=0.5)
    q, _ = fb.quantize_fp8_block(w, tile=True)
    wide = torch.full((333, 512), float("nan"), device="cuda", dtype=torch.bfloat16)
    wide[:200] = x
    with torch.no_grad():
        assert torch.equal(fb.linear_fp8_block(wide, q)[:200], fb.linear_fp8_block(x, q))


# ------------------------------------------------------------------------------------------------
# Models
# ------------------------------------------------------------------------------------------------
def test_a_run_through_models_training_and_encoding():
    """The recipe in the engine, its gradients beside the bf16 ones, and the trained kind of model encoding with kept
    weights."""
    from lset_b200.models import Qwen3Config
    from lset_b200.train.data.collator import PackedCollator
    from lset_b200.train.data.dataset import SyntheticPairDataset
    from lset_b200.train.engine import TrainingEngine
    from lset_b200.train.quantization.fp8 import Float8Linear, Fp8KeptLinear, apply_fp8_inference

    cfg = Qwen3Config(vocab_size=2048, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=128)
    ds = SyntheticPairDataset(64, 2048, (8, 24), (40, 200), seed=3)
    batch = PackedCollator()([ds[i] for i in range(8)])

    def engine(fused, **kw):
        torch.manual_seed(0)
        return TrainingEngine("qwen3", None, None, batch_size=8, lr=1e-3, packed=True, model_config=cfg,
                              log_interval=0, scheduler_type="constant", fused_projections=fused, device="cuda", **kw)

    for fused in (True, False):
        ref, eng = engine(fused), engine(fused, fp8=True, fp8_recipe="block128")
        assert sum(isinstance(m, Float8Linear) for m in eng.model.modules()) == (8 if fused else 14)
        l_ref, l_fp8 = float(ref.forward_backward(batch, True)), float(eng.forward_backward(batch, True))
        nv.check_status()
        assert abs(l_fp8 - l_ref) < 0.1 * max(1.0, abs(l_ref))
        flat = lambda e: torch.cat([g.flat_grad.float().cpu() for g in e.store.groups])  # noqa: E731
        # an e4m3 value is off by 2^-4 / sqrt(3) of itself in the mean: a few percent a product, over two layers
        assert torch.nn.functional.cosine_similarity(flat(eng), flat(ref), dim=0).item() > 0.95
        eng.optimizer_step()

    model = ref.model.eval()
    ids = torch.randint(0, 2048, (3, 50), device="cuda")
    with torch.no_grad():
        want = model(ids)["hidden_states"].float()
        apply_fp8_inference(model)
        got = model(ids)["hidden_states"].float()
    assert sum(isinstance(m, Fp8KeptLinear) for m in model.modules()) == 2 * 6
    assert torch.nn.functional.cosine_similarity(got, want, dim=-1).min().item() > 0.97
    nv.check_status()


# ------------------------------------------------------------------------------------------------
# Sums
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,H,I", [(1024, 8192, 1024), (1000, 2560, 2048), (2600, 2048, 1024), (64, 4096, 4096)])
@pytest.mark.parametrize("kind", ["swiglu", "geglu"])
def test_what_a_step_rounds_twice_is_summed_as_in_32_bits(T, H, I, kind):
    """Gate and up products are rounded to bf16 and, as gradients, to 8 bits, where a sum on the wrong side of a border
    moves a value by 2^-4 of itself. So no more of them may fall on another side than 64 bits put them than of sums in
    plain fp32: half as many again, and six standard deviations of such a count."""
    x, w, wd = _rand(T, H, spread=0.5), _rand(2 * I, H, seed=1, spread=0.3) * H ** -0.5, _rand(H, I, seed=2, spread=0.3)
    y = fb.gated_mlp_fp8_block(x, w.requires_grad_(), None, wd, kind)
    nv.check_status()
    saved = y.grad_fn.saved_tensors[-1]                   # gate and up products come first in it
    gu = saved[:4 * T * I].view(torch.bfloat16).view(T, 2 * I)
    xv, wv = _value(x, 1, 128), _value(w, 128, 128)
    exact = (xv @ wv.t()).to(torch.float32).to(torch.bfloat16)
    plain = int(((xv.float() @ wv.float().t()).to(torch.bfloat16) != exact).sum())
    own = int((gu != exact).sum())
    assert own <= 1.5 * plain + 6 * max(plain, 1) ** 0.5, (own, plain)


@pytest.mark.parametrize("T", [40, 3000])
def test_gradients_of_a_deep_step_against_64_bits(T):
    """The gradient of gate and up, in an fp32 accumulator, beside the formula's in 64 bits: no further off than where the
    sums in front of the two roundings are plain fp32 ones, twice that and what its own sums add."""
    H, I = 8192, 512
    x, dy = _rand(T, H, spread=0.5), _rand(T, H, seed=1, spread=1.0)
    w, wd = _rand(2 * I, H, seed=2, spread=0.3) * H ** -0.5, _rand(H, I, seed=3, spread=0.3) * I ** -0.5
    w.requires_grad_()
    w.main_grad = torch.zeros(2 * I, H, device="cuda")
    fb.gated_mlp_fp8_block(x, w, None, wd).backward(dy)
    nv.check_status()

    def gradient(dtype):
        xv, wv, dv, yv = (_value(*a).to(dtype) for a in ((x, 1, 128), (w, 128, 128), (wd, 128, 128), (dy, 1, 128)))
        gu, dh = (xv @ wv.t()).to(torch.bfloat16).to(dtype), (yv @ dv).to(torch.bfloat16).to(dtype)
        g, u = gu.chunk(2, dim=1)
        s = 1 / (1 + torch.exp(-g))
        d = torch.cat([dh * u * s * (1 + g * (1 - s)), dh * g * s], dim=1).to(torch.bfloat16)
        return _value(d, 128, 1).t() @ _value(x, 128, 1)

    want = gradient(torch.float64)
    assert _off(w.main_grad, want) <= 2 * _off(gradient(torch.float32), want) + (T // 32 + 3) * 2.0 ** -22


@pytest.mark.parametrize("kind", ["swiglu", "geglu"])
@pytest.mark.parametrize("T", [24, None])
def test_activation_and_derivative_of_every_gate(kind, T):
    """Gates of every bf16 value from 2^-40 to 2^20 (the upper and the lower half of the bits lie in blocks of their own,
    so nothing is rounded on the way to the product), up projections of 1. y is 2^67 times act(g) in 8 bits, the gradient
    of x's first column 128 times the derivative."""
    bits = torch.arange((127 - 40) << 7, (127 + 20) << 7, device="cuda", dtype=torch.int32)
    g = (torch.cat([bits, bits | 0x8000]) << 16).view(torch.float32)
    if T is not None:       # gates whose sigmoid is far from 0 and 1, and at its lower end
        near = torch.tensor([-88.5, -88, -87.5, -87, -60, -17, -5, -3, -1, -0.5, 0.5, 3], device="cuda")
        g = torch.cat([near, torch.linspace(-4, 4, T - 12, device="cuda").to(torch.bfloat16).float()])
    low = (g.view(torch.int32) & 0x000F0000) != 0
    top = (g.view(torch.int32) & ~0x000FFFFF).view(torch.float32)
    x = torch.zeros(len(g), 384, device="cuda")
    x[:, 0], x[:, 128], x[:, 256] = top, torch.where(low, g - top, torch.zeros_like(g)), 1
    w = torch.zeros(256, 384, device="cuda")
    w[:128, 0] = w[:128, 128] = w[128:, 256] = 1
    wd, dy = torch.zeros(384, 128, device="cuda"), torch.zeros(len(g), 384, device="cuda")
    wd[0], dy[:, 0] = 2.0 ** 60, 2.0 ** -60
    x, w, wd, dy = (t.to(torch.bfloat16).requires_grad_() for t in (x, w, wd, dy))
    y = fb.gated_mlp_fp8_block(x, w, None, wd, kind)
    (dx,) = torch.autograd.grad(y, x, dy)
    nv.check_status()
    if kind == "swiglu":
        s = 1 / (1 + torch.exp(-g))
        a, da = g * s, s * (1 + g * (1 - s))
        v = g.double()
        s = 1 / (1 + torch.exp(-v))
        exact = v * s, s * (1 + v * (1 - s))
    else:
        c, k = 0.7978845608028654, 0.044715
        t = torch.tanh(c * (g + k * g * g * g))
        a, da = 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * k * g * g)
        exact = None
    for i, (got, plain) in enumerate(((y[:, 0].double() * 2.0 ** -67, a), (dx[:, 0].double() / 128, da))):
        want = _value(plain.to(torch.bfloat16).view(-1, 1).expand(-1, 8), 1, 128)[:, 0]
        # the formula in 32 bits, operation by operation, as far as the sigmoid is not 0 (below -87.3). Gates below -1, one in
        # 16 here, have it off by up to 2^-24 |g| of itself, 2^-18: between bf16 values 2^-8 apart one in 2^9 then falls
        # to another side, and of those one in 2^4 in 8 bits, which have 16 steps of bf16 to one of their own.
        some = g >= -87.25
        assert int((got != want)[some].sum()) <= 3 + len(g) * 2.0 ** -17, int((got != want)[some].sum())
        assert (got[~some].abs() <= 2.0 ** -116).all()
        if exact is not None:
            e, v = exact[i][some], got[some]
            # 1 - s and 1 + g (1 - s) cancel next to the derivative's zero: an absolute error there
            assert ((v - e).abs() <= (2.0 ** -4 + 2.0 ** -8) * e.abs() + 2.0 ** -20 * (e.abs() > 2.0 ** -30)).all()


# contractions that CTA pairs split over several products in fp32 (few tiles, great depth), ragged ones among them
SPLIT = [(333, 1024, 8192), (300, 1016, 8328), (1000, 512, 9728), (700, 776, 16392), (1024, 1024, 16384)]


@pytest.mark.parametrize("M,N,K", SPLIT)
def test_split_products_with_bias(M, N, K):
    assert fb._product_bytes(M, N, K, N) >= 2 * 4 * M * N
    a, _ = fb.quantize_fp8_block(_rand(M, K, spread=1.0))
    b, _ = fb.quantize_fp8_block(_rand(N, K, seed=1, spread=1.0), tile=True)
    wide = _rand(N + 1, spread=0.5) * K ** 0.5
    for bias in (wide[:N], wide[1:]):      # the second at no multiple of 4 bytes
        for dt in (torch.bfloat16, torch.float32):
            _check_product(fb.matmul_fp8_block(a, b, bias=bias, out_dtype=dt), a, b, bias)
    nv.check_status()


@pytest.mark.parametrize("T,N,K", [(333, 1024, 8192), (1000, 512, 9728)])
def test_split_layers_with_bias(T, N, K):
    x, w, b = _rand(T, K, spread=1.0), _rand(N, K, seed=1, spread=0.5), _rand(N, seed=2, spread=0.5) * K ** 0.5
    xq, _ = fb.quantize_fp8_block(x)
    wq, _ = fb.quantize_fp8_block(w, tile=True)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    y = fb.linear_fp8_block(x, w, b)
    _check_product(y.detach(), xq, wq, b.detach())
    dy = _rand(T, N, seed=3)
    (db,) = torch.autograd.grad(y, b, dy)
    assert ((db.double() - dy.double().sum(0)).abs()
            <= 2.0 ** -8 * dy.double().sum(0).abs() + T * 2.0 ** -24 * dy.double().abs().sum(0)).all()
    with torch.no_grad():
        assert torch.equal(fb.linear_fp8_block(x, wq, b), y)
    nv.check_status()


def test_copies_of_kept_weights_are_on_memory_of_their_own():
    import copy
    import pickle

    x = _rand(20, 512, spread=0.5)
    q, _ = fb.quantize_fp8_block(_rand(256, 512, seed=1, spread=0.3), tile=True)
    with torch.no_grad():
        want = fb.linear_fp8_block(x, q)
        for c in (copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
            q.data.zero_(), q.scales.fill_(127)
            assert c.data.is_cuda and torch.equal(fb.linear_fp8_block(x, c), want)
            q.data.copy_(c.data), q.scales.copy_(c.scales)
        other, _ = fb.quantize_fp8_block(_rand(256, 512, seed=2, spread=0.3), tile=True)
        q.data.data, q.scales.data = other.data, other.scales
        assert torch.equal(fb.linear_fp8_block(x, q), fb.linear_fp8_block(x, other))
        q.scales.data = torch.zeros(1025, dtype=torch.uint8, device="cuda")[1:].view(1, 256, 4)
        with pytest.raises(ValueError, match="multiples of"):
            fb.linear_fp8_block(x, q)


def test_the_gated_kernel_is_chosen_where_it_is_the_faster():
    """Its tiles run whole, whatever is left for the last wave: 64 rows of 9728 on 2560 take it 22.6 us for 18.4 of a
    product and an activation (whose products then have storage), 500 of 4096 on 1024 10.3 for 15.8."""
    assert fb._mlp_kept_bytes(64, 2560, 9728) >= 4 * 64 * 9728
    assert fb._mlp_kept_bytes(500, 1024, 4096) < 4 * 500 * 4096


def _sums(a, b, depth):
    """What fp32 sums of |a| |b|ᵀ that deep may be off (_check_product says why)."""
    return (depth // 32 + 3) * 2.0 ** -22 * (a.abs() @ b.abs().t())


@pytest.mark.parametrize("T", [1, 5, 129, 700])
@pytest.mark.parametrize("bias_type", [torch.float32, torch.bfloat16])
def test_values_of_an_fp32_linear_layer(T, bias_type):
    """fp32 activations and weights: operands are rounded to bf16 on their way to 8 bits, results are fp32, and the
    gradient of the bias is the sum of dy as it comes."""
    K, N = 272, 136
    g = torch.Generator("cuda").manual_seed(T)
    x, w, dy = (torch.randn(*s, generator=g, device="cuda") for s in ((T, K), (N, K), (T, N)))
    b = torch.randn(N, generator=g, device="cuda").to(bias_type)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = fb.linear_fp8_block(x, w, b)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    nv.check_status()
    xr, xc, dr, dc, wv = _value(x, 1, 128), _value(x, 128, 1), _value(dy, 1, 128), _value(dy, 128, 1), _value(w, 128, 128)
    bv = b.detach().to(torch.bfloat16).double()
    for got, want, off in ((y.detach(), xr @ wv.t() + bv, _sums(xr, wv, K)), (dx, dr @ wv, _sums(dr, wv.t(), N)),
                           (dw, dc.t() @ xc, _sums(dc.t(), xc.t(), T))):
        assert got.dtype == torch.float32
        assert ((got.double() - want).abs() <= 2.0 ** -23 * want.abs() + off).all()
    want = dy.double().sum(0)
    assert db.dtype == bias_type
    half = 2.0 ** -8 if bias_type is torch.bfloat16 else 2.0 ** -23
    assert ((db.double() - want).abs() <= half * want.abs() + (130 + T // 128) * 2.0 ** -24 * dy.double().abs().sum(0)).all()
    (only,) = torch.autograd.grad(fb.linear_fp8_block(x, w, b), b, dy.expand(T, N))
    assert torch.equal(only, db)
    (ones,) = torch.autograd.grad(fb.linear_fp8_block(x, w, b).sum(), b)
    assert (ones == T).all()


@pytest.mark.parametrize("T", [1, 130])
def test_values_of_an_fp32_gated_block(T):
    """fp32 activations, weights and accumulators: what bf16 ones of the same values give, rounded to bf16 in between."""
    H, I = 264, 256
    x, dy = _rand(T, H, spread=0.5), _rand(T, H, seed=1, spread=1.0)
    w, wd = _rand(2 * I, H, seed=2, spread=0.3) * H ** -0.5, _rand(H, I, seed=3, spread=0.3) * I ** -0.5
    leaves = [t.requires_grad_() for t in (x, w, wd)]
    y = fb.gated_mlp_fp8_block(x, w, None, wd)
    want = torch.autograd.grad(y, leaves, dy)
    fp32 = [t.detach().float().requires_grad_() for t in leaves]
    z = fb.gated_mlp_fp8_block(fp32[0], fp32[1], None, fp32[2])
    got = torch.autograd.grad(z, fp32, dy.float())
    assert z.dtype == torch.float32 and torch.equal(z, y.float()) and torch.equal(got[0], want[0].float())
    for a, b in zip(got[1:], want[1:]):      # fp32 sums, and those rounded to bf16
        assert a.dtype == torch.float32 and torch.equal(a.to(torch.bfloat16), b)
    for t in leaves[1:]:
        t.main_grad = torch.full(t.shape, 2.0, device="cuda")
    fb.gated_mlp_fp8_block(x, w, None, wd).backward(dy)
    for t, a in zip(leaves[1:], got[1:]):    # added to what is there: half a step of the sum's type
        assert t.grad is None and ((t.main_grad - 2 - a).abs() <= 2.0 ** -23 * (2 + a.abs())).all()
    nv.check_status()


@pytest.mark.parametrize("M,N,K", SPLIT)
def test_split_products_into_given_outputs(M, N, K):
    a, _ = fb.quantize_fp8_block(_rand(M, K, spread=1.0))
    b, _ = fb.quantize_fp8_block(_rand(N, K, seed=1, spread=1.0), tile=True)
    for dt in (torch.bfloat16, torch.float32):
        wide = torch.full((M + 2, N + 24), 7.0, dtype=dt, device="cuda")
        out = wide[1:M + 1, 8:N + 8]
        assert fb._product_bytes(M, N, K, N + 24) >= 2 * 4 * M * N
        fb.matmul_fp8_block(a, b, out=out)
        _check_product(out, a, b)
        out.fill_(7)
        assert (wide == 7).all()                 # nothing around it
    base = torch.randn(M, N, device="cuda") * K ** 0.5
    out = base.clone()
    fb.matmul_fp8_block(a, b, out=out, accumulate=True)
    _check_product(out, a, b, base=base)
    nv.check_status()


def test_split_weight_gradients_of_a_long_batch():
    T, K, N = 16384, 768, 768
    assert fb._product_bytes(N, K, T, K) >= 2 * 4 * N * K
    x, w, dy = _rand(T, K, spread=0.5), _rand(N, K, seed=1, spread=0.5), _rand(T, N, seed=2, spread=0.5)
    a, b = _value(dy, 128, 1).t(), _value(x, 128, 1).t()
    want, off = a @ b.t(), _sums(a, b, T)
    x.requires_grad_(), w.requires_grad_()
    y = fb.linear_fp8_block(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    assert ((dw.double() - want).abs() <= 2.0 ** -8 * want.abs() + off).all()
    wv, dr = _value(w, 128, 128), _value(dy, 1, 128)
    assert ((dx.double() - dr @ wv).abs() <= 2.0 ** -8 * (dr @ wv).abs() + _sums(dr, wv.t(), N)).all()
    w.main_grad = torch.full((N, K), 3.0, device="cuda")
    for n in (1, 2):
        y.backward(dy, retain_graph=True)
        assert w.grad is None
        assert ((w.main_grad.double() - 3 - n * want).abs() <= n * (2.0 ** -23 * (3 + n * want.abs()) + off)).all()
    nv.check_status()


@pytest.mark.parametrize("T", [1, 17, 129, 1000, 2600])
@pytest.mark.parametrize("K,N,bias", [(136, 264, True), (640, 72, True), (2568, 1032, False)])
def test_linear_layers_value_by_value(T, K, N, bias):
    x, w, dy = _rand(T, K, spread=1.0), _rand(N, K, seed=1, spread=0.5), _rand(T, N, seed=2, spread=1.0)
    b = _rand(N, seed=3, spread=0.5) if bias else None
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = fb.linear_fp8_block(x, w, b)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    nv.check_status()
    xr, xc, dr, dc, wv = _value(x, 1, 128), _value(x, 128, 1), _value(dy, 1, 128), _value(dy, 128, 1), _value(w, 128, 128)
    want = [(xr @ wv.t() + (0 if b is None else b.detach().double()), _sums(xr, wv, K)), (dr @ wv, _sums(dr, wv.t(), N)),
            (dc.t() @ xc, _sums(dc.t(), xc.t(), T))]
    if bias:
        want.append((dy.double().sum(0), (130 + T // 128) * 2.0 ** -24 * dy.double().abs().sum(0)))
    for a, (c, off) in zip(got, want):
        assert ((a.double() - c).abs() <= 2.0 ** -8 * c.abs() + off).all()


def _rows_close(got, a, b, flips=2):
    """Each row of ``got`` beside ``a @ b``: half a step of bf16, what its sums may be off, and ``flips`` values of a's row that
    fell to the other side of a rounding to 8 bits, by 2^-3 of themselves."""
    want = a @ b
    off = ((a.shape[1] // 32 + 3) * 2.0 ** -22) * (a.abs() @ b.abs())
    one = (a.abs() * b.norm(dim=1)).amax(dim=1)
    bound = 2.0 ** -8 * want.norm(dim=1) + off.norm(dim=1) + flips * 2.0 ** -3 * one
    err = (got.double() - want).norm(dim=1)
    assert (err <= bound).all(), (int((err > bound).sum()), float((err / bound).max()))


@pytest.mark.parametrize("kind", ["swiglu", "geglu"])
@pytest.mark.parametrize("T,H,I", [(1, 264, 384), (33, 1032, 256), (129, 2568, 128), (333, 1152, 1280), (1500, 4104, 640),
                                   (2600, 2048, 1024), (4097, 1288, 2432)])
def test_gated_blocks_row_by_row(T, H, I, kind):
    """Sums of one part and of several, few rows and many, ragged widths; gate and up products value by value, the rest by rows
    (of weight gradients, by features)."""
    x, dy = _rand(T, H, spread=0.5), _rand(T, H, seed=1, spread=0.5)
    w, wd = _rand(2 * I, H, seed=2, spread=0.3) * H ** -0.5, _rand(H, I, seed=3, spread=0.3) * I ** -0.5
    leaves = [t.requires_grad_() for t in (x, w, wd)]
    y = fb.gated_mlp_fp8_block(x, w, None, wd, kind)
    gu = y.grad_fn.saved_tensors[-1][:4 * T * I].view(torch.bfloat16).view(T, 2 * I).clone()
    dx, dw, dwd = torch.autograd.grad(y, leaves, dy)
    nv.check_status()
    xr, xc, wv, dv = _value(x, 1, 128), _value(x, 128, 1), _value(w, 128, 128), _value(wd, 128, 128)
    dr, dc = _value(dy, 1, 128), _value(dy, 128, 1)
    want = xr @ wv.t()
    assert ((gu.double() - want).abs() <= 2.0 ** -8 * want.abs() + _sums(xr, wv, H)).all()
    leaf = gu.float().requires_grad_()
    g, u = leaf[:, :I], leaf[:, I:]
    act = torch.nn.functional.silu(g) if kind == "swiglu" else 0.5 * g * (
        1 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g)))
    h = act * u
    dh = (dr @ dv).to(torch.bfloat16).float()
    (dgu,) = torch.autograd.grad(h, leaf, dh)
    hb, db = h.detach().to(torch.bfloat16), dgu.to(torch.bfloat16)
    _rows_close(y.detach(), _value(hb, 1, 128), dv.t())
    _rows_close(dx, _value(db, 1, 128), wv)
    _rows_close(dw, _value(db, 128, 1).t(), xc)
    _rows_close(dwd.t(), _value(hb, 128, 1).t(), dc)
    with torch.no_grad():
        kept = [fb.quantize_fp8_block(t, tile=True)[0] for t in (w, wd)]
        z = fb.gated_mlp_fp8_block(x, kept[0], None, kept[1], kind)
    if H <= 1024:
        assert torch.equal(z, y)       # (deeper, a step's gate and up are sums of parts)
    _rows_close(z, _value(hb, 1, 128), dv.t(), flips=4)


def test_a_deep_training_step_captured_and_replayed_on_another_stream():
    T, H, I = 1300, 2056, 256
    x, dy = _rand(T, H, spread=0.5), _rand(T, H, seed=1, spread=0.5)
    w, wd = _rand(2 * I, H, seed=2, spread=0.3) * H ** -0.5, _rand(H, I, seed=3, spread=0.3) * I ** -0.5
    x.requires_grad_(), w.requires_grad_(), wd.requires_grad_()
    step = lambda: torch.autograd.grad(fb.gated_mlp_fp8_block(x, w, None, wd), (x, w, wd), dy)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    nv.check_status()


@pytest.mark.parametrize("fused", [True, False])
def test_a_run_through_models_checkpointed_and_captured(fused):
    """Recomputed forwards write the gradients that kept ones do; an encoder on kept weights replays from a graph."""
    from lset_b200.models import Qwen3Config
    from lset_b200.train.cuda_graph import CUDAGraphWrapper
    from lset_b200.train.data.collator import PackedCollator
    from lset_b200.train.data.dataset import SyntheticPairDataset
    from lset_b200.train.engine import TrainingEngine
    from lset_b200.train.quantization.fp8 import apply_fp8_inference

    cfg = Qwen3Config(vocab_size=2048, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=128)
    ds = SyntheticPairDataset(64, 2048, (8, 24), (40, 200), seed=3)
    batch = PackedCollator()([ds[i] for i in range(8)])
    grads = []
    for kw in ({}, dict(activation_checkpoint=True, ac_mode="full"), dict(activation_checkpoint=True, ac_mode="selective")):
        torch.manual_seed(0)
        eng = TrainingEngine("qwen3", None, None, batch_size=8, lr=1e-3, packed=True, model_config=cfg, log_interval=0,
                             scheduler_type="constant", fused_projections=fused, device="cuda", fp8=True,
                             fp8_recipe="block128", **kw)
        eng.forward_backward(batch, True)
        nv.check_status()
        grads.append({n: p.main_grad.clone() for n, p in eng.model.named_parameters()})
    for name, want in grads[0].items():
        assert want.abs().sum() > 0
        for got in (grads[1][name], grads[2][name]):
            # norms and the embedding are added up with atomics, in another order each time, whatever the layers are
            assert torch.equal(got, want) if "_proj" in name else _off(got, want.double()) < 2.0 ** -20, name

    model = apply_fp8_inference(TrainingEngine("qwen3", None, None, batch_size=8, packed=True, model_config=cfg,
                                               log_interval=0, fused_projections=fused, device="cuda").model.eval())
    ids = torch.randint(0, 2048, (3, 64), device="cuda")
    with torch.no_grad():
        graph = CUDAGraphWrapper(model, 3, 64, "cuda")
        for _ in range(2):
            assert torch.equal(graph(ids)["hidden_states"], model(ids)["hidden_states"])
            ids = ids.flip(0)
    nv.check_status()

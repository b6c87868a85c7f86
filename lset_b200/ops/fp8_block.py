"""8-bit float products with one power-of-two scale for each block of 128, and the layers built on them.

``quantize_fp8_block`` casts a bf16 matrix to e4m3 (or e5m2) in blocks: runs of 128 values along a row for
activations and gradients, 128 x 128 tiles for weights (the same values then serve the forward product and, in
the transposed copy, the input gradient). ``matmul_fp8_block`` multiplies two such matrices on the tensor cores
(``tcgen05.mma kind::mxf8f6f4.block_scale``: the scales enter the product there, sums are fp32).
``linear_fp8_block`` is the linear layer: its three products with operands cast along their own contraction.
``gated_mlp_fp8_block`` is the gated feed-forward block: the activation's result is cast where it is computed, and
one pass over the activations of the backward casts the operands of its three products.

A block's scale is ``2^e`` with the smallest ``e`` for which its largest magnitude is at most 448 (57344 in
e5m2) times it: scaling is exact and a value is rounded once, to nearest even. A block of zeros has the scale 1; a
block that holds a NaN or an infinity is NaN throughout.

On the CPU the same arithmetic runs in plain PyTorch. Beside ``ops/fp8.py``, whose scales are those of a tensor,
a row or a column; the recipe ``block128`` of ``train/quantization/fp8.py`` selects these layers.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import _native as nv
from .activation import glu_ref
from ._grads import main_grad_of

BLOCK = 128
E4M3_MAX, E5M2_MAX = 448.0, 57344.0


@dataclass
class Fp8BlockTensor:
    """A matrix ``[rows, cols]`` in 8 bits: ``data`` ``[rows, ld]`` bytes (the first ``cols`` of a row are
    valid; ``ld`` a multiple of 16), ``scales`` ``[ceil(cols / 512), rows, 4]`` bytes: ``scales[b // 4, r,
    b % 4]`` is the exponent, biased by 127, of the scale of columns ``128 b .. 128 b + 127`` of row ``r``."""
    data: torch.Tensor
    cols: int
    scales: torch.Tensor
    e5m2: bool = False

    @property
    def rows(self) -> int:
        return self.data.shape[0]

    @property
    def shape(self):
        return (self.data.shape[0], self.cols)

    def dequantize(self) -> torch.Tensor:
        """The values, in fp32."""
        q = self.data[:, :self.cols].view(torch.float8_e5m2 if self.e5m2 else torch.float8_e4m3fn)
        e = self.scales.transpose(0, 1).reshape(self.rows, 4 * self.scales.shape[0]).int()
        s = (e << 23).view(torch.float32).repeat_interleave(BLOCK, dim=1)[:, :self.cols]
        return q.float() * s

    def check(self, what: str) -> None:
        d, s = self.data, self.scales
        if d.dim() != 2 or d.dtype != torch.uint8 or s.dim() != 3 or s.dtype != torch.uint8:
            raise TypeError(f"{what}: data is a 2-D and scales a 3-D tensor of bytes")
        if not 0 <= self.cols <= d.shape[1] or tuple(s.shape) != (-(-self.cols // 512), d.shape[0], 4):
            raise ValueError(f"{what}: data {tuple(d.shape)} with {self.cols} columns and scales "
                             f"{tuple(s.shape)} do not belong together")
        if (d.stride(1) != 1 and d.shape[1] > 1) or (d.shape[0] > 1 and d.stride(0) < self.cols):
            raise ValueError(f"{what}: the bytes of a row lie next to one another")
        if d.is_cuda and d.numel() and (_row_bytes(d) % 16 or d.data_ptr() % 16):
            raise ValueError(f"{what}: rows start at multiples of 16 bytes")
        if not s[0].is_contiguous() if s.shape[0] else False:
            raise ValueError(f"{what}: the scales of four blocks lie next to one another, row by row")
        if s.device != d.device:
            raise ValueError(f"{what}: data and scales are on one device")


def _row_bytes(d: torch.Tensor) -> int:
    """Bytes between two rows (of a single row: enough of them)."""
    return d.stride(0) if d.shape[0] > 1 else (d.shape[1] + 15) // 16 * 16


def _scale_rows(s: torch.Tensor) -> int:
    """Words between the scales of one group of four blocks and the next."""
    return s.stride(0) // 4 if s.shape[0] > 1 else s.shape[1]


# ------------------------------------------------------------------------------------------------
# Calls into the library
# ------------------------------------------------------------------------------------------------
_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
_SIGNATURES = {
    "lb_block_cast": [_P, _I, _I, _L, _I, _I, _P, _L, _P, _L, _P, _L, _P, _L, _I, _P],
    "lb_block_glu_fwd": [_I, _P, _P, _L, _I, _I, _P, _L, _P, _L, _P],
    "lb_block_glu_bwd": [_I, _P, _L, _P, _P, _L, _I, _I] + 3 * [_P, _L, _P, _L] + [_P],
    "lb_gemm_block": [_P, _P, _P, _I, _I, _I, _L, _L, _L, _I, _I, _P, _L, _P, _L, _I, _I, _P, _P, _P],
}
_fns = {}


def _fn(name):
    """A launcher with its argument types set: plain numbers then pass without a wrapper each."""
    f = _fns.get(name)
    if f is None:
        f = getattr(nv.load(), name)
        f.argtypes, f.restype = _SIGNATURES[name], _I
        _fns[name] = f
    return f


def _on_device(*tensors):
    """The tensors' one CUDA device as a context; launches go to the current stream of that device."""
    dev = None
    for t in tensors:
        if t is not None:
            if dev is not None and t.device != dev:
                raise ValueError(f"operands are on {dev} and {t.device}")
            dev = t.device
    return torch.cuda.device(dev)


# ------------------------------------------------------------------------------------------------
# Casts
# ------------------------------------------------------------------------------------------------
def _eager_blocks(x, rows, cols, e5m2):
    """Bytes and exponents of ``x`` in blocks of ``rows x cols``, exponents one for each row and block."""
    R, C = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -C % cols, 0, -R % rows))
    v = v.view(v.shape[0] // rows, rows, v.shape[1] // cols, cols)
    amax = v.abs().nan_to_num(nan=float("inf"), posinf=float("inf")).amax(dim=(1, 3), keepdim=True)
    bits = amax.view(torch.int32)
    e = ((bits >> 23) - (15 if e5m2 else 8) + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(1, 254)
    bad = ~torch.isfinite(amax)
    e = torch.where((amax == 0) | bad, torch.full_like(e, 127), e)
    q = v * ((254 - e) << 23).view(torch.float32)
    q = q.to(torch.float8_e5m2 if e5m2 else torch.float8_e4m3fn).view(torch.uint8)
    q = torch.where(bad, torch.full_like(q, 0x7F), q)
    return q.reshape(v.shape[0] * rows, -1)[:R, :C], e[:, 0, :, 0]


def _pack(q, e):
    """The ``Fp8BlockTensor`` layout of bytes ``[rows, cols]`` and exponents ``[rows, blocks]``."""
    R, C = q.shape
    data = torch.zeros(R, (C + 15) // 16 * 16, dtype=torch.uint8, device=q.device)
    data[:, :C] = q
    words = torch.nn.functional.pad(e.to(torch.uint8), (0, -e.shape[1] % 4), value=127)
    return data, words.reshape(R, -1, 4).transpose(0, 1).contiguous()


def _quantize_eager(x, tile, e5m2, want, want_t):
    R, C = x.shape
    if x.numel() == 0:
        return (_empty(R, C, e5m2, x.device) if want else None), (_empty(C, R, e5m2, x.device) if want_t else None)
    x = x.to(torch.bfloat16)
    out = out_t = None
    if tile:
        q, e = _eager_blocks(x, BLOCK, BLOCK, e5m2)
        if want:
            d, s = _pack(q, e.repeat_interleave(BLOCK, dim=0)[:R])
            out = Fp8BlockTensor(d, C, s, e5m2)
        if want_t:
            d, s = _pack(q.t(), e.t().repeat_interleave(BLOCK, dim=0)[:C])
            out_t = Fp8BlockTensor(d, R, s, e5m2)
        return out, out_t
    if want:
        d, s = _pack(*_eager_blocks(x, 1, BLOCK, e5m2))
        out = Fp8BlockTensor(d, C, s, e5m2)
    if want_t:
        d, s = _pack(*_eager_blocks(x.t(), 1, BLOCK, e5m2))
        out_t = Fp8BlockTensor(d, R, s, e5m2)
    return out, out_t


def _empty(rows, cols, e5m2, device) -> Fp8BlockTensor:
    return Fp8BlockTensor(torch.empty(rows, (cols + 15) // 16 * 16, dtype=torch.uint8, device=device), cols,
                          torch.empty(-(-cols // 512), rows, 4, dtype=torch.uint8, device=device), e5m2)


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """``x`` [R, C] in bf16 with rows that a kernel can read in 16-byte pieces."""
    if x.dtype != torch.bfloat16:
        x = x.to(torch.bfloat16)
    if x.stride(1) != 1 or x.stride(0) % 8 or x.stride(0) < x.shape[1] or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _where(q: Optional[Fp8BlockTensor]):
    """A cast matrix as the launchers take it: bytes, their row stride, scale words, words of a group."""
    if q is None:
        return 0, 0, 0, 0
    return q.data.data_ptr(), _row_bytes(q.data), q.scales.data_ptr(), _scale_rows(q.scales)


def _cast_into(x, tile, e5m2, out: Optional[Fp8BlockTensor], out_t: Optional[Fp8BlockTensor]) -> None:
    R, C = x.shape
    rc = _fn("lb_block_cast")(x.data_ptr(), R, C, x.stride(0), tile, e5m2, *_where(out), *_where(out_t), 0,
                              nv.stream_ptr())
    if rc != 0:
        nv.check_rc(rc, f"lb_block_cast(R={R},C={C})")
    nv.count_launch()


def quantize_fp8_block(x: torch.Tensor, *, tile: bool = False, e5m2: bool = False, want: bool = True,
                       want_t: bool = False):
    """Cast a 2-D matrix ``x [R, C]`` (bf16; other types are rounded to it first) to 8 bits in blocks of 128.

    Returns ``(q, q_t)``, either None when not requested: ``q`` is ``x`` with one scale for each row and 128
    columns, ``q_t`` is ``xᵀ`` (``[C, R]``) with one for each column of ``x`` and 128 rows, so each is scaled
    along the dimension that a product contracts. ``tile``: both have the same values, one scale for each
    128 x 128 block of ``x``. On the GPU ``C`` is a multiple of 8.
    """
    if x.dim() != 2 or not x.is_floating_point():
        raise ValueError("quantize_fp8_block takes a 2-D matrix of floating-point values")
    if not nv.use_native(x):
        return _quantize_eager(x, tile, e5m2, want, want_t)
    R, C = x.shape
    if C % 8:
        raise ValueError("quantize_fp8_block needs a multiple of 8 columns")
    with _on_device(x):
        x = _aligned(x.detach())
        out = _empty(R, C, e5m2, x.device) if want else None
        out_t = _empty(C, R, e5m2, x.device) if want_t else None
        if R and C:
            _cast_into(x, tile, e5m2, out, out_t)
    return out, out_t


# ------------------------------------------------------------------------------------------------
# Products
# ------------------------------------------------------------------------------------------------
def _matmul(a: Fp8BlockTensor, b: Fp8BlockTensor, out: torch.Tensor, accumulate: bool, bias) -> None:
    """The product of checked operands on the current device."""
    M, N, K = a.data.shape[0], b.data.shape[0], a.cols
    rc = _fn("lb_gemm_block")(
        a.data.data_ptr(), b.data.data_ptr(), out.data_ptr(), M, N, K, _row_bytes(a.data), _row_bytes(b.data),
        out.stride(0) if M > 1 else N, a.e5m2, b.e5m2, a.scales.data_ptr(), _scale_rows(a.scales),
        b.scales.data_ptr(), _scale_rows(b.scales), out.dtype == torch.float32, accumulate,
        0 if bias is None else bias.data_ptr(), nv.status_word(out.device).data_ptr(), nv.stream_ptr())
    if rc != 0:
        nv.check_rc(rc, f"lb_gemm_block(M={M},N={N},K={K})")
    nv.count_launch()


def matmul_fp8_block(a: Fp8BlockTensor, b: Fp8BlockTensor, *, out: Optional[torch.Tensor] = None,
                     out_dtype=torch.bfloat16, accumulate: bool = False, bias=None) -> torch.Tensor:
    """``C[M, N] = A · Bᵀ (+ bias)`` of block-scaled ``a [M, K]`` and ``b [N, K]``, in bf16 or fp32.

    ``out`` may be given (rows of unit inner stride); ``accumulate`` adds into it (fp32, no bias). Sums are
    fp32 and their order depends on the sizes alone. e4m3 and e5m2 operands may be mixed.
    """
    a.check("a")
    b.check("b")
    M, N, K = a.rows, b.rows, a.cols
    if b.cols != K:
        raise ValueError(f"contraction mismatch: {K} vs {b.cols}")
    if out is not None:
        out_dtype = out.dtype
        if tuple(out.shape) != (M, N) or (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
            raise ValueError(f"out has to be [{M}, {N}] with neighbouring columns next to one another")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("output must be bf16 or fp32")
    if accumulate and (out is None or out_dtype != torch.float32 or bias is not None):
        raise ValueError("accumulate adds into a given fp32 output, without a bias")
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"bias has to be [{N}]")
    if not nv.use_native(a.data, b.data):
        c = a.dequantize() @ b.dequantize().t()
        if bias is not None:
            c = c + bias.to(torch.bfloat16).float()
        if out is None:
            return c.to(out_dtype)
        return out.add_(c) if accumulate else out.copy_(c)
    with _on_device(a.data, b.data, out, bias):
        if out is None:
            out = torch.empty(M, N, dtype=out_dtype, device=a.data.device)
        if M == 0 or N == 0:
            return out
        if K == 0:
            if not accumulate:
                out.zero_() if bias is None else out.copy_(bias.to(torch.bfloat16).expand(M, N))
            return out
        if bias is not None:
            bias = bias.to(torch.bfloat16).contiguous()
        _matmul(a, b, out, accumulate, bias)
    return out


# ------------------------------------------------------------------------------------------------
# Layers
# ------------------------------------------------------------------------------------------------
def _weight_gradient(w, a_t: Fp8BlockTensor, b_t: Fp8BlockTensor):
    """``dyᵀ · x`` into the weight's fp32 accumulator (returns None), or in the weight's type."""
    main = main_grad_of(w)
    if main is not None and a_t.data.is_cuda:
        matmul_fp8_block(a_t, b_t, out=main, accumulate=True)
        return None
    if w.dtype == torch.bfloat16:
        return matmul_fp8_block(a_t, b_t)
    return matmul_fp8_block(a_t, b_t, out_dtype=torch.float32).to(w.dtype)


class _LinearFp8Block(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias):
        x2 = x.reshape(-1, x.shape[-1])
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        xq, xq_t = quantize_fp8_block(x2, want_t=need_w)
        wq, wq_t = quantize_fp8_block(w, tile=True, want_t=need_x)
        ctx.shape, ctx.tokens, ctx.features = x.shape, x2.shape[0], w.shape
        ctx.act_dtype = x.dtype if x.dtype in (torch.bfloat16, torch.float32) else torch.bfloat16
        ctx.x_dtype, ctx.bias_dtype = x.dtype, None if bias is None else bias.dtype
        # the backward pass needs only the transposed 8-bit copies (and the weight as an address)
        ctx.save_for_backward(*((xq_t.data, xq_t.scales) if need_w else (None, None)),
                              *((wq_t.data, wq_t.scales) if need_x else (None, None)), w)
        y = matmul_fp8_block(xq, wq, out_dtype=ctx.act_dtype, bias=bias)
        return y.view(*x.shape[:-1], w.shape[0])

    @staticmethod
    def backward(ctx, dy):
        xt, xs, wt, ws, w = ctx.saved_tensors
        dy2 = dy.reshape(-1, dy.shape[-1])
        dx = dw = db = None
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        if need_x or need_w:
            dyq, dyq_t = quantize_fp8_block(dy2, want=need_x, want_t=need_w)
        if need_x:
            dx = matmul_fp8_block(dyq, Fp8BlockTensor(wt, ctx.features[0], ws), out_dtype=ctx.act_dtype)
            dx = dx.view(ctx.shape).to(ctx.x_dtype)
        if need_w:
            dw = _weight_gradient(w, dyq_t, Fp8BlockTensor(xt, ctx.tokens, xs))
        if ctx.bias_dtype is not None and ctx.needs_input_grad[2]:
            db = dy2.float().sum(0).to(ctx.bias_dtype)
        return dx, dw, db


def linear_fp8_block(x: torch.Tensor, w, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y = x · wᵀ (+ bias)`` with block-scaled 8-bit products, forward and backward.

    ``w [N, K]`` is a bf16 (or fp32) weight, cast here for the three products of a training step, or an
    ``Fp8BlockTensor`` from ``quantize_fp8_block(w, tile=True)`` that an inference program keeps (no gradients
    then). ``x`` is ``[..., K]``; ``y`` has its type if that is bf16 or fp32, else bf16. On the GPU ``K`` and
    ``N`` are multiples of 8. The weight gradient goes into the fp32 accumulator of the sharding runtime
    where the weight has one.
    """
    if w.shape[1] != x.shape[-1]:
        raise ValueError(f"x has {x.shape[-1]} features and w takes {w.shape[1]}")
    if isinstance(w, Fp8BlockTensor):
        if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
            raise ValueError("a kept 8-bit weight is for passes without gradients")
        xq, _ = quantize_fp8_block(x.reshape(-1, x.shape[-1]))
        y = matmul_fp8_block(xq, w, out_dtype=x.dtype if x.dtype == torch.float32 else torch.bfloat16, bias=bias)
        return y.view(*x.shape[:-1], w.rows)
    return _LinearFp8Block.apply(x, w, bias)


_KINDS = {"swiglu": 0, "geglu": 1}


def _glu_forward(gu, kind) -> Fp8BlockTensor:
    """``act(gate) * up`` (bf16 values) of ``gu = [gate | up]``, cast in blocks of a row."""
    T, I = gu.shape[0], gu.shape[1] // 2
    if not nv.use_native(gu):
        return _quantize_eager(glu_ref(gu[:, :I], gu[:, I:], kind), False, False, True, False)[0]
    h = _empty(T, I, False, gu.device)
    if T:
        rc = _fn("lb_block_glu_fwd")(_KINDS[kind], gu.data_ptr(), gu.data_ptr() + 2 * I, gu.stride(0), T, I, *_where(h),
                                     nv.stream_ptr())
        if rc != 0:
            nv.check_rc(rc, f"lb_block_glu_fwd(T={T},I={I})")
        nv.count_launch()
    return h


def _glu_grad_ref(g, u, dh, kind):
    g, u, dh = g.float(), u.float(), dh.float()
    if kind == "swiglu":
        s = torch.sigmoid(g)
        a, da = g * s, s * (1 + g * (1 - s))
    else:
        c, k = 0.7978845608028654, 0.044715
        t = torch.tanh(c * (g + k * g * g * g))
        a, da = 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * k * g * g)
    return torch.cat([dh * u * da, dh * a], dim=1).to(torch.bfloat16)


def _glu_backward(dh, gu, kind, want, want_t, want_h):
    """Gradients of ``gu`` in blocks of a row and of 128 tokens, and ``h`` in blocks of 128 tokens."""
    T, I = gu.shape[0], gu.shape[1] // 2
    if not nv.use_native(dh):
        d, d_t = _quantize_eager(_glu_grad_ref(gu[:, :I], gu[:, I:], dh, kind), False, False, want, want_t)
        h_t = _quantize_eager(glu_ref(gu[:, :I], gu[:, I:], kind), False, False, False, True)[1] if want_h else None
        return d, d_t, h_t
    d = _empty(T, 2 * I, False, gu.device) if want else None
    d_t = _empty(2 * I, T, False, gu.device) if want_t else None
    h_t = _empty(I, T, False, gu.device) if want_h else None
    if T:
        rc = _fn("lb_block_glu_bwd")(_KINDS[kind], dh.data_ptr(), dh.stride(0), gu.data_ptr(), gu.data_ptr() + 2 * I,
                                     gu.stride(0), T, I, *_where(d), *_where(d_t), *_where(h_t), nv.stream_ptr())
        if rc != 0:
            nv.check_rc(rc, f"lb_block_glu_bwd(T={T},I={I})")
        nv.count_launch()
    return d, d_t, h_t


def _cast_pair(w_gate, w_up, want_t):
    """Gate and up weights as one block-scaled ``[2 I, K]`` matrix (and its transpose), wherever they lie."""
    if w_up is None:
        return quantize_fp8_block(w_gate, tile=True, want_t=want_t)
    if not nv.use_native(w_gate, w_up):
        return _quantize_eager(torch.cat([w_gate, w_up]), True, False, True, want_t)
    I, K = w_gate.shape
    if K % 8:
        raise ValueError("quantize_fp8_block needs a multiple of 8 columns")
    q = _empty(2 * I, K, False, w_gate.device)
    q_t = _empty(K, 2 * I, False, w_gate.device) if want_t else None
    for lo, w in ((0, _aligned(w_gate.detach())), (I, _aligned(w_up.detach()))):
        part = Fp8BlockTensor(q.data[lo:lo + I], K, q.scales[:, lo:lo + I])
        part_t = (0, 0, 0, 0)
        if want_t:
            part_t = (q_t.data.data_ptr() + lo, _row_bytes(q_t.data), q_t.scales.data_ptr(), K)
        rc = _fn("lb_block_cast")(w.data_ptr(), I, K, w.stride(0), True, False, *_where(part), *part_t, lo // BLOCK,
                                  nv.stream_ptr())
        if rc != 0:
            nv.check_rc(rc, f"lb_block_cast(R={I},C={K})")
    nv.count_launch(2)
    return q, q_t


def _mlp_forward(xq, w, wd, kind):
    """Gate and up products (bf16) and the block's output."""
    gu = matmul_fp8_block(xq, w)
    return gu, matmul_fp8_block(_glu_forward(gu, kind), wd)


class _GatedMlpFp8Block(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, kind):
        x2 = x.reshape(-1, x.shape[-1])
        need_x, need_g, need_u, need_d = ctx.needs_input_grad[:4]
        need_gu = need_g or need_u
        xq, xq_t = quantize_fp8_block(x2, want_t=need_gu)
        wq, wq_t = _cast_pair(w_gate, w_up, need_x)
        dq, dq_t = quantize_fp8_block(w_down, tile=True, want_t=need_x or need_gu)
        gu, y = _mlp_forward(xq, wq, dq, kind)
        ctx.save_for_backward(gu, *(t for q in (xq_t, wq_t, dq_t) for t in ((q.data, q.scales) if q else (None, None))),
                              w_gate, w_up, w_down)
        ctx.kind, ctx.shape, ctx.dtype = kind, x.shape, x.dtype
        return y.view(x.shape).to(x.dtype if x.dtype == torch.float32 else torch.bfloat16)

    @staticmethod
    def backward(ctx, dy):
        gu, xt, xs, wt, ws, dt, ds, w_gate, w_up, w_down = ctx.saved_tensors
        need_x, need_g, need_u, need_d = ctx.needs_input_grad[:4]
        need_gu = need_g or need_u
        T, I = gu.shape[0], gu.shape[1] // 2
        dx = dg = du = dd = None
        dyq, dyq_t = quantize_fp8_block(dy.reshape(T, -1), want=need_x or need_gu, want_t=need_d)
        if need_x or need_gu:
            dh = matmul_fp8_block(dyq, Fp8BlockTensor(dt, w_down.shape[0], ds))
        else:
            dh = gu[:, :I]      # not read for h
        d, d_t, h_t = _glu_backward(dh, gu, ctx.kind, need_x, need_gu, need_d)
        if need_x:
            dx = matmul_fp8_block(d, Fp8BlockTensor(wt, 2 * I, ws)).view(ctx.shape).to(ctx.dtype)
        if need_gu:
            x_t = Fp8BlockTensor(xt, T, xs)
            if w_up is None:
                dg = _weight_gradient(w_gate, d_t, x_t)
            else:
                half = lambda lo: Fp8BlockTensor(d_t.data[lo:lo + I], T, d_t.scales[:, lo:lo + I])  # noqa: E731
                dg = _weight_gradient(w_gate, half(0), x_t) if need_g else None
                du = _weight_gradient(w_up, half(I), x_t) if need_u else None
        if need_d:
            dd = _weight_gradient(w_down, dyq_t, h_t)
        return dx, dg, du, dd, None


def gated_mlp_fp8_block(x: torch.Tensor, w_gate, w_up, w_down, kind: str = "swiglu") -> torch.Tensor:
    """``y = (act(x · w_gateᵀ) * (x · w_upᵀ)) · w_downᵀ`` with block-scaled 8-bit products, both directions.

    ``x`` is ``[..., H]``, ``w_gate`` and ``w_up`` ``[I, H]``, ``w_down`` ``[H, I]``; with ``w_up`` None
    ``w_gate`` is the fused ``[2 I, H]`` weight (gate rows first). ``kind`` is "swiglu" or "geglu" (tanh). ``I`` is a
    multiple of 128, so that no block holds gate and up columns; on the GPU ``H`` is a multiple of 8. Weights are
    bf16 (or fp32) and cast here, or, in a pass without gradients, the ``Fp8BlockTensor`` forms that
    ``quantize_fp8_block(w, tile=True)`` gives, all of them, with a fused gate and up weight.

    Gate and up products, ``act(gate) * up`` and its gradient, and the gradients of gate and up are rounded to
    bf16, as they are between separate layers, before they are cast.
    """
    if kind not in _KINDS:
        raise ValueError(f"unknown activation {kind!r}; choose from {tuple(_KINDS)}")
    H, I = w_down.shape
    rows = I if w_up is not None else 2 * I
    for w in (w_gate, w_up):
        if w is not None and tuple(w.shape) != (rows, H):
            raise ValueError(f"gate and up weights {tuple(w.shape)} do not fit w_down {tuple(w_down.shape)}")
    if x.shape[-1] != H:
        raise ValueError(f"x has {x.shape[-1]} features and the weights take {H}")
    if I % BLOCK:
        raise ValueError(f"the inner width has to be a multiple of {BLOCK}, got {I}")
    kept = [isinstance(w, Fp8BlockTensor) for w in (w_gate, w_up, w_down)]
    if any(kept):
        if not (kept[0] and kept[2]) or w_up is not None:
            raise ValueError("8-bit weights come as a fused gate and up weight and a down weight")
        if torch.is_grad_enabled() and x.requires_grad:
            raise ValueError("a kept 8-bit weight is for passes without gradients")
        xq, _ = quantize_fp8_block(x.reshape(-1, H))
        y = _mlp_forward(xq, w_gate, w_down, kind)[1].view(x.shape)
        return y.to(x.dtype) if x.dtype == torch.float32 else y
    return _GatedMlpFp8Block.apply(x, w_gate, w_up, w_down, kind)

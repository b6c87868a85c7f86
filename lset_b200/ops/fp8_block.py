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

import contextlib
import ctypes
import functools
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native as nv
from .activation import glu_ref
from ._grads import main_grad_of

BLOCK = 128
_MOST = 1 << 30      # rows and columns are counted in 32 bits


class Fp8BlockTensor:
    """A matrix ``[rows, cols]`` in 8 bits: ``data`` ``[rows, ld]`` bytes (the first ``cols`` of a row are
    valid; ``ld`` a multiple of 16), ``scales`` ``[ceil(cols / 512), rows, 4]`` bytes: ``scales[b // 4, r,
    b % 4]`` is the exponent (1 to 254, biased by 127) of the scale of columns ``128 b .. 128 b + 127`` of row ``r``;
    bytes of blocks that a row does not have are not read.

    The two are checked here, once; a product takes them as they are, and looks again where one lies elsewhere than it
    did (its ``.data`` exchanged). Copies (``copy``, ``pickle``) are made and checked anew, on memory of their own.
    """
    __slots__ = ("_data", "_cols", "_scales", "_e5m2", "_seen", "_at")

    def __init__(self, data: torch.Tensor, cols: int, scales: torch.Tensor, e5m2: bool = False):
        self._data, self._cols, self._scales, self._e5m2 = data, cols, scales, bool(e5m2)
        self._check()

    def _check(self):
        data, cols, scales = self._data, self._cols, self._scales
        if data.dtype is not torch.uint8 or scales.dtype is not torch.uint8 or data.dim() != 2 or scales.dim() != 3:
            raise TypeError("data is a 2-D and scales a 3-D tensor of bytes")
        strides, s_strides = data.stride(), scales.stride()
        (rows, width), (ld, step) = data.shape, strides
        (groups, s_rows, four), (s_group, s_row, s_byte) = scales.shape, s_strides
        if not 0 <= cols <= width or groups != (cols + 511) // 512 or s_rows != rows or four != 4:
            raise ValueError(f"data {tuple(data.shape)} with {cols} columns and scales {tuple(scales.shape)} do not "
                             f"belong together")
        if rows <= 1:       # strides of a dimension of one say nothing
            ld, s_row = (width + 15) // 16 * 16, 4
        if groups <= 1:
            s_group = 4 * rows
        if width and rows and ((step != 1 and width > 1) or ld < cols):
            raise ValueError("the bytes of a row lie next to one another")
        if rows and groups and (s_byte != 1 or s_row != 4 or s_group % 4 or s_group < 4 * rows):
            raise ValueError("the scales of four blocks lie next to one another, row by row")
        ptr, s_ptr = data.data_ptr(), scales.data_ptr()
        if data.is_cuda and (ld % 16 or ptr % 16 or s_ptr % 4) and width and rows:
            raise ValueError("rows start at multiples of 16 bytes, their scales at multiples of 4")
        if data.get_device() != scales.get_device():
            raise ValueError("data and scales are on one device")
        if not (ptr and s_ptr) and data.numel() and scales.numel():
            raise ValueError("the memory of a block-scaled matrix was released")
        self._seen = ptr, s_ptr, strides, s_strides
        # as the launchers take it: bytes, their row stride, scale words, words of a group of four blocks
        self._at = ptr, ld, s_ptr, s_group // 4

    def __reduce__(self):
        return Fp8BlockTensor, (self._data, self._cols, self._scales, self._e5m2)

    @property
    def _where(self):
        data, scales = self._data, self._scales
        if (data.data_ptr(), scales.data_ptr(), data.stride(), scales.stride()) != self._seen:
            self._check()
        return self._at

    data = property(lambda self: self._data)
    cols = property(lambda self: self._cols)
    scales = property(lambda self: self._scales)
    e5m2 = property(lambda self: self._e5m2)
    rows = property(lambda self: self._data.shape[0])
    shape = property(lambda self: (self._data.shape[0], self._cols))

    def dequantize(self) -> torch.Tensor:
        """The values, in fp32."""
        q = self.data[:, :self.cols].view(torch.float8_e5m2 if self.e5m2 else torch.float8_e4m3fn)
        e = self.scales.transpose(0, 1).reshape(self.rows, 4 * self.scales.shape[0]).int()
        s = (e << 23).view(torch.float32).repeat_interleave(BLOCK, dim=1)[:, :self.cols]
        return q.float() * s


# ------------------------------------------------------------------------------------------------
# Calls into the library
# ------------------------------------------------------------------------------------------------
_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
_SIGNATURES = {
    "lb_block_cast": [_P, _I, _I, _L, _I, _I, _P, _L, _P, _L, _P, _L, _P, _L, _I, _P],
    "lb_gemm_block_bytes": [_I, _I, _I, _L],
    "lb_gemm_block": [_P, _P, _P, _I, _I, _I, _L, _L, _L, _I, _I, _P, _L, _P, _L, _I, _I, _P, _P, _L, _P, _P],
    "lb_linear_block_bytes": [_I] * 4 + [_P],
    "lb_linear_block_fwd": [_P, _L, _P, _L, _P, _I, _I, _I, _I, _I] + [_P] * 5,
    "lb_linear_block_bwd": [_P, _L, _P, _L, _I, _I, _I, _I, _P, _P, _P, _I, _P, _I, _P, _I, _P, _P],
    "lb_linear_kept_bytes": [_I] * 3,
    "lb_linear_kept_fwd": [_P, _L, _P, _L, _P, _L, _I, _P, _I, _I, _I, _I, _P, _P, _P, _P],
    "lb_mlp_block_bytes": [_I] * 4 + [_P],
    "lb_mlp_block_fwd": [_I, _P, _L, _P, _L, _P, _L, _P, _L, _I, _I, _I, _I] + [_P] * 5,
    "lb_mlp_block_bwd": [_I, _P, _L, _I, _I, _I, _I, _I] + [_P] * 9,
    "lb_mlp_kept_bytes": [_I] * 3,
    "lb_mlp_kept_fwd": [_I, _P, _L, _P, _L, _P, _L, _I, _P, _L, _P, _L, _I, _I, _I, _I] + [_P] * 4,
}
_RETURNS = {"lb_gemm_block_bytes": _L, "lb_linear_kept_bytes": _L, "lb_mlp_kept_bytes": _L}
_fns = {}


def _fn(name):
    """A launcher with its argument types set: plain numbers then pass without a wrapper each."""
    f = _fns.get(name)
    if f is None:
        f = getattr(nv.load(), name)
        f.argtypes, f.restype = _SIGNATURES[name], _RETURNS.get(name, _I)
        _fns[name] = f
    return f


def _call(name, *args):
    rc = _fn(name)(*args)
    if rc != 0:
        nv.check_rc(rc, f"{name}{tuple(a for a in args if a is not None and not a >> 24)}")


_HERE = contextlib.nullcontext()


def _on_device(first, *others):
    """The tensors' one CUDA device as a context: launches go to the current stream of that device."""
    dev = first.get_device()
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"operands are on {first.device} and {t.device}")
    return _HERE if dev == _current_device() else torch.cuda.device(dev)


_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_status = {}


def _status_ptr(device) -> int:
    """Address of the device's status word, which stays where it is."""
    p = _status.get(device.index)
    if p is None:
        p = _status[device.index] = nv.status_word(device).data_ptr()
    return p


def _bytes(n: int, device) -> torch.Tensor:
    return torch.empty(n, dtype=torch.uint8, device=device)


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
    if x.dtype is not torch.bfloat16:
        x = x.to(torch.bfloat16)
    ld, step = x.stride()
    if step != 1 or ld % 8 or ld < x.shape[1] or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _rows(x: torch.Tensor, width: int) -> torch.Tensor:
    return x if x.dim() == 2 else x.reshape(-1, width)


_NONE = (0, 0, 0, 0)


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
    if R >= _MOST or C >= _MOST:
        raise ValueError(f"more rows or columns than the kernels count: {R}, {C}")
    with _on_device(x):
        x = _aligned(x.detach())
        out = _empty(R, C, e5m2, x.device) if want else None
        out_t = _empty(C, R, e5m2, x.device) if want_t else None
        if R and C and (want or want_t):
            _call("lb_block_cast", x.data_ptr(), R, C, x.stride(0), tile, e5m2, *(out._where if want else _NONE),
                  *(out_t._where if want_t else _NONE), 0, nv.stream_ptr())
            nv.count_launch()
    return out, out_t


# ------------------------------------------------------------------------------------------------
# Products
# ------------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=4096)
def _product_bytes(M, N, K, ldc) -> int:
    return _fn("lb_gemm_block_bytes")(M, N, K, ldc)


def matmul_fp8_block(a: Fp8BlockTensor, b: Fp8BlockTensor, *, out: Optional[torch.Tensor] = None,
                     out_dtype=torch.bfloat16, accumulate: bool = False, bias=None) -> torch.Tensor:
    """``C[M, N] = A · Bᵀ (+ bias)`` of block-scaled ``a [M, K]`` and ``b [N, K]``, in bf16 or fp32.

    ``out`` may be given (rows of unit inner stride); ``accumulate`` adds into it (fp32, no bias). Sums are
    fp32, in an order that the sizes and whether ``out``'s rows start at multiples of 16 bytes decide, and nothing
    else. e4m3 and e5m2 operands may be mixed.
    """
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
    if max(M, N, K) >= _MOST:
        raise ValueError(f"more rows or columns than the kernels count: {M}, {N}, {K}")
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
        ldc, fp32 = (out.stride(0) if M > 1 else N), out_dtype == torch.float32
        n = _product_bytes(M, N, K, ldc)
        ws = _bytes(n, out.device) if n else None
        (pa, lda, sa, rows_a), (pb, ldb, sb, rows_b) = a._where, b._where
        _call("lb_gemm_block", pa, pb, out.data_ptr(), M, N, K, lda, ldb, ldc, a.e5m2, b.e5m2, sa, rows_a, sb, rows_b, fp32,
              accumulate, nv.ptr(bias), nv.ptr(ws), n, _status_ptr(out.device), nv.stream_ptr())
        nv.count_launch()
    return out


# ------------------------------------------------------------------------------------------------
# Layers
# ------------------------------------------------------------------------------------------------
_BF16, _FP32, _ADD = 0, 1, 2     # where a result goes: a bf16 or fp32 tensor, or added to an fp32 one


def _mode(dtype) -> int:
    return _FP32 if dtype == torch.float32 else _BF16


def _gradient_of(w):
    """``(tensor, mode)`` that a native call writes the gradient of weight ``w`` to: its fp32 accumulator where the
    sharding runtime has given it one, else a tensor of its type (fp32 for types other than bf16)."""
    main = main_grad_of(w)
    if main is None:
        bf16 = w.dtype is torch.bfloat16
        return torch.empty(w.shape, dtype=torch.bfloat16 if bf16 else torch.float32, device=w.device), not bf16
    if main.dtype is torch.float32 and main.is_contiguous():
        return main, _ADD
    return torch.empty(w.shape, dtype=torch.float32, device=w.device), _FP32


def _returned(w, out, mode):
    """What autograd gets for ``w`` once ``_gradient_of``'s tensor is written."""
    if mode == _ADD:
        return None
    main = None if mode == _BF16 else main_grad_of(w)
    if main is None:
        return out if out.dtype is w.dtype else out.to(w.dtype)
    main.add_(out)
    return None


def _storage(n_saved, n_tmp, device):
    """A tensor of ``n_saved`` bytes for the backward, a tensor to hold during the call (or None), and the address of
    ``n_tmp`` bytes: behind the first where they are few (an allocation costs the host 2 us), else in the second."""
    small = n_tmp <= 1 << 20
    saved = _bytes(n_saved + n_tmp if small else n_saved, device)
    tmp = None if small else _bytes(n_tmp, device)
    return saved, tmp, saved.data_ptr() + n_saved if small else tmp.data_ptr()


@functools.lru_cache(maxsize=4096)
def _linear_bytes(T, K, N, need):
    out = (_L * 3)()
    _fn("lb_linear_block_bytes")(T, K, N, need, ctypes.addressof(out))
    return tuple(out)


@functools.lru_cache(maxsize=4096)
def _linear_kept_bytes(T, K, N):
    return _fn("lb_linear_kept_bytes")(T, K, N)


def _check_widths(T, K, N=0):
    if K % 8 or N % 8:
        raise ValueError(f"block-scaled layers need multiples of 8 features, got {K} and {N}")
    if T >= _MOST or K >= _MOST or N >= _MOST:
        raise ValueError(f"more rows or columns than the kernels count: {T}, {K}, {N}")


class _LinearFp8Block(torch.autograd.Function):
    """On the GPU: one native call each way. ``saved`` holds the transposed 8-bit copies of x and w, all that the
    backward reads of them."""

    @staticmethod
    def forward(ctx, x, w, bias):
        x2 = _rows(x, x.shape[-1])
        T, K = x2.shape
        N = w.shape[0]
        ctx.need = need = ctx.needs_input_grad[0] + 2 * ctx.needs_input_grad[1] + 4 * ctx.needs_input_grad[2]
        ctx.x_like = (x.shape, x.dtype)
        ctx.bias_dtype = None if bias is None else bias.dtype
        act = torch.float32 if x.dtype == torch.float32 else torch.bfloat16
        if not x.is_cuda:
            xq, xq_t = _quantize_eager(x2, False, False, True, True)
            wq, _ = _quantize_eager(w, True, False, True, False)
            ctx.save_for_backward(w, xq_t.dequantize(), wq.dequantize())
            return matmul_fp8_block(xq, wq, out_dtype=act, bias=bias).view(*x.shape[:-1], N)
        _check_widths(T, K, N)
        with _on_device(x, w, bias):
            x2, w2 = _aligned(x2), _aligned(w)
            if bias is not None and (bias.dtype is not torch.bfloat16 or not bias.is_contiguous()):
                bias = bias.to(torch.bfloat16).contiguous()
            n_saved, n_tmp, _ = _linear_bytes(T, K, N, need)
            saved, tmp, at = _storage(n_saved, n_tmp, x.device)
            y = torch.empty(*x.shape[:-1], N, dtype=act, device=x.device)
            _call("lb_linear_block_fwd", x2.data_ptr(), x2.stride(0), w2.data_ptr(), w2.stride(0), nv.ptr(bias), T, K, N,
                  need, _mode(act), y.data_ptr(), saved.data_ptr(), at,
                  _status_ptr(x.device), nv.stream_ptr())
            nv.count_launch(2)
        ctx.save_for_backward(w, saved)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w, *kept = ctx.saved_tensors
        shape, x_dtype = ctx.x_like
        N, K = w.shape
        dy2 = _rows(dy, N)
        T, need = dy2.shape[0], ctx.need
        dx = dw = db = None
        if len(kept) == 2:      # on the CPU
            xv_t, wv = kept
            dq, dq_t = _quantize_eager(dy2, False, False, True, True)
            if need & 1:
                dx = (dq.dequantize() @ wv).view(shape).to(x_dtype)
            if need & 2:
                dw = (dq_t.dequantize() @ xv_t.t()).to(w.dtype)
            if need & 4:
                db = dy2.float().sum(0).to(ctx.bias_dtype)
            return dx, dw, db
        saved, dev = kept[0], dy.device
        with _on_device(dy, w):
            dy32 = dy2.contiguous() if need & 4 and dy2.dtype is torch.float32 else None
            dy2 = _aligned(dy2)
            x_mode = x_dtype is torch.float32
            if need & 1:
                dx = torch.empty(shape, dtype=torch.float32 if x_mode else torch.bfloat16, device=dev)
            g, g_mode = _gradient_of(w) if need & 2 else (None, _BF16)
            b_mode = ctx.bias_dtype is not torch.bfloat16
            if need & 4:
                db = torch.empty(N, dtype=torch.float32 if b_mode else torch.bfloat16, device=dev)
            tmp = _bytes(_linear_bytes(T, K, N, need)[2], dev)
            _call("lb_linear_block_bwd", dy2.data_ptr(), dy2.stride(0), nv.ptr(dy32), N, T, K, N, need, saved.data_ptr(),
                  tmp.data_ptr(), nv.ptr(dx), x_mode, nv.ptr(g), g_mode, nv.ptr(db), b_mode, _status_ptr(dev), nv.stream_ptr())
            nv.count_launch(1 + bool(need & 1) + bool(need & 2) + bool(need & 4) + (dy32 is not None))
            if need & 2:
                dw = _returned(w, g, g_mode)
            if need & 1 and dx.dtype is not x_dtype:
                dx = dx.to(x_dtype)
            if need & 4 and db.dtype is not ctx.bias_dtype:
                db = db.to(ctx.bias_dtype)
        return dx, dw, db


def linear_fp8_block(x: torch.Tensor, w, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y = x · wᵀ (+ bias)`` with block-scaled 8-bit products, forward and backward.

    ``w [N, K]`` is a bf16 (or fp32) weight, cast here for the three products of a training step, or an
    ``Fp8BlockTensor`` from ``quantize_fp8_block(w, tile=True)`` that an inference program keeps (no gradients
    then). ``x`` is ``[..., K]``; ``y`` has its type if that is bf16 or fp32, else bf16. Operands (``x``, ``w``, the gradient
    of ``y``) of other types are rounded to bf16 on their way to 8 bits, and so is ``bias``; its gradient is the sum of
    the gradient of ``y`` as it comes. On the GPU ``K`` and ``N`` are multiples of 8. The weight gradient goes into the fp32 accumulator of the sharding runtime
    where the weight has one.
    """
    N, K = w.shape
    if K != x.shape[-1]:
        raise ValueError(f"x has {x.shape[-1]} features and w takes {K}")
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"bias has to be [{N}]")
    if not isinstance(w, Fp8BlockTensor):
        if x.numel() == 0 or N == 0:
            y = torch.nn.functional.linear(x, w.to(x.dtype), None if bias is None else bias.to(x.dtype))
            return y if x.dtype is torch.float32 else y.to(torch.bfloat16)
        if not torch.is_grad_enabled():      # nothing is kept for a backward then
            x, w, bias = x.detach(), w.detach(), None if bias is None else bias.detach()
        return _LinearFp8Block.apply(x, w, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        raise ValueError("a kept 8-bit weight is for passes without gradients")
    fp32 = x.dtype is torch.float32
    act = torch.float32 if fp32 else torch.bfloat16
    x2 = _rows(x, K)
    T = x2.shape[0]
    if T * K * N == 0 or not (x.is_cuda and w._data.is_cuda):
        xq, _ = quantize_fp8_block(x2)
        return matmul_fp8_block(xq, w, out_dtype=act, bias=bias).view(*x.shape[:-1], N)
    _check_widths(T, K, N)
    with _on_device(x, w._data, bias):
        x2 = _aligned(x2)
        if bias is not None and (bias.dtype is not torch.bfloat16 or not bias.is_contiguous()):
            bias = bias.to(torch.bfloat16).contiguous()
        y = torch.empty((T, N), dtype=act, device=x.device)
        n = _linear_kept_bytes(T, K, N)
        tmp = _bytes(n, x.device) if n else None      # none: the product casts x itself
        _call("lb_linear_kept_fwd", x2.data_ptr(), x2.stride(0), *w._where, w._e5m2, nv.ptr(bias), T, K, N, fp32,
              y.data_ptr(), nv.ptr(tmp), _status_ptr(x.device), nv.stream_ptr())
        nv.count_launch(2 if n else 1)
    return y if x2.dim() == x.dim() else y.view(*x.shape[:-1], N)


_KINDS = {"swiglu": 0, "geglu": 1}


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


def _mlp_eager(xq, w, wd, kind):
    """Gate and up products, ``h`` (both bf16 values) and the output."""
    gu = matmul_fp8_block(xq, w)
    I = gu.shape[1] // 2
    h = glu_ref(gu[:, :I], gu[:, I:], kind)
    return gu, h, matmul_fp8_block(_quantize_eager(h, False, False, True, False)[0], wd)


@functools.lru_cache(maxsize=4096)
def _mlp_bytes(T, H, I, need):
    out = (_L * 3)()
    _fn("lb_mlp_block_bytes")(T, H, I, need, ctypes.addressof(out))
    return tuple(out)


@functools.lru_cache(maxsize=4096)
def _mlp_kept_bytes(T, H, I):
    return _fn("lb_mlp_kept_bytes")(T, H, I)


class _GatedMlpFp8Block(torch.autograd.Function):
    """On the GPU: one native call each way. ``saved`` holds gate and up products and the transposed 8-bit copies of x and
    the weights."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, kind):
        H, I = w_down.shape
        x2 = _rows(x, H)
        T = x2.shape[0]
        nx, ng, nu, nd = ctx.needs_input_grad[:4]
        ctx.need = need = nx + 2 * (ng or nu) + 4 * nd
        ctx.kind, ctx.x_like = kind, (x.shape, x.dtype)
        act = torch.float32 if x.dtype == torch.float32 else torch.bfloat16
        if not x.is_cuda:
            xq, xq_t = _quantize_eager(x2, False, False, True, True)
            w = w_gate if w_up is None else torch.cat([w_gate, w_up])
            wq, dq = (_quantize_eager(t, True, False, True, False)[0] for t in (w, w_down))
            gu, h, y = _mlp_eager(xq, wq, dq, kind)
            ctx.save_for_backward(w_gate, w_up, w_down, gu, h, xq_t.dequantize(), wq.dequantize(), dq.dequantize())
            return y.view(x.shape).to(act)
        _check_widths(T, H, I)
        with _on_device(x, w_gate, w_up, w_down):
            x2, wg, wd = _aligned(x2), _aligned(w_gate), _aligned(w_down)
            wu = None if w_up is None else _aligned(w_up)
            n_saved, n_tmp, _ = _mlp_bytes(T, H, I, need)
            saved, tmp, at = _storage(n_saved, n_tmp, x.device)
            y = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
            _call("lb_mlp_block_fwd", _KINDS[kind], x2.data_ptr(), x2.stride(0), wg.data_ptr(), wg.stride(0), nv.ptr(wu),
                  0 if wu is None else wu.stride(0), wd.data_ptr(), wd.stride(0), T, H, I, need, y.data_ptr(),
                  saved.data_ptr(), at, _status_ptr(x.device), nv.stream_ptr())
            nv.count_launch(3)
        ctx.save_for_backward(w_gate, w_up, w_down, saved)
        return y.to(act)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w_gate, w_up, w_down, *kept = ctx.saved_tensors
        shape, x_dtype = ctx.x_like
        H, I = w_down.shape
        dy2 = _rows(dy, H)
        T, need = dy2.shape[0], ctx.need
        nx, ng, nu, nd = ctx.needs_input_grad[:4]
        dx = dg = du = dd = None
        if len(kept) > 1:       # on the CPU
            gu, h, xv_t, wv, dv = kept
            dq, dq_t = _quantize_eager(dy2, False, False, True, True)
            dh = (dq.dequantize() @ dv).to(torch.bfloat16)
            d, d_t = _quantize_eager(_glu_grad_ref(gu[:, :I], gu[:, I:], dh, ctx.kind), False, False, True, True)
            if nx:
                dx = (d.dequantize() @ wv).to(torch.bfloat16).view(shape).to(x_dtype)
            if need & 2:
                dw = d_t.dequantize() @ xv_t.t()
                if w_up is None:
                    dg = dw.to(w_gate.dtype)
                else:
                    dg, du = (t.to(w_gate.dtype) if n else None for t, n in ((dw[:I], ng), (dw[I:], nu)))
            if nd:
                h_t = _quantize_eager(h, False, False, False, True)[1].dequantize()
                dd = (dq_t.dequantize() @ h_t.t()).to(w_down.dtype)
            return dx, dg, du, dd, None
        saved = kept[0]
        with _on_device(dy, w_down):
            dy2 = _aligned(dy2)
            dx = torch.empty(shape, dtype=torch.bfloat16, device=dy.device) if nx else None
            grads = [_gradient_of(w) if n else (None, _BF16)
                     for w, n in ((w_gate, ng), (w_up, nu), (w_down, nd))]
            modes = [g[1] for g in grads]
            tmp = _bytes(_mlp_bytes(T, H, I, need)[2], dy.device)
            m = (_I * 3)(*modes)
            _call("lb_mlp_block_bwd", _KINDS[ctx.kind], dy2.data_ptr(), dy2.stride(0), T, H, I, need, w_up is None,
                  saved.data_ptr(), tmp.data_ptr(), nv.ptr(dx), *(nv.ptr(g[0]) for g in grads), ctypes.addressof(m),
                  _status_ptr(dy.device), nv.stream_ptr())
            nv.count_launch(2 + bool(need & 3) + nx + ng + nu + nd)
            dg, du, dd = (_returned(w, *g) if n else None
                          for w, n, g in zip((w_gate, w_up, w_down), (ng, nu, nd), grads))
            if nx and dx.dtype is not x_dtype:
                dx = dx.to(x_dtype)
        return dx, dg, du, dd, None


def gated_mlp_fp8_block(x: torch.Tensor, w_gate, w_up, w_down, kind: str = "swiglu") -> torch.Tensor:
    """``y = (act(x · w_gateᵀ) * (x · w_upᵀ)) · w_downᵀ`` with block-scaled 8-bit products, both directions.

    ``x`` is ``[..., H]``, ``w_gate`` and ``w_up`` ``[I, H]``, ``w_down`` ``[H, I]``; with ``w_up`` None
    ``w_gate`` is the fused ``[2 I, H]`` weight (gate rows first). ``kind`` is "swiglu" or "geglu" (tanh). ``I`` is a
    multiple of 128, so that no block holds gate and up columns; on the GPU ``H`` is a multiple of 8. Weights are
    bf16 (or fp32) and cast here, or, in a pass without gradients, the ``Fp8BlockTensor`` forms that
    ``quantize_fp8_block(w, tile=True)`` gives, all of them, with a fused gate and up weight.

    Gate and up products, ``act(gate) * up`` and its gradient, and the gradients of gate and up are rounded to
    bf16, as they are between separate layers, before they are cast; so are ``y`` and ``dx``, whatever ``x``'s type. A
    training step adds gate, up and dh from parts 1024 deep (an error in them can move a gradient by a step of 8
    bits); with kept weights they are summed whole, and above ``H`` = 1024 may differ from a step's in the last bit.
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
    if I % BLOCK or I == 0:
        raise ValueError(f"the inner width has to be a multiple of {BLOCK}, got {I}")
    kept = [isinstance(w, Fp8BlockTensor) for w in (w_gate, w_up, w_down)]
    if not any(kept):
        if x.numel() == 0:
            zero = sum(w.sum() for w in (w_gate, w_up, w_down) if w is not None) * 0
            y = x * zero.to(x.dtype)      # keeps the graph: gradients of zero
            return y if x.dtype is torch.float32 else y.to(torch.bfloat16)
        if not torch.is_grad_enabled():      # nothing is kept for a backward then
            x, w_gate, w_up, w_down = (t if t is None else t.detach() for t in (x, w_gate, w_up, w_down))
        return _GatedMlpFp8Block.apply(x, w_gate, w_up, w_down, kind)
    if not (kept[0] and kept[2]) or w_up is not None:
        raise ValueError("8-bit weights come as a fused gate and up weight and a down weight")
    if torch.is_grad_enabled() and x.requires_grad:
        raise ValueError("a kept 8-bit weight is for passes without gradients")
    act = torch.float32 if x.dtype == torch.float32 else torch.bfloat16
    if x.numel() == 0:
        return torch.empty(x.shape, dtype=act, device=x.device)
    x2 = _rows(x, H)
    if not x.is_cuda:
        xq, _ = _quantize_eager(x2, False, False, True, False)
        return _mlp_eager(xq, w_gate, w_down, kind)[2].view(x.shape).to(act)
    T = x2.shape[0]
    _check_widths(T, H, I)
    with _on_device(x, w_gate._data, w_down._data):
        x2 = _aligned(x2)
        y = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
        tmp = _bytes(_mlp_kept_bytes(T, H, I), x.device)
        _call("lb_mlp_kept_fwd", _KINDS[kind], x2.data_ptr(), x2.stride(0), *w_gate._where, w_gate._e5m2,
              *w_down._where, w_down._e5m2, T, H, I, y.data_ptr(), tmp.data_ptr(),
              _status_ptr(x.device), nv.stream_ptr())
        nv.count_launch(4)
    return y.to(act)

"""4-bit weights with group scales: the codec, and the operators that read the codes.

A matrix (N, K) is held as ``w[n, k] = scale * scales[n, k // group] * q[n, k]`` (:class:`Q4`): q whole numbers in
-8 .. 7, one E4M3 scale per group of 32, 64, 128 or 256 values of a row, one float32 per matrix.  4.25 bits a weight at
group 32.  ``scales * q`` has at most 8 significant bits, so the products of bfloat16 or float16 activations with the
weights are exact and only their float32 sums and the result round.

* ``enc_q4`` / ``deq_q4``  -- the codec, beside ``q8.enc_q8`` / ``q8.deq_q8``
* ``linear``               -- y = x W^T, from one token up
* ``grouped_linear``       -- the same with one matrix for each run of rows (experts), ragged
* ``embedding``            -- rows by token, scaled
* ``round_scales``         -- float32 group scales into the stored form

``linear``, ``grouped_linear`` and ``embedding`` are differentiable with respect to the activations and, like
``qat.recon_torch``, to the scales with the codes held fixed: ``scales`` is the float32 tensor that is trained, in units
of ``w.scale * w.scales`` (``w.group_scales()`` starts one).  The product uses the scales stored in ``w`` and passes the
gradient straight through their rounding; after an optimizer step ``round_scales`` stores the new ones.

Everything runs on the current stream of the operands' device; nothing synchronises.  ``check_errors`` reports what
kernels met on the device (a token or offset out of range).  The reference has no counterpart.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from . import _device as D
from . import _lib
from ._lib import UQ_BF16, UQ_F16, UQ_F32, UQ_F64

__all__ = ["Q4", "enc_q4", "deq_q4", "round_scales", "linear", "grouped_linear", "embedding", "check_errors"]

GROUPS = (32, 64, 128, 256)
_CODE = {torch.float32: UQ_F32, torch.float64: UQ_F64, torch.bfloat16: UQ_BF16, torch.float16: UQ_F16}
_ACT = {torch.bfloat16: UQ_BF16, torch.float16: UQ_F16}
_OUT = {torch.float32: UQ_F32, torch.bfloat16: UQ_BF16, torch.float16: UQ_F16}


class Q4:
    """4-bit weights: ``codes`` (..., N, K/2) uint8, ``scales`` (..., N, K/group) float8_e4m3fn, ``scale`` (...) float32,
    with no leading dimension or one (experts).  Contiguous CUDA tensors of one device; the byte order of the codes is
    include/uq_b200.h's."""

    __slots__ = ("codes", "scales", "scale", "mats", "rows", "cols", "group", "device", "form")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, scale: torch.Tensor):
        cs, ss = codes.shape, scales.shape
        if codes.dtype != torch.uint8 or scales.dtype != torch.float8_e4m3fn or scale.dtype != torch.float32:
            raise TypeError(f"Q4: codes uint8, scales float8_e4m3fn and scale float32 are expected, got {codes.dtype}, "
                            f"{scales.dtype}, {scale.dtype}")
        if len(cs) not in (2, 3) or len(ss) != len(cs) or ss[:-1] != cs[:-1] or scale.numel() != (cs[0] if len(cs) == 3 else 1):
            raise ValueError(f"Q4: shapes do not match: codes {tuple(cs)}, scales {tuple(ss)}, scale {tuple(scale.shape)}")
        cols, per = 2 * cs[-1], ss[-1]
        group = cols // per if per else 0
        if group not in GROUPS or group * per != cols:
            raise ValueError(f"Q4: {cols} columns and {per} scales a row: groups of {GROUPS} are built")
        if not codes.is_cuda or scales.device != codes.device or scale.device != codes.device:
            raise ValueError("Q4: codes, scales and scale have to be CUDA tensors of one device")
        if not (codes.is_contiguous() and scales.is_contiguous() and scale.is_contiguous()):
            raise ValueError("Q4: codes, scales and scale have to be contiguous")
        if codes.data_ptr() & 15 or scales.data_ptr() & 15:
            raise ValueError("Q4: codes and scales have to start on a 16-byte boundary")
        self._set(codes, scales, scale, cs[0] if len(cs) == 3 else 1, cs[-2], cols, group)

    def _set(self, codes, scales, scale, mats, rows, cols, group):
        self.codes, self.scales, self.scale = codes, scales, scale
        self.mats, self.rows, self.cols, self.group, self.device = mats, rows, cols, group, codes.device
        self.form = (mats, rows, cols, group)

    @classmethod
    def _of(cls, codes, scales, scale, mats, rows, cols, group):
        """Of tensors made here, which need no check."""
        w = cls.__new__(cls)
        w._set(codes, scales, scale, mats, rows, cols, group)
        return w

    @property
    def ptrs(self):
        return self.codes.data_ptr(), self.scales.data_ptr(), self.scale.data_ptr()

    @property
    def shape(self):
        return (*self.codes.shape[:-1], self.cols)

    def group_scales(self) -> torch.Tensor:
        """scale * scales in float32, (..., N, K/group): a start for trained scales."""
        return self.scales.float() * self.scale.reshape(*self.codes.shape[:-2], 1, 1)

    def __repr__(self):
        return f"Q4(shape={self.shape}, group={self.group}, device={self.device})"


def _weights(W):
    """numpy or torch weights on the device, in a dtype that the encoder reads."""
    if not isinstance(W, torch.Tensor):
        W = D.as_device(W)
    if W.dtype not in _CODE:
        raise TypeError(f"enc_q4: dtype {W.dtype} is not built (float32, float64, bfloat16, float16)")
    if not W.is_cuda:
        W = W.to(D.device())
    return W if W.is_contiguous() else W.contiguous()


def enc_q4(W, group: int = 32) -> Q4:
    """(N, K) or (experts, N, K) weights -> :class:`Q4`; K a multiple of ``group``.  Each group's scale takes its value of
    largest size to -8; values round to the nearest step, ties to even.  A group with a non-finite value decodes to NaN."""
    w = _weights(W)
    if w.dim() not in (2, 3):
        raise ValueError(f"enc_q4: expected (N, K) or (experts, N, K), got shape {tuple(w.shape)}")
    if group not in GROUPS:
        raise ValueError(f"enc_q4: group {group} is not one of {GROUPS}")
    *lead, rows, cols = w.shape
    if cols == 0 or cols % group:
        raise ValueError(f"enc_q4: {cols} columns are not whole groups of {group}")
    dev = w.device
    mats = lead[0] if lead else 1
    codes = w.new_empty((*lead, rows, cols // 2), dtype=torch.uint8)
    scales = w.new_empty((*lead, rows, cols // group), dtype=torch.float8_e4m3fn)
    scale = w.new_empty(tuple(lead), dtype=torch.float32)
    nbytes = _workspace_bytes("uq_q4_encode", mats, rows, cols)
    ws = _scratch(nbytes, dev)
    _run(dev, "uq_q4_encode", w.data_ptr(), _CODE[w.dtype], mats, rows, cols, cols, group, codes.data_ptr(),
         scales.data_ptr(), scale.data_ptr(), D.ptr(ws), nbytes)
    return Q4._of(codes, scales, scale, mats, rows, cols, group)


def deq_q4(w: Q4, dtype=torch.float32) -> torch.Tensor:
    """The values: scale * scales * q.  With a power of two as ``scale`` (the encoder's) float32 holds them exactly and a
    16-bit ``dtype`` rounds once; with any other the float32 products round as well."""
    if dtype not in _OUT:
        raise TypeError(f"deq_q4: dtype {dtype} is not built (float32, bfloat16, float16)")
    out = w.codes.new_empty(w.shape, dtype=dtype)
    _run(w.device, "uq_q4_decode", *w.ptrs, *w.form, out.data_ptr(), _OUT[dtype])
    return out


def round_scales(w: Q4, scales: torch.Tensor) -> Q4:
    """``w``'s codes with the float32 group scales ``scales`` rounded into the stored form (new scale tensors; the codes
    are shared)."""
    c = _trained(w, scales).detach().contiguous()
    e, s = torch.empty_like(w.scales), torch.empty_like(w.scale)
    _run(w.device, "uq_q4_round_scales", c.data_ptr(), w.mats, c.numel() // max(w.mats, 1), e.data_ptr(),
         s.data_ptr())
    return Q4._of(w.codes, e, s, *w.form)


def check_errors(device=None) -> None:
    """Waits for the current stream and raises what the operators' kernels of the device have met since the last call:
    UQError for a wait that gave up, else ValueError for a token or an offset out of range; the message names all."""
    dev = torch.device(device) if device is not None else D.device()
    _run(dev if dev.index is not None else D.device(), "uq_q4_errors")


def _trained(w: Q4, scales) -> torch.Tensor:
    if scales.dtype != torch.float32 or scales.shape != w.scales.shape or scales.device != w.device:
        raise ValueError(f"q4: trained scales have to be float32 {tuple(w.scales.shape)} on {w.device}, got {scales.dtype} "
                         f"{tuple(scales.shape)} on {scales.device}")
    return scales


def _rows(x: torch.Tensor) -> torch.Tensor:
    """(..., n) as a matrix whose rows the kernels can read: unit inner stride, 16-byte aligned base and row stride."""
    if x.dim() != 2:
        x = x.reshape(x.shape[:-1].numel(), x.shape[-1])     # not -1: there may be no columns
    T, n = x.shape
    ld, inner = x.stride()
    if T <= 1:
        ld = n
    if (inner == 1 and not ld & 7 and ld >= n and not x.data_ptr() & 15) or T == 0 or n == 0:
        return x
    pad = torch.empty((T, -(-n // 8) * 8), dtype=x.dtype, device=x.device)
    pad[:, :n] = x
    return pad[:, :n]


def _ld(x: torch.Tensor) -> int:
    """Row stride; of a single row, what the kernels ask of it."""
    return x.stride(0) if x.shape[0] > 1 else -(-x.shape[1] // 8) * 8


def _extent(t: torch.Tensor) -> tuple[int, int, int, int]:
    """(first byte, rows, bytes from row to row, bytes of a row) of a matrix with unit inner stride or a contiguous tensor."""
    size = t.element_size()
    if t.dim() != 2 or t.shape[0] <= 1 or t.is_contiguous():
        return t.data_ptr(), 1, 0, t.numel() * size
    return t.data_ptr(), t.shape[0], t.stride(0) * size, t.shape[1] * size


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the two share a byte.  Columns of the same rows do not; of interleaved rows of different strides this is not
    looked into (they count as sharing)."""
    if not a.numel() or not b.numel():
        return False
    (pa, ra, sa, wa), (pb, rb, sb, wb) = _extent(a), _extent(b)
    if pa + (ra - 1) * sa + wa <= pb or pb + (rb - 1) * sb + wb <= pa:
        return False
    step = sa or sb
    if not step or (ra > 1 and rb > 1 and sa != sb):
        return True
    d = (pb - pa) % step          # where b's rows begin between two of a's
    return d < wa or d + wb > step


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


@lru_cache(maxsize=None)
def _fn(name: str):
    return getattr(_lib.load(), name)


def _run(dev: torch.device, name: str, *args) -> None:
    """The entry point ``name`` on the current stream of ``dev``, raising for its status."""
    fn, i = _fn(name), dev.index
    stream = _raw_stream(i) if _raw_stream is not None else D.stream_handle(dev)
    if torch.cuda.current_device() == i:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(i):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc, name)


@lru_cache(maxsize=4096)
def _workspace_bytes(name: str, *sizes) -> int:
    return _fn(name + "_workspace_bytes")(*sizes)


def _scratch(nbytes: int, dev: torch.device):
    """Of its own for each call: calls on several streams and captured graphs share nothing."""
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _checked(x: torch.Tensor, w: Q4, offsets, what: str) -> None:
    if x.dtype not in _ACT:
        raise TypeError(f"{what}: activations of dtype {x.dtype} are not built (bfloat16, float16)")
    if x.device != w.device:
        raise ValueError(f"{what}: activations on {x.device}, weights on {w.device}")
    if x.dim() == 0 or x.shape[-1] != w.cols:
        raise ValueError(f"{what}: activations {tuple(x.shape)} do not match weights {w.shape}")
    if offsets is None:
        if w.codes.dim() != 2:
            raise ValueError(f"{what}: weights {w.shape} are those of several experts")
    else:
        if w.codes.dim() != 3:
            raise ValueError(f"{what}: weights {w.shape} have no experts")
        if x.dim() != 2:
            raise ValueError(f"{what}: activations have to be (rows, {w.cols}), got {tuple(x.shape)}")
        if offsets.dtype != torch.int32 or offsets.shape != (w.mats + 1,) or offsets.device != w.device or not offsets.is_contiguous():
            raise ValueError(f"{what}: offsets have to be {w.mats + 1} contiguous int32 on {w.device}")


def _call(name: str, T: int, a: torch.Tensor, w: Q4, offsets, out: torch.Tensor, zero_rest: bool) -> None:
    """uq_q4_linear or uq_q4_linear_dx on rows ``a``."""
    mats, rows, cols, group = w.form
    nbytes = _workspace_bytes(name, T, mats, rows, cols) if offsets is None else 0
    ws = _scratch(nbytes, w.device)
    _run(w.device, name, a.data_ptr(), _ACT[a.dtype], T, _ld(a), *w.ptrs, mats, rows, cols, group,
         offsets.data_ptr() if offsets is not None else None, out.data_ptr(), out.stride(0) if T > 1 else out.shape[1],
         zero_rest, ws.data_ptr() if nbytes else None, nbytes)


def _forward(x2: torch.Tensor, w: Q4, offsets, out=None) -> torch.Tensor:
    T = x2.shape[0]
    zero_rest = out is None
    if out is None:
        out = x2.new_empty((T, w.rows))
    if T and w.rows:
        _call("uq_q4_linear", T, x2, w, offsets, out, zero_rest)
    return out


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scales, w, offsets):
        x2 = _rows(x)
        ctx.w, ctx.shape = w, x.shape
        ctx.save_for_backward(x2 if scales is not None else None, offsets, w.codes, w.scales, w.scale)
        return _shaped(_forward(x2, w, offsets), x, w)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x2, offsets, *_ = ctx.saved_tensors
        w = ctx.w
        d2 = _rows(dy)
        T = d2.shape[0]
        dx = dc = None
        if ctx.needs_input_grad[0]:
            dx = torch.empty((T, w.cols), dtype=dy.dtype, device=w.device)
            if T and w.rows:
                _call("uq_q4_linear_dx", T, d2, w, offsets, dx, True)
            else:
                dx.zero_()
            dx = dx.reshape(ctx.shape)
        if ctx.needs_input_grad[1]:
            dc = torch.empty(w.scales.shape, dtype=torch.float32, device=w.device)
            if dc.numel():
                nbytes = _workspace_bytes("uq_q4_linear_dscale", T, *w.form)
                ws = _scratch(nbytes, w.device)
                _run(w.device, "uq_q4_linear_dscale", D.ptr(d2), D.ptr(x2), _ACT[dy.dtype], T,
                     _ld(d2), _ld(x2), w.ptrs[0], *w.form, D.ptr(offsets), dc.data_ptr(), D.ptr(ws), nbytes)
        return dx, dc, None, None


def _shaped(y: torch.Tensor, x: torch.Tensor, w: Q4) -> torch.Tensor:
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], w.rows)


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def linear(x: torch.Tensor, w: Q4, scales: torch.Tensor | None = None) -> torch.Tensor:
    """y = x W^T: x (..., K) bfloat16 or float16, w (N, K) -> (..., N) in x's dtype; float32 sums over exact products, one
    rounding.  Differentiable in x and in ``scales`` (see the module's text)."""
    _checked(x, w, None, "linear")
    if scales is not None:
        _trained(w, scales)
    if _wants_grad(x, scales):
        return _Product.apply(x, scales, w, None)
    return _shaped(_forward(_rows(x), w, None), x, w)


def grouped_linear(x: torch.Tensor, offsets: torch.Tensor, w: Q4, scales: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows offsets[i] .. offsets[i + 1] - 1 of x (rows, K) times matrix i of w (experts, N, K), each expert with any number
    of rows, none among them; offsets int32 on the device, never falling, at most the rows of x (each is taken as at least
    its predecessors; ``check_errors`` reports one that is not).  Returns (rows, N); rows outside offsets[0] ..
    offsets[-1] are zero, or, in an ``out`` that is given, left as they were.  ``out`` may be columns of a larger matrix; it
    shares no memory with what is read.  Differentiable like ``linear``, without ``out``."""
    _checked(x, w, offsets, "grouped_linear")
    if scales is not None:
        _trained(w, scales)
    if _wants_grad(x, scales):
        if out is not None:
            raise ValueError("grouped_linear: out cannot be given where a gradient is wanted")
        return _Product.apply(x, scales, w, offsets)
    if out is not None:
        if out.dtype != x.dtype or out.shape != (x.shape[0], w.rows) or out.device != w.device or out.stride(1) != 1 or (
                out.shape[0] > 1 and out.stride(0) < w.rows):
            raise ValueError(f"grouped_linear: out has to be {x.dtype} {(x.shape[0], w.rows)} with rows of unit stride")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("grouped_linear: out wants a gradient, which is not passed through it")
        x = _rows(x)
        if any(_overlap(out, t) for t in (x, offsets, w.codes, w.scales, w.scale)):
            raise ValueError("grouped_linear: out overlaps the activations, offsets or weights that are read")
        torch.autograd.graph.increment_version(out)   # a backward pass that needs what was there notices
    return _forward(_rows(x), w, offsets, out)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, scales, w, alpha, dtype):
        ctx.w, ctx.alpha = w, alpha
        ctx.save_for_backward(tokens, w.codes)
        return _lookup(tokens, w, alpha, dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        tokens, _ = ctx.saved_tensors
        w = ctx.w
        d2 = _rows(dout)
        T = d2.shape[0]
        dc = torch.empty(w.scales.shape, dtype=torch.float32, device=w.device)
        if dc.numel():
            nbytes = _workspace_bytes("uq_q4_embed_dscale", T, *w.form[1:])
            ws = _scratch(nbytes, w.device)
            _run(w.device, "uq_q4_embed_dscale", D.ptr(tokens), tokens.dtype == torch.int64, T,
                 D.ptr(d2), _OUT[d2.dtype], _ld(d2), w.ptrs[0], *w.form[1:], ctx.alpha, dc.data_ptr(), D.ptr(ws), nbytes)
        return None, dc, None, None, None


def _lookup(tokens, w, alpha, dtype):
    out = w.codes.new_empty((*tokens.shape, w.cols), dtype=dtype)
    if out.numel():
        _run(w.device, "uq_q4_embed", tokens.data_ptr(), tokens.dtype == torch.int64, tokens.numel(), *w.ptrs,
             *w.form[1:], alpha, out.data_ptr(), _OUT[dtype])
    return out


def embedding(tokens: torch.Tensor, w: Q4, alpha: float = 1.0, scales: torch.Tensor | None = None,
              dtype=torch.bfloat16) -> torch.Tensor:
    """alpha * w[tokens]: tokens int32 or int64 of any shape, w (V, K) -> (*tokens.shape, K) in ``dtype`` (bfloat16,
    float16 or float32).  A token outside 0 .. V - 1 gives a row of NaN (and no gradient); ``check_errors`` reports it.
    Differentiable in ``scales``: the rows of each token are found by a stable sort and added in their order, so the
    gradient's bits are the same every time."""
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"embedding: tokens have to be int32 or int64, got {tokens.dtype}")
    if tokens.device != w.device:
        raise ValueError(f"embedding: tokens on {tokens.device}, weights on {w.device}")
    if w.codes.dim() != 2:
        raise ValueError(f"embedding: a table (V, K) is expected, got {w.shape}")
    if dtype not in _OUT:
        raise TypeError(f"embedding: dtype {dtype} is not built (float32, bfloat16, float16)")
    tokens = tokens.contiguous()
    if scales is not None:
        _trained(w, scales)
        if _wants_grad(scales):
            return _Embedding.apply(tokens, scales, w, float(alpha), dtype)
    return _lookup(tokens, w, float(alpha), dtype)

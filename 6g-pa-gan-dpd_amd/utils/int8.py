"""The linear layer in 8 bits, with one scale for each token and each output channel (csrc/int8_linear.hip).

`QuantizedLinear` quantises with fixed power-of-two scales; here the scales follow the data, so that wide layers keep
7 bits of every row.  `quantize_rows_int8` and `int8_matmul` are the two parts, `int8_linear` / `Int8Linear` train through
them with the straight-through estimator, `Int8Inference` serves weights that are quantised once.  The reference has no
counterpart."""
from typing import Dict, Optional, Tuple

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import _lib as L

TYPES = L.TYPES
_NEEDS_WORKSPACE = 4            # DPD_ERR_WORKSPACE
_MOST_STRIDE = (1 << 23) - 128  # bytes from row to row of an int8 factor
_MOST_OUTS = {torch.float32: 1398080, torch.bfloat16: 2097088, torch.float16: 2097088}      # with a gradient of x
_MOST_TOKENS = 1 << 20          # of one backward call: bounds its workspace, and below what the weight's gradient can sum over


def _type(t: torch.Tensor, what: str) -> int:
    try:
        return TYPES[t.dtype]
    except KeyError:
        raise RuntimeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}") from None


def _rows(x: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """x as rows [M, K] whose elements lie one behind the other, and the row stride: x itself where its layout allows."""
    if x.dim() == 0:
        raise ValueError("expected at least one dimension")
    k = x.shape[-1]
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= k:
        return x, x.stride(0)
    return x.contiguous().view(-1, k) if x.numel() else x.new_empty(x.shape[:-1].numel(), k), k


def _near_rows(x: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """The same for the product, whose offsets inside a tile of 256 rows have 32 bits: rows further apart are copied."""
    x2, ld = _rows(x)
    return (x2, ld) if ld <= _MOST_STRIDE else (x2.contiguous(), x2.shape[1])


def _check_scale(s: torch.Tensor, rows: int, device, what: str) -> torch.Tensor:
    if s.dtype != torch.float32 or s.numel() != rows or s.device != device:
        raise ValueError(f"{what} must be {rows} float32 values on {device}, got {tuple(s.shape)} {s.dtype} on {s.device}")
    return s.contiguous()


def _check_bias(b: Optional[torch.Tensor], n: int, device) -> Tuple[Optional[torch.Tensor], int]:
    if b is None:
        return None, 0
    if b.dim() != 1 or b.shape[0] != n or b.device != device:
        raise ValueError(f"bias must be {n} values on {device}, got {tuple(b.shape)} on {b.device}")
    return b.contiguous(), _type(b, "bias")


def _quantize(x2: torch.Tensor, ldx: int, ldq: int) -> Tuple[torch.Tensor, torch.Tensor]:
    m, k = x2.shape
    q = torch.empty(m, ldq, dtype=torch.int8, device=x2.device)
    s = torch.empty(m, dtype=torch.float32, device=x2.device)
    L.call("dpd_quantize_rows_int8", L.c_p(x2.data_ptr()), _type(x2, "x"), m, k, ldx, L.c_p(q.data_ptr()), ldq, L.c_p(s.data_ptr()), L.stream())
    return q, s


def _row_bytes(k: int) -> int:
    return (k + 127) // 128 * 128


def quantize_rows_int8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of the rows of x [..., K]: scale = max(max|row|, 2^-100) times fl32(1 / 127) in fp32, q = round-half-even(row / scale)
    as int8.  A row that holds a NaN or an infinity gets the scale NaN and zeros, so every product with it is NaN.  The results
    have no history (`int8_linear` is what has a gradient)."""
    L.need_gpu(x)
    with torch.no_grad():                # a tangent only: a leaf that is trained may be looked at
        L.refuse_gradient("quantize_rows_int8", x)
    x = x.detach()
    x2, ldx = _rows(x)
    with L.device(x):
        q, s = _quantize(x2, ldx, x2.shape[1])
    return q.view(x.shape), s.view(x.shape[:-1])


def _matmul(a, lda, sa, b, ldb, sb, bias, bias_type, m, n, k, dtype):
    out = torch.empty(m, n, dtype=dtype, device=a.device)
    ws = None
    nbytes = 0
    if k % 16 or lda % 16 or ldb % 16 or a.data_ptr() % 16 or b.data_ptr() % 16:
        nbytes = L.lib().dpd_int8_matmul_workspace_bytes(m, n, k)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=a.device)
    L.call("dpd_int8_matmul", L.c_p(a.data_ptr()), lda, L.c_p(sa.data_ptr()), L.c_p(b.data_ptr()), ldb, L.c_p(sb.data_ptr()),
           L.c_p(bias.data_ptr() if bias is not None else 0), bias_type, m, n, k, L.c_p(out.data_ptr()), TYPES[dtype], n,
           L.c_p(ws.data_ptr() if ws is not None else 0), nbytes, L.stream())
    return out


def int8_matmul(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """a [..., K] int8 with one scale a row, b [N, K] int8 with one scale a row: (a b^T) a_scale b_scale + bias as [..., N].
    The sum is exact (K <= 131071); scales and bias enter in fp32, and the result is rounded once.  Not differentiable: scales or a
    bias that require a gradient are refused."""
    L.need_gpu(a, a_scale, b, b_scale, bias)
    if a.dtype != torch.int8 or b.dtype != torch.int8:
        raise RuntimeError(f"int8_matmul takes int8 matrices, got {a.dtype} and {b.dtype}")
    if out_dtype not in TYPES:
        raise RuntimeError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    if b.dim() != 2 or a.dim() < 1 or a.shape[-1] != b.shape[1] or a.device != b.device:
        raise ValueError(f"cannot multiply rows of {tuple(a.shape)} on {a.device} with rows of {tuple(b.shape)} on {b.device}")
    a2, lda = _near_rows(a)
    b2, ldb = _near_rows(b)
    m, n, k = a2.shape[0], b2.shape[0], b2.shape[1]
    sa, sb = _check_scale(a_scale, m, a.device, "a_scale"), _check_scale(b_scale, n, a.device, "b_scale")
    bc, bt = _check_bias(bias, n, a.device)
    L.refuse_gradient("int8_matmul (training: int8_linear)", sa, sb, bc)
    with L.device(a):
        return _matmul(a2, lda, sa, b2, ldb, sb, bc, bt, m, n, k, out_dtype).view(*a.shape[:-1], n)


def _addresses(kept, m, n, ld):
    base = kept.data_ptr()
    return base, base + m * ld, base + (m + n) * ld, base + (m + n) * ld + 4 * m


class _Int8LinearFn(torch.autograd.Function):
    """Both factors quantised on the way; the backward reads the 8-bit factors, so x and the weight are not kept."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        x2, ldx = _rows(x)
        w2, ldw = _rows(weight)
        (m, k), n = x2.shape, w2.shape[0]
        ld, dev = _row_bytes(k), x.device
        bc, bt = _check_bias(bias, n, dev)
        out = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=dev)
        # one buffer for what the backward reads: qx [m, ld], qw [n, ld], the scales of x, the scales of the weight
        kept = torch.empty((m + n) * (ld + 4), dtype=torch.int8, device=dev)
        at = _addresses(kept, m, n, ld)
        with L.device(x):
            L.check(L.entry("dpd_int8_linear_forward")(
                x2.data_ptr(), TYPES[x.dtype], m, k, ldx, w2.data_ptr(), TYPES[weight.dtype], n, ldw, 0 if bc is None else bc.data_ptr(), bt,
                out.data_ptr(), n, at[0], at[2], at[1], at[3], L.raw_stream(dev.index)))
        ctx.save_for_backward(kept)
        ctx.sizes, ctx.lead, ctx.types = (m, n, k, ld), x.shape[:-1], (x.dtype, weight.dtype, bias.dtype if bias is not None else None)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        kept, = ctx.saved_tensors
        m, n, k, ld = ctx.sizes
        tx, tw, tb = ctx.types
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        need_b = tb is not None and ctx.needs_input_grad[2]
        dev = kept.device
        g2, ldg = _rows(gy)
        gx = torch.empty((*ctx.lead, k), dtype=tx, device=dev) if need_x else None
        ptr = lambda t: t.data_ptr() if t is not None else 0
        t, (qx, qw, sx, sw) = TYPES[tx], _addresses(kept, m, n, ld)
        # more tokens than one call takes: in parts, whose weight and bias gradients are added in fp32, in their order
        part = max(64, min(_MOST_TOKENS, (1 << 35) // max(n, 64) // 64 * 64))
        whole = m <= part
        with L.device(kept):
            gw = torch.empty(n, k, dtype=tw if whole else torch.float32, device=dev) if need_w else None
            gb = torch.empty(n, dtype=tb if whole else torch.float32, device=dev) if need_b else None
            nbytes = L.entry("dpd_int8_linear_backward_workspace_bytes")(min(m, part), n, k, t, need_x, need_w, need_b)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            type_w, type_b = TYPES[tw if whole else torch.float32], (TYPES[tb if whole else torch.float32] if need_b else 0)
            size_g, size_x = g2.element_size(), tx.itemsize
            for at in range(0, max(m, 1), part):
                w, b = (gw, gb) if at == 0 else (torch.empty_like(gw) if need_w else None, torch.empty_like(gb) if need_b else None)
                L.check(L.entry("dpd_int8_linear_backward")(
                    g2.data_ptr() + at * ldg * size_g, t, min(m - at, part), n, k, ldg, qx + at * ld, ld, sx + at * 4, qw, ld, sw,
                    gx.data_ptr() + at * k * size_x if need_x else 0, ptr(w), type_w, ptr(b), type_b, ws.data_ptr(), nbytes, L.raw_stream(dev.index)))
                if at:
                    if need_w:
                        gw += w
                    if need_b:
                        gb += b
        return gx, gw if whole or not need_w else gw.to(tw), gb if whole or not need_b else gb.to(tb)


def int8_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q(x) q(weight)^T + bias in the type of x, both factors quantised by rows in this call; differentiable in x, weight
    and bias with the straight-through estimator (the quantisers count as the identity).  x [..., K], weight [N, K].
    Any number of tokens; where x has a gradient, up to 1,398,080 (fp32) or 2,097,088 (bf16, fp16) output features.

    What a graph captures: the pass may be captured together with its gradients; as with every torch module, an eager graph of
    the same leaf tensors must not be alive then (let go of earlier losses first, or use torch.autograd.grad)."""
    L.need_gpu(x, weight, bias)
    _type(x, "x")
    _type(weight, "weight")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or x.device != weight.device:
        raise ValueError(f"cannot apply a weight of shape {tuple(weight.shape)} on {weight.device} to {tuple(x.shape)} on {x.device}")
    _check_bias(bias, weight.shape[0], x.device)
    if weight.shape[0] > _MOST_OUTS[x.dtype] and x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{weight.shape[0]} output features are too many for the gradient of a {x.dtype} x (at most {_MOST_OUTS[x.dtype]})")
    return _Int8LinearFn.apply(x, weight, bias)


class Int8Linear(nn.Module):
    """A linear layer trained through its 8-bit form (see `int8_linear`); the weight stays in floating point."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.weight = nn.Parameter(torch.randn(out_features, in_features) * 0.1)
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return int8_linear(x, self.weight, self.bias)

    @torch.no_grad()
    def get_quantized_weights(self) -> Dict[str, torch.Tensor]:
        """weight int8 [out, in], scale fp32 [out] and the bias: what `Int8Inference` serves."""
        q, s = quantize_rows_int8(self.weight)
        out = {"weight": q, "scale": s}
        if self.bias is not None:
            out["bias"] = self.bias.detach().clone()
        return out


class Int8Inference:
    """Serves a linear layer from 8-bit weights: tokens are quantised on the way.  `weights`: "weight" int8 [N, K],
    "scale" float32 [N] and, optionally, "bias" [N], as `Int8Linear.get_quantized_weights` gives them.  The weights are laid
    out once, here; they are a copy, and later changes of the tensors that were passed do not show."""

    def __init__(self, weights: Dict[str, torch.Tensor]):
        w, s, b = weights["weight"], weights["scale"], weights.get("bias")
        L.need_gpu(w, s, b)
        if w.dtype != torch.int8 or w.dim() != 2:
            raise ValueError(f"weight must be an int8 matrix, got {w.dtype} {tuple(w.shape)}")
        n, k = w.shape
        if k < 1 or k > 131071:
            raise ValueError(f"{k} input features; 1 to 131071 keep the 32-bit sum exact")
        self.out_features, self.in_features, self.device = n, k, w.device
        # held where nobody rebinds them: the calls pass their addresses
        self._image = torch.zeros(n, _row_bytes(k), dtype=torch.int8, device=w.device)
        self._image[:, :k] = w
        self._scale = _check_scale(s, n, w.device, "scale").detach().clone()
        bc, self._bias_type = _check_bias(b, n, w.device)
        self._bias = None if bc is None else bc.detach().clone()
        self._w = (self._image.data_ptr(), self._scale.data_ptr(), 0 if self._bias is None else self._bias.data_ptr())
        self._fn = L.entry("dpd_int8_linear")
        self._index = self.device.index

    # what is served, to look at; other weights are another engine
    image = property(lambda self: self._image)
    scale = property(lambda self: self._scale)
    bias = property(lambda self: self._bias)

    def __call__(self, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [..., K] -> [..., N] in the type of x.  `out` (optional: [..., N], contiguous, the type of x, apart from x in
        memory, from its first element to its last) receives the result in place of a new tensor."""
        k, n = self.in_features, self.out_features
        t = TYPES.get(x.dtype)
        if t is None:
            _type(x, "x")
        shape = x.shape
        if not shape or shape[-1] != k:
            raise ValueError(f"expected {k} input features, got {tuple(shape)}")
        if x.device != self.device:
            raise RuntimeError(f"the weights are on {self.device}, the tokens on {x.device}")
        L.refuse_gradient("Int8Inference (training: Int8Linear)", x)
        x2, ldx = _rows(x)
        m = x2.shape[0]
        if out is None:
            out = torch.empty((*shape[:-1], n), dtype=x.dtype, device=self.device)
        elif out.shape != (*shape[:-1], n) or out.dtype != x.dtype or not out.is_contiguous() or out.device != x.device or out.requires_grad:
            raise RuntimeError(f"out must be a contiguous {x.dtype} tensor of shape {(*shape[:-1], n)} on {x.device} without gradient")
        elif m:
            at, to, size = x2.data_ptr(), out.data_ptr(), x.element_size()
            if at < to + m * n * size and to < at + ((m - 1) * ldx + k) * size:
                raise RuntimeError("out must not share memory with x")
        qw, sw, b = self._w
        with L.device(x):
            args = (x2.data_ptr(), t, m, k, ldx, qw, sw, b, self._bias_type, n, out.data_ptr(), n)
            stream = L.raw_stream(self._index)
            rc = self._fn(*args, 0, 0, stream) if m <= 32 else _NEEDS_WORKSPACE
            if rc == _NEEDS_WORKSPACE:       # the tokens are quantised by a launch of their own
                nbytes = m * _row_bytes(k) + (m * 4 + 255) // 256 * 256 + 256        # dpd_int8_linear_workspace_bytes
                ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
                rc = self._fn(*args, ws.data_ptr(), nbytes, stream)
            if rc:
                L.check(rc)
        return out

"""Orthogonalised updates: the Newton-Schulz iteration that takes the singular values of a matrix towards one
(csrc/orthogonal.hip).  The critic's spectral normalisation bounds the largest singular value of a weight; this spreads all
of an update's.  The reference has no counterpart."""
import ctypes
from functools import lru_cache
from typing import Optional, Sequence, Tuple, Union

import torch

from .. import _lib as L

Coefficients = Union[Tuple[float, float, float], Sequence[Tuple[float, float, float]]]
COEFFICIENTS = (3.4445, -4.7750, 2.0315)      # steep at zero: singular values end between about 0.7 and 1.2


@lru_cache(maxsize=64)
def _table(coefficients, steps: int):
    rows = coefficients if coefficients and isinstance(coefficients[0], tuple) else (coefficients,) * steps
    if len(rows) != steps or any(not isinstance(r, tuple) or len(r) != 3 for r in rows):
        raise ValueError(f"coefficients must be one triple (a, b, c) or one for each of {steps} steps")
    flat = [float(v) for r in rows for v in r]
    return (ctypes.c_float * len(flat))(*flat)


def coefficient_table(coefficients: Coefficients, steps: int):
    """steps triples as a host array; one triple serves every step."""
    if not 1 <= int(steps) <= 32:
        raise ValueError(f"steps must be 1 to 32, got {steps}")
    if type(coefficients) is not tuple or (coefficients and type(coefficients[0]) is list):
        coefficients = tuple(tuple(v) if isinstance(v, (tuple, list)) else v for v in coefficients)
    return _table(coefficients, int(steps))


def orthogonalize(x: torch.Tensor, steps: int = 5, coefficients: Coefficients = COEFFICIENTS, eps: float = 1e-7,
                  accurate: Optional[bool] = None) -> torch.Tensor:
    """The Newton-Schulz iterate of each matrix of x [..., rows, cols] in the type of x:

        X <- X / max(|X|_F, eps);   `steps` times:  A = X X^T,  X <- a X + (b A + c A A) X

    (on the transposed matrix where rows > cols).  `coefficients`: one triple (a, b, c), or one for each step; triples that
    could take a singular value above 3.9 raise ValueError.  `accurate`: fp32 accuracy (the default: 22 bits
    of every entry above 2^-28 of its matrix's norm, an absolute 2^-50 of the norm below), or, with False,
    factors rounded to fp16 with sums in fp32, in a third of the time where the products are large (4096 x 4096: 1.3 instead of
    4.2 ms; a bf16 matrix comes out 1.9e-3 off, of which the rounding to its type is 1.7e-3; small singular values next to large
    ones feel the factors' rounding more, since the iteration amplifies them).  Matrices of up to 64 x 128 are
    always computed in fp32.  A matrix that holds a NaN or an infinity comes out as NaN.  Not differentiable."""
    L.need_gpu(x)
    if x.dtype not in L.TYPES:
        raise RuntimeError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() < 2:
        raise ValueError(f"expected matrices [..., rows, cols], got {tuple(x.shape)}")
    L.refuse_gradient("orthogonalize", x)
    coef = coefficient_table(coefficients, steps)
    xc = x.detach().contiguous()
    rows, cols = x.shape[-2:]
    batch = x.shape[:-2].numel()
    out = torch.empty_like(xc)
    acc = int(accurate is None or bool(accurate))
    with L.device(x):
        nbytes = L.entry("dpd_orthogonalize_workspace_bytes")(batch, rows, cols, acc)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        L.check(L.entry("dpd_orthogonalize")(xc.data_ptr(), L.TYPES[x.dtype], batch, rows, cols, int(steps), coef, float(eps), acc, out.data_ptr(),
                                             ws.data_ptr(), nbytes, L.raw_stream(x.device.index)))
    return out

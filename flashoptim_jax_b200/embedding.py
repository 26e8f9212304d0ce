"""Embedding lookup on the weights as this package keeps them, and its gradient by sorted tokens, on the GPU.

The reference takes the gradients of a pytree as they come.  That of an embedding table, the largest leaf of a language
model, is no matrix product but a sum of rows by token: `embed_grad` makes it in the leaf's layout, in one fixed order, rounded once,
or adds it to what a tied output head left there; a leaf of `grads` may also be a `TokenGradient`, which `tx.step` and
`clip_by_global_norm` turn into it.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any, List, Optional, Tuple

import torch

from . import _lib
from . import tree as pytree
from ._dev import DTYPE_CODE, ECC_BITS_OF, LOW_PRECISION, as_tensor, dtype_name, refuse_tangent, require_cuda, stream_ptr
from .dropping import checked_dropout, fill_dropout

_IDS_BITS = {torch.int32: 32, torch.int64: 64}
_MOST_STRIDE = 2**28


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """A matrix whose rows are without gaps, and the distance between them in elements."""
    rows, dim = t.shape
    stride = t.stride(0) if rows > 1 else dim
    if (dim > 1 and t.stride(1) != 1) or stride < dim or stride >= _MOST_STRIDE:
        t, stride = t.contiguous(), dim
    return t, stride


def _check_ids(ids: Any, device: torch.device) -> None:
    require_cuda(ids, "ids")
    if ids.dtype not in _IDS_BITS:
        raise ValueError(f"ids must be int32 or int64, got {dtype_name(ids.dtype)}")
    if ids.device != device:
        raise ValueError(f"ids live on {ids.device}, not on {device}")


def _check_scale(scale) -> float:
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    return scale


def _lookup(table, ids, ecc, scale, p, seed, offset, dtype) -> torch.Tensor:
    p, seed, host_offset, on_device = checked_dropout(p, seed, offset, table.device)
    rows, dim = table.shape
    ids = ids.contiguous()
    out = torch.empty((*ids.shape, dim), dtype=dtype, device=table.device)
    table, stride = _rows(table)
    f = _lib.FoEmbed(struct_size=ctypes.sizeof(_lib.FoEmbed), table_dtype=DTYPE_CODE[table.dtype], out_dtype=DTYPE_CODE[dtype], ids_bits=_IDS_BITS[ids.dtype],
                     table=table.data_ptr(), ids=ids.data_ptr(), out=out.data_ptr(), n_tokens=ids.numel(), rows=rows, dim=dim, row_stride=stride, scale=scale)
    if ecc is not None:
        ecc, f.ecc_stride = _rows(ecc)
        f.ecc, f.ecc_bits = ecc.data_ptr(), ECC_BITS_OF[ecc.dtype]
    fill_dropout(f.dropout, p, seed, host_offset, on_device)
    with torch.cuda.device(table.device):
        _lib.check(_lib.lib().fo_embed(ctypes.byref(f), stream_ptr(table.device)))
    return out


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, ecc, scale, p, seed, offset, dtype):
        on_device = isinstance(offset, torch.Tensor)
        ctx.how = (table.shape[0], table.dtype, scale, p, seed, None if on_device else offset)
        ctx.save_for_backward(ids, *([offset] if on_device else []))
        return _lookup(table, ids, ecc, scale, p, seed, offset, dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        rows, dtype, scale, p, seed, offset = ctx.how
        ids, *rest = ctx.saved_tensors
        grad = embed_grad(dy, ids, rows, scale=scale, p=p, seed=seed, offset=rest[0] if offset is None else offset, dtype=dtype)
        return grad, None, None, None, None, None, None, None


def embed(table: torch.Tensor, ids: torch.Tensor, *, scale: float = 1.0, ecc: Optional[torch.Tensor] = None, p: float = 0.0, seed: int = 0,
          offset=0, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """scale * table[ids], with dropout of probability `p` (seed and offset as for `dropout`): shape ids.shape + (dim,).

    `table`: (rows, dim) in float32, bfloat16 or float16.  With `ecc`, the error-correction codes of the same leaf in the optimizer state, the rows
    are the fp32 weights that `reconstruct_leaf` gives; the 0-d marker of a leaf without codes is taken for none.  The result has the table's dtype, with
    `ecc` fp32; `dtype` may ask for either.  scale / (1 - p), one factor in fp32, has to be 0 or a normal
    fp32 number.  `ids`: int32 or int64.  A negative id is no token: its row is 0 and it has no part in the
    gradient.  An id behind the last row cannot be reported without waiting for the GPU: its row is NaN, which the loss shows.
    Differentiable in the table (once, in reverse mode): the gradient is `embed_grad`'s, in the table's dtype.  A step that is captured in a CUDA graph calls
    `embed_grad` by hand."""
    if dtype is None:
        out = _lib.host().embed(table, ids, ecc, scale, p, seed, offset)  # None: something to differentiate or convert first, or an error to report
        if out is not None:
            return out
    require_cuda(table, "table")
    refuse_tangent(table, "table")
    if table.dim() != 2 or table.dtype not in DTYPE_CODE:
        raise ValueError(f"table must be a float32, bfloat16 or float16 matrix, got shape {tuple(table.shape)}, {dtype_name(table.dtype)}")
    _check_ids(ids, table.device)
    if ecc is not None:
        ecc = as_tensor(ecc)
        if ecc.dim() == 0 and ecc.dtype == torch.int32:
            ecc = None
        elif ecc.dtype not in ECC_BITS_OF or table.dtype not in LOW_PRECISION or ecc.shape != table.shape or ecc.device != table.device:
            raise ValueError(f"ecc of shape {tuple(ecc.shape)}, {dtype_name(ecc.dtype)}, on {ecc.device} does not belong to a table of shape "
                             f"{tuple(table.shape)}, {dtype_name(table.dtype)}, on {table.device}")
    if dtype is None:
        dtype = table.dtype if ecc is None else torch.float32
    elif dtype not in (table.dtype, torch.float32):
        raise ValueError(f"dtype must be the table's ({dtype_name(table.dtype)}) or float32, got {dtype_name(dtype)}")
    scale = _check_scale(scale)
    if torch.is_grad_enabled() and table.requires_grad:
        checked_dropout(p, seed, offset, table.device)
        return _Embed.apply(table, ids, ecc, scale, p, seed, offset, dtype)
    return _lookup(table, ids, ecc, scale, p, seed, offset, dtype)


def embed_grad(dy: torch.Tensor, ids: torch.Tensor, rows: int, *, scale: float = 1.0, p: float = 0.0, seed: int = 0, offset=0,
               dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """Gradient of `embed(table, ids, ...)` for a table of `rows` rows, given that of its result: (rows, dim), in dy's dtype or `dtype`.

    Row v is the sum of scale * dropout(dy) over the tokens with id v, in fp32 and in an order fixed by the ids, the sizes, `accumulate` and whether there is
    dropout (same inputs, same bits), rounded once; rows without a token are 0.  Into `out` where it is given (a leaf of `Zero1Optimizer.grads`, say); with `accumulate` the sums
    go on from what `out` holds (the gradient that the output head of a tied model left there, or an earlier micro-batch's), and rows without a
    token are not written.  `out` must not overlap dy, nor require a gradient (but under torch.no_grad()).  Not differentiable
    itself."""
    if dtype is None:
        grad = _lib.host().embed_grad(dy, ids, rows, scale, p, seed, offset, out, accumulate)  # None: something to convert first, or an error to report
        if grad is not None:
            return grad
    require_cuda(dy, "dy")
    refuse_tangent(dy, "dy")
    _check_ids(ids, dy.device)
    if dy.dtype not in DTYPE_CODE:
        raise ValueError(f"dy must be float32, bfloat16 or float16, got {dtype_name(dy.dtype)}")
    if dy.dim() != ids.dim() + 1 or dy.shape[:-1] != ids.shape:
        raise ValueError(f"dy of shape {tuple(dy.shape)} does not belong to ids of shape {tuple(ids.shape)}")
    rows = int(rows)
    if rows < 0:
        raise ValueError(f"rows must not be negative, got {rows}")
    dim = dy.shape[-1]
    scale = _check_scale(scale)
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs the gradient to add to: give it as out")
        dtype = dy.dtype if dtype is None else dtype
        if dtype not in DTYPE_CODE:
            raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype_name(dtype)}")
    else:
        require_cuda(out, "out")
        refuse_tangent(out, "out")
        if out.requires_grad and torch.is_grad_enabled():  # (as torch's own operators with out=)
            raise RuntimeError("embed_grad writes into out behind autograd's back, but out requires a gradient")
        if tuple(out.shape) != (rows, dim) or out.dtype not in DTYPE_CODE or (dtype is not None and out.dtype != dtype) or out.device != dy.device:
            raise ValueError(f"out of shape {tuple(out.shape)}, {dtype_name(out.dtype)}, on {out.device} is not a gradient of shape {(rows, dim)} on {dy.device}")
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
    p, seed, host_offset, on_device = checked_dropout(p, seed, offset, dy.device)
    ids = ids.contiguous()
    n = ids.numel()
    dy, stride = _rows(dy.reshape(n, dim))
    need = ctypes.c_uint64()
    lib = _lib.lib()
    _lib.check(lib.fo_embed_grad_workspace(rows, dim, n, ctypes.byref(need)))
    grad = torch.empty((rows, dim), dtype=dtype, device=dy.device) if out is None else out
    workspace = torch.empty(need.value, dtype=torch.uint8, device=dy.device)  # its own: streams do not share one
    f = _lib.FoEmbedGrad(struct_size=ctypes.sizeof(_lib.FoEmbedGrad), dy_dtype=DTYPE_CODE[dy.dtype], out_dtype=DTYPE_CODE[grad.dtype], ids_bits=_IDS_BITS[ids.dtype],
                         accumulate=int(bool(accumulate)), dy=dy.data_ptr(), ids=ids.data_ptr(), out=grad.data_ptr(), n_tokens=n, rows=rows, dim=dim,
                         dy_stride=stride, scale=scale, workspace=workspace.data_ptr(), workspace_bytes=need.value)
    fill_dropout(f.dropout, p, seed, host_offset, on_device)
    with torch.cuda.device(dy.device):
        _lib.check(lib.fo_embed_grad(ctypes.byref(f), stream_ptr(dy.device)))
    if out is not None and not out.is_inference():
        torch.autograd.graph.increment_version(out)
    return grad


class TokenGradient:
    """The gradient of an embedding table as the backward pass has it: that of the looked-up rows, and their ids.

    Stands in the place of the table's leaf in the `grads` of `tx.step`, `clip_by_global_norm(...).step` and `Zero1Optimizer.step`, which make the leaf's
    gradient from it with `embed_grad`; the arguments are those of the lookup."""

    __slots__ = ("dy", "ids", "scale", "p", "seed", "offset")

    def __init__(self, dy: torch.Tensor, ids: torch.Tensor, *, scale: float = 1.0, p: float = 0.0, seed: int = 0, offset=0):
        self.dy, self.ids, self.scale, self.p, self.seed, self.offset = dy, ids, scale, p, seed, offset

    def dense(self, param: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The gradient of `param`, a table of (rows, dim)."""
        if param.dim() != 2 or self.dy.dim() == 0 or self.dy.shape[-1] != param.shape[1]:
            raise ValueError(f"a TokenGradient of rows of {tuple(self.dy.shape)[-1:]} does not belong to a parameter of shape {tuple(param.shape)}")
        return embed_grad(self.dy, self.ids, param.shape[0], scale=self.scale, p=self.p, seed=self.seed, offset=self.offset, out=out)


def has_tokens(leaves: List[Any]) -> bool:
    return any(type(g) is TokenGradient for g in leaves)


def dense_leaves(params: List[Any], grads: List[Any]) -> List[Any]:
    """Leaves of gradients with every TokenGradient replaced by the gradient of its parameter; the same list where there is none."""
    if not has_tokens(grads):
        return grads
    return [g.dense(as_tensor(p)) if type(g) is TokenGradient else g for g, p in zip(grads, params)]


def dense_gradients(params: Any, grads: Any) -> Any:
    """`grads` with every TokenGradient in it replaced by the gradient of its leaf of `params`; the same object where there is none."""
    if not has_tokens(pytree.tree_leaves(grads)):
        return grads
    leaves, treedef = pytree.tree_flatten(grads)
    param_leaves, param_def = pytree.tree_flatten(params)
    if treedef != param_def:
        return grads  # (refused where the trees are compared)
    return treedef.unflatten(dense_leaves(param_leaves, leaves))

"""Embedding lookup with scaling (``m3_embed``) and its gradient by sorted tokens (``m3_embed_bwd``).

`embed_tokens` is ``(scale * table[tokens]).to(dtype)`` with one rounding and no intermediate
copy; its gradient sums each token's rows in the order of their positions, in fp32, so that it
is the same every run.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _capi as C
from . import _tensors as T

_MOST_VOCAB = 2 ** 31 - 1


def _check_tokens(tokens, ref):
    """The tokens as the kernels read them (int64)."""
    T.require_here(ref.device, tokens)
    if tokens.dtype != torch.int64:
        if tokens.dtype != torch.int32:
            raise ValueError(f"tokens must be int64 or int32, got {tokens.dtype}")
        tokens = tokens.to(torch.int64)
    return tokens


def _lookup(table, tokens, scale, dtype):
    lead, dev = tokens.shape, table.device
    vocab, dim = table.shape
    outer, inner = T.row_counts(lead)
    tokens, (t_outer, t_inner) = T.row_input(tokens, len(lead))
    ld, unit = table.stride()
    if unit != 1 or ld < dim:
        table = table.detach().contiguous()
        ld = dim
    out = torch.empty((*lead, dim), dtype=dtype, device=dev)
    a = C.M3EmbedArgs(outer, inner, vocab, dim, T.io_dtype(table.dtype), T.io_dtype(dtype), scale, 0,
                      tokens.data_ptr(), t_outer, t_inner, table.data_ptr(), ld, out.data_ptr(), dim)
    T.call(C.lib().m3_embed, a, dev)
    return out


class _EmbedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale, dtype):
        ctx.save_for_backward(tokens)
        ctx.vocab, ctx.scale, ctx.dtype = table.shape[0], scale, table.dtype
        return _lookup(table, tokens, scale, dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        tokens, = ctx.saved_tensors
        return embedding_grad(dy, tokens, ctx.vocab, scale=ctx.scale, dtype=ctx.dtype), None, None, None


def embed_tokens(table: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0,
                 dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``table (V, D)`` bf16 or f32, ``tokens (...)`` int -> ``(..., D)`` in ``dtype`` (the table's
    by default).  A negative token is padding: a zero row without gradient; one at or past V
    gives a NaN row.  Differentiable in ``table``, once and in reverse mode (a dense gradient in its
    dtype)."""
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError(f"table must be (vocab, dim), got {tuple(table.shape)}")
    T.vocab_of(table.shape[0], _MOST_VOCAB)
    T.no_tangent("embed_tokens", table)
    tokens = _check_tokens(tokens, table)
    dtype = table.dtype if dtype is None else dtype
    if table.requires_grad and torch.is_grad_enabled():
        return _EmbedFn.apply(table, tokens, float(scale), dtype)
    return _lookup(table, tokens, scale, dtype)


def embedding_grad(dy: torch.Tensor, tokens: torch.Tensor, vocab: int, scale: float = 1.0,
                   dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of `embed_tokens` with respect to its table: ``dy (..., D)`` -> ``(vocab, D)``
    in ``dtype``.  With ``out`` it is added to that ``(vocab, D)`` tensor instead (only the rows
    of tokens that occur are touched; each sum is rounded once), e.g. the gradient a tied head
    has left there.  It shares no memory with ``dy``, and its version is raised."""
    if dy.dim() != tokens.dim() + 1 or dy.shape[:-1] != tokens.shape or dy.shape[-1] < 1:
        raise ValueError(f"dy must be {tuple(tokens.shape)} + (dim,), got {tuple(dy.shape)}")
    T.vocab_of(vocab, _MOST_VOCAB)
    tokens = _check_tokens(tokens, dy)
    lead, dim, dev = tokens.shape, dy.shape[-1], dy.device
    add = out is not None
    if not add:
        out = torch.empty((vocab, dim), dtype=dtype, device=dev)
    elif out.shape != (vocab, dim) or out.device != dev or (dim > 1 and out.stride(1) != 1) or out.stride(0) < dim:
        raise ValueError(f"out must be ({vocab}, {dim}) on {dev} with contiguous rows")
    elif out.requires_grad and out.is_leaf and torch.is_grad_enabled():
        raise ValueError("out must not be a leaf that requires grad")
    nd = len(lead)
    outer, inner = T.row_counts(lead)
    tokens, (t_outer, t_inner) = T.row_input(tokens, nd)
    dy, (dy_outer, dy_inner) = T.row_input(dy, nd)
    if add and not T.apart(dy, out):
        raise ValueError("out must share no memory with dy")
    lib = C.lib()
    size = lib.m3_embed_bwd_workspace_size(outer * inner, dim)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    a = C.M3EmbedBwdArgs(outer, inner, vocab, dim, T.io_dtype(dy.dtype), T.io_dtype(out.dtype), scale, int(add),
                         tokens.data_ptr(), t_outer, t_inner, dy.data_ptr(), dy_outer, dy_inner, out.data_ptr(),
                         out.stride(0), ws.data_ptr(), size)
    T.call(lib.m3_embed_bwd, a, dev)
    if add:
        T.written(out)
    return out

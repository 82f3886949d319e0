"""Embedding of tokens, its gradient, and the grouping of ids both the gradient and a router's dispatch need, over the C ABI
(``loops_embedding_*``, ``loops_group_tokens``): the product of a token matrix (tokens x rows of a table, one 1 per token) with
the table, and of its transpose with the gradient of the result.

``lookup`` -> ``out[t] = scale * table[token - first_id]``; ``group_tokens`` sorts the positions by id; ``gradient`` sums the gradient
rows of every id.  Tables, gradients and results are float32, float16 or bfloat16, token ids int32 or int64.  An id outside
``[first_id, first_id + rows)`` (padding, another rank's shard of the vocabulary) gives a zero row and takes no part in the gradient.
Calls are asynchronous on the current stream of the tensors' device and may be captured into a graph; there is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib as L

VALUE_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # enum loops_value_type
INDEX_TYPES = {torch.int32: 0, torch.int64: 1}  # enum loops_index_type


def value_type(t: torch.Tensor, what: str) -> int:
    v = VALUE_TYPES.get(t.dtype)
    if v is None:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, not {t.dtype}")
    return v


def index_type(t: torch.Tensor, what: str) -> int:
    v = INDEX_TYPES.get(t.dtype)
    if v is None:
        raise TypeError(f"{what} must be int32 or int64, not {t.dtype}")
    return v


def require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def same_device(first: torch.Tensor, *others: Optional[torch.Tensor]) -> torch.device:
    device = first.device
    require(device.type == "cuda", "tensors must be on the GPU")
    for t in others:
        require(t is None or t.device == device, "tensors must be on one device")
    return device


def pitch_of(t: torch.Tensor, what: str) -> int:
    """Elements between the rows of a matrix with unit column stride."""
    require(t.dim() == 2, f"{what} must have two dimensions")
    rows, cols = t.shape
    at, step = t.stride()
    if rows <= 1 or cols == 0:
        at = cols
        step = 1 if rows == 0 else step
    require((step == 1 or cols <= 1) and at >= cols, f"{what}: columns must be adjacent and rows must not overlap")
    return at


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory between the first and the last element of one tensor meets the other's."""
    def ends(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = ends(a), ends(b)
    return a0 < b1 and b0 < a1


def launch(device: torch.device, name: str, *args) -> None:
    """The C entry point on the current stream of `device` (appended as the last argument)."""
    index = device.index
    fn = getattr(L.lib(), name)
    if index == torch.cuda.current_device():
        code = fn(*args, torch.cuda.current_stream(index).cuda_stream)
    else:
        with torch.cuda.device(index):
            code = fn(*args, torch.cuda.current_stream(index).cuda_stream)
    if code:
        L.check(code, name)


def workspace(device: torch.device, name: str, *args):
    """(tensor or None, pointer, bytes): scratch of a call, from torch's allocator -- one per call, ordered by the stream."""
    size = C.c_size_t(0)
    L.check(getattr(L.lib(), name)(*args, C.byref(size)), name)
    if size.value == 0:
        return None, None, 0
    t = torch.empty(size.value, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), size.value


def lookup(table: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0, first_id: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[..., :] = scale * table[tokens[...] - first_id, :]``, zeros for ids the table does not hold.

    ``table``: [rows, dim], columns adjacent, any distance between rows.  ``tokens``: any shape, contiguous.  ``out``:
    [*tokens.shape, dim] (or [tokens, dim] with any distance between rows) of the table's type; made when not given."""
    value, index = value_type(table, "table"), index_type(tokens, "tokens")
    pitch = pitch_of(table, "table")
    require(tokens.is_contiguous(), "tokens must be contiguous")
    require(first_id >= 0, "first_id must not be negative")
    device = same_device(table, tokens, out)
    rows, dim = table.shape
    n = tokens.numel()
    if out is None:
        out = torch.empty(*tokens.shape, dim, dtype=table.dtype, device=device)
        out_pitch = dim
    else:
        require(out.dtype is table.dtype and tuple(out.shape) in ((*tokens.shape, dim), (n, dim)), "out must be [*tokens.shape, dim] of the table's type")
        out_pitch = pitch_of(out if out.dim() == 2 else out.view(n, dim), "out")
        require(not overlap(out, table) and not overlap(out, tokens), "out must not overlap the inputs")
    launch(device, "loops_embedding_lookup", value, index, rows, dim, table.data_ptr(), pitch, n, tokens.data_ptr(), first_id, scale, out.data_ptr(),
           out_pitch)
    return out


class TokenGroups(NamedTuple):
    """Positions in the order of their ids (``group_tokens``)."""
    ids: torch.Tensor        # int32 [tokens]: id - first_id, ascending; `rows` for tokens without a row
    positions: torch.Tensor  # int32 [tokens]: where they stand in the flattened tokens, ascending within an id
    rows: int


def group_tokens(tokens: torch.Tensor, rows: int, first_id: int = 0, drop_id: int = -1) -> TokenGroups:
    """The positions of ``tokens`` (any shape, contiguous) sorted by id, stably; ids outside [first_id, first_id + rows) and ``drop_id``
    (a padding id; -1: none) become ``rows`` and stand at the end."""
    index = index_type(tokens, "tokens")
    require(tokens.is_contiguous(), "tokens must be contiguous")
    require(first_id >= 0 and rows >= 0, "first_id and rows must not be negative")
    device = same_device(tokens)
    n = tokens.numel()
    both = torch.empty(2, n, dtype=torch.int32, device=device)
    ids, positions = both[0], both[1]
    _keep, ws, size = workspace(device, "loops_group_tokens_workspace", n, rows)
    launch(device, "loops_group_tokens", index, n, tokens.data_ptr(), rows, first_id, drop_id, ids.data_ptr(), positions.data_ptr(), ws, size)
    return TokenGroups(ids, positions, rows)


def gradient(groups: TokenGroups, grad: torch.Tensor, scale: float = 1.0, dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
             accumulate: bool = False) -> torch.Tensor:
    """``out[v, :] = scale * sum of grad[t, :] over the tokens t of row v``: the gradient of ``lookup``'s table from the gradient of its
    result, for the tokens that ``groups`` was made of.

    ``grad``: [tokens, dim] with any distance between rows, or [*tokens.shape, dim] contiguous.  ``out``: [rows, dim] in grad's type or
    float32 (``dtype`` when it is made here).  ``accumulate``: add to what ``out`` holds in the rows that have tokens and leave the
    others.  Sums are held in float32 and rounded once; their order is fixed."""
    value = value_type(grad, "grad")
    n, rows = groups.ids.numel(), groups.rows
    require(grad.dim() >= 1, "grad must have the tokens' shape and a last dimension")
    dim = grad.shape[-1]
    if grad.dim() != 2:
        require(grad.is_contiguous(), "grad of more than two dimensions must be contiguous")
        grad = grad.view(grad.numel() // dim if dim else n, dim)
    require(grad.shape[0] == n, "grad must have a row for each token")
    pitch = pitch_of(grad, "grad")
    device = same_device(grad, groups.ids, groups.positions, out)
    if out is None:
        require(not accumulate, "accumulate needs out")
        out = torch.empty(rows, dim, dtype=grad.dtype if dtype is None else dtype, device=device)
    else:
        require(dtype is None or out.dtype is dtype, "out has another type than dtype")
        require(tuple(out.shape) == (rows, dim), "out must be [rows, dim]")
        require(not overlap(out, grad) and not overlap(out, groups.ids) and not overlap(out, groups.positions), "out must not overlap the inputs")
    if out.dtype is not grad.dtype and out.dtype is not torch.float32:
        raise TypeError("out must have grad's type or float32")
    out_pitch = pitch_of(out, "out")
    add = 1 if accumulate else 0
    _keep, ws, size = workspace(device, "loops_embedding_gradient_workspace", value, n, rows, dim, add)
    launch(device, "loops_embedding_gradient", value, VALUE_TYPES[out.dtype], n, groups.ids.data_ptr(), groups.positions.data_ptr(), rows, dim,
           grad.data_ptr(), pitch, scale, add, out.data_ptr(), out_pitch, ws, size)
    return out

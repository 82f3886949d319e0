"""Embedding of tokens, its gradient, and the grouping of ids both the gradient and a router's dispatch need, over the C ABI
(``loops_embedding_*``, ``loops_group_tokens``): the product of a token matrix (tokens x rows of a table, one 1 per token) with
the table, and of its transpose with the gradient of the result.

``lookup`` -> ``out[t] = scale * table[token - first_id]``; ``group_tokens`` sorts the positions by id; ``gradient`` sums the gradient
rows of every id.  Tables, gradients and results are float32, float16 or bfloat16, token ids int32 or int64.  An id outside
``[first_id, first_id + rows)`` (padding, another rank's shard of the vocabulary) gives a zero row and takes no part in the gradient.
Calls are asynchronous on the current stream of the tensors' device and may be captured into a graph; there is no CPU path.  Arguments
of a wrong type raise TypeError, of a wrong shape or layout ValueError; what the library itself refuses (an output that overlaps an
input, sizes beyond its range) LoopsError.

Autograd records none of these calls; the gradients are calls of their own.  A table that requires a gradient is therefore refused
(ValueError) where autograd records, as is any ``out`` that does: call under ``torch.no_grad()``, on ``table.detach()``, or from the forward
and backward of a ``torch.autograd.Function``, where it does not.
"""
from __future__ import annotations

import ctypes as C
import functools
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


def same_device(first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """The index of the GPU that holds all of them."""
    if not first.is_cuda:
        raise ValueError("tensors must be on the GPU")
    device = first.get_device()
    for t in others:
        if t is not None and t.get_device() != device:  # (-1 on the CPU)
            raise ValueError("tensors must be on one device")
    return device


def pitch_of(t: torch.Tensor, what: str) -> int:
    """Elements between the rows of a matrix with adjacent columns."""
    if t.dim() != 2:
        raise ValueError(f"{what} must have two dimensions")
    rows, cols = t.shape
    pitch, step = t.stride()
    if rows == 0 or cols == 0:
        return cols
    if rows == 1:
        pitch = cols
    if (step != 1 and cols != 1) or pitch < cols:
        raise ValueError(f"{what}: columns must be adjacent and rows must not overlap")
    return pitch


def not_recorded(what: str) -> None:
    """Refuses a tensor that requires a gradient where autograd would record an operation on it: the gradient would be lost without an error."""
    if torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, which this call does not record: use torch.no_grad(), {what}.detach() or an autograd.Function")


INT_MAX = 2 ** 31 - 1
LONG_MAX = 2 ** 63 - 1


def c_int(name: str, *sizes: int) -> None:
    """Refuses sizes that the C entry point's int arguments do not hold."""
    if max(sizes) > INT_MAX or min(sizes) < -INT_MAX:
        L.check(-2, name)


_entries = {}


def launch(device: int, name: str, *args) -> None:
    """The C entry point on the current stream of `device` (appended as the last argument)."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(L.lib(), name)
    try:
        if device == torch._C._cuda_getDevice():
            code = fn(*args, torch._C._cuda_getCurrentRawStream(device))
        else:
            with torch.cuda.device(device):
                code = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    except C.ArgumentError as e:
        raise TypeError(f"{name}: {e}") from None
    if code:
        L.check(code, name)


@functools.lru_cache(maxsize=4096)
def workspace_bytes(name: str, *args) -> int:
    size = C.c_size_t(0)
    try:
        L.check(getattr(L.lib(), name)(*args, C.byref(size)), name)
    except C.ArgumentError as e:
        raise TypeError(f"{name}: {e}") from None
    return size.value


def workspace(device: int, name: str, *args):
    """(tensor or None, pointer, bytes): scratch of one call, from torch's allocator and so in the stream's order."""
    size = workspace_bytes(name, *args)
    if size == 0:
        return None, None, 0
    t = torch.empty(size, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), size


def lookup(table: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0, first_id: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[..., :] = scale * table[tokens[...] - first_id, :]``, zeros for ids the table does not hold.

    ``table``: [rows, dim], columns adjacent, any distance between rows.  ``tokens``: any shape, contiguous.  ``out``:
    [*tokens.shape, dim] contiguous (or [tokens, dim] with any distance between rows), of the table's type; made when not given."""
    value, index = value_type(table, "table"), index_type(tokens, "tokens")
    if table.requires_grad:
        not_recorded("table")
    if out is not None and out.requires_grad:
        not_recorded("out")
    pitch = pitch_of(table, "table")
    if not tokens.is_contiguous():
        raise ValueError("tokens must be contiguous")
    if not 0 <= first_id <= LONG_MAX:
        raise ValueError("first_id must not be negative or beyond 64 bits")
    device = same_device(table, tokens, out)
    rows, dim = table.shape
    n = tokens.numel()
    c_int("loops_embedding_lookup", n, rows, dim)
    if out is None:
        out = torch.empty(*tokens.shape, dim, dtype=table.dtype, device=device)
        out_pitch = dim
    else:
        if out.dtype is not table.dtype:
            raise TypeError("out must have the table's type")
        if tuple(out.shape) not in ((*tokens.shape, dim), (n, dim)) or (out.dim() != 2 and not out.is_contiguous()):
            raise ValueError("out must be [*tokens.shape, dim] contiguous, or [tokens, dim]")
        out_pitch = pitch_of(out, "out") if out.dim() == 2 else dim
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
    if not tokens.is_contiguous():
        raise ValueError("tokens must be contiguous")
    if rows < 0 or not 0 <= first_id <= LONG_MAX or not -LONG_MAX <= drop_id <= LONG_MAX:
        raise ValueError("first_id and rows must not be negative, ids not beyond 64 bits")
    device = same_device(tokens)
    n = tokens.numel()
    c_int("loops_group_tokens", n, rows)
    _keep, ws, size = workspace(device, "loops_group_tokens_workspace", n, rows)
    ids = torch.empty(n, dtype=torch.int32, device=device)
    positions = torch.empty(n, dtype=torch.int32, device=device)
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
    if out is not None and out.requires_grad:
        not_recorded("out")
    ids, positions, rows = groups
    n = ids.numel()
    if ids.dtype is not torch.int32 or positions.dtype is not torch.int32:
        raise TypeError("groups must hold int32")
    if positions.numel() != n or not ids.is_contiguous() or not positions.is_contiguous():
        raise ValueError("groups must hold as many ids as positions, contiguous")
    if grad.dim() == 0:
        raise ValueError("grad must have the tokens' shape and a last dimension")
    dim = grad.shape[-1]
    if grad.dim() != 2:
        if not grad.is_contiguous():
            raise ValueError("grad of other than two dimensions must be contiguous")
        grad = grad.view(grad.numel() // dim if dim else n, dim)
    if grad.shape[0] != n:
        raise ValueError("grad must have a row for each token")
    pitch = pitch_of(grad, "grad")
    device = same_device(grad, ids, positions, out)
    c_int("loops_embedding_gradient", n, rows, dim)
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = torch.empty(rows, dim, dtype=grad.dtype if dtype is None else dtype, device=device)
        out_pitch = dim
    else:
        if dtype is not None and out.dtype is not dtype:
            raise TypeError("out has another type than dtype")
        if out.shape != (rows, dim):
            raise ValueError("out must be [rows, dim]")
        out_pitch = pitch_of(out, "out")
    if out.dtype is not grad.dtype and out.dtype is not torch.float32:
        raise TypeError("out must have grad's type or float32")
    to, add = VALUE_TYPES[out.dtype], 1 if accumulate else 0
    _keep, ws, size = workspace(device, "loops_embedding_gradient_workspace", value, to, n, rows, dim, add)
    launch(device, "loops_embedding_gradient", value, to, n, ids.data_ptr(), positions.data_ptr(), rows, dim, grad.data_ptr(), pitch, scale, add,
           out.data_ptr(), out_pitch, ws, size)
    return out

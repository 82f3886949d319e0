"""What the embedding and routing entry points refuse, at the C boundary (before any runtime call, so the addresses are never read) and
in Python (tensors on the CPU): no GPU needed."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from loops_amd import _lib, embedding, routing

F32, F16, BF16, I32, I64 = 0, 1, 2, 0, 1
BADARG, RANGE, CONFIG = -1, -2, -3
A, B, D, G, H = (1 << 40, 2 << 40, 3 << 40, 4 << 40, 5 << 40)  # addresses far apart
BIG = 2 ** 31 - 1


def _lookup(value=F32, index=I64, rows=10, dim=8, table=A, pitch=8, tokens=5, ids=B, first=0, out=D, out_pitch=8):
    return _lib.lib().loops_embedding_lookup(value, index, rows, dim, table, pitch, tokens, ids, first, 1.0, out, out_pitch, None)


@pytest.mark.parametrize("change,code", [
    (dict(value=3), CONFIG), (dict(value=-1), CONFIG), (dict(index=2), CONFIG), (dict(rows=-1), BADARG), (dict(dim=-1), BADARG), (dict(tokens=-1), BADARG),
    (dict(pitch=7), BADARG), (dict(out_pitch=7), BADARG), (dict(first=-1), BADARG), (dict(first=2 ** 63 - 10), BADARG), (dict(table=None), BADARG),
    (dict(ids=None), BADARG), (dict(out=None), BADARG),
    (dict(out=A + 4), BADARG), (dict(out=A - 4), BADARG), (dict(out=A + 10 * 8 * 4 - 4), BADARG), (dict(out=B + 5 * 8 - 4), BADARG), (dict(out=B - 5 * 8 * 4 + 4), BADARG),
    (dict(tokens=0, table=None, ids=None, out=None), 0), (dict(dim=0, pitch=0, out_pitch=0, table=None, ids=None, out=None), 0),
])
def test_lookup(change, code):
    assert _lookup(**change) == code


def _group(index=I64, tokens=9000, ids=A, rows=100, first=0, out=B, positions=D, ws=G, size=1 << 30):
    return _lib.lib().loops_group_tokens(index, tokens, ids, rows, first, -1, out, positions, ws, size, None)


@pytest.mark.parametrize("change,code", [
    (dict(index=2), CONFIG), (dict(tokens=-1), BADARG), (dict(rows=-1), BADARG), (dict(first=-1), BADARG), (dict(first=2 ** 63 - 50), BADARG),
    (dict(tokens=BIG - 100), RANGE), (dict(tokens=2 ** 30, rows=2 ** 30), RANGE), (dict(ids=None), BADARG), (dict(out=None), BADARG),
    (dict(positions=None), BADARG), (dict(ws=None), BADARG), (dict(size=100), BADARG), (dict(out=A + 8), BADARG), (dict(positions=A - 8), BADARG),
    (dict(positions=B + 8999 * 4), BADARG), (dict(tokens=0, ids=None, out=None, positions=None, ws=None, size=0), 0),
])
def test_group_tokens(change, code):
    assert _group(**change) == code


def _gradient(value=BF16, to=F32, tokens=2000, ids=A, positions=B, rows=30, dim=16, grad=D, pitch=16, add=0, out=G, out_pitch=16, ws=H, size=1 << 40):
    return _lib.lib().loops_embedding_gradient(value, to, tokens, ids, positions, rows, dim, grad, pitch, 1.0, add, out, out_pitch, ws, size, None)


@pytest.mark.parametrize("change,code", [
    (dict(value=3), CONFIG), (dict(value=F32, to=BF16), CONFIG), (dict(value=F16, to=BF16), CONFIG), (dict(tokens=-1), BADARG), (dict(rows=-1), BADARG),
    (dict(dim=-1), BADARG), (dict(tokens=2 ** 30, rows=2 ** 30), RANGE), (dict(pitch=15), BADARG), (dict(out_pitch=15), BADARG), (dict(ids=None), BADARG),
    (dict(positions=None), BADARG), (dict(grad=None), BADARG), (dict(out=None), BADARG), (dict(ws=None), BADARG), (dict(size=64), BADARG),
    (dict(out=D + 4), BADARG), (dict(out=A), BADARG), (dict(out=B - 4), BADARG),
    (dict(rows=0, ids=None, positions=None, grad=None, out=None, ws=None, size=0), 0), (dict(tokens=0, add=1, ids=None, positions=None, grad=None, out=None, ws=None, size=0), 0),
])
def test_gradient(change, code):
    assert _gradient(**change) == code


def _counts(index=I64, tokens=10, choices=4, chosen=A, mask=B, experts=16, counts=D, ws=None, size=0):
    return _lib.lib().loops_expert_counts(index, tokens, choices, chosen, mask, experts, counts, ws, size, None)


@pytest.mark.parametrize("change,code", [
    (dict(index=2), CONFIG), (dict(tokens=-1), BADARG), (dict(choices=0), BADARG), (dict(experts=0), BADARG), (dict(experts=1025), CONFIG),
    (dict(tokens=2 ** 29, choices=4), RANGE), (dict(chosen=None), BADARG), (dict(counts=None), BADARG), (dict(tokens=100000), BADARG),
    (dict(counts=A + 10 * 4 * 8 - 4), BADARG), (dict(counts=B - 4), BADARG),
])
def test_expert_counts(change, code):
    assert _counts(**change) == code


def _loss(value=F32, index=I64, tokens=10, experts=16, choices=4, logits=A, pitch=16, chosen=B, mask=D, loss=G, counts=G + 64, probability=G + 256, counted=G + 512,
          ws=None, size=0):
    return _lib.lib().loops_balance_loss(value, index, tokens, experts, choices, logits, pitch, chosen, mask, 1.0, loss, counts, probability, counted, ws, size, None)


@pytest.mark.parametrize("change,code", [
    (dict(value=3), CONFIG), (dict(index=2), CONFIG), (dict(tokens=-1), BADARG), (dict(experts=0), BADARG), (dict(experts=1025, pitch=1025), CONFIG),
    (dict(choices=0), BADARG), (dict(tokens=2 ** 29), RANGE), (dict(pitch=15), BADARG), (dict(logits=None), BADARG), (dict(chosen=None), BADARG),
    (dict(loss=None), BADARG), (dict(counts=None), BADARG), (dict(probability=None), BADARG), (dict(counted=None), BADARG), (dict(tokens=10000), BADARG),
    (dict(loss=A), BADARG), (dict(counts=B - 4), BADARG), (dict(probability=A + 10 * 16 * 4 - 4), BADARG), (dict(counted=D + 9), BADARG),
])
def test_balance_loss(change, code):
    assert _loss(**change) == code


def _backward(value=F32, tokens=10, experts=16, choices=4, logits=A, pitch=16, counts=B, counted=B + 64, mask=D, upstream=G, grad=H, grad_pitch=16):
    return _lib.lib().loops_balance_loss_backward(value, tokens, experts, choices, logits, pitch, counts, counted, mask, 1.0, upstream, grad, grad_pitch, None)


@pytest.mark.parametrize("change,code", [
    (dict(value=3), CONFIG), (dict(tokens=-1), BADARG), (dict(experts=0), BADARG), (dict(experts=1025, pitch=1025, grad_pitch=1025), CONFIG),
    (dict(choices=0), BADARG), (dict(tokens=2 ** 29), RANGE), (dict(pitch=15), BADARG), (dict(grad_pitch=15), BADARG), (dict(logits=None), BADARG),
    (dict(counts=None), BADARG), (dict(counted=None), BADARG), (dict(grad=None), BADARG), (dict(grad=A), BADARG), (dict(grad=B), BADARG), (dict(grad=D - 8), BADARG),
    (dict(grad=G), BADARG), (dict(tokens=0, logits=None, counts=None, counted=None, grad=None), 0),
])
def test_balance_loss_backward(change, code):
    assert _backward(**change) == code


def test_workspace_functions():
    L = _lib.lib()
    size = C.c_size_t(7)
    at = C.byref(size)
    assert L.loops_group_tokens_workspace(8192, 100, at) == 0 and size.value == 0
    assert L.loops_group_tokens_workspace(8193, 100, at) == 0 and size.value > 0
    assert L.loops_group_tokens_workspace(-1, 100, at) == BADARG and L.loops_group_tokens_workspace(1, 1, None) == BADARG
    assert L.loops_group_tokens_workspace(2 ** 30, 2 ** 30, at) == RANGE
    assert L.loops_embedding_gradient_workspace(BF16, F32, 100, 50, 64, 0, at) == 0 and size.value > 0
    assert L.loops_embedding_gradient_workspace(BF16, F16, 100, 50, 64, 0, at) == CONFIG
    assert L.loops_embedding_gradient_workspace(BF16, F32, 100, 50, -1, 0, at) == BADARG and L.loops_embedding_gradient_workspace(0, 0, 1, 1, 1, 0, None) == BADARG
    assert L.loops_expert_counts_workspace(10, 4, 1025, at) == CONFIG and L.loops_expert_counts_workspace(10, 4, 16, None) == BADARG
    assert L.loops_balance_loss_workspace(10, 0, at) == BADARG and L.loops_balance_loss_workspace(10, 16, None) == BADARG
    assert L.loops_balance_loss_workspace(100000, 256, at) == 0 and size.value > 0


def _z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def _ids(*shape, dtype=torch.int64):
    return torch.zeros(*shape, dtype=dtype)


GROUPS = embedding.TokenGroups(_ids(4, dtype=torch.int32), _ids(4, dtype=torch.int32), 9)
FORWARD = routing.BalanceLoss(_z(()), _ids(6, dtype=torch.int32), _z(6), _ids((), dtype=torch.int32), 2, 1.0)


@pytest.mark.parametrize("call,error", [
    (lambda: embedding.lookup(_z(9, 8, dtype=torch.float64), _ids(4)), TypeError),
    (lambda: embedding.lookup(_z(9, 8), _ids(4, dtype=torch.int16)), TypeError),
    (lambda: embedding.lookup(_z(9, 8), _z(4)), TypeError),
    (lambda: embedding.lookup(_z(9, 8, 2), _ids(4)), ValueError),
    (lambda: embedding.lookup(_z(8, 9).t(), _ids(4)), ValueError),                  # columns apart
    (lambda: embedding.lookup(_z(1, 8).expand(9, 8), _ids(4)), ValueError),         # rows on top of each other
    (lambda: embedding.lookup(_z(9, 8), _ids(8)[::2]), ValueError),
    (lambda: embedding.lookup(_z(9, 8), _ids(4), first_id=-1), ValueError),
    (lambda: embedding.lookup(_z(9, 8), _ids(4), first_id=2 ** 63), ValueError),
    (lambda: embedding.lookup(_z(9, 8), _ids(4)), ValueError),                      # no CPU path
    (lambda: embedding.group_tokens(_z(4), 9), TypeError),
    (lambda: embedding.group_tokens(_ids(8)[::2], 9), ValueError),
    (lambda: embedding.group_tokens(_ids(4), -1), ValueError),
    (lambda: embedding.group_tokens(_ids(4), 9, first_id=-3), ValueError),
    (lambda: embedding.group_tokens(_ids(4), 9, drop_id=2 ** 64), ValueError),
    (lambda: embedding.group_tokens(_ids(4), 9), ValueError),
    (lambda: embedding.gradient(GROUPS, _z(4, 8, dtype=torch.float64)), TypeError),
    (lambda: embedding.gradient(GROUPS._replace(ids=_ids(4)), _z(4, 8)), TypeError),
    (lambda: embedding.gradient(GROUPS._replace(positions=_ids(3, dtype=torch.int32)), _z(4, 8)), ValueError),
    (lambda: embedding.gradient(GROUPS._replace(ids=_ids(8, dtype=torch.int32)[::2]), _z(4, 8)), ValueError),
    (lambda: embedding.gradient(GROUPS, _z(())), ValueError),
    (lambda: embedding.gradient(GROUPS, _z(3, 8)), ValueError),
    (lambda: embedding.gradient(GROUPS, _z(2, 8, 2).transpose(1, 2)), ValueError),
    (lambda: embedding.gradient(GROUPS, _z(1, 8).expand(4, 8)), ValueError),
    (lambda: embedding.gradient(GROUPS, _z(4, 8)), ValueError),
    (lambda: routing.expert_counts(_z(4, 2), 6), TypeError),
    (lambda: routing.expert_counts(_ids(4, 2, 2), 6), ValueError),
    (lambda: routing.expert_counts(_ids(2, 4).t(), 6), ValueError),
    (lambda: routing.expert_counts(_ids(4, 2), 6), ValueError),
    (lambda: routing.balance_loss(_z(4, 6, dtype=torch.float64), _ids(4, 2)), TypeError),
    (lambda: routing.balance_loss(_z(4, 6), _z(4, 2)), TypeError),
    (lambda: routing.balance_loss(_z(4, 6), _ids(3, 2)), ValueError),
    (lambda: routing.balance_loss(_z(4, 6), _ids(4)), ValueError),
    (lambda: routing.balance_loss(_z(4, 6), _ids(2, 4).t()), ValueError),
    (lambda: routing.balance_loss(_z(6, 4).t(), _ids(4, 2)), ValueError),
    (lambda: routing.balance_loss(_z(4, 6), _ids(4, 2)), ValueError),
    (lambda: routing.balance_loss_backward(_z(4, 6, dtype=torch.int32), FORWARD), TypeError),
    (lambda: routing.balance_loss_backward(_z(4, 7), FORWARD), ValueError),
    (lambda: routing.balance_loss_backward(_z(4, 6), FORWARD._replace(counts=_z(6))), TypeError),
    (lambda: routing.balance_loss_backward(_z(4, 6), FORWARD._replace(tokens=_ids(2, dtype=torch.int32))), ValueError),
    (lambda: routing.balance_loss_backward(_z(4, 6), FORWARD), ValueError),
])
def test_python_refusals(call, error):
    with pytest.raises(error):
        call()


def test_sizes_that_are_no_integers_are_refused():
    with pytest.raises(TypeError):
        embedding.workspace_bytes("loops_expert_counts_workspace", 10, 2, 6.5)


def test_sizes_beyond_the_int_arguments_are_refused_and_not_cut():
    embedding.c_int("loops_group_tokens", BIG, 0)
    for bad in (BIG + 1, 2 ** 32 + 5, -2 ** 32 + 5):
        with pytest.raises(_lib.LoopsError, match="LOOPS_E_RANGE"):
            embedding.c_int("loops_group_tokens", 7, bad)

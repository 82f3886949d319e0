"""The embedding and routing calls beside autograd, which records none of them: refused where a gradient would be lost without an error, and
used from autograd.Functions."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from loops_amd import embedding, routing


def _z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def _ids(*shape, dtype=torch.int64):
    return torch.zeros(*shape, dtype=dtype)


GROUPS = embedding.TokenGroups(_ids(4, dtype=torch.int32), _ids(4, dtype=torch.int32), 9)
FORWARD = routing.BalanceLoss(_z(()), _ids(6, dtype=torch.int32), _z(6), _ids((), dtype=torch.int32), 2, 1.0)
CALLS = {
    "lookup table": lambda grad: embedding.lookup(_z(9, 8).requires_grad_(grad), _ids(4)),
    "lookup table of a graph": lambda grad: embedding.lookup(_z(9, 8).requires_grad_(grad) * 2, _ids(4)),
    "lookup out": lambda grad: embedding.lookup(_z(9, 8), _ids(4), out=_z(4, 8).requires_grad_(grad)),
    "gradient out": lambda grad: embedding.gradient(GROUPS, _z(4, 8), out=_z(9, 8).requires_grad_(grad), accumulate=True),
    "balance_loss logits": lambda grad: routing.balance_loss(_z(4, 6).requires_grad_(grad), _ids(4, 2)),
    "balance_loss_backward out": lambda grad: routing.balance_loss_backward(_z(4, 6), FORWARD, out=_z(4, 6).requires_grad_(grad)),
}


@pytest.mark.parametrize("call", CALLS)
def test_a_gradient_that_would_be_lost_is_refused(call):
    with pytest.raises(ValueError, match="requires a gradient"):
        CALLS[call](True)
    with pytest.raises(ValueError, match="must be on"):  # (the next check: these tensors are on the CPU)
        CALLS[call](False)
    with torch.no_grad(), pytest.raises(ValueError, match="must be on"):
        CALLS[call](True)


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale):
        ctx.save_for_backward(tokens)
        ctx.rows, ctx.scale = table.shape[0], scale
        return embedding.lookup(table, tokens, scale=scale)

    @staticmethod
    def backward(ctx, grad):
        tokens, = ctx.saved_tensors
        return embedding.gradient(embedding.group_tokens(tokens, ctx.rows), grad.contiguous(), scale=ctx.scale), None, None


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, chosen, coefficient, mask):
        ctx.kept = routing.balance_loss(logits, chosen, coefficient=coefficient, mask=mask)
        ctx.save_for_backward(logits, mask)
        return ctx.kept.loss

    @staticmethod
    def backward(ctx, grad):
        logits, mask = ctx.saved_tensors
        return routing.balance_loss_backward(logits, ctx.kept, mask=mask, grad_loss=grad), None, None, None


@pytest.mark.gpu
def test_functions_around_them_give_autograd_its_gradients():
    """Embedding, a router on it, the balance loss and a loss of its own on the rows, against the same in float64 on the CPU (inputs that float32
    holds exactly).

    e = 2^-24.  A logit is a sum of `dim` products of rounded rows: off by (dim + 3) e H, H the largest sum of magnitudes; twice that relative in a
    probability, four times in p (f - d).  The balance loss's gradient adds (4 D + 3 experts + 32) e of s p (f + d) of its own (D: largest distance of a
    logit to its row's maximum), the products with the router and the rows' sums (experts + 3), (n + 3) e and the sums over tokens (n + 3) e.  With
    the magnitudes M of the terms in place of the values: |error| <= M e ((4 (dim + 3) H + 4 D + 4 experts + 2 n + 41), a factor 1.01 for higher orders."""
    rng = np.random.default_rng(0)
    rows, dim, experts, n, k, a = 30, 16, 12, 70, 3, 5.0
    normal = lambda *shape: torch.from_numpy(rng.standard_normal(shape).astype(np.float32))  # noqa: E731
    table, router, weight = normal(rows, dim) / 4, normal(dim, experts) / 4, normal(n, dim)
    tokens = torch.from_numpy(rng.integers(0, rows, n))
    mask = torch.from_numpy(rng.random(n) < 0.8)

    w64, r64 = table.double().requires_grad_(), router.double().requires_grad_()
    hidden = w64[tokens] * 2.0
    logits = hidden @ r64
    chosen = torch.topk(logits.detach(), k, dim=1).indices.contiguous()
    p = torch.softmax(logits[mask], 1)
    f = torch.bincount(chosen[mask].reshape(-1), minlength=experts).double() / (mask.sum() * k)
    ((hidden * weight.double()).sum() + a * experts * (f * p.mean(0)).sum()).backward()

    w, r = table.cuda().requires_grad_(), router.cuda().requires_grad_()
    hidden = _Lookup.apply(w, tokens.cuda(), 2.0)
    loss = _Balance.apply(hidden @ r, chosen.cuda(), a, mask.cuda())
    ((hidden * weight.cuda()).sum() + loss).backward()

    with torch.no_grad():
        size = torch.zeros(n, experts, dtype=torch.float64)
        size[mask] = a * experts / mask.sum() * p * (f + (p @ f)[:, None])
        rows_abs, logits = 2 * w64.abs()[tokens], logits.detach()
        h = (rows_abs @ r64.abs()).max().item()
        d = (logits.amax(1, keepdim=True) - logits).max().item()
        rel = 1.01 * 2.0 ** -24 * (4 * (dim + 3) * h + 4 * d + 4 * experts + 2 * n + 41)
        w_size = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, tokens, 2 * (weight.double().abs() + size @ r64.abs().t()))
        for got, want, size in ((w.grad, w64.grad, w_size), (r.grad, r64.grad, rows_abs.t() @ size)):
            assert got is not None and ((got.cpu().double() - want).abs() <= rel * size).all()

"""Tokens per expert and the balance loss (loops_amd/routing.py) against plain fp64 arithmetic on the host.

Tolerances, e = 2^-24 (one float32 rounding), u = finfo(type).eps / 2 (one store).  A probability: the difference to the row's maximum
is rounded (e |x - max|, |x - max| <= D), the exponential of it is exp2 of a rounded product (D / ln 2 in magnitude, so the result is off by
another D e relative) with at most 1 ulp (2 e) of its own; the sum of E terms adds (log2-tree and per-lane chains: at most E) E e, the
reciprocal and the product 2 ulp each: relative P = (2 D + E + 8) e.  Probabilities whose exponential is below float32's normal range
come out as 0 or rounded to 2^-149: absolute 2^-126 each.
Mean over n tokens: at most n further additions, 2 products: relative P + (n + 3) e (all terms positive).
Loss: E more additions and 4 products: relative P + (n + E + 8) e.
Gradient: s p_e (f_e - d), d = sum f_j p_j: the weights f carry 3 e, d relative P + (E + 4) e, so the bracket is off by at most
(P + (E + 8) e) (f_e + d), the product with p_e s by relative P + 8 e more: |error| <= s p_e (f_e + d) (2 P + (E + 16) e), and the store u |result|
(float16: half a spacing of the smallest, 2^-25).  All with a factor 1.01 for the higher orders."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype is not torch.float32 else E32


def _case(rng, tokens, experts, choices, dtype, masked, pitch=None, spread=2.0):
    x = (rng.standard_normal((tokens, pitch or experts)) * spread).astype(np.float32)
    logits = torch.from_numpy(x).to(dtype).cuda()[:, :experts]
    chosen = np.argsort(-logits.cpu().float().numpy(), axis=1, kind="stable")[:, :choices].copy()
    mask = None if masked is None else rng.random(tokens) >= masked
    return logits, chosen, mask


def _reference(logits, chosen, mask, coefficient, upstream):
    x = logits.cpu().double().numpy()
    tokens, experts = x.shape
    keep = np.ones(tokens, bool) if mask is None else mask
    k = chosen.shape[1]
    flat = chosen[keep].reshape(-1)
    counts = np.bincount(flat[(flat >= 0) & (flat < experts)], minlength=experts)
    n = int(keep.sum())
    top = x[keep].max(1, keepdims=True) if n else np.zeros((0, 1))
    with np.errstate(invalid="ignore"):
        dist = np.where(np.isneginf(top), np.inf, top - x[keep])
        p_kept = np.exp(-dist)
        sums = p_kept.sum(1, keepdims=True)
        p_kept = np.where(sums > 0, p_kept / np.where(sums > 0, sums, 1), 0.0)
    finite = dist[np.isfinite(dist)]
    spread = min(float(finite.max()), 104.0) if finite.size else 0.0  # (beyond that the exponential is 0 in float32)
    coefficient, upstream = float(np.float32(coefficient)), float(np.float32(upstream))
    f = counts / max(n * k, 1)
    mean = p_kept.sum(0) / max(n, 1)
    loss = coefficient * experts * (f * mean).sum()
    s = upstream * coefficient * experts / max(n, 1)
    d = p_kept @ f
    grad, size = np.zeros((tokens, experts)), np.zeros((tokens, experts))
    grad[keep] = s * p_kept * (f - d[:, None])
    size[keep] = abs(s) * p_kept * (f + d[:, None])
    rel = 1.01 * (2 * spread + experts + 8) * E32
    return dict(counts=counts, n=n, mean=mean, loss=loss, grad=grad, size=size, rel=rel, s=abs(s))


def _compare(logits, chosen, mask, forward, grad, coefficient, upstream):
    want = _reference(logits, chosen, mask, coefficient, upstream)
    experts = logits.shape[1]
    n = want["n"]
    assert np.array_equal(forward.counts.cpu().numpy(), want["counts"])
    assert forward.tokens.item() == n
    tiny = 2.0 ** -126
    mean = forward.probability.cpu().double().numpy()
    assert (np.abs(mean - want["mean"]) <= (want["rel"] + 1.01 * (n + 3) * E32) * want["mean"] + tiny).all()
    assert abs(forward.loss.item() - want["loss"]) <= (want["rel"] + 1.01 * (n + experts + 8) * E32) * abs(want["loss"]) + tiny
    got = grad.cpu().double().numpy()
    bound = want["size"] * (2 * want["rel"] + 1.01 * (experts + 16) * E32) + _half_step(grad.dtype) * 1.01 * np.abs(want["grad"])
    bound = bound + (2.0 ** -25 if grad.dtype is torch.float16 else 0) + (want["s"] + 1) * tiny * experts
    assert (np.abs(got - want["grad"]) <= bound).all(), np.max(np.abs(got - want["grad"]) - bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("experts,choices", [(1, 1), (3, 2), (7, 7), (8, 2), (9, 1), (26, 4), (34, 6), (64, 6), (65, 8), (128, 8), (200, 3), (256, 8), (257, 1),
                                             (384, 8), (512, 4), (1000, 5), (1024, 8)])
def test_balance_loss(dtype, experts, choices):
    from loops_amd import routing
    rng = np.random.default_rng(experts)
    for tokens, masked, pitch, id_type in [(1, None, None, torch.int64), (2, 0.5, experts + 5, torch.int32), (37, 0.3, None, torch.int32),
                                           (130, None, experts + 3, torch.int64), (4099, 0.1, None, torch.int64)]:
        logits, chosen, mask = _case(rng, tokens, experts, choices, dtype, masked, pitch)
        where = None if mask is None else torch.from_numpy(mask).cuda()
        forward = routing.balance_loss(logits, torch.from_numpy(chosen).to(id_type).cuda(), coefficient=0.3, mask=where)
        upstream = torch.full((), -2.5, device="cuda")
        grad = routing.balance_loss_backward(logits, forward, mask=where, grad_loss=upstream)
        assert grad.dtype is dtype and forward.choices == choices
        _compare(logits, chosen, mask, forward, grad, 0.3, -2.5)
        if mask is not None:
            assert (grad[~where] == 0).all()


def test_balance_loss_large_and_repeatable():
    from loops_amd import routing
    rng = np.random.default_rng(1)
    for dtype, tokens, experts in [(torch.bfloat16, 70003, 256), (torch.float32, 30000, 129)]:
        logits, chosen, mask = _case(rng, tokens, experts, 8, dtype, 0.2)
        where = torch.from_numpy(mask).cuda()
        ids = torch.from_numpy(chosen).cuda()
        runs = []
        for _ in range(2):
            forward = routing.balance_loss(logits, ids, coefficient=0.01, mask=where)
            runs.append((forward, routing.balance_loss_backward(logits, forward, mask=where)))
        _compare(logits, chosen, mask, *runs[0], 0.01, 1.0)
        (a, ga), (b, gb) = runs
        assert torch.equal(ga, gb) and torch.equal(a.probability, b.probability) and torch.equal(a.loss, b.loss) and torch.equal(a.counts, b.counts)


def test_gradient_against_differences():
    """Central differences of the loss in float64 (counts held): exact to h^2 of a smooth function, and to the kernel's own bound."""
    from loops_amd import routing
    rng = np.random.default_rng(2)
    logits, chosen, mask = _case(rng, 23, 12, 3, torch.float32, 0.2)
    where = torch.from_numpy(mask).cuda()
    forward = routing.balance_loss(logits, torch.from_numpy(chosen).cuda(), coefficient=1.0, mask=where)
    grad = routing.balance_loss_backward(logits, forward, mask=where).cpu().double().numpy()
    x = logits.cpu().double().numpy()
    h = 1e-4

    def loss(x):
        p = np.exp(x - x.max(1, keepdims=True))
        p = p / p.sum(1, keepdims=True)
        n = mask.sum()
        f = np.bincount(chosen[mask].reshape(-1), minlength=12) / (n * 3)
        return 12 * (f * p[mask].sum(0) / n).sum()

    for t, e in [(0, 0), (1, 5), (7, 11), (22, 3), (13, 8)]:
        up, down = x.copy(), x.copy()
        up[t, e] += h
        down[t, e] -= h
        assert abs((loss(up) - loss(down)) / (2 * h) - grad[t, e]) < 1e-7


def test_masked_rows_may_hold_anything():
    from loops_amd import routing
    rng = np.random.default_rng(3)
    for dtype in TYPES:
        for tokens, experts in [(50, 40), (9000, 64)]:
            logits, chosen, mask = _case(rng, tokens, experts, 4, dtype, 0.4)
            where = torch.from_numpy(mask).cuda()
            ids = torch.from_numpy(chosen).cuda()
            dirty = logits.clone()
            dirty[~where] = float("nan")
            dirty_ids = ids.clone()
            dirty_ids[~where] = 10 ** 12
            a = routing.balance_loss(logits, ids, mask=where)
            b = routing.balance_loss(dirty, dirty_ids, mask=where)
            assert torch.equal(a.loss, b.loss) and torch.equal(a.counts, b.counts) and torch.equal(a.probability, b.probability)
            ga, gb = routing.balance_loss_backward(logits, a, mask=where), routing.balance_loss_backward(dirty, b, mask=where)
            assert torch.equal(ga, gb) and (gb[~where] == 0).all()


def test_nothing_left():
    """Every token masked; no tokens; rows of -infinity; the lowest finite value; choices outside the experts."""
    from loops_amd import routing
    rng = np.random.default_rng(4)
    logits, chosen, _ = _case(rng, 33, 20, 2, torch.float32, None)
    ids = torch.from_numpy(chosen).cuda()
    none = torch.zeros(33, dtype=torch.bool, device="cuda")
    forward = routing.balance_loss(logits, ids, mask=none)
    assert forward.loss.item() == 0 and forward.tokens.item() == 0 and (forward.counts == 0).all() and (forward.probability == 0).all()
    assert (routing.balance_loss_backward(logits, forward, mask=none) == 0).all()
    forward = routing.balance_loss(logits[:0], ids[:0])
    assert forward.loss.item() == 0 and forward.tokens.item() == 0 and (forward.counts == 0).all() and (forward.probability == 0).all()
    assert routing.balance_loss_backward(logits[:0], forward).shape == (0, 20)
    for dtype in TYPES:
        holes = logits.clone().to(dtype)
        holes[::5] = float("-inf")          # no expert left
        holes[1::5, ::2] = float("-inf")    # half of them
        holes[2::5] = torch.finfo(dtype).min
        outside = chosen.copy()
        outside[::3, 0] = -1
        outside[1::3, 1] = 20
        out_ids = torch.from_numpy(outside).cuda()
        forward = routing.balance_loss(holes, out_ids, coefficient=2.0)
        grad = routing.balance_loss_backward(holes, forward)
        _compare(holes, outside, None, forward, grad, 2.0, 1.0)
        assert (grad[::5] == 0).all() and (grad[1::5, ::2] == 0).all()


def test_values_that_are_not_finite_show():
    from loops_amd import routing
    rng = np.random.default_rng(5)
    for bad in (float("inf"), float("nan")):
        logits, chosen, _ = _case(rng, 40, 16, 2, torch.float32, None)
        logits[9, 3] = bad
        forward = routing.balance_loss(logits, torch.from_numpy(chosen).cuda())
        grad = routing.balance_loss_backward(logits, forward)
        assert forward.loss.isnan() and grad[9].isnan().all() and not grad[torch.arange(40, device="cuda") != 9].isnan().any()


@pytest.mark.parametrize("tokens", [0, 1, 100, 2048, 2049, 5000, 262147])
@pytest.mark.parametrize("experts,choices", [(1, 1), (5, 2), (256, 8), (1000, 3), (1024, 1)])
def test_expert_counts(tokens, experts, choices):
    from loops_amd import routing
    rng = np.random.default_rng(tokens + experts)
    chosen = rng.integers(-2, experts + 2, (tokens, choices))
    mask = rng.random(tokens) < 0.7
    for id_type in (torch.int32, torch.int64):
        for where in (None, mask):
            ids = torch.from_numpy(chosen).to(id_type).cuda()
            got = routing.expert_counts(ids, experts, None if where is None else torch.from_numpy(where).cuda())
            flat = (chosen if where is None else chosen[where]).reshape(-1)
            assert np.array_equal(got.cpu().numpy(), np.bincount(flat[(flat >= 0) & (flat < experts)], minlength=experts))
    if choices == 1:
        assert torch.equal(routing.expert_counts(ids[:, 0].contiguous(), experts), routing.expert_counts(ids, experts))

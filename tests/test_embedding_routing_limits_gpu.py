"""The embedding and routing operators at the largest sizes: token numbers near 2^31, checked against what whole numbers give."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_counts_and_loss_of_the_most_tokens():
    """2^31 - 4 097 tokens of one choice: every one of them is counted.  One expert has probability 1 whatever its logit, so that the loss is
    the coefficient; its sums are whole numbers up to a workgroup's 4.2 million (exact), the join of the 512 workgroups rounds at most 512
    times, a reciprocal and three products once or twice each: 2^-24 (512 + 8) relative."""
    from loops_amd import routing
    tokens, experts = 2 ** 31 - 4097, 16
    chosen = torch.arange(tokens, dtype=torch.int32, device="cuda").remainder_(experts)
    got = routing.expert_counts(chosen, experts)
    assert got.tolist() == [len(range(e, tokens, experts)) for e in range(experts)]
    chosen.zero_()
    chosen[-5:] = -1
    logits = torch.ones(tokens, 1, dtype=torch.float16, device="cuda")
    forward = routing.balance_loss(logits, chosen[:, None], coefficient=0.5)
    assert forward.tokens.item() == tokens and forward.counts.tolist() == [tokens - 5]
    bound = 2.0 ** -24 * 520
    assert abs(forward.probability.item() - 1.0) <= bound
    assert abs(forward.loss.item() - 0.5 * (tokens - 5) / tokens) <= 0.5 * 2 * bound


def _whole(rows, cols, seed):
    """Whole numbers in [-4, 4], half, made a row at a time."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    out = torch.empty(rows, cols, dtype=torch.float16, device="cuda")
    for r in range(rows):
        out[r] = torch.randint(-4, 5, (cols,), generator=g, dtype=torch.int8, device="cuda")
    return out


def _same(got, want):
    """Equal, compared a piece at a time (a comparison of all of it makes a temporary as large)."""
    assert got.shape == want.shape
    for at in range(0, got.numel(), 2 ** 28):
        assert torch.equal(got[at:at + 2 ** 28], want[at:at + 2 ** 28]), at


def test_the_widest_rows():
    """2^31 - 1 columns, and 2^28 + 5, which end in a range narrower than an access; whole numbers and a scale of 2: exact sums."""
    from loops_amd import embedding
    dim = 2 ** 31 - 1
    table = _whole(2, dim, 1)
    got = embedding.lookup(table, torch.tensor([1, 7], device="cuda"), scale=2.0)
    _same(got[0], table[1] * 2)
    assert not got[1].any()
    del got
    groups = embedding.group_tokens(torch.tensor([2, 2], device="cuda"), 3)
    got = embedding.gradient(groups, table, scale=2.0)
    assert not got[0].any() and not got[1].any()
    _same(got[2], (table[0] + table[1]) * 2)
    embedding.gradient(groups, table, scale=2.0, out=got, accumulate=True)  # in one launch per range
    assert not got[0].any() and not got[1].any()
    _same(got[2], (table[0] + table[1]) * 4)
    del got, table
    dim, tokens = 2 ** 28 + 5, 70  # (the row is cut into tiles and joined in the last, narrow range)
    grad = _whole(tokens, dim, 2)
    groups = embedding.group_tokens(torch.ones(tokens, dtype=torch.int64, device="cuda"), 2)
    got = embedding.gradient(groups, grad)
    assert not got[0].any()
    want = torch.zeros(dim, dtype=torch.float16, device="cuda")  # (sums of 70 numbers up to 4 are exact in half)
    for t in range(tokens):
        want += grad[t]
    _same(got[1], want)


def test_more_narrow_lookups_than_a_launch_holds():
    """2^30 tokens of rows of 4 halves, moved one by one: more than 2^32 threads."""
    from loops_amd import embedding
    rows, dim, tokens = 1000, 4, 2 ** 30 + 77
    table = _whole(rows, dim, 3)
    ids = torch.arange(tokens, dtype=torch.int32, device="cuda").remainder_(rows + 3)  # three in 1 003 lie outside
    got = embedding.lookup(table, ids, scale=0.5)
    padded = torch.cat([table * 0.5, torch.zeros(3, dim, dtype=torch.float16, device="cuda")])
    for at in range(0, tokens, 2 ** 26):
        assert torch.equal(got[at:at + 2 ** 26], padded[ids[at:at + 2 ** 26].long()]), at


def test_balance_loss_and_gradient_beyond_32_bit_offsets():
    """2 100 003 x 1 024 logits (2.15e9 of them), whole rows at both ends and between against float64.

    Bounds as in test_routing_gpu.py: e = 2^-24, a probability is off by P = (2 D + E + 8) e relative, their mean over n tokens by (n + 3) e more (the
    sums are of at most n terms, all positive), the loss by (n + E + 8) e instead; the gradient by (2 P + (E + 16) e) s p (f + d) and half a step of
    bfloat16, 2^-8, of its value.  n e would be 1/8 here; no sum adds more than 1 024 terms after each other (4 102 tokens per workgroup are 257 rows per
    wavefront, then 16 wavefronts, then 512 workgroups), which stand in n's place.  Float32's least normal number, 2^-126, for each exponential."""
    from loops_amd import routing
    tokens, experts, choices, e = 2100003, 1024, 2, 2.0 ** -24
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    logits = torch.empty(tokens, experts, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    chosen = torch.randint(-1, experts, (tokens, choices), generator=g, dtype=torch.int32, device="cuda")
    mask = torch.rand(tokens, generator=g, device="cuda") < 0.9
    forward = routing.balance_loss(logits, chosen, coefficient=1.0, mask=mask)
    n = int(mask.sum())
    kept = chosen[mask].reshape(-1).long()
    counts = torch.bincount(kept[kept >= 0], minlength=experts)
    total, distance = torch.zeros(experts, dtype=torch.float64, device="cuda"), 0.0
    for at in range(0, tokens, 2 ** 17):
        x = logits[at:at + 2 ** 17].double()
        x -= x.amax(1, keepdim=True)
        distance = max(distance, -x.min().item())
        p = x.exp_()
        p /= p.sum(1, keepdim=True)
        total += (p * mask[at:at + 2 ** 17, None]).sum(0)
    f, mean = counts.double() / (n * choices), total / n
    loss = experts * (f * mean).sum().item()
    rel = 1.01 * (2 * distance + experts + 8) * e
    assert forward.tokens.item() == n and torch.equal(forward.counts.long(), counts)
    assert ((forward.probability.double() - mean).abs() <= (rel + 1.01 * (1024 + 3) * e) * mean + 2.0 ** -126).all()
    assert abs(forward.loss.item() - loss) <= (rel + 1.01 * (1024 + experts + 8) * e) * loss

    grad = routing.balance_loss_backward(logits, forward, mask=mask, grad_loss=torch.full((), float(n), device="cuda"))
    middle = 2 ** 31 // experts  # the row behind the last element that 31 bits number
    at = torch.cat([torch.arange(300), torch.arange(middle - 300, middle + 300), torch.arange(tokens - 300, tokens),
                    torch.randint(tokens, (3000,))]).cuda()
    p = torch.softmax(logits[at].double(), 1) * mask[at, None]
    d = (p * f).sum(1, keepdim=True)
    want, size = experts * p * (f - d), experts * p * (f + d)
    bound = size * (2 * rel + 1.01 * (experts + 16) * e) + 2.0 ** -8 * 1.01 * want.abs() + experts * 2.0 ** -126
    assert ((grad[at].double() - want).abs() <= bound).all()
    assert (grad[at][~mask[at]] == 0).all() and (grad[at][mask[at]] != 0).any(1).all()


@pytest.mark.parametrize("n", [131071, 131072, 131073, 262145, 1200008])
@pytest.mark.parametrize("rows", [256, 131072])
def test_group_tokens_in_spans_of_more_than_1024(n, rows):
    """Up to 128 spans of 1 024 positions each; beyond that longer spans."""
    from loops_amd import embedding
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    ids = torch.randint(-1, rows, (n,), generator=g, device="cuda")
    got = embedding.group_tokens(ids, rows)
    key, order = torch.sort(torch.where(ids < 0, rows, ids), stable=True)
    assert torch.equal(got.ids.long(), key) and torch.equal(got.positions.long(), order)

"""The embedding and routing operators as a training step of a sparse model uses them: together, captured into a graph, on streams of their
own, over storage whose offsets pass 32 bits; and what they refuse on the GPU.

Where values are small integers and scales powers of two every sum is exact in float32 and results are compared bit for bit; the balance
loss (float) is compared with itself run another way, which its fixed order of summation makes equal bit for bit."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _whole(rng, *shape, dtype=torch.float32):
    return torch.from_numpy(rng.integers(-4, 5, shape).astype(np.float32)).to(dtype).cuda()


def _step(s):
    """Lookup, the loss of the router with its gradient, the order of the experts' products, the table's gradient."""
    from loops_amd import embedding, routing
    hidden = embedding.lookup(s["table"], s["tokens"], scale=2.0)
    forward = routing.balance_loss(s["logits"], s["chosen"], coefficient=0.01, mask=s["mask"])
    grad_logits = routing.balance_loss_backward(s["logits"], forward, mask=s["mask"], grad_loss=s["upstream"])
    counts = routing.expert_counts(s["chosen"], s["experts"], s["mask"])
    order = embedding.group_tokens(s["chosen"], s["experts"])
    groups = embedding.group_tokens(s["tokens"], s["table"].shape[0], drop_id=0)
    grad_table = embedding.gradient(groups, s["grad"], scale=2.0, dtype=torch.float32)
    embedding.gradient(groups, s["grad"], scale=2.0, out=s["sum"], accumulate=True)
    return dict(hidden=hidden, loss=forward.loss, counts=forward.counts, probability=forward.probability, tokens=forward.tokens, grad_logits=grad_logits, again=counts,
                ids=order.ids, positions=order.positions, grad_table=grad_table, sum=s["sum"])


def _state(seed, n, rows=501, dim=72, experts=24, choices=3, dtype=torch.bfloat16):
    rng = np.random.default_rng(seed)
    s = dict(table=_whole(rng, rows, dim, dtype=dtype), tokens=torch.from_numpy(rng.integers(0, rows, n)).cuda(), grad=_whole(rng, n, dim, dtype=dtype),
             sum=_whole(rng, rows, dim), experts=experts, mask=torch.from_numpy(rng.random(n) < 0.8).cuda(), upstream=torch.full((), 0.5, device="cuda"))
    s["logits"] = torch.from_numpy(rng.standard_normal((n, experts)).astype(np.float32)).to(dtype).cuda()
    chosen = torch.topk(s["logits"].float(), choices, dim=1).indices
    s["chosen"] = torch.where(s["mask"][:, None], chosen, -1).contiguous()
    return s


def _expected(s, total_before):
    """What integer arithmetic on the host gives."""
    ids, chosen = s["tokens"].cpu().numpy(), s["chosen"].cpu().numpy()
    table, grad = s["table"].cpu().double().numpy(), s["grad"].cpu().double().numpy()
    grad_table = np.zeros(table.shape)
    np.add.at(grad_table, ids[ids != 0], 2 * grad[ids != 0])
    flat = chosen.reshape(-1)
    key = np.where(flat >= 0, flat, s["experts"])
    return dict(hidden=2 * table[ids], grad_table=grad_table, sum=total_before.cpu().double().numpy() + grad_table, ids=np.sort(key, kind="stable"),
                positions=np.argsort(key, kind="stable"), again=np.bincount(flat[flat >= 0], minlength=s["experts"]), tokens=s["mask"].cpu().numpy().sum())


def _equal(got, want):
    for k, v in want.items():
        assert np.array_equal(got[k].cpu().double().numpy(), v), k
    assert torch.equal(got["again"], got["counts"])


@pytest.mark.parametrize("n", [1, 300, 9001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_training_step(n, dtype):
    s = _state(n, n, dtype=dtype)
    before = s["sum"].clone()
    got = _step(s)
    _equal(got, _expected(s, before))
    # tokens sorted by expert: each expert's products take a run of them, as long as its count
    starts = torch.cumsum(got["counts"], 0) - got["counts"]
    for e in range(s["experts"]):
        rows = got["positions"][starts[e]:starts[e] + got["counts"][e]] // 3
        assert (s["chosen"][rows.long()] == e).any(1).all()


@pytest.mark.parametrize("n", [200, 9001])
def test_captured_steps(n):
    """Two graphs of the step over the same inputs, replayed in turn with eager work between: every replay against the eager result."""
    s = _state(7, n)
    before = s["sum"].clone()
    _step(s)  # libraries and kernels are loaded
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(s))
        graphs.append(g)
    for replay in range(4):
        new = _state(100 + replay, n)
        for k in ("table", "tokens", "grad", "mask", "logits", "chosen"):
            s[k].copy_(new[k])
        s["sum"].copy_(before)
        want = {k: v.clone() for k, v in _step(s).items()}
        _equal(want, _expected(s, before))
        for g, out in zip(graphs, outs):
            s["sum"].copy_(before)
            g.replay()
            torch.zeros(1 << 20, device="cuda").add_(1.0)
            torch.cuda.synchronize()
            for k, v in want.items():
                assert torch.equal(out[k], v), (replay, k)


def test_two_streams_at_once():
    states = [_state(20 + i, 20011, dim=200) for i in range(2)]
    before = [s["sum"].clone() for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    outs = [None, None]
    for _ in range(5):
        for i, (s, stream) in enumerate(zip(states, streams)):
            with torch.cuda.stream(stream):
                s["sum"].copy_(before[i])
                outs[i] = _step(s)
    torch.cuda.synchronize()
    for s, out, old in zip(states, outs, before):
        _equal(out, _expected(s, old))
        s["sum"].copy_(old)
        again = _step(s)
        assert all(torch.equal(out[k], again[k]) for k in out)


def test_offsets_beyond_32_bits():
    """Table, gradient and logits of more than 2^31 elements: rows at both ends, checked one by one."""
    from loops_amd import embedding, routing
    rng = np.random.default_rng(30)
    rows, dim = 600011, 4096  # 4.9 GB
    table = torch.empty(rows, dim, dtype=torch.bfloat16, device="cuda")
    table.copy_((torch.arange(rows, device="cuda") % 97)[:, None].expand(rows, dim))
    ids = torch.cat([torch.arange(5), torch.arange(rows - 5, rows)]).cuda()
    got = embedding.lookup(table, ids)
    assert torch.equal(got, table[ids])
    # every row once, in another order; the table is the gradient
    tokens = torch.randperm(rows, device="cuda")
    groups = embedding.group_tokens(tokens, rows)
    out = embedding.gradient(groups, table, scale=0.5)
    at = torch.cat([torch.arange(3), torch.arange(rows - 300, rows), torch.from_numpy(rng.integers(0, rows, 300))]).cuda()
    assert torch.equal(out[tokens[at]], table[at] * 0.5)
    embedding.gradient(groups, table, scale=0.5, out=out, accumulate=True)
    assert torch.equal(out[tokens[at]], table[at])
    del out, groups
    tokens, experts = rows * 4, 1024
    logits = table.view(-1)[:tokens * experts].view(tokens, experts)
    chosen = torch.full((tokens, 1), 5, dtype=torch.int32, device="cuda")
    forward = routing.balance_loss(logits, chosen)  # equal logits in a row: p = 1 / experts, loss = 1 (a power of two: exact terms)
    assert forward.counts[5].item() == tokens and abs(forward.loss.item() - 1.0) < 1e-3
    grad = routing.balance_loss_backward(logits, forward, grad_loss=torch.full((), float(tokens), device="cuda"))
    # p (f_e - 1 / experts) * experts, f_5 = 1: 1 - 2^-10 and -2^-10, exp2(0) and 1 / 1024 are exact
    want = torch.full((experts,), -2.0 ** -10)
    want[5] = 1 - 2.0 ** -10
    for t in (0, 1, tokens // 2, tokens - 2, tokens - 1):
        assert (grad[t].cpu().float() - want).abs().max().item() <= 2.0 ** -8  # one bf16 store of a value below 1
    assert (grad[:, 0].float() < 0).all() and (grad[:, 5].float() > 0.9).all()


def test_outputs_may_be_slices_and_inputs_shared():
    """The same tokens twice, one gradient for two tables, outputs inside a larger buffer."""
    from loops_amd import embedding
    rng = np.random.default_rng(31)
    table, other = _whole(rng, 40, 24), _whole(rng, 40, 24)
    tokens = torch.full((70,), 7, dtype=torch.int32, device="cuda")
    buffer = torch.full((2, 40, 30), 3.0, device="cuda")
    groups = embedding.group_tokens(tokens, 40)
    grad = _whole(rng, 70, 24)
    for i in range(2):
        embedding.gradient(groups, grad, out=buffer[i, :, 2:26])
    want = torch.zeros(40, 24, device="cuda")
    want[7] = grad.sum(0)
    for i in range(2):
        assert torch.equal(buffer[i, :, 2:26], want) and (buffer[i, :, :2] == 3).all() and (buffer[i, :, 26:] == 3).all()
    assert torch.equal(embedding.lookup(table, tokens), table[tokens.long()]) and torch.equal(embedding.lookup(other, tokens), other[tokens.long()])


@pytest.mark.parametrize("dtype,dim,pitch", [(torch.float32, 4096, 4096), (torch.float32, 6176, 6176), (torch.float32, 6176, 6208), (torch.float32, 9001, 9001),
                                             (torch.bfloat16, 64, 64), (torch.bfloat16, 64, 128), (torch.float16, 8200, 8200), (torch.bfloat16, 3, 3)])
def test_rows_without_tokens_are_cleared(dtype, dim, pitch):
    """Rows of a part of a clearing workgroup and of many to one, none or all of them without a token, the padding left as it was; whole numbers."""
    from loops_amd import embedding
    rng = np.random.default_rng(dim)
    for rows, ids in [(1, [0]), (1, []), (700, []), (700, list(range(700))), (700, [0] * 70 + [699]), (701, [350] * 1500 + [351, 353, 700]), (65, [1, 3, 64, 3])]:
        tokens = torch.tensor(ids, dtype=torch.int64, device="cuda")
        grad = _whole(rng, len(ids), dim, dtype=dtype).clamp_(0, 1)
        buffer = torch.full((rows, pitch), 5.0, device="cuda", dtype=dtype if dim < 5000 else torch.float32)
        embedding.gradient(embedding.group_tokens(tokens, rows), grad, out=buffer[:, :dim])
        want = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, tokens.cpu(), grad.cpu().double())
        assert torch.equal(buffer[:, :dim].cpu().double(), want.to(buffer.dtype).double()), (rows, len(ids))
        assert (buffer[:, dim:] == 5).all()


@pytest.mark.parametrize("n", [63, 64, 639, 640, 641, 1024, 1025])
def test_adding_few_tokens_and_some_more(n):
    """Both sides of the one-launch form, tokens of one row, of all different rows and of some without a row."""
    from loops_amd import embedding
    rng = np.random.default_rng(n)
    for ids in (np.full(n, 17), np.arange(n) % 2000, np.where(np.arange(n) % 3 == 0, -1, 1999), np.sort(rng.integers(0, 30, n)), np.full(n, -1)):
        for dim in (1, 77, 520):
            grad, old = _whole(rng, n, dim, dtype=torch.bfloat16), _whole(rng, 2000, dim)
            tokens = torch.from_numpy(ids).cuda()
            got = embedding.gradient(embedding.group_tokens(tokens, 2000), grad, scale=0.5, out=old.clone(), accumulate=True)
            keep = torch.from_numpy(ids >= 0)
            want = old.cpu().double().index_add_(0, torch.from_numpy(ids)[keep], 0.5 * grad.cpu().double()[keep])
            assert torch.equal(got.cpu().double(), want), dim


def test_refusals():
    from loops_amd import LoopsError, embedding, routing
    table, tokens = torch.zeros(9, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError):
        embedding.lookup(table, tokens, out=torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        embedding.lookup(table, tokens, out=torch.zeros(5, 8, device="cuda"))
    with pytest.raises(ValueError):
        embedding.lookup(table, tokens.cpu())
    with pytest.raises(LoopsError):
        embedding.lookup(table, tokens, out=table[2:6])
    with pytest.raises(TypeError):
        embedding.lookup(table, tokens, scale="2")
    with pytest.raises(LoopsError):
        embedding.group_tokens(tokens, 2 ** 32 + 5)
    groups, grad = embedding.group_tokens(tokens, 9), torch.zeros(4, 8, device="cuda")
    with pytest.raises(ValueError):
        embedding.gradient(groups, grad, accumulate=True)
    with pytest.raises(ValueError):
        embedding.gradient(groups, grad, out=torch.zeros(8, 8, device="cuda"))
    with pytest.raises(TypeError):
        embedding.gradient(groups, grad, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        embedding.gradient(groups, grad, dtype=torch.float32, out=torch.zeros(9, 8, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(LoopsError):
        embedding.gradient(embedding.group_tokens(tokens, 4), grad, out=grad)
    logits, chosen = torch.zeros(4, 6, device="cuda"), torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError):
        routing.balance_loss(logits, chosen, mask=torch.ones(4, device="cuda"))
    with pytest.raises(ValueError):
        routing.balance_loss(logits, chosen, mask=torch.ones(5, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError):
        routing.balance_loss(logits, chosen, mask=torch.ones(4, dtype=torch.bool))
    with pytest.raises(LoopsError):
        routing.balance_loss(torch.zeros(4, 1025, device="cuda"), chosen)
    with pytest.raises(LoopsError):
        routing.expert_counts(chosen, 1025)
    forward = routing.balance_loss(logits, chosen)
    with pytest.raises(TypeError):
        routing.balance_loss_backward(logits, forward, grad_loss=torch.zeros((), dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError):
        routing.balance_loss_backward(logits, forward, grad_loss=torch.zeros(2, device="cuda"))
    with pytest.raises(TypeError):
        routing.balance_loss_backward(logits, forward, out=torch.zeros(4, 6, dtype=torch.float16, device="cuda"))
    with pytest.raises(LoopsError):
        routing.balance_loss_backward(logits, forward, out=logits)

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

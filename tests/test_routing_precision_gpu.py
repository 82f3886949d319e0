"""The balance loss of float logits far below their row's maximum, where a rounding of the exponential's argument would show.

Logits 0 (the maximum) and multiples of -2^-10: their distances are exact.  e = 2^-24.  An exponential: 1 ulp of the hardware's 2^x (2 e), the factor
that brings back its argument's rounding (e, and its own terms left out, below e / 100); the sum of E of them E e; the reciprocal e, the
product e: a probability is off by less than (E + 6) e relative, whatever the distance, and one token's is its mean.  The gradient s p_e (f_e - d), d =
sum f p: |error| <= s p (f + d) (2 (E + 6) + E + 16) e, and its store e.  All with a factor 1.01 for the higher orders."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24


@pytest.mark.parametrize("experts", [2, 8, 13, 128, 300])
@pytest.mark.parametrize("depth", [1.0, 20.0, 60.0, 87.0])
def test_probabilities_far_below_the_maximum(experts, depth):
    from loops_amd import routing
    rng = np.random.default_rng(experts)
    for trial in range(10):
        x = -np.floor(rng.random((1, experts)) * depth * 1024) / 1024
        x[0, rng.integers(experts)] = 0.0
        x[0, -1] = min(x[0, -1], -depth / 2) if x[0, -1] else 0.0
        logits = torch.from_numpy(x.astype(np.float32)).cuda()
        chosen = torch.from_numpy(np.argsort(x, axis=1)[:, :2].copy()).cuda()  # (the least likely: the gradient's terms do not cancel)
        forward = routing.balance_loss(logits, chosen, coefficient=1.0)
        grad = routing.balance_loss_backward(logits, forward).cpu().double().numpy()[0]
        p = np.exp(x[0])
        p /= p.sum()
        assert (np.abs(forward.probability.cpu().double().numpy() - p) <= 1.01 * (experts + 6) * E32 * p).all()
        f = np.bincount(chosen.cpu().numpy().reshape(-1), minlength=experts) / 2
        d = (f * p).sum()
        want = experts * p * (f - d)
        size = experts * p * (f + d)
        assert (np.abs(grad - want) <= 1.01 * E32 * (size * (2 * (experts + 6) + experts + 16) + np.abs(want)) + 2.0 ** -126 * experts).all()


def test_distances_beyond_every_exponent():
    """-infinity, the lowest finite value under the highest, and distances whose exponential is below float's range: probability 0, no NaN."""
    from loops_amd import routing
    top = torch.finfo(torch.float32).max
    for row in ([0.0, float("-inf"), -200.0, -1e30], [top, -top, 0.0, float("-inf")], [-top, -top, float("-inf"), float("-inf")]):
        for experts in (4, 37):
            x = torch.full((1, experts), float("-inf"))
            x[0, :4] = torch.tensor(row)
            chosen = torch.zeros(1, 1, dtype=torch.int64, device="cuda")
            forward = routing.balance_loss(x.cuda(), chosen)
            want = torch.zeros(experts)
            at = x[0] == x[0].max()
            want[at] = 1.0 / at.sum()
            assert torch.equal(forward.probability.cpu(), want)
            grad = routing.balance_loss_backward(x.cuda(), forward).cpu()
            f = torch.zeros(experts)
            f[0] = 1.0
            assert torch.equal(grad[0], experts * want * (f - (f * want).sum()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_factors_of_the_whole_result_are_rounded_once(dtype):
    """Two experts of equal logits, all tokens to the first: probabilities of 1/2, f = (1, 0), every sum exact.  The loss is the coefficient
    itself, the gradient +- upstream coefficient 2 / n / 4 rounded once (e), and once more by its store."""
    from loops_amd import routing
    coefficient, upstream = float(np.float32(0.3)), float(np.float32(0.7))
    for n in [*range(1, 130), 1000, 4099, 20011, 70003]:
        for choices in (1, 3):
            logits = torch.zeros(n, 2, dtype=dtype, device="cuda")
            chosen = torch.zeros(n, choices, dtype=torch.int32, device="cuda")
            forward = routing.balance_loss(logits, chosen, coefficient=coefficient)
            assert forward.loss.item() == coefficient and (forward.probability == 0.5).all(), (n, choices)
            grad = routing.balance_loss_backward(logits, forward, grad_loss=torch.full((), upstream, device="cuda")).double()
            want = upstream * coefficient * 2 / n / 4
            store = 0.0 if dtype is torch.float32 else torch.finfo(dtype).eps / 2
            bound = 1.01 * (E32 + store) * want + (2.0 ** -25 if dtype is torch.float16 else 0.0)
            assert (grad[:, 0] - want).abs().max() <= bound and (grad[:, 1] + want).abs().max() <= bound, (n, choices)

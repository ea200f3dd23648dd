"""sample_tokens where settings and logits are at their ends together, against its definition in 64 bits; bounds are those
of test_sampling.py."""
import math

import pytest
import torch
from shared_oracle import sample
from test_sampling import TYPES, _check, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [4099, 20000])
def test_infinite_temperature_and_infinite_logits(pkg, cuda, kind, vocab):
    """Parts with an infinity, with finite logits alone and with nothing, under every filter; all that is drawn is the
    infinities, all of the same weight."""
    x, u = _logits(6, vocab, TYPES[kind], 83)
    x[0, 4097] = math.inf
    x[1, [3, 1000, 4098]] = math.inf
    x[2, 0] = math.inf
    x[2, 1:4096] = -math.inf
    x[3, :4096] = math.nan
    x[3, 4096:4098] = math.inf
    x[4] = math.inf
    # row 5 stays finite: all of it weighs the same
    for settings in (dict(), dict(top_k=1), dict(top_k=2), dict(top_k=4000), dict(top_p=0.4), dict(top_p=0.99), dict(min_p=0.3),
                     dict(min_p=1.0), dict(top_k=3, top_p=0.6, min_p=0.1)):
        _check(pkg, cuda, x, u, temperature=math.inf, **settings)
        mixed = torch.tensor([math.inf, 1.0, math.inf, math.inf, 0.5, 0.0])
        _check(pkg, cuda, x, u, temperature=mixed, **settings)


@pytest.mark.parametrize("kind", ["fp16", "fp32"])
def test_light_tokens_in_earlier_parts(pkg, cuda, kind):
    """Weights of 2^-58 of the largest, kept by top-k and before it: random numbers of 0 and 2^-100 draw the first of them."""
    x = torch.full((3, 9000), -200.0)
    x[:, 8500:8510] = torch.linspace(7.0, 8.0, 10)
    x[:, 5] = 4.0
    x[:, 4097] = 4.125
    x[:, 6000:6025] = 3.875
    x = x.to(TYPES[kind])
    u = torch.tensor([0.0, 2.0 ** -100, 2.0 ** -57])
    for settings in (dict(top_k=20), dict(top_k=12), dict(top_k=300)):
        tokens, logs = pkg.sample_tokens(x.to(cuda), u.to(cuda), temperature=0.1, return_logprobs=True, **settings)
        # borders are 2^-58 of the total apart, and at least a tenth of that from these numbers
        want = [sample(x[r], u[r].item(), temperature=0.1, **settings)[:2] for r in range(3)]
        assert [w[0] for w in want] == [5, 5, 4097] and tokens.tolist() == [5, 5, 4097]
        assert all(abs(float(got) - w[1]) <= abs(w[1]) * 2.0 ** -24 * 1.0001 + 2.0 ** -40 for got, w in zip(logs, want))


def _tail(count, units, vocab, seed):
    """One logit of 0 and `count` light ones, whose weights are units[0] to units[1] times 2^-43."""
    g = torch.Generator().manual_seed(seed)
    x = torch.full((1, vocab), -math.inf)
    at = torch.randperm(vocab, generator=g)[:count + 1]
    x[0, at[0]] = 0.0
    w = (units[0] + (units[1] - units[0]) * torch.rand((count,), generator=g).double()) * 2.0 ** -43
    x[0, at[1:]] = torch.log(w).float()
    return x


@pytest.mark.parametrize("count,units,vocab,top_p,u,seed", [
    (8000, (512.40, 512.49), 12000, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 2),  # a list of them
    (8000, (512.40, 512.49), 12000, 1 - 2.0 ** -24, 1 - 2.0 ** -23, 2),
    (40000, (50.40, 50.49), 50001, 1 - 2.0 ** -23, 1 - 2.0 ** -24, 1),   # more than a list holds
    (40000, (50.40, 50.49), 50001, 1 - 2.0 ** -23, 1 - 2.0 ** -24, 3)])
def test_sums_of_light_tokens(pkg, cuda, count, units, vocab, top_p, u, seed):
    """Thresholds and draws among tokens that weigh a few times 2^-43 of the largest each: rounded to that, their sums would
    be off by many of them."""
    _check(pkg, cuda, _tail(count, units, vocab, seed), torch.tensor([u]), top_p=top_p)


@pytest.mark.parametrize("kind", list(TYPES))
def test_least_weights_above_the_largest(pkg, cuda, kind):
    """A min-p above 1 keeps the first of the largest logits alone, as a top-k of 1 does."""
    x, u = _logits(6, 9000, TYPES[kind], 97)
    x[:, [100, 5000, 8999]] = 50.0
    x[4, [7, 70]] = math.inf
    x[5] = 2.0
    u[:] = 0.999
    least = torch.tensor([1.0, 1.0000001, 1.5, math.inf, 2.0, 3.0])
    for settings in (dict(), dict(top_k=2), dict(top_p=0.9), dict(temperature=math.inf), dict(temperature=0.3, top_k=500, top_p=0.5)):
        tokens = _check(pkg, cuda, x, u, min_p=least, **settings)
        assert tokens[1:].tolist() == [100, 100, 100, 7, 0]

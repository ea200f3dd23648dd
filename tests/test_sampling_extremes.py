"""sample_tokens where settings and logits are at their ends together, against its definition in 64 bits; bounds are those
of test_sampling.py."""
import math

import pytest
import torch
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

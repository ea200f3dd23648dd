"""sample_tokens against its definition in 64 bits, row by row.  Tokens have to be equal: the weights and sums are of 64
bits on both sides, off by less than 2^-40 of the total in any order (2^20 terms of 2^-52, and the exponent's argument, at
most 2^10, with 2^-52), so a row may differ only where one of its decisions lies within 2^-40 of a border, of which random
rows have none.  Logarithms are rounded once to 32 bits: 2^-24 of the value, and 2^-40 from the sums."""
import math

import pytest
import torch
from shared_oracle import sample

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _logits(rows, vocab, dtype, seed, scale=2.0, likely=20):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g) * scale
    for r in range(rows):
        at = torch.randint(vocab, (min(likely, vocab),), generator=g)
        x[r, at] = 4 + 8 * torch.rand((len(at),), generator=g)
    return x.to(dtype), torch.rand((rows,), generator=g)


def _check(pkg, cuda, x, u, logits=None, **settings):
    """x: the CPU's logits; logits: the tensor of the call (x on the GPU by default)."""
    on_gpu = {k: v.to(cuda) if torch.is_tensor(v) else v for k, v in settings.items()}
    tokens, logs = pkg.sample_tokens(x.to(cuda) if logits is None else logits, u.to(cuda), return_logprobs=True, **on_gpu)
    assert tokens.dtype == torch.int64 and logs.dtype == torch.float32 and tokens.shape == u.shape == logs.shape
    alone = pkg.sample_tokens(x.to(cuda) if logits is None else logits, u.to(cuda), **on_gpu)
    assert torch.equal(alone, tokens)
    for r in range(x.shape[0]):
        row = {k: v[r].item() if torch.is_tensor(v) else v for k, v in settings.items()}
        token, log, near = sample(x[r], u[r].item(), **row)
        assert near > 2.0 ** -40 or near == 0, f"row {r} lies on a border: choose inputs by the definition, not by luck"
        got = int(tokens[r])
        assert got == token, f"row {r}: {got} for {token} ({row}, u {u[r].item()})"
        if math.isinf(log):
            assert float(logs[r]) == log
        else:
            assert abs(float(logs[r]) - log) <= abs(log) * 2.0 ** -24 * 1.0001 + 2.0 ** -40
    return tokens


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=7), dict(top_k=300, temperature=1.5), dict(top_p=0.9),
            dict(top_p=0.3), dict(top_p=0.9999), dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1.0), dict(temperature=0.0),
            dict(temperature=0.6, top_k=20, top_p=0.95), dict(temperature=1.2, top_k=50, top_p=0.8, min_p=0.02),
            dict(top_p=0.7, min_p=0.3), dict(temperature=100.0), dict(temperature=1e-3), dict(temperature=1e-30),
            dict(temperature=math.inf)]


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("kind", list(TYPES))
def test_settings(pkg, cuda, settings, kind):
    x, u = _logits(6, 1003, TYPES[kind], 1)
    _check(pkg, cuda, x, u, **settings)


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 1000, 1024, 1025, 4099, 32000, 50257])
@pytest.mark.parametrize("kind", list(TYPES))
def test_vocabularies(pkg, cuda, vocab, kind):
    x, u = _logits(3, vocab, TYPES[kind], vocab)
    for settings in (dict(), dict(top_k=5), dict(top_p=0.8), dict(temperature=0.8, top_k=40, top_p=0.9, min_p=0.01)):
        _check(pkg, cuda, x, u, **settings)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows", [1, 2, 40])
def test_a_model_s_vocabulary(pkg, cuda, kind, rows):
    x, u = _logits(rows, 151936, TYPES[kind], 7, likely=60)
    for settings in (dict(), dict(temperature=0.7, top_k=20, top_p=0.8), dict(top_p=0.95), dict(top_k=3000),
                     dict(temperature=2.0, top_p=0.99), dict(min_p=0.1)):
        _check(pkg, cuda, x, u, **settings)


def test_settings_per_row(pkg, cuda):
    rows = 96
    x, u = _logits(rows, 2000, torch.float16, 3)
    g = torch.Generator().manual_seed(4)
    pick = lambda values, dtype: torch.tensor(values, dtype=dtype)[torch.randint(len(values), (rows,), generator=g)]  # noqa: E731
    every = dict(temperature=pick([0.0, -1.0, math.nan, 0.5, 1.0, 2.0], torch.float32),
                 top_k=pick([-5, 0, 1, 2, 50, 1999, 2000, 5000, 2 ** 31 - 1], torch.int32),
                 top_p=pick([-1.0, 0.0, 0.5, 0.9, 1.0, 2.0], torch.float32), min_p=pick([-1.0, 0.0, 0.1, 0.5, 1.0], torch.float32))
    _check(pkg, cuda, x, u, **every)
    for name, value in every.items():
        _check(pkg, cuda, x, u, **{name: value})


@pytest.mark.parametrize("kind", list(TYPES))
def test_ties(pkg, cuda, kind):
    """Equal logits rank by index: the first of them stay, and are drawn in order."""
    g = torch.Generator().manual_seed(9)
    x = torch.randint(0, 4, (12, 3001), generator=g).to(TYPES[kind])
    u = torch.rand((12,), generator=g)
    for settings in (dict(), dict(top_k=1), dict(top_k=100), dict(top_k=1500), dict(top_p=0.2003), dict(top_p=0.9001), dict(temperature=0.0),
                     dict(top_k=777, top_p=0.501), dict(min_p=0.3), dict(top_k=900, min_p=0.9)):
        _check(pkg, cuda, x, u, **settings)
    x = torch.zeros((5, 4000), dtype=TYPES[kind])
    x[1::2] = -0.0
    x[2, ::2] = -0.0
    u = torch.tensor([0.0, 0.24999, 0.50001, 0.75001, 0.999999])
    for settings in (dict(), dict(top_k=1), dict(top_k=1001), dict(top_p=0.40011), dict(temperature=0.0), dict(top_k=10, top_p=0.55)):
        _check(pkg, cuda, x, u, **settings)


@pytest.mark.parametrize("kind", list(TYPES))
def test_infinities_and_nan(pkg, cuda, kind):
    t = TYPES[kind]
    x, u = _logits(10, 500, t, 11)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 1:] = -math.inf
    x[3, :499] = -math.inf
    x[4, ::2] = math.nan
    x[5, 7] = math.inf
    x[6, [3, 100, 499]] = math.inf
    x[6, 50] = math.nan
    x[7] = math.inf
    x[8] = torch.finfo(t).min
    x[9, ::3] = torch.finfo(t).min
    x[9, 5] = torch.finfo(t).max
    for settings in (dict(), dict(temperature=0.0), dict(top_k=2), dict(top_k=400), dict(top_p=0.49), dict(min_p=0.5),
                     dict(temperature=0.5, top_k=3, top_p=0.9, min_p=0.1), dict(temperature=math.inf)):
        tokens = _check(pkg, cuda, x, u, **settings)
        assert tokens[:2].tolist() == [-1, -1]


def test_random_numbers_at_the_ends(pkg, cuda):
    x, _ = _logits(1, 300, torch.float32, 13)
    x[0, 0] = x[0, 299] = -200.0  # weights of 10^-93: u = 0 draws the first token of any weight
    for u in (0.0, -0.5, math.nan, 2.0 ** -30, 1 - 2.0 ** -24, 1.0, 7.0, math.inf):
        for settings in (dict(), dict(top_k=4), dict(top_p=0.5)):
            _check(pkg, cuda, x, torch.tensor([u]), **settings)


def test_shapes_and_strides(pkg, cuda):
    x, u = _logits(12, 777, torch.bfloat16, 17)
    want = pkg.sample_tokens(x.to(cuda), u.to(cuda), top_k=50)
    # rows of a wider buffer, from an odd element on: no alignment at all
    wide = torch.full((12, 1001), 50.0, dtype=torch.bfloat16, device=cuda)
    wide[:, 3:780] = x.to(cuda)
    assert torch.equal(_check(pkg, cuda, x, u, logits=wide[:, 3:780], top_k=50), want)
    # a model's logits [batch, tokens, vocab], last positions; a transposed tensor; one row; none
    three = x.to(cuda).view(4, 3, 777)
    assert torch.equal(pkg.sample_tokens(three, u.to(cuda).view(4, 3), top_k=50), want.view(4, 3))
    assert torch.equal(pkg.sample_tokens(three[:, -1], u.to(cuda).view(4, 3)[:, -1], top_k=50), want.view(4, 3)[:, -1])
    assert torch.equal(pkg.sample_tokens(x.to(cuda).t().contiguous().t(), u.to(cuda), top_k=50), want)
    assert torch.equal(pkg.sample_tokens(x[5].to(cuda), u[5].to(cuda), top_k=50), want[5])
    assert pkg.sample_tokens(x[:0].to(cuda), u[:0].to(cuda)).shape == (0,)
    # one row for all: stride 0
    many = torch.rand((9,))
    _check(pkg, cuda, x[2:3].expand(9, 777), many, logits=x[2:3].to(cuda).expand(9, 777), top_p=0.9)


def test_draws_follow_the_distribution(pkg, cuda):
    """Evenly spread numbers draw every token as often as its probability says, off by 1 in 4096 at each of its ends."""
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5]).to(cuda)
    n = 4096
    u = (torch.arange(n, device=cuda) + 0.5) / n
    tokens = pkg.sample_tokens(x.expand(n, 5), u, temperature=1.5)
    share = torch.bincount(tokens, minlength=5).double().cpu() / n
    assert ((share - torch.softmax(x.double().cpu() / 1.5, 0)).abs() <= 1.0 / n + 1e-9).all()


def test_equal_calls_give_equal_bits_in_a_graph_and_on_another_stream(pkg, cuda):
    x, u = (t.to(cuda) for t in _logits(33, 20000, torch.float16, 19))
    flat = torch.randn((33, 20000), generator=torch.Generator().manual_seed(23)).half().to(cuda)
    calls = [dict(), dict(top_p=0.9), dict(top_k=64, top_p=0.9, min_p=0.01), dict(top_p=0.999)]

    def run(logits, uniform):
        return [t for c in calls for t in pkg.sample_tokens(logits, uniform, return_logprobs=True, **c)]

    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        xs, us = x.clone(), u.clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(xs, us)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(xs, us)
        graphs.append((graph, xs, us, out))
    for i in range(6):
        logits, uniform = (x, flat)[i % 2], torch.rand((33,), generator=torch.Generator().manual_seed(i)).to(cuda)
        want = run(logits, uniform)
        for graph, xs, us, _ in graphs:
            xs.copy_(logits)
            us.copy_(uniform)
            graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = run(logits, uniform)
        torch.cuda.synchronize()
        for got in (again, *(g[3] for g in graphs)):
            assert all(torch.equal(a, b) for a, b in zip(got, want))

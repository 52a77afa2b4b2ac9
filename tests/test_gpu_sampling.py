"""Sampling against the definition in 64 bits.

A draw is a comparison of running sums, so the exact one can fall to a neighbour where float32
exponentials (relative error below 2^-21 at |z| <= 8, below 2^-18 at any z that still has a weight;
1e-5 covers them) or the weights' whole numbers (each floor loses less than 2^-31 of the largest
weight, so the sum, at least that weight, moves by less than vocab 2^-31 of itself) move the sums.
Every row is therefore drawn five times in 64 bits, with the random number and top_p moved by that
share of the mass either way: where all agree (asserted for nearly all rows) the kernel's token is
that one, elsewhere it lies, in index order, between the first and the last of them. Tokens are
also compared, without any tolerance, with the whole-number definition evaluated by torch on the
same device.
"""

from __future__ import annotations

import math

import pytest
import torch

from augur_b200.sampling import sample_tokens

pytestmark = pytest.mark.gpu

_INF = math.inf


def exact_row(x, u, t, k, p, m):
    """(token, logprob) of one row in 64 bits."""
    x = torch.where(torch.isnan(x), -_INF, x).double()
    most = x.max()
    if most == -_INF:
        return -1, -_INF
    if not t > 0:
        return int((x == most).nonzero()[0]), 0.0
    z = torch.where(x == most, 0.0, (x - most) / t)
    z = torch.where(torch.isnan(z), -_INF, z)
    e = z.exp()
    e = torch.where(e < 2.0 ** -31, 0.0, e)
    order = torch.argsort(z, descending=True, stable=True)
    if 0 < k < order.numel():
        order = order[:k]
    mass = e[order].cumsum(0)
    keep = (e[order] >= min(m, 1.0)) & ((mass - e[order] < max(p, 1e-300) * mass[-1]) if p < 1 else True)
    keep[0] = True
    order = order[keep].sort().values
    mass = e[order].cumsum(0)
    at = min(int((mass <= min(max(u, 0.0), 1.0) * mass[-1]).sum()), int((mass < mass[-1]).sum()))
    return int(order[at]), float(z[order[at]] - mass[-1].log())


def whole_number_rows(logits, uniform, temperature, top_k, top_p, min_p):
    """The whole-number definition, by torch on the logits' device."""
    x = logits.float()
    x = torch.where(torch.isnan(x), -_INF, x)
    vocab = x.shape[1]
    most = x.amax(1, keepdim=True)
    t = temperature.unsqueeze(1)
    greedy = ~(t > 0)
    z = (x - most) * (1.0 / torch.where(greedy, 1.0, t))
    z = torch.where(torch.isnan(z) | greedy, -_INF, z)
    z = torch.where(x == most, 0.0, z)
    w = (z.exp() * 2.0 ** 31).floor().long()
    k = top_k.unsqueeze(1).long()
    k = torch.where(greedy, 1, torch.where((k <= 0) | (k > vocab), vocab, k))
    down, order = z.sort(dim=1, descending=True, stable=True)
    rank = torch.arange(vocab, device=x.device)
    ws = w.gather(1, order) * (rank < k)
    run = ws.cumsum(1)
    p = top_p.double().unsqueeze(1)
    need = torch.where(p < 1, (p * run[:, -1:].double()).ceil().long().clamp(min=1), run[:, -1:] + 1)
    kept = (run - ws < need) & (rank < k) & (down.exp() >= min_p.clamp(max=1.0).unsqueeze(1))
    keep = torch.zeros_like(kept).scatter_(1, order, kept)
    run = (w * keep).cumsum(1)
    total = run[:, -1:]
    target = torch.minimum((uniform.double().unsqueeze(1) * total.double()).floor().long().clamp(min=0), total - 1)
    token = (run <= target).sum(1).clamp(max=vocab - 1)
    logprob = z.gather(1, token.unsqueeze(1))[:, 0].double() - (total[:, 0].double() * 2.0 ** -31).log()
    nothing = most[:, 0] == -_INF
    return torch.where(nothing, -1, token), torch.where(nothing, -_INF, logprob)


def check(logits, uniform, temperature, top_k, top_p, min_p, sure=0.75):
    rows, device = logits.shape[0], logits.device

    def full(v, dtype):
        return v.to(dtype) if isinstance(v, torch.Tensor) else torch.full((rows,), v, dtype=dtype, device=device)

    tokens, logprobs = sample_tokens(logits, uniform, temperature, top_k, top_p, min_p)
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32 and tokens.shape == logprobs.shape == (rows,)
    per_row = [full(temperature, torch.float32), full(top_k, torch.int32), full(top_p, torch.float32), full(min_p, torch.float32)]
    whole_tokens, whole_logprobs = whole_number_rows(logits, uniform, *per_row)
    assert torch.equal(tokens, whole_tokens)
    # the same kept sum, its logarithm and one subtraction in float32: 2^-22 of each, and of the sum's rounding
    some = torch.isfinite(whole_logprobs)
    assert torch.equal(torch.isfinite(logprobs), some)
    assert ((logprobs.double() - whole_logprobs).abs()[some] <= 2.0 ** -21 * (1 + 25 + whole_logprobs.abs()[some])).all()
    settings = list(zip(uniform.tolist(), *(v.tolist() for v in per_row)))
    agree, vocab = 0, logits.shape[1]
    share = 1e-5 + vocab * 2.0 ** -31
    for b, (u, t, k, p, m) in enumerate(settings):
        token, logprob = exact_row(logits[b], u, t, k, p, m)
        near = {token} | {exact_row(logits[b], u + du, t, k, p + dp if p < 1 else p, m)[0]
                          for du, dp in ((share, 0), (-share, 0), (0, share), (0, -share))}
        assert min(near) <= int(tokens[b]) <= max(near), (b, int(tokens[b]), near)
        if len(near) == 1:
            agree += 1
            if math.isinf(logprob):
                assert float(logprobs[b]) == logprob
            else:  # float32: z's relative error 2^-22 (|z| < 21.5), the sum's share, a moved nucleus edge below 1e-3
                assert abs(float(logprobs[b]) - logprob) <= share + 1e-5 * abs(logprob) + (2e-3 if p < 1 else 0)
    assert agree >= sure * rows, (agree, rows)
    return tokens


def make(cuda, rows, vocab, dtype, seed=0, spread=2.0, likely=20):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, device=cuda) * spread
    if likely:
        at = torch.randint(0, vocab, (rows, likely), generator=g, device=cuda)
        x.scatter_add_(1, at, 4 + 8 * torch.rand(rows, likely, generator=g, device=cuda))
    return x.to(dtype), torch.rand(rows, generator=g, device=cuda)


_SETTINGS = [
    (1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.8, 40, 0.95, 0.02), (1.2, 0, 1.0, 0.1),
    (0.0, 0, 1.0, 0.0), (1.0, 1, 0.5, 0.5), (1.5, 3000, 0.8, 0.0), (1.0, 900, 0.99, 0.0), (0.05, 7, 0.3, 0.0),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 32003, 151936])
def test_settings_per_row(cuda, dtype, vocab):
    rows = 2 * len(_SETTINGS) + 1
    logits, u = make(cuda, rows, vocab, dtype, seed=vocab)
    cols = list(zip(*(_SETTINGS[b % len(_SETTINGS)] for b in range(rows))))
    check(logits, u, *(torch.tensor(c, device=cuda, dtype=torch.int32 if i == 1 else torch.float32) for i, c in enumerate(cols)))


@pytest.mark.parametrize("rows", [1, 3, 40, 300])
@pytest.mark.parametrize("setting", _SETTINGS[:5])
def test_scalar_settings(cuda, rows, setting):
    check(*make(cuda, rows, 20011, torch.bfloat16, seed=rows), *setting)


@pytest.mark.parametrize("setting", _SETTINGS)
@pytest.mark.parametrize("kind", ["equal", "flat", "two values", "coarse"])
def test_rows_that_hold_too_many_candidates(cuda, kind, setting):
    """Flat rows, whose candidates do not fit a sorted list, and rows of ties."""
    rows, vocab = 4, 40013
    g = torch.Generator(device=cuda).manual_seed(2)
    u = torch.rand(rows, generator=g, device=cuda)
    x = torch.randn(rows, vocab, generator=g, device=cuda)
    if kind == "equal":
        x = torch.zeros_like(x)
    elif kind == "flat":
        x = x * 0.01
    elif kind == "two values":
        x = (x > 1.0).float()
    else:
        x = (x * 4).round() / 4
    check(x.to(torch.bfloat16 if kind == "coarse" else torch.float32), u, *setting, sure=0.0)


def test_rows_without_a_choice(cuda):
    vocab = 5003
    x, u = make(cuda, 9, vocab, torch.float32, likely=0)
    x[0] = -_INF
    x[1] = torch.nan
    x[2, :] = -_INF
    x[2, 4321] = -5.0
    x[3, 17] = torch.nan
    x[4, 100] = x[4, 3000] = _INF
    x[5] = torch.finfo(torch.float32).min
    x[6, ::2] = torch.finfo(torch.float32).min
    x[7] = -_INF
    x[7, :2] = torch.finfo(torch.float32).min
    for setting in _SETTINGS:
        tokens = check(x, u, *setting, sure=0.0)
        assert tokens[0] == tokens[1] == -1 and tokens[2] == 4321
        assert int(tokens[4]) in (100, 3000) and int(tokens[7]) in (0, 1)


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 1.0, -1.0, math.nan])
@pytest.mark.parametrize("setting", _SETTINGS[:4])
def test_random_numbers_at_the_ends(cuda, u, setting):
    x, _ = make(cuda, 3, 3001, torch.float32)
    tokens, logprobs = sample_tokens(x, torch.full((3,), u, device=cuda), *setting)
    low = 0.0 if not u > 0 else u
    ends = [exact_row(x[b], low, *setting)[0] for b in range(3)]
    near = [exact_row(x[b], min(low, 1.0) * (1 - 1e-5), *setting)[0] for b in range(3)]
    assert all(int(t) in (e, n) for t, e, n in zip(tokens, ends, near)) and torch.isfinite(logprobs).all()


@pytest.mark.parametrize("temperature,top_p,min_p", [(math.inf, 1.0, 0.0), (1e-30, 1.0, 0.0), (1e-45, 0.9, 0.0),
                                                     (-1.0, 1.0, 0.0), (math.nan, 1.0, 0.0), (1.0, 0.0, 0.0),
                                                     (1.0, -1.0, 0.0), (1.0, 1.0, 7.0), (1.0, math.nan, 0.0)])
def test_settings_at_the_ends(cuda, temperature, top_p, min_p):
    x, u = make(cuda, 4, 3001, torch.float32)
    tokens, logprobs = sample_tokens(x, u, temperature, 0, top_p, min_p)
    if temperature == math.inf:  # uniform over the vocabulary
        assert torch.equal(tokens, (u.double() * 3001).floor().long())
    elif math.isnan(top_p):
        assert torch.equal(tokens, sample_tokens(x, u)[0])
    else:
        assert torch.equal(tokens, x.argmax(1)) and (logprobs.abs() < 1e-5).all()


def test_layouts_streams_and_batches(cuda):
    """A row's token depends on the row, its number and its settings alone."""
    vocab = 30011
    x, u = make(cuda, 37, vocab, torch.float16)
    args = dict(temperature=0.9, top_k=60, top_p=0.9)
    want, logp = sample_tokens(x, u, **args)
    padded = torch.zeros(37, vocab + 13, dtype=torch.float16, device=cuda)
    for shift in (0, 1, 3, 8):  # rows that start anywhere in a 16-byte granule
        padded[:, shift:shift + vocab] = x
        got = sample_tokens(padded[:, shift:shift + vocab], u, **args)
        assert torch.equal(got[0], want) and torch.equal(got[1], logp)
    assert torch.equal(sample_tokens(x.t().contiguous().t(), u, **args)[0], want)
    for b in (0, 5, 36):
        assert torch.equal(sample_tokens(x[b:b + 1], u[b:b + 1], **args)[0], want[b:b + 1])
    wide = x.repeat(20, 1)
    assert torch.equal(sample_tokens(wide, u.repeat(20), **args)[0], want.repeat(20))
    assert torch.equal(sample_tokens(x, u.repeat_interleave(2)[::2], **args)[0], want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = sample_tokens(x, u, **args, stream=side)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = sample_tokens(x, u, **args)[0]
    torch.cuda.current_stream().wait_stream(side)
    x.copy_(x.flip(0))
    u.copy_(u.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want.flip(0))


@pytest.mark.parametrize("vocab", [420001, 900001, 1 << 21])
def test_vocabularies_beyond_shared_memory(cuda, vocab):
    x, u = make(cuda, 5, vocab, torch.float32, likely=200)
    t, k, p, m = (torch.tensor(c, device=cuda) for c in zip(*(_SETTINGS[i] for i in (0, 1, 2, 3, 7))))
    check(x, u, t, k, p, m, sure=0.0)


def test_refusals(cuda):
    x, u = make(cuda, 3, 100, torch.float32)
    with pytest.raises(ValueError, match=r"\[rows, vocab\]"):
        sample_tokens(x[0], u)
    with pytest.raises(ValueError, match="no CPU fallback"):
        sample_tokens(x.cpu(), u.cpu())
    with pytest.raises(ValueError, match="uniform must be"):
        sample_tokens(x, u[:2])
    with pytest.raises(ValueError, match="uniform must be"):
        sample_tokens(x, u.double())
    with pytest.raises(ValueError, match="unsupported logits dtype"):
        sample_tokens(x.double(), u)
    with pytest.raises(ValueError, match="temperature must be"):
        sample_tokens(x, u, temperature=u[:2])
    with pytest.raises(ValueError, match="logits' device"):
        sample_tokens(x, u, top_p=u.cpu())
    with pytest.raises(ValueError, match="vocab must be"):
        sample_tokens(x[:, :0], u)
    tokens, logprobs = sample_tokens(x[:0], u[:0])
    assert tokens.shape == logprobs.shape == (0,)


@pytest.mark.parametrize("vocab", [3001, 40013, 151936])
@pytest.mark.parametrize("depth", [1.0, 3.0, 6.0, 9.0, 12.0, 15.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nucleus_ends_close_to_a_depth(cuda, vocab, depth, dtype):
    """Entries crowded around one depth below the maximum, a nucleus that ends at every place among them."""
    rows = 24
    g = torch.Generator(device=cuda).manual_seed(int(depth))
    x = -depth + 0.2 * (torch.rand(rows, vocab, generator=g, device=cuda) - 0.5)
    x[:, 77] = 0.0
    x = x.to(dtype)
    top_p = torch.linspace(0.02, 0.999, rows, device=cuda)
    settings = (torch.rand(rows, generator=g, device=cuda), torch.ones(rows, device=cuda),
                torch.zeros(rows, dtype=torch.int32, device=cuda), top_p, torch.zeros(rows, device=cuda))
    tokens, logprobs = sample_tokens(x, settings[0], top_p=top_p)
    want, want_logprobs = whole_number_rows(x, *settings)
    assert torch.equal(tokens, want)
    assert ((logprobs.double() - want_logprobs).abs() <= 2.0 ** -21 * (1 + 25 + want_logprobs.abs())).all()


@pytest.mark.parametrize("seed", range(8))
def test_wide_nuclei(cuda, seed):
    """Many rows of top-p alone: the kept sum is the definition's to the last unit."""
    rows, vocab = 96, 32003
    x, u = make(cuda, rows, vocab, torch.float16 if seed % 2 else torch.float32, seed=100 + seed)
    g = torch.Generator(device=cuda).manual_seed(seed)
    top_p = torch.tensor([0.7, 0.8, 0.9, 0.95, 0.99], device=cuda)[torch.randint(0, 5, (rows,), generator=g, device=cuda)]
    t = 0.8 + 0.6 * torch.rand(rows, generator=g, device=cuda)
    tokens, logprobs = sample_tokens(x, u, temperature=t, top_p=top_p)
    zero = torch.zeros(rows, device=cuda)
    want, want_logprobs = whole_number_rows(x, u, t, zero.int(), top_p, zero)
    assert torch.equal(tokens, want)
    assert ((logprobs.double() - want_logprobs).abs() <= 2.0 ** -21 * (1 + 25 + want_logprobs.abs())).all()


@pytest.mark.parametrize("temperature", [0.03, 1.0, 40.0])
@pytest.mark.parametrize("move", ["maximum 0", "cut near 0", "far up", "far down", "tiny", "huge"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_limits_anywhere_among_the_floats(cuda, move, temperature, dtype):
    g = torch.Generator(device=cuda).manual_seed(17)
    rows, vocab = 12, 20011
    x = torch.randn(rows, vocab, generator=g, device=cuda) * 2.0 * temperature
    if move == "maximum 0":
        x = x - x.amax(1, keepdim=True)
    elif move == "cut near 0":  # where the floats are densest
        x = x - x.topk(400, dim=1).values[:, -1:]
    elif move in ("far up", "far down"):
        x = x + (1e5 if move == "far up" else -1e5) * temperature
    elif move in ("tiny", "huge"):
        scale = 1e-30 if move == "tiny" else 1e30
        x, temperature = x * scale, temperature * scale
    logits = x.to(dtype)
    uniform = torch.rand(rows, generator=g, device=cuda)
    for k, p, m in ((50, 1.0, 0.0), (0, 0.9, 0.0), (3000, 0.7, 0.0), (0, 1.0, 0.05), (0, 0.97, 0.001)):
        per_row = (torch.full((rows,), v, dtype=d, device=cuda)
                   for v, d in ((temperature, torch.float32), (k, torch.int32), (p, torch.float32), (m, torch.float32)))
        tokens, logprobs = sample_tokens(logits, uniform, temperature, k, p, m)
        want, want_logprobs = whole_number_rows(logits, uniform, *per_row)
        assert torch.equal(tokens, want), (k, p, m)
        # as in check: float32 roundings of z, of the kept sum's logarithm and of their difference
        assert ((logprobs.double() - want_logprobs).abs() <= 2.0 ** -21 * (26 + want_logprobs.abs())).all()

"""sample_tokens against its definition in 64 bits, token by token: vocabularies of every size, ties, settings by row and for all,
flat and steep rows that defeat each of the ways a border is found, masked rows, and random numbers at the ends."""
from __future__ import annotations

import pytest
import torch

from forge_amd import _lib, ops_gemm
from forge_amd.errors import ConfigError
from forge_amd.ops_sampling import sample_tokens
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")


def _reference(logits, uniform, temperature, top_k, top_p, min_p):
    """(tokens, log probabilities, distance of u from the nearest border as a share of the total) row by row, in 64 bits."""
    tokens, logs, far = [], [], []
    for row, u, t, k, p, m in zip(logits.double(), uniform.double().tolist(), temperature, top_k, top_p, min_p):
        row = torch.where(row.isnan(), -INF, row)
        top = row.max()
        if top == -INF:
            tokens.append(-1), logs.append(-INF), far.append(1.0)
            continue
        order = torch.sort(row, descending=True, stable=True)[1]
        if not t > 0:
            token, gap = int(order[0]), 1.0
        else:
            w = torch.exp((row - top) / t)
            w[row == top] = 1.0
            ranked = w[order]
            n = min(k, len(row)) if k > 0 else len(row)
            sums = ranked[:n].cumsum(0)
            before = torch.cat((torch.zeros(1, dtype=torch.float64), sums[:-1]))
            keep = torch.ones(n, dtype=torch.bool) if not p < 1 else before < max(p, 1e-300) * sums[-1]
            keep &= (ranked[:n] >= min(m, 1.0)) & (ranked[:n] > 0)
            kept = torch.zeros_like(w)
            kept[order[:n][keep]] = ranked[:n][keep]
            cum = kept.cumsum(0)
            mark = min(max(u, 0.0), 1.0) * cum[-1] if u == u else 0.0
            index = torch.nonzero(kept).flatten()
            at = int((cum[index] <= mark).sum())
            token = int(index[min(at, len(index) - 1)])
            gap = float((cum[index] - mark).abs().min() / cum[-1])
        tokens.append(token), far.append(gap)
        logs.append(float(row[token] - torch.logsumexp(row, 0)) if top < INF else float("nan"))
    return torch.tensor(tokens), torch.tensor(logs, dtype=torch.float64), torch.tensor(far)


def _each(x, b, none):
    return [none] * b if x is None else (x.double().tolist() if isinstance(x, torch.Tensor) else [x] * b)


def _check(logits, uniform, temperature=1.0, top_k=None, top_p=None, min_p=None):
    b = logits.shape[0]
    # numbers reach the kernel in 32 bits
    one = lambda x: x if x is None or isinstance(x, (int, torch.Tensor)) else float(torch.tensor(x, dtype=FP))  # noqa: E731
    top_k_rows = [int(k) for k in _each(top_k, b, 0)]
    want, logs, _ = _reference(logits, uniform, _each(one(temperature), b, 1.0), top_k_rows, _each(one(top_p), b, 1.0), _each(one(min_p), b, 0.0))
    on = lambda x: x.to(DEV) if isinstance(x, torch.Tensor) else x  # noqa: E731
    token, logprob = sample_tokens(logits.to(DEV), uniform.to(DEV), temperature=on(temperature), top_k=on(top_k), top_p=on(top_p),
                                   min_p=on(min_p), return_logprobs=True)
    assert token.dtype == torch.int64 and logprob.dtype == FP
    assert torch.equal(token.cpu(), want), (token.cpu() - want).nonzero().flatten()
    fine = torch.isfinite(logs)
    got = logprob.cpu().double()
    # a difference, a sum of V powers (of hardware's 2^x) and a logarithm in fp32
    assert bool(((got - logs)[fine].abs() <= 2.0 ** -17 * (1 + logs[fine].abs())).all())
    assert torch.equal(got[~fine].isnan(), logs[~fine].isnan()) and torch.equal(got[~fine] == -INF, logs[~fine] == -INF)
    return token


def _logits(b, v, dt, seed=0, spread=2.5):
    g = gen(seed + 3 * v + b)
    x = spread * torch.randn(b, v, generator=g) - 3 * torch.log(torch.rand(b, v, generator=g).clamp_min(1e-30)) * (torch.rand(b, v, generator=g) < 0.003)
    return x.to(dt), torch.rand(b, generator=g)


SETTINGS = [dict(), dict(top_k=1), dict(top_k=5), dict(top_p=0.3), dict(top_p=0.9), dict(top_p=0.0), dict(min_p=0.1), dict(top_k=40, top_p=0.8),
            dict(top_k=700, top_p=0.99, min_p=0.001), dict(temperature=0.0), dict(temperature=0.3, top_p=0.95), dict(temperature=5.0, top_k=100),
            dict(temperature=100.0, top_p=0.5), dict(temperature=0.01), dict(top_k=10 ** 9, top_p=1.0), dict(min_p=1.0), dict(min_p=3.0)]


@pytest.mark.parametrize("dt", [FP, BF, HF])
@pytest.mark.parametrize("v", [1, 2, 63, 1000, 4096, 4097, 20011])
def test_vocabularies_and_settings(v, dt):
    x, u = _logits(7, v, dt)
    for kw in SETTINGS:
        _check(x, u, **kw)


@pytest.mark.parametrize("dt", [FP, BF])
@pytest.mark.parametrize("b,v", [(1, 150001), (3, 131072), (600, 5000), (40, 32000)])
def test_batches_and_long_rows(b, v, dt):
    x, u = _logits(b, v, dt)
    for kw in (dict(top_k=50, top_p=0.9), dict(top_p=0.95), dict(temperature=0.7, min_p=0.02), dict(temperature=1.5, top_k=6000, top_p=0.999)):
        _check(x, u, **kw)


def test_settings_by_row():
    b = 64
    for v, dt in ((9001, FP), (32000, BF)):
        x, u = _logits(b, v, dt)
        g = gen(v)
        t = torch.where(torch.rand(b, generator=g) < 0.2, 0.0, 0.2 + 2 * torch.rand(b, generator=g))
        k = torch.where(torch.rand(b, generator=g) < 0.4, 0, torch.exp(9 * torch.rand(b, generator=g)).int()).to(torch.int32)
        p = torch.where(torch.rand(b, generator=g) < 0.3, 1.0, torch.rand(b, generator=g))
        m = torch.where(torch.rand(b, generator=g) < 0.6, 0.0, 0.2 * torch.rand(b, generator=g))
        k[0], p[1], m[2], t[3], t[4], p[5] = -7, -1.0, -1.0, -2.0, float("nan"), float("nan")
        _check(x, u, t, k, p, m)
        _check(x, u, 0.9, k, 0.9, None)
        wide = torch.zeros(b, v + 5, dtype=dt)
        wide[:, 3:-2] = x
        token = sample_tokens(wide.to(DEV)[:, 3:-2], u.to(DEV), temperature=t.to(DEV), top_k=k.to(DEV), top_p=p.to(DEV), min_p=m.to(DEV))
        assert torch.equal(token, _check(x, u, t, k, p, m))
        same = sample_tokens(x[:1].to(DEV).expand(b, v), u.to(DEV), top_p=0.9)
        assert torch.equal(same, _check(x[:1].expand(b, v), u, top_p=0.9))


@pytest.mark.parametrize("v", [1000, 30000])
def test_ties(v):
    """Few distinct logits: borders among equal ones go by the index."""
    g = gen(v)
    for distinct in (1, 2, 7):
        x = torch.randint(0, distinct, (9, v), generator=g).float()
        u = torch.rand(9, generator=g)
        for kw in (dict(), dict(top_k=1), dict(top_k=17), dict(top_k=v // 2), dict(top_k=v - 1), dict(top_p=0.5), dict(top_p=0.01),
                   dict(top_k=v // 3, top_p=0.7), dict(min_p=0.5), dict(temperature=0.0)):
            _check(x.to(BF), u, **kw)
    x = torch.where(torch.rand(9, v, generator=g) < 0.5, 0.0, -0.0)
    _check(x, u, top_k=v // 4)


def test_rows_that_crowd_a_bin():
    """Most tokens next to each other far below, or next to, a few others: more of them lie in a border's bin than a list holds."""
    g = gen(5)
    v = 50000
    x = torch.randn(6, v, generator=g) * 1e-4
    x[0, 7], x[1, 11], x[2, 3] = 30.0, 9.0, 12.0
    x[3] = torch.randn(v, generator=g) * 1e-6 + 1
    x[4, ::2] -= 20.0
    x[5, :5] = torch.tensor([40.0, 39.0, 38.0, 20.0, 10.0])
    u = torch.rand(6, generator=g)
    for kw in (dict(top_k=20000), dict(top_p=0.5), dict(top_k=30000, top_p=0.6), dict(temperature=3.0, top_p=0.9, top_k=45000), dict(top_k=10, top_p=0.9)):
        _check(x, u, **kw)


def test_rows_of_large_and_infinite_logits():
    g = gen(6)
    x = torch.randn(8, 5000, generator=g)
    x[0] *= 1e37
    x[1] = -INF
    x[1, 77] = -3e38
    x[2] = -INF
    x[3, ::3] = float("nan")
    x[4, 100] = x[4, 4000] = INF
    x[5] = float("nan")
    x[6] = -INF
    x[6, 4999] = x[6, 17] = 2.0
    x[7] *= 1e-40
    u = torch.tensor([0.3, 0.5, 0.5, 0.7, 0.6, 0.1, 0.99, 0.5])
    for kw in SETTINGS:
        token = _check(x, u, **kw)
        assert token[2] == -1 and token[5] == -1 and token[1] == 77


def test_random_numbers_at_the_ends():
    x, _ = _logits(1, 3000, FP)
    x = x.expand(9, 3000).contiguous()
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan"), INF, -INF, 2.0 ** -149])
    for kw in (dict(), dict(top_k=10), dict(top_p=0.9), dict(top_k=2000, top_p=0.999)):
        _check(x, u, **kw)


def test_every_token_of_a_row():
    """Random numbers on either side of each border of a small distribution, and equal shares to the bit."""
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5]).log_softmax(0)
    edges = x.double().exp().cumsum(0)[:-1]
    u = torch.cat([(edges + d).float() for d in (-1e-6, 1e-6)])
    want = torch.cat((torch.arange(4), torch.arange(1, 5)))
    assert torch.equal(sample_tokens(x.expand(8, 5).contiguous().to(DEV), u.to(DEV)).cpu(), want)
    even = torch.zeros(16, 4096)
    u = torch.arange(16) / 16
    assert torch.equal(sample_tokens(even.to(DEV), u.to(DEV)).cpu(), 256 * torch.arange(16))
    assert torch.equal(sample_tokens(even.to(DEV), u.to(DEV), top_k=1024).cpu(), 64 * torch.arange(16))
    assert torch.equal(sample_tokens(even.to(DEV), u.to(DEV), top_p=0.5).cpu(), 128 * torch.arange(16))


def test_graph_and_streams():
    x, u = (t.to(DEV) for t in _logits(5, 40000, BF))
    k = torch.tensor([0, 3, 50, 20000, 0], dtype=torch.int32, device=DEV)
    run = lambda: sample_tokens(x, u, temperature=0.9, top_k=k, top_p=0.95, return_logprobs=True)  # noqa: E731
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want[0], other[0]) and torch.equal(want[1], other[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i in range(4):
        x.copy_(_logits(5, 40000, BF, seed=i + 1)[0])
        u.copy_(torch.rand(5, generator=gen(i)))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(kept, run()))


def test_no_rows_and_refusals():
    x, u = torch.zeros(3, 100, device=DEV), torch.zeros(3, device=DEV)
    token, logprob = sample_tokens(x[:0], u[:0], return_logprobs=True)
    assert token.shape == logprob.shape == (0,)
    assert torch.equal(sample_tokens(torch.randn(100, 3, device=DEV).t(), u), sample_tokens(x, u) * 0)
    for bad in (dict(logits=x[0]), dict(logits=x.int()), dict(logits=x[:, :0]), dict(uniform=u[:2]), dict(uniform=u.double()), dict(uniform=u.cpu()),
                dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=-0.1), dict(min_p=-0.1),
                dict(temperature=u.half()), dict(top_k=u), dict(top_p=u[:2]), dict(min_p=u.cpu())):
        with pytest.raises(ConfigError):
            sample_tokens(**{"logits": x, "uniform": u, **bad})
    with pytest.raises(ops_gemm.HardwareUnsupported):
        sample_tokens(x.cpu(), u.cpu())
    with pytest.raises(_lib.KernelLaunchError, match="sizes"):
        sample_tokens(x[:1].expand(1 << 16, 100), torch.zeros(1 << 16, device=DEV))


@pytest.mark.parametrize("dt", [FP, BF])
@pytest.mark.parametrize("spread", [0.01, 0.7, 2.5, 9.0])
def test_borders_of_both_kinds_near_and_far(spread, dt):
    """Top-k's border in front of top-p's, behind it and in the same bin, in rows of few and of many tokens up to there."""
    k = torch.tensor([1, 2, 40, 255, 256, 257, 300, 1000, 4095, 4097, 5000, 12000, 20010, 0], dtype=torch.int32)
    for p in (1e-6, 0.2, 0.7, 0.95, 0.9999):
        logits, uniform = _logits(len(k), 20011, dt, seed=int(1000 * p), spread=spread)
        _check(logits, uniform, top_k=k, top_p=p)
    _check(logits, uniform, top_k=k, min_p=0.02)
    _check(logits[:2], uniform[:2], top_k=5000, top_p=0.8, temperature=0.5)  # a row in more chunks


@pytest.mark.parametrize("b,v", [(270, 40001), (1, 3000000), (9, 1200000)])
def test_rows_that_are_cut_up_more_finely_for_the_sums(b, v):
    """Many rows of long vocabularies, of which some are settled by few tokens and others need every sum; rows of most chunks."""
    logits, uniform = _logits(b, v, FP)
    k = torch.tensor([0, 5, 0, 0], dtype=torch.int32).repeat(b)[:b]
    p = torch.tensor([1.0, 0.9, 0.97, 0.3]).repeat(b)[:b]
    _check(logits, uniform, top_k=k, top_p=p)
    _check(logits[:9], uniform[:9])

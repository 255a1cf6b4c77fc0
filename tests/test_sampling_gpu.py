"""Sampling against its definition: token by token the torch statement (whole-number weights, so equal bit for bit), and a 64-bit
one of the probabilities.

The 64-bit bounds: a weight is off by half of 2^-31 and by fp32's exp of a rounded argument: (|y| + 4) 2^-24 of itself, at most 2^-19 for
the 22 units of |y| whose weights are not zero; so a cumulative share is off by at most 2^-19 + V 2^-32 of the kept sum (which is at
least the largest weight), and logprobs and log_norm by that and a few roundings of fp32 (2^-22 of their size)."""
import math

import pytest
import torch

import triton_distributed_b200 as tdist
from triton_distributed_b200 import _lib
from triton_distributed_b200.ops.sampling import ref_sample_tokens
from triton_distributed_b200.runtime import check_status

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _check(logits, u, t, k, p, m):
    got = tdist.sample_tokens(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)
    check_status()
    ref = ref_sample_tokens(logits, u, t, k, p, m)
    B, V = logits.shape
    assert torch.equal(got.tokens, ref.tokens), (got.tokens[got.tokens != ref.tokens], ref.tokens[got.tokens != ref.tokens])
    torch.testing.assert_close(got.logprobs, ref.logprobs, atol=2.0 ** -18, rtol=2.0 ** -22)
    torch.testing.assert_close(got.log_norm, ref.log_norm, atol=2.0 ** -18, rtol=2.0 ** -22)

    def at(v, b):
        return float(v[b]) if isinstance(v, torch.Tensor) else float(v)

    slack = 2.0 ** -19 + V * 2.0 ** -32
    for b in range(min(B, 12)):
        x = logits[b].double()
        x = torch.where(torch.isnan(x), -math.inf, x)
        if float(x.max()) in (-math.inf, math.inf):
            continue
        tok, tb = int(got.tokens[b]), at(t, b)
        if tb <= 0:
            assert tok == int((x == x.max()).nonzero()[0, 0]) and float(got.logprobs[b]) == 0 and float(got.log_norm[b]) == float(x.max())
            continue
        z = x / tb
        order = torch.sort(z, descending=True, stable=True).indices
        prob = torch.softmax(z[order], 0)
        kk, pp, mm = int(at(k, b)), at(p, b), at(m, b)
        n = V if kk <= 0 else min(kk, V)
        share = (torch.cumsum(prob, 0) - prob) / prob[:n].sum()
        low = high = torch.arange(V, device=x.device) < n
        if pp < 1:
            first = torch.arange(V, device=x.device) == 0
            low, high = low & ((share < pp - slack) | first), high & ((share < pp + slack) | first)
        low, high = low & (prob >= prob[0] * mm * (1 + slack) + slack * 0), high & (prob >= prob[0] * min(mm, 1.0) * (1 - slack))
        high = high & (prob > 0)
        low[0] = high[0] = True
        keep = torch.zeros(V, dtype=torch.bool, device=x.device).scatter_(0, order, high)
        assert bool(keep[tok]), (b, tok)
        # the share below the token lies at u, as far as the kept set is known
        full = torch.zeros(V, dtype=torch.float64, device=x.device).scatter_(0, order, prob)
        unsure = float((prob[high & ~low]).sum() / prob[low].sum()) + slack
        kept = full * keep
        total = float(kept.sum())
        upto = float(kept[:tok + 1].sum()) / total
        assert upto - float(kept[tok]) / total <= float(u[b]) + unsure and float(u[b]) <= upto + unsure, (b, tok)
        assert abs(float(got.log_norm[b]) - (float(torch.logsumexp(z[order][high], 0)))) <= unsure * 2 + 2.0 ** -20 * (1 + abs(float(z.max())))
    return got


def _settings(B, dev, seed):
    g = torch.Generator().manual_seed(seed)
    pick = lambda vals: torch.tensor([vals[int(i)] for i in torch.randint(len(vals), (B,), generator=g)], device=dev)   # noqa: E731
    return (pick([0.0, 0.3, 0.7, 1.0, 1.0, 2.5]), pick([0, 0, 1, 3, 50, 1000]).to(torch.int32), pick([1.0, 1.0, 0.0, 0.1, 0.5, 0.9, 0.999]),
            pick([0.0, 0.0, 0.02, 0.3, 1.0]))


@pytest.mark.parametrize("V", [1, 2, 7, 33, 1000, 4097, 32000, 100003])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B", [1, 5, 40])
def test_mixed_settings(cuda_device, V, dtype, B):
    torch.manual_seed(V + B)
    for spread in (0.1, 2.5, 12.0):
        logits = (torch.randn(B, V, device=cuda_device) * spread).to(DTYPES[dtype])
        logits[::3, ::2] = float("-inf") if V > 2 else 0.0
        _check(logits, torch.rand(B, device=cuda_device), *_settings(B, cuda_device, V + int(spread)))


@pytest.mark.parametrize("B,V", [(1, 200000), (3, 524032), (300, 2000), (200, 70000)])
def test_sizes_of_cluster(cuda_device, B, V):
    """One to eight CTAs per row; rows that take more CTAs than fill the machine."""
    torch.manual_seed(B)
    logits = torch.randn(B, V, device=cuda_device).mul_(3).to(torch.bfloat16)
    _check(logits, torch.rand(B, device=cuda_device), *_settings(B, cuda_device, B))


@pytest.mark.parametrize("V", [5000, 100003])
@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (1, 1.0, 0.0), (2500, 1.0, 0.0), (4999, 1.0, 0.0), (0, 0.3, 0.0), (0, 0.0, 0.0), (2500, 0.5, 0.0), (0, 0.99, 1.0),
                                   (3000, 0.9999, 0.5)])
def test_ties_by_the_thousand(cuda_device, V, k, p, m):
    """Flat rows; rows of two and of a few values; a peak over a flat rest; values one unit of fp32 apart."""
    dev = cuda_device
    torch.manual_seed(V)
    rows = [torch.zeros(V, device=dev), torch.full((V,), -3.5, device=dev), torch.randint(0, 2, (V,), device=dev).float(),
            torch.randint(-3, 3, (V,), device=dev) * 0.25, torch.zeros(V, device=dev).index_fill_(0, torch.tensor([V // 2], device=dev), 5.0),
            1.0 + torch.randint(0, 9, (V,), device=dev) * 2.0 ** -23, torch.where(torch.rand(V, device=dev) < 0.5, -0.0, 0.0),
            torch.where(torch.rand(V, device=dev) < 0.5, -1e-40, 1e-40)]
    logits = torch.stack(rows)
    for u in (0.0, 0.37, 1.0 - 2.0 ** -24):
        _check(logits, torch.full((len(rows),), u, device=dev), 1.0, k, p, m)


def test_rows_with_nothing_and_with_extremes(cuda_device):
    dev, V = cuda_device, 3001
    inf, nan = float("inf"), float("nan")
    torch.manual_seed(0)
    logits = torch.randn(9, V, device=dev)
    logits[0] = -inf
    logits[1] = nan
    logits[2] = -inf
    logits[2, 1234] = -200.0
    logits[3, [7, 2000]] = inf
    logits[4, ::5] = nan
    logits[5] = torch.finfo(torch.float32).min
    logits[6] = torch.finfo(torch.float32).min
    logits[6, 17] = torch.finfo(torch.float32).max
    logits[7] *= 1e-30
    logits[8, 5:] = torch.finfo(torch.float32).min
    for t in (0.0, 0.001, 1.0, 50.0):
        for k, p in ((0, 1.0), (2, 1.0), (0, 0.6), (40, 0.6)):
            got = tdist.sample_tokens(logits, torch.full((9,), 0.6, device=dev), t, k, p)
            ref = ref_sample_tokens(logits, torch.full((9,), 0.6, device=dev), t, k, p)
            check_status()
            assert torch.equal(got.tokens, ref.tokens), (t, k, p)
            assert got.tokens[:2].tolist() == [-1, -1] and int(got.tokens[2]) == 1234 and int(got.tokens[3]) in (7, 2000) and int(got.tokens[6]) == 17
            assert (got.logprobs[:2] == -inf).all() and (got.log_norm[:2] == -inf).all()
            assert int(got.tokens[4]) % 5 != 0 and int(got.tokens[8]) < 5
            torch.testing.assert_close(got.logprobs, ref.logprobs, atol=2.0 ** -18, rtol=2.0 ** -22)


def test_rows_apart_and_unaligned(cuda_device):
    """Rows that are views of a wider tensor and start on any element; the whole is not contiguous."""
    torch.manual_seed(2)
    for dtype in DTYPES.values():
        wide = torch.randn(6, 1037, device=cuda_device).to(dtype)
        for off, V in ((0, 1000), (1, 1000), (3, 777), (13, 1024), (5, 3)):
            _check(wide[:, off:off + V], torch.rand(6, device=cuda_device), *_settings(6, cuda_device, off))
        _check(wide.t()[:900], torch.rand(900, device=cuda_device), 0.8, 0, 0.9, 0.0)


def test_draws_follow_the_probabilities(cuda_device):
    """20000 evenly spaced numbers over one row: every token as often as its share, one more or less."""
    torch.manual_seed(5)
    n = 20000
    row = torch.randn(50, device=cuda_device) * 2
    u = (torch.arange(n, device=cuda_device) + 0.5) / n
    got = tdist.sample_tokens(row.expand(n, 50), u, 0.9, 20, 0.95, 0.01)
    ref = ref_sample_tokens(row.view(1, -1).expand(n, 50).contiguous(), u, 0.9, 20, 0.95, 0.01)
    assert torch.equal(got.tokens, ref.tokens)
    counts = torch.bincount(got.tokens.long(), minlength=50).double()
    share = torch.zeros(50, dtype=torch.float64, device=cuda_device)
    share[got.tokens.long()] = got.logprobs.double().exp()
    assert ((counts - share * n).abs() <= 1.01).all()


def test_a_row_alone_and_in_a_batch(cuda_device):
    """The same row, settings and number give the same bits on one CTA and on eight."""
    torch.manual_seed(6)
    logits = torch.randn(400, 50000, device=cuda_device)
    u = torch.rand(400, device=cuda_device)
    all_rows = tdist.sample_tokens(logits, u, 1.1, 0, 0.97, 0.001)
    for b in (0, 399):
        alone = tdist.sample_tokens(logits[b:b + 1], u[b:b + 1], 1.1, 0, 0.97, 0.001)
        assert all(torch.equal(x[b:b + 1], y) for x, y in zip(all_rows, alone))


def test_replays_from_a_graph(cuda_device):
    torch.manual_seed(7)
    logits, u = torch.randn(8, 30000, device=cuda_device), torch.rand(8, device=cuda_device)
    settings = _settings(8, cuda_device, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tdist.sample_tokens(logits, u, *settings)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = tdist.sample_tokens(logits, u, *settings)
    for _ in range(3):
        logits.normal_()
        u.uniform_()
        g.replay()
        assert torch.equal(out.tokens, ref_sample_tokens(logits, u, *settings).tokens)


def test_refusals(cuda_device):
    x, u = torch.zeros(2, 10, device=cuda_device), torch.zeros(2, device=cuda_device)
    with pytest.raises(ValueError):
        tdist.sample_tokens(x[0], u)
    with pytest.raises(ValueError):
        tdist.sample_tokens(x, u[:1])
    with pytest.raises(ValueError):
        tdist.sample_tokens(x, u.cpu())
    with pytest.raises(ValueError):
        tdist.sample_tokens(x[:, :0], u)
    with pytest.raises(TypeError):
        tdist.sample_tokens(x.double(), u)
    with pytest.raises(TypeError):
        tdist.sample_tokens(x, u.half())
    with pytest.raises(TypeError):
        tdist.sample_tokens(x, u, top_k=u)
    with pytest.raises(ValueError):
        tdist.sample_tokens(x, u, temperature=u[:1])
    with pytest.raises(_lib.TdistError):
        tdist.sample_tokens(torch.zeros(1, 1, device=cuda_device).expand(1, 600000).contiguous(), u[:1])
    assert tdist.sample_tokens(x[:0], u[:0]).tokens.shape == (0,)


@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (0, 0.5, 0.0), (5, 0.5, 0.1), (0, 1.0, 0.2)])
def test_a_temperature_that_is_no_number(cuda_device, k, p, m):
    """NaN among the rows' temperatures: the largest logit, whatever the filters, as for 0."""
    torch.manual_seed(8)
    logits, u = torch.randn(3, 9001, device=cuda_device), torch.rand(3, device=cuda_device)
    t = torch.tensor([float("nan"), 0.7, -1.0], device=cuda_device)
    got, ref = tdist.sample_tokens(logits, u, t, k, p, m), ref_sample_tokens(logits, u, t, k, p, m)
    check_status()
    assert torch.equal(got.tokens, ref.tokens)
    assert torch.equal(got.tokens[::2].long(), logits[::2].argmax(1))
    assert torch.equal(got.log_norm[::2], logits[::2].amax(1)) and got.logprobs[::2].tolist() == [0.0, 0.0]
    one = tdist.sample_tokens(logits, u, float("nan"), k, p, m)
    assert torch.equal(one.tokens.long(), logits.argmax(1))

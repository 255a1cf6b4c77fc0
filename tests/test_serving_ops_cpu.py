"""Windowed, prefill and shared-prefix attention and sampling on CPU tensors: the plain statements against loops in 64 bits, the
dispatcher's registrations, the checks of arguments, the example that runs them together."""
import importlib.util
import math
import os

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import triton_distributed_b200 as tdist
import triton_distributed_b200.torch_ops  # noqa: F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _loop(q, keys, values, scale, cap):
    """One query head over lists of key and value vectors, in Python floats."""
    if not keys:
        return [0.0] * q.shape[0]
    s = [float((q.double() * k.double()).sum()) * scale for k in keys]
    s = [cap * math.tanh(x / cap) if cap > 0 else x for x in s]
    m = max(s)
    p = [math.exp(x - m) for x in s]
    return [sum(w * float(v[d]) for w, v in zip(p, values)) / sum(p) for d in range(q.shape[0])]


@pytest.mark.parametrize("window,sinks,cap", [(None, 0, 0.0), (3, 0, 0.0), (1, 2, 5.0), (4, 9, 0.0)])
def test_window_statements(window, sinks, cap):
    torch.manual_seed(1)
    page, Hkv, G, D = 3, 2, 2, 4
    k, v = torch.randn(9, page, Hkv, D), torch.randn(9, page, Hkv, D)
    table = torch.tensor([[4, 0, 7], [8, 2, 1]], dtype=torch.int32)
    starts, lens = torch.tensor([0, 3, 8]), torch.tensor([9, 3])     # the second: two tokens before its first key
    q = torch.randn(8, Hkv * G, D)
    out = tdist.gqa_fwd_window_prefill(q, k, v, starts, lens, table, window=window, sinks=sinks, scale=0.7, soft_cap=cap)
    for b in range(2):
        n, kv = int(starts[b + 1] - starts[b]), int(lens[b])
        for i in range(n):
            p = kv - n + i
            seen = [j for j in range(kv) if j <= p and (window is None or j > p - window or j < sinks)]
            for h in range(Hkv * G):
                ref = _loop(q[int(starts[b]) + i, h], [k[table[b, j // page], j % page, h // G] for j in seen],
                            [v[table[b, j // page], j % page, h // G] for j in seen], 0.7, cap)
                torch.testing.assert_close(out[int(starts[b]) + i, h].double(), torch.tensor(ref, dtype=torch.float64), atol=1e-5, rtol=1e-5)
    last = torch.stack([q[2], q[7]])
    dec = tdist.gqa_fwd_window_decode(last, k, v, lens, table, window=window, sinks=sinks, scale=0.7, soft_cap=cap)
    torch.testing.assert_close(dec, torch.stack([out[2], out[7]]), atol=1e-5, rtol=1e-5)


def test_shared_prefix_statement():
    torch.manual_seed(2)
    page, Hkv, G, D = 4, 1, 3, 4
    k, v = torch.randn(8, page, Hkv, D), torch.randn(8, page, Hkv, D)
    pre, own, lens = torch.tensor([5, 2]), torch.tensor([[0], [1], [3]]), torch.tensor([3, 0, 4])
    q = torch.randn(3, G, D)
    for P in (0, 1, 7):
        out = tdist.gqa_fwd_shared_prefix_decode(q, k, v, P, pre, lens, own)
        for b in range(3):
            keys = [k[pre[j // page], j % page, 0] for j in range(P)] + [k[own[b, 0], j, 0] for j in range(int(lens[b]))]
            vals = [v[pre[j // page], j % page, 0] for j in range(P)] + [v[own[b, 0], j, 0] for j in range(int(lens[b]))]
            for h in range(G):
                torch.testing.assert_close(out[b, h].double(), torch.tensor(_loop(q[b, h], keys, vals, 0.5, 0.0), dtype=torch.float64), atol=1e-5, rtol=1e-5)


def _draw(row, u, t, k, p, m):
    """The definition of sampling in Python numbers, on one row."""
    x = [-math.inf if math.isnan(v) else v for v in row]
    top = max(x)
    if top == -math.inf:
        return -1
    if t <= 0:
        return x.index(top)
    w = [round(2.0 ** 31 * math.exp((v - top) / t)) if v > -math.inf else 0 for v in x]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if k > 0:
        order = order[:k]
    mass, kept, before = sum(w[i] for i in order), [], 0
    for i in order:
        if (p >= 1 or before < p * mass or not kept) and w[i] >= m * 2.0 ** 31:
            kept.append(i)
        before += w[i]
    target, total = math.floor(u * sum(w[i] for i in kept)), 0
    for i in sorted(kept):
        total += w[i]
        if total > target:
            return i


@pytest.mark.parametrize("t,k,p,m", [(1.0, 0, 1.0, 0.0), (0.5, 3, 1.0, 0.0), (1.5, 0, 0.6, 0.0), (1.0, 5, 0.8, 0.1), (0.0, 0, 1.0, 0.0), (2.0, 0, 0.0, 0.0)])
def test_sampling_statement(t, k, p, m):
    torch.manual_seed(3)
    rows = torch.randn(40, 12) * 2
    rows[0], rows[1, ::2], rows[2] = float("-inf"), float("nan"), 1.0   # nothing, some missing, all alike
    u = torch.rand(40)
    got = tdist.sample_tokens(rows, u, t, k, p, m)
    assert got.tokens.tolist() == [_draw(r.tolist(), float(x), t, k, p, m) for r, x in zip(rows, u)]
    assert float(got.logprobs[0]) == -math.inf and (got.logprobs[1:] <= 0).all()
    if k == 0 and p == 1.0 and m == 0.0 and t > 0:
        torch.testing.assert_close(got.log_norm[3:], torch.logsumexp(rows[3:] / t, 1), atol=1e-5, rtol=1e-5)


def test_settings_as_numbers_and_tensors():
    torch.manual_seed(4)
    x, u = torch.randn(6, 30), torch.rand(6)
    a = tdist.sample_tokens(x, u, 0.7, 9, 0.9, 0.02)
    b = tdist.sample_tokens(x, u, torch.full((6,), 0.7), torch.full((6,), 9), torch.full((6,), 0.9), torch.full((6,), 0.02))
    assert all(torch.equal(i, j) for i, j in zip(a, b))


def test_through_the_dispatcher():
    torch.manual_seed(5)
    k, v, q = torch.randn(6, 4, 2, 8), torch.randn(6, 4, 2, 8), torch.randn(2, 4, 8)
    table, lens = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32), torch.tensor([7, 5], dtype=torch.int32)
    pre, plen, starts = torch.tensor([4, 5], dtype=torch.int32), torch.tensor([6], dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32)
    ops = torch.ops.tdist
    torch.testing.assert_close(ops.gqa_fwd_window_decode(q, k, v, lens, table, 3, 1, 0.3, 0.0), tdist.gqa_fwd_window_decode(q, k, v, lens, table, 3, 1, 0.3))
    torch.testing.assert_close(ops.gqa_fwd_window_prefill(q, k, v, starts, lens, table, None, 0, 0.3, 2.0),
                               tdist.gqa_fwd_window_prefill(q, k, v, starts, lens, table, scale=0.3, soft_cap=2.0))
    torch.testing.assert_close(ops.gqa_fwd_shared_prefix_decode(q, k, v, plen, pre, lens, table, 0.3, 0.0),
                               tdist.gqa_fwd_shared_prefix_decode(q, k, v, plen, pre, lens, table, 0.3))
    x, u = torch.randn(2, 20), torch.rand(2)
    args = (torch.ones(2), torch.zeros(2, dtype=torch.int32), torch.ones(2), torch.zeros(2))
    assert torch.equal(ops.sample_tokens(x, u, *args)[0], tdist.sample_tokens(x, u).tokens)
    with FakeTensorMode():
        f = torch.empty
        out = ops.gqa_fwd_window_prefill(f(5, 4, 8), f(6, 4, 2, 8), f(6, 4, 2, 8), f(3, dtype=torch.int32), f(2, dtype=torch.int32),
                                         f(2, 2, dtype=torch.int32), 3, 0, 0.3, 0.0)
        assert out.shape == (5, 4, 8)
        assert ops.sample_tokens(f(3, 9), f(3), f(3), f(3, dtype=torch.int32), f(3), f(3))[0].dtype == torch.int32


def test_refusals():
    k, q = torch.zeros(6, 4, 2, 8), torch.zeros(2, 4, 8)
    table, lens, starts = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.arange(3)
    for bad in (dict(window=0), dict(window=-3), dict(sinks=-1), dict(soft_cap=-1.0), dict(soft_cap=float("nan"))):
        with pytest.raises(ValueError):
            tdist.gqa_fwd_window_prefill(q, k, k, starts, lens, table, **bad)
    with pytest.raises(ValueError):
        tdist.gqa_fwd_window_prefill(q, k, k, lens, lens, table)
    with pytest.raises(TypeError):
        tdist.gqa_fwd_window_decode(q, k, k, lens.float(), table)
    with pytest.raises(ValueError):
        tdist.gqa_fwd_window_decode(q, k, k[:5], lens, table)
    with pytest.raises(ValueError):
        tdist.gqa_fwd_window_decode(q[:, :3], k, k, lens, table)
    with pytest.raises(ValueError):
        tdist.gqa_fwd_shared_prefix_decode(q, k, k, torch.ones(2, dtype=torch.int32), table[0], lens, table)
    with pytest.raises(ValueError):
        tdist.sample_tokens(torch.zeros(2, 5), torch.zeros(3))
    with pytest.raises(TypeError):
        tdist.sample_tokens(torch.zeros(2, 5), torch.zeros(2), top_k=torch.zeros(2))
    with pytest.raises(TypeError):
        tdist.sample_tokens(torch.zeros(2, 5, dtype=torch.int32), torch.zeros(2))


def _example():
    spec = importlib.util.spec_from_file_location("shared_prompt_serving", os.path.join(ROOT, "examples", "shared_prompt_serving.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_the_example_on_cpu():
    drawn = _example().run(torch.device("cpu"), batch=3, prompt=64, steps=18)
    assert drawn.shape == (3, 18) and (drawn >= 0).all()


@pytest.mark.gpu
def test_the_example_on_a_gpu(cuda_device):
    from triton_distributed_b200.runtime import check_status
    drawn = _example().run(cuda_device)
    check_status()
    assert drawn.shape == (6, 20) and (drawn >= 0).all()


def test_a_temperature_that_is_no_number():
    torch.manual_seed(6)
    x, u = torch.randn(3, 30), torch.rand(3)
    got = tdist.sample_tokens(x, u, torch.tensor([math.nan, 0.0, math.nan]), 5, 0.9, 0.1)
    assert torch.equal(got.tokens.long(), x.argmax(1)) and torch.equal(got.log_norm, x.amax(1)) and not got.logprobs.any()

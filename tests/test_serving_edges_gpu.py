"""Serving operators where they can go wrong: calls interleaved on one stream, lengths and pages beyond the tensors."""
import pytest
import torch

import triton_distributed_b200 as tdist
from triton_distributed_b200.ops import paged_attention as PA
from triton_distributed_b200.runtime import check_status

pytestmark = pytest.mark.gpu


def _pool(pages, page, Hkv, D, dt, dev):
    return torch.randn(pages, page, Hkv, D, device=dev).to(dt), torch.randn(pages, page, Hkv, D, device=dev).to(dt)


def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def test_interleaved_shared_prefix_calls_on_one_stream(cuda_device, monkeypatch):
    """Two threads that call on one stream may launch prefix A, prefix B, own keys A, own keys B. Both own keys' launches use the stream's
    scratch, so the second must not begin before the first is done with it."""
    dev, page = cuda_device, 16
    torch.manual_seed(5)
    k, v = _pool(1200, page, 1, 128, torch.bfloat16, dev)
    calls = []
    for _ in range(2):
        order = torch.randperm(1200, device=dev).to(torch.int32)
        calls.append((torch.randn(1, 8, 128, device=dev).to(torch.bfloat16), k, v, _ints([700], dev), order[:44], _ints([16000], dev), order[44:1044].view(1, 1000)))
    want = [tdist.gqa_fwd_shared_prefix_decode(*c) for c in calls]
    torch.cuda.synchronize()
    attention, decode, kept, waiting = PA._run_attention, PA._run_decode, [], []

    def keep(*args):
        kept.append(args)   # each call's partials live until its own keys' launch, as in a thread of its own
        return attention(*args)

    monkeypatch.setattr(PA, "_run_attention", keep)
    monkeypatch.setattr(PA, "_run_decode", waiting.append)
    got = []
    for _ in range(100):
        got.append([tdist.gqa_fwd_shared_prefix_decode(*c) for c in calls])
        assert waiting[0].partial == waiting[1].partial and waiting[0].splits > 8   # one scratch, in global memory
        for a in waiting:
            decode(a)
        waiting.clear()
    check_status()
    for pair in got:
        assert all(torch.equal(a, b) for a, b in zip(pair, want))


@pytest.mark.parametrize("D,page", [(64, 16), (64, 1), (128, 16), (256, 64)])
@pytest.mark.parametrize("splits", [-1, 1, 16])
def test_lengths_beyond_the_table_are_cut(cuda_device, D, page, splits):
    """As many keys as the table has room for, whatever the length says; lengths below zero are none."""
    dev = cuda_device
    torch.manual_seed(D + page)
    room = 320 // page
    k, v = _pool(3 * room, page, 2, D, torch.bfloat16, dev)
    table = torch.randperm(3 * room, device=dev).view(3, room).to(torch.int32)
    q = torch.randn(3, 8, D, device=dev).to(torch.bfloat16)
    for window, sinks in ((None, 0), (100, 3)):
        args = dict(window=window, sinks=sinks, kv_split=splits)
        got = tdist.gqa_fwd_window_decode(q, k, v, _ints([321, 2 ** 31 - 1, -5], dev), table, **args)
        want = tdist.gqa_fwd_window_decode(q, k, v, _ints([320, 320, 0], dev), table, **args)
        check_status()
        assert torch.equal(got, want) and not got[2].any()
    pre = torch.randperm(3 * room, device=dev)[:room].to(torch.int32)
    got = tdist.gqa_fwd_shared_prefix_decode(q, k, v, 77, pre, _ints([1000, 320, -1], dev), table)
    want = tdist.gqa_fwd_shared_prefix_decode(q, k, v, 77, pre, _ints([320, 320, 0], dev), table)
    check_status()
    assert torch.equal(got, want)


@pytest.mark.parametrize("D,page", [(64, 16), (64, 1), (128, 16), (256, 64), (128, 3)])
@pytest.mark.parametrize("bad", [-1, 10 ** 9])
def test_pages_that_the_cache_does_not_have_read_as_zeros(cuda_device, D, page, bad):
    dev = cuda_device
    torch.manual_seed(D + page)
    room = -(-320 // page)
    k, v = _pool(2 * room + 1, page, 2, D, torch.bfloat16, dev)
    k[-1], v[-1] = 0, 0
    order = torch.randperm(2 * room, device=dev).view(2, room).to(torch.int32)
    wrong, zeros = order.clone(), order.clone()
    for i in (0, room // 2, room - 1):
        wrong[0, i], zeros[0, i] = bad, 2 * room
    q = torch.randn(2, 8, D, device=dev).to(torch.bfloat16)
    lens = _ints([315, 320], dev)
    for window, sinks in ((None, 0), (200, 3)):
        for splits in (-1, 1, 16):
            a, b = (tdist.gqa_fwd_window_decode(q, k, v, lens, t, window=window, sinks=sinks, kv_split=splits) for t in (wrong, zeros))
            check_status()
            assert torch.equal(a, b)
        a, b = (tdist.gqa_fwd_window_prefill(q, k, v, _ints([0, 1, 2], dev), lens, t, window=window, sinks=sinks) for t in (wrong, zeros))
        check_status()
        assert torch.equal(a, b)

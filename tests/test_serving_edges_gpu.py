"""Serving operators where they can go wrong: calls interleaved on one stream."""
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

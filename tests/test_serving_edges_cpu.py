"""What the serving operators refuse before any launch, and their CPU statements on infinities, NaN and empty batches."""
import ctypes as C
import math

import pytest
import torch

import triton_distributed_b200 as tdist
from triton_distributed_b200 import _lib


def _decode_args(**changed):
    """A call that nothing is wrong with but ``changed``. The addresses are numbers: nothing may come of the call but its refusal."""
    a = _lib.DecodeArgs()
    base = 1 << 20
    a.q, a.k_cache, a.v_cache, a.block_table, a.kv_lens, a.partial, a.counters, a.out = (base * (i + 1) for i in range(8))
    a.B, a.Hq, a.Hkv, a.head_dim, a.page_size, a.max_blocks, a.splits, a.world = 2, 8, 2, 128, 16, 4, 1, 1
    a.stride_block, a.stride_token, a.stride_head, a.scale, a.dtype = 16 * 256, 256, 128, 1.0, _lib.DT_BF16
    for name, value in changed.items():
        setattr(a, name, value)
    return a


WINDOW = dict(window=64, sinks=4, blocks=9)


@pytest.mark.parametrize("ext", [{}, WINDOW])
@pytest.mark.parametrize("field,address", [("k_cache", (2 << 20) + 8), ("v_cache", (3 << 20) + 8), ("k_cache", (2 << 20) + 2), ("q", (1 << 20) + 2),
                                           ("out", (8 << 20) + 4), ("partial", (6 << 20) + 4)])
def test_decode_refuses_misaligned_addresses(ext, field, address):
    """Every copy and store of the kernel needs its width's alignment; a slice of a cache has it in its strides but not in its base."""
    code = _lib.lib().tdist_flash_decode(C.byref(_decode_args(**ext, **{field: address})))
    assert code != 0 and b"aligned" in _lib.lib().tdist_last_error()


def test_decode_refuses_misaligned_earlier_partials():
    a = _decode_args(**WINDOW, priors=2, prior_o=(9 << 20) + 4, prior_lse=10 << 20)
    code = _lib.lib().tdist_flash_decode(C.byref(a))
    assert code != 0 and b"aligned" in _lib.lib().tdist_last_error()


def test_windowed_decode_needs_the_number_of_pages():
    code = _lib.lib().tdist_flash_decode(C.byref(_decode_args(window=64, sinks=4, blocks=0)))
    assert code != 0 and b"blocks" in _lib.lib().tdist_last_error()


@pytest.mark.parametrize("tokens", [4, 10])   # 10: the first two lie before the first key
def test_what_is_no_number_shows_beside_rows_that_see_nothing(tokens):
    torch.manual_seed(1)
    k, v, q = torch.randn(4, 4, 1, 8), torch.randn(4, 4, 1, 8), torch.randn(tokens, 2, 8)
    k[1, 1] = math.nan   # key 5 of 8: the last three queries see it
    out = tdist.gqa_fwd_window_prefill(q, k, v, torch.tensor([0, tokens]), torch.tensor([8]), torch.arange(4).view(1, 4))
    assert out[-3:].isnan().all() and not out[:-3].isnan().any()
    assert not out[:-8].any()


def test_a_query_whose_scores_are_all_minus_infinity_gives_zeros():
    k, v, q = torch.zeros(1, 4, 1, 8), torch.randn(1, 4, 1, 8), torch.ones(1, 2, 8)
    k[..., 0] = -math.inf
    assert not tdist.gqa_fwd_window_decode(q, k, v, torch.tensor([3]), torch.zeros(1, 1, dtype=torch.int32)).any()


def test_results_go_into_a_given_tensor_on_the_cpu_too():
    torch.manual_seed(2)
    k, v, q = torch.randn(6, 4, 2, 8), torch.randn(6, 4, 2, 8), torch.randn(2, 4, 8)
    table, lens, pre = torch.tensor([[0, 1], [2, 3]]), torch.tensor([7, 5]), torch.tensor([4, 5])
    for call in (lambda **o: tdist.gqa_fwd_window_decode(q, k, v, lens, table, window=3, **o),
                 lambda **o: tdist.gqa_fwd_window_prefill(q, k, v, torch.arange(3), lens, table, **o),
                 lambda **o: tdist.gqa_fwd_shared_prefix_decode(q, k, v, 6, pre, lens, table, **o)):
        out = torch.full_like(q, math.nan)
        assert call(out=out) is out and torch.equal(out, call())
        with pytest.raises(ValueError):
            call(out=torch.empty(2, 4, 9))


@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (0, 0.5, 0.0), (700, 0.9, 0.0), (0, 0.3, 0.5)])
def test_an_infinite_temperature_draws_evenly_from_what_is_there(k, p, m):
    torch.manual_seed(3)
    x = torch.randn(9, 1001)
    x[:, ::2] = -math.inf      # 500 of 1001 are left
    x[:, 5::10] = math.nan     # and 400 of these
    got = tdist.sample_tokens(x, torch.linspace(0, 0.999, 9), math.inf, k, p, m)
    kept = math.ceil(float(torch.tensor(p)) * 400)   # top_p is fp32; top_k lets all 400 through
    assert x.gather(1, got.tokens.long().view(-1, 1)).isfinite().all()
    torch.testing.assert_close(got.logprobs, torch.full((9,), -math.log(kept)), atol=1e-6, rtol=1e-6)
    order = torch.sort(x.nan_to_num(nan=-math.inf, neginf=-math.inf), dim=1, descending=True, stable=True).indices[:, :kept].sort(1).values
    at = torch.floor(torch.linspace(0, 0.999, 9).double() * kept * 2.0 ** 31).div(2.0 ** 31).floor().long()
    assert torch.equal(got.tokens.long(), order.gather(1, at.view(-1, 1)).view(-1))


@pytest.mark.parametrize("p", [1.0, 0.5])
def test_infinite_logits_at_an_infinite_temperature(p):
    """They weigh alike and the finite ones nothing, as at any temperature."""
    x = torch.randn(4, 31)
    x[:, 3::9] = math.inf   # 3, 12, 21, 30
    u = torch.tensor([0.0, 0.3, 0.6, 0.99])
    for t in (1.0, math.inf):
        got = tdist.sample_tokens(x, u, t, top_p=p)
        assert got.tokens.tolist() == ([3, 12, 21, 30] if p == 1.0 else [3, 3, 12, 12])
        torch.testing.assert_close(got.logprobs, torch.full((4,), -math.log(4 * p)))

"""GPU: prompt attention where the softmax has no value."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,m", [(5, 5), (64, 64), (300, 300), (1000, 1000), (3, 2000), (130, 9000)])
def test_logits_of_minus_infinity(dtype, n, m):
    """A row all of whose logits are -inf is NaN wherever its keys lie, one that sees no key zeros, and one finite logit has all of the weight."""
    from tq_local_b200.runtime.prompt_attention import prompt_attention

    gen = torch.Generator(device="cuda").manual_seed(n)
    q, k, v = (torch.randn(3, h, s, 128, device="cuda", generator=gen).to(dtype) for h, s in ((4, n), (2, m), (2, m)))
    q[..., 0] = 1
    k[..., 0] = -math.inf
    starts = torch.tensor([0, m, m - n + n // 2], dtype=torch.int32, device="cuda")
    for causal in (True, False):
        out = prompt_attention(q, k, v, causal=causal)
        assert out.isnan().all()
        out = prompt_attention(q, k, v, causal=causal, seq_start=starts)
        empty = n // 2 if causal else 0
        assert out[0].isnan().all() and (out[1] == 0).all() and (out[2, :, :empty] == 0).all() and out[2, :, empty:].isnan().all()
    for at in {0, m - n, m - n + n // 3, m - 1}:
        one = k.clone()
        one[:, :, at, 0] = 0
        out = prompt_attention(q, one, v)
        before = max(0, at - (m - n))
        assert out[:, :, :before].isnan().all()
        want = v[:, :, at].repeat_interleave(2, 1).unsqueeze(2).expand(3, 4, n - before, 128).double()
        # (the weight 1 and the sum 1 are exact, others are 0 or 2^-125)
        assert ((out[:, :, before:].double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -25).all()


def test_the_status_waits_for_every_stream():
    """What a kernel on a stream of its own reports is not missed."""
    from tq_local_b200.runtime.prompt_attention import prompt_attention, raise_on_status

    q = torch.zeros(1, 2, 8, 128, device="cuda", dtype=BF16)
    prompt_attention(q, q, q)  # (loads the kernel)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)  # some 50 ms
        prompt_attention(q, q, q)
    assert not side.query()
    raise_on_status(q.device, "test")
    assert side.query()


def test_the_status_can_be_cleared():
    import ctypes as C

    from tq_local_b200.runtime import ffi

    word = C.c_int32(-1)
    assert ffi.lib().tq_prompt_status_clear() == 0
    assert ffi.lib().tq_prompt_status(C.byref(word)) == 0 and word.value == 0

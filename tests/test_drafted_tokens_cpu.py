"""CPU: what the entry points of prompt attention, drafted tokens and cache moves refuse before anything is launched."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

OK, ARG, UNSUPPORTED = 0, -1, -2


def lib():
    from tq_local_b200.runtime import ffi

    return ffi.lib()


def desc(data=4096, dtype=1, b=8 * 128, h=128, t=128):
    from tq_local_b200.runtime.ffi import DenseDesc

    return C.byref(DenseDesc(data, dtype, b, h, t))


def test_prompt_kernels_replace_sdpa_alone():
    """Another implementation may add terms that neither the kernels nor their fall-back compute."""
    from types import SimpleNamespace

    from tq_local_b200.runtime.generation import _prompt_kernels

    ids = torch.zeros(2, 4, dtype=torch.long)
    inside = lambda mask=None, enabled=True, **config: _inside(_prompt_kernels, SimpleNamespace(config=SimpleNamespace(**config)),
                                                                {"input_ids": ids, "attention_mask": mask}, enabled)
    assert inside(_attn_implementation="sdpa") == ("turboquant_prompt", "sdpa")
    assert inside(_attn_implementation="sdpa", enabled=False) == ("sdpa", "sdpa")
    assert inside(_attn_implementation="eager") == ("eager", "eager")
    assert inside(_attn_implementation="sdpa", attention_chunk_size=8192) == ("sdpa", "sdpa")
    assert inside(torch.tensor([[0, 0, 1, 1], [1, 1, 1, 1]]), _attn_implementation="sdpa") == ("turboquant_prompt", "sdpa")
    assert inside(torch.tensor([[1, 0, 1, 1], [1, 1, 1, 1]]), _attn_implementation="sdpa") == ("sdpa", "sdpa")


def _inside(manager, model, inputs, enabled):
    with manager(model, inputs, enabled):
        seen = model.config._attn_implementation
    return seen, model.config._attn_implementation


def test_prompt_refuses_bad_arguments():
    d = desc()
    call = lambda q=d, k=d, v=d, b=1, hq=4, hkv=2, n=8, m=8, start=None, out=d, ws=None, size=0, causal=1: lib().tq_prompt_attn(
        q, k, v, b, hq, hkv, n, m, start, 0.1, causal, ws, size, out, None)
    assert call(q=None) == ARG and call(out=None) == ARG and call(k=desc(data=None)) == ARG
    assert call(q=desc(dtype=0)) == UNSUPPORTED and call(q=desc(dtype=9)) == ARG and call(k=desc(dtype=2)) == ARG
    assert call(q=desc(data=4098)) == ARG and call(v=desc(t=129)) == ARG and call(out=desc(h=4)) == ARG
    assert call(hq=3) == ARG and call(hkv=0) == ARG and call(n=9) == ARG and call(b=-1) == ARG and call(n=-1) == ARG
    assert call(hq=65, hkv=1) == UNSUPPORTED and call(start=2) == ARG
    assert call(b=0) == OK and call(n=0) == OK  # nothing to do, nothing launched
    packed = lambda cu=4096, n=1, total=8, most=8: lib().tq_prompt_attn_packed(d, d, d, n, total, 4, 2, cu, most, 0.1, 1, None, 0, d, None)
    assert packed(cu=None) == ARG and packed(cu=4098) == ARG and packed(total=-1) == ARG and packed(most=-1) == ARG
    assert packed(n=0) == OK and packed(most=0) == OK
    assert lib().tq_prompt_status(None) == ARG


def test_calls_without_a_context_are_refused():
    from tq_local_b200.runtime.ffi import CacheDesc

    cache = C.byref(CacheDesc())
    assert lib().tq_tree_attn(None, desc(), 4, 1, cache, 0, None, None, None, 0, desc(), None) == ARG
    assert lib().tq_cache_keep_tokens(None, cache, 0, 4096, 1, 4096, 4096, 8192, None) == ARG
    assert lib().tq_cache_select_rows(None, cache, cache, 4096, 0, 0, None, None) == ARG


def test_prompt_attention_takes_cuda_tensors_only():
    from tq_local_b200.runtime.ffi import TQError
    from tq_local_b200.runtime.prompt_attention import prompt_attention, prompt_attention_packed

    x = torch.zeros(1, 2, 4, 128, dtype=torch.float16)
    with pytest.raises(TQError):
        prompt_attention(x, x, x)
    with pytest.raises(TQError):
        prompt_attention_packed(x[0], x[0], x[0], torch.zeros(2, dtype=torch.int32), 1)
    with pytest.raises(ValueError):
        prompt_attention(x, x[:, :0], x[:, :0])


def test_rows_that_kernels_cannot_address_are_copied():
    from tq_local_b200.runtime.codec import aligned_view, strided_desc

    x = torch.zeros(2, 3, 4, 256, dtype=torch.float16)
    whole = x[..., :128]
    assert aligned_view(whole) is whole
    for t in (x[..., ::2], x[..., 1:129], x[:, :1, :, :128].expand(2, 3, 4, 128), torch.zeros(2, 3, 4, 129, dtype=torch.float16)[..., :128]):
        assert aligned_view(t) is not t and aligned_view(t).stride() == (3 * 4 * 128, 4 * 128, 128, 1)
    odd = torch.zeros(5, 129, dtype=torch.float16)[:1, :128].view(1, 1, 1, 128)  # one row: its stride is nobody's business
    assert aligned_view(odd) is odd
    d = strided_desc(odd)
    assert (d.stride_b, d.stride_h, d.stride_t) == (0, 0, 0)


def test_operands_are_aligned_views_with_their_strides():
    from tq_local_b200.runtime.codec import aligned_view, operand, strided_desc

    x = torch.zeros(2, 3, 4, 256, dtype=torch.bfloat16)
    for t in (x[..., :128], x[..., ::2], x[..., 1:129], x[:, :1, :, :128].expand(2, 3, 4, 128), x[:1, :, :1, :128], x[..., :128].transpose(1, 2),
              torch.zeros(2, 3, 4, 129, dtype=torch.float16)[..., :128], torch.zeros(5, 129, dtype=torch.float16)[:1, :128].view(1, 1, 1, 128)):
        view, d = operand(t)
        same = aligned_view(t)
        assert (view is t) == (same is t) and view.stride() == same.stride()
        want = strided_desc(view)
        assert [getattr(d, name) for name, _ in d._fields_] == [getattr(want, name) for name, _ in d._fields_]


def test_dense_rows_follow_an_index():
    from tq_local_b200.runtime.packed_qmse_cache import _GrowingDense

    dense = _GrowingDense()
    dense.take_rows(torch.tensor([0]))
    assert dense.buf is None
    x = torch.arange(6.0).view(3, 1, 2, 1)
    dense.append(x)
    dense.take_rows(torch.tensor([2, 0, 0, 1]))
    assert torch.equal(dense.view(), x[[2, 0, 0, 1]])

"""CPU: prompt attention's host side - what the C entry points take, and where the HF backend sends what the kernels do not compute."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

OK, ARG = 0, -1


def desc(b=1024, h=128, t=128):
    from tq_local_b200.runtime.ffi import DenseDesc

    return C.byref(DenseDesc(4096, 1, b, h, t))


def test_strides_of_axes_with_one_element_are_not_looked_at():
    """No query or no sequence: strides are checked, nothing is launched."""
    from tq_local_b200.runtime import ffi

    plain = desc()
    call = lambda q=plain, k=plain, v=plain, out=plain, b=1, hq=1, hkv=1, n=0, m=1: ffi.lib().tq_prompt_attn(
        q, k, v, b, hq, hkv, n, m, None, 0.1, 1, None, 0, out, None)
    assert call() == OK
    for odd in (desc(b=3), desc(h=5), desc(t=7), desc(3, 5, 7)):
        for name in ("q", "k", "v", "out"):
            assert call(**{name: odd}) == OK
    for many, odd in ((dict(b=2), desc(b=3)), (dict(hq=2, hkv=2), desc(h=5)), (dict(m=2), desc(t=7))):
        for name in ("k", "v") if "m" in many else ("q", "k", "v", "out"):
            assert call(**many, **{name: odd}) == ARG
    assert call(hq=2, k=desc(h=5)) == OK and call(hq=2, q=desc(h=5)) == ARG
    packed = lambda d, n=0, total=8, h=2: ffi.lib().tq_prompt_attn_packed(d, d, d, n, total, h, h, 4096, 8, 0.1, 1, None, 0, d, None)
    assert packed(desc(b=3)) == OK and packed(desc(h=5)) == ARG and packed(desc(t=7)) == ARG
    assert packed(desc(h=5), h=1) == OK and packed(desc(t=7), total=1) == OK


def test_what_the_backend_takes():
    """Everything that a call of the kernels would refuse goes to the model's own attention instead, the values' type, size and gradient among it."""
    from types import SimpleNamespace

    from tq_local_b200.runtime.prompt_attention import _takes

    def tensor(*shape, dtype=torch.bfloat16, device="cuda", grad=False):
        return SimpleNamespace(shape=torch.Size(shape), dtype=dtype, device=torch.device(device), requires_grad=grad)

    q, kv = tensor(2, 8, 30, 128), tensor(2, 2, 30, 128)
    takes = lambda q=q, k=kv, v=kv, mask=None, causal=True, dropout=0.0, **kw: _takes(q, k, v, mask, causal, dropout, kw)
    with torch.enable_grad():
        assert takes() and takes(q=tensor(2, 8, 3, 128)) and takes(sliding_window=None)
        for name, shape in (("q", (2, 8, 30, 128)), ("k", (2, 2, 30, 128)), ("v", (2, 2, 30, 128))):
            assert not takes(**{name: tensor(*shape, grad=True)}) and not takes(**{name: tensor(*shape, dtype=torch.float16)})
            with torch.no_grad():
                assert takes(**{name: tensor(*shape, grad=True)})
    assert not takes(v=tensor(2, 2, 30, 64)) and not takes(k=tensor(2, 2, 30, 64)) and not takes(q=tensor(2, 8, 31, 128))
    assert not takes(causal=False) and not takes(dropout=0.1) and not takes(sliding_window=4096) and not takes(softcap=30.0)
    assert not takes(q=tensor(2, 8, 30, 128, device="cpu")) and not takes(q=tensor(2, 130, 30, 128))


def test_what_the_kernels_do_not_compute_is_the_models_own_attention():
    """Not causal, a mask, dropout: as ``sdpa`` computes it."""
    from types import SimpleNamespace

    import torch.nn.functional as F

    from tq_local_b200.runtime.prompt_attention import turboquant_prompt_forward

    gen = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, h, 9, 16, generator=gen) for h in (4, 2, 2))
    plain = lambda **kw: F.scaled_dot_product_attention(q, k.repeat_interleave(2, 1), v.repeat_interleave(2, 1), **kw).transpose(1, 2)
    module = lambda causal: SimpleNamespace(is_causal=causal, num_key_value_groups=2, training=False)
    for causal in (False, True):
        out, weights = turboquant_prompt_forward(module(causal), q, k, v, None, scaling=0.3)
        assert weights is None
        torch.testing.assert_close(out, plain(is_causal=causal, scale=0.3))
        torch.testing.assert_close(turboquant_prompt_forward(module(not causal), q, k, v, None, is_causal=causal)[0], plain(is_causal=causal))
    mask = torch.rand(2, 1, 9, 9, generator=gen) < 0.7
    mask[..., 0] = True
    torch.testing.assert_close(turboquant_prompt_forward(module(True), q, k, v, mask)[0], plain(attn_mask=mask))
    assert (turboquant_prompt_forward(module(False), q, k, v, None, dropout=1.0)[0] == 0).all()


@pytest.mark.parametrize("before", [None, "sdpa"])
@pytest.mark.parametrize("fails", [False, True])
def test_a_models_implementation_is_put_back_as_it_was(before, fails):
    from types import SimpleNamespace

    from transformers import LlamaConfig

    from tq_local_b200.runtime.generation import _prompt_kernels

    model = SimpleNamespace(config=LlamaConfig(hidden_size=256, num_attention_heads=2, num_hidden_layers=1))
    model.config._attn_implementation = before
    try:
        with _prompt_kernels(model, {"input_ids": torch.zeros(1, 4, dtype=torch.long)}, True):
            assert model.config._attn_implementation == "turboquant_prompt"
            if fails:
                raise KeyError
    except KeyError:
        assert fails
    assert model.config._attn_implementation == before


def test_a_lost_wait_is_reported_once(monkeypatch):
    """The device's word stays until it is cleared, so that it must be once it has been reported: later calls are not at fault."""
    from contextlib import nullcontext
    from types import SimpleNamespace

    from tq_local_b200.runtime import ffi, prompt_attention

    word = {"now": 0}

    def status(out):
        out._obj.value = word["now"]
        return 0

    def clear():
        word["now"] = 0
        return 0

    monkeypatch.setattr(ffi, "lib", lambda: SimpleNamespace(tq_prompt_status=status, tq_prompt_status_clear=clear))
    monkeypatch.setattr(torch.cuda, "device", lambda device: nullcontext())
    prompt_attention.raise_on_status("cuda:0", "here")
    for lost in (1, 2):
        word["now"] = lost
        with pytest.raises(ffi.TQError, match=f"here.*status {lost}"):
            prompt_attention.raise_on_status("cuda:0", "here")
        prompt_attention.raise_on_status("cuda:0", "here")

"""GPU: prompt attention against softmax attention in 64 bits.

Tolerances.  u = eps / 2 is the largest relative error of one rounding to the tensors' type.  A weight is rounded once to
that type before it meets the values, its exponential is good to u / 4, and the sum of the weights carries the same
errors once more at most; the logits are exact products summed in fp32, whose error (128 terms of 2^-24 of the sum of their magnitudes)
moves a weight by 2^-17 of that sum at most.  With A = sum_j p_ij |v_j| an output is thus off by at most (2.5 u + 2^-16 L) A for the products'
sum L of a row, then rounded once: u |out|.  fp16 keeps nothing below 2^-25."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def reference(q, k, v, starts=None, causal=True, scale=None):
    """[B, H, S, 128] in 64 bits -> (out, what it may be off by)."""
    u = torch.finfo(q.dtype).eps / 2
    scale = 128 ** -0.5 if scale is None else scale
    g, n, m = q.shape[1] // k.shape[1], q.shape[2], k.shape[2]
    q64, k64, v64 = q.double(), k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    i, j = torch.arange(n, device=q.device)[:, None], torch.arange(m, device=q.device)[None, :]
    seen = torch.ones(n, m, dtype=torch.bool, device=q.device) if not causal else j <= i + m - n
    seen = seen.expand(q.shape[0], 1, n, m)
    if starts is not None:
        seen = seen & (j >= starts.clamp(min=0).view(-1, 1, 1, 1))
    k64, v64 = k64.masked_fill(~seen.any(2).unsqueeze(-1), 0.0), v64.masked_fill(~seen.any(2).unsqueeze(-1), 0.0)
    s = (q64 @ k64.mT * scale).masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    out = p @ v64
    reach = (q64.abs() @ k64.abs().mT * abs(scale)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    return out, (2.5 * u + 2.0 ** -16 * reach) * (p @ v64.abs()) + u * out.abs() + 2.0 ** -25


def check(got, want, tol):
    bad = (got.double() - want).abs() > tol
    assert not bad.any() and got.isfinite().all(), f"{int(bad.sum())} outputs off, by up to {float(((got.double() - want).abs() / tol).max()):.3g} x"


def make(b, hq, hkv, n, m, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = lambda h, s: torch.randn(b, s, h, 128, device="cuda", generator=gen).to(dtype).transpose(1, 2)
    return t(hq, n), t(hkv, m), t(hkv, m)


@pytest.mark.parametrize("n,m", [(1, 1), (2, 2), (31, 31), (33, 33), (63, 64), (127, 127), (128, 128), (129, 129), (255, 255), (257, 257),
                                 (513, 513), (1, 700), (5, 133), (64, 1000), (100, 129), (1000, 1001)])
@pytest.mark.parametrize("hq,hkv,dtype", [(4, 1, BF16), (7, 1, F16), (2, 2, F16), (16, 2, BF16)])
def test_causal(n, m, hq, hkv, dtype):
    from tq_local_b200.runtime.prompt_attention import prompt_attention

    q, k, v = make(2, hq, hkv, n, m, dtype, n + m)
    out = prompt_attention(q, k, v)
    assert out.shape == q.shape and out.dtype == dtype and out.transpose(1, 2).is_contiguous()
    check(out, *reference(q, k, v))


@pytest.mark.parametrize("group", [1, 3, 5, 6, 12, 33, 64])
def test_group_sizes(group):
    from tq_local_b200.runtime.prompt_attention import prompt_attention

    q, k, v = make(1, 2 * group, 2, 150, 150, BF16, group)
    check(prompt_attention(q, k, v), *reference(q, k, v))


@pytest.mark.parametrize("n,m", [(40, 40), (300, 300), (3, 500), (300, 120), (1, 1)])
def test_without_causal_mask(n, m):
    from tq_local_b200.runtime.prompt_attention import prompt_attention

    q, k, v = make(2, 8, 2, n, m, F16, 1)
    starts = torch.tensor([0, m // 2], dtype=torch.int32, device="cuda")
    check(prompt_attention(q, k, v, causal=False), *reference(q, k, v, causal=False))
    check(prompt_attention(q, k, v, causal=False, seq_start=starts), *reference(q, k, v, starts, causal=False))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,n,m", [(8, 2, 400, 400), (14, 2, 130, 130), (4, 4, 50, 300)])
def test_left_padding_hides_what_it_covers(dtype, hq, hkv, n, m):
    from tq_local_b200.runtime.prompt_attention import prompt_attention

    starts = torch.tensor([0, 1, 37, 128, m - 1, m, m + 5, -3], dtype=torch.int32, device="cuda")
    q, k, v = make(len(starts), hq, hkv, n, m, dtype, 3)
    want, tol = reference(q, k, v, starts)
    junk = [math.nan, math.inf, -math.inf, torch.finfo(dtype).min, torch.finfo(dtype).max]
    for b, s in enumerate(starts.clamp(0, m).tolist()):  # the padding holds anything
        for x in (k, v):
            x[b, :, :s] = torch.tensor([junk[i % 5] for i in range(s)], device="cuda").to(dtype).view(1, s, 1) if s else x[b, :, :s]
    out = prompt_attention(q, k, v, seq_start=starts)
    check(out, want, tol)
    for b, s in enumerate(starts.tolist()):
        empty = max(0, min(s - (m - n), n))
        assert (out[b, :, :empty] == 0).all()


def test_scales_and_large_logits():
    from tq_local_b200.runtime.prompt_attention import prompt_attention

    q, k, v = make(1, 4, 2, 300, 300, BF16, 5)
    for scale in (0.0, -0.05, 0.02, 1.0):
        check(prompt_attention(q, k, v, scale=scale), *reference(q, k, v, scale=scale))
    # keys that grow: the running maximum moves by hundreds from tile to tile, and back
    grow = torch.linspace(0.1, 30.0, 300, device="cuda").view(1, 1, 300, 1)
    for ramp in (grow, grow.flip(2)):
        kk = (k.float() * ramp).to(BF16)
        check(prompt_attention(q, kk, v), *reference(q, kk, v))


def test_equal_logits_average_the_values():
    from tq_local_b200.runtime.prompt_attention import prompt_attention

    q, k, v = make(1, 4, 1, 700, 700, F16, 6)
    q.zero_()
    check(prompt_attention(q, k, v), *reference(q, k, v))


def test_strides_and_orders():
    """[B, S, H, D] and [B, H, S, D] memory, a slice of fused projections, unaligned rows, expanded heads, a given output."""
    from tq_local_b200.runtime.prompt_attention import prompt_attention

    b, n = 2, 200
    fused = torch.randn(b, n, 8 + 2 * 2, 128, device="cuda").to(BF16)
    q, k, v = (t.transpose(1, 2) for t in fused.split((8, 2, 2), dim=2))
    want, tol = reference(q, k, v)
    check(prompt_attention(q, k, v), want, tol)
    check(prompt_attention(q.contiguous(), k.contiguous(), v.contiguous()), want, tol)
    odd = torch.empty(b, 8, n, 131, dtype=BF16, device="cuda")[..., 1:129].copy_(q)
    check(prompt_attention(odd, k, v), want, tol)
    wide = torch.empty(b, 8, n, 256, dtype=BF16, device="cuda")[..., ::2].copy_(q)
    check(prompt_attention(wide, k, v), want, tol)
    out = torch.empty(b, 8, n, 136, dtype=BF16, device="cuda")[..., 8:]
    assert prompt_attention(q, k, v, out=out) is out
    check(out, want, tol)
    one = k[:, :1].expand(b, 2, n, 128)  # one head for all: a stride of 0
    check(prompt_attention(q, one, v), *reference(q, one, v))


@pytest.mark.parametrize("hq,hkv,dtype", [(8, 2, BF16), (7, 1, F16), (2, 2, BF16)])
def test_packed_sequences(hq, hkv, dtype):
    from tq_local_b200.runtime.prompt_attention import prompt_attention_packed

    lens = [1, 0, 130, 77, 0, 256, 3, 500, 64, 1]
    cu = torch.tensor([0] + [sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32, device="cuda")
    total = sum(lens) + 9
    q, k, v = (t[0].transpose(0, 1) for t in make(1, hq, hkv, total, total, dtype, 7))
    k[sum(lens):], v[sum(lens):] = math.nan, math.inf  # what lies behind the last sequence
    for causal in (True, False):
        out = torch.full_like(q, 7.0)
        assert prompt_attention_packed(q, k, v, cu, 500, causal=causal, out=out) is out
        for s, n in zip(cu.tolist(), lens):
            if n:
                part = [t[s:s + n].transpose(0, 1).unsqueeze(0) for t in (q, k, v, out)]
                check(part[3], *reference(*part[:3], causal=causal))
        assert (out[sum(lens):] == 7.0).all()  # rows behind the last sequence
    # a sequence's neighbours hold anything
    mine = prompt_attention_packed(q, k, v, cu, 500)[131:131 + 77]
    k[:131], v[:131], k[208:], v[208:] = math.nan, math.inf, -math.inf, math.nan
    assert torch.equal(prompt_attention_packed(q, k, v, cu, 500)[131:131 + 77], mine)


def test_sequence_bounds_outside_the_tensor_are_cut():
    from tq_local_b200.runtime.prompt_attention import prompt_attention_packed

    q, k, v = (t[0].transpose(0, 1) for t in make(1, 4, 2, 300, 300, BF16, 4))
    room = torch.full((400, 4, 128), 7.0, dtype=BF16, device="cuda")
    out = room[:300]
    cu = torch.tensor([-50, 100, 90, 250, 1000], dtype=torch.int32, device="cuda")  # [0, 100), nothing, [90, 250), [250, 300)
    prompt_attention_packed(q, k, v, cu, 300, out=out)
    for lo, hi in ((0, 90), (250, 300)):  # (what two sequences share is either's)
        part = [t[(0 if lo == 0 else lo):hi].transpose(0, 1).unsqueeze(0) for t in (q, k, v, out)]
        check(part[3], *reference(*part[:3]))
    assert (room[300:] == 7.0).all()


def test_many_short_sequences():
    from tq_local_b200.runtime.prompt_attention import prompt_attention_packed

    lens = [1 + i % 5 for i in range(400)]
    cu = torch.tensor([0] + [sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32, device="cuda")
    q, k, v = (t[0].transpose(0, 1) for t in make(1, 4, 2, sum(lens), sum(lens), BF16, 8))
    out = prompt_attention_packed(q, k, v, cu, max(lens))
    for s, n in list(zip(cu.tolist(), lens))[::37]:
        part = [t[s:s + n].transpose(0, 1).unsqueeze(0) for t in (q, k, v, out)]
        check(part[3], *reference(*part[:3]))


def test_long_keys_few_queries_and_equal_runs():
    from tq_local_b200.runtime.prompt_attention import prompt_attention

    for hq, hkv, n, m in ((8, 2, 3, 20011), (4, 1, 70, 9001), (2, 2, 1, 40000)):
        q, k, v = make(1, hq, hkv, n, m, F16, m)
        starts = torch.tensor([m // 3], dtype=torch.int32, device="cuda")
        for s in (None, starts):
            out = prompt_attention(q, k, v, seq_start=s)
            check(out, *reference(q, k, v, s))
            assert torch.equal(out, prompt_attention(q, k, v, seq_start=s))


def test_many_tiles():
    """More tiles than SMs, again and again."""
    from tq_local_b200.runtime.prompt_attention import prompt_attention, raise_on_status

    for b, hq, hkv, n in ((1, 8, 8, 4000), (6, 16, 4, 700), (60, 4, 1, 130)):
        q, k, v = make(b, hq, hkv, n, n, BF16, n)
        for _ in range(30):
            out = prompt_attention(q, k, v)
        check(out[:2], *reference(q[:2], k[:2], v[:2]))
    raise_on_status(q.device, "test")


def test_other_stream_and_recorded():
    from tq_local_b200.runtime.prompt_attention import prompt_attention, raise_on_status

    q, k, v = make(1, 8, 2, 40, 5000, BF16, 9)
    want, tol = reference(q, k, v)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = prompt_attention(q, k, v)
    side.synchronize()
    check(out, want, tol)
    graphs, outs = [], []
    for _ in range(2):  # two recorded calls do not share scratch
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(prompt_attention(q, k, v))
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        for g, s in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o in outs:
            check(o, want, tol)
    raise_on_status(q.device, "test")


def test_generate_runs_its_prompt_on_these_kernels(monkeypatch):
    """``activate(..., prompt_attention=True)``: the prompt's logits agree with the model's own attention within what 16-bit
    activations allow, on an unpadded and a left-padded batch, and the model's implementation is put back."""
    from transformers import LlamaConfig, LlamaForCausalLM

    import turboquant
    from tq_local_b200.runtime import generation, prompt_attention as pa

    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=128, max_position_embeddings=512)
    model = LlamaForCausalLM(cfg).eval().to("cuda", BF16)
    ids = torch.randint(0, 512, (3, 90), device="cuda")
    mask = torch.ones_like(ids)
    mask[1, :40], mask[2, :89] = 0, 0

    class Tokenizer:
        eos_token_id = None

        def decode(self, ids, skip_special_tokens=True):
            return ""

    calls = []
    real = pa.prompt_attention
    monkeypatch.setattr(pa, "prompt_attention", lambda *a, **kw: calls.append(1) or real(*a, **kw))
    for m in (None, mask):
        logits = {}
        for on in (False, True):
            seen = {}
            kept = generation._prefill

            def prefill(*a, **kw):
                out = kept(*a, **kw)
                seen["logits"] = out.logits[:, -1].float()
                return out

            monkeypatch.setattr(generation, "_prefill", prefill)
            turboquant.activate(model, Tokenizer(), quiet=True, norm_guard=False, verify=not on, prompt_attention=on)
            out = model.generate(ids, attention_mask=m, max_new_tokens=4)
            turboquant.deactivate(model, quiet=True)
            monkeypatch.setattr(generation, "_prefill", kept)
            assert out.shape == (3, 94) and model.config._attn_implementation == "sdpa"
            logits[on] = seen["logits"]
            assert len(calls) == (2 if on else 0), calls
            if on:
                calls.clear()
        # two layers of bf16 activations: 2^-8 for each of the dozen roundings between attention and logits
        assert (logits[True] - logits[False]).norm() <= 12 * 2.0 ** -8 * logits[False].norm()


def test_refusals():
    from tq_local_b200.runtime.ffi import TQError
    from tq_local_b200.runtime.prompt_attention import prompt_attention, prompt_attention_packed

    q, k, v = make(1, 4, 2, 8, 8, BF16)
    with pytest.raises(TypeError):
        prompt_attention(q.float(), k.float(), v.float())
    with pytest.raises(TypeError):
        prompt_attention(q, k.half(), v)
    with pytest.raises(ValueError):
        prompt_attention(q[..., :64], k[..., :64], v[..., :64])
    with pytest.raises(ValueError):
        prompt_attention(q[:, :3], k, v)
    with pytest.raises(ValueError):
        prompt_attention(q, k[:, :, :7], v[:, :, :7])
    with pytest.raises(ValueError):
        prompt_attention(q, k, v[:, :, :7])
    with pytest.raises(ValueError):
        prompt_attention(q, k, v, seq_start=torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        prompt_attention(q, k, v, out=torch.empty(1, 4, 8, 128, device="cuda"))
    with pytest.raises(TQError):
        prompt_attention(q, k.cpu(), v.cpu())
    with pytest.raises(TQError):
        prompt_attention(q.detach().requires_grad_(), k, v)
    with torch.no_grad():
        prompt_attention(q.detach().requires_grad_(), k, v)
    big = torch.zeros(1, 65, 1, 128, dtype=BF16, device="cuda")
    with pytest.raises(TQError):
        prompt_attention(big, big[:, :1], big[:, :1])
    p = [t[0].transpose(0, 1) for t in (q, k, v)]
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        prompt_attention_packed(*p, cu, 9)
    with pytest.raises(ValueError):
        prompt_attention_packed(*p, cu.long(), 8)
    # nothing to do
    assert prompt_attention(q[:, :, :0], k, v).shape == (1, 4, 0, 128)
    assert (prompt_attention(q, k[:, :, :0], v[:, :, :0], causal=False) == 0).all()
    assert prompt_attention(q[:0], k[:0], v[:0]).shape == (0, 4, 8, 128)
    assert prompt_attention_packed(*p, cu[:1], 0).shape == p[0].shape


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_nan_keys_reach_the_queries_that_see_them_and_no_others(dtype):
    """One NaN key at each place of a block, a batch entry each: what sees it is NaN, what comes before it is not."""
    from tq_local_b200.runtime.prompt_attention import prompt_attention

    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(128, 1, 300, 128, device="cuda", generator=gen).to(dtype) for _ in range(3))
    at = torch.arange(128, device="cuda")
    k[at, 0, at, 7] = math.nan
    out = prompt_attention(q, k, v)
    sees = torch.arange(300, device="cuda")[None, :] >= at[:, None]
    assert out[:, 0].isnan().all(-1).equal(sees) and out[:, 0].isfinite().all(-1).equal(~sees)
    few = prompt_attention(q[:2, :, -3:], k[:2], v[:2])  # pieces of the keys, joined
    assert few.isnan().all()

"""Attention of a whole prompt over its dense keys and values (``tq_prompt_attn``).

The prompt pass of a packed-cache generation attends dense tensors; these are its kernels: causal, with grouped heads, over a
left-padded batch, a chunk of a prompt behind keys that are there already, or sequences of different lengths laid end to end.
``"turboquant_prompt"`` is the HF attention backend that calls them (``activate(..., prompt_attention=True)``).
"""

from __future__ import annotations

import ctypes as C

import torch

from tq_local_b200.runtime import ffi
from tq_local_b200.runtime.codec import aligned_view, operand, refuse_grad, strided_desc


_SCALE = 128 ** -0.5


def _check(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, dims: int) -> None:
    """Shapes, devices and types of [..., heads, ..., 128] tensors whose heads are the second axis."""
    qs, ks = query.shape, key.shape
    if len(qs) != dims or len(ks) != dims or ks != value.shape or qs[-1] != 128 or ks[-1] != 128:
        raise ValueError(f"expected queries, keys and values of {dims} axes with 128 coordinates, keys and values alike; got {tuple(qs)}, "
                         f"{tuple(ks)}, {tuple(value.shape)}")
    if ks[1] == 0 or qs[1] == 0 or qs[1] % ks[1]:
        raise ValueError(f"query heads must be a multiple of KV heads, got {tuple(qs)}, {tuple(ks)}")
    device, dtype = query.device, query.dtype
    if device.type != "cuda":
        raise ffi.TQError("TurboQuant-B200 runs on CUDA devices only; there is no CPU path")
    if key.device != device or value.device != device:
        raise ffi.TQError(f"queries on {device}, keys on {key.device}, values on {value.device}")
    if dtype not in (torch.float16, torch.bfloat16) or key.dtype != dtype or value.dtype != dtype:
        raise TypeError(f"expected float16 or bfloat16 for all three, got {dtype}, {key.dtype}, {value.dtype}")
    refuse_grad("prompt attention", query, key, value)


def _int32(t: torch.Tensor, shape: tuple, device: torch.device, what: str) -> torch.Tensor:
    if t.dtype != torch.int32 or t.device != device or t.shape != shape:
        raise ValueError(f"{what} must be an int32 tensor {list(shape)} on {device}")
    return t.contiguous()


def _output(out: torch.Tensor | None, query: torch.Tensor, make) -> torch.Tensor:
    if out is None:
        return make()
    if out.shape != query.shape or out.dtype != query.dtype or out.device != query.device or aligned_view(out) is not out:
        raise ValueError("out must have the queries' shape, dtype and device, with rows on 16-byte boundaries")
    return out


def _workspace(device: torch.device, *shape: int) -> tuple[torch.Tensor | None, int]:
    """Scratch of this call alone (calls may overlap or be recorded); mostly none is needed."""
    need = ffi.lib().tq_prompt_workspace_bytes(*shape)
    return (torch.empty(need, dtype=torch.uint8, device=device) if need else None), need


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *, scale: float | None = None,
                     causal: bool = True, seq_start: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``query`` [B, Hq, Sq, 128], ``key`` / ``value`` [B, Hkv, Skv, 128] (fp16 or bf16, any outer strides) -> [B, Hq, Sq, 128], a view of
    [B, Sq, Hq, 128].  Causal: query ``i`` sees the keys up to ``i + Skv - Sq`` (so ``Sq`` < ``Skv`` is a chunk behind
    ``Skv - Sq`` earlier tokens).  ``seq_start`` (int32 [B] on the device): entry ``b`` attends keys from there on, a
    left-padded batch; a query that sees no key gets zeros, one whose logits are all -inf NaN.  ``scale`` defaults to 1/sqrt(128)."""
    _check(query, key, value, 4)
    (b, hq, n_q, _), (b_kv, hkv, n_kv, _) = query.shape, key.shape
    if b_kv != b or (causal and n_kv < n_q):
        raise ValueError(f"keys {tuple(key.shape)} do not go with queries {tuple(query.shape)}" + (" under a causal mask" if causal else ""))
    if seq_start is not None:
        seq_start = _int32(seq_start, (b,), query.device, "seq_start")
    out = _output(out, query, lambda: torch.empty_strided((b, hq, n_q, 128), (n_q * hq * 128, 128, hq * 128, 1), dtype=query.dtype,
                                                          device=query.device))
    if out.numel() == 0:
        return out
    if n_kv == 0:
        return out.zero_()
    (q, qd), (k, kd), (v, vd), od = operand(query), operand(key), operand(value), strided_desc(out)
    ws, need = _workspace(query.device, b, hq, hkv, n_q, n_kv)
    ffi.launch("tq_prompt_attn", query.device, (
        C.byref(qd), C.byref(kd), C.byref(vd), b, hq, hkv, n_q, n_kv, None if seq_start is None else seq_start.data_ptr(),
        _SCALE if scale is None else float(scale), int(causal), None if ws is None else ws.data_ptr(), need, C.byref(od)))
    return out


def prompt_attention_packed(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int, *,
                            scale: float | None = None, causal: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """Sequences laid end to end: ``query`` [total, Hq, 128], ``key`` / ``value`` [total, Hkv, 128] -> [total, Hq, 128].  Sequence
    ``s`` is the tokens ``[cu_seqlens[s], cu_seqlens[s + 1])`` (int32 on the device, ascending) and attends itself alone;
    none is longer than ``max_seqlen``.  Tokens behind the last sequence are left as they were in ``out``."""
    _check(query, key, value, 3)
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be an int32 tensor [sequences + 1]")
    cu_seqlens = _int32(cu_seqlens, (int(cu_seqlens.numel()),), query.device, "cu_seqlens")
    total, hq, hkv, n = int(query.shape[0]), int(query.shape[1]), int(key.shape[1]), int(cu_seqlens.numel()) - 1
    if key.shape[0] != total or not 0 <= int(max_seqlen) <= total:
        raise ValueError(f"{total} queries, {int(key.shape[0])} keys and sequences of up to {max_seqlen} tokens do not go together")
    out = _output(out, query, lambda: torch.empty(total, hq, 128, dtype=query.dtype, device=query.device))
    if n == 0 or max_seqlen == 0:
        return out
    (q, qd), (k, kd), (v, vd) = (operand(t.transpose(0, 1).unsqueeze(0)) for t in (query, key, value))
    od = strided_desc(out.transpose(0, 1).unsqueeze(0))
    ws, need = _workspace(query.device, n, hq, hkv, int(max_seqlen), int(max_seqlen))
    ffi.launch("tq_prompt_attn_packed", query.device, (
        C.byref(qd), C.byref(kd), C.byref(vd), n, total, hq, hkv, cu_seqlens.data_ptr(), int(max_seqlen),
        _SCALE if scale is None else float(scale), int(causal), None if ws is None else ws.data_ptr(), need, C.byref(od)))
    return out


def raise_on_status(device: torch.device, where: str) -> None:
    """Raise :class:`TQError` when a prompt kernel of this device has given up waiting (synchronises with the device).  What is reported is
    cleared: it says nothing of later calls."""
    v = C.c_int32()
    with torch.cuda.device(device):
        ffi.check(ffi.lib().tq_prompt_status(C.byref(v)), "tq_prompt_status")
        if v.value:
            ffi.check(ffi.lib().tq_prompt_status_clear(), "tq_prompt_status_clear")
    if v.value:
        raise ffi.TQError(f"{where}: a prompt attention kernel gave up (status {v.value}: 1 a wait ran out, 2 its shared memory did not fit); "
                          "its outputs are not valid")


def _takes(query, key, value, attention_mask, is_causal, dropout, kwargs) -> bool:
    """Whether the kernels compute what the model asks for here: causal attention of 16-bit tensors with 128 coordinates per head
    and at most left padding."""
    return (query.device.type == "cuda" and query.dtype in (torch.float16, torch.bfloat16) and key.dtype == query.dtype
            and value.dtype == query.dtype and query.shape[-1] == 128 and key.shape[-1] == 128 and value.shape == key.shape and query.shape[2] <= key.shape[2] and is_causal and not dropout
            and query.shape[1] // key.shape[1] <= 64
            and not (torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad))
            and (attention_mask is None or attention_mask.dim() == 4)
            and not any(kwargs.get(name) is not None for name in ("sliding_window", "softcap", "s_aux", "position_bias")))


def turboquant_prompt_forward(module, query, key, value, attention_mask, dropout: float = 0.0, scaling: float | None = None,
                              is_causal: bool | None = None, **kwargs):
    """HF attention function of the prompt pass, ``(module, query[B,Hq,Sq,D], key, value, mask, ...) -> (out[B,Sq,Hq,D], None)``.  The
    mask is that of a causal, at most left-padded batch (``generate`` switches here only for those); what the kernels do not compute
    goes to the ``sdpa`` that the model runs otherwise, with all that the model hands down."""
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS

    from tq_local_b200.runtime.packed_qmse_cache import leading_masked_tokens

    causal = getattr(module, "is_causal", True) if is_causal is None else is_causal
    if not _takes(query, key, value, attention_mask, causal, dropout, kwargs):
        return ALL_ATTENTION_FUNCTIONS["sdpa"](module, query, key, value, attention_mask, dropout=dropout, scaling=scaling, is_causal=is_causal, **kwargs)
    starts = None if attention_mask is None else leading_masked_tokens(attention_mask).expand(query.shape[0])
    return prompt_attention(query, key, value, scale=scaling, seq_start=starts).transpose(1, 2), None


def register_prompt_backend() -> None:
    """Register ``"turboquant_prompt"`` with ``transformers`` (and the SDPA mask builder under the same key); idempotent."""
    try:
        from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    except ImportError:
        return
    ALL_ATTENTION_FUNCTIONS.register("turboquant_prompt", turboquant_prompt_forward)
    try:
        from transformers.masking_utils import ALL_MASK_ATTENTION_FUNCTIONS

        ALL_MASK_ATTENTION_FUNCTIONS.register("turboquant_prompt", ALL_MASK_ATTENTION_FUNCTIONS["sdpa"])
    except (ImportError, KeyError):
        pass

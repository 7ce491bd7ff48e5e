"""GPU: attention of drafted tokens, every output bounded by what went into its own row.

Tolerance.  u = 2^-11 is half a step of fp16, and a rounding to fp16 is off by at most u times the number or, among the smallest numbers, by
a = 2^-25.

* The operands are rounded: the rotated (times log2 e) and the projected query, a centre (a value's times 2^e, the power of two that brings the largest to
  [1/2, 1)), and centre times norm.  These errors are not independent of each other: all coordinates of a token with the same code share theirs (with two
  centres a logit s is off by up to 2 u s), all tokens share the query's, and where two tokens have most of the weight one number moves all outputs of
  the row.  So what rounded operands make of an output is computed, not estimated.  The kernel rounds queries that are good to 2^-20: one in 2^8
  rounds the other way, which gives a logit the variance 2^-8 (2u)^2 (sum_d Q_d^2 K_d^2 + sum_i P_i^2 r^2) for rotated query Q and key K, projected
  query P and residual factor r; four times that is allowed, since tokens share these too.
* A weight, relative to a row's largest, is rounded once: uniform errors, independent from token to token.  In the rotated frame they give an output the
  variance sum_j p_j^2 v_j^2 (u^2 + (max p / p_j a)^2) / 3, which R_v mixes.  Six standard deviations hold for millions of outputs.

fp32 sums of 24 steps add at most 2^-19 of a logit's terms, and the output is rounded once."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import tq_oracle as O

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
U, A, LOG2E = 2.0 ** -11, 2.0 ** -25, math.log2(math.e)


def codec_of(bits, qjl):
    from tq_local_b200.runtime.codec import Codec

    return Codec.get(torch.device("cuda", torch.cuda.current_device()), bits, qjl)


def store_of(bits, qjl, k, v, capacity=None):
    from tq_local_b200.runtime.packed_store import PackedStore

    b, h, n, _ = k.shape
    store = PackedStore(codec_of(bits, qjl), b, h, capacity or n)
    for t in store.streams():  # room behind the tokens holds anything
        t.view(torch.uint8).fill_(0xFF)
    store.pack(k, v)
    return store


def normal(*shape, seed=0, spread=0.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, 128, device="cuda", generator=gen)
    return x * torch.exp(spread * torch.randn(*shape, 1, device="cuda", generator=gen))


def expected(store, q, start, mask=None, lengths=None, starts=None):
    """[B, Hq, T, 128] in 64 bits from the cache's bytes -> (out, what it may be off by).  mask: bool [B, T, T]."""
    c, n, scale = store.codec, store.length, 1 / math.sqrt(128)
    b, hq, t, _ = q.shape
    table = lambda name: torch.from_numpy(getattr(c, name)).double().cuda()
    codes = lambda x, bits: torch.from_numpy(O.unpack_codes(x[:, :, :n].reshape(-1, 16 * bits).cpu().numpy(), bits, 128)).cuda().long().view(
        store.batch, store.kv_heads, n, 128)
    j = torch.arange(n, device="cuda")
    ends = torch.full((b,), start, device="cuda") if lengths is None else lengths.long().clamp(0, start)
    first = torch.zeros(b, device="cuda", dtype=torch.long) if starts is None else starts.long().clamp(min=0)
    seen = ((j < ends[:, None]) & (j >= first[:, None]))[:, None, :].repeat(1, t, 1)
    seen[:, :, start:start + t] = torch.ones(t, t, dtype=torch.bool, device="cuda").tril() if mask is None else mask
    used = seen.any(1)[:, None, :]  # (what no node sees holds anything)
    norm = lambda x: torch.where(used, x[:, :, :n].double(), 0.0)
    kn, vn = norm(store.k_norms), norm(store.v_norms)
    fit = 2.0 ** -math.frexp(float(table("cen_v").abs().max()))[1]
    code_k, code_v = codes(store.k_codes, c.key_bits), codes(store.v_codes, c.bits)
    rn = norm(store.k_rnorms) if c.use_qjl else None
    signs = 2.0 * codes(store.k_signs, 1).double() - 1 if c.use_qjl else None
    out, tol = torch.empty(2, b, hq, t, 128, dtype=torch.float64, device="cuda")
    g, rot = hq // store.kv_heads, table("rot_v")
    for h in range(hq):
        x = q[:, h].double()
        rq = x @ table("rot_k").T * scale
        if c.use_qjl:
            r, sq = rn[:, h // g, None], x @ table("qjl").T * (scale * math.sqrt(math.pi / 2) / 128)
        half = lambda query: (query * LOG2E).half().double() / LOG2E

        def attend(kk, vv, query):
            s = query(rq) @ kk.mT
            if c.use_qjl:
                s = s + query(sq) @ signs[:, h // g].mT * r
            s = s.masked_fill(~seen, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
            return s, p, p @ vv

        cen_k, cen_v = table("cen_k")[code_k[:, h // g]], table("cen_v")[code_v[:, h // g]]
        knh, vnh = kn[:, h // g, :, None], vn[:, h // g, :, None]
        kk, vv = cen_k * knh, cen_v * vnh
        s, p, o = attend(kk, vv, lambda query: query)
        rounded = lambda centre, norm: (centre.half().double() * norm).half().double()
        operands = (attend(rounded(cen_k, knh), rounded(cen_v * fit, vnh) / fit, half)[-1] @ rot - o @ rot).abs()
        terms = rq.square() @ kk.square().mT
        if c.use_qjl:
            terms = terms + sq.square().sum(-1, keepdim=True) * r.square()
        w, v2 = p.square() * (4 * 2.0 ** -8 * 4 * U * U * terms), vv.square()
        moved = w @ v2 - 2 * o * (w @ vv) + o.square() * w.sum(-1, keepdim=True)
        least = p.amax(-1, keepdim=True).square() * (A * A / 3) * (seen.double() @ v2)
        off = moved.clamp_min(0) + U * U / 3 * (p.square() @ v2) + least
        reach = (s.masked_fill(~seen, 0.0).abs() + 6 * terms.sqrt()).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
        out[:, h] = o @ rot
        sure = 2.0 ** -19 * (1 + reach) * (p @ vv.abs()).amax(-1, keepdim=True)
        tol[:, h] = 6 * (off @ rot.square()).sqrt() + sure + operands
    return out, tol + torch.finfo(q.dtype).eps / 2 * (out.abs() + tol) + (A if q.dtype == F16 else 0.0)


def check(got, want, tol):
    off = (got.double() - want).abs() / tol.clamp_min(1e-300)
    assert got.isfinite().all() and float(off.max()) <= 1, f"{int((off > 1).sum())} outputs off, by up to {float(off.max()):.3g} x"


def queries(b, hq, t, dtype, seed=1):
    return normal(b, t, hq, seed=seed, spread=0.0).to(dtype).transpose(1, 2)


@pytest.mark.parametrize("bits,qjl", [(4, True), (3, False), (2, True)])
@pytest.mark.parametrize("order", ["up", "down", "by turns"])
@pytest.mark.parametrize("b,hkv,t", [(1, 8, 16), (2, 2, 3), (40, 4, 1)])
def test_maxima_that_move_from_block_to_block(bits, qjl, order, b, hkv, t):
    """Keys that grow, shrink or do both from 64 tokens to the next, so that each half of a row has a maximum of its own in every block and the
    running one moves at most of them; every call gives the same bits."""
    n = 3000 if b < 40 else 700
    at = torch.arange(n + t, device="cuda") // 64
    last = int(at[-1])
    steps = {"up": at / last, "down": 1 - at / last, "by turns": (at % 5) / 4}[order]
    k, v = normal(b, hkv, n + t, seed=7, spread=0.2), normal(b, hkv, n + t, seed=8)
    store = store_of(bits, qjl, (k * (0.1 + 6 * steps)[:, None]).to(BF16), v.to(BF16))
    q = queries(b, 4 * hkv, t, F16)
    want, tol = expected(store, q, n)
    first = store.tree_attn(q)
    check(first, want, tol)
    for _ in range(20):
        assert torch.equal(store.tree_attn(q), first)
    assert store.codec.device_status() == 0


@pytest.mark.parametrize("bits,qjl", [(4, True), (3, False), (2, False)])
@pytest.mark.parametrize("power", [-10, -12, -14, -16])
@pytest.mark.parametrize("t", [1, 12])
def test_small_values(bits, qjl, power, t):
    """A cache whose values all have norms around 2^power: centres times norm would be among fp16's smallest numbers but for the factor 2^e."""
    k, v = normal(2, 2, 300 + t, seed=3), normal(2, 2, 300 + t, seed=4) * (2.0 ** power / math.sqrt(128))
    store = store_of(bits, qjl, k, v)
    q = queries(2, 8, t, BF16)
    check(store.tree_attn(q), *expected(store, q, 300))


@pytest.mark.parametrize("bits,qjl", [(4, True), (3, False), (2, False)])
def test_the_largest_values(bits, qjl):
    """Norms up to fp16's largest number."""
    k, v = normal(1, 2, 200, seed=3), normal(1, 2, 200, seed=4)
    store = store_of(bits, qjl, k, v)
    store.v_norms[:, :, ::3] = 65504.0
    q = queries(1, 8, 5, BF16)
    check(store.tree_attn(q), *expected(store, q, 195))


def words(mask):
    """bool [..., T, T] -> int64 [..., T]"""
    t = mask.shape[-1]
    return (mask.long() << torch.arange(t, device=mask.device)).sum(-1)


def random_tree(b, t, seed):
    gen = torch.Generator().manual_seed(seed)
    mask = torch.zeros(b, t, t, dtype=torch.bool)
    for r in range(b):
        for i in range(t):
            up = int(torch.randint(-1, i, (1,), generator=gen)) if i else -1
            if up >= 0:
                mask[r, i] = mask[r, up]
            mask[r, i, i] = True
    return mask.cuda()


@pytest.mark.parametrize("bits,qjl", [(4, True), (3, False), (2, True)])
@pytest.mark.parametrize("t,dtype", [(1, F16), (12, BF16)])
def test_rows_of_histories_of_different_lengths(bits, qjl, t, dtype):
    """Rows that see one token lie beside rows that see hundreds, whose outputs are many times smaller."""
    lengths = torch.tensor([700, 0, 1, 127, 128, 129, 512, 699, -5, 10_000], dtype=torch.int32, device="cuda")
    starts = torch.tensor([699, 0, 1, 5, 128, 64, 130, 700, 3, -1], dtype=torch.int32, device="cuda")
    b = len(lengths)
    store = store_of(bits, qjl, normal(b, 2, 700 + t, seed=t).to(BF16), normal(b, 2, 700 + t, seed=t + 1).to(BF16), capacity=900)
    q, mask = queries(b, 8, t, dtype), random_tree(b, t, 5)
    check(store.tree_attn(q, words(mask), lengths=lengths), *expected(store, q, 700, mask, lengths))
    store.set_seq_start(starts)
    check(store.tree_attn(q, words(mask), lengths=lengths), *expected(store, q, 700, mask, lengths, starts))
    check(store.tree_attn(q, lengths=lengths), *expected(store, q, 700, None, lengths, starts))
    assert store.codec.device_status() == 0


@pytest.mark.parametrize("bits,qjl", [(4, True), (2, False)])
@pytest.mark.parametrize("b,hq,hkv,n,t,dtype", [(3, 16, 8, 4500, 3, F16), (2, 28, 4, 3001, 64, BF16), (40, 16, 8, 200, 1, F16), (1, 4, 2, 30_000, 40, F16),
                                                (1, 8, 1, 5000, 200, BF16)])
def test_rows_that_are_joined_from_pieces(bits, qjl, b, hq, hkv, n, t, dtype):
    store = store_of(bits, qjl, normal(b, hkv, n + t, seed=b).to(BF16), normal(b, hkv, n + t, seed=b + 1).to(BF16))
    lengths = torch.randint(0, n + 1, (b,), generator=torch.Generator().manual_seed(b), dtype=torch.int32).cuda()
    q, mask = queries(b, hq, t, dtype), random_tree(b, t, 9) if t <= 64 else None
    check(store.tree_attn(q, None if mask is None else words(mask), lengths=lengths), *expected(store, q, n, mask, lengths))
    assert store.codec.device_status() == 0


@pytest.mark.parametrize("bits,qjl", [(4, True), (3, False), (2, True)])
def test_rows_over_norms_of_all_sizes(bits, qjl):
    """Keys and values from 2^-20 to 2^10 of their usual length, zeros among them; each head's values of one size of their own."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    sizes = lambda lo, hi, *s: torch.exp2(torch.randint(lo, hi, (*s, 1), device="cuda", generator=gen).float())
    k = normal(3, 4, 400, seed=3, spread=0.0) * sizes(-20, 3, 3, 4, 400)
    v = normal(3, 4, 400, seed=4, spread=0.0) * sizes(-3, 3, 3, 4, 400) * sizes(-9, 8, 3, 4, 1)
    k[:, :, ::17] = 0
    v[:, :, 5::19] = 0
    store = store_of(bits, qjl, k, v)
    q = queries(3, 16, 9, BF16)
    check(store.tree_attn(q), *expected(store, q, 391))


def test_a_sample_on_the_bounds_checked_build():
    """Every bulk copy and every stored piece lies inside the cache's rows and the workspace: the cases assert a clean status word
    themselves."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = os.path.join(root, "tq_local_b200", "libtq_b200_checked.so")
    assert os.path.isfile(lib), "build it with `python -m tq_local_b200.build --checked`"
    out = subprocess.run([sys.executable, "-m", "pytest", os.path.abspath(__file__), "-m", "gpu", "-x", "-q", "-k",
                          "different_lengths or joined or (block_to_block and 40)"], capture_output=True, text=True, timeout=600,
                         env=dict(os.environ, TQ_B200_LIBRARY=lib), cwd=root)
    assert out.returncode == 0, out.stdout[-3000:] + out.stderr[-2000:]
    assert " passed" in out.stdout and "failed" not in out.stdout

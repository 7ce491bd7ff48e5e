"""GPU: attention of drafted tokens over the packed cache against the same in 64 bits from the cache's own bytes.

Tolerance.  Queries, centres times norms, weights and values enter the products as fp16, five roundings of at most 2^-11 each, of
independent sign from coordinate to coordinate and token to token.  A logit of vectors of norms |q|, |k| = sqrt(128) x 1 .. 4 moves by
2^-11 |q| |k| / 128 = 5e-4 .. 2e-3, a weight by as much, and what is summed over tokens by less: 2e-3 of the largest output, the bound the
one-token kernel is held to, and one rounding of the output, u |out| (u = eps / 2)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import tq_oracle as O

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
MODES = [(4, True), (4, False), (3, True), (3, False), (2, True), (2, False)]


def make_store(bits, qjl, b, hkv, n, capacity=None, seed=0, dtype=BF16):
    from tq_local_b200.runtime.codec import Codec
    from tq_local_b200.runtime.packed_store import PackedStore

    store = PackedStore(Codec.get(torch.device("cuda", torch.cuda.current_device()), bits, qjl), b, hkv, capacity or n)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kv = torch.randn(2, b, hkv, n, 128, device="cuda", generator=gen)
    kv *= torch.exp(0.5 * torch.randn(2, b, hkv, n, 1, device="cuda", generator=gen))
    for t in store.streams():  # room behind the tokens holds anything
        t.view(torch.uint8).fill_(0xFF)
    store.pack(kv[0].to(dtype), kv[1].to(dtype))
    return store


def dense(store):
    """Keys and values of the store in 64 bits, from its bytes and the codec's tables."""
    c, n = store.codec, store.length
    tab = lambda name: torch.from_numpy(getattr(c, name)).double().cuda()
    codes = lambda t, bits: torch.from_numpy(O.unpack_codes(t[:, :, :n].reshape(-1, 16 * bits).cpu().numpy(), bits, 128)).cuda().long().view(
        store.batch, store.kv_heads, n, 128)
    norm = lambda t: t[:, :, :n].double().unsqueeze(-1)
    k = tab("cen_k")[codes(store.k_codes, c.key_bits)] @ tab("rot_k") * norm(store.k_norms)
    if c.use_qjl:
        k += (2.0 * codes(store.k_signs, 1).double() - 1) @ tab("qjl") * norm(store.k_rnorms) * (math.sqrt(math.pi / 2) / 128)
    return k, tab("cen_v")[codes(store.v_codes, c.bits)] @ tab("rot_v") * norm(store.v_norms)


def reference(store, q, t0, mask=None, lengths=None, starts=None):
    """mask: bool [B, T, T]."""
    k, v = dense(store)
    b, hq, t, _ = q.shape
    g = hq // store.kv_heads
    j = torch.arange(store.length, device="cuda")
    ends = torch.full((b,), t0, device="cuda") if lengths is None else lengths.long().clamp(0, t0)
    first = torch.zeros(b, device="cuda", dtype=torch.long) if starts is None else starts.long().clamp(min=0)
    seen = ((j < ends[:, None]) & (j >= first[:, None]))[:, None, :].repeat(1, t, 1)
    if mask is None:
        mask = torch.ones(t, t, dtype=torch.bool, device="cuda").tril().expand(b, t, t)
    seen[:, :, t0:t0 + t] = mask
    seen = seen[:, None]
    s = (q.double() @ k.repeat_interleave(g, 1).mT / math.sqrt(128)).masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    return p @ v.repeat_interleave(g, 1)


def check(got, want):
    u = torch.finfo(got.dtype).eps / 2
    assert got.isfinite().all()
    off = (got.double() - want).abs() - u * want.abs()
    assert float(off.max()) <= 2e-3 * float(want.abs().max()), float(off.max()) / float(want.abs().max())


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


def queries(b, hq, t, dtype, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(b, t, hq, 128, device="cuda", generator=gen).to(dtype).transpose(1, 2)


@pytest.mark.parametrize("bits,qjl", MODES)
@pytest.mark.parametrize("n,t,hq,hkv,dtype", [(300, 7, 8, 2, BF16), (129, 64, 7, 1, F16), (1000, 33, 16, 2, F16), (1, 1, 4, 1, BF16)])
def test_trees(bits, qjl, n, t, hq, hkv, dtype):
    store = make_store(bits, qjl, 2, hkv, n + t, seed=n)
    mask, q = random_tree(2, t, n), queries(2, hq, t, dtype)
    out = store.tree_attn(q, words(mask))
    assert out.shape == q.shape and out.dtype == dtype and out.transpose(1, 2).is_contiguous()
    check(out, reference(store, q, n, mask))
    assert store.codec.device_status() == 0


@pytest.mark.parametrize("n", [0, 1, 63, 64, 127, 128, 129, 255, 257, 640, 4099])
@pytest.mark.parametrize("t", [1, 5, 64])
def test_lengths_around_tiles(n, t):
    store = make_store(4, True, 1, 2, n + t, seed=n + t)
    q = queries(1, 8, t, BF16)
    check(store.tree_attn(q), reference(store, q, n))
    mask = random_tree(1, t, t)
    check(store.tree_attn(q, words(mask)[0]), reference(store, q, n, mask))


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8])
def test_group_sizes(group):
    store = make_store(3, True, 2, 2, 500, seed=group)
    q = queries(2, 2 * group, 21, F16)
    check(store.tree_attn(q), reference(store, q, 479))


@pytest.mark.parametrize("t,n", [(65, 10), (200, 333), (300, 0)])
def test_long_chains(t, n):
    store = make_store(4, False, 2, 1, n + t, seed=t)
    q = queries(2, 4, t, BF16)
    check(store.tree_attn(q), reference(store, q, n))


@pytest.mark.parametrize("t", [1, 12])
@pytest.mark.parametrize("qjl", [True, False])
def test_histories_of_different_lengths(t, qjl):
    """Histories from nothing to all, offsets before, inside and behind them, a gap of stale tokens before the drafted ones."""
    lengths = torch.tensor([700, 0, 1, 127, 128, 129, 512, 699, -5, 10_000], dtype=torch.int32, device="cuda")
    b = len(lengths)
    store = make_store(4, qjl, b, 2, 700 + t, capacity=900, seed=t)
    q, mask = queries(b, 8, t, BF16), random_tree(b, t, 5)
    check(store.tree_attn(q, words(mask), lengths=lengths), reference(store, q, 700, mask, lengths))
    starts = torch.tensor([699, 0, 1, 5, 128, 64, 130, 700, 3, -1], dtype=torch.int32, device="cuda")
    store.set_seq_start(starts)
    check(store.tree_attn(q, words(mask), lengths=lengths), reference(store, q, 700, mask, lengths, starts))
    check(store.tree_attn(q, lengths=lengths), reference(store, q, 700, None, lengths, starts))


def test_rows_that_see_nothing_and_odd_masks():
    t = 40
    store = make_store(4, True, 2, 1, 200 + t)
    q = queries(2, 4, t, F16)
    mask = torch.rand(2, t, t, device="cuda") < 0.3  # any mask: not even itself
    mask[:, 3] = False
    lengths = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    out = store.tree_attn(q, words(mask), lengths=lengths)
    check(out, reference(store, q, 200, mask, lengths))
    assert (out[0, :, 3] == 0).all()
    assert torch.equal(store.tree_attn(q, words(mask) | -1 << t, lengths=lengths), out)  # bits of nodes that do not exist
    store.set_seq_start(torch.tensor([0, 200], dtype=torch.int32, device="cuda"))
    none = torch.zeros(2, t, dtype=torch.int64, device="cuda")
    assert (store.tree_attn(q, none, lengths=lengths) == 0).all()


def test_hidden_tokens_hold_anything():
    """Norms outside [start, length) and beyond the drafted tokens are not looked at."""
    store = make_store(4, True, 2, 2, 420, capacity=1024)
    starts, lengths = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 130], [300, 390]))
    store.set_seq_start(starts)
    q = queries(2, 8, 20, BF16)
    want = reference(store, q, 400, None, lengths, starts)
    for t in (store.k_norms, store.v_norms, store.k_rnorms):
        t[0, :, 300:400], t[1, :, :130], t[1, :, 390:400], t[:, :, 420:] = math.nan, math.inf, -math.inf, math.nan
    check(store.tree_attn(q, lengths=lengths), want)


def test_extreme_norms():
    """Keys and values from 2^-20 to 2^10 of their usual length, zeros among them."""
    from tq_local_b200.runtime.codec import Codec
    from tq_local_b200.runtime.packed_store import PackedStore

    gen = torch.Generator(device="cuda").manual_seed(3)
    kv = torch.randn(2, 1, 2, 400, 128, device="cuda", generator=gen) * torch.exp2(torch.randint(-20, 3, (2, 1, 2, 400, 1), device="cuda", generator=gen).float())
    kv[:, :, :, ::17] = 0
    kv[1, :, :, 5::23] *= 1000
    store = PackedStore(Codec.get(torch.device("cuda", 0), 4, True), 1, 2, 400)
    store.pack(kv[0], kv[1])
    q = queries(1, 8, 9, BF16)
    check(store.tree_attn(q), reference(store, q, 391))


@pytest.mark.parametrize("b,hkv,n,t", [(3, 8, 4500, 3), (2, 16, 3001, 64), (40, 8, 200, 1), (1, 2, 30_000, 40)])
def test_many_blocks_and_many_rows_a_cta(b, hkv, n, t):
    """More blocks than SMs: a CTA goes through several, and from one row of the cache to the next."""
    store = make_store(4, True, b, hkv, n + t, seed=b)
    lengths = torch.randint(0, n + 1, (b,), generator=torch.Generator().manual_seed(b), dtype=torch.int32).cuda()
    q, mask = queries(b, 2 * hkv, t, F16), random_tree(b, t, 9)
    for _ in range(20):
        out = store.tree_attn(q, words(mask), lengths=lengths)
    check(out, reference(store, q, n, mask, lengths))
    assert store.codec.device_status() == 0


def test_query_layouts_and_given_output():
    store = make_store(4, True, 2, 2, 300)
    q = queries(2, 8, 10, BF16)
    want = reference(store, q, 290)
    check(store.tree_attn(q.contiguous()), want)
    check(store.tree_attn(torch.empty(2, 8, 10, 131, dtype=BF16, device="cuda")[..., 3:].copy_(q)), want)
    out = torch.empty(2, 8, 10, 160, dtype=BF16, device="cuda")[..., 16:144]
    assert store.tree_attn(q, out=out) is out
    check(out, want)
    same = q[:, :, :1].expand(2, 8, 10, 128)
    check(store.tree_attn(same), reference(store, same, 290))


def test_agrees_with_the_one_token_kernel():
    store = make_store(4, True, 3, 2, 2000)
    q = queries(3, 8, 1, BF16)
    a, b = store.tree_attn(q).double(), store.decode_attn(q).double()
    assert float((a - b).abs().max()) <= (2 * 2e-3 + 2 ** -7) * float(b.abs().max())


def test_other_stream_recorded_and_repeatable():
    store = make_store(4, True, 1, 2, 9000)
    q, mask = queries(1, 8, 12, BF16), random_tree(1, 12, 2)
    m, lengths = words(mask), torch.tensor([8500], dtype=torch.int32, device="cuda")
    want = store.tree_attn(q, m, lengths=lengths)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(store.tree_attn(q, m, lengths=lengths))
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        for g, s in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
    lengths.fill_(100)  # a replay takes lengths and masks as they are then
    graphs[0].replay()
    torch.cuda.synchronize()
    check(outs[0], reference(store, q, 8988, mask, lengths))


# ------------------------------------------------------------------------------------------------ accepted tokens
def streams(store):
    return [t.clone() for t in store.streams()]


@pytest.mark.parametrize("bits,qjl", MODES)
def test_keep_tokens(bits, qjl):
    b, t = 6, 30
    store = make_store(bits, qjl, b, 3, 200 + t, capacity=240)
    lengths = torch.tensor([200, 0, 7, 150, 199, 200], dtype=torch.int32, device="cuda")
    gen = torch.Generator().manual_seed(1)
    counts = torch.tensor([5, 30, 0, 12, 1, 30], dtype=torch.int32)
    path = torch.zeros(b, t, dtype=torch.int32)
    for r, c in enumerate(counts.tolist()):
        path[r, :c] = torch.randperm(t, generator=gen)[:c].sort().values
    before = streams(store)
    new = store.keep_tokens(path.cuda(), counts.cuda(), tree_start=200, lengths=lengths)
    assert new.tolist() == (lengths.cpu() + counts).tolist()
    for was, now in zip(before, store.streams()):
        for r, c in enumerate(counts.tolist()):
            n = int(lengths[r])
            was[r, :, n:n + c] = was[r, :, 200 + path[r, :c].long().cuda()].clone()
        assert torch.equal(was.view(torch.uint8), now.view(torch.uint8))
    assert store.codec.device_status() == 0


def test_keep_long_paths_in_place():
    """More tokens than a block stages at once, landing among their sources."""
    store = make_store(4, True, 1, 2, 50 + 400)
    path = torch.arange(0, 400, dtype=torch.int32, device="cuda")[::2].reshape(1, -1).contiguous()
    path[0, 150:] = torch.arange(350, 400, device="cuda")
    before = streams(store)
    new = store.keep_tokens(path, torch.tensor([200], dtype=torch.int32, device="cuda"), tree_start=50,
                            lengths=torch.tensor([50], dtype=torch.int32, device="cuda"))
    assert new.tolist() == [250]
    for was, now in zip(before, store.streams()):
        assert torch.equal(now[:, :, 50:250].view(torch.uint8), was[:, :, 50 + path[0].long()].view(torch.uint8))
        assert torch.equal(now[:, :, :50].view(torch.uint8), was[:, :, :50].view(torch.uint8))
        assert torch.equal(now[:, :, 250:].view(torch.uint8), was[:, :, 250:].view(torch.uint8))


def test_keep_drops_what_is_out_of_range():
    from tq_local_b200.runtime.codec import Codec
    from tq_local_b200.runtime.packed_store import PackedStore

    store = PackedStore(Codec(torch.device("cuda", torch.cuda.current_device()), 4, True), 6, 1, 104)
    kv = torch.randn(2, 6, 1, 104, 128, device="cuda")
    store.pack(kv[0], kv[1])
    before = streams(store)
    path = torch.tensor([[0, 1], [1, 1], [-1, 0], [0, 4], [0, 1], [0, 1]], dtype=torch.int32, device="cuda")
    counts = torch.tensor([2, 2, 2, 2, 3, -1], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([101, 10, 10, 10, 10, 10], dtype=torch.int32, device="cuda")
    assert store.keep_tokens(path, counts, tree_start=100, lengths=lengths).tolist() == lengths.tolist()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, store.streams()))
    assert store.codec.device_status() == 7


# ------------------------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("bits,qjl", MODES)
@pytest.mark.parametrize("b,lo,hi", [(2, 0, None), (5, 3, 77), (16, 13, 14), (17, 0, 100), (70, 1, 100), (300, 9, None)])
def test_select_rows(bits, qjl, b, lo, hi):
    store = make_store(bits, qjl, b, 2, 101, capacity=120, seed=b)
    starts = torch.arange(b, dtype=torch.int32, device="cuda")
    gen = torch.Generator().manual_seed(b)
    for index in (torch.randperm(b, generator=gen), torch.randint(0, b, (b,), generator=gen), torch.arange(b), torch.zeros(b, dtype=torch.long)):
        store.set_seq_start(starts)
        before = streams(store)
        store.select_rows(index.cuda() if b != 5 else index.cuda().int(), lo, hi)
        assert torch.equal(store._seq_start, starts[index.cuda()])
        for was, now in zip(before, store.streams()):
            end = 101 if hi is None else hi
            want = was.clone()
            want[:, :, lo:end] = was[index.cuda(), :, lo:end]
            assert torch.equal(want.view(torch.uint8), now.view(torch.uint8))
    assert store.codec.device_status() == 0


@pytest.mark.parametrize("bits,qjl", MODES)
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_take_rows(bits, qjl, rows):
    store = make_store(bits, qjl, 5, 2, 61, seed=rows)
    index = torch.randint(0, 5, (rows,), generator=torch.Generator().manual_seed(rows)).cuda()
    other = store.take_rows(index, capacity=300)
    assert (other.batch, other.length, other.capacity, other._seq_start) == (rows, 61, 304, None)
    for a, b in zip(store.streams(), other.streams()):
        assert torch.equal(a[index, :, :61].view(torch.uint8), b[:, :, :61].view(torch.uint8))
    store.set_seq_start(torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device="cuda"))
    assert torch.equal(store.take_rows(index)._seq_start.long(), index)


def test_rows_out_of_range_are_dropped():
    from tq_local_b200.runtime.codec import Codec
    from tq_local_b200.runtime.packed_store import PackedStore

    store = PackedStore(Codec(torch.device("cuda", torch.cuda.current_device()), 3, False), 4, 1, 16)
    kv = torch.randn(2, 4, 1, 16, 128, device="cuda")
    store.pack(kv[0], kv[1])
    store.set_seq_start(torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda"))
    before = streams(store)
    store.select_rows(torch.tensor([-1, 4, 3, 2], device="cuda"))
    for was, now in zip(before, store.streams()):
        assert torch.equal(was[[0, 1, 3, 2]].view(torch.uint8), now.view(torch.uint8))
    assert store._seq_start.tolist() == [0, 1, 3, 2] and store.codec.device_status() == 7


def test_too_many_rows_in_place_are_refused():
    from tq_local_b200.runtime.ffi import TQError

    store = make_store(2, False, 449, 1, 8)
    with pytest.raises(TQError):
        store.select_rows(torch.arange(449, device="cuda"))
    assert store.take_rows(torch.arange(449, device="cuda")).batch == 449


# ------------------------------------------------------------------------------------------------ together
def test_refusals():
    from tq_local_b200.runtime.ffi import TQError

    store = make_store(4, True, 2, 2, 80)
    q = queries(2, 8, 4, BF16)
    with pytest.raises(TQError):
        store.tree_attn(q.float())
    with pytest.raises(TQError):
        store.tree_attn(queries(2, 18, 4, BF16))  # nine queries per KV head
    with pytest.raises(TQError):
        store.tree_attn(queries(2, 8, 65, BF16), torch.zeros(2, 65, dtype=torch.int64, device="cuda"))
    with pytest.raises(TQError):
        store.tree_attn(q.cpu())
    with pytest.raises(TQError):
        store.tree_attn(q.detach().requires_grad_())
    for bad in (dict(tree_start=77), dict(tree_start=-1), dict(lengths=torch.zeros(2, device="cuda")), dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda")),
                dict(tree_mask=torch.zeros(2, 4, dtype=torch.int32, device="cuda")), dict(tree_mask=torch.zeros(2, 5, dtype=torch.int64, device="cuda")),
                dict(out=torch.empty(2, 8, 4, 128, device="cuda"))):
        with pytest.raises(ValueError):
            store.tree_attn(q, **bad)
    with pytest.raises(ValueError):
        store.tree_attn(q[:1])
    with pytest.raises(ValueError):
        store.tree_attn(queries(2, 7, 4, BF16))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        store.keep_tokens(i32(0, 1), i32(1, 1), tree_start=70, lengths=i32(1, 1))
    with pytest.raises(ValueError):
        store.keep_tokens(i32(0, 1).view(2, 1), i32(1, 1), tree_start=81, lengths=i32(1, 1))
    for index, lo in ((torch.zeros(3, dtype=torch.long, device="cuda"), 0), (torch.zeros(2, device="cuda"), 0), (torch.zeros(2, dtype=torch.long), 0),
                      (torch.zeros(2, dtype=torch.long, device="cuda"), 81)):
        with pytest.raises(ValueError):
            store.select_rows(index, lo)
    with pytest.raises(ValueError):
        store.take_rows(torch.zeros(0, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError):
        store.truncate(81)
    assert store.tree_attn(q[:, :, :0]).shape == (2, 8, 0, 128)
    assert store.keep_tokens(torch.zeros(2, 0, dtype=torch.int32, device="cuda"), i32(0, 0), tree_start=80, lengths=i32(3, 4)).tolist() == [3, 4]


def test_a_drafting_loop():
    """Prompt attention, packing, a fork, two rounds of drafting with ragged acceptance, one more token: every step against
    64 bits, and the cache's bytes against the same tokens packed in their final order."""
    from tq_local_b200.runtime.codec import Codec
    from tq_local_b200.runtime.packed_store import PackedStore
    from tq_local_b200.runtime.prompt_attention import prompt_attention

    gen = torch.Generator(device="cuda").manual_seed(11)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(BF16)
    codec = Codec.get(torch.device("cuda", torch.cuda.current_device()), 4, True)
    k, v = rnd(2, 2, 100, 128), rnd(2, 2, 100, 128)
    assert prompt_attention(rnd(2, 8, 100, 128), k, v).isfinite().all()
    base = PackedStore(codec, 2, 2, 100)
    base.pack(k, v)
    rows = torch.tensor([0, 0, 1], device="cuda")
    store = base.take_rows(rows, capacity=160)
    kept = [(k[r], v[r]) for r in rows.tolist()]
    lengths = torch.full((3,), 100, dtype=torch.int32, device="cuda")
    for paths in ([[0, 2, 5], [1], []], [[0, 1, 2, 3, 4, 5, 6], [3, 6], [0]]):
        start, t = store.length, 7
        kt, vt = rnd(3, 2, t, 128), rnd(3, 2, t, 128)
        store.pack(kt, vt)
        q, mask = rnd(3, 8, t, 128), random_tree(3, t, start)
        check(store.tree_attn(q, words(mask), lengths=lengths), reference(store, q, start, mask, lengths))
        path = torch.zeros(3, t, dtype=torch.int32)
        for r, p in enumerate(paths):
            path[r, :len(p)] = torch.tensor(p, dtype=torch.int32)
            kept[r] = tuple(torch.cat((old, new[r][:, p]), dim=1) for old, new in zip(kept[r], (kt, vt)))
        counts = torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda")
        lengths = store.keep_tokens(path.cuda(), counts, tree_start=start, lengths=lengths)
        store.truncate(int(lengths.max()))
    assert lengths.tolist() == [110, 103, 101]
    for r, (kr, vr) in enumerate(kept):
        alone = PackedStore(codec, 1, 2, 160)
        alone.pack(kr.unsqueeze(0), vr.unsqueeze(0))
        n = alone.length
        assert n == int(lengths[r])
        for a, b in zip(alone.streams(), store.streams()):
            assert torch.equal(a[:, :, :n].view(torch.uint8), b[r:r + 1, :, :n].view(torch.uint8))
    start = store.length
    store.pack(rnd(3, 2, 1, 128), rnd(3, 2, 1, 128))
    q = rnd(3, 8, 1, 128)
    check(store.tree_attn(q, lengths=lengths), reference(store, q, start, None, lengths))
    assert codec.device_status() == 0


def _tiny_model():
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=128, max_position_embeddings=512)
    return LlamaForCausalLM(cfg).eval().to("cuda", BF16)


@torch.inference_mode()
def test_a_model_step_of_drafted_tokens_and_the_cache_hooks():
    """A model's forward pass over a tree of drafted tokens gives every branch the hidden states it has when its tokens are fed
    one at a time, and Cache.reorder_cache / batch_* / crop move the packed layers."""
    from tq_local_b200.adapters.transformers import disable_turboquant_attention, enable_turboquant_attention
    from tq_local_b200.runtime.packed_qmse_cache import build_packed_mse_cache

    model = _tiny_model()
    ids = torch.randint(0, 512, (1, 50), device="cuda")

    def fresh():
        return build_packed_mse_cache(model(input_ids=ids, use_cache=True).past_key_values, bits=4, use_qjl_keys=True, quantize_decode=True,
                                      norm_guard=False, reserve_tokens=32)

    drafted = torch.tensor([[3, 14, 15, 92, 65]], device="cuda")
    parents = [-1, 0, 0, 2, 1]
    mask = torch.zeros(1, 5, 5, dtype=torch.bool, device="cuda")
    depth = []
    for i, p in enumerate(parents):
        if p >= 0:
            mask[0, i] = mask[0, p]
        mask[0, i, i] = True
        depth.append(0 if p < 0 else depth[p] + 1)
    position = torch.tensor([[50 + d for d in depth]], device="cuda")
    cache = fresh()
    old = enable_turboquant_attention(model, cache)
    for layer in cache.layers:
        layer.bind_tree(words(mask))
    tree = model(input_ids=drafted, position_ids=position, past_key_values=cache, use_cache=True).logits.float()
    for layer in cache.layers:
        layer.unbind_tree()
    path, lengths = torch.tensor([[0, 2, 3]], dtype=torch.int32, device="cuda"), torch.tensor([50], dtype=torch.int32, device="cuda")
    new = [layer.keep_tokens(path, torch.tensor([3], dtype=torch.int32, device="cuda"), tree_start=50, lengths=lengths) for layer in cache.layers]
    cache.crop(int(new[0]))
    assert cache.get_seq_length() == 53
    nxt = model(input_ids=drafted[:, :1], position_ids=torch.tensor([[53]], device="cuda"), past_key_values=cache, use_cache=True).logits.float()
    disable_turboquant_attention(model, cache, old)

    for leaf in ([0, 1, 4], [0, 2, 3]):
        single = fresh()
        old = enable_turboquant_attention(model, single)
        for d, i in enumerate(leaf):
            one = model(input_ids=drafted[:, i:i + 1], position_ids=torch.tensor([[50 + d]], device="cuda"), past_key_values=single,
                        use_cache=True).logits.float()
            # two layers of bf16 activations: a dozen roundings of 2^-8
            assert (one[0, 0] - tree[0, i]).norm() <= 12 * 2.0 ** -8 * one.norm()
        if leaf == [0, 2, 3]:
            one = model(input_ids=drafted[:, :1], position_ids=torch.tensor([[53]], device="cuda"), past_key_values=single, use_cache=True).logits.float()
            assert (one - nxt).norm() <= 12 * 2.0 ** -8 * one.norm()
        disable_turboquant_attention(model, single, old)

    cache.batch_repeat_interleave(3)
    store = cache.layers[1].store
    assert store.batch == 3 and torch.equal(store.k_codes[0, :, :53], store.k_codes[2, :, :53])
    store.k_norms[:, :, 0] = torch.tensor([1.0, 2.0, 3.0], device="cuda").half().view(3, 1)
    cache.reorder_cache(torch.tensor([2, 0, 0], device="cuda"))
    assert store.k_norms[:, 0, 0].tolist() == [3.0, 1.0, 1.0]
    cache.batch_select_indices(torch.tensor([1], device="cuda"))
    assert cache.layers[1].store.batch == 1 and cache.layers[1].store.k_norms[0, 0, 0] == 1.0
    cache.crop(-3)  # 50 of the prompt, three kept, one fed after them
    assert cache.get_seq_length() == 51


def test_hooks_of_layers_with_a_dense_tail_and_of_dense_layers():
    from tq_local_b200.runtime.packed_qmse_cache import PackedMSELayer

    k, v = torch.randn(2, 2, 20, 128, device="cuda"), torch.randn(2, 2, 20, 128, device="cuda")
    for dense_layer in (False, True):
        layer = PackedMSELayer(bits=4, use_qjl_keys=True, quantize_decode=False)
        layer.initialize_from_dense(k, v, force_dense=dense_layer)
        layer._lazy_update = True
        layer.update(k[:, :, :3], v[:, :, :3])
        with pytest.raises((RuntimeError, NotImplementedError)):
            layer.bind_tree(None)
        layer.reorder_cache(torch.tensor([1, 0], device="cuda"))
        assert torch.equal(layer._dense_k.view()[:, :, -3:], k[[1, 0], :, :3])
        layer.crop(-2)
        assert layer.get_seq_length() == 21
        layer.crop(10)
        assert layer.get_seq_length() == 10 and layer._dense_k.length == (10 if dense_layer else 0)
        layer.batch_repeat_interleave(2)
        assert (layer._dense_k.buf if dense_layer else layer.store.k_codes).shape[0] == 4


def test_rows_of_a_padded_cache_are_not_recorded():
    """The row offsets go to a tensor of their own, which a replay would fill from the old ones again; without offsets a replay moves rows again."""
    from tq_local_b200.runtime import ffi

    store = make_store(4, True, 3, 2, 24)
    index = torch.tensor([1, 2, 0], device="cuda")
    store.select_rows(index)  # (loads the kernel)
    before = store.k_codes.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        store.select_rows(index)
    graph.replay(), graph.replay()
    assert torch.equal(store.k_codes, before[index][index])
    starts = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda")
    store.set_seq_start(starts)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ffi.TQError):
            store.select_rows(index)
    store.select_rows(index)
    assert store._seq_start.tolist() == [3, 5, 0] and starts.tolist() == [0, 3, 5]


def test_more_rows_in_place_than_fit_are_refused():
    import ctypes as C

    from tq_local_b200.runtime import ffi

    store = make_store(4, True, 2, 2, 24)
    for rows in (449, 4_194_304, 8_388_608):  # refused on the host, before anything is read
        d = ffi.CacheDesc.from_buffer_copy(store._desc_ref._obj)
        d.batch = rows
        assert ffi.lib().tq_cache_select_rows(store.codec.handle, C.byref(d), C.byref(d), store.k_codes.data_ptr(), 0, 24, None, None) == -2


@pytest.mark.parametrize("name", ["k_norms", "k_rnorms", "v_norms"])
def test_nan_norms_reach_the_head_that_holds_them_alone(name):
    store = make_store(4, True, 2, 2, 700)
    q = queries(2, 8, 5, F16)
    getattr(store, name)[1, 0, 130] = math.nan
    out = store.tree_attn(q)
    assert out[1, :4].isnan().all() and out[0].isfinite().all() and out[1, 4:].isfinite().all()

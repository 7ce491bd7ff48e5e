"""Prompt attention, attention of drafted tokens, and the moves of a packed cache: cases that can be timed and compared.

Four kinds, each one pass through one operator:

* ``prompt``  attention of a whole prompt over dense keys and values: a (left-padded) batch, a chunk of a prompt behind keys
              that are there already, or sequences of different lengths laid end to end
* ``tree``    attention of drafted tokens over one layer's packed cache: every batch entry has a history of its own
              length, and its drafted tokens (at one common position behind all histories) see the history and
              their ancestors, or, as a chain, all tokens before them
* ``keep``    the accepted ones of the drafted tokens move behind their history, in all streams of the layer's cache
* ``rows``    batch entries of the layer's cache become copies of others, in place or as a cache of another batch size

Queries, keys and values are iid N(0,1) coordinates with lognormal(0, 0.5) norms per key and value; a packed cache holds
the codes of such vectors, encoded here from the definition.  With ``own`` set, ``run`` calls the library; otherwise it
computes the same with elementary tensor operations in 32 bits.
"""

from __future__ import annotations

import functools
import math
import random

import numpy as np
import torch

own = False

D = 128
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
HEADS = ((32, 8), (28, 4), (8, 2), (16, 2))  # query heads, KV heads: 4, 7, 4 and 8 queries per KV head
SKETCH = math.sqrt(math.pi / 2.0) / D
MOST_PAIRS = 32 * 32768 * 32768 // 2         # visible (query head, key) pairs of the largest listed prompt
MOST_TREE = 8 * 8 * 32768                    # packed tokens of the largest listed tree (its queries fill one block of 128 per KV head)
MOST_ROWS = 16 * 8 * 32768                   # packed tokens of the largest listed row move


# ---------------------------------------------------------------------------------------------------- cases
def _prompt(batch, s_q, s_kv=None, q_heads=32, kv_heads=8, dtype="bf16", layout="batch", padded=False, cut=1):
    return dict(kind="prompt", batch=batch, s_q=s_q, s_kv=s_q if s_kv is None else s_kv, q_heads=q_heads, kv_heads=kv_heads,
                dtype=dtype, layout=layout, padded=padded, cut=cut)


def _tree(batch, ctx, nodes, q_heads=32, kv_heads=8, bits=4, qjl=True, dtype="bf16", chain=False, ragged=True, cut=1):
    return dict(kind="tree", batch=batch, ctx=ctx, nodes=nodes, q_heads=q_heads, kv_heads=kv_heads, bits=bits, qjl=qjl,
                dtype=dtype, chain=chain, ragged=ragged, cut=cut)


def _keep(batch, ctx, nodes, kv_heads=8, bits=4, qjl=True, cut=1):
    return dict(kind="keep", batch=batch, ctx=ctx, nodes=nodes, kv_heads=kv_heads, bits=bits, qjl=qjl, cut=cut)


def _rows(batch, ctx, lo=0, rows_out=0, kv_heads=8, bits=4, qjl=True, cut=1):
    """``rows_out`` 0: in place, tokens [lo, ctx); otherwise a new cache of that many rows."""
    return dict(kind="rows", batch=batch, ctx=ctx, lo=lo, rows_out=rows_out, kv_heads=kv_heads, bits=bits, qjl=qjl, cut=cut)


def listed():
    return [
        # a chat turn: one short prompt, launch latency is everything
        dict(_prompt(1, 77), name="prompt_b1_s77"),
        # a small left-padded batch of middle-sized prompts, 7 queries per KV head, fp16
        dict(_prompt(4, 1000, q_heads=28, kv_heads=4, dtype="f16", padded=True), name="prompt_b4_s1000_padded_g7_f16"),
        # sixteen requests of very different lengths laid end to end
        dict(_prompt(16, 24001, layout="packed"), name="prompt_16_packed_24001"),
        # one long document
        dict(_prompt(1, 32768), name="prompt_b1_s32768"),
        # one drafted token per sequence: single-token decoding of a batch whose lengths have drifted apart
        dict(_tree(4, 4099, 1), name="tree_b4_ctx4099_t1"),
        # one user, a small tree of drafted tokens
        dict(_tree(1, 8191, 12, ragged=False), name="tree_b1_ctx8191_t12"),
        # a batch of long contexts, sixteen drafted tokens each
        dict(_tree(8, 32768, 16), name="tree_b8_ctx32768_t16"),
        # the widest tree under 7 queries per KV head, 3 bits without the sketch, fp16
        dict(_tree(2, 16001, 64, 28, 4, bits=3, qjl=False, dtype="f16"), name="tree_b2_ctx16001_t64_g7_3bit_f16"),
        # a drafted branch accepted by one user
        dict(_keep(1, 8191, 12), name="keep_b1_t12"),
        # a large batch of wide trees
        dict(_keep(64, 2047, 64), name="keep_b64_t64"),
        # four beams that share their prompt: only the generated tokens differ
        dict(_rows(4, 2100, lo=2000), name="rows_b4_last100"),
        # a batch of long contexts, some abandoned for copies of others
        dict(_rows(16, 32768), name="rows_b16_ctx32768"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("prompt", "prompt", "prompt", "tree", "tree", "tree", "keep", "rows"))
    q_heads, kv_heads = rng.choice(HEADS)
    bits, qjl = rng.choice((2, 3, 4, 4)), rng.random() < 0.7
    dtype = "f16" if rng.random() < 0.4 else "bf16"
    cut = rng.randrange(1 << 30)
    if kind == "prompt":
        layout = rng.choice(("batch", "batch", "chunk", "packed"))
        batch = _log_int(rng, 1, 24)
        s_kv = _log_int(rng, max(batch, 1), 32768)
        if layout == "batch":
            while batch > 1 and batch * q_heads * s_kv * s_kv // 2 > MOST_PAIRS:
                batch //= 2
            return _prompt(batch, s_kv, None, q_heads, kv_heads, dtype, "batch", rng.random() < 0.4, cut)
        if layout == "chunk":
            s_q = _log_int(rng, 1, s_kv)
            while batch > 1 and batch * q_heads * s_q * s_kv > MOST_PAIRS:
                batch //= 2
            return _prompt(batch, s_q, s_kv, q_heads, kv_heads, dtype, "batch", rng.random() < 0.4, cut)
        return _prompt(batch, s_kv, None, q_heads, kv_heads, dtype, "packed", False, cut)
    batch = _log_int(rng, 1, 64)
    ctx = _log_int(rng, 1, 65536)
    if kind == "tree":
        chain = rng.random() < 0.3
        nodes = _log_int(rng, 1, 512) if chain else _log_int(rng, 1, 64)
        tiles = -(-nodes * (q_heads // kv_heads) // D)
        while batch > 1 and batch * kv_heads * ctx * tiles > MOST_TREE:
            batch //= 2
        ctx = max(1, min(ctx, MOST_TREE // (batch * kv_heads * tiles)))
        return _tree(batch, ctx, nodes, q_heads, kv_heads, bits, qjl, dtype, chain, rng.random() < 0.7, cut)
    if kind == "keep":
        return _keep(batch, _log_int(rng, 1, 4096), _log_int(rng, 1, 64), kv_heads, bits, qjl, cut)
    batch = max(2, batch)
    ctx = max(1, min(ctx, MOST_ROWS // (2 * batch * kv_heads)))
    if rng.random() < 0.4:
        return _rows(batch, ctx, 0, _log_int(rng, 1, 2 * batch), kv_heads, bits, qjl, cut)
    return _rows(batch, ctx, rng.randrange(ctx) if rng.random() < 0.5 else 0, 0, kv_heads, bits, qjl, cut)


def _lengths(case):
    """Tokens of every sequence of a packed prompt: at least one each, cut at random."""
    rng = random.Random(case["cut"])
    marks = sorted(rng.sample(range(1, case["s_q"]), case["batch"] - 1)) if case["batch"] > 1 else []
    return [b - a for a, b in zip([0] + marks, marks + [case["s_q"]])]


def _starts(case):
    """Left padding of every batch entry of a prompt (the longest one has none; the chunk's own tokens are never padding)."""
    if not case["padded"]:
        return [0] * case["batch"]
    rng = random.Random(case["cut"])
    most = case["s_kv"] - 1 if case["s_q"] == case["s_kv"] else case["s_kv"] - case["s_q"]
    return [0] + [rng.randint(0, most) for _ in range(case["batch"] - 1)]


def _histories(case):
    """Tokens of every batch entry's history; the drafted tokens lie at ``ctx`` for all of them."""
    rng = random.Random(case["cut"])
    if case["kind"] == "keep":  # (behind the longest history there is room for what is kept)
        return [max(0, case["ctx"] - rng.randint(0, case["ctx"] // 4)) for _ in range(case["batch"])]
    if not case["ragged"]:
        return [case["ctx"]] * case["batch"]
    return [case["ctx"]] + [rng.randint(case["ctx"] // 2, case["ctx"]) for _ in range(case["batch"] - 1)]


def _tree_start(case):
    return case["ctx"] + (case["nodes"] if case["kind"] == "keep" else 0)


def _parents(case):
    """Random trees: node i hangs under one of the nodes before it, or directly under the history (-1)."""
    rng = random.Random(case["cut"] + 1)
    return [[rng.randint(max(-1, i - 9), i - 1) for i in range(case["nodes"])] for _ in range(case["batch"])]


def _paths(case):
    """The accepted nodes: from a random node up to its root, in ascending order."""
    rng, out = random.Random(case["cut"] + 2), []
    for up in _parents(case):
        node, path = rng.randint(len(up) // 2, len(up) - 1), []
        while node >= 0:
            path.append(node)
            node = up[node]
        out.append(path[::-1])
    return out


def _index(case):
    """Which row each row becomes: some rows stay, the others become copies of rows that stay."""
    rng = random.Random(case["cut"])
    if case["rows_out"]:
        return [rng.randrange(case["batch"]) for _ in range(case["rows_out"])]
    stay = sorted(rng.sample(range(case["batch"]), max(1, case["batch"] // 2)))
    return [b if b in stay else rng.choice(stay) for b in range(case["batch"])]


def _token_bytes(case):
    return 16 * (2 * case["bits"] - (1 if case["qjl"] else 0)) + 4 + (18 if case["qjl"] else 0)


def work(case):
    if case["kind"] == "prompt":
        if case["layout"] == "packed":
            lens = _lengths(case)
            pairs, tokens, queries = sum(n * (n + 1) // 2 for n in lens), sum(lens), sum(lens)
        else:
            n_q, n_kv = case["s_q"], case["s_kv"]
            pairs = tokens = 0
            for start in _starts(case):
                first = n_kv - n_q - start + 1  # keys that the first query sees (less than 1: it sees none)
                last = n_kv - start
                low = max(first, 1)
                pairs += (low + last) * (last - low + 1) // 2
                tokens += last
            queries = case["batch"] * n_q
        return {"bytes": 2 * D * (2 * queries * case["q_heads"] + 2 * tokens * case["kv_heads"]),
                "flops": 4 * D * pairs * case["q_heads"]}
    if case["kind"] == "tree":
        per = _token_bytes(case) * case["kv_heads"]
        nodes, rows = case["nodes"], case["batch"] * case["nodes"] * case["q_heads"]
        tokens = sum(_histories(case)) + case["batch"] * nodes
        inner = nodes * (nodes + 1) // 2 * case["batch"]
        if not case["chain"]:
            inner = 0
            for up in _parents(case):
                depth = []
                for p in up:
                    depth.append(1 if p < 0 else depth[p] + 1)
                inner += sum(depth)
        pairs = (sum(_histories(case)) * nodes + inner) * case["q_heads"]
        return {"bytes": tokens * per + 4 * D * rows,
                "flops": pairs * 2 * D * (3 if case["qjl"] else 2) + rows * 2 * D * D * (3 if case["qjl"] else 2)}
    if case["kind"] == "keep":
        return {"bytes": 2 * sum(len(p) for p in _paths(case)) * case["kv_heads"] * _token_bytes(case), "flops": 0}
    index = _index(case)
    if case["rows_out"]:
        reads, writes = len(set(index)), len(index)
    else:
        moved = [i for b, i in enumerate(index) if i != b]
        reads, writes = len(set(moved)), len(moved)
    return {"bytes": (reads + writes) * (case["ctx"] - case["lo"]) * case["kv_heads"] * _token_bytes(case), "flops": 0}


# ---------------------------------------------------------------------------------------------------- inputs
@functools.lru_cache(maxsize=8)
def _centres(bits):
    """Lloyd-Max centres for a coordinate of a uniform point on the unit sphere in 128 dimensions."""
    x = np.linspace(-1.0, 1.0, 32769)
    pdf = math.gamma(D / 2) / (math.sqrt(math.pi) * math.gamma((D - 1) / 2)) * np.power(1.0 - x * x, (D - 3) / 2)
    cdf = np.cumsum(pdf) * (x[1] - x[0])
    cdf /= cdf[-1]
    cdf[0], cdf[-1] = 0.0, 1.0
    centres = np.interp(np.linspace(0.0, 1.0, 2 ** bits + 2)[1:-1], cdf, x)
    for _ in range(200):
        edges = np.concatenate(([-1.0], (centres[:-1] + centres[1:]) / 2, [1.0]))
        moved = np.empty_like(centres)
        for i in range(len(centres)):
            inside = (x >= edges[i]) & (x <= edges[i + 1])
            moved[i] = np.trapezoid(x[inside] * pdf[inside], x[inside]) / np.trapezoid(pdf[inside], x[inside])
        done = np.max(np.abs(moved - centres)) < 1e-10
        centres = moved
        if done:
            break
    return centres.astype(np.float32)


@functools.lru_cache(maxsize=4)
def _rotation(seed):
    q, r = np.linalg.qr(np.random.default_rng(seed).standard_normal((D, D)))
    return (q * np.sign(np.diag(r))).astype(np.float32)


class _Tables:
    """The codec's tables of seed 0 as float32 tensors."""

    def __init__(self, bits, qjl, device):
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(device)
        self.bits, self.qjl, self.key_bits = bits, qjl, bits - 1 if qjl else bits
        self.cen_v, self.rot_v = put(_centres(bits)), put(_rotation(0))
        self.cen_k, self.rot_k = (put(_centres(self.key_bits)), put(_rotation(1))) if qjl else (self.cen_v, self.rot_v)
        self.sketch = torch.randn(D, D, generator=torch.Generator().manual_seed(31337)).to(device) if qjl else None


def _pack_bits(codes, bits):
    """[..., 128] codes -> [..., 16 * bits] bytes, least significant bit first."""
    planes = torch.stack([(codes >> i) & 1 for i in range(bits)], dim=-1).to(torch.uint8)
    planes = planes.reshape(*codes.shape[:-1], 16 * bits, 8)
    return (planes << torch.arange(8, device=codes.device, dtype=torch.uint8)).sum(-1, dtype=torch.uint8)


def _unpack_bits(data, bits):
    """[..., 16 * bits] bytes -> [..., 128] codes."""
    planes = (data.unsqueeze(-1) >> torch.arange(8, device=data.device, dtype=torch.uint8)) & 1
    planes = planes.reshape(*data.shape[:-1], D, bits)
    return (planes << torch.arange(bits, device=data.device, dtype=torch.uint8)).sum(-1, dtype=torch.uint8)


def _encode(x, centres):
    """Codes and fp16 norms of vectors given in the rotated frame, and what the codes leave of the unit vectors."""
    norms = x.norm(dim=-1, keepdim=True)
    unit = x / norms
    bounds = (centres[:-1] + centres[1:]) / 2
    codes = torch.bucketize(unit, bounds)
    return codes, norms.squeeze(-1).half(), unit - centres[codes]


def _streams(case, batch, tokens, gen, device):
    """The six streams of a layer's packed cache with ``tokens`` encoded tokens per row."""
    t = _Tables(case["bits"], case["qjl"], device)
    heads, cap = case["kv_heads"], max(8, -(-tokens // 8) * 8)
    u8 = lambda n: torch.zeros(batch, heads, cap, n, dtype=torch.uint8, device=device)
    f16 = lambda: torch.zeros(batch, heads, cap, dtype=torch.float16, device=device)
    s = {"k_codes": u8(16 * t.key_bits), "k_norms": f16(), "k_signs": u8(16) if t.qjl else None,
         "k_rnorms": f16() if t.qjl else None, "v_codes": u8(16 * t.bits), "v_norms": f16()}
    for b in range(batch):
        for lo in range(0, tokens, 16384):
            n = min(16384, tokens - lo)
            x = torch.randn(2, heads, n, D, generator=gen, device=device)
            x *= torch.exp(0.5 * torch.randn(2, heads, n, 1, generator=gen, device=device))
            codes, norms, rest = _encode(x[0], t.cen_k)
            s["k_codes"][b, :, lo:lo + n], s["k_norms"][b, :, lo:lo + n] = _pack_bits(codes.to(torch.uint8), t.key_bits), norms
            if t.qjl:
                rest = (rest @ t.rot_k) * x[0].norm(dim=-1, keepdim=True)
                signs = (rest @ t.sketch.T >= 0).to(torch.uint8)
                s["k_signs"][b, :, lo:lo + n], s["k_rnorms"][b, :, lo:lo + n] = _pack_bits(signs, 1), rest.norm(dim=-1).half()
            codes, norms, _ = _encode(x[1], t.cen_v)
            s["v_codes"][b, :, lo:lo + n], s["v_norms"][b, :, lo:lo + n] = _pack_bits(codes.to(torch.uint8), t.bits), norms
    return s, t


def _store(case, streams, batch, tokens, device):
    """The library's cache of one layer, holding the same tokens."""
    from tq_local_b200.runtime.codec import Codec
    from tq_local_b200.runtime.packed_store import PackedStore

    store = PackedStore(Codec.get(device, case["bits"], case["qjl"]), batch, case["kv_heads"], tokens)
    for name, data in streams.items():
        if data is not None:
            getattr(store, name).copy_(data)
    store.length = tokens
    return store


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=device).manual_seed(seed)
    put = lambda rows, dtype=torch.int32: torch.tensor(rows, dtype=dtype, device=device)
    if case["kind"] == "prompt":
        dtype, hq, hkv = DTYPES[case["dtype"]], case["q_heads"], case["kv_heads"]

        def dense(batch, n, heads, spread):  # [B, H, S, 128] as a model's projections leave it: heads side by side
            x = torch.empty(batch, n, heads, D, dtype=dtype, device=device)
            for b in range(batch):
                row = torch.randn(n, heads, D, generator=gen, device=device)
                if spread:
                    row *= torch.exp(0.5 * torch.randn(n, heads, 1, generator=gen, device=device))
                x[b] = row
            return x.transpose(1, 2)

        packed = case["layout"] == "packed"
        batch = 1 if packed else case["batch"]
        state = {"case": case, "q": dense(batch, case["s_q"], hq, False), "k": dense(batch, case["s_kv"], hkv, True),
                 "v": dense(batch, case["s_kv"], hkv, True)}
        if packed:
            lens = _lengths(case)
            for name in "qkv":
                state[name] = state[name][0].transpose(0, 1)  # [tokens, heads, 128]
            state["lens"], state["longest"] = lens, max(lens)
            state["cu_seqlens"] = put([0] + [sum(lens[:i + 1]) for i in range(len(lens))])
        elif case["padded"]:
            state["seq_start"] = put(_starts(case))
        return state
    if case["kind"] == "rows":
        streams, tables = _streams(case, case["batch"], case["ctx"], gen, device)
        state = {"case": case, "index": put(_index(case), torch.int64)}
        if own:
            state["store"] = _store(case, streams, case["batch"], case["ctx"], device)
        else:
            state["streams"] = streams
        return state
    tokens = _tree_start(case) + case["nodes"]
    streams, tables = _streams(case, case["batch"], tokens, gen, device)
    state = {"case": case, "lengths": put(_histories(case))}
    if case["kind"] == "tree":
        dtype = DTYPES[case["dtype"]]
        q = torch.randn(case["batch"], case["nodes"], case["q_heads"], D, generator=gen, device=device)
        state["q"] = q.to(dtype).transpose(1, 2)
        if not case["chain"]:
            masks = []
            for up in _parents(case):
                rows = []
                for i, p in enumerate(up):
                    rows.append((rows[p] if p >= 0 else 0) | 1 << i)
                masks.append([m - (1 << 64) if m >> 63 else m for m in rows])
            state["tree_mask"] = put(masks, torch.int64)
    else:
        paths = _paths(case)
        most = max(len(p) for p in paths)
        state["path"] = put([p + [0] * (most - len(p)) for p in paths])
        state["counts"] = put([len(p) for p in paths])
    if own:
        state["store"] = _store(case, streams, case["batch"], tokens, device)
    else:
        state["streams"], state["tables"] = streams, tables
    return state


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_attention(q, k, v, first, offset):
    """q [H, n, 128], k / v [Hkv, m, 128] in 32 bits; query i sees keys [first, i + offset]."""
    hkv, m, n = k.shape[0], k.shape[1], q.shape[1]
    q = q.reshape(hkv, -1, n, D)
    out = torch.empty_like(q)
    step = max(1, (1 << 28) // (q.shape[1] * max(m, 1)))  # queries at a time: a gigabyte of logits
    cols = torch.arange(m, device=q.device)
    for h in range(hkv):
        for lo in range(0, n, step):
            rows = torch.arange(lo, min(lo + step, n), device=q.device).unsqueeze(1)
            top = min(m, lo + step + offset)
            if top <= first:
                out[h, :, lo:lo + step] = 0
                continue
            logits = (q[h, :, lo:lo + step] @ k[h, :top].T) * (1.0 / math.sqrt(D))
            logits.masked_fill_((cols[:top] > rows + offset) | (cols[:top] < first), -math.inf)
            peak = logits.max(dim=-1, keepdim=True).values
            weights = logits.sub_(torch.where(peak == -math.inf, 0.0, peak)).exp_()
            total = weights.sum(dim=-1, keepdim=True)
            out[h, :, lo:lo + step] = (weights @ v[h, :top]) / torch.where(total == 0, 1.0, total)
    return out.reshape(-1, n, D)


def _plain_prompt(state):
    q, k, v = state["q"], state["k"], state["v"]
    out = torch.empty_like(q)
    if "lens" in state:
        at = 0
        for n in state["lens"]:
            part = [x[at:at + n].transpose(0, 1).float() for x in (q, k, v)]
            out[at:at + n] = _plain_attention(*part, 0, 0).transpose(0, 1).to(q.dtype)
            at += n
        return out
    starts = _starts(state["case"])
    for b in range(q.shape[0]):
        out[b] = _plain_attention(q[b].float(), k[b].float(), v[b].float(), starts[b], k.shape[2] - q.shape[2]).to(q.dtype)
    return out


def _plain_tree(state):
    case, s, t, q = state["case"], state["streams"], state["tables"], state["q"]
    nodes, start, out = case["nodes"], _tree_start(case), torch.empty_like(q)
    at = torch.arange(nodes, device=q.device)
    for b, n in enumerate(_histories(case)):
        if case["chain"]:
            inner = at.unsqueeze(0) <= at.unsqueeze(1)
        else:
            inner = (state["tree_mask"][b].unsqueeze(1) >> at) & 1 == 1
        for h in range(case["kv_heads"]):
            rows = torch.cat((torch.arange(n, device=q.device), start + at))
            take = lambda name: s[name][b, h].index_select(0, rows)
            g = q.shape[1] // case["kv_heads"]
            x = q[b, h * g:(h + 1) * g].float().reshape(-1, D)  # (head, node) rows
            keys = t.cen_k[_unpack_bits(take("k_codes"), t.key_bits).int()]
            logits = (x @ t.rot_k.T) @ keys.T * take("k_norms").float()
            if t.qjl:
                signs = _unpack_bits(take("k_signs"), 1).float() * 2 - 1
                logits += (x @ t.sketch.T) @ signs.T * (take("k_rnorms").float() * SKETCH)
            logits *= 1.0 / math.sqrt(D)
            logits.view(g, nodes, -1)[:, :, n:].masked_fill_(~inner, -math.inf)
            weights = (logits - logits.max(dim=-1, keepdim=True).values).exp()
            values = t.cen_v[_unpack_bits(take("v_codes"), t.bits).int()] * take("v_norms").float().unsqueeze(-1)
            y = (weights @ values) / weights.sum(dim=-1, keepdim=True) @ t.rot_v
            out[b, h * g:(h + 1) * g] = y.reshape(g, nodes, D).to(q.dtype)
    return out


def _bits(x):
    """A stream as whole numbers: what is moved arrives bit for bit."""
    return x.view(torch.int16) if x.dtype == torch.float16 else x


def _plain_keep(state):
    case, s, lengths = state["case"], state["streams"], state["lengths"]
    path, counts = state["path"], state["counts"]
    nth = torch.arange(path.shape[1], device=path.device)
    b, i = torch.nonzero(nth < counts.unsqueeze(1), as_tuple=True)
    src, dst = _tree_start(case) + path[b, i], lengths[b] + i
    for data in s.values():
        if data is not None:
            data[b, :, dst] = data[b, :, src]
    return [_bits(x) for x in s.values() if x is not None] + [lengths + counts]


def _plain_rows(state):
    case, s, index = state["case"], state["streams"], state["index"]
    out = []
    for data in s.values():
        if data is None:
            continue
        if case["rows_out"]:
            out.append(_bits(data[:, :, :case["ctx"]].index_select(0, index)))
        else:
            moved = torch.nonzero(index != torch.arange(len(index), device=index.device)).squeeze(1)
            data[moved, :, case["lo"]:case["ctx"]] = data[index[moved], :, case["lo"]:case["ctx"]]
            out.append(_bits(data[:, :, :case["ctx"]]))
    return out


def _cache(store, tokens):
    """The streams that hold something, in the order of the plain forms."""
    names = ("k_codes", "k_norms", "k_signs", "k_rnorms", "v_codes", "v_norms")
    return [_bits(x[:, :, :tokens]) for x in (getattr(store, name) for name in names) if x is not None]


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"prompt": _plain_prompt, "tree": _plain_tree, "keep": _plain_keep, "rows": _plain_rows}[kind](state)
    if kind == "prompt":
        from tq_local_b200.runtime.prompt_attention import prompt_attention, prompt_attention_packed

        if case["layout"] == "packed":
            return prompt_attention_packed(state["q"], state["k"], state["v"], state["cu_seqlens"], state["longest"])
        return prompt_attention(state["q"], state["k"], state["v"], seq_start=state.get("seq_start"))
    store = state["store"]
    if kind == "tree":
        return store.tree_attn(state["q"], state.get("tree_mask"), tree_start=_tree_start(case), lengths=state["lengths"])
    if kind == "keep":
        lengths = store.keep_tokens(state["path"], state["counts"], tree_start=_tree_start(case), lengths=state["lengths"])
        return _cache(store, store.capacity) + [lengths]
    if case["rows_out"]:
        return _cache(store.take_rows(state["index"]), case["ctx"])
    store.select_rows(state["index"], case["lo"])
    return _cache(store, case["ctx"])


# ---------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    if case["kind"] not in ("prompt", "tree"):
        return None
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    return _exact_prompt(case, state) if case["kind"] == "prompt" else _exact_tree(case, state)


def _exact_softmax(scores, seen):
    """Softmax over the seen entries of every row in 64 bits; rows that see nothing get zeros."""
    scores = torch.where(seen, scores, torch.full((), -math.inf, dtype=scores.dtype, device=scores.device))
    best = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.nan_to_num(best, neginf=0.0))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-300)


def _exact_prompt(case, state):
    q, k, v = state["q"], state["k"], state["v"]
    if 4 * D * case["q_heads"] * case["batch"] * case["s_q"] * case["s_kv"] > 1 << 46 and case["layout"] != "packed":
        return None
    group = case["q_heads"] // case["kv_heads"]
    if case["layout"] == "packed":
        spans, at = [], 0
        for n in state["lens"]:
            spans.append((q[at:at + n], k[at:at + n], v[at:at + n], 0))
            at += n
    else:
        by_token = lambda x, b: x[b].permute(1, 0, 2)
        spans = [(by_token(q, b), by_token(k, b), by_token(v, b), s) for b, s in enumerate(_starts(case))]
    results = []
    for qs, ks, vs, start in spans:  # [tokens, heads, 128]
        n, m = qs.shape[0], ks.shape[0]
        res = torch.empty(qs.shape, dtype=torch.float64, device=qs.device)
        for head in range(case["q_heads"]):
            kk, vv = ks[:, head // group].double(), vs[:, head // group].double()
            for lo in range(0, n, 2048):
                hi = min(lo + 2048, n)
                end = m - n + hi
                pos = torch.arange(m - n + lo, end, device=qs.device)
                key = torch.arange(end, device=qs.device)
                seen = (key[None, :] <= pos[:, None]) & (key[None, :] >= start)
                w = _exact_softmax(qs[lo:hi, head].double() @ kk[:end].mT / math.sqrt(D), seen)
                res[lo:hi, head] = w @ vv[:end]
        results.append(res)
    if case["layout"] == "packed":
        return torch.cat(results)
    return torch.stack(results).transpose(1, 2)


def _exact_tree(case, state):
    """Keys and values brought back to their own frame in 64 bits, then ordinary attention, a node at a time over its path."""
    t, s, q = state["tables"], state["streams"], state["q"]
    group, start = case["q_heads"] // case["kv_heads"], _tree_start(case)
    res = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    parents = _parents(case)
    for b, n in enumerate(_histories(case)):
        visible = torch.zeros(case["nodes"], n + case["nodes"], dtype=torch.bool)
        visible[:, :n] = True
        for i in range(case["nodes"]):
            if case["chain"]:
                visible[i, n:n + i + 1] = True
                continue
            j = i
            while j >= 0:
                visible[i, n + j] = True
                j = parents[b][j]
        visible = visible.to(q.device)
        for h in range(case["kv_heads"]):
            def tokens(name):
                x = s[name][b, h]
                return torch.cat((x[:n], x[start:start + case["nodes"]]))

            keys = t.cen_k.double()[_unpack_bits(tokens("k_codes"), t.key_bits).long()] @ t.rot_k.double()
            keys *= tokens("k_norms").double()[:, None]
            if t.qjl:
                sign = torch.where(_unpack_bits(tokens("k_signs"), 1) > 0, 1.0, -1.0).double()
                keys += sign @ t.sketch.double() * (tokens("k_rnorms").double() * SKETCH)[:, None]
            values = t.cen_v.double()[_unpack_bits(tokens("v_codes"), t.bits).long()] @ t.rot_v.double()
            values *= tokens("v_norms").double()[:, None]
            for head in range(h * group, (h + 1) * group):
                scores = q[b, head].double() @ keys.T / math.sqrt(D)
                res[b, head] = _exact_softmax(scores, visible) @ values
    return res

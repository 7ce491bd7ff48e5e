"""GPU: the row offsets of a left-padded cache when its rows move and calls are recorded."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def padded_store(starts):
    from tq_local_b200.runtime.codec import Codec
    from tq_local_b200.runtime.packed_store import PackedStore

    store = PackedStore(Codec.get(torch.device("cuda", torch.cuda.current_device()), 4, True), len(starts), 2, 300)
    gen = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(len(starts), 2, 300, 128, device="cuda", generator=gen).to(BF16) for _ in range(2))
    store.pack(k, v)
    store.set_seq_start(torch.tensor(starts, dtype=torch.int32, device="cuda"))
    return store


def recorded(f):
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    return graph, out


def test_what_was_recorded_follows_the_rows():
    """Attention that was recorded before rows moved attends the tokens that they have after it."""
    store = padded_store([0, 100, 250])
    store.select_rows(torch.arange(3, device="cuda"))  # the offsets are the cache's own from here on
    held = store._seq_start
    q = torch.randn(3, 8, 1, 128, device="cuda", dtype=BF16)
    one, out_one = recorded(lambda: store.decode_attn(q))
    tree, out_tree = recorded(lambda: store.tree_attn(q))
    store.select_rows(torch.tensor([2, 0, 1], device="cuda"))
    one.replay(), tree.replay()
    assert store._seq_start.tolist() == [250, 0, 100] and store._seq_start is held
    assert torch.equal(out_one, store.decode_attn(q)) and torch.equal(out_tree, store.tree_attn(q))


def test_rows_with_offsets_of_the_caches_own_are_recorded():
    store = padded_store([0, 100, 250]).take_rows(torch.arange(3, device="cuda"))
    index = torch.tensor([1, 2, 0], device="cuda")
    before = [t.clone() for t in store.streams()]
    store.select_rows(index)
    graph, _ = recorded(lambda: store.select_rows(index))  # once more before it is recorded
    graph.replay(), graph.replay()
    moved = index[index][index][index]
    assert store._seq_start.tolist() == [[0, 100, 250][i] for i in moved.tolist()]
    assert all(torch.equal(now.view(torch.uint8)[:, :, :300], was.view(torch.uint8)[moved][:, :, :300]) for was, now in zip(before, store.streams()))


def test_a_tensor_that_the_caller_keeps_is_not_written():
    store = padded_store([0, 100, 250])
    starts = store._seq_start
    store.select_rows(torch.tensor([2, 2, 2], device="cuda"))
    assert starts.tolist() == [0, 100, 250] and store._seq_start.tolist() == [250, 250, 250]
    store.set_seq_start(starts)
    store.select_rows(torch.tensor([1, 1, 1], device="cuda"))
    assert starts.tolist() == [0, 100, 250] and store._seq_start.tolist() == [100, 100, 100]

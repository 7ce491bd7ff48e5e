"""CPU: what a layer does with a bound tree of drafted tokens apart from attending."""

from __future__ import annotations

import pytest
import torch


def layer_of(mask, lengths):
    from tq_local_b200.runtime.packed_qmse_cache import PackedMSELayer

    layer = PackedMSELayer(bits=4, use_qjl_keys=True, quantize_decode=True)
    layer._tree = (mask, lengths)
    return layer


@pytest.mark.parametrize("rows", [[2, 0, 0], [1], [0, 0, 1, 1, 2, 2]])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_masks_and_lengths_follow_their_rows(rows, dtype):
    mask, lengths = torch.arange(12).view(3, 4), torch.tensor([5, 6, 7], dtype=torch.int32)
    index = torch.tensor(rows, dtype=dtype)
    for move in ("batch_select_indices", "reorder_cache"):
        layer = layer_of(mask, lengths)
        getattr(layer, move)(index)
        assert torch.equal(layer._tree[0], mask[rows]) and torch.equal(layer._tree[1], lengths[rows])
        layer = layer_of(mask[0], None)  # one mask for all rows, histories of one length
        getattr(layer, move)(index)
        assert torch.equal(layer._tree[0], mask[0]) and layer._tree[1] is None
        layer = layer_of(None, lengths)
        getattr(layer, move)(index)
        assert layer._tree[0] is None and torch.equal(layer._tree[1], lengths[rows])
    layer.unbind_tree()
    layer.reorder_cache(index)
    assert layer._tree is None


def test_a_static_decode_does_not_begin_under_a_bound_tree():
    """Its steps would attend every row up to the longest and none of the mask."""
    from types import SimpleNamespace

    layer = layer_of(None, torch.tensor([5], dtype=torch.int32))
    layer.store = SimpleNamespace(length=5, reserve=lambda n: None)
    pos = torch.zeros((), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="unbind_tree"):
        layer.begin_static_decode(pos, 4)
    assert layer._static_pos is None
    layer.unbind_tree()
    layer.begin_static_decode(pos, 4)
    assert layer._static_pos is pos
    with pytest.raises(RuntimeError):
        layer.bind_tree(None)


def test_layers_of_float32_models_are_refused_before_a_step_has_changed_them():
    from types import SimpleNamespace

    layer = layer_of(None, None)
    layer.unbind_tree()
    layer.store = SimpleNamespace(length=5)
    layer.dtype = torch.float32
    with pytest.raises(NotImplementedError, match="float32"):
        layer.bind_tree(None)
    assert layer._tree is None
    for dtype in (torch.float16, torch.bfloat16):
        layer.dtype = dtype
        layer.bind_tree(None)
        assert layer._tree == (None, None)

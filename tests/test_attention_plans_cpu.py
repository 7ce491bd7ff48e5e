"""CPU: how the attention kernels cut their work, as far as the sizes of their scratch tell."""

from __future__ import annotations

import ctypes as C

import pytest


def context(sm_count: int, qjl: bool = True):
    """The first fields of a context - device, bits, key bits, sketch, SMs -, which is what sizes are told from."""
    return (C.c_int32 * 256)(0, 4, 3 if qjl else 4, int(qjl), sm_count)


@pytest.mark.parametrize("qjl", [True, False])
@pytest.mark.parametrize("batch,q_heads,kv_heads,nodes,start", [(1, 32, 8, 12, 8191), (4, 32, 8, 1, 4099), (1, 4, 1, 1, 300), (3, 28, 4, 64, 5000)])
def test_a_drafted_token_call_has_a_cta_on_any_number_of_sms(qjl, batch, q_heads, kv_heads, nodes, start):
    """Scratch for a piece of every tile and one more of every CTA, of which there is one an SM."""
    from tq_local_b200.runtime import ffi

    group = q_heads // kv_heads
    positions = 128 // group
    tiles, rows = -(-nodes // positions) * batch * kv_heads, min(nodes, positions) * group
    up = lambda n: -(-n // 256) * 256
    for sms in (1, 2, 3, 4, 8, 9, 16, 132, 148):
        pieces = tiles + min(sms, tiles * -(-(start + nodes + 21) // 128))
        want = up(tiles * rows * (512 if qjl else 256)) + up(pieces * rows * 8) + up(pieces * rows * 512)
        assert ffi.lib().tq_tree_workspace_bytes(context(sms, qjl), batch, q_heads, kv_heads, nodes, start) == want

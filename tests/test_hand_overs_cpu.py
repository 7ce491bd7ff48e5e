"""CPU: hand-overs between threads that no run on a GPU can be relied on to show, from the sources."""

from __future__ import annotations

import os
import re

from tq_local_b200.build import CSRC


def source(name: str) -> str:
    return open(os.path.join(CSRC, name)).read()


def exchange_goes_wrong(copies: int, blocks: int = 6) -> bool:
    """Two warps tell each other a number per block: store it (to copy ``block % copies``), meet at a barrier, load the other's.
    Whether, in some order of their steps, a warp loads what belongs to another block."""
    start = ((0, 0), (0, 0), ((None,) * copies,) * 2)  # of each warp: block, step (0 store, 1 at the barrier, 2 load); what it has stored
    seen, todo = {start}, [start]
    while todo:
        a, b, held = state = todo.pop()
        warps = (a, b)
        nexts = []
        if a[1] == 1 and b[1] == 1:  # both at the barrier: they pass
            assert a[0] == b[0]
            nexts.append(((a[0], 2), (b[0], 2), held))
        for w in (0, 1):
            block, step = warps[w]
            if block == blocks or step == 1:
                continue
            if step == 0:
                mine = list(held[w])
                mine[block % copies] = block
                other, new = held[1 - w], (block, 1)
                stored = (tuple(mine), other) if w == 0 else (other, tuple(mine))
            else:
                if held[1 - w][block % copies] != block:
                    return True
                new, stored = (block + 1, 0), held
            nexts.append((new, b, stored) if w == 0 else (a, new, stored))
        for s in nexts:
            if s not in seen:
                seen.add(s), todo.append(s)
    return False


def test_halves_of_a_row_tell_each_other_the_maximum_of_the_same_block():
    """Nothing but the barrier between store and load orders the two warps: the next block's logits do not wait for this block's weights."""
    text = source("tq_tree.cu")
    assert exchange_goes_wrong(1) and not exchange_goes_wrong(2)
    sizes = re.search(r"__shared__ float s_half((?:\[\w+\])+);", text).group(1)
    block_loop = text[text.index("for (int k = g.k; k < g.k_end; ++k, ++n) {\n                const uint32_t t_s"):text.index("float l0, l1;")]
    uses = re.findall(r"s_half((?:\[[^\]]+\])+)", block_loop)
    assert len(uses) == 2
    copies = 2 if sizes == "[2][2][kUmmaRows]" and all(u.startswith("[n & 1]") for u in uses) else 1
    assert not exchange_goes_wrong(copies)


def test_waits_for_tensor_memory_name_the_registers_that_arrive():
    """A load from tensor memory is asynchronous: what does arithmetic on its registers must depend on the statement that waits, or the compiler may
    move it ahead of that."""
    found = 0
    for name in sorted(os.listdir(CSRC)):
        for statement in re.findall(r"asm volatile\(((?:[^;\"]|\"(?:[^\"\\]|\\.)*\")*)\);", source(name)):
            if "tcgen05.wait::ld" in statement:
                found += 1
                assert "tcgen05.ld." in statement or '"+r"' in statement, (name, statement)
    assert found == 2


def test_every_shared_piece_has_a_caller():
    """Functions of the headers, each named at least once outside its own definition."""
    files = {name: re.sub(r"//[^\n]*", "", source(name)) for name in os.listdir(CSRC) if name.endswith((".cu", ".cuh"))}
    for name in ("tq_attn_tc.cuh", "tq_umma.cuh", "tq_bulk.cuh"):
        for function in set(re.findall(r"__forceinline__ [\w:]+ \*?(\w+)\(", files[name])):
            uses = sum(len(re.findall(rf"\b{function}\b", text)) for text in files.values())
            defined = len(re.findall(rf"__forceinline__ [\w:]+ \*?{function}\(", files[name]))
            assert uses > defined, (name, function)


def test_copies_and_products_end_before_their_cta():
    """A thread whose wait ran out waits for nothing more, but before the CTA ends what it set going is waited for: a copy that lands later would land
    in another CTA's shared memory."""
    for name, copies in (("tq_prompt.cu", ("mbar_wait(bar_full", "mbar_wait(bar_q")), ("tq_tree.cu", ("mbar_wait(bar_raw",))):
        text = source(name)
        end = text[text.index("if (__syncthreads_or(lost)) {"):]
        end = end[:end.index("tcgen05.dealloc")]
        for wait in copies + ("umma_commit(bar", "mbar_wait(bar"):
            assert wait in end, (name, wait)
    assert re.search(r"if \(lost\) \{[^}]*mbar_wait\(bar_image, 0\), mbar_wait\(bar_mma, 0\);", source("tq_tree.cu"))

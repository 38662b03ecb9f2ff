"""The source of the 8-bit products' kernels: what a test on the GPU cannot show, as it may work by the luck of a compilation.

``tcgen05.ld``, ``tcgen05.wait::ld`` and ``bar.red`` are ``.aligned``: undefined unless all lanes of a warp execute them
together. So in the code that reads the sums from tensor memory a lane never leaves a turn of a loop by itself, what lanes
do apart ends in ``__syncwarp()`` before the next such instruction, and a wait whose outcome decides which of them come
next is one decision of the warp."""
from __future__ import annotations

import re
from pathlib import Path

SOURCE = Path(__file__).resolve().parent.parent / "nvcr_b200" / "csrc" / "k_token_bytes.cu"


def block_at(text, start):
    """The braces from the first one at or after `start` to the one that closes it."""
    first = text.index("{", start)
    depth = 0
    for at in range(first, len(text)):
        depth += {"{": 1, "}": -1}.get(text[at], 0)
        if depth == 0:
            return text[first:at + 1]
    raise AssertionError("braces that do not close")


def without_comments(text):
    return re.sub(r"//[^\n]*", "", text)


def test_lanes_meet_before_tensor_memory_is_read():
    text = without_comments(SOURCE.read_text())
    body = block_at(text, re.search(r"\bvoid store_tile\(", text).end())
    before, loop = body[:body.index("for (int column")], block_at(body, body.index("for (int column"))
    assert before.index("__syncwarp()") < before.index("tmem_load16")
    assert "tmem_load_wait" in loop and "tmem_load16" in loop
    for word in ("continue", "break", "return;"):
        assert word not in loop, word
    assert re.search(r"__syncwarp\(\);\s*\}$", loop)


def test_barriers_of_the_epilogue_take_whole_warps():
    text = without_comments(SOURCE.read_text())
    body = block_at(text, re.search(r"\bbool epilogue_any\(", text).end())
    assert body.index("__syncwarp()") < body.index("bar.red")


def test_a_warp_takes_one_decision_about_a_tile():
    """Lanes poll for themselves and may run out of time one by one."""
    text = re.sub(r"\s+", "", without_comments(SOURCE.read_text()))
    waits = re.findall(r".{0,40}(?:barrier_wait|barrier_wait_for)\(smem_address\(&tail\.tmem_full", text)
    assert len(waits) == 2
    for wait in waits:
        assert "__all_sync(0xffffffffu," in wait, wait

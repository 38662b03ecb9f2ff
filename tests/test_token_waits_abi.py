"""What the self-test of the 8-bit products' waits refuses (no GPU)."""
from __future__ import annotations


def test_the_limit_and_the_block_are_checked(built_library):
    from nvcr_b200.executor import library

    for limit, block in ((0, 0), (4001, 0), (20, -1)):
        assert library().nvcr_sm100_token_test_wait_timeout(limit, block) == 1  # NVCR_SM100_INVALID_ARGUMENT

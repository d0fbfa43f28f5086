"""Step tables: memory that is read and written in one call is refused on the host, before any launch."""

from __future__ import annotations

import ctypes

import pytest

from vllm_ascend_kvcompress import _native as N

R, TOKENS, BLOCKS = 3, 10, 4
SIZES = {"computed": 8 * R, "scheduled": 4 * R, "offsets": 8 * R, "pages": 4 * (2 * 9 + 5), "starts": 4 * (R + 1),
         "lens": 4 * R, "positions": 8 * TOKENS, "slots": 8 * TOKENS, "request": 4 * TOKENS, "blocks": 4 * R * BLOCKS}
INPUTS = ("computed", "scheduled", "offsets", "pages")


def call(at):
    p = {k: ctypes.c_void_p(v) for k, v in at.items()}
    return N.lib().kvc_step_tables(p["computed"], 8, p["scheduled"], 4, p["offsets"], R, p["pages"], 4, 9, 5, 1, TOKENS,
                                   BLOCKS, p["starts"], p["lens"], p["positions"], p["slots"], p["request"], p["blocks"],
                                   None, None)


def apart():
    """Made-up addresses, each array right behind the one before it."""
    at, end = {}, 0x10000
    for k, size in SIZES.items():
        at[k], end = end, end + size
    return at


@pytest.mark.parametrize("one", [k for k in SIZES if k not in INPUTS])
@pytest.mark.parametrize("other", list(SIZES))
def test_tables_may_not_share_memory_with_inputs_or_each_other(one, other):
    if one == other:
        return
    at = apart()
    for start in (at[other], at[other] + SIZES[other] - 4, at[other] - SIZES[one] + 4):
        assert call({**at, one: start}) == -22


def test_inputs_may_share_memory_and_arrays_may_touch():
    """Without a GPU the launch itself fails, with another status than a refusal."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("the addresses are made up: only for hosts where nothing can be launched")
    at = apart()
    assert call(at) not in (-22, -14, -95)
    assert call({**at, "offsets": at["computed"], "pages": at["scheduled"]}) not in (-22, -14, -95)

"""Paged attention and step tables at their edges: values that are not finite, small weights, counts and ids past a range."""

from __future__ import annotations

import math

import pytest
import torch

import serving_reference as R
from test_gpu_serving import BF16, FP16, attend, attention_case, check_attention, ints  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- values that are not finite --------------------------------------------------------------------


@pytest.mark.parametrize("bad", [math.nan, -math.inf])
@pytest.mark.parametrize("dim,kvh,short,long", [(64, 2, 3, 16), (128, 2, 3, 16), (256, 2, 3, 16)])
def test_tiles_of_one_and_two_halves_in_turn_with_anything_past_the_lengths(bad, dim, kvh, short, long):
    """Several tiles a CTA, those of few rows beside those of many, each with a partly masked block to clear."""
    new = [short if i % 2 else long for i in range(700)]
    lens = [n + (29 * i) % 150 for i, n in enumerate(new)]
    c = attention_case(new, lens, 16 * kvh, kvh, dim, BF16)
    for r, n in enumerate(lens):
        if n % 128:
            last = c["table"][r, (n - 1) // 128]
            c["kc"][last, (n - 1) % 128 + 1:] = bad
            c["vc"][last, (n - 1) % 128 + 1:] = bad
    got = attend(c)
    check_attention(c, got)
    again = attend(c)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])

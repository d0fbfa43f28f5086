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


@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, BF16), (256, BF16)])
@pytest.mark.parametrize("longest", [1, 64])  # 1: the kernel of single tokens
@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("where", ["query", "key"])
def test_nan_scores_answer_nan(dim, dtype, longest, window, where):
    """Rows whose every seen score is NaN, beside masked keys, in prompts shorter and longer than a block of keys."""
    new = [40, 1, 200, 3]
    lens = [40, 1, 200, 90]
    c = attention_case(new, lens, 4, 2, dim, dtype)
    want = torch.zeros(sum(new), 4, dtype=torch.bool)
    for r, (n, length) in enumerate(zip(new, lens)):
        first = c["starts"][r]
        if where == "query":  # one head of the request's second (or only) new token
            row = first + min(1, n - 1)
            c["q"][row, 2, 5] = math.nan
            want[row, 2] = True
        else:  # key 0 of the second KV head, which the first new token of a prompt sees alone
            c["kc"][c["table"][r, 0], 0, 1, 7] = math.nan
            for j in range(n):
                p = length - n + j
                want[first + j, 2:] = window == 0 or p < window
    out, lse = (x.cpu() for x in attend(c, window=window, max_query_len=longest))
    assert torch.equal(lse.isnan(), want)
    assert torch.equal(out.isnan(), want[..., None].expand_as(out))
    clean = dict(c, q=c["q"].nan_to_num(), kc=c["kc"].nan_to_num())
    fine = [x.cpu() for x in attend(clean, window=window, max_query_len=longest)]
    out[want], lse[want] = fine[0][want], fine[1][want]  # the other rows are as they are without the NaN
    check_attention(clean, (out, lse), window)


@pytest.mark.parametrize("longest", [1, 64])
def test_nan_scores_in_a_part_of_a_request_cut_over_the_gpu(longest):
    """The part that holds the NaN key goes through the workspace."""
    c = attention_case([2], [9001], 4, 1, 128, BF16)
    for at in (0, 4500, 8990):
        d = dict(c, kc=c["kc"].clone())
        d["kc"][c["table"][0, at // 128], at % 128, 0, 3] = math.nan
        out, lse = attend(d, max_query_len=longest)
        assert out.isnan().all() and lse.isnan().all()
    q = dict(c, q=c["q"].clone())
    q["q"][1, 3, 0] = math.nan
    out, lse = (x.cpu() for x in attend(q, max_query_len=longest))
    assert out[1, 3].isnan().all() and lse[1, 3].isnan()
    assert out.isnan().sum() == 128 and lse.isnan().sum() == 1

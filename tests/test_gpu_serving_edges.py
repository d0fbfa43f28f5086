"""Paged attention and step tables at their edges: values that are not finite, small weights, counts and ids past a range."""

from __future__ import annotations

import math

import pytest
import torch

import serving_reference as R
from test_gpu_serving import BF16, FP16, attend, attention_case, check_attention, ints
from vllm_ascend_kvcompress import _native as N
from vllm_ascend_kvcompress.methods.triattention import kernels as K

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


# ---- fp16 weights far below the largest ------------------------------------------------------------


def bits_below(kind, n, g):
    """log2 of each key's weight against the largest, as how far below it lies."""
    i = torch.arange(n, dtype=torch.float64)
    if kind == "spread":
        return 40 * torch.rand(n, generator=g, dtype=torch.float64)
    if kind == "rising":  # every part has a new maximum
        return 60 * (1 - i / n)
    if kind == "plateaus":  # 64 weights alike, then 64 that are 3 bits higher, over and over
        return 3.0 * (7 - (i // 64) % 8) + 24.0 * (n - 1 - i).div(512, rounding_mode="floor")
    far = torch.full((n,), float(kind), dtype=torch.float64)  # one strong first token, all others alike
    far[0] = 0
    return far


@pytest.mark.parametrize("kind,n", [("0", 5000), ("12", 65536), ("20", 65536), ("25.1", 65536), ("25.1", 700), ("28", 65536),
                                    ("spread", 20000), ("rising", 9000), ("plateaus", 4100)])
@pytest.mark.parametrize("dim,new", [(64, 1), (128, 1), (256, 1), (64, 30), (128, 30), (256, 30)])
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_many_small_weights_beside_a_strong_one(kind, n, dim, new, dtype):
    """The first token's value is 0, so the others' weights are all of the output.  150 requests read one cache, so
    that most are not cut into parts, each with a largest weight of its own.

    Bound of an output, relative to sum w |v|: half a step of the type for each weight and for the output; products
    and sums in fp32, of up to n / 16 terms one after another (2^-23 each); the exponential and the scores (here one
    product of at most 60 bits, so 2^-23 * 60 of a weight, and 2^-18 for the rest).  And of weights under fp16's
    normal range half of its smallest subnormal, 2^-25: 64 of them beside the first token, whose weight is 2^3 (128
    beside 2^7 at head_dim 256), and any others as 2^9 of what they are against it, 2^-22 + n 2^-34 of the row's
    sum; in blocks of mixed weights, which average 2^-10 at least, 2^-15 of it.
    """
    g = torch.Generator().manual_seed(n + dim)
    heads, blocks = 4, -(-n // 128)
    q = torch.zeros(new, heads, dim)
    q[..., 3] = 4.0
    q[:, 1, 3], q[:, 2, 3] = 3.0, 3.5
    kc = torch.zeros(blocks * 128, dim)
    kc[:n, 3] = (-bits_below(kind, n, g) * math.log(2) / 4).float()
    vc = 0.5 + torch.rand(blocks * 128, dim, generator=g)
    vc[0] = 0
    q, kc, vc = (x.to(dtype).cuda() for x in (q, kc, vc))
    many = 150
    out, lse = attend({"q": q.repeat(many, 1, 1), "kc": kc.view(blocks, 128, 1, dim), "vc": vc.view(blocks, 128, 1, dim),
                       "table": torch.arange(blocks, dtype=torch.int32).repeat(many, 1),
                       "starts": [new * i for i in range(many + 1)], "lens": [n] * many, "longest": new}, scale=1.0)
    out, lse = out.unflatten(0, (many, new)), lse.unflatten(0, (many, new))
    score = (q[..., 3].double().flatten()[:, None] * kc[:n, 3].double()).unflatten(0, (new, heads))
    last = torch.arange(n - new, n, device="cuda")[:, None, None]
    score = score.masked_fill(torch.arange(n, device="cuda") > last, -math.inf)
    w = torch.softmax(score, -1)
    want = w @ vc[:n].double()
    u = torch.finfo(dtype).eps / 2
    bound = want * (2 * u + 60 * 2.0 ** -23 + 2.0 ** -18 + n / 16 * 2.0 ** -23)
    coarse = 2.0 ** -22 + n * 2.0 ** -34 if kind[0].isdigit() else 2.0 ** -15
    bound += (coarse if dtype == FP16 else 0) * vc[:n].double().amax(0) + torch.finfo(dtype).tiny * 2 * u
    over = (out.double() - want).abs() - bound
    assert (over <= 0).all(), f"{over.max().item():.3g} past its bound where {want.mean().item():.3g} is usual"
    off = (lse.double() - torch.logsumexp(score, -1)).abs()
    assert (off <= 2.0 ** -16 + n / 16 * 2.0 ** -23).all()


# ---- bounds and counts that are wrong --------------------------------------------------------------


@pytest.mark.parametrize("new", [[1, 5, 0, 40], [1, 1, 1, 1]])
def test_a_longest_length_of_zero_still_serves_the_tokens(new):
    c = attention_case(new, [300, 900, 7, 40], 10, 2, 128, BF16)
    want = attend(c, max_query_len=1)
    out = torch.full(c["q"].shape, 7.0, dtype=BF16, device="cuda")
    got = attend(c, max_query_len=0, out=out)
    check_attention(c, got)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


TOP = 2 ** 31 - 1


def step(computed, scheduled, pages, num_tokens=4, max_blocks=3, page_dtype=torch.int32, **kw):
    err = ints([0])
    t = K.step_tables(ints(computed, torch.int64), ints(scheduled), torch.tensor(pages).to("cuda", page_dtype),
                      num_tokens=num_tokens, max_blocks=max_blocks, error_flag=err, **kw)
    return t, err.item()


@pytest.mark.parametrize("scheduled", [[TOP, TOP, 4], [2, TOP, TOP, 2], [1] + [1 << 24] * 256 + [1], [1, 1, TOP] * 200])
def test_counts_whose_sum_passes_32_bits_are_flagged_and_stay_in_order(scheduled):
    requests = len(scheduled)
    t, err = step([0] * requests, scheduled, [[3 + r % 2, 9] for r in range(requests)])
    assert err & N.DEV_TOKEN_RANGE
    starts = [min(sum(scheduled[:r]), TOP) for r in range(requests + 1)]
    assert t.query_start_loc.tolist() == starts
    first = [next(r for r in range(requests) if starts[r] <= i < starts[r + 1]) for i in range(4)]
    assert t.request_indices.tolist() == first
    assert t.positions.tolist() == [i - starts[r] for i, r in enumerate(first)]
    assert t.slot_mapping.tolist() == [(3 + r % 2) * 128 + i - starts[r] for i, r in enumerate(first)]


@pytest.mark.parametrize("bpp,page,block,slot", [
    (4, 1 << 62, -1, -1),                        # 4 * 2^62 is 0 in 64 bits
    (16, (1 << 60) + 5, -1, -1),
    (1, (1 << 56) + 7, -1, -1),                  # a slot of 2^63 and more
    (1, 1 << 40, -1, (1 << 47) + 10),            # a slot that 64 bits hold, a block that an int32 does not
    (2, 1 << 30, -1, (1 << 38) + 10),
    (2, (1 << 30) - 1, (1 << 31) - 2, ((1 << 30) - 1) * 256 + 10),  # the last page whose blocks an int32 holds
])
def test_page_ids_past_the_range_are_flagged(bpp, page, block, slot):
    t, err = step([10], [1], [[page]], num_tokens=1, max_blocks=1, page_dtype=torch.int64, blocks_per_page=bpp)
    assert t.block_table.tolist() == [[block]] and t.slot_mapping.tolist() == [slot]
    assert err == (0 if block >= 0 else N.DEV_BLOCK_RANGE)


@pytest.mark.parametrize("longest", [1, 64])
@pytest.mark.parametrize("tail", [[0], [0, 3]])
def test_starts_that_name_the_rows_thousands_of_times_are_flagged(longest, tail):
    """4,096 requests of 2^20 rows each: 2^32 rows, as starts that go back and forth name them."""
    n = 1 << 20
    starts = ([0, n] * 4096 + tail)[: 8193]
    memory = [torch.full((8 * n + 16 * 64,), 3.0, dtype=BF16, device="cuda") for _ in range(2)]  # rows overlap: 16 MB
    q, out = (x.as_strided((n, 16, 64), (8, 64, 1)) for x in memory)
    cache = torch.zeros(1, 128, 1, 64, dtype=BF16, device="cuda")
    requests = len(starts) - 1
    err = ints([0])
    K.paged_attention(q, cache, cache, torch.zeros(requests, 1, dtype=torch.int32, device="cuda"), ints(starts),
                      ints([5] * requests), max_query_len=longest, out=out, error_flag=err)
    assert err.item() == N.DEV_INDEX_RANGE
    assert (memory[1] == 3.0).all()


def test_tables_that_are_also_inputs_are_refused():
    t, err = step([10, 300], [1, 1], [[0, 1, 2], [3, 4, 5]], num_tokens=2)
    assert err == 0
    pages = ints([[0, 1, 2], [3, 4, 5]])
    with pytest.raises(RuntimeError, match="kvc_step_tables"):  # the last step's lengths, and its tables again
        K.step_tables(t.seq_lens, ints([1, 1]), pages, num_tokens=2, max_blocks=3, out=t)
    with pytest.raises(RuntimeError, match="kvc_step_tables"):
        K.step_tables(ints([11, 301]), ints([1, 1]), t.block_table, num_tokens=2, max_blocks=3, out=t)
    with pytest.raises(RuntimeError, match="kvc_step_tables"):
        K.step_tables(ints([11, 301]), ints([1, 1]), pages, num_tokens=2, max_blocks=3, out=t._replace(slot_mapping=t.positions))
    both = torch.arange(2, device="cuda", dtype=torch.int32)  # inputs alone may
    u = K.step_tables(both, both, pages, num_tokens=2, max_blocks=3, out=t)
    assert u.query_start_loc.tolist() == [0, 0, 1] and u.seq_lens.tolist() == [0, 2]
    v = K.step_tables(u.seq_lens, ints([1, 1]), pages, num_tokens=2, max_blocks=3)  # into tables of its own
    assert v.seq_lens.tolist() == [1, 3]


@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 20, 2.0 ** 24, 2.0 ** 26])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("dim,longest", [(64, 1), (128, 1), (256, 1), (64, 64), (128, 64), (256, 64)])
def test_scores_whose_rounding_is_bits(size, dtype, dim, longest):
    """Scores near `size` that differ by small whole numbers answer a mean of the values, never inf or NaN.

    The scores are exact here (two products of powers of two and small integers; at 2^24 and past it the integers
    are multiples of the step).  A maximum in units of log2 rounds by up to 2^-24 of itself, which moves all weights
    taken with it by as many bits; parts that were taken with two of them are up to twice as far apart, so the
    weights of a mean are each within a factor 2^s and the mean within 2^2s, and never outside the values.
    """
    n, heads = 600, 4
    step = max(1.0, size * 2.0 ** -23)
    g = torch.Generator().manual_seed(dim)
    below = step * torch.randint(0, 7, (n,), generator=g).float()
    half = size ** 0.5 if math.log2(size) % 2 == 0 else None
    q, k = torch.zeros(3, heads, dim), torch.zeros(640, dim)
    q[..., 0], k[:, 0] = half, half
    q[..., 9], k[:n, 9] = step, -below / step
    v = 0.5 + torch.rand(640, dim, generator=g)
    q, k, v = (x.to(dtype) for x in (q, k, v))
    assert q[0, 0, 0] == half and k[0, 0] == half and (k[:n, 9].float() == -below / step).all()
    out, lse = attend({"q": q, "kc": k.view(5, 128, 1, dim), "vc": v.view(5, 128, 1, dim),
                       "table": torch.arange(5, dtype=torch.int32).repeat(3, 1), "starts": [0, 1, 2, 3],
                       "lens": [n] * 3, "longest": longest}, scale=1.0)
    w = torch.softmax(-below.double(), 0)
    want = w @ v[:n].double()
    u = torch.finfo(dtype).eps / 2
    s = 2 * size * math.log2(math.e) * 2.0 ** -24
    out = out.double().cpu()
    top, bottom = v[:n].double().amax(0), v[:n].double().amin(0)
    assert (out <= top * (1 + 2 * u + 2.0 ** -18)).all() and (out >= bottom * (1 - 2 * u - 2.0 ** -18)).all()
    assert ((out - want).abs() <= want * (2 * u + 2.0 ** -18 + 4.0 ** s - 1)).all()
    assert (lse.double().cpu() - size).abs().max() <= 8 + size * 2.0 ** -21


@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, BF16), (256, BF16), (256, FP16)])
@pytest.mark.parametrize("longest", [1, 64])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5)])
def test_scattered_values_that_are_not_finite_reach_the_rows_that_see_them(dim, dtype, longest, window, sinks):
    """Single infinite and NaN values anywhere in the values, beside tails that hold nothing else."""
    new, lens = [130, 1, 7, 64], [400, 129, 7, 300]
    c = attention_case(new, lens, 4, 2, dim, dtype)
    g = torch.Generator().manual_seed(dim + longest)
    hit = torch.rand(c["vc"].shape, generator=g) < 3e-5
    c["vc"][hit] = torch.tensor([math.inf, -math.inf, math.nan])[torch.randint(0, 3, (int(hit.sum()),), generator=g)].to(dtype)
    for r, n in enumerate(lens):
        if n % 128:
            c["vc"][c["table"][r, (n - 1) // 128], n % 128:] = math.nan
    out, lse, ob, lb = R.attention(c["q"], c["kc"], c["vc"], c["table"], c["starts"], c["lens"], dim ** -0.5, window, sinks)
    got = [x.double().cpu() for x in attend(c, window=window, sinks=sinks, max_query_len=longest)]
    assert 0 < (~out.isfinite()).sum() < out.numel() / 2
    assert torch.equal(got[0].isnan(), out.isnan())
    odd = out.isinf()
    assert torch.equal(got[0].isinf(), odd) and torch.equal(got[0][odd], out[odd])
    fine = out.isfinite()
    # a value that is not finite makes its own dim's bound infinite or NaN: the finite dims' are as they were
    assert ((got[0] - out).abs() <= ob)[fine].all()
    assert ((got[1] - lse).abs() <= lb).all()

"""Serving-step operators on the GPU against their plain 64-bit forms (tests/serving_reference.py)."""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

import serving_reference as R
from vllm_ascend_kvcompress import _native as N
from vllm_ascend_kvcompress.methods.triattention import kernels as K
from vllm_ascend_kvcompress.provider import ActiveCompression, BatchedCompressionProvider

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


# ---- step tables ----------------------------------------------------------------------------------


def check_tables(t, want):
    got = (t.query_start_loc, t.seq_lens, t.positions, t.slot_mapping, t.request_indices, t.block_table)
    for g, w in zip(got, want):
        assert g.tolist() == w


@pytest.mark.parametrize("requests,bpp,dtype,page_dtype", [
    (1, 1, torch.int32, torch.int32), (3, 9, torch.int64, torch.int64), (300, 16, torch.int32, torch.int64),
    (1000, 1, torch.int64, torch.int32)])
def test_step_tables(requests, bpp, dtype, page_dtype):
    g = torch.Generator().manual_seed(requests)
    rand = lambda hi: torch.randint(0, hi, (requests,), generator=g).tolist()  # noqa: E731
    computed, scheduled = rand(9000), [n if n < 40 else 0 for n in rand(60)]  # a third of them without new tokens
    computed[0] = 0
    offsets = [min(c, o) if o % 3 == 0 else 0 for c, o in zip(computed, rand(9000))]
    width = -(-9100 // (128 * bpp))
    pages = torch.randint(0, 1 << 20, (requests, width), generator=g)
    total, blocks = sum(scheduled), 73
    want = R.step_tables(computed, scheduled, offsets, pages.tolist(), bpp, total + 5, blocks)
    err = ints([0])
    t = K.step_tables(ints(computed, dtype), ints(scheduled, dtype), pages.to("cuda", page_dtype),
                      num_tokens=total + 5, max_blocks=blocks, offsets=ints(offsets, torch.int64),
                      blocks_per_page=bpp, error_flag=err)
    check_tables(t, want)
    assert err.item() == 0
    # tables of an earlier call, and no offsets
    want = R.step_tables(computed, scheduled, [0] * requests, pages.tolist(), bpp, total + 5, blocks)
    again = K.step_tables(ints(computed, dtype), ints(scheduled, dtype), pages.to("cuda", page_dtype),
                          num_tokens=total + 5, max_blocks=blocks, blocks_per_page=bpp, out=t)
    assert again is t
    check_tables(t, want)


def test_step_tables_takes_rows_of_a_wider_page_table_and_an_empty_step():
    pages = torch.arange(40, dtype=torch.int32, device="cuda").view(4, 10)[::2, 2:8]
    t = K.step_tables(ints([130, 5]), ints([0, 0]), pages, num_tokens=0, max_blocks=3)
    check_tables(t, ([0, 0, 0], [130, 5], [], [], [], [[2, 3, -1], [22, -1, -1]]))


@pytest.mark.parametrize("computed,scheduled,offsets,pages,bit", [
    ([300], [1], [0], [[4, 5]], N.DEV_BLOCK_RANGE),     # the table ends before the token's page
    ([100], [1], [0], [[-1, 5]], N.DEV_BLOCK_RANGE),    # a page that was never assigned
    ([10], [2], [11], [[4, 5]], N.DEV_TOKEN_RANGE),     # a token before the cache
    ([10], [-2], [0], [[4, 5]], N.DEV_TOKEN_RANGE),     # a negative count
    ([10], [9], [0], [[4, 5]], N.DEV_TOKEN_RANGE),      # more new tokens than the tables hold
])
def test_step_tables_flags_what_it_cannot_place(computed, scheduled, offsets, pages, bit):
    err = ints([0])
    t = K.step_tables(ints(computed), ints(scheduled), ints(pages), num_tokens=4, max_blocks=3,
                      offsets=ints(offsets, torch.int64), error_flag=err)
    assert err.item() & bit
    assert all(-1 <= s < 6 * 128 for s in t.slot_mapping.tolist())


# ---- rotary positions and cache write ---------------------------------------------------------------


def rotary_case(n, heads, kvh, dim, rot, axes, dtype, far, seed=0, blocks=None):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(n, (heads + 2 * kvh) * dim + 8, generator=g).to(dtype)  # rows of a wider projection
    blocks = blocks or -(-n // 128) + 1
    return {"qkv": qkv, "split": (heads * dim, kvh * dim, kvh * dim, 8), "dim": dim,
            "positions": torch.randint(0, far, (axes, n), generator=g),
            "slots": torch.randperm(blocks * 128, generator=g)[:n],
            "omega": 1e6 ** (-torch.arange(rot // 2) / (rot // 2)), "axis": (torch.arange(rot // 2) * 7 % axes).int(),
            "kc": torch.randn(blocks, 128, kvh, dim, generator=g).to(dtype),
            "vc": torch.randn(blocks, 128, kvh, dim, generator=g).to(dtype)}


def views(qkv, c):
    return [x.unflatten(1, (-1, c["dim"])) for x in qkv.split(c["split"], 1)[:3]]


def check_rotary(c, q_got, kc_got, vc_got, slots):
    q, k, v = views(c["qkv"], c)
    for x, got in ((q, q_got), (k, None)):
        want, bound = R.rotate(x, c["positions"], c["omega"], c["axis"]), R.rotate_bound(x, c["omega"], x.dtype)
        if got is None:
            keep = slots >= 0
            kc, vc = c["kc"].double().flatten(0, 1), c["vc"].flatten(0, 1)
            kb = torch.zeros_like(kc)
            kc[slots[keep]], kb[slots[keep]] = want[keep], bound[keep]
            vc[slots[keep]] = v[keep]
            assert (kc_got.double().flatten(0, 1) - kc).abs().le(kb).all()
            assert torch.equal(vc_got.flatten(0, 1), vc)
        else:
            assert (got.double() - want).abs().le(bound).all()


@pytest.mark.parametrize("n,heads,kvh,dim,rot,axes,dtype,far", [
    (1, 5, 1, 128, 128, 1, BF16, 100), (37, 16, 2, 256, 64, 3, BF16, 52000), (130, 8, 8, 64, 64, 1, FP16, 1 << 20),
    (300, 20, 4, 128, 64, 4, FP16, 40000), (9, 3, 1, 72, 48, 2, BF16, 1 << 40), (5, 2, 2, 256, 256, 1, BF16, 7),
    (3, 2, 1, 16, 16, 1, FP16, 50), (2371, 3, 1, 64, 32, 3, BF16, 9000), (4000, 2, 2, 16, 16, 1, BF16, 70000)])
def test_rotary_write(n, heads, kvh, dim, rot, axes, dtype, far):
    c = rotary_case(n, heads, kvh, dim, rot, axes, dtype, far)
    if n > 4:
        c["slots"][2] = -1  # a padded token
    d = {k: t.cuda() for k, t in c.items() if torch.is_tensor(t)}
    q, k, v = views(d["qkv"], c)
    err = ints([0])
    got = K.rotary_write(q, k, v, d["positions"][0] if axes == 1 else d["positions"], d["slots"], d["kc"], d["vc"],
                         omega=d["omega"], axis_of_frequency=d["axis"] if axes > 1 else None, error_flag=err)
    assert err.item() == 0
    check_rotary(c, got.cpu(), d["kc"].cpu(), d["vc"].cpu(), c["slots"])
    assert torch.equal(d["qkv"].cpu(), c["qkv"])  # inputs as they were
    # in place, into caches that interleave in one padded buffer
    both = torch.zeros(c["kc"].shape[0], 2, c["kc"][0].numel() + 64, dtype=dtype, device="cuda")
    kc, vc = (both[:, i, : c["kc"][0].numel()].unflatten(1, c["kc"].shape[1:]) for i in (0, 1))
    kc.copy_(c["kc"])
    vc.copy_(c["vc"])
    same = K.rotary_write(q, k, v, d["positions"], d["slots"], kc, vc, omega=d["omega"], axis_of_frequency=d["axis"],
                          q_out=q)
    assert same is q and torch.equal(q, got) and torch.equal(kc, d["kc"]) and torch.equal(vc, d["vc"])
    assert not both[:, :, c["kc"][0].numel():].any()


def test_rotary_write_flags_bad_slots_and_axes_and_takes_no_tokens():
    c = rotary_case(4, 2, 1, 64, 32, 2, BF16, 50)
    c["slots"] = torch.tensor([5, c["kc"].shape[0] * 128, -7, 1 << 40])
    d = {k: t.cuda() for k, t in c.items() if torch.is_tensor(t)}
    q, k, v = views(d["qkv"], c)
    err = ints([0])
    got = K.rotary_write(q, k, v, d["positions"], d["slots"], d["kc"], d["vc"], omega=d["omega"],
                         axis_of_frequency=d["axis"], error_flag=err)
    assert err.item() == N.DEV_TOKEN_RANGE
    check_rotary(c, got.cpu(), d["kc"].cpu(), d["vc"].cpu(), torch.tensor([5, -1, -1, -1]))
    err.zero_()
    d["axis"][3] = 2
    K.rotary_write(q, k, v, d["positions"], d["slots"], d["kc"], d["vc"], omega=d["omega"],
                   axis_of_frequency=d["axis"], error_flag=err)
    assert err.item() == N.DEV_TOKEN_RANGE | N.DEV_INDEX_RANGE
    empty = K.rotary_write(q[:0], k[:0], v[:0], d["positions"][:, :0], d["slots"][:0], d["kc"], d["vc"],
                           omega=d["omega"], axis_of_frequency=d["axis"])
    assert empty.shape == (0, 2, 64)


# ---- paged attention ------------------------------------------------------------------------------


def attention_case(new, lens, heads, kvh, dim, dtype, seed=0, gain=1.5):
    g = torch.Generator().manual_seed(seed)
    need = [max(0, -(-n // 128)) for n in lens]
    blocks = sum(need) + 3
    ids = torch.randperm(blocks, generator=g)[: sum(need)].int()
    table = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = ids[at: at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    rand = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return {"q": (gain * rand(starts[-1], heads, dim)).to(dtype), "kc": rand(blocks, 128, kvh, dim).to(dtype),
            "vc": rand(blocks, 128, kvh, dim).to(dtype), "table": table, "starts": starts, "lens": lens,
            "longest": max(new)}


def attend(c, **kw):
    kw.setdefault("max_query_len", c["longest"])
    return K.paged_attention(c["q"].cuda(), c["kc"].cuda(), c["vc"].cuda(), c["table"].cuda(), ints(c["starts"]),
                             ints(c["lens"]), return_lse=True, **kw)


def check_attention(c, got, window=0, sinks=0, scale=None):
    scale = scale or c["q"].shape[2] ** -0.5
    out, lse, ob, lb = R.attention(c["q"], c["kc"], c["vc"], c["table"], c["starts"], c["lens"], scale, window, sinks)
    o, l = got[0].double().cpu(), got[1].double().cpu()
    assert torch.equal(o.isfinite(), out.isfinite())
    fine = out.isfinite()
    over = ((o - out).abs() - ob)[fine]  # rows that see nothing have the bound 0
    assert (over <= 0).all(), f"an output is {over.max().item():.3g} past its bound"
    seen = lse > -math.inf
    assert torch.equal(l > -math.inf, seen)
    over = ((l - lse).abs() - lb)[seen]
    assert (over <= 0).all(), f"an lse is {over.max().item():.3g} past its bound"


GEOMETRIES = [(40, 8, 128, BF16), (16, 2, 256, FP16), (8, 8, 64, FP16), (5, 1, 128, BF16), (16, 1, 64, BF16),
              (6, 2, 256, BF16), (13, 1, 128, FP16)]


@pytest.mark.parametrize("heads,kvh,dim,dtype", GEOMETRIES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 4), (1, 0), (64, 130), (5000, 9)])
def test_decode(heads, kvh, dim, dtype, window, sinks):
    lens = [1, 2, 127, 128, 129, 1000, 63, 64, 65, 700]
    c = attention_case([1] * len(lens), lens, heads, kvh, dim, dtype)
    check_attention(c, attend(c, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("heads,kvh,dim,dtype", GEOMETRIES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4), (1, 0), (33, 300)])
def test_short_and_ragged_chunks(heads, kvh, dim, dtype, window, sinks):
    c = attention_case([3, 1, 0, 17, 130, 2], [3, 400, 50, 20, 300, 129], heads, kvh, dim, dtype)
    check_attention(c, attend(c, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, FP16), (256, BF16)])
@pytest.mark.parametrize("new", [1, 2, 64])
def test_one_long_request_is_cut_over_the_whole_gpu(dim, dtype, new):
    c = attention_case([new], [9001], 4, 1, dim, dtype)
    check_attention(c, attend(c))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_requests_and_a_chunk_of_a_whole_prompt(dim):
    new = [1] * 70 + [333] + [1] * 70
    lens = [(37 * i) % 400 + 1 for i in range(70)] + [333] + [(91 * i) % 300 + 1 for i in range(70)]
    c = attention_case(new, lens, 2, 1, dim, BF16)
    check_attention(c, attend(c))
    check_attention(c, attend(c, window=50, sinks=3), 50, 3)


@pytest.mark.parametrize("longest,extra", [(1, 0), (3, 0), (1, 64), (150, 64)])
def test_more_tiles_than_threads_of_a_block(longest, extra):
    new = [(i * 7) % (longest + 1) if i % 50 == 3 else i % 3 != 0 for i in range(1100)]
    new[-1] = longest
    lens = [n + (53 * i) % 300 for i, n in enumerate(new)]
    c = attention_case([int(n) for n in new], lens, 4, 2, 64, BF16)
    kw = {"max_query_len": max(longest, extra)}  # 64: the kernel for chunks, whatever the lengths
    check_attention(c, attend(c, **kw))
    check_attention(c, attend(c, window=40, sinks=130, **kw), 40, 130)


def test_rows_that_see_nothing_and_requests_without_keys():
    c = attention_case([1, 5, 1, 3], [0, 2, 7, -4], 8, 2, 128, BF16)
    out, lse = attend(c)
    check_attention(c, (out, lse))
    assert not out[:4].any() and out[4:7].any() and not out[7:].any()
    assert (lse[:4] == -math.inf).all() and (lse[7:] == -math.inf).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim,new", [(128, [1, 4, 30]), (64, [1, 3, 200]), (256, [2, 1, 40])])
def test_masked_places_may_hold_anything(bad, dim, new):
    """Slots past each request's length, keys before the window, and later new tokens."""
    lens = [100, 300, 333]
    c = attention_case(new, lens, 6, 2, dim, BF16)
    for window, sinks in ((0, 0), (40, 2)):
        d = dict(c, kc=c["kc"].clone(), vc=c["vc"].clone())
        for r, n in enumerate(lens):
            last = c["table"][r, (n - 1) // 128]
            d["kc"][last, (n - 1) % 128 + 1:] = bad
            d["vc"][last, (n - 1) % 128 + 1:] = bad
        if window:  # a key that no row sees, in a block that rows do see
            at = lens[1] - new[1] - window
            d["kc"][c["table"][1, at // 128], at % 128] = bad
            d["vc"][c["table"][1, at // 128], at % 128] = bad
        # the last new token of the third request: its own row alone sees it
        d["vc"][c["table"][2, (lens[2] - 1) // 128], (lens[2] - 1) % 128, 1, 5] = bad
        out, lse = attend(d, window=window, sinks=sinks)
        check_attention(d, (out, lse), window, sinks)
        assert out[: sum(new) - 1].isfinite().all() and lse.isfinite().all()
        assert (~out[-1].isfinite()).sum() == 3  # the three heads of the second KV head, one dim


def test_infinite_and_nan_values_in_seen_places():
    c = attention_case([2, 1], [200, 5], 4, 2, 128, BF16)
    c["vc"][c["table"][0, 0], 17, 0, 3] = math.inf
    c["vc"][c["table"][1, 0], 2, 1, 100] = math.nan
    out, lse = attend(c)
    check_attention(c, (out, lse))
    assert (out[:2, :2, 3] == math.inf).all() and out[2, 2:, 100].isnan().all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_large_scores(dtype):
    c = attention_case([1, 40, 2], [500, 600, 20], 8, 2, 128, dtype, gain=60.0)
    check_attention(c, attend(c))
    check_attention(c, attend(c, scale=0.01), scale=0.01)


@pytest.mark.parametrize("new", [[1, 2, 1], [100, 1, 60]])
def test_strided_inputs_padded_pages_and_rows_of_no_request(new):
    c = attention_case(new, [300, 129, 64], 10, 2, 128, BF16)
    n = sum(new)
    want = attend(c)
    wide = torch.randn(n + 7, 14, 128, device="cuda").to(BF16)  # q inside a fused projection, rows behind the last
    wide[:n, 2:12] = c["q"].cuda()
    both = torch.full((c["kc"].shape[0], 2 * c["kc"][0].numel() + 64), math.nan, dtype=BF16, device="cuda")
    size = c["kc"][0].numel()
    kc, vc = (both[:, i * size: (i + 1) * size].unflatten(1, c["kc"].shape[1:]) for i in (0, 1))
    kc.copy_(c["kc"])
    vc.copy_(c["vc"])
    table = torch.full((3, 9), 7, dtype=torch.int32, device="cuda")
    table[:, : c["table"].shape[1]] = c["table"].cuda()
    out = torch.full((n + 7, 12, 128), 3.0, dtype=BF16, device="cuda")
    view = out[:, 1:11]
    err = ints([0])
    got, lse = K.paged_attention(wide[:, 2:12], kc, vc, table[:, :5], ints(c["starts"]), ints(c["lens"]),
                                 max_query_len=c["longest"], out=view, return_lse=True, error_flag=err)
    assert got is view and err.item() == 0
    assert torch.equal(out[:n, 1:11], want[0]) and torch.equal(lse[:n], want[1])
    assert (out[n:] == 3.0).all() and (out[:, 0] == 3.0).all() and (out[:, 11] == 3.0).all()


@pytest.mark.parametrize("new", [[1, 1], [50, 1]])
def test_bad_block_ids_and_row_ranges_are_flagged(new):
    c = attention_case(new, [300, 100], 4, 2, 64, BF16)
    want = attend(c)
    err = ints([0])
    bad = dict(c, table=c["table"].clone())
    bad["table"][0, 1] = c["kc"].shape[0]
    out, _ = attend(bad, error_flag=err)
    assert err.item() == N.DEV_BLOCK_RANGE
    assert torch.equal(out[new[0]:], want[0][new[0]:])  # the other request is served
    err.zero_()
    short = dict(c, table=c["table"][:, :2])
    attend(short, error_flag=err)
    assert err.item() == N.DEV_BLOCK_RANGE
    err.zero_()
    far = dict(c, starts=[0, new[0], new[0] + 9])
    out, _ = attend(far, error_flag=err)
    assert err.item() == N.DEV_INDEX_RANGE
    assert torch.equal(out[: new[0]], want[0][: new[0]])


@pytest.mark.parametrize("new", [[1, 1, 1, 1, 1], [9, 1, 50, 1, 3]])
@pytest.mark.parametrize("window", [0, 60])
def test_lengths_that_no_table_holds_are_flagged_and_leave_the_others(new, window):
    top = 2 ** 31 - 1
    for c, lens, rows in (
            (attention_case(new, [300, 0, 200, 10, 129], 4, 2, 64, BF16), [300, top, 200, -top - 1, 129], (0, 2, 4)),
            (attention_case([1] * 500 + [new[0]], [5] * 500 + [300], 4, 2, 64, BF16), [top] * 500 + [300], (500,))):
        out, lse, ob, lb = R.attention(c["q"], c["kc"], c["vc"], c["table"], c["starts"], c["lens"], 64 ** -0.5, window, 0)
        err = ints([0])
        got, l = (x.double().cpu() for x in attend(dict(c, lens=lens), window=window, error_flag=err))
        assert err.item() == N.DEV_BLOCK_RANGE
        for r in rows:
            s = slice(c["starts"][r], c["starts"][r + 1])
            assert ((got[s] - out[s]).abs() <= ob[s]).all() and ((l[s] - lse[s]).abs() <= lb[s]).all()
        for r in [r for r, n in enumerate(lens) if n < 0]:
            s = slice(c["starts"][r], c["starts"][r + 1])
            assert (got[s] == 0).all() and (l[s] == -math.inf).all()


@pytest.mark.parametrize("new", [[1] * 5, [1, 200, 3, 1, 64]])
def test_captured_and_replayed_with_other_lengths(new):
    lens = [300, 900, 500, 65, 64]
    c = attention_case(new, lens, 10, 2, 128, BF16)
    q, kc, vc, table = (c[x].cuda() for x in ("q", "kc", "vc", "table"))
    starts, length = ints(c["starts"]), ints(lens)
    run = lambda: K.paged_attention(q, kc, vc, table, starts, length, max_query_len=c["longest"],  # noqa: E731
                                    return_lse=True)
    run()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graphs, results = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(run())
    for shift in (0, 30):
        c["lens"] = [n - shift for n in lens]
        length.copy_(ints(c["lens"]))
        for x in results:
            x[0].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):  # both at once: each graph has a workspace of its own
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        check_attention(c, results[0])
        assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


def test_results_do_not_depend_on_timing():
    c = attention_case([1, 300, 1, 2], [5000, 2300, 700, 3], 10, 2, 128, BF16)
    d = [c[x].cuda() for x in ("q", "kc", "vc", "table")] + [ints(c["starts"]), ints(c["lens"])]
    first = K.paged_attention(*d, max_query_len=300)
    for _ in range(20):
        assert torch.equal(K.paged_attention(*d, max_query_len=300), first)


@pytest.mark.parametrize("new", [[1, 1], [60, 1]])
def test_offsets_past_32_bits(new):
    """Blocks past 4 GB of a cache that interleaves K and V, written by the rotary write and read by attention."""
    kvh, dim, heads, blocks, n = 8, 128, 16, 9000, sum(new)
    g = torch.Generator().manual_seed(1)
    both = torch.zeros(blocks, 2, 128 * kvh * dim, dtype=BF16, device="cuda")
    kc, vc = (both[:, i].unflatten(1, (128, kvh, dim)) for i in (0, 1))
    lens, ids = [300, 129], [[8999, 3, 8700], [8500, 8998, -1]]
    used = [8999, 3, 8700, 8500, 8998]
    for c in (kc, vc):
        c[used] = torch.randn(len(used), 128, kvh, dim, generator=g).to(BF16).cuda()
    x = torch.randn(n, heads + 2 * kvh, dim, generator=g).to(BF16)
    starts = [0, new[0], n]
    slots = [ids[r][p // 128] * 128 + p % 128 for r in range(2) for p in range(lens[r] - new[r], lens[r])]
    pos = torch.arange(n)[None]
    omega = 1e6 ** (-torch.arange(dim // 2) / (dim // 2))
    q, k, v = x.cuda().split([heads, kvh, kvh], 1)
    q = K.rotary_write(q, k, v, pos.cuda(), ints(slots, torch.int64), kc, vc, omega=omega.cuda())
    small = {i: j for j, i in enumerate(used)}
    hk, hv = kc[used].cpu(), vc[used].cpu()
    at = [small[s // 128] * 128 + s % 128 for s in slots]
    want = R.rotate(x[:, heads: heads + kvh], pos, omega, torch.zeros(dim // 2).long())
    assert (hk.flatten(0, 1)[at].double() - want).abs().le(R.rotate_bound(x[:, heads: heads + kvh], omega, BF16)).all()
    assert torch.equal(hv.flatten(0, 1)[at], x[:, heads + kvh:])
    got = K.paged_attention(q, kc, vc, ints(ids), ints(starts), ints(lens), max_query_len=max(new), return_lse=True)
    c = {"q": q.cpu(), "kc": hk, "vc": hv, "table": torch.tensor([[small.get(i, -1) for i in row] for row in ids]),
         "starts": starts, "lens": lens}
    check_attention(c, got)


# ---- a step of all three --------------------------------------------------------------------------


@pytest.mark.parametrize("scheduled", [[1, 1, 1, 1], [1, 70, 3, 0]])
def test_a_step_over_a_compressed_cache(scheduled):
    """Tables, rotary write and attention as a serving step runs them; two requests were compressed."""
    g = torch.Generator().manual_seed(3)
    computed, offsets = [700, 0, 5000, 130], [0, 0, 4700, 2]
    heads, kvh, dim, rot, bpp = 16, 2, 128, 64, 2
    pages = torch.randperm(40, generator=g)[:16].view(4, 4)
    total = sum(scheduled)
    want = R.step_tables(computed, scheduled, offsets, pages.tolist(), bpp, total, 8)
    x = torch.randn(total, (heads + 2 * kvh) * dim, generator=g).to(BF16)
    kc, vc = (torch.randn(80, 128, kvh, dim, generator=g).to(BF16) for _ in range(2))
    omega = 1e7 ** (-torch.arange(rot // 2) / (rot // 2))
    t = K.step_tables(ints(computed), ints(scheduled), pages.int().cuda(), num_tokens=total, max_blocks=8,
                      offsets=ints(offsets, torch.int64), blocks_per_page=bpp)
    check_tables(t, want)
    gk, gv = kc.cuda(), vc.cuda()
    q, k, v = (y.unflatten(1, (-1, dim)) for y in x.cuda().split([heads * dim, kvh * dim, kvh * dim], 1))
    q = K.rotary_write(q, k, v, t.positions, t.slot_mapping, gk, gv, omega=omega.cuda())
    got = K.paged_attention(q, gk, gv, t.block_table, t.query_start_loc, t.seq_lens, max_query_len=max(scheduled),
                            return_lse=True)
    # each stage against its 64-bit form, on what the stage before left
    hq, hk, hv = (y.unflatten(1, (-1, dim)) for y in x.split([heads * dim, kvh * dim, kvh * dim], 1))
    pos, slots, axis = torch.tensor([want[2]]), torch.tensor(want[3]), torch.zeros(rot // 2).long()
    assert (q.cpu().double() - R.rotate(hq, pos, omega, axis)).abs().le(R.rotate_bound(hq, omega, BF16)).all()
    gk, gv = gk.cpu(), gv.cpu()
    assert (gk.flatten(0, 1)[slots].double() - R.rotate(hk, pos, omega, axis)).abs().le(
        R.rotate_bound(hk, omega, BF16)).all()
    assert torch.equal(gv.flatten(0, 1)[slots], hv)
    c = {"q": q.cpu(), "kc": gk, "vc": gv, "table": torch.tensor(want[5]), "starts": want[0], "lens": want[1]}
    check_attention(c, got)


def test_the_provider_makes_the_tables_of_its_batch():
    ids = ["a", "b", "c"]
    runner = SimpleNamespace(device=torch.device("cuda"), requests={r: None for r in ids}, max_num_reqs=4,
                             max_num_tokens=64, input_batch=SimpleNamespace(req_ids=ids, num_reqs=3))
    p = BatchedCompressionProvider(SimpleNamespace(runtime_spec=None), runner, scheduler_block_size=256)
    p.active["b"] = ActiveCompression(5000, 300)
    p.after_update_states(None)
    pages = torch.arange(30).view(3, 10)
    t = p.step_tables(ints([10, 5003, 700]), ints([4, 1, 1]), pages.cuda(), num_tokens=6, max_blocks=6)
    check_tables(t, R.step_tables([10, 5003, 700], [4, 1, 1], [0, 4700, 0], pages.tolist(), 2, 6, 6))
    p.check_device_errors()
    p.step_tables(ints([10, 5003, 9000]), ints([4, 1, 1]), pages.cuda(), num_tokens=6, max_blocks=6)
    with pytest.raises(RuntimeError, match="step_tables"):
        p.check_device_errors()
    with pytest.raises(RuntimeError, match="max_num_reqs"):
        p.step_tables(ints([1] * 5), ints([1] * 5), pages.cuda(), num_tokens=5, max_blocks=1)


# ---- refusals of the wrappers ---------------------------------------------------------------------


def test_wrappers_refuse_what_does_not_fit():
    i32 = ints([3, 4])
    pages = ints([[0, 1], [2, 3]])
    for bad in (dict(offsets=i32), dict(max_blocks=-1), dict(num_tokens=-1), dict(blocks_per_page=0)):
        with pytest.raises((RuntimeError, ValueError)):
            K.step_tables(i32, i32, pages, **{"num_tokens": 7, "max_blocks": 1, **bad})
    for bad in ((i32[:1], i32, pages), (i32.float(), i32, pages), (i32, i32, pages[:, :1].T), (i32[:0], i32[:0], pages[:0])):
        with pytest.raises((RuntimeError, ValueError)):
            K.step_tables(*bad, num_tokens=7, max_blocks=1)
    with pytest.raises(ValueError, match="must have shape"):
        K.step_tables(i32, i32, pages, num_tokens=7, max_blocks=1, out=K.StepTables.empty(2, 6, 1, "cuda"))
    with pytest.raises(RuntimeError, match="CUDA"):
        K.step_tables(i32, i32, pages, num_tokens=7, max_blocks=1, error_flag=torch.zeros(1, dtype=torch.int32))

    c = rotary_case(4, 2, 1, 64, 32, 2, BF16, 50)
    d = {k: t.cuda() for k, t in c.items() if torch.is_tensor(t)}
    q, k, v = views(d["qkv"], c)
    good = dict(positions=d["positions"], slot_mapping=d["slots"], k_cache=d["kc"], v_cache=d["vc"], omega=d["omega"],
                axis_of_frequency=d["axis"])
    K.rotary_write(q, k, v, **good)
    for bad in (dict(axis_of_frequency=None), dict(positions=d["positions"].int()), dict(slot_mapping=d["slots"][:3]),
                dict(k_cache=d["kc"][:, :64]), dict(k_cache=d["kc"].to(FP16), v_cache=d["vc"].to(FP16)),
                dict(omega=d["omega"].double()), dict(q_out=q[:3]), dict(omega=d["omega"][:12], axis_of_frequency=d["axis"][:12])):
        with pytest.raises((RuntimeError, ValueError)):
            K.rotary_write(q, k, v, **{**good, **bad})
    for q1, k1, v1 in ((q[:, :, :32], k, v), (q, k[:3], v[:3]), (q.float(), k, v), (q.transpose(1, 2), k, v)):
        with pytest.raises((RuntimeError, ValueError)):
            K.rotary_write(q1, k1, v1, **good)

    a = attention_case([1, 2], [100, 200], 4, 2, 64, BF16)
    args = [a[x].cuda() for x in ("q", "kc", "vc", "table")] + [ints(a["starts"]), ints(a["lens"])]
    K.paged_attention(*args, max_query_len=2)
    for i, bad in ((0, args[0].to(FP16)), (0, args[0].float()), (1, args[1][:, :, :1]), (1, args[1][:, :, :, :32]),
                   (3, args[3].long()), (3, args[3][:1]), (4, args[4].long()), (4, args[4][:2]), (5, args[5].float())):
        with pytest.raises((RuntimeError, ValueError)):
            K.paged_attention(*args[:i], bad, *args[i + 1:], max_query_len=2)
    for bad in (dict(scale=0.0), dict(window=-1), dict(sinks=-1), dict(max_query_len=-1), dict(out=args[0][:2]),
                dict(workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))):
        with pytest.raises((RuntimeError, ValueError)):
            K.paged_attention(*args, **{"max_query_len": 2, **bad})


@pytest.mark.parametrize("longest", [1, 2, 5, 1000])
def test_the_longest_length_picks_the_kernel_alone(longest):
    """A bound that is wrong or generous changes which kernel runs, and nothing past rounding."""
    c = attention_case([1, 5, 0, 40], [300, 900, 7, 40], 10, 2, 128, BF16)
    check_attention(c, attend(c, max_query_len=longest))


@pytest.mark.parametrize("new", [[1, 1], [1, 90]])
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 2 ** 31 - 1), (30, 2 ** 31 - 1), (2 ** 31 - 1, 0)])
def test_windows_and_first_tokens_past_any_cache(new, window, sinks):
    c = attention_case(new, [200, 300], 4, 2, 128, BF16)
    check_attention(c, attend(c, window=window, sinks=sinks), window, sinks)


def test_calls_on_two_streams_at_once():
    c = attention_case([1, 70, 2], [3000, 1200, 64], 10, 2, 128, BF16)
    d = [c[x].cuda() for x in ("q", "kc", "vc", "table")] + [ints(c["starts"]), ints(c["lens"])]
    want = K.paged_attention(*d, max_query_len=70)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(K.paged_attention(*d, max_query_len=70))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_a_step_in_one_graph_follows_new_lengths():
    """Tables, rotary write and attention captured together, padded to a fixed number of tokens."""
    g = torch.Generator().manual_seed(9)
    heads, kvh, dim, cap = 8, 2, 64, 8
    pages = torch.randperm(24, generator=g).view(3, 8)
    computed, scheduled = ints([100, 500, 3]), ints([1, 1, 1])
    x = torch.randn(cap, (heads + 2 * kvh) * dim, generator=g).to(BF16).cuda()
    caches = [torch.randn(24, 128, kvh, dim, generator=g).to(BF16).cuda() for _ in range(2)]
    omega = (1e6 ** (-torch.arange(dim // 2) / (dim // 2))).cuda()
    page_table = pages.int().cuda()
    q, k, v = (y.unflatten(1, (-1, dim)) for y in x.split([heads * dim, kvh * dim, kvh * dim], 1))

    def step():
        t = K.step_tables(computed, scheduled, page_table, num_tokens=cap, max_blocks=8)
        turned = K.rotary_write(q, k, v, t.positions, t.slot_mapping, *caches, omega=omega)
        return (t, turned, *K.paged_attention(turned, *caches, t.block_table, t.query_start_loc, t.seq_lens,
                                              max_query_len=cap, return_lse=True))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t, turned, out, lse = step()
    for lens, new in (([100, 500, 3], [1, 1, 1]), ([101, 0, 900], [2, 5, 1]), ([7, 700, 0], [0, 0, 3])):
        computed.copy_(ints(lens))
        scheduled.copy_(ints(new))
        graph.replay()
        torch.cuda.synchronize()
        want = R.step_tables(lens, new, [0, 0, 0], pages.tolist(), 1, cap, 8)
        check_tables(t, want)
        n = sum(new)
        c = {"q": turned[:n].cpu(), "kc": caches[0].cpu(), "vc": caches[1].cpu(), "table": torch.tensor(want[5]),
             "starts": want[0], "lens": want[1]}
        check_attention(c, (out[:n], lse[:n]))

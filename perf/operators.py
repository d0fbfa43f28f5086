"""The serving step's operators around the paged (and possibly compressed) KV cache, as measured cases.

Four operators, in the order a decode or chunked-prefill step runs them:

* ``tables``  block tables, slot map, positions and physical lengths of a step from the request lengths;
* ``rotary``  rotary positions with one to three axes, keys and values written into the paged cache;
* ``attend``  attention of each request's new tokens (one, or a chunk) over its paged cache;
* ``window``  the same with a sliding window and a few first tokens that stay visible.

``run`` computes the plain form with elementary torch operations in 32 bits (angles in 64), or, with
``own`` set, makes the framework's calls.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- the cases -----------------------------------------------------------------------------------


def _tables(name, requests, ctx_lo, ctx_hi, new_lo, new_hi, decodes, budget, bpp, salt):
    return {"name": name, "op": "tables", "requests": requests, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "new_lo": new_lo,
            "new_hi": new_hi, "decodes": decodes, "budget": budget, "bpp": bpp, "salt": salt}


def _rotary(name, tokens, heads, kv_heads, dim, rotary, axes, far, dtype, salt):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "axes": axes, "far": far, "dtype": dtype, "salt": salt}


def _attend(name, requests, ctx_lo, ctx_hi, new_lo, new_hi, decodes, heads, kv_heads, dim, dtype, budget, window, sinks,
            salt):
    return {"name": name, "op": "window" if window else "attend", "requests": requests, "ctx_lo": ctx_lo,
            "ctx_hi": ctx_hi, "new_lo": new_lo, "new_hi": new_hi, "decodes": decodes, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "budget": budget, "window": window, "sinks": sinks,
            "salt": salt}


def listed():
    return [
        # a decode step of four requests, 128-token scheduler pages: latency
        _tables("tables_decode4", 4, 1000, 6000, 1, 1, 4, 0, 1, 11),
        # 128 decodes of 2k-64k tokens, the long ones compressed to a 4608-token budget
        _tables("tables_decode128", 128, 2048, 65536, 1, 1, 128, 4608, 1, 12),
        # chunked prefill beside decodes: 2048-token scheduler pages, each sixteen kernel blocks
        _tables("tables_chunked96", 96, 0, 52000, 64, 700, 72, 4608, 16, 13),
        # one new token of 32 requests, 40 query heads on 8 KV heads
        _rotary("rotary_decode32", 32, 40, 8, 128, 128, 1, 32768, "bf16", 21),
        # a long prompt with image and video positions: partial rotary over 64 of 256 dims, three axes
        _rotary("rotary_chunk8191_axes3", 8191, 16, 2, 256, 64, 3, 52000, "bf16", 22),
        # a small decode step: latency
        _attend("decode4", 4, 1000, 6000, 1, 1, 4, 40, 8, 128, "bf16", 0, 0, 0, 31),
        # decode after compression: every cache at its 4608-token budget and a few tokens
        _attend("decode32_compressed", 32, 4096, 32768, 1, 1, 32, 40, 8, 128, "bf16", 4608, 0, 0, 32),
        # decode over long uncompressed caches, head_dim 256
        _attend("decode16_long_fp16", 16, 8192, 52000, 1, 1, 16, 16, 2, 256, "fp16", 0, 0, 0, 33),
        # one prefill chunk over a long prefix
        _attend("chunk2048_over16k", 1, 16384, 16384, 2048, 2048, 0, 40, 8, 128, "bf16", 0, 0, 0, 34),
        # ragged chunks beside decodes, head_dim 256
        _attend("mixed12_d256", 12, 300, 9000, 65, 900, 6, 16, 2, 256, "bf16", 0, 0, 0, 35),
        # streaming decode: 128 first tokens and the last 512 of 4k-32k
        _attend("window_decode32", 32, 4096, 32768, 1, 1, 32, 40, 8, 128, "bf16", 0, 512, 128, 41),
        # a whole prompt with the window, head_dim 64
        _attend("window_prompt8191_d64", 1, 0, 0, 8191, 8191, 0, 16, 8, 64, "fp16", 0, 1024, 4, 42),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["tables", "rotary", "attend", "attend", "window"])
    salt = rng.randrange(1 << 30)
    if op == "tables":
        requests = _log(rng, 1, 128)
        decodes = requests if rng.random() < 0.5 else rng.randint(0, requests)
        new_hi = max(1, min(_log(rng, 1, 2000), 9000 // requests))
        hi = _log(rng, 1, 60000)
        case = _tables(None, requests, rng.randint(0, hi), hi, rng.randint(1, new_hi), new_hi, decodes,
                       rng.choice([0, 4608]), rng.choice([1, 9, 16]), salt)
    elif op == "rotary":
        heads, kv, dim, rotary = rng.choice([(40, 8, 128, 128), (16, 2, 256, 64), (8, 8, 64, 64), (20, 4, 128, 64),
                                             (5, 1, 128, 128), (16, 2, 256, 256)])
        tokens = _log(rng, 1, 8000 * 20 * 256 // ((heads + 2 * kv) * dim))
        case = _rotary(None, tokens, heads, kv, dim, rotary, rng.choice([1, 1, 3]), _log(rng, 16, 1000000),
                       rng.choice(["bf16", "fp16"]), salt)
    else:
        heads, kv, dim = rng.choice([(40, 8, 128), (16, 2, 256), (8, 8, 64), (20, 4, 128), (5, 1, 128), (16, 8, 64),
                                     (24, 4, 64)])
        window = _log(rng, 1, 4096) if op == "window" else 0
        sinks = rng.choice([0, 4, 128, rng.randint(1, 200)]) if window else 0
        dtype = rng.choice(["bf16", "fp16"])
        if rng.random() < 0.5:
            requests = _log(rng, 1, 32)
            hi = min(_log(rng, 1, 32768), 240000000 // (kv * dim * requests))
            case = _attend(None, requests, rng.randint(hi // 8, hi), hi, 1, rng.choice([1, 1, 3]), 0, heads, kv, dim,
                           dtype, rng.choice([0, 0, 4608]), window, sinks, salt)
        else:
            requests = _log(rng, 1, 8)
            hi, new = _log(rng, 1, 12000), max(1, _log(rng, 2, 2000) // requests)
            case = _attend(None, requests, rng.randint(0, hi), hi, rng.randint(1, new), new,
                           rng.randint(0, requests - 1), heads, kv, dim, dtype, 0, window, sinks, salt)
    del case["name"]
    return case


def _lengths(case):
    """(tokens before the step, new tokens, removed tokens) of each request, from the case alone."""
    rng = random.Random(case["salt"])
    ctx, new, removed = [], [], []
    for i in range(case["requests"]):
        c = rng.randint(case["ctx_lo"], case["ctx_hi"])
        n = 1 if i < case["decodes"] else rng.randint(case["new_lo"], case["new_hi"])
        grown = rng.randrange(128)
        ctx.append(c)
        new.append(n)
        removed.append(c - case["budget"] - grown if case["budget"] and c >= case["budget"] + 128 else 0)
    order = list(range(len(ctx)))
    rng.shuffle(order)
    return [ctx[i] for i in order], [new[i] for i in order], [removed[i] for i in order]


def _visible(last, window, sinks):
    """Keys that a query at physical position `last` attends to."""
    if not window or last + 1 <= window:
        return last + 1
    return window + min(sinks, last + 1 - window)


def work(case):
    if case["op"] == "tables":
        ctx, new, removed = _lengths(case)
        width = max(-(-(c + n - d) // BLOCK) for c, n, d in zip(ctx, new, removed))
        pages = sum(-(-(c + n - d) // (BLOCK * case["bpp"])) for c, n, d in zip(ctx, new, removed))
        requests, tokens = len(ctx), sum(new)
        # lengths, offsets and page ids read; prefix sums, lengths, blocks, positions, slots and indices written
        return {"bytes": requests * (4 + 4 + 8) + 4 * pages + 4 * (2 * requests + 1) + 4 * requests * width + 20 * tokens,
                "flops": 8 * tokens + 2 * requests * width}
    if case["op"] == "rotary":
        n, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": n * (4 * (h + 2 * kv) * d + 8 * case["axes"] + 8),
                "flops": 3 * n * (h + kv) * case["rotary"]}
    ctx, new, removed = _lengths(case)
    pairs = keys = 0
    for c, n, d in zip(ctx, new, removed):
        first = c - d
        pairs += sum(_visible(first + j, case["window"], case["sinks"]) for j in range(n))
        keys += min(first + n, _visible(first, case["window"], case["sinks"]) + n - 1)
    tokens, h, kv, dim = sum(new), case["heads"], case["kv_heads"], case["dim"]
    return {"bytes": 4 * keys * kv * dim + 4 * tokens * h * dim + 4 * tokens * h,
            "flops": 4 * pairs * h * dim}


# ---- inputs --------------------------------------------------------------------------------------


def _pages(lengths, page, device, generator):
    """A page table of random distinct page ids, -1 past each request's pages, and the pages that it names."""
    need = [-(-n // page) for n in lengths]
    ids = torch.randperm(sum(need) + 3, generator=generator, device=device)[: sum(need)].to(torch.int32)
    table = torch.full((len(need), max(max(need), 1)), -1, dtype=torch.int32, device=device)
    inside = torch.arange(table.shape[1], device=device) < torch.tensor(need, device=device)[:, None]
    table[inside] = ids
    return table, sum(need) + 3


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(1000003 * seed + case["salt"])
    if case["op"] == "tables":
        ctx, new, removed = _lengths(case)
        table, _ = _pages([c + n - d for c, n, d in zip(ctx, new, removed)], BLOCK * case["bpp"], device, g)
        as_tensor = lambda v, t: torch.tensor(v, dtype=t, device=device)  # noqa: E731
        return {"case": case, "computed": as_tensor(ctx, torch.int32), "scheduled": as_tensor(new, torch.int32),
                "offsets": as_tensor(removed, torch.int64), "pages": table, "tokens": sum(new),
                "width": max(-(-(c + n - d) // BLOCK) for c, n, d in zip(ctx, new, removed)) or 1}
    dtype, kv, d = DTYPES[case["dtype"]], case["kv_heads"], case["dim"]
    rand = lambda *shape: torch.randn(shape, generator=g, device=device, dtype=dtype)  # noqa: E731
    if case["op"] == "rotary":
        n, h, f = case["tokens"], case["heads"], case["rotary"] // 2
        # one fused projection's output, as a layer has it: q, k and v are views of its rows
        qkv = rand(n, (h + 2 * kv) * d)
        q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([h * d, kv * d, kv * d], dim=1))
        blocks = -(-n // BLOCK) + 2
        start = torch.randint(0, case["far"], (case["axes"], 1), generator=g, device=device)
        positions = start + torch.arange(n, device=device) // torch.tensor([[1], [7], [3]], device=device)[: case["axes"]]
        slots = torch.randperm(blocks * BLOCK, generator=g, device=device)[:n]
        slots[torch.rand(n, generator=g, device=device) < 0.01] = -1  # padded tokens of a captured step
        theta = 1e7 if d == 256 else 1e6
        omega = (theta ** (-torch.arange(f, dtype=torch.float64, device=device) / f)).float()
        axis = (torch.arange(f, device=device) % case["axes"]).to(torch.int32)
        return {"case": case, "q": q, "k": k, "v": v, "positions": positions, "slots": slots, "omega": omega,
                "axis": axis, "k_cache": rand(blocks, BLOCK, kv, d), "v_cache": rand(blocks, BLOCK, kv, d)}
    ctx, new, removed = _lengths(case)
    lengths = [c + n - r for c, n, r in zip(ctx, new, removed)]
    table, blocks = _pages(lengths, BLOCK, device, g)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return {"case": case, "q": 1.5 * rand(starts[-1], case["heads"], d), "k_cache": rand(blocks, BLOCK, kv, d),
            "v_cache": rand(blocks, BLOCK, kv, d), "table": table,
            "starts": torch.tensor(starts, dtype=torch.int32, device=device),
            "lengths": torch.tensor(lengths, dtype=torch.int32, device=device),
            "new": new, "ends": lengths, "longest": max(new)}


# ---- plain forms ---------------------------------------------------------------------------------


def _plain_tables(s):
    bpp = s["case"]["bpp"]
    computed, scheduled, offsets = s["computed"].long(), s["scheduled"].long(), s["offsets"]
    ends = torch.cumsum(scheduled, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    request = torch.repeat_interleave(torch.arange(len(computed), device=computed.device), scheduled,
                                      output_size=s["tokens"])
    positions = computed[request] + torch.arange(s["tokens"], device=computed.device) - starts[request].long()
    physical = positions - offsets[request]
    page = BLOCK * bpp
    slots = s["pages"][request, physical // page].long() * page + physical % page
    lengths = computed + scheduled - offsets
    index = torch.arange(s["width"], device=computed.device)
    width = s["pages"].shape[1]
    blocks = s["pages"][:, (index // bpp).clamp(max=width - 1)].long() * bpp + index % bpp
    blocks = torch.where(index * BLOCK < lengths[:, None], blocks, -1)
    return [starts, lengths.to(torch.int32), positions, slots, request.to(torch.int32), blocks.to(torch.int32)]


def _plain_rotary(s):
    case = s["case"]
    f = case["rotary"] // 2
    angle = s["positions"][s["axis"].long()].double() * s["omega"].double()[:, None]
    cos, sin = (t.float().t()[:, None] for t in (torch.cos(angle), torch.sin(angle)))

    def turn(x):
        x = x.float()
        a, b, rest = x[..., :f], x[..., f: 2 * f], x[..., 2 * f:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)

    q = turn(s["q"]).to(s["q"].dtype)
    k = turn(s["k"]).to(s["k"].dtype)
    keep = s["slots"] >= 0
    slots = s["slots"][keep]
    s["k_cache"].flatten(0, 1)[slots] = k[keep]
    s["v_cache"].flatten(0, 1)[slots] = s["v"][keep]
    return [q, s["k_cache"], s["v_cache"]]


def _softmax_of(scores, seen, values, how):
    """exp and sum over the seen keys, the weighted values and the logarithm of the sum."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    return torch.einsum(how, p / total, values), (top + torch.log(total)).squeeze(-1)


def _plain_attend(s):
    case = s["case"]
    h, kv, d, window, sinks = (case[x] for x in ("heads", "kv_heads", "dim", "window", "sinks"))
    q = s["q"].float().unflatten(1, (kv, h // kv)) / math.sqrt(d)
    if s["longest"] == 1:  # single tokens: every request at once, padded to the longest
        pages = s["table"].clamp(min=0).long()
        k, v = (c[pages].flatten(1, 2).float() for c in (s["k_cache"], s["v_cache"]))
        at = torch.arange(k.shape[1], device=q.device)
        last = s["lengths"].long()[:, None] - 1
        seen = at <= last
        if window:
            seen = seen & ((at > last - window) | (at < sinks))
        out, lse = _softmax_of(torch.einsum("rhgd,rthd->rhgt", q, k), seen[:, None, None], v, "rhgt,rthd->rhgd")
        return [out.flatten(1, 2).to(s["q"].dtype), lse.flatten(1, 2)]
    outs, lses, start = [], [], 0
    for r, (n, end) in enumerate(zip(s["new"], s["ends"])):  # chunks of unlike lengths, one request at a time
        pages = s["table"][r, : -(-end // BLOCK)].long()
        k, v = (c[pages].flatten(0, 1)[:end].float() for c in (s["k_cache"], s["v_cache"]))
        at = torch.arange(end, device=q.device)
        last = torch.arange(end - n, end, device=q.device)[:, None]
        seen = at <= last
        if window:
            seen = seen & ((at > last - window) | (at < sinks))
        out, lse = _softmax_of(torch.einsum("nhgd,thd->hgnt", q[start: start + n], k), seen, v, "hgnt,thd->nhgd")
        outs.append(out.flatten(1, 2))
        lses.append(lse.permute(2, 0, 1).flatten(1, 2))
        start += n
    return [torch.cat(outs).to(s["q"].dtype), torch.cat(lses)]


# ---- the framework's calls -----------------------------------------------------------------------


def _kernels():
    root = str(Path(__file__).resolve().parents[1] / "vllm-ascend-kvcompress-hust_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from vllm_ascend_kvcompress.methods.triattention import kernels

    return kernels


def _own(s):
    kernels, case = _kernels(), s["case"]
    if case["op"] == "tables":
        t = kernels.step_tables(s["computed"], s["scheduled"], s["pages"], num_tokens=s["tokens"],
                                max_blocks=s["width"], offsets=s["offsets"], blocks_per_page=case["bpp"])
        return [t.query_start_loc, t.seq_lens, t.positions, t.slot_mapping, t.request_indices, t.block_table]
    if case["op"] == "rotary":
        q = kernels.rotary_write(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["k_cache"], s["v_cache"],
                                 omega=s["omega"], axis_of_frequency=s["axis"])
        return [q, s["k_cache"], s["v_cache"]]
    return list(kernels.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["lengths"],
                                        max_query_len=s["longest"], window=case["window"], sinks=case["sinks"],
                                        return_lse=True))


def run(state):
    if own:
        return _own(state)
    if state["case"]["op"] == "tables":
        return _plain_tables(state)
    if state["case"]["op"] == "rotary":
        return _plain_rotary(state)
    return _plain_attend(state)


# ---- the definition in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "rotary":
        # each pair is a complex number, turned by its angle
        f = case["rotary"] // 2
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           torch.stack([s["positions"][a].double() for a in s["axis"].tolist()], 1) *
                           s["omega"].double())[:, None]
        results = []
        for x in (s["q"].double(), s["k"].double()):
            z = torch.complex(x[..., :f].contiguous(), x[..., f: 2 * f].contiguous()) * turn
            results.append(torch.cat([z.real, z.imag, x[..., 2 * f:]], -1))
        caches = [s["k_cache"].double(), s["v_cache"].double()]
        live = (s["slots"] >= 0).nonzero().squeeze(1)
        block, within = s["slots"][live] // BLOCK, s["slots"][live] % BLOCK
        caches[0][block, within] = results[1][live]
        caches[1][block, within] = s["v"].double()[live]
        return [results[0], *caches]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(sum(s["new"]), h, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(sum(s["new"]), h, dtype=torch.float64, device="cuda")
    row = 0
    for r, (n, end) in enumerate(zip(s["new"], s["ends"])):
        ids = s["table"][r].tolist()[: -(-end // BLOCK)]
        keys, values = (c[ids].reshape(-1, kv, d)[:end] for c in (s["k_cache"], s["v_cache"]))
        position = torch.arange(end, device="cuda")
        for head in range(kv):
            key, value = keys[:, head].double(), values[:, head].double()
            for first in range(0, n, 512):
                at = torch.arange(end - n + first, end - n + min(n, first + 512), device="cuda")
                seen = position[None] <= at[:, None]
                if case["window"]:
                    seen &= (at[:, None] - position[None] < case["window"]) | (position[None] < case["sinks"])
                rows = slice(row + first, row + first + len(at))
                for g in range(head * (h // kv), (head + 1) * (h // kv)):
                    logits = (s["q"][rows, g].double() @ key.T * d ** -0.5).masked_fill(~seen, -math.inf)
                    lse[rows, g] = torch.logsumexp(logits, 1)
                    out[rows, g] = torch.softmax(logits, 1) @ value
        row += n
    return [out, lse]

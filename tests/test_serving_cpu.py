"""Serving-step operators: what the C entries and their wrappers refuse on the host, before any launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

from vllm_ascend_kvcompress import _native as N
from vllm_ascend_kvcompress.methods.triattention import kernels as K

FAKE = ctypes.c_void_p(0x1000)


def tables(**kw):
    a = dict(computed=FAKE, cb=4, scheduled=FAKE, sb=4, offsets=None, R=2, pages=FAKE, pb=4, stride=8, width=8, bpp=1,
             n=4, blocks=8, o0=FAKE, o1=FAKE, o2=FAKE, o3=FAKE, o4=FAKE, o5=FAKE, err=None, stream=None)
    a.update(kw)
    return N.lib().kvc_step_tables(*a.values())


def test_step_tables_refusals():
    for name in ("computed", "scheduled", "pages", "o0", "o1", "o2", "o3", "o4", "o5"):
        assert tables(**{name: None}) == -14, name
    for bad in ({"R": 0}, {"n": -1}, {"blocks": -1}, {"width": 0}, {"bpp": 0}, {"cb": 2}, {"sb": 1}, {"pb": 16},
                {"stride": -1}, {"n": 1 << 31}):
        assert tables(**bad) == -22, bad
    assert tables(R=8193) == -95


def rotary(**kw):
    a = dict(q=FAKE, q0=512, q1=128, k=FAKE, k0=256, k1=128, v=FAKE, v0=256, v1=128, dtype=0, n=4, heads=4, kvh=2,
             dim=128, rot=128, pos=FAKE, axes=1, ps=0, omega=FAKE, axis=None, slots=FAKE, out=FAKE, o0=512, o1=128,
             kc=FAKE, kb=128 * 256, vc=FAKE, vb=128 * 256, blocks=10, err=None, stream=None)
    a.update(kw)
    return N.lib().kvc_rotary_write(*a.values())


def test_rotary_write_refusals():
    for name in ("q", "k", "v", "pos", "omega", "slots", "out", "kc", "vc"):
        assert rotary(**{name: None}) == -14, name
    assert rotary(axes=3) == -14  # several axes need the axis of each frequency
    for bad in ({"dtype": 2}, {"n": -1}, {"heads": 0}, {"kvh": 0}, {"blocks": 0}, {"rot": 0}, {"rot": 144},
                {"axes": 0}, {"axes": 9}, {"kb": 128 * 256 - 8}, {"ps": -1}, {"o0": 0}, {"o1": 0}):
        assert rotary(**bad) == -22, bad
    for bad in ({"rot": 24}, {"dim": 132, "rot": 128}, {"dim": 512, "rot": 272, "kb": 1 << 20, "vb": 1 << 20}):
        assert rotary(**bad) == -95, bad
    for bad in ({"q0": 513}, {"k1": 130}, {"o0": 516}, {"vb": 128 * 256 + 4}, {"q": ctypes.c_void_p(0x1002)},
                {"kc": ctypes.c_void_p(0x1008)}, {"v0": -256}):
        assert rotary(**bad) == -71, bad
    assert rotary(n=0, q=None) == 0  # nothing to do, nothing launched


def attend(**kw):
    a = dict(q=FAKE, q0=512, q1=128, dtype=0, n=4, longest=1, heads=4, kvh=2, dim=128, kc=FAKE, kb=128 * 256, vc=FAKE,
             vb=128 * 256, blocks=10, table=FAKE, ts=8, tw=8, starts=FAKE, lens=FAKE, R=4, scale=0.1, window=0,
             sinks=0, out=FAKE, o0=512, o1=128, lse=None, ws=FAKE, wsize=1 << 40, err=None, stream=None)
    a.update(kw)
    return N.lib().kvc_paged_attention(*a.values())


def test_paged_attention_refusals():
    for name in ("q", "kc", "vc", "table", "starts", "lens", "out", "ws"):
        assert attend(**{name: None}) == -14, name
    for bad in ({"dtype": 5}, {"n": -1}, {"longest": -1}, {"heads": 5}, {"heads": 0}, {"blocks": 0}, {"window": -1},
                {"sinks": -4}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")}, {"scale": float("inf")},
                {"kb": 128 * 256 - 8}, {"R": -1}, {"tw": -1}):
        assert attend(**bad) == -22, bad
    for bad in ({"dim": 96}, {"heads": 34}, {"R": 8193}):
        assert attend(**bad) == -95, bad
    for bad in ({"q0": 516}, {"o1": 4}, {"q": ctypes.c_void_p(0x1008)}, {"ws": ctypes.c_void_p(0x1008)},
                {"vb": 128 * 256 + 4}):
        assert attend(**bad) == -71, bad
    assert attend(wsize=1000) == -22
    for none in ({"R": 0}, {"n": 0}, {"longest": 0}):
        assert attend(**none) == 0, none  # nothing to do, nothing launched


def test_workspace_size_of_unsupported_geometries_is_zero():
    size = N.lib().kvc_paged_attention_workspace_bytes
    assert size(1, 40, 8, 128) > 0 and size(1, 16, 2, 256) > size(1, 16, 2, 64) > 0
    assert size(1, 40, 7, 128) == size(1, 40, 8, 96) == size(1, 34, 2, 128) == size(-1, 40, 8, 128) == 0


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    cache = torch.zeros(3, 128, 4, 128, dtype=torch.bfloat16)
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.step_tables(i32, i32, i32[:, None], num_tokens=2, max_blocks=1)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.rotary_write(x, x, x, i32.long(), i32.long(), cache, cache, omega=torch.ones(64))
    with pytest.raises(RuntimeError, match="CUDA"):
        K.paged_attention(x, cache, cache, i32[:, None], torch.zeros(3, dtype=torch.int32), i32, max_query_len=1)

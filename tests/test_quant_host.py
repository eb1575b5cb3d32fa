"""Refusals of the 8-bit cache's entry points, on the host, before any launch."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from paged_serve_b200 import _lib, ops


def _msg():
    return _lib.load().ps_last_error_string().decode()


def _append(**kw):
    a = dict(t=4, ks=256, vs=256, hkv=2, d=128, bs=16, nb=8, dtype=2, code=1, pool=16, rope=False)
    a.update(kw)
    lib = _lib.load()
    head = [a["pool"], 16, 16, 16, 16, 16, 16]
    geo = [a["t"], a["ks"], a["vs"], a["hkv"], a["d"], a["bs"], a["nb"]]
    if a["rope"]:
        return lib.ps_cache_append_rope_quant(*head, a.get("pos", 16), *geo, a.get("table", 16), 10,
                                              a.get("rope_dim", a["d"]), a["dtype"], a["code"], None, None)
    return lib.ps_cache_append_quant(*head, *geo, a["dtype"], a["code"], None, None)


def test_append_refusals():
    assert _append(dtype=3) == _lib.PS_ERR_UNSUPPORTED and "dtype" in _msg()
    assert _append(code=3) == _lib.PS_ERR_UNSUPPORTED and "code" in _msg()
    assert _append(d=96) == _lib.PS_ERR_UNSUPPORTED
    assert _append(t=-1) == _lib.PS_ERR_INVALID
    assert _append(t=0) == _lib.PS_OK
    assert _append(pool=None) == _lib.PS_ERR_INVALID
    assert _append(pool=8) == _lib.PS_ERR_INVALID and "aligned" in _msg()
    assert _append(ks=128) == _lib.PS_ERR_INVALID
    assert _append(ks=260) == _lib.PS_ERR_INVALID
    assert _append(nb=1 << 40) == _lib.PS_ERR_INVALID
    assert _append(t=1 << 60) == _lib.PS_ERR_INVALID
    assert _append(rope=True, rope_dim=64) == _lib.PS_ERR_UNSUPPORTED
    assert _append(rope=True, table=None) == _lib.PS_ERR_INVALID
    assert _append(rope=True, pos=None) == _lib.PS_ERR_INVALID


def _read(**kw):
    a = dict(nb=8, onb=8, ts=4, ots=4, b=2, hkv=2, d=128, bs=16, mb=4, dtype=2, code=2, out=16)
    a.update(kw)
    return _lib.load().ps_cache_read_quant(16, 16, 16, 16, a["nb"], a["out"], 16, a["onb"], 16, a["ts"], 16,
                                           a["ots"], 16, a["b"], a["hkv"], a["d"], a["bs"], a["mb"],
                                           a["dtype"], a["code"], None, None)


def test_read_refusals():
    assert _read(dtype=0) == _lib.PS_ERR_UNSUPPORTED
    assert _read(code=0) == _lib.PS_ERR_UNSUPPORTED
    assert _read(d=32) == _lib.PS_ERR_UNSUPPORTED
    assert _read(b=0) == _lib.PS_OK
    assert _read(b=70000) == _lib.PS_ERR_INVALID
    assert _read(onb=0) == _lib.PS_ERR_INVALID
    assert _read(ts=3) == _lib.PS_ERR_INVALID
    assert _read(ots=3) == _lib.PS_ERR_INVALID
    assert _read(out=None) == _lib.PS_ERR_INVALID
    assert _read(out=24) == _lib.PS_ERR_INVALID
    assert _read(mb=1 << 28, ts=1 << 28, ots=1 << 28) == _lib.PS_ERR_INVALID


def _decode(**kw):
    a = dict(os=1024, qs=1024, ks=16, nb=8, bts=4, b=2, order=None, listed=-1, hq=8, hkv=2, d=128, bs=16, mb=4,
             split=0, planned=0, ws=None, wsb=0, dtype=2, code=1)
    a.update(kw)
    return _lib.load().ps_paged_decode_quant(
        16, a["os"], 16, a["qs"], 16, 16, a["ks"], 16, a["nb"], 16, a["bts"], 16, a["b"], a["order"],
        a["listed"], a["hq"], a["hkv"], a["d"], a["bs"], a["mb"], 0.1, a["split"], a["planned"], a["ws"], a["wsb"],
        a["dtype"], a["code"], None, None)


def test_decode_refusals():
    assert _decode(code=7) == _lib.PS_ERR_UNSUPPORTED
    assert _decode(dtype=7) == _lib.PS_ERR_UNSUPPORTED
    assert _decode(d=256) == _lib.PS_ERR_UNSUPPORTED
    assert _decode(bs=4) == _lib.PS_ERR_UNSUPPORTED
    assert _decode(hq=34, os=34 * 128, qs=34 * 128) == _lib.PS_ERR_UNSUPPORTED
    assert _decode(hq=9) == _lib.PS_ERR_INVALID
    assert _decode(ks=None) == _lib.PS_ERR_INVALID and "scale" in _msg()
    assert _decode(ks=20) == _lib.PS_ERR_INVALID
    assert _decode(listed=1) == _lib.PS_ERR_INVALID
    assert _decode(listed=3, order=16) == _lib.PS_ERR_INVALID
    assert _decode(listed=0) == _lib.PS_OK
    assert _decode(listed=0, planned=1) == _lib.PS_ERR_INVALID and "plan" in _msg()
    assert _decode(b=0) == _lib.PS_OK
    assert _decode(split=24) == _lib.PS_ERR_INVALID
    assert _decode(split=16) == _lib.PS_ERR_INVALID and "workspace" in _msg()
    assert _decode(split=16, ws=256, wsb=100) == _lib.PS_ERR_INVALID


def test_plan_refusals():
    def plan(b=4, mb=64, split=16, ws=256, wsb=1 << 62):
        return _lib.load().ps_paged_decode_plan(16, b, None, 8, 128, 16, mb, split, ws, wsb, None)

    assert plan(ws=None) == _lib.PS_ERR_INVALID and "workspace" in _msg()
    assert plan(ws=16) == _lib.PS_ERR_INVALID
    assert plan(wsb=100) == _lib.PS_ERR_INVALID and "workspace" in _msg()
    assert plan(split=24) == _lib.PS_ERR_INVALID
    # 65,535 sequences of 40,000 partitions: more units than 32 bits count
    assert plan(b=65535, mb=40000) == _lib.PS_ERR_INVALID and "units" in _msg()
    assert plan(mb=1) == _lib.PS_OK  # nothing is split


def test_ops_refuse_host_tensors():
    kp = torch.zeros((2, 1, 16, 64), dtype=torch.int8)
    sc = torch.zeros((2, 1, 16))
    x = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    slots = torch.zeros(1, dtype=torch.int64)
    tables = torch.zeros((1, 2), dtype=torch.int32)
    n = torch.ones(1, dtype=torch.int32)
    out = torch.zeros((2, 1, 16, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.cache_append_quant(kp, kp, sc, sc, x, x, slots)
    with pytest.raises(ValueError, match="CUDA"):
        ops.cache_read_quant(kp, kp, sc, sc, tables, n, out, out, tables)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_decode_quant(x, kp, kp, sc, sc, tables, n, 1.0)


def test_quant_pools_are_checked():
    kp = torch.zeros((2, 1, 16, 64), dtype=torch.int8)
    sc = torch.zeros((2, 1, 16))
    assert ops._check_quant_pools(kp, kp, sc, sc) == _lib.PS_CODE_INT8
    f8 = kp.view(torch.float8_e4m3fn)
    assert ops._check_quant_pools(f8, f8, sc, sc) == _lib.PS_CODE_E4M3
    for bad in ((kp.to(torch.uint8), kp, sc, sc), (kp, f8, sc, sc), (kp, kp[:1], sc, sc), (kp, kp, sc[:1], sc),
                (kp, kp, sc, sc.double()), (kp, kp, sc.transpose(0, 2), sc), (kp[0], kp, sc, sc)):
        with pytest.raises(ValueError):
            ops._check_quant_pools(*bad)


def _shared(**kw):
    a = dict(b=4, starts=16, groups=2, shared=16, max_group=2, max_shared=64, hq=8, hkv=2, d=128, bs=16, mb=8,
             split_keys=0, split=0, ws=256, wsb=1 << 30, dtype=2)
    a.update(kw)
    return _lib.load().ps_paged_decode_shared(
        16, 1024, 16, 1024, 16, 16, 8, 16, a["mb"], 16, a["b"], a["starts"], a["groups"], a["shared"],
        a["max_group"], a["max_shared"], a["hq"], a["hkv"], a["d"], a["bs"], a["mb"], 0.1, a["split_keys"],
        a["split"], a["ws"], a["wsb"], a["dtype"], None, None, None)


def test_shared_refusals():
    assert _shared(dtype=3) == _lib.PS_ERR_UNSUPPORTED
    assert _shared(d=32) == _lib.PS_ERR_UNSUPPORTED
    assert _shared(b=0) == _lib.PS_OK
    assert _shared(max_shared=-1) == _lib.PS_ERR_INVALID
    assert _shared(max_shared=129) == _lib.PS_ERR_INVALID and "max_shared" in _msg()
    assert _shared(split_keys=64) == _lib.PS_ERR_INVALID
    assert _shared(groups=5) == _lib.PS_ERR_INVALID
    assert _shared(max_group=5) == _lib.PS_ERR_INVALID
    assert _shared(starts=None) == _lib.PS_ERR_INVALID
    assert _shared(shared=None) == _lib.PS_ERR_INVALID
    assert _shared(ws=None) == _lib.PS_ERR_INVALID and "workspace" in _msg()
    assert _shared(wsb=100) == _lib.PS_ERR_INVALID
    assert _shared(ws=16) == _lib.PS_ERR_INVALID


def test_shared_workspace_and_pieces():
    size = ops.decode_shared_workspace_bytes
    one = size(4, 8, 128, 16, 8, 64, 0, 0)
    assert one == 2 * (4 * 8 * 128 * 4 + 4 * 8 * 8)  # two partials a piece
    assert size(4, 8, 128, 16, 80, 1280, 128, 0) == 10 * one
    assert size(4, 8, 128, 16, 8, 0, 0, 0) == 0
    assert size(4, 8, 128, 16, 8, 64, (1 << 31) - 128, 0) == one  # one piece, however long
    assert size(4, 8, 128, 16, 8, 64, -128, 0) == 0 and size(4, 8, 128, 16, 8, -1, 0, 0) == 0
    assert size(4, 8, 128, 16, 8, 64, 0, 32) == one + ops.decode_workspace_bytes(4, 8, 128, 16, 8, 32)
    # 256 rows x 4 heads = 4 pairs of tiles x 8 KV heads = 32 items: four pieces of 16 tiles
    # are one wave of 128 units
    assert ops.shared_split_keys([256], 32, 8, 8192, 148) == 2048
    assert ops.shared_split_keys([256], 32, 8, 128, 148) == 0
    assert ops.shared_split_keys([], 32, 8, 8192, 148) == 0
    for sizes, hq, hkv, keys in (([8], 64, 8, 32768), ([17, 3, 40], 14, 2, 2000), ([1], 8, 8, 64), ([500], 16, 1, 100000)):
        split = ops.shared_split_keys(sizes, hq, hkv, keys, 148)
        assert split % 128 == 0 and 0 <= split < keys


@pytest.mark.parametrize("qmax", [448.0, 127.0])
def test_division_by_the_code_range(qmax):
    """fma(x, hi, x * lo) with hi + lo ~ 1 / qmax is x / qmax, rounded once, for every significand.

    Both sides scale with powers of two, so x runs over the 2^23 integers of 24 bits. The sum
    x * hi + fl(x * lo) is held exactly, as an integer multiple of 2^-36: hi is a multiple of 2^-32
    (1/512 < hi), and a product rounded to 24 bits of at least 2^-13 one of 2^-36.
    """
    x = np.arange(1 << 23, 1 << 24, dtype=np.int64)
    hi = np.float32(1.0 / qmax)
    lo = np.float32(1.0 / qmax - float(hi))
    small = (x.astype(np.float32) * lo).astype(np.float64) * 2.0**36
    assert np.array_equal(small, np.rint(small))
    exact = x * np.int64(float(hi) * 2.0**36) + small.astype(np.int64)
    fma = exact.astype(np.float32) * np.float32(2.0**-36)  # one rounding; the scaling is exact
    assert np.array_equal(fma, x.astype(np.float32) / np.float32(qmax))

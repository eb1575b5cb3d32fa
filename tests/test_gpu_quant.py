"""GPU parity of the 8-bit KV cache: append, read back, decode, and a run of them together."""

from __future__ import annotations

import math

import pytest
import torch

from paged_serve_b200 import _lib, ops
from paged_serve_b200.rope import cos_sin_table
from tests.gpu_util import random_tables
from tests.quant_util import assert_within, attend, dequantise, quantise, rotate, sequence

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
CODES = [E4M3, INT8]
NAN = float("nan")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _empty_cache(nb, hkv, bs, d, code, fill=0):
    pools = [torch.full((nb, hkv, bs, d), fill, dtype=torch.uint8, device=DEV).view(code) for _ in range(2)]
    scales = [torch.full((nb, hkv, bs), NAN if fill else 0.0, device=DEV) for _ in range(2)]
    return *pools, *scales


def _random_cache(nb, hkv, bs, d, code, seed, k_gain=1.0, v_spread=0.5):
    g = _gen(seed)
    k = torch.randn((nb, hkv, bs, d), device=DEV, generator=g) * 0.5 * k_gain
    v = torch.randn((nb, hkv, bs, d), device=DEV, generator=g) * 0.5
    v *= torch.exp(v_spread * torch.randn((nb, hkv, bs, 1), device=DEV, generator=g))
    kp, ks = quantise(k, code)
    vp, vs = quantise(v, code)
    return kp, vp, ks, vs


def _spoil_tails(cache, tables, lens):
    """NaN codes (e4m3) and scales behind every sequence's last token and in unused blocks."""
    kp, vp, ks, vs = cache
    nb, _, bs, _ = kp.shape
    used = torch.zeros(nb, bs, dtype=torch.bool)
    for row, n in zip(tables, lens):
        for j in range((n + bs - 1) // bs):
            used[int(row[j]), : min(bs, n - j * bs)] = True
    stale = (~used).to(DEV)[:, None, :].expand(ks.shape)
    for pool, scale in ((kp, ks), (vp, vs)):
        pool.view(torch.uint8).masked_fill_(stale.unsqueeze(-1), 0x7F)
        scale.masked_fill_(stale, NAN)


def _decode(q, cache, tables, lens, split=0, **kw):
    b, hq, d = q.shape
    bs = cache[0].shape[2]
    need = ops.decode_workspace_bytes(b, hq, d, bs, tables.shape[1], split)
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=DEV) if split else None
    return ops.paged_decode_quant(q, *cache, tables, lens, 1.0 / math.sqrt(d), split, workspace=ws, **kw)


def _check_decode(out, q, cache, tables, lens, what=""):
    kp, vp, ks, vs = cache
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all(), f"{what}: an empty sequence's output is zeros"
            continue
        k = dequantise(sequence(kp, tables[b].to(DEV), n), sequence(ks, tables[b].to(DEV), n))
        v = dequantise(sequence(vp, tables[b].to(DEV), n), sequence(vs, tables[b].to(DEV), n))
        ref, weight = attend(q[b], k, v, 1.0 / math.sqrt(q.shape[-1]))
        assert_within(out[b], ref, weight, f"{what} sequence {b} ({n} keys)")


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hkv,d,bs,t", [(8, 128, 16, 1), (8, 128, 16, 257), (2, 64, 8, 63), (3, 64, 32, 1037),
                                        (1, 128, 5, 40)])
@pytest.mark.parametrize("rope", [False, True])
def test_append_is_bit_exact(code, dtype, hkv, d, bs, t, rope):
    g = _gen(t)
    nb = (t + bs - 1) // bs + 3
    fused = torch.randn((t, 3 * hkv, d), device=DEV, generator=g)
    fused = (fused * torch.exp(torch.randn((t, 3 * hkv, 1), device=DEV, generator=g))).to(dtype)
    key, value = fused[:, :hkv], fused[:, 2 * hkv:]  # rows strided over a wider buffer
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(t))[:t]
    slots[::7] = -1
    if t > 1:
        slots[1] = nb * bs - 1 if not (slots == nb * bs - 1).any() else slots[1]
    cache = _empty_cache(nb, hkv, bs, d, code)
    want = [x.clone() for x in cache]
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    k = key
    if rope:
        pos = torch.randint(0, 500, (t,), device=DEV, generator=g)
        table = cos_sin_table(d, 10000.0, 500, dtype, DEV)
        ops.cache_append_rope_quant(*cache, key, value, slots.to(DEV), pos, table, err)
        k = rotate(key, pos, table)
    else:
        ops.cache_append_quant(*cache, key, value, slots.to(DEV), err)
    for x, pool, scale in ((k, want[0], want[2]), (value, want[1], want[3])):
        codes, sc = quantise(x, code)
        for i, s in enumerate(slots.tolist()):
            if s >= 0:
                pool.view(torch.uint8)[s // bs, :, s % bs] = codes.view(torch.uint8)[i]
                scale[s // bs, :, s % bs] = sc[i]
    assert int(err) == 0
    for got, ref in zip(cache, want):
        same = got.view(torch.uint8) == ref.view(torch.uint8) if got.element_size() == 1 else got == ref
        assert same.all()


@pytest.mark.parametrize("code", CODES)
def test_append_special_rows(code):
    """Zeros, the type's extremes, tiny values, infinities and NaN, each in a row of its own."""
    d, hkv, bs = 64, 1, 16
    rows = torch.zeros(7, hkv, d)
    rows[1] = torch.finfo(torch.bfloat16).max
    rows[2, :, 3] = 1e-38
    rows[2, :, 5] = -2e-38
    rows[3, :, 0] = float("inf")
    rows[4, :, 0] = NAN
    rows[5] = torch.linspace(-3, 3, d)
    rows[6, :, 1] = 2.0**-133
    x = rows.to(torch.bfloat16).to(DEV)
    cache = _empty_cache(1, hkv, bs, d, code)
    ops.cache_append_quant(*cache, x, x, torch.arange(7, device=DEV))
    codes, scale = quantise(x, code)
    for r in (0, 1, 2, 5, 6):
        for pool, sc in ((cache[0], cache[2]), (cache[1], cache[3])):
            assert torch.equal(pool[0, 0, r].view(torch.uint8), codes[r, 0].view(torch.uint8)), r
            assert float(sc[0, 0, r]) == float(scale[r, 0]), r
    assert math.isnan(float(cache[2][0, 0, 3])) and math.isnan(float(cache[3][0, 0, 4]))
    out = torch.zeros((1, hkv, bs, d), device=DEV, dtype=torch.bfloat16)
    table = torch.zeros((1, 1), dtype=torch.int32, device=DEV)
    ops.cache_read_quant(*cache, table, torch.tensor([7], dtype=torch.int32, device=DEV), out, out.clone(), table)
    assert out[0, 0, 3].isnan().all() and out[0, 0, 4].isnan().all()
    assert (out[0, 0, 0] == 0).all() and out[0, 0, 1].isfinite().all()


def test_append_reports_bad_slots_and_positions():
    cache = _empty_cache(2, 2, 16, 64, E4M3)
    before = [c.clone() for c in cache]
    x = torch.ones((3, 2, 64), device=DEV, dtype=torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.cache_append_quant(*cache, x, x, torch.tensor([32, -1, 1 << 40], device=DEV), err)
    assert int(err) == _lib.PS_DEVERR_SLOT
    err.zero_()
    table = cos_sin_table(64, 10000.0, 8, torch.bfloat16, DEV)
    ops.cache_append_rope_quant(*cache, x, x, torch.tensor([0, 1, 2], device=DEV),
                                torch.tensor([8, -1, 1 << 33], device=DEV), table, err)
    assert int(err) == _lib.PS_DEVERR_POSITION
    for a, b in zip(cache, before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ------------------------------------------------------------------ read back
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hkv,d,bs", [(8, 128, 16), (2, 64, 8), (3, 64, 32), (1, 128, 4)])
def test_read_is_bit_exact(code, dtype, hkv, d, bs):
    lens = [0, 1, bs - 1, bs, bs + 1, 77, 300]
    nb = sum((n + bs - 1) // bs for n in lens) + 5
    cache = _random_cache(nb, hkv, bs, d, code, seed=bs)
    width = (max(lens) + bs - 1) // bs + 2
    tables = random_tables(lens, bs, nb, seed=1, width=width)
    out_tables = random_tables(lens, bs, nb + 2, seed=2, width=width)
    _spoil_tails(cache, tables, lens)
    k_out = torch.full((nb + 2, hkv, bs, d), 9.0, dtype=dtype, device=DEV)
    v_out = k_out.clone()
    want = [k_out.clone(), v_out.clone()]
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.cache_read_quant(*cache, tables.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), k_out,
                         v_out, out_tables.to(DEV), err)
    for b, n in enumerate(lens):
        for j in range((n + bs - 1) // bs):
            live = min(bs, n - j * bs)
            for x, (pool, scale) in enumerate(((cache[0], cache[2]), (cache[1], cache[3]))):
                src, dst = int(tables[b, j]), int(out_tables[b, j])
                want[x][dst] = 0
                want[x][dst, :, :live] = (pool[src, :, :live].float() * scale[src, :, :live, None]).to(dtype)
    assert int(err) == 0
    assert torch.equal(k_out, want[0]) and torch.equal(v_out, want[1])


def test_read_reports_bad_blocks_and_lengths():
    cache = _random_cache(4, 1, 16, 64, INT8, seed=3)
    out = torch.zeros((4, 1, 16, 64), dtype=torch.bfloat16, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)

    def read(table, out_table, n):
        err.zero_()
        ops.cache_read_quant(*cache, torch.tensor([table], dtype=torch.int32, device=DEV),
                             torch.tensor([n], dtype=torch.int32, device=DEV), out, out.clone(),
                             torch.tensor([out_table], dtype=torch.int32, device=DEV), err)
        return int(err)

    assert read([0, 4], [0, 1], 17) == _lib.PS_DEVERR_BLOCK_ID
    assert read([0, -1], [0, 1], 17) == _lib.PS_DEVERR_BLOCK_ID
    assert read([0, 1], [0, 9], 17) == _lib.PS_DEVERR_BLOCK_ID
    assert read([0, 99], [0, 99], 16) == 0  # the second block holds no token
    out.zero_()
    assert read([0, 1], [0, 1], 33) == _lib.PS_DEVERR_LENGTH
    assert (out == 0).all()


# ------------------------------------------------------------------ decode
LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 500, 1000]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d,bs", [(32, 8, 128, 16), (14, 2, 64, 16), (4, 4, 128, 8), (16, 1, 64, 32),
                                         (27, 3, 128, 32), (8, 1, 64, 8)])
@pytest.mark.parametrize("split", [0, 64])
def test_decode_vs_float64(code, dtype, hq, hkv, d, bs, split):
    nb = sum((n + bs - 1) // bs for n in LENS) + 7
    cache = _random_cache(nb, hkv, bs, d, code, seed=hq + d)
    tables = random_tables(LENS, bs, nb, seed=4, width=1024 // bs + 1)
    _spoil_tails(cache, tables, LENS)
    q = torch.randn((len(LENS), hq, d), device=DEV, generator=_gen(5)).to(dtype)
    lens = torch.tensor(LENS, dtype=torch.int32, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = _decode(q, cache, tables.to(DEV), lens, split, device_error=err)
    assert int(err) == 0
    _check_decode(out, q, cache, tables, LENS, f"{code} {dtype} {hq}/{hkv} d{d} bs{bs} split{split}")


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d,bs", [(32, 2, 128, 16), (27, 3, 128, 8), (20, 2, 128, 32), (30, 3, 64, 8),
                                         (12, 1, 64, 16)])
@pytest.mark.parametrize("split", [0, 64])
def test_decode_with_more_than_eight_heads_vs_float64(code, dtype, hq, hkv, d, bs, split):
    """Both head tiles, full and part full, at every block size."""
    nb = sum((n + bs - 1) // bs for n in LENS) + 7
    cache = _random_cache(nb, hkv, bs, d, code, seed=hq + bs)
    tables = random_tables(LENS, bs, nb, seed=31, width=1024 // bs + 1)
    _spoil_tails(cache, tables, LENS)
    q = torch.randn((len(LENS), hq, d), device=DEV, generator=_gen(32)).to(dtype)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = _decode(q, cache, tables.to(DEV), torch.tensor(LENS, dtype=torch.int32, device=DEV), split,
                  device_error=err)
    assert int(err) == 0
    _check_decode(out, q, cache, tables, LENS, f"{code} {dtype} {hq}/{hkv} d{d} bs{bs} split{split}")


@pytest.mark.parametrize("code", CODES)
def test_decode_with_wide_ranges(code):
    """Loud tokens among quiet ones (V scales over six decades, in rising and falling
    order), large scores and queries of large and small size."""
    hq, hkv, d, bs, n = 32, 8, 128, 16, 700
    nb = (n + bs - 1) // bs
    kp, vp, ks, vs = _random_cache(nb, hkv, bs, d, code, seed=8, k_gain=4.0)
    up = torch.logspace(-4, 2, nb * bs, device=DEV).view(nb, 1, bs)
    tables = torch.arange(nb, dtype=torch.int32).view(1, nb)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    for gain in (up, up.flip(0, 2), torch.full_like(up, 1e-30), torch.full_like(up, 1e30)):
        for qs in (1.0, 4.0, 1e-3):
            cache = (kp, vp, ks, vs * gain)
            q = (torch.randn((1, hq, d), device=DEV, generator=_gen(9)) * qs).to(torch.bfloat16)
            out = _decode(q, cache, tables.to(DEV), lens)
            v_abs = float((dequantise(vp, vs * gain)).abs().max())
            # values near 1e-30 and 1e30 are compared after bringing them to about 1
            norm = 1.0 / v_abs if v_abs < 1e-6 or v_abs > 1e6 else 1.0
            k = dequantise(sequence(kp, tables[0].to(DEV), n), sequence(ks, tables[0].to(DEV), n))
            v = dequantise(sequence(vp, tables[0].to(DEV), n), sequence(vs * gain, tables[0].to(DEV), n))
            ref, weight = attend(q[0], k, v * norm, 1.0 / math.sqrt(d))
            assert_within(out[0].double() * norm, ref, weight, f"wide range, q x {qs}", half=2.0**-8)


def test_decode_nan_stays_in_its_sequence():
    cache = _random_cache(8, 2, 16, 64, E4M3, seed=10)
    cache[2][1, 0, 3] = NAN  # a key of sequence 0, KV head 0
    tables = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32)
    lens = [32, 32, 20]
    q = torch.randn((3, 8, 64), device=DEV, generator=_gen(11)).to(torch.bfloat16)
    out = _decode(q, cache, tables.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    assert out[0, :4].isnan().all()
    assert out[0, 4:].isfinite().all() and out[1:].isfinite().all()


def test_decode_order_list_and_plan_give_the_same_bits():
    lens = [5, 400, 33, 0, 129, 64]
    hq, hkv, d, bs, split = 28, 4, 128, 16, 64
    nb = sum((n + bs - 1) // bs for n in lens) + 2
    cache = _random_cache(nb, hkv, bs, d, E4M3, seed=12)
    tables = random_tables(lens, bs, nb, seed=13).to(DEV)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = torch.randn((len(lens), hq, d), device=DEV, generator=_gen(14)).to(torch.float16)
    for sp in (0, split):
        base = _decode(q, cache, tables, ctx, sp)
        order = ops.decode_order(ctx)
        assert torch.equal(base, _decode(q, cache, tables, ctx, sp, seq_order=order))
        out = torch.full_like(base, 7.0)
        seqs = torch.tensor([4, 1], dtype=torch.int32, device=DEV)
        _decode(q, cache, tables, ctx, sp, seq_list=seqs, out=out)
        assert torch.equal(out[[1, 4]], base[[1, 4]]) and (out[[0, 2, 3, 5]] == 7.0).all()
        none = torch.full_like(base, 7.0)
        _decode(q, cache, tables, ctx, sp, seq_list=seqs[:0], out=none)
        assert (none == 7.0).all()
        # one plan for two calls, as the layers of a step use it
        need = ops.decode_workspace_bytes(len(lens), hq, d, bs, tables.shape[1], sp)
        ws = torch.empty(max(need, 256), dtype=torch.uint8, device=DEV)
        ops.decode_plan(ctx, ws, hq, d, bs, tables.shape[1], sp, seq_order=order)
        for _ in range(2):
            got = ops.paged_decode_quant(q, *cache, tables, ctx, 1.0 / math.sqrt(d), sp, workspace=ws,
                                         seq_order=order, planned=True)
            assert torch.equal(got, base)


def test_decode_rows_do_not_depend_on_the_batch():
    """A sequence's output has the same bits alone and in a batch, wherever its blocks lie."""
    lens = [700, 45, 260]
    bs = 16
    nb = 90
    cache = _random_cache(nb, 8, bs, 128, INT8, seed=15)
    tables = random_tables(lens, bs, nb, seed=16).to(DEV)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = torch.randn((3, 32, 128), device=DEV, generator=_gen(17)).to(torch.bfloat16)
    for split in (0, 128):
        whole = _decode(q, cache, tables, ctx, split)
        for b in range(3):
            one = _decode(q[b:b + 1], cache, tables[b:b + 1], ctx[b:b + 1], split)
            assert torch.equal(one[0], whole[b])
        assert torch.equal(whole, _decode(q, cache, tables, ctx, split))


def test_decode_strides_and_wide_tables():
    lens = [40, 7]
    cache = _random_cache(6, 2, 16, 64, E4M3, seed=18)
    wide = torch.full((2, 40), -5, dtype=torch.int32, device=DEV)  # entries past the context are never read
    wide[0, :3] = torch.tensor([5, 0, 2])
    wide[1, :1] = 4
    buf = torch.randn((2, 3, 14, 64), device=DEV, generator=_gen(19)).to(torch.bfloat16)
    out_buf = torch.full((2, 2, 14, 64), 3.0, device=DEV, dtype=torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    _decode(buf[:, 2], cache, wide[:, :20], ctx, out=out_buf[:, 1], device_error=err)
    assert int(err) == 0 and (out_buf[:, 0] == 3.0).all()
    _check_decode(out_buf[:, 1], buf[:, 2], cache, wide.cpu(), lens, "strided")


def test_decode_reports_bad_tables():
    cache = _random_cache(4, 2, 16, 64, E4M3, seed=20)
    q = torch.randn((2, 8, 64), device=DEV, generator=_gen(21)).to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    for split in (0, 16):
        err.zero_()
        _decode(q, cache, torch.tensor([[0, 4], [1, -1]], dtype=torch.int32, device=DEV),
                torch.tensor([20, 20], dtype=torch.int32, device=DEV), split, device_error=err)
        assert int(err) == _lib.PS_DEVERR_BLOCK_ID
        err.zero_()
        out = _decode(q, cache, torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV),
                      torch.tensor([33, 20], dtype=torch.int32, device=DEV), split, device_error=err)
        assert int(err) == _lib.PS_DEVERR_LENGTH and (out[0] == 0).all()
        err.zero_()
        _decode(q, cache, torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV),
                torch.tensor([20, 20], dtype=torch.int32, device=DEV), split, device_error=err,
                seq_list=torch.tensor([1, 2], dtype=torch.int32, device=DEV))
        assert int(err) == _lib.PS_DEVERR_LENGTH


def test_on_another_stream_and_in_graphs():
    """The launches go to the current stream; two graphs that share a split workspace
    replay in turn with the eager result."""
    lens = [300, 20, 90]
    bs, split = 16, 64
    cache = _random_cache(40, 8, bs, 128, E4M3, seed=22)
    tables = random_tables(lens, bs, 40, seed=23).to(DEV)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = torch.randn((3, 32, 128), device=DEV, generator=_gen(24)).to(torch.bfloat16)
    q2 = q.flip(1).contiguous()
    want, want2 = _decode(q, cache, tables, ctx, split), _decode(q2, cache, tables, ctx, split)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _decode(q, cache, tables, ctx, split)
    side.synchronize()
    assert torch.equal(got, want)
    ws = torch.empty(ops.decode_workspace_bytes(3, 32, 128, bs, tables.shape[1], split), dtype=torch.uint8,
                     device=DEV)
    graphs, outs = [], []
    for x in (q, q2):
        g, out = torch.cuda.CUDAGraph(), torch.empty_like(x)
        with torch.cuda.graph(g):
            ops.paged_decode_quant(x, *cache, tables, ctx, 128**-0.5, split, out=out, workspace=ws)
        graphs.append(g)
        outs.append(out)
    for _ in range(3):
        for out in outs:
            out.zero_()
        graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,at", [(64, 0), (128, 45), (64, 99)])
def test_decode_of_a_top_key_with_a_row_of_zeros(code, dtype, d, at):
    """The key with nearly all of the softmax has zeros for values (their scale 2^-126), and
    the others, 2^gap below it, have values of any size: finite, and the attention of the rest.

    Beside the roundings of assert_within, in units of the largest probability: a probability
    below 2^-126 may count as 0 (n 2^-126 max|v| in all); P b is held to 2^-25 2^-119 or better, which
    meets codes of at most 448 (n 2^-135); the output's smallest step."""
    hq, bs, n = 8, 16, 100
    nb = (n + bs - 1) // bs
    g = _gen(30)
    tables = torch.arange(nb, dtype=torch.int32).view(1, nb)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    q = torch.randn((1, hq, d), device=DEV, generator=g) * 0.1
    q[..., 0] = 1.0
    q = q.to(dtype)
    k = torch.randn((nb, 1, bs, d), device=DEV, generator=g)
    k[..., 0] = 0.0
    v = torch.randn((nb, 1, bs, d), device=DEV, generator=g)
    v /= v.abs().amax(-1, keepdim=True)
    v[at // bs, 0, at % bs] = 0.0
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the output's smallest step
    for gap in (0, 40, 100, 112, 118, 125, 127, 140, 210, 250):
        k[at // bs, 0, at % bs] = 0.0
        k[at // bs, 0, at % bs, 0] = gap * math.log(2.0)
        kp, ks = quantise(k, code)
        for size in (1e-30, 1.0, 6e4, 1e20, 1e30, 1e38):
            vp, vs = quantise(v * size, code)
            out = ops.paged_decode_quant(q, kp, vp, ks, vs, tables.to(DEV), lens, 1.0)
            kk = dequantise(sequence(kp, tables[0].to(DEV), n), sequence(ks, tables[0].to(DEV), n))
            vv = dequantise(sequence(vp, tables[0].to(DEV), n), sequence(vs, tables[0].to(DEV), n))
            ref, weight = attend(q[0], kk, vv, 1.0)
            # refused by the documentation: sum(p |v|) in units of the top probability, up to
            # 100 x 1e38 here, is formed in float32 (3.4e38); or beyond the output's range
            p_v = torch.softmax(torch.einsum("hd,nd->hn", q[0].double(), kk[0]), -1)
            if float((p_v / p_v.amax(-1, keepdim=True) @ vv[0].abs()).max()) > 2.0**127 or                     float(ref.abs().max()) > torch.finfo(dtype).max / 2:
                continue
            bound = (torch.finfo(dtype).eps / 2 * ref.abs() + 1.1 * 2.0**-11 * weight
                     + 2.0**-21 * weight.amax(-1, keepdim=True) + tiny / 2
                     + n * (2.0**-126 * float(vv.abs().max()) + 2.0**-135))
            err = (out[0].double() - ref).abs()
            assert (err <= bound).all(), (gap, size, float((err / bound).nan_to_num(nan=math.inf).max()))


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("code", CODES)
def test_prompt_then_decode_steps(code):
    """A prompt is appended and prefilled from the read-back pool, blocks are copied on
    write with the 16-bit cache's entry point, and decode steps follow; every
    attention output is checked against float64 over the cache's values."""
    hq, hkv, d, bs, dtype = 28, 4, 128, 16, torch.bfloat16
    prompts, steps = [70, 5, 33], 3
    nb = 24
    cache = _empty_cache(nb, hkv, bs, d, code, fill=0x7F)
    width = 6
    tables = random_tables([n + steps + bs for n in prompts], bs, nb, seed=25, width=width)
    dt = tables.to(DEV)
    g = _gen(26)
    rope = cos_sin_table(d, 10000.0, 128, dtype, DEV)
    held = list(prompts)
    ids = torch.cat([torch.arange(n) + (b << 20) for b, n in enumerate(prompts)])
    owner, pos = ids >> 20, ids & 0xFFFFF
    slots = tables[owner, pos // bs].long() * bs + pos % bs
    kv = torch.randn((len(ids), 2 * hkv, d), device=DEV, generator=g).to(dtype)
    ops.cache_append_rope_quant(*cache, kv[:, :hkv], kv[:, hkv:], slots.to(DEV), pos.to(DEV), rope)
    # prefill over the read-back tokens
    q = torch.randn((len(ids), hq, d), device=DEV, generator=g).to(dtype)
    pools = [torch.full((nb, hkv, bs, d), NAN, dtype=dtype, device=DEV) for _ in range(2)]
    ctx = torch.tensor(held, dtype=torch.int32, device=DEV)
    ops.cache_read_quant(*cache, dt, ctx, *pools, dt)
    starts = torch.tensor([0, prompts[0], prompts[0] + prompts[1]], dtype=torch.int32, device=DEV)
    zero = torch.zeros(3, dtype=torch.int32, device=DEV)
    out = ops.paged_prefill(q, *pools, dt, starts, ctx, zero, max(prompts), d**-0.5)
    for b, n in enumerate(prompts):
        k, v = (sequence(x, dt[b], n) for x in pools)
        for i in (0, n // 2, n - 1):
            ref, weight = attend(q[int(starts[b]) + i], k[:, : i + 1], v[:, : i + 1], d**-0.5)
            # the prefill rounds its probabilities to bf16: 2^-8 in place of fp16's 2^-11
            assert_within(out[int(starts[b]) + i], ref, weight * 8, f"prefill {b} row {i}")
    # copy-on-write: sequence 0's last block moves to a free block
    free = next(x for x in range(nb) if not (tables == x).any())
    old = int(tables[0, (held[0] - 1) // bs])
    pair = torch.tensor([[old, free]], device=DEV)
    ops.copy_blocks(cache[0], cache[1], pair)
    ops.copy_blocks(cache[2].unsqueeze(-1), cache[3].unsqueeze(-1), pair)
    cache[0].view(torch.uint8)[old] = 0x7F
    tables[0, (held[0] - 1) // bs] = free
    dt = tables.to(DEV)
    for _ in range(steps):
        pos = torch.tensor(held)
        slots = tables[torch.arange(3), pos // bs].long() * bs + pos % bs
        kv = torch.randn((3, 2 * hkv, d), device=DEV, generator=g).to(dtype)
        ops.cache_append_rope_quant(*cache, kv[:, :hkv], kv[:, hkv:], slots.to(DEV), pos.to(DEV), rope)
        held = [n + 1 for n in held]
        q = torch.randn((3, hq, d), device=DEV, generator=g).to(dtype)
        out = _decode(q, cache, dt, torch.tensor(held, dtype=torch.int32, device=DEV), 32)
        _check_decode(out, q, cache, tables, held, "step")

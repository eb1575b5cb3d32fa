"""GPU parity of shared-prefix decode against a plain float64 attention of each sequence."""

from __future__ import annotations

import math

import pytest
import torch

from paged_serve_b200 import _lib, ops
from tests.gpu_util import random_pool
from tests.quant_util import assert_within, attend, dequantise, quantise, sequence

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN = float("nan")


def _case(groups, own, bs, seed=0, spare=3):
    """Tables for groups [(rows, prefix tokens)] with own[b] tokens behind each prefix."""
    pre, starts = [], [0]
    for n, p in groups:
        assert p % bs == 0
        pre += [p] * n
        starts.append(starts[-1] + n)
    lens = [p + o for p, o in zip(pre, own)]
    need = sum(p // bs for _, p in groups) + sum((o + bs - 1) // bs for o in own)
    ids = torch.randperm(need + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(1, max((n + bs - 1) // bs for n in lens)) + 1
    tables = torch.zeros((len(lens), width), dtype=torch.int32)
    at, b = 0, 0
    for n, p in groups:
        head = ids[at:at + p // bs]
        at += p // bs
        for _ in range(n):
            m = (own[b] + bs - 1) // bs
            row = head + ids[at:at + m]
            at += m
            if row:
                tables[b, : len(row)] = torch.tensor(row, dtype=torch.int32)
            b += 1
    return pre, starts, lens, tables, need + spare


def _spoil_tails(pools, tables, lens):
    nb, _, bs, _ = pools[0].shape
    used = torch.zeros(nb, bs, dtype=torch.bool)
    for row, n in zip(tables, lens):
        for j in range((n + bs - 1) // bs):
            used[int(row[j]), : min(bs, n - j * bs)] = True
    for p in pools:
        p.masked_fill_((~used).to(DEV)[:, None, :, None], NAN)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _shared(q, pools, tables, lens, pre, starts, split_keys=0, split=0, **kw):
    sizes = [b - a for a, b in zip(starts, starts[1:])]
    return ops.paged_decode_shared(q, *pools, tables.to(DEV), _i32(lens), _i32(starts), _i32(pre),
                                   max(sizes, default=0), max(pre, default=0), q.shape[-1] ** -0.5,
                                   split_keys=split_keys, split_tokens=split, **kw)


def _check(out, q, pools, tables, lens, what, prob_half=2.0**-8):
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        k, v = (sequence(p, tables[b].to(DEV), n) for p in pools)
        ref, weight = attend(q[b], k, v, q.shape[-1] ** -0.5)
        # probabilities are rounded to the pools' type here, where assert_within counts fp16's half step
        assert_within(out[b], ref, weight * (prob_half / 2.0**-11), f"{what} row {b} ({n} keys)")


HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d,bs", [(32, 8, 128, 16), (14, 2, 64, 8), (4, 4, 128, 32), (16, 1, 64, 16),
                                         (27, 3, 128, 8), (8, 1, 64, 32)])
@pytest.mark.parametrize("split_keys,split", [(0, 0), (128, 0), (0, 64), (256, 32)])
def test_groups_vs_float64(dtype, hq, hkv, d, bs, split_keys, split):
    groups = [(5, 352), (1, 32), (3, 0), (40, 160), (2, 1024)]
    own = [(7 * i * i) % 131 for i in range(51)]
    own[0] = own[5] = own[8] = 0  # a row that ends with its prefix, a lone one, one with no keys at all
    own[6] = 0
    pre, starts, lens, tables, nb = _case(groups, own, bs)
    pools = random_pool(nb, hkv, bs, d, dtype, DEV, seed=hq)
    _spoil_tails(pools, tables, lens)
    q = torch.randn((len(lens), hq, d), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dtype)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    order = ops.decode_order(_i32([n - p for n, p in zip(lens, pre)]))
    out = _shared(q, pools, tables, lens, pre, starts, split_keys, split, device_error=err, seq_order=order)
    assert int(err) == 0
    _check(out, q, pools, tables, lens, f"{dtype} {hq}/{hkv} d{d} bs{bs} {split_keys}/{split}", HALF[dtype])
    # the same bits again, and without the order
    assert torch.equal(out, _shared(q, pools, tables, lens, pre, starts, split_keys, split))


def test_a_whole_batch_under_one_prefix():
    """More rows than a tile pair holds, and a prefix that ends inside a key tile."""
    groups, own = [(150, 432)], [i % 40 for i in range(150)]
    pre, starts, lens, tables, nb = _case(groups, own, 16)
    pools = random_pool(nb, 8, 16, 128, torch.bfloat16, DEV, seed=3)
    _spoil_tails(pools, tables, lens)
    q = torch.randn((150, 32, 128), device=DEV).to(torch.bfloat16)
    keys = ops.shared_split_keys([150], 32, 8, 432, 148)
    out = _shared(q, pools, tables, lens, pre, starts, keys)
    _check(out, q, pools, tables, lens, "one prefix")


def test_large_scores_in_either_part():
    """The softmax's weight wholly in the prefix for one row and behind it for another."""
    pre, starts, lens, tables, nb = _case([(2, 256)], [40, 40], 16)
    kp, vp = random_pool(nb, 1, 16, 64, torch.bfloat16, DEV, seed=4)
    q = torch.randn((2, 4, 64), device=DEV).to(torch.bfloat16)
    kp[int(tables[0, 3]), 0, 5] = q[0, 0] * 8
    kp[int(tables[1, 17]), 0, 2] = q[1, 0] * 8
    out = _shared(q, (kp, vp), tables, lens, pre, starts, 128)
    _check(out, q, (kp, vp), tables, lens, "large scores")


def test_nothing_shared_is_paged_decode():
    lens = [5, 0, 130]
    pre, starts, lens, tables, nb = _case([(3, 0)], lens, 16)
    pools = random_pool(nb, 2, 16, 64, torch.float16, DEV, seed=5)
    q = torch.randn((3, 8, 64), device=DEV).to(torch.float16)
    ref = ops.paged_decode(q, *pools, tables.to(DEV), _i32(lens), 0.125)
    assert torch.equal(_shared(q, pools, tables, lens, pre, starts), ref)
    # A maximum that no row uses: another instantiation runs, which promises the
    # same attention, not the same bits.
    out = ops.paged_decode_shared(q, *pools, tables.to(DEV), _i32(lens), _i32(starts), _i32(pre), 3, 16, 0.125)
    _check(out, q, pools, tables, lens, "nothing shared", HALF[torch.float16])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d,bs", [(32, 8, 128, 16), (14, 2, 64, 8), (16, 1, 64, 32)])
@pytest.mark.parametrize("split", [0, 32])
def test_nothing_shared_ignores_stale_rows(dtype, hq, hkv, d, bs, split):
    lens = [1, 7, 8, 0, 15, 16, 17, 33, 130, 255]
    pre, starts, lens, tables, nb = _case([(len(lens), 0)], lens, bs, seed=9)
    pools = random_pool(nb, hkv, bs, d, dtype, DEV, seed=10)
    _spoil_tails(pools, tables, lens)
    q = torch.randn((len(lens), hq, d), device=DEV).to(dtype)
    out = _shared(q, pools, tables, lens, pre, starts, split=split)
    _check(out, q, pools, tables, lens, "nothing shared", HALF[dtype])


def test_bad_lengths_are_reported():
    pre, starts, lens, tables, nb = _case([(2, 64), (2, 128)], [10, 20, 30, 40], 16)
    pools = random_pool(nb, 2, 16, 64, torch.bfloat16, DEV, seed=6)
    q = torch.randn((4, 8, 64), device=DEV).to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)

    def code(pre=pre, starts=starts, lens=lens, max_group=2, max_shared=128, tables=tables):
        err.zero_()
        for split in (0, 32):
            ops.paged_decode_shared(q, *pools, tables.to(DEV), _i32(lens), _i32(starts), _i32(pre), max_group,
                                    max_shared, 0.125, split_keys=128, split_tokens=split, device_error=err)
        return int(err)

    length = _lib.PS_DEVERR_LENGTH
    assert code() == 0
    assert code(pre=[60, 60, 128, 128]) == length  # not whole blocks
    assert code(pre=[-16, -16, 128, 128]) == length
    assert code(pre=[64, 32, 128, 128]) == length  # rows of a group differ
    assert code(pre=[64, 64, 144, 144]) == length  # more than max_shared
    assert code(lens=[60, 84, 158, 168]) == length  # a prefix longer than its sequence
    assert code(starts=[0, 2, 5]) == length
    assert code(starts=[-1, 2, 4]) == length
    assert code(starts=[0, 40, 80]) == length
    wide = _case([(40, 64)], [1] * 40, 16)
    pools40 = random_pool(wide[4], 2, 16, 64, torch.bfloat16, DEV, seed=7)
    err.zero_()  # more rows than max_group's tiles hold (4 heads: 64 rows a pair of tiles)
    big = torch.randn((40, 16, 64), device=DEV).to(torch.bfloat16)
    ops.paged_decode_shared(big, *pools40, wide[3].to(DEV), _i32(wide[2]), _i32([0, 40]), _i32(wide[0]), 1, 64,
                            0.125, device_error=err)
    assert int(err) == length
    bad = tables.clone()
    bad[0, 1] = nb
    assert code(tables=bad) & _lib.PS_DEVERR_BLOCK_ID


def test_rows_outside_their_group_are_reported():
    pre, starts, lens, tables, nb = _case([(2, 64), (2, 128), (3, 0), (1, 32)], [10, 20, 30, 40, 5, 6, 7, 8], 16)
    pools = random_pool(nb, 2, 16, 64, torch.bfloat16, DEV, seed=6)
    q = torch.randn((8, 8, 64), device=DEV).to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)

    def code(pre=pre, starts=starts, max_group=3):
        err.zero_()
        for group in (max_group, 8):
            for split in (0, 32):
                ops.paged_decode_shared(q, *pools, tables.to(DEV), _i32(lens), _i32(starts), _i32(pre), group,
                                        128, 0.125, split_keys=128, split_tokens=split, device_error=err)
        return int(err)

    length = _lib.PS_DEVERR_LENGTH
    assert code() == 0
    assert code(starts=[0, 2, 4, 4, 4, 7, 8]) == 0  # groups without rows
    assert code(starts=[0, 2, 3, 4, 7, 8]) == 0  # neighbours of one length in two groups
    assert code(pre=[0, 0, 128, 128, 0, 0, 0, 0], starts=[2, 4]) == 0  # rows in no group
    assert code(pre=[0] * 8, starts=[3, 3]) == 0
    assert code(starts=[0, 2, 4, 7]) == length  # the last row's prefix in no group
    assert code(starts=[2, 4, 7, 8]) == length  # the first rows'
    assert code(pre=[0, 64, 128, 128, 0, 0, 0, 32]) == length  # the first row of a group has none
    assert code(pre=[64, 64, 128, 128, 0, 16, 0, 32]) == length
    assert code(starts=[0, 2, 4, 3, 7, 8]) == length  # not in order
    assert code(pre=[64] * 8, starts=[0, 7], max_group=7) == length


@pytest.mark.parametrize("split", [0, 32])
def test_a_prefix_of_a_sequence_without_keys_is_reported(split):
    """A row of a group with a prefix but no keys at all breaks the rule as one with too few does."""
    pre, starts, lens, tables, nb = _case([(2, 64), (2, 0)], [10, 20, 30, 0], 16)
    pools = random_pool(nb, 2, 16, 64, torch.bfloat16, DEV, seed=11)
    q = torch.randn((4, 8, 64), device=DEV).to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = _shared(q, pools, tables, lens, pre, starts, 128, split, device_error=err)
    assert int(err) == 0 and (out[3] == 0).all()
    for empty in (0, -5):
        for row in (0, 1):
            err.zero_()
            bad = list(lens)
            bad[row] = empty
            _shared(q, pools, tables, bad, pre, starts, 128, split, device_error=err)
            assert int(err) == _lib.PS_DEVERR_LENGTH, (empty, row)
        err.zero_()  # without a prefix a row without keys is no error
        out = _shared(q, pools, tables, [*lens[:3], empty], pre, starts, 128, split, device_error=err)
        assert int(err) == 0 and (out[3] == 0).all()


@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 2), (32, 2)])
def test_a_group_longer_than_max_group_is_reported(hq, hkv):
    """Also where a query tile would hold the rows; a long group that shares nothing is none."""
    pre, starts, lens, tables, nb = _case([(3, 64), (5, 0), (2, 32)], [9] * 10, 16)
    pools = random_pool(nb, hkv, 16, 64, torch.bfloat16, DEV, seed=12)
    q = torch.randn((10, hq, 64), device=DEV).to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    for max_group, want in ((1, _lib.PS_DEVERR_LENGTH), (2, _lib.PS_DEVERR_LENGTH), (3, 0), (10, 0)):
        err.zero_()
        out = ops.paged_decode_shared(q, *pools, tables.to(DEV), _i32(lens), _i32(starts), _i32(pre), max_group, 64,
                                      0.125, device_error=err)
        assert int(err) == want, max_group
        if not want:
            _check(out, q, pools, tables, lens, f"max_group {max_group}")


def test_streams_and_graphs():
    """Another stream, and two captured calls that share a workspace replayed in turn,
    with the inputs of the calls written by the kernels just before them."""
    groups, own = [(6, 512), (2, 48)], [33, 1, 100, 17, 0, 60, 5, 70]
    pre, starts, lens, tables, nb = _case(groups, own, 16)
    pools = random_pool(nb, 8, 16, 128, torch.bfloat16, DEV, seed=8)
    dt, ctx, st, pr = tables.to(DEV), _i32(lens), _i32(starts), _i32(pre)
    src = [torch.randn((8, 32, 128), device=DEV).to(torch.bfloat16) for _ in range(2)]
    for split in (0, 32):
        ws = torch.empty(ops.decode_shared_workspace_bytes(8, 32, 128, 16, tables.shape[1], 512, 128, split),
                         dtype=torch.uint8, device=DEV)

        def call(q, out=None):
            return ops.paged_decode_shared(q, *pools, dt, ctx, st, pr, 6, 512, 128**-0.5, split_keys=128,
                                           split_tokens=split, out=out, workspace=ws)

        want = [call(q).clone() for q in src]
        _check(want[0], src[0], pools, tables, lens, "eager")
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = call(src[1])
        side.synchronize()
        assert torch.equal(got, want[1])
        graphs, outs = [], []
        for x in src:
            q, out = torch.zeros_like(x), torch.empty_like(x)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                q.copy_(x)
                call(q, out)
                again = call(out)  # reads what the call before it wrote
            graphs.append((g, again))
            outs.append(out)
        for _ in range(3):
            for g, _ in reversed(graphs):
                g.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert torch.equal(graphs[0][1], call(want[0]))


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
def test_over_a_read_back_cache(code):
    """A prefix held in 8 bits is read back once and shared by the batch; the decode of
    the 8-bit cache itself gives the same attention to the two kernels' roundings."""
    pre, starts, lens, tables, nb = _case([(9, 320)], [(11 * i) % 50 + 1 for i in range(9)], 16)
    g = torch.Generator(device=DEV).manual_seed(9)
    kp, ks = quantise(torch.randn((nb, 8, 16, 128), device=DEV, generator=g), code)
    vp, vs = quantise(torch.randn((nb, 8, 16, 128), device=DEV, generator=g), code)
    q = torch.randn((9, 32, 128), device=DEV, generator=g).to(torch.bfloat16)
    pools = [torch.full((nb, 8, 16, 128), NAN, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    dt = tables.to(DEV)
    ops.cache_read_quant(kp, vp, ks, vs, dt, _i32(lens), *pools, dt)
    out = _shared(q, pools, tables, lens, pre, starts, 128)
    _check(out, q, pools, tables, lens, "read back")
    direct = ops.paged_decode_quant(q, kp, vp, ks, vs, dt, _i32(lens), 128**-0.5)
    for b, n in enumerate(lens):
        k, v = (sequence(p, dt[b], n) for p in pools)
        ref, weight = attend(q[b], k, v, 128**-0.5)
        # the read-back values are off by bf16's half step, 2^-8 of v and, through the
        # scores (|s| <= 2^4 in all), at most 2^-8 * 2^4 of a probability
        assert_within(direct[b], ref, weight * (2.0**-4 + 2.0**-8) / 2.0**-11, f"row {b}")


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("split", [0, 32])
def test_a_read_back_prefix_and_the_codes_agree(code, split):
    """The decode over the codes against float64 over what the codes stand for, at its own
    roundings, on the tables of a shared prompt; and the shared path over the values read back
    against float64 over those."""
    pre, starts, lens, tables, nb = _case([(9, 320)], [(11 * i) % 50 + 1 for i in range(9)], 16, seed=2)
    g = torch.Generator(device=DEV).manual_seed(13)
    kp, ks = quantise(torch.randn((nb, 8, 16, 128), device=DEV, generator=g), code)
    vp, vs = quantise(torch.randn((nb, 8, 16, 128), device=DEV, generator=g), code)
    q = torch.randn((9, 32, 128), device=DEV, generator=g).to(torch.bfloat16)
    dt, ctx = tables.to(DEV), _i32(lens)
    ws = torch.empty(max(256, ops.decode_workspace_bytes(9, 32, 128, 16, dt.shape[1], split)), dtype=torch.uint8,
                     device=DEV)
    direct = ops.paged_decode_quant(q, kp, vp, ks, vs, dt, ctx, 128**-0.5, split, workspace=ws)
    pools = [torch.full((nb, 8, 16, 128), NAN, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    ops.cache_read_quant(kp, vp, ks, vs, dt, ctx, *pools, dt)
    out = _shared(q, pools, tables, lens, pre, starts, 128, split)
    for b, n in enumerate(lens):
        k, v = (dequantise(sequence(c, dt[b], n), sequence(s, dt[b], n)) for c, s in ((kp, ks), (vp, vs)))
        ref, weight = attend(q[b], k, v, 128**-0.5)
        assert_within(direct[b], ref, weight, f"codes, row {b}")
    _check(out, q, pools, tables, lens, "read back")

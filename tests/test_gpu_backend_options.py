"""PagedCudaBackend with an 8-bit cache (kv_codes) and with shared prefixes (share_prefixes)."""

from __future__ import annotations

import random
import time
import weakref
from array import array

import pytest
import torch

from oracle import contiguous_attention
from paged_serve_b200 import backend as backend_module
from paged_serve_b200.backend import PagedCudaBackend, shared_groups
from paged_serve_b200.config import ModelConfig
from paged_serve_b200.graphs import DecodeGraph
from paged_serve_b200.interface import StepInput
from tests.gpu_util import assert_attention_close
from tests.quant_util import dequantise, quantise

DEV = "cuda"
BS = 16
CODES = [torch.float8_e4m3fn, torch.int8]
MODEL = ModelConfig(name="gqa4", num_layers=2, num_q_heads=8, num_kv_heads=2, head_dim=128)


class TestGroups:
    """The host's choice of groups (no GPU)."""

    def test_a_common_prompt(self):
        tables = [[1, 2, 3, 10], [1, 2, 3, 11], [1, 2, 3, 12]]
        assert shared_groups(tables, [50, 60, 64], 16, 1) == ([0, 3], [48, 48, 48])

    def test_the_newest_token_is_never_in_the_prefix(self):
        tables = [[1, 2, 3], [1, 2, 3]]
        assert shared_groups(tables, [48, 48], 16, 1) == ([0, 2], [32, 32])
        assert shared_groups(tables, [16, 48], 16, 1) is None

    def test_neighbours_split_where_the_prefix_would_shrink_too_far(self):
        a, b = [1, 2, 3, 4, 5], [1, 8, 9]
        tables = [a + [20], a + [21], b + [22], b + [23], [7]]
        assert shared_groups(tables, [90, 90, 60, 60, 5], 16, 1) == ([0, 2, 4, 5], [80, 80, 48, 48, 0])

    def test_a_saving_too_small_is_none(self):
        tables = [[1, 2], [1, 3]]
        assert shared_groups(tables, [20, 20], 16, 17) is None
        assert shared_groups(tables, [20, 20], 16, 16) == ([0, 2], [16, 16])
        assert shared_groups([], [], 16, 1) is None
        assert shared_groups([[], [5]], [0, 1], 16, 1) is None

    def test_every_first_difference(self):
        """Two tables that agree in any number of blocks, as arrays, as lists and as one of each."""
        base = list(range(100, 121))
        for n in range(len(base) + 1):
            other = base[:n] + [-1] * (len(base) - n)
            # 20 whole blocks lie before the newest of 336 tokens
            want = ([0, 2], [16 * min(n, 20)] * 2) if n else None
            for a, b in ((base, other), (array("i", base), array("i", other)), (array("i", base), other)):
                assert shared_groups([a, b], [336, 336], 16, 1) == want

    def test_as_the_comparison_block_by_block(self):
        rng = random.Random(3)
        for _ in range(300):
            heads = [[rng.randrange(4) for _ in range(rng.randrange(1, 9))] for _ in range(3)]
            tables, lens = [], []
            for i in range(rng.randrange(1, 9)):
                t = list(rng.choice(heads))[: rng.randrange(0, 9)] + [100 + i] * rng.randrange(0, 3)
                tables.append(array("i", t))
                lens.append(rng.randrange(0, len(t) * 4 + 1))
            got = shared_groups(tables, lens, 4, 1)
            starts, pre, i = [0], [], 0
            while i < len(tables):
                limit = [min(len(t), max(x - 1, 0) // 4) for t, x in zip(tables, lens)]
                common, j = limit[i], i + 1
                while j < len(tables):
                    c = 0
                    while c < min(common, limit[j]) and tables[j][c] == tables[i][c]:
                        c += 1
                    if c == 0 or (j - i) * c < (j - i - 1) * common:
                        break
                    common, j = c, j + 1
                pre += [4 * common if j - i > 1 else 0] * (j - i)
                starts.append(j)
                i = j
            saved = sum((z - a - 1) * pre[a] for a, z in zip(starts, starts[1:]))
            assert got == ((starts, pre) if saved else None)

    @pytest.mark.parametrize("shared", [True, False])
    def test_the_search_is_short_beside_a_step(self, shared):
        """256 rows over 8,192 tokens, whose attention takes 2.5 ms or more over 32 layers."""
        common = list(range(512))
        tables = [array("i", (common if shared else [1000 + i] * 512) + [5000 + i]) for i in range(256)]
        lens = [8192 + 7] * 256
        times = []
        for _ in range(9):
            start = time.perf_counter()
            got = shared_groups(tables, lens, 16, 1)
            times.append(time.perf_counter() - start)
        assert got == (([0, 256], [8192] * 256) if shared else None)
        assert min(times) < 3e-3, f"{min(times) * 1e3:.2f} ms"  # 0.2 to 0.6; id by id 6 to 11


def test_options_are_checked():
    with pytest.raises(ValueError, match="kv_codes"):
        PagedCudaBackend(MODEL, device="cpu", dtype=torch.bfloat16, kv_codes=torch.uint8)
    with pytest.raises(ValueError, match="share_prefixes"):
        PagedCudaBackend(MODEL, device="cpu", dtype=torch.bfloat16, kv_codes=torch.int8, share_prefixes=True)


@pytest.mark.parametrize("code", CODES)
def test_an_8_bit_reservation_is_reported(code):
    be = PagedCudaBackend(MODEL, device="cpu", dtype=torch.bfloat16, kv_codes=code)
    be.allocate(2, 64)
    row = 128 + 4  # codes and scale of one token and KV head
    assert be.memory_stats().allocated_bytes == 2 * 2 * 8 * 16 * 2 * row
    assert be.block_usage()["held_bytes"] == 8 * 16 * 2 * 2 * 2 * row
    be.free()
    assert be.k_scale is None and be.memory_stats().allocated_bytes == 0


@pytest.mark.parametrize("code", CODES)
def test_a_steps_scratch_lives_as_long_as_its_metadata(code):
    """A captured graph holds the addresses that its step was planned with: a later, larger step
    takes a pool of its own."""
    be = PagedCudaBackend(MODEL, device="cpu", dtype=torch.bfloat16, kv_codes=code)
    be.allocate(2, 64)
    zeros = torch.zeros(2, dtype=torch.int32)
    tables = torch.arange(4, dtype=torch.int32).view(2, 2)
    base = backend_module.PagedMetadata(
        query_len=2, context_len=0, key_len=32, num_seqs=2, block_tables=tables, slot_mapping=zeros.long(),
        positions=zeros.long(), ctx_lens=zeros, ctx_before=zeros, q_lens=zeros, q_starts=zeros, live_tokens=zeros)
    first = be._plan_read(base, tables, zeros, 4)
    held = [weakref.ref(x) for x in be._scratch]
    second = be._plan_read(base, tables, zeros, 400)
    assert be._scratch[0].shape[0] == 400 and all(r() is not None and r().shape[0] == 4 for r in held)
    assert first.read_tables is not None and second.read_tables is not None  # both still in use


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["read back", "shared prefix", "split prefill"])
def test_a_captured_step_survives_a_larger_one(kind, monkeypatch):
    """forward() captured with one step's metadata, replayed after a step that needed more
    scratch or workspace: the same outputs, and no write to memory that others now hold."""
    monkeypatch.setattr(backend_module, "SHARED_MIN_VALUES", 1)
    be = PagedCudaBackend(MODEL, device=DEV, dtype=torch.bfloat16, num_blocks=1400, split_tokens=32,
                          kv_codes=torch.int8 if kind == "read back" else None,
                          share_prefixes=kind == "shared prefix")
    be.allocate(24, 8192)
    mgr = be.make_block_manager(enable_prefix_caching=kind == "shared prefix")
    if kind != "read back":
        be.k_cache.normal_(0.0, 0.5)
        be.v_cache.normal_(0.0, 0.5)
    rng = torch.Generator().manual_seed(5)
    new_id = iter(range(100))

    def plan(rows, prompt, prefix):
        """A prefill of `prompt` new tokens a row, or (prefix > 0) a decode behind a common prompt."""
        common = torch.randint(0, 50000, (prefix,), generator=rng).tolist()
        ids = [next(new_id) for _ in range(rows)]
        for i in ids:
            own = torch.randint(0, 50000, (prompt,), generator=rng).tolist()
            mgr.allocate(i, prefix + prompt, common + own)
            if prefix:
                mgr.schedule([i])
                mgr.append_slots(i, 1, [7])
        return mgr.schedule(ids)

    def size():
        held = {"read back": be._scratch and be._scratch[0], "shared prefix": be._shared_ws,
                "split prefill": be._prefill_ws}[kind]
        return 0 if held is None else held.numel() * held.element_size()

    small = {"read back": (2, 40, 0), "shared prefix": (3, 9, 64), "split prefill": (1, 2000, 0)}[kind]
    large = {"read back": (2, 900, 0), "shared prefix": (20, 9, 1024), "split prefill": (1, 6000, 0)}[kind]
    p = plan(*small)
    md = be.begin_plan(p)
    first = size()
    assert first > 0 and (kind != "shared prefix" or md.group_starts is not None)
    b, tq = len(p.seq_ids), p.query_len
    q, k, v = ((torch.randn((b, tq, h, 128), generator=rng) * 0.5).to(torch.bfloat16).to(DEV) for h in (8, 2, 2))
    want = be.forward(0, q, k, v, md).clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = be.forward(0, q, k, v, md)
    be.begin_plan(plan(*large))
    assert size() > first
    torch.cuda.synchronize()
    junk = [torch.full((first,), 77, dtype=torch.uint8, device=DEV) for _ in range(64)]
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert all((j == 77).all() for j in junk)
    assert int(be.device_error) == 0


@pytest.mark.parametrize("layers,heads,rows,prefix,worth", [
    (32, (32, 8, 128), 16, 4096, False), (32, (32, 8, 128), 64, 2048, True), (80, (64, 8, 128), 64, 512, False),
    (80, (64, 8, 128), 64, 1024, True), (24, (14, 2, 64), 256, 1024, False), (24, (14, 2, 64), 256, 4096, True),
    (4, (14, 2, 64), 256, 4096, False)])
def test_groups_are_taken_where_whole_steps_get_shorter(layers, heads, rows, prefix, worth):
    """Each measured as whole steps of both kinds (the figures beside SHARED_MIN_VALUES)."""
    model = ModelConfig(name="m", num_layers=layers, num_q_heads=heads[0], num_kv_heads=heads[1], head_dim=heads[2])
    be = PagedCudaBackend(model, device="cpu", dtype=torch.bfloat16, share_prefixes=True)
    common = list(range(prefix // BS))
    tables = [array("i", common + [5000 + i]) for i in range(rows)]
    got = shared_groups(tables, [prefix + 5] * rows, BS, be._min_shared_keys())
    assert got == (([0, rows], [prefix] * rows) if worth else None)


class _History:
    """Token ids per sequence and the K/V a model would produce for them, prefix by prefix."""

    def __init__(self, seed=0):
        g = torch.Generator().manual_seed(seed)
        shape = (MODEL.num_layers, 2, MODEL.num_kv_heads, MODEL.head_dim)
        self.freq = torch.rand(shape, generator=g) * 3.0 + 0.5
        self.phase = torch.rand(shape, generator=g) * 6.283
        self.tokens: dict[int, list[int]] = {}

    def kv(self, layer, sid, start, stop):
        h, hs = 0, []
        for t in self.tokens[sid][:stop]:
            h = (h * 1000003 + t + 1) % (1 << 31)
            hs.append(h / (1 << 31) * 1000.0)
        x = torch.tensor(hs[start:stop], dtype=torch.float64).view(-1, 1, 1)
        return tuple((0.5 * torch.sin(x * self.freq[layer, i] + self.phase[layer, i])).to(torch.bfloat16)
                     for i in range(2))


def _held(x, code):
    """What an 8-bit cache holds for rows x."""
    if code is None:
        return x.float()
    return dequantise(*quantise(x, code)).float()


def _run_step(backend, mgr, hist, seq_ids, gen, code=None):
    plan = mgr.schedule(seq_ids)
    md = backend.begin_plan(plan)
    b, tq = len(seq_ids), plan.query_len
    hq, hkv, d = MODEL.num_q_heads, MODEL.num_kv_heads, MODEL.head_dim
    for layer in range(MODEL.num_layers):
        q = (torch.randn((b, tq, hq, d), generator=gen) * 0.5).to(torch.bfloat16)
        k = (torch.randn((b, tq, hkv, d), generator=gen) * 0.5).to(torch.bfloat16)  # pads: junk
        v = (torch.randn((b, tq, hkv, d), generator=gen) * 0.5).to(torch.bfloat16)
        for i, sid in enumerate(seq_ids):
            c, n = plan.ctx_before[i], plan.q_lens[i]
            if n:
                k[i, tq - n:], v[i, tq - n:] = hist.kv(layer, sid, c, c + n)
        out = backend.forward(layer, q.to(DEV), k.to(DEV), v.to(DEV), md).cpu()
        for i, sid in enumerate(seq_ids):
            c, n = plan.ctx_before[i], plan.q_lens[i]
            if not n:
                continue
            kk, vv = (_held(x, code) for x in hist.kv(layer, sid, 0, c + n))
            decodes = n == 1 and (tq == 1 or backend.split_mixed_steps)
            if code is not None and not decodes:  # the prefill reads the values rounded to 16 bits
                kk, vv = kk.to(torch.bfloat16).float(), vv.to(torch.bfloat16).float()
            ref = contiguous_attention(q[i:i + 1, tq - n:].float(), kk[None], vv[None],
                                       torch.ones((1, c + n), dtype=torch.bool), c)
            assert_attention_close(out[i, tq - n:], ref[0], f"seq {sid} layer {layer} ctx {c}")
    return plan, md


def _scenario(backend, code):
    backend.allocate(num_seq_slots=8, max_seq_len=512)
    backend.allocate_swap_space(16)
    mgr = backend.make_block_manager(enable_prefix_caching=True)
    hist = _History()
    rng, gen = torch.Generator().manual_seed(1), torch.Generator().manual_seed(2)
    shared_steps = 0

    def new_tokens(n):
        return torch.randint(0, 50000, (n,), generator=rng).tolist()

    def admit(sid, prompt):
        hist.tokens[sid] = list(prompt)
        mgr.allocate(sid, len(prompt), prompt)

    def step(sids, decode=()):
        nonlocal shared_steps
        for sid in decode:
            t = new_tokens(1)
            hist.tokens[sid] += t
            mgr.append_slots(sid, 1, t)
        plan, md = _run_step(backend, mgr, hist, sids, gen, code)
        shared_steps += md.group_starts is not None
        return plan

    system = new_tokens(150)
    admit(0, system + new_tokens(30))
    admit(1, new_tokens(45))
    step([0, 1])
    for _ in range(2):
        step([0, 1], [0, 1])
    admit(2, system + new_tokens(21))  # shares the system prompt's blocks, in a mixed step
    admit(3, system + new_tokens(1))
    step([0, 2, 3, 1], [0, 1])
    mgr.fork(0, 4)
    hist.tokens[4] = list(hist.tokens[0])
    plan = step([0, 4, 2, 3, 1], [0, 4, 2, 3, 1])  # copy-on-write, then a decode of five
    assert len(plan.copies) == 1
    for _ in range(2):
        step([0, 4, 2, 3, 1], [0, 4, 2, 3, 1])
    # a sequence leaves for host memory and comes back to other blocks
    mgr.swap_out(1)
    step([0, 4, 2, 3], [0, 4, 2, 3])
    mgr.swap_in(1)
    step([0, 4, 2, 3, 1], [0, 4, 2, 3, 1])
    mgr.check_invariants()
    torch.cuda.synchronize()
    assert int(backend.device_error.item()) == 0
    return shared_steps


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("split_mixed", [True, False])
def test_continuous_batching_over_an_8_bit_cache(code, split_mixed):
    be = PagedCudaBackend(MODEL, device=DEV, dtype=torch.bfloat16, num_blocks=96, split_tokens=32,
                          debug_invariants=True, split_mixed_steps=split_mixed, kv_codes=code)
    assert _scenario(be, code) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("split", [0, 32])
def test_continuous_batching_with_shared_prefixes(split, monkeypatch):
    monkeypatch.setattr(backend_module, "SHARED_MIN_VALUES", 1)
    be = PagedCudaBackend(MODEL, device=DEV, dtype=torch.bfloat16, num_blocks=96, split_tokens=split,
                          debug_invariants=True, share_prefixes=True)
    assert _scenario(be, None) == 5  # every pure decode step in which two sequences share blocks


@pytest.mark.gpu
@pytest.mark.parametrize("share", [True, False])
def test_a_step_sorts_its_sequences_once(share, monkeypatch):
    """By their own keys where prefixes are shared, else by their lengths."""
    monkeypatch.setattr(backend_module, "SHARED_MIN_VALUES", 1)
    be = PagedCudaBackend(MODEL, device=DEV, dtype=torch.bfloat16, num_blocks=96, share_prefixes=share)
    be.allocate(4, 512)
    mgr = be.make_block_manager(enable_prefix_caching=True)
    common = list(range(64))
    for i, own in enumerate((40, 5, 90)):
        mgr.allocate(i, 64 + own, common + [100 + i] * own)
        mgr.schedule([i])
        mgr.append_slots(i, 1, [7])
    sorted_by = []
    order = backend_module.ops.decode_order

    def counted(lens, **kw):
        sorted_by.append(lens.tolist())
        return order(lens, **kw)

    monkeypatch.setattr(backend_module.ops, "decode_order", counted)
    md = be.begin_plan(mgr.schedule([0, 1, 2]))
    assert (md.group_starts is not None) == share
    assert sorted_by == ([[41, 6, 91]] if share else [[105, 70, 155]])
    assert md.seq_order.tolist() == [2, 0, 1]


@pytest.mark.gpu
def test_small_savings_keep_the_plain_decode():
    be = PagedCudaBackend(MODEL, device=DEV, dtype=torch.bfloat16, num_blocks=96, split_tokens=32,
                          share_prefixes=True)
    assert _scenario(be, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("use_tables", [False, True])
def test_static_engine_over_an_8_bit_cache(code, use_tables):
    """The reference's static batching: a left-padded prefill of uneven prompts, then decodes."""
    prompts, steps = [37, 5, 130], 4
    total = max(prompts) + steps
    be = PagedCudaBackend(MODEL, device=DEV, dtype=torch.bfloat16, split_tokens=64, kv_codes=code,
                          debug_invariants=True)
    be.allocate(len(prompts), total)
    gen = torch.Generator().manual_seed(3)
    b, hq, hkv, d = len(prompts), 8, 2, 128
    mask = torch.zeros((b, total), dtype=torch.bool)
    for i, n in enumerate(prompts):
        mask[i, max(prompts) - n: max(prompts)] = True
    width = (total + BS - 1) // BS
    tables = torch.randperm(be.num_blocks, generator=gen)[: b * width].view(b, width).to(torch.int32)
    hist = torch.zeros((2, MODEL.num_layers, b, total, hkv, d), dtype=torch.bfloat16)
    lens = torch.tensor(prompts, dtype=torch.int32)
    for ctx, tq in [(0, max(prompts))] + [(max(prompts) + s, 1) for s in range(steps)]:
        if tq == 1:
            mask[:, ctx] = True
            lens = lens + 1
        real = mask[:, ctx:ctx + tq]
        logical = mask[:, :ctx].sum(1, keepdim=True) + real.cumsum(1) - 1
        slots = torch.where(real, tables.long().gather(1, logical.clamp(min=0) // BS) * BS + logical % BS, -1)
        md = be.begin_step(StepInput(
            query_len=tq, context_len=ctx, seq_lens=lens.to(DEV), padding_mask=mask[:, :ctx + tq].to(DEV),
            is_prefill=tq > 1, block_tables=tables.to(DEV) if use_tables else None,
            slot_mapping=slots.reshape(-1).to(DEV) if use_tables else None))
        for layer in range(MODEL.num_layers):
            q, k, v = ((torch.randn((b, tq, h, d), generator=gen) * 0.5).to(torch.bfloat16) for h in (hq, hkv, hkv))
            out = be.forward(layer, q.to(DEV), k.to(DEV), v.to(DEV), md).cpu()
            hist[0, layer, :, ctx:ctx + tq], hist[1, layer, :, ctx:ctx + tq] = k, v
            kk, vv = (_held(x[layer, :, :ctx + tq], code) for x in hist)
            if tq > 1:
                kk, vv = kk.to(torch.bfloat16).float(), vv.to(torch.bfloat16).float()
            ref = contiguous_attention(q.float(), kk, vv, mask[:, :ctx + tq], ctx)
            assert_attention_close(out[real], ref[real], f"layer {layer} ctx {ctx}")
    assert be.memory_stats().live_bytes == int(lens.sum()) * be._kv_bytes_per_token()


@pytest.mark.gpu
@pytest.mark.parametrize("code", [None, *CODES])
def test_a_prefill_leaves_zeros_in_padding_rows(code):
    """Left-padded prompts: the rows before a prompt are zeros, whatever the memory held before."""
    prompts = [37, 5, 64]
    b, tq, hq, hkv, d = 3, 64, 8, 2, 128
    be = PagedCudaBackend(MODEL, device=DEV, dtype=torch.bfloat16, kv_codes=code)
    be.allocate(b, 128)
    mask = torch.zeros((b, tq), dtype=torch.bool, device=DEV)
    for i, n in enumerate(prompts):
        mask[i, tq - n:] = True
    md = be.begin_step(StepInput(query_len=tq, context_len=0, seq_lens=mask.sum(1).to(torch.int32),
                                 padding_mask=mask, is_prefill=True))
    q, k, v = (torch.randn((b, tq, h, d), device=DEV).to(torch.bfloat16) for h in (hq, hkv, hkv))
    for _ in range(2):
        junk = [torch.full((b * tq, hq, d), float("nan"), device=DEV, dtype=torch.bfloat16) for _ in range(4)]
        del junk
        out = be.forward(0, q, k, v, md)
        assert (out[~mask] == 0).all() and out[mask].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
def test_decode_graph_over_an_8_bit_cache(code):
    """DecodeGraph replays equal eager steps, with growing contexts and an inactive row."""
    lens = [40, 17, 90]
    outs = []
    for graph in (True, False):
        be = PagedCudaBackend(MODEL, device=DEV, dtype=torch.bfloat16, split_tokens=32, kv_codes=code)
        be.allocate(4, 128)
        gen = torch.Generator(device=DEV).manual_seed(4)
        for pool, scale in ((be.k_cache, be.k_scale), (be.v_cache, be.v_scale)):
            c, s = quantise(torch.randn(pool.shape, device=DEV, generator=gen) * 0.5, code)
            pool.copy_(c)
            scale.copy_(s)
        tables = torch.arange(3 * 8, dtype=torch.int32).view(3, 8)
        g = DecodeGraph(be, batch=4) if graph else None
        md = None if graph else be.static_decode_metadata(4)
        got = []
        for t in range(3):
            ctx = torch.tensor(lens, dtype=torch.int32) + t
            x = [torch.randn((MODEL.num_layers, 4, 1, h, 128), device=DEV, generator=gen).to(torch.bfloat16)
                 for h in (8, 2, 2)]
            if graph:
                g.query.copy_(x[0])
                g.key.copy_(x[1])
                g.value.copy_(x[2])
                g.load(tables, ctx)
                got += [o.clone() for o in g.replay()]
            else:
                be.load_decode(md, tables, ctx)
                got += [be.forward(i, x[0][i], x[1][i], x[2][i], md).clone() for i in range(MODEL.num_layers)]
        torch.cuda.synchronize()
        assert (got[-1][3] == 0).all()
        outs.append(got + [be.k_cache.view(torch.uint8).clone(), be.v_scale.clone()])
    for a, z in zip(*outs):
        assert torch.equal(a, z)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
def test_write_kv_rope_quantises_the_rotated_rows(code):
    from paged_serve_b200.rope import cos_sin_table
    from tests.quant_util import rotate

    be = PagedCudaBackend(MODEL, device=DEV, dtype=torch.bfloat16, kv_codes=code)
    be.allocate(2, 64)
    mask = torch.ones((2, 20), dtype=torch.bool, device=DEV)
    md = be.begin_step(StepInput(query_len=20, context_len=0, seq_lens=mask.sum(1).to(torch.int32),
                                 padding_mask=mask, is_prefill=True))
    k, v = (torch.randn((2, 20, 2, 128), device=DEV).to(torch.bfloat16) for _ in range(2))
    be.write_kv_rope(1, k, v, md)
    table = cos_sin_table(128, 10000.0, 64, torch.bfloat16, DEV)
    codes, scale = quantise(rotate(k.view(40, 2, 128), torch.arange(20, device=DEV).repeat(2), table), code)
    for b in range(2):
        for t in range(20):
            blk = b * 4 + t // BS
            assert torch.equal(be.k_cache[1, blk, :, t % BS].view(torch.uint8), codes[b * 20 + t].view(torch.uint8))
            assert torch.equal(be.k_scale[1, blk, :, t % BS], scale[b * 20 + t])

"""The quantised paged KV cache and shared-prefix decode: cases, plain forms and exact values.

Four operators over the paged pools ``[num_blocks, num_kv_heads, block_size, head_dim]``:

* ``append``  - quantise the step's K and V rows (K rotated on the way, where asked) to
  8 bits with one fp32 scale per (token, kv head) and write them at their slots:
  ``scale = max(max|x| / qmax, 2^-126)``, ``code = round(x * (1 / scale))``, with qmax 448
  for e4m3 and 127 for int8, every step rounded to fp32, so codes are reproducible to the bit.
* ``read``    - the codes of whole sequences back as 16-bit values ``code * scale`` in a pool
  of their own, rows past a sequence's last token as zeros.
* ``decode``  - one query per sequence over its 8-bit keys and values.
* ``shared``  - one query per sequence over 16-bit pools, where groups of neighbouring
  sequences share their leading blocks.

``own`` false computes them in elementary torch operations, ``own`` true through the package.
"""

import math
import random

import torch

own = False

QMAX = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
KV = {"bf16": torch.bfloat16, "f16": torch.float16}

# (query heads, kv heads, head dim) of the repository's workloads and tests
HEADS = [(32, 8, 128), (64, 8, 128), (14, 2, 64), (8, 2, 64), (28, 4, 128), (32, 2, 128), (9, 3, 64),
         (8, 8, 128)]


def listed():
    return [
        # One decode step of a Llama-3-8B-shaped layer: 256 new tokens, K rotated.
        dict(name="append_step_8b", op="append", tokens=256, hkv=8, d=128, bs=16, kv="bf16", code="e4m3",
             rope=True, pad=0, lens_seed=1),
        # The append workload's step: 256 decode tokens and eight prompts of 2048.
        dict(name="append_prompt_8b", op="append", tokens=16640, hkv=8, d=128, bs=16, kv="bf16", code="e4m3",
             rope=True, pad=0, lens_seed=2),
        # A left-padded step of a small model at head dim 64, int8 codes, no rotation.
        dict(name="append_padded_int8", op="append", tokens=1037, hkv=2, d=64, bs=32, kv="f16", code="int8",
             rope=False, pad=211, lens_seed=3),
        # A long prompt's cached tokens brought back for its next chunk's prefill.
        dict(name="read_long_prompt", op="read", hkv=8, d=128, bs=16, kv="bf16", code="e4m3", lens="fixed",
             batch=1, lo=32256, hi=32256, lens_seed=4),
        # Many short ragged sequences, an empty one among them, small blocks.
        dict(name="read_ragged_int8", op="read", hkv=2, d=64, bs=8, kv="f16", code="int8", lens="uniform",
             batch=37, lo=0, hi=700, lens_seed=5),
        # The headline decode batch of a Llama-3-8B-shaped layer from an e4m3 cache.
        dict(name="decode_8b", op="decode", hq=32, hkv=8, d=128, bs=16, kv="bf16", code="e4m3",
             lens="uniform", batch=256, lo=512, hi=4096, split=0, lens_seed=6),
        # A rank's share of the skewed long-context 70B batch, partitions of 512 keys.
        dict(name="decode_70b_long", op="decode", hq=64, hkv=8, d=128, bs=16, kv="bf16", code="e4m3",
             lens="lognormal", batch=64, lo=128, hi=32768, split=512, lens_seed=7),
        # A single user's stream, where latency counts: int8, fp16, short partitions.
        dict(name="decode_one", op="decode", hq=32, hkv=8, d=128, bs=16, kv="f16", code="int8", lens="fixed",
             batch=1, lo=1531, hi=1531, split=128, lens_seed=8),
        # The reference's default model geometry (head dim 64, seven query heads a kv head), ragged.
        dict(name="decode_qwen_int8", op="decode", hq=14, hkv=2, d=64, bs=32, kv="bf16", code="int8",
             lens="uniform", batch=96, lo=1, hi=2000, split=0, lens_seed=9),
        # A batch under one long system prompt, each with a short conversation of its own.
        dict(name="shared_prompt_8b", op="shared", hq=32, hkv=8, d=128, bs=16, kv="bf16", groups="256x8192",
             lo=1, hi=512, split=0, lens_seed=10),
        # Several few-shot prompts of different lengths and group sizes, and sequences that share nothing.
        dict(name="shared_groups_qwen", op="shared", hq=14, hkv=2, d=64, bs=8, kv="f16",
             groups="17x1040 3x2000 5x0 40x336", lo=0, hi=300, split=0, lens_seed=11),
        # Eight samples drawn from one long document, eight query heads a kv head.
        dict(name="shared_document_70b", op="shared", hq=64, hkv=8, d=128, bs=16, kv="bf16", groups="8x32768",
             lo=1, hi=64, split=0, lens_seed=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "decode", "shared", "shared"])
    hq, hkv, d = rng.choice(HEADS)
    case = dict(op=op, hkv=hkv, d=d, bs=rng.choice([8, 16, 32]), kv=rng.choice(["bf16", "f16"]),
                lens_seed=rng.randrange(1 << 30))
    if op != "shared":
        case["code"] = rng.choice(["e4m3", "int8"])
    if op == "append":
        case.update(tokens=_log(rng, 1, 16640), rope=rng.random() < 0.5)
        case["pad"] = _log(rng, 1, 300) if rng.random() < 0.4 else 0
    elif op == "read":
        batch = _log(rng, 1, 200)
        hi = _log(rng, 1, max(1, 120000 // batch // hkv))
        case.update(lens=rng.choice(["fixed", "uniform"]), batch=batch, lo=rng.randint(0, hi), hi=hi)
    elif op == "decode":
        batch = _log(rng, 1, 256)
        hi = _log(rng, 1, min(32768, max(1, 4000000 // batch // hkv)))
        lens = rng.choice(["fixed", "uniform", "lognormal"])
        case.update(hq=hq, lens=lens, batch=batch, lo=rng.randint(0, hi) if lens != "lognormal" else 1, hi=hi)
        case["split"] = rng.choice([0, 128, 256, 512]) if hi <= 8192 else rng.choice([256, 512, 1024])
    else:
        groups, room = [], 1500000 // hkv
        for _ in range(rng.choice([1, 1, 2, 3, 6])):
            n = _log(rng, 1, 96)
            pre = _log(rng, 32, 32768)
            pre = min(pre, room // n) // case["bs"] * case["bs"] if rng.random() < 0.85 else 0
            groups.append("%dx%d" % (n, pre))
            room = max(room - n * (pre + 256), 0)
        hi = _log(rng, 1, 400)
        case.update(hq=hq, groups=" ".join(groups), lo=rng.randint(0, min(hi, 32)), hi=hi, split=rng.choice([0, 0, 128]))
    return case


# ------------------------------------------------------------------ lengths and tables
def _groups(case):
    """[(sequences, shared prefix tokens)] of a `shared` case, from text such as "17x1040 5x0"."""
    return [tuple(int(x) for x in g.split("x")) for g in case["groups"].split()]


def _lens(case):
    """Tokens of each sequence; for `shared`, those behind the shared prefix."""
    rng = random.Random(case["lens_seed"])
    if case["op"] == "shared":
        return [rng.randint(case["lo"], case["hi"]) for _ in range(sum(n for n, _ in _groups(case)))]
    n, lo, hi = case["batch"], case["lo"], case["hi"]
    if case["lens"] == "fixed":
        return [hi] * n
    if case["lens"] == "uniform":
        return [rng.randint(lo, hi) for _ in range(n)]
    return [max(lo, min(hi, int(rng.lognormvariate(math.log(max(1, min(2048, hi))), 1.0)))) for _ in range(n)]


def _shared(case):
    """(shared prefix tokens of each sequence, group start indices)."""
    pre, starts = [], [0]
    for n, p in _groups(case):
        pre += [p] * n
        starts.append(starts[-1] + n)
    return pre, starts


def _tables(case, lens, pre=None, starts=None):
    """Block tables (lists of ids in a shuffled pool) and the pool's block count."""
    bs = case["bs"]
    rng = random.Random(case["lens_seed"] + 1)
    need = [(n + bs - 1) // bs for n in lens]
    heads = [p // bs for p in pre] if pre else [0] * len(lens)
    total = sum(need) + (sum(heads[a] for a in starts[:-1]) if pre else 0)
    blocks = total + max(4, total // 4)
    ids = list(range(blocks))
    rng.shuffle(ids)
    tables, at = [], 0
    first = []
    group_of = {a for a in starts[:-1]} if pre else set()
    for b, n in enumerate(need):
        if b in group_of:
            first, at = ids[at:at + heads[b]], at + heads[b]
        tables.append((first if pre else []) + ids[at:at + n])
        at += n
    return tables, blocks


def _width(tables):
    return max(1, max((len(t) for t in tables), default=1))


def _table_tensor(tables, width):
    t = torch.zeros((len(tables), width), dtype=torch.int32)
    for b, row in enumerate(tables):
        if row:
            t[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
    return t


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(shape, gen, dtype, loud):
    """Rows like a model's K or V: normal, a few loud channels (K) or tokens (V)."""
    x = torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, 0.5, generator=gen)
    if loud == "channels":
        x *= 1.0 + 5.0 * (torch.rand(shape[-1], device="cuda", generator=gen) < 0.04)
    else:
        x *= torch.exp(0.5 * torch.randn(shape[:-1] + (1,), device="cuda", generator=gen))
    return x.to(dtype)


def _quantise(x, code):
    """(codes, scales) of rows x [..., D] in fp32."""
    x = x.float()
    qmax = torch.full(x.shape[:-1], QMAX[code], device=x.device)
    scale = (x.abs().amax(-1) / qmax).clamp_min(2.0 ** -126)
    y = x * (torch.ones_like(scale) / scale).unsqueeze(-1)
    if code == "int8":
        return torch.round(y).clamp(-127, 127).to(torch.int8), scale
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _fill_pools(case, state, seed, quantised):
    """Pools whose used rows hold drawn values and whose other rows hold NaN, as stale memory may."""
    gen = _gen(seed)
    shape = (state["blocks"], case["hkv"], case["bs"], case["d"])
    bs = case["bs"]
    used = torch.zeros(state["blocks"], bs, dtype=torch.bool)
    for row, n in zip(state["tables"], state["ctx"]):
        full = n // bs
        if full:
            used[torch.tensor(row[:full])] = True
        if n % bs:
            used[row[full], :n % bs] = True
    stale = (~used).cuda()[:, None, :].expand(shape[:3])
    for name, loud in (("k", "channels"), ("v", "tokens")):
        x = _rows(shape, gen, KV[case["kv"]], loud)
        if not quantised:
            state[name] = x.masked_fill_(stale.unsqueeze(-1), float("nan"))
            continue
        codes, scale = _quantise(x, case["code"])
        del x
        if case["code"] == "e4m3":
            codes.view(torch.uint8).masked_fill_(stale.unsqueeze(-1), 0x7F)  # NaN
        state[name], state[name + "_scale"] = codes, scale.masked_fill_(stale, float("nan"))
    return gen


def prepare(case, seed):
    dt = KV[case["kv"]]
    if case["op"] == "append":
        return _prepare_append(case, seed, dt)
    lens = _lens(case)
    state = {"case": case}
    if case["op"] == "shared":
        pre, starts = _shared(case)
        state["pre"], state["starts"] = pre, starts
        state["tables"], state["blocks"] = _tables(case, lens, pre, starts)
        state["ctx"] = [a + b for a, b in zip(pre, lens)]
    else:
        state["tables"], state["blocks"] = _tables(case, lens)
        state["ctx"] = lens
    gen = _fill_pools(case, state, seed, case["op"] != "shared")
    width = _width(state["tables"])
    state["block_tables"] = _table_tensor(state["tables"], width).cuda()
    state["ctx_lens"] = torch.tensor(state["ctx"], dtype=torch.int32).cuda()
    state["ids"] = [torch.tensor(t, dtype=torch.long).cuda() for t in state["tables"]]
    n = len(state["ctx"])
    if case["op"] == "read":
        bs = case["bs"]
        need = [(c + bs - 1) // bs for c in state["ctx"]]
        starts = [sum(need[:b]) for b in range(n)]
        out_tables = [list(range(a, a + m)) for a, m in zip(starts, need)]
        state["out_starts"] = starts
        state["out_tables"] = _table_tensor(out_tables, width).cuda()
        shape = (max(1, sum(need)), case["hkv"], bs, case["d"])
        state["k_out"] = torch.zeros(shape, device="cuda", dtype=dt)
        state["v_out"] = torch.zeros(shape, device="cuda", dtype=dt)
        return state
    state["query"] = torch.empty((n, case["hq"], case["d"]), device="cuda").normal_(
        0.0, 1.0, generator=gen).to(dt)
    state["sm_scale"] = 1.0 / math.sqrt(case["d"])
    if case["op"] == "shared":
        state["shared_lens"] = torch.tensor(state["pre"], dtype=torch.int32).cuda()
        state["group_starts"] = torch.tensor(state["starts"], dtype=torch.int32).cuda()
    if own:
        _plan(case, state)
    return state


def _prepare_append(case, seed, dt):
    gen = _gen(seed)
    t, hkv, d, bs = case["tokens"], case["hkv"], case["d"], case["bs"]
    rng = random.Random(case["lens_seed"])
    blocks = (t + bs - 1) // bs + 8
    slots = torch.tensor(rng.sample(range(blocks * bs), t), dtype=torch.int64)
    if case["pad"]:
        slots[torch.tensor(rng.sample(range(t), min(case["pad"], t)))] = -1
    state = {"case": case, "slots": slots.cuda(), "real": (slots >= 0).nonzero().squeeze(1).cuda()}
    # K and V as a fused projection leaves them: two column ranges of one buffer.
    fused = torch.cat([_rows((t, hkv, d), gen, dt, "channels"), _rows((t, hkv, d), gen, dt, "tokens")], 1)
    state["key"], state["value"] = fused[:, :hkv], fused[:, hkv:]
    shape = (blocks, hkv, bs, d)
    for name in ("k", "v"):
        state[name] = torch.zeros(shape, device="cuda", dtype=torch.int8).view(CODE[case["code"]])
        state[name + "_scale"] = torch.zeros(shape[:3], device="cuda")
    if case["rope"]:
        table_len = 4096
        state["positions"] = torch.randint(0, table_len, (t,), device="cuda", generator=gen)
        inv = 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        ang = torch.arange(table_len, device="cuda", dtype=torch.float64)[:, None] * inv
        state["table"] = torch.cat([ang.cos(), ang.sin()], -1).to(dt)
    return state


def _plan(case, state):
    """What a serving loop keeps per step: the launch order, the workspace and the split plan."""
    from paged_serve_b200 import ops

    n, width = state["block_tables"].shape
    if case["op"] == "decode":
        state["order"] = ops.decode_order(state["ctx_lens"])
        need = ops.decode_workspace_bytes(n, case["hq"], case["d"], case["bs"], width, case["split"])
        state["workspace"] = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
        ops.decode_plan(state["ctx_lens"], state["workspace"], case["hq"], case["d"], case["bs"], width,
                        case["split"], seq_order=state["order"])
        return
    state["max_group"] = max(m for m, _ in _groups(case))
    state["max_shared"] = max(p for _, p in _groups(case))
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    state["split_keys"] = ops.shared_split_keys([m for m, p in _groups(case) if p], case["hq"], case["hkv"],
                                                state["max_shared"], sms)
    own_lens = state["ctx_lens"] - state["shared_lens"]
    state["order"] = ops.decode_order(own_lens)
    need = ops.decode_shared_workspace_bytes(n, case["hq"], case["d"], case["bs"], width, state["max_shared"],
                                             state["split_keys"], case["split"])
    state["workspace"] = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")


# ------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state["case"], state)


def _run_own(case, s):
    from paged_serve_b200 import ops

    if case["op"] == "append":
        if case["rope"]:
            ops.cache_append_rope_quant(s["k"], s["v"], s["k_scale"], s["v_scale"], s["key"], s["value"],
                                        s["slots"], s["positions"], s["table"])
        else:
            ops.cache_append_quant(s["k"], s["v"], s["k_scale"], s["v_scale"], s["key"], s["value"], s["slots"])
        return s["k"], s["v"], s["k_scale"], s["v_scale"]
    if case["op"] == "read":
        ops.cache_read_quant(s["k"], s["v"], s["k_scale"], s["v_scale"], s["block_tables"], s["ctx_lens"],
                             s["k_out"], s["v_out"], s["out_tables"])
        return s["k_out"], s["v_out"]
    if case["op"] == "decode":
        return ops.paged_decode_quant(s["query"], s["k"], s["v"], s["k_scale"], s["v_scale"],
                                      s["block_tables"], s["ctx_lens"], s["sm_scale"], case["split"],
                                      workspace=s["workspace"], seq_order=s["order"], planned=True)
    return ops.paged_decode_shared(s["query"], s["k"], s["v"], s["block_tables"], s["ctx_lens"],
                                   s["group_starts"], s["shared_lens"], s["max_group"], s["max_shared"],
                                   s["sm_scale"], split_keys=s["split_keys"], split_tokens=case["split"],
                                   workspace=s["workspace"], seq_order=s["order"])


def _run_plain(case, s):
    if case["op"] == "append":
        key = s["key"].float()
        if case["rope"]:
            half = case["d"] // 2
            cs = s["table"].float()[s["positions"]][:, None]
            c, sn = cs[..., :half], cs[..., half:]
            lo, hi = key[..., :half], key[..., half:]
            key = torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1)
        rows = s["real"]  # the rows that are no padding
        slots = s["slots"][rows]
        blk, off = slots // case["bs"], slots % case["bs"]
        for name, x in (("k", key), ("v", s["value"].float())):
            codes, scale = _quantise(x, case["code"])
            s[name].view(torch.uint8)[blk, :, off] = codes.view(torch.uint8)[rows]
            s[name + "_scale"][blk, :, off] = scale[rows]
        return s["k"], s["v"], s["k_scale"], s["v_scale"]
    if case["op"] == "read":
        bs = case["bs"]
        for ids, n, a in zip(s["ids"], s["ctx"], s["out_starts"]):
            if n == 0:
                continue
            live = (torch.arange(len(ids) * bs, device="cuda") < n).view(len(ids), 1, bs, 1)
            for name in ("k", "v"):
                x = s[name][ids].float() * s[name + "_scale"][ids].unsqueeze(-1)
                s[name + "_out"][a:a + len(ids)] = torch.where(live, x, torch.zeros_like(x)).to(
                    s[name + "_out"].dtype)
        return s["k_out"], s["v_out"]
    out = torch.zeros_like(s["query"])
    for b, (ids, n) in enumerate(zip(s["ids"], s["ctx"])):
        if n == 0:
            continue
        k, v = (_sequence(case, s, name, ids, n) for name in ("k", "v"))  # [Hkv, n, D] fp32
        q = s["query"][b].float().view(case["hkv"], -1, case["d"])
        x = (q @ k.transpose(1, 2)) * s["sm_scale"]
        p = torch.exp(x - x.amax(-1, keepdim=True))
        o = (p @ v) / p.sum(-1, keepdim=True)
        out[b] = o.reshape(case["hq"], case["d"]).to(out.dtype)
    return out


def _sequence(case, s, name, ids, n):
    x = s[name][ids].float()
    if case["op"] == "decode":
        x = x * s[name + "_scale"][ids].unsqueeze(-1)
    return x.transpose(0, 1).reshape(case["hkv"], -1, case["d"])[:, :n]


# ------------------------------------------------------------------ work and exact values
def work(case):
    size = 2  # bytes of a bf16 or fp16 value
    if case["op"] == "append":
        rows = case["tokens"] - min(case["pad"], case["tokens"])
        elems = 2 * rows * case["hkv"] * case["d"]
        b = elems * (size + 1) + 2 * rows * case["hkv"] * 4 + case["tokens"] * 8
        if case["rope"]:
            b += case["tokens"] * 8 + min(rows, 4096) * case["d"] * size
        return {"bytes": b, "flops": elems * (5 if case["rope"] else 3)}
    lens = _lens(case)
    bs, hkv, d = case["bs"], case["hkv"], case["d"]
    if case["op"] == "read":
        rows = sum(lens)
        padded = sum((n + bs - 1) // bs * bs for n in lens)
        return {"bytes": 2 * hkv * (rows * (d + 4) + padded * d * size) + 8 * len(lens), "flops": 2 * rows * hkv * d}
    n = len(lens)
    io = 2 * n * case["hq"] * d * size + 4 * n
    if case["op"] == "decode":
        keys = sum(lens)
        return {"bytes": 2 * keys * hkv * (d + 4) + io + sum((x + bs - 1) // bs for x in lens) * 4,
                "flops": 4 * d * case["hq"] * keys}
    once = sum(p for _, p in _groups(case)) + sum(lens)
    keys = sum(lens) + sum(m * p for m, p in _groups(case))
    return {"bytes": 2 * once * hkv * d * size + io + (once + bs * n) // bs * 4, "flops": 4 * d * case["hq"] * keys}


def exact(case, seed):
    """The operators' definitions in float64, token by token rather than block by block."""
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "append":
        k, v = s["key"].to(f8), s["value"].to(f8)
        if case["rope"]:
            tab = s["table"].to(f8)[s["positions"]].unsqueeze(1)
            z = torch.complex(*k.chunk(2, -1)) * torch.complex(*tab.chunk(2, -1))
            k = torch.cat([z.real, z.imag], -1)
        outs = []
        for x in (k, v):
            code = torch.zeros(s["k"].shape, dtype=f8, device="cuda").transpose(1, 2).flatten(0, 1)
            scale = torch.zeros(code.shape[:2], dtype=f8, device="cuda")
            keep = s["slots"] >= 0
            top = (x.abs().amax(-1) / QMAX[case["code"]]).clamp_min(2.0 ** -126)
            scale[s["slots"][keep]] = top[keep]
            code[s["slots"][keep]] = (x / top.unsqueeze(-1))[keep]
            back = (s["k"].shape[0], case["bs"], case["hkv"])
            outs.append((code.view(*back, -1).transpose(1, 2), scale.view(back).transpose(1, 2)))
        codes = [None if case["code"] == "int8" else o[0] for o in outs]
        return codes[0], codes[1], outs[0][1], outs[1][1]
    pos_of = []
    for row, n in zip(s["tables"], s["ctx"]):
        t = torch.arange(n)
        ids = torch.tensor(row, dtype=torch.long)[t // case["bs"]] if n else torch.zeros(0, dtype=torch.long)
        pos_of.append((ids.cuda(), (t % case["bs"]).cuda()))

    def tokens(name, b):  # [n, Hkv, D]
        blk, off = pos_of[b]
        x = s[name][blk, :, off] if case["op"] == "shared" else s[name].view(torch.uint8)[blk, :, off].view(
            s[name].dtype)
        x = x.to(f8) if case["op"] == "shared" else x.float().to(f8)
        return x if case["op"] == "shared" else x * s[name + "_scale"].to(f8)[blk, :, off].unsqueeze(-1)

    if case["op"] == "read":
        outs = []
        for name in ("k", "v"):
            o = torch.zeros(s["k_out"].shape, dtype=f8, device="cuda").transpose(1, 2).flatten(0, 1)
            for b, n in enumerate(s["ctx"]):
                o[s["out_starts"][b] * case["bs"]:][:n] = tokens(name, b)
            outs.append(o.view(-1, case["bs"], case["hkv"], case["d"]).transpose(1, 2))
        return tuple(outs)
    q = s["query"].to(f8)
    out = torch.zeros_like(q)
    share = case["hq"] // case["hkv"]
    for b, n in enumerate(s["ctx"]):
        if n:
            k, v = tokens("k", b), tokens("v", b)
            x = torch.einsum("hgd,nhd->hgn", q[b].view(case["hkv"], share, -1), k) / math.sqrt(case["d"])
            out[b] = torch.einsum("hgn,nhd->hgd", torch.softmax(x, -1), v).reshape(case["hq"], -1)
    return out

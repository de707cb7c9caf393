"""Workloads of the 4-bit KV cache operators, their plain forms and their 64-bit definition.

The cache: a layer is a uint8 tensor [kv, blocks, heads, tokens_per_block / 16, 9 * dim].  The last axis is one
unit, 16 tokens of one head: 16 rows of dim / 2 bytes with two e2m1 values each (the even channel in the low bits),
then 16 rows of dim / 16 scale bytes, one for each 16 channels.  A scale byte c stands for the half-precision number
with the bits c << 7 (5 exponent bits, 3 mantissa bits, no sign).  A group of 16 channels is stored with the scale
nearest to amax / 6 (at most 10240), and each value as the e2m1 number nearest to x / scale, ties to the even code.
"""
import math
import random

import torch

own = False

GROUP = 16
UNIT = 16  # tokens of a unit
SCALE_MAX = 10240.0
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One sequence's next token, every decode step of an engine with a 4-bit cache: latency alone counts.
        dict(name="append one token", kind="append", tokens=1, heads=8, dim=128, tpb=16, dtype="bf16", fused=True, padded=0, mla=False),
        # A prompt chunk of ragged requests as the projection leaves it (k and v are slices of one row), padded rows behind it.
        dict(name="append 1021 of 1024", kind="append", tokens=1024, heads=4, dim=128, tpb=16, dtype="bf16", fused=True, padded=3, mla=False),
        # A cached 32k-token prefix handed to 16-bit kernels.
        dict(name="read 32768", kind="read", tokens=32768, heads=8, dim=128, tpb=16, dtype="bf16", mla=False),
        # A latent cache: one vector of 576 channels for each token, an odd number of tokens.
        dict(name="read latent 4099", kind="read", tokens=4099, heads=1, dim=576, tpb=64, dtype="bf16", mla=True),
        # One request's few blocks on their way to the host tier and back, all layers.
        dict(name="blocks 28x9", kind="blocks", layers=28, blocks=9, heads=4, dim=128, tpb=16, dtype="bf16", mla=False),
        # A batch of blocks, all layers of a larger model.
        dict(name="blocks 32x256", kind="blocks", layers=32, blocks=256, heads=8, dim=128, tpb=16, dtype="bf16", mla=False),
        # One chat of middling length, the smallest decode step.
        dict(name="decode 1x1000", kind="attend", batch=1, heads=8, group=4, dim=128, tpb=16, dtype="bf16", len_min=1000, len_max=1000, new_min=1, new_max=1, pick=0),
        # One rank of eight reads its only head of a very long context.
        dict(name="decode 1x131071, one head", kind="attend", batch=1, heads=1, group=8, dim=128, tpb=64, dtype="bf16", len_min=131071, len_max=131071, new_min=1, new_max=1, pick=0),
        # A serving batch of requests of all lengths, seven query heads to a key head.
        dict(name="decode 64 ragged", kind="attend", batch=64, heads=4, group=7, dim=128, tpb=16, dtype="bf16", len_min=1, len_max=8192, new_min=1, new_max=1, pick=1),
        # A full batch of long requests: the largest decode step.
        dict(name="decode 48 long", kind="attend", batch=48, heads=8, group=4, dim=128, tpb=16, dtype="bf16", len_min=6000, len_max=16384, new_min=1, new_max=1, pick=2),
        # Proposed tokens checked in one pass: one to five for each request, half precision, small heads.
        dict(name="verify 16x1-5", kind="attend", batch=16, heads=8, group=2, dim=64, tpb=16, dtype="fp16", len_min=300, len_max=6000, new_min=1, new_max=5, pick=3),
        # Chunks of prompts behind cached prefixes, packed.
        dict(name="prompts 3 packed", kind="attend", batch=3, heads=8, group=4, dim=128, tpb=16, dtype="bf16", len_min=4500, len_max=8000, new_min=3500, new_max=4096, pick=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "read", "blocks", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "fp16"])
    tpb = rng.choice([16, 32, 64])
    mla = kind != "attend" and rng.random() < 0.25
    heads = 1 if mla else rng.choice([1, 2, 4, 8])
    dim = 576 if mla else rng.choice([64, 128])
    if kind in ("append", "read"):
        tokens = _log(rng, 1, 32768 // heads)
        c = dict(kind=kind, tokens=tokens, heads=heads, dim=dim, tpb=tpb, dtype=dtype, mla=mla)
        if kind == "append":
            c.update(fused=rng.random() < 0.5, padded=rng.choice([0, 0, rng.randint(0, tokens - 1)]))
        return c
    if kind == "blocks":
        return dict(kind=kind, layers=rng.randint(1, 32), blocks=_log(rng, 1, 1024 // (heads * tpb // 16)), heads=heads, dim=dim, tpb=tpb,
                    dtype=dtype, mla=mla)
    group = rng.randint(1, 16)
    c = dict(kind=kind, heads=heads, group=group, dim=dim, tpb=tpb, dtype=dtype, pick=rng.randrange(1 << 30))
    form = rng.choice(["decode", "decode", "verify", "prompt"])
    if form == "prompt":
        longest = _log(rng, 64, 6000)
        c.update(group=min(group, 32 // heads), batch=rng.randint(1, 3), len_min=max(1, longest // 3), len_max=longest, new_min=max(1, longest // 6), new_max=max(1, longest // 2))
    else:
        longest = _log(rng, 16, 65536)
        c.update(batch=_log(rng, 1, max(1, min(256, (1 << 19) // longest))), len_min=1, len_max=longest, new_min=1,
                 new_max=1 if form == "decode" else rng.randint(2, 8))
    return c


def _lengths(case):
    """(cached tokens with the new ones among them, new tokens) of each sequence."""
    rng = random.Random(case["pick"])
    lens = [rng.randint(case["len_min"], case["len_max"]) for _ in range(case["batch"])]
    return lens, [min(n, rng.randint(case["new_min"], case["new_max"])) for n in lens]


_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _values(shape, dtype, gen):
    """Keys or values: normal numbers with channels of different strength (as learned projections give), a few far out."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    x *= torch.exp(0.5 * torch.randn(shape[-2:], generator=gen, device="cuda"))
    return x.to(dtype)


def _slots(tokens, tpb, blocks, gen):
    """Slots of a sequence of `tokens` tokens over pages that lie anywhere in the pool."""
    pages = torch.randperm(blocks, generator=gen, device="cuda")[: -(-tokens // tpb)]
    return (pages[:, None] * tpb + torch.arange(tpb, device="cuda")).reshape(-1)[:tokens].contiguous()


def _filled(kv, blocks, heads, dim, tpb, gen):
    """A layer of the cache with quantised content, and its bytes."""
    layer = torch.empty(kv, blocks, heads, tpb // UNIT, 9 * dim, dtype=torch.uint8, device="cuda")
    part = max(1, (1 << 27) // (heads * tpb * dim))
    for side in range(kv):
        for b in range(0, blocks, part):
            n = min(part, blocks - b)
            x = _values((n, tpb, heads, dim), torch.bfloat16, gen)
            layer[side, b : b + n] = _bytes(x.transpose(1, 2).reshape(n, heads, tpb // UNIT, UNIT, dim))
    return layer


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, heads, dim, tpb, dtype = case["kind"], case["heads"], case["dim"], case["tpb"], _TYPES[case["dtype"]]
    if kind == "attend":
        lens, new = _lengths(case)
        pages = [-(-n // tpb) for n in lens]
        layer = _filled(2, sum(pages) + 3, heads, dim, tpb, gen)
        order = torch.randperm(layer.shape[1], generator=gen, device="cuda").to(torch.int32)
        starts = torch.tensor([sum(pages[:i]) for i in range(len(pages))], device="cuda")
        at = torch.arange(max(pages), device="cuda")
        counts = torch.tensor(pages, device="cuda")
        tables = torch.where(at < counts[:, None], order[(starts[:, None] + at).clamp(max=len(order) - 1)], 0).to(torch.int32)
        q = torch.randn(sum(new), heads * case["group"], dim, generator=gen, device="cuda").to(dtype)
        ends = [sum(new[: i + 1]) for i in range(len(new))]
        same = max(new) == 1 and min(new) == 1
        return dict(case=case, layer=layer, q=q, tables=tables, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                    starts=None if same else torch.tensor([0] + ends, dtype=torch.int32, device="cuda"), longest=max(new),
                    scale=dim ** -0.5)
    kv = 1 if case["mla"] else 2
    if kind == "blocks":
        layers, n = case["layers"], case["blocks"]
        pool = n + 7
        source = _values((layers, kv, pool, tpb, heads, dim), dtype, gen)
        ids = [torch.randperm(pool, generator=gen, device="cuda")[:n].contiguous() for _ in range(3)]
        target = torch.zeros_like(source)
        return dict(case=case, source=list(source), target=target, targets=list(target), ids=ids,
                    packed=[torch.zeros(kv, pool, heads, tpb // UNIT, 9 * dim, dtype=torch.uint8, device="cuda") for _ in range(layers)])
    tokens = case["tokens"]
    blocks = -(-tokens // tpb) + 5
    slots = _slots(tokens, tpb, blocks, gen)
    if kind == "read":
        return dict(case=case, layer=_filled(kv, blocks, heads, dim, tpb, gen), slots=slots, dtype=dtype)
    if case["padded"]:
        slots[-case["padded"]:] = -1
    if case["fused"]:  # slices of what one projection gives: queries, keys and values of a token in one row
        rows = _values((tokens, 3 * kv * heads, dim), dtype, gen)
        k, v = rows[:, -kv * heads :][:, :heads], rows[:, -heads:]
    else:
        k, v = _values((tokens, heads, dim), dtype, gen), _values((tokens, heads, dim), dtype, gen)
    return dict(case=case, layer=torch.zeros(kv, blocks, heads, tpb // UNIT, 9 * dim, dtype=torch.uint8, device="cuda"), slots=slots,
                k=k, v=v if kv == 2 else None, dtype=dtype)


# ---- plain forms ---------------------------------------------------------------------------------------------


def _quantised(x):
    """Codes and scale codes of the groups of x [..., dim]: uint8 [..., dim / 16, 16] and uint8 [..., dim / 16]."""
    x = x.float().unflatten(-1, (-1, GROUP))
    x = torch.where(x.isnan(), 0.0, x)
    s = (x.abs().amax(-1) / 6).clamp(max=SCALE_MAX)
    e = torch.frexp(s.clamp(min=2.0 ** -14))[1] - 1
    step = torch.ldexp(torch.ones_like(s), e - 3)
    s = (s / step).round() * step
    code = (s.half().view(torch.int16) >> 7).to(torch.uint8)
    y = torch.where(s[..., None] > 0, x / s[..., None], 0.0)
    a = y.abs().clamp(max=6)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (a / step).round() * step
    c = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    return c + 8 * (y < 0).to(torch.uint8), code


def _bytes(x):
    """Units of x [..., 16 tokens, dim]: uint8 [..., 9 * dim]."""
    c, code = _quantised(x)
    c = c.flatten(-2).unflatten(-1, (-1, 2))
    return torch.cat([(c[..., 0] + 16 * c[..., 1]).flatten(-2), code.flatten(-2)], -1)


def _dequantised(rows, codes):
    """float32 [..., dim] of payload rows [..., dim / 2] and scale codes [..., dim / 16]."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=rows.device)
    q = table[torch.stack([rows & 15, rows >> 4], -1).flatten(-2).int()]
    s = (codes.to(torch.int16) << 7).view(torch.float16).float()
    return (q.unflatten(-1, (-1, GROUP)) * s[..., None]).flatten(-2)


def _rows(units, dim):
    """Payload rows and scale codes of units [..., 9 * dim]: [..., 16, dim / 2], [..., 16, dim / 16]."""
    return units[..., : 8 * dim].unflatten(-1, (UNIT, -1)), units[..., 8 * dim :].unflatten(-1, (UNIT, -1))


def _read(layer, slots, dim, dtype):
    tpb = layer.shape[3] * UNIT
    at = slots.clamp(min=0)
    rows, codes = _rows(layer, dim)
    pick = lambda t: t.permute(1, 3, 4, 0, 2, 5)[at // tpb, at % tpb // UNIT, at % UNIT]  # [tokens, kv, heads, bytes]  # noqa: E731
    x = _dequantised(pick(rows), pick(codes))
    x = torch.where((slots >= 0)[:, None, None, None], x, 0.0).to(dtype)
    return [x[:, i].contiguous() for i in range(x.shape[1])]


def _append(s):
    layer, slots, case = s["layer"], s["slots"], s["case"]
    dim, tpb = case["dim"], case["tpb"]
    x = torch.stack([s["k"]] + ([s["v"]] if s["v"] is not None else []), 1)  # [tokens, kv, heads, dim]
    n = slots.numel() - case["padded"]
    c, code = _quantised(x[:n])
    c = c.flatten(-2).unflatten(-1, (-1, 2))
    rows, codes = _rows(layer, dim)
    at = slots[:n]
    rows.permute(1, 3, 4, 0, 2, 5)[at // tpb, at % tpb // UNIT, at % UNIT] = c[..., 0] + 16 * c[..., 1]
    codes.permute(1, 3, 4, 0, 2, 5)[at // tpb, at % tpb // UNIT, at % UNIT] = code
    return _read(layer, slots, dim, s["dtype"])


def _blocks(s):
    case, (a, b, c) = s["case"], s["ids"]
    x = torch.stack([t[:, a] for t in s["source"]])  # [layers, kv, blocks, tpb, heads, dim]
    units = _bytes(x.transpose(3, 4).unflatten(4, (-1, UNIT)))
    rows, codes = _rows(units, case["dim"])
    back = _dequantised(rows, codes).flatten(4, 5).transpose(3, 4)
    s["target"][:, :, c] = back.to(s["target"].dtype)
    return s["target"]


def _attend(s):
    case, q, tables, lens = s["case"], s["q"], s["tables"].long(), s["lens"].long()
    batch, heads, group, dim, tpb = case["batch"], case["heads"], case["group"], case["dim"], case["tpb"]
    rows, codes = _rows(s["layer"][:, tables], dim)  # [2, batch, pages, heads, units, 16, bytes]
    kv = _dequantised(rows, codes).permute(0, 1, 3, 2, 4, 5, 6).flatten(3, 5)  # [2, batch, heads, positions, dim]
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(batch + 1, device=q.device)
    new = starts[1:] - starts[:-1]
    row = torch.arange(s["longest"], device=q.device)
    there = row < new[:, None]  # [batch, rows]
    at = (starts[:-1, None] + row).clamp(max=q.shape[0] - 1)
    x = q[at].float().view(batch, -1, heads, group, dim).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [batch, heads, rows * group, dim]
    scores = (x @ kv[0].transpose(-1, -2)).mul_(s["scale"]).unflatten(2, (-1, group))
    last = lens[:, None] - new[:, None] + row
    hidden = torch.arange(kv.shape[3], device=q.device) > last[..., None]
    scores.masked_fill_(hidden[:, None, :, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    o = (scores.flatten(2, 3) @ kv[1]).unflatten(2, (-1, group)) / total
    o = o.permute(0, 2, 1, 3, 4).flatten(2, 3)  # [batch, rows, query heads, dim]
    return o[there].to(q.dtype)


def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        from flexkv_b200 import fp4_cache

        if kind == "append":
            fp4_cache.fp4_write(s["layer"], s["k"], s["v"], s["slots"])
            return [x for x in fp4_cache.fp4_read(s["layer"], s["slots"], s["dtype"]) if x is not None]
        if kind == "read":
            return [x for x in fp4_cache.fp4_read(s["layer"], s["slots"], s["dtype"]) if x is not None]
        if kind == "blocks":
            a, b, c = s["ids"]
            fp4_cache.fp4_pack_blocks(s["source"], s["packed"], a, b)
            fp4_cache.fp4_unpack_blocks(s["packed"], s["targets"], b, c)
            return s["target"]
        return fp4_cache.fp4_attention(s["layer"], s["q"], s["tables"], s["lens"], cu_seqlens_q=s["starts"], max_q_len=s["longest"],
                                       softmax_scale=s["scale"])
    if kind == "append":
        return _append(s)
    if kind == "read":
        return _read(s["layer"], s["slots"], s["case"]["dim"], s["dtype"])
    if kind == "blocks":
        return _blocks(s)
    return _attend(s)


def work(case):
    heads, dim, kind = case["heads"], case["dim"], case["kind"]
    if kind == "attend":
        lens, new = _lengths(case)
        seen = sum(m * n - m * (m - 1) // 2 for n, m in zip(lens, new))  # pairs of a new token and a key that it sees
        cache = sum(lens) * 2 * heads * dim * 9 // 16 + 4 * sum(-(-n // case["tpb"]) for n in lens)
        return {"bytes": cache + 2 * 2 * sum(new) * heads * case["group"] * dim, "flops": 4 * seen * heads * case["group"] * dim}
    kv = 1 if case["mla"] else 2
    if kind == "blocks":
        values = case["layers"] * kv * case["blocks"] * case["tpb"] * heads * dim
        return {"bytes": values * (2 + 9 / 16) * 2, "flops": 6 * values}
    values = case["tokens"] * kv * heads * dim
    if kind == "read":
        return {"bytes": values * (2 + 9 / 16) + 8 * case["tokens"], "flops": values}
    values = (case["tokens"] - case["padded"]) * kv * heads * dim
    return {"bytes": values * (2 + 2 * 9 / 16) + 2 * case["tokens"] * kv * heads * dim + 8 * case["tokens"], "flops": 6 * values}


# ---- the definition, in 64 bits ------------------------------------------------------------------------------


def _nearest(x, grid):
    """The value of the ascending grid nearest to x >= 0, the one with the even index where two are as near."""
    mid = (grid[1:] + grid[:-1]) / 2
    low = torch.searchsorted(mid, x, right=False)  # a tie goes down ...
    high = torch.searchsorted(mid, x, right=True)  # ... or up
    return grid[torch.where(low % 2 == 0, low, high)]


def _stored64(x):
    """What the cache holds of x [..., dim], in 64 bits."""
    code = torch.arange(227, device=x.device)
    scales = torch.where(code < 8, code * 2.0 ** -17, (8 + code % 8) * 2.0 ** (code // 8 - 18.0)).double()
    values = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    x = x.double().unflatten(-1, (-1, GROUP)).nan_to_num(0.0)
    s = _nearest(x.abs().amax(-1) / 6, scales)[..., None]
    return (torch.where(s > 0, _nearest(x.abs() / s.clamp(min=2.0 ** -20), values) * s, 0.0) * x.sign()).flatten(-2)


def _held64(layer, dim):
    """Every value of a layer: [kv, blocks, heads, tpb, dim], in 64 bits."""
    u = layer.long()
    codes, c = u[..., 8 * dim :].reshape(*u.shape[:-1], UNIT, -1), u[..., : 8 * dim].reshape(*u.shape[:-1], UNIT, -1)
    s = torch.where(codes < 8, codes.double() * 2.0 ** -17, (8 + codes % 8).double() * torch.exp2((codes // 8).double() - 18))
    c = torch.stack([c % 16, c // 16], -1).flatten(-2)
    m, e = c % 2, c // 2 % 4
    v = torch.where(e == 0, m * 0.5, (1 + m * 0.5) * torch.exp2(e.double() - 1)) * (1 - 2 * (c // 8))
    return (v * s.repeat_interleave(GROUP, -1)).flatten(3, 4)


def exact(case, seed):
    s, kind, dim, tpb = prepare(case, seed), case["kind"], case["dim"], case["tpb"]
    if kind == "append":
        keep = (s["slots"] >= 0)[:, None, None]
        return [torch.where(keep, _stored64(x), 0.0) for x in (s["k"], s["v"]) if x is not None]
    if kind == "read":
        held = _held64(s["layer"], dim).transpose(2, 3).flatten(1, 2)  # [kv, slots, heads, dim]
        return [side[s["slots"]] for side in held]
    if kind == "blocks":
        a, _, c = s["ids"]
        out = torch.zeros(s["target"].shape, dtype=torch.float64, device="cuda")
        for layer, x in enumerate(s["source"]):
            out[layer][:, c] = _stored64(x[:, a])
        return out
    lens, new = _lengths(case)
    outs, first = [], 0
    for b, (n, m) in enumerate(zip(lens, new)):
        k, v = _held64(s["layer"][:, s["tables"][b, : -(-n // tpb)].long()], dim).transpose(2, 3).flatten(1, 2)[:, :n]
        o = torch.empty(m, case["heads"], case["group"], dim, dtype=torch.float64, device="cuda")
        for h in range(case["heads"]):
            q = s["q"][first : first + m].double().view(m, case["heads"], case["group"], dim)[:, h]
            w = torch.einsum("mgd,nd->mgn", q, k[:, h]) * s["scale"]
            seen = torch.arange(n, device="cuda") <= torch.arange(n - m, n, device="cuda")[:, None]
            w = torch.softmax(torch.where(seen[:, None], w, -math.inf), -1)
            o[:, h] = torch.einsum("mgn,nd->mgd", w, v[:, h])
        outs.append(o.flatten(1, 2))
        first += m
    return torch.cat(outs)

"""GPU: the 4-bit cache's operators against their 64-bit definition
(fp4_model), bit for bit where they store or read values, within derived
bounds where they sum."""
import numpy as np
import pytest
import torch

import fp4_model as M
from flexkv_b200 import c_ext, fp4_cache
from flexkv_b200.layout import KVCacheLayout, KVCacheLayoutType, cpu_byte_strides, gpu_byte_strides

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def f64(t):
    return t.detach().cpu().double().numpy()


def noise(shape, dtype, seed, spread=4.0):
    """Normal values whose magnitude varies by group over a range that reaches the scale grid's ends."""
    r = np.random.RandomState(seed)
    x = r.randn(*shape).reshape(*shape[:-1], -1, 16)
    x = x * np.exp(spread * r.randn(*x.shape[:-1], 1))
    x[r.rand(*x.shape[:-1]) < 0.05] = 0
    x[r.rand(*x.shape[:-1]) < 0.05] *= 1e-7
    return torch.from_numpy(np.clip(x.reshape(shape), -6e4, 6e4)).to(DT[dtype]).cuda()


def garbage(kv, blocks, heads, tpb, dim):
    """A layer of 0xFF bytes: what is not written decodes to NaN."""
    return torch.full((kv, blocks, heads, tpb // 16, 9 * dim), 255, dtype=torch.uint8, device="cuda")


def written(kv, blocks, heads, tpb, dim, seed, spread=0.5):
    """A layer with every slot written, by the model."""
    r = np.random.RandomState(seed)
    layer = np.zeros((kv, blocks, heads, tpb // 16, 9 * dim), dtype=np.uint8)
    for side in range(kv):
        x = r.randn(blocks, heads, tpb // 16, 16, dim) * np.exp(spread * r.randn(heads, 1, 1, dim))
        layer[side] = M.unit_bytes(*M.quantise(x))
    return layer


# ---- write and read -------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kv,heads,dim,tpb,n", [
    (2, 8, 128, 16, 1), (2, 4, 128, 16, 15), (2, 2, 64, 32, 16), (2, 1, 64, 16, 17), (1, 1, 576, 64, 100),
    (2, 3, 16, 48, 333), (1, 5, 80, 16, 31), (2, 8, 256, 128, 70)])
def test_write_and_read(dtype, kv, heads, dim, tpb, n):
    blocks = -(-n // tpb) + 3
    k = noise((n, heads, dim), dtype, 1)
    v = noise((n, heads, dim), dtype, 2) if kv == 2 else None
    r = np.random.RandomState(3)
    slots = r.permutation(blocks * tpb)[:n].astype(np.int64)
    if n > 4:
        slots[[1, n - 1]] = -1, blocks * tpb + 5  # dropped
    layer = garbage(kv, blocks, heads, tpb, dim)
    want = layer.cpu().numpy()
    fp4_cache.fp4_write(layer, k, v, torch.from_numpy(slots).cuda())
    M.write(want, [f64(x) for x in (k, v) if x is not None], slots)
    # the byte of a negative zero is the kernel's own affair: compare values, and unwritten bytes
    assert np.array_equal(np.nan_to_num(M.held(layer.cpu().numpy()), nan=7e7), np.nan_to_num(M.held(want), nan=7e7))
    untouched = np.setdiff1d(np.arange(blocks * tpb), slots)
    full = np.full_like(want, 255)
    assert np.array_equal(M.held(full)[:, untouched], M.held(layer.cpu().numpy())[:, untouched], equal_nan=True)
    for out_dtype in ("bf16", "fp16"):
        got = fp4_cache.fp4_read(layer, torch.from_numpy(slots).cuda(), DT[out_dtype])
        assert (got[1] is None) == (kv == 1)
        held = M.held(want)
        ok = (slots >= 0) & (slots < blocks * tpb)
        for side in range(kv):
            w = np.where(ok[:, None, None], held[side][np.where(ok, slots, 0)], 0.0)
            assert got[side].dtype == DT[out_dtype] and np.array_equal(f64(got[side]), w)


def test_every_value_of_both_types():
    """Every finite 16-bit pattern, infinities and NaN, against a group maximum of its own size."""
    bits = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    for dtype in ("bf16", "fp16"):
        x = torch.from_numpy(bits.view(np.int16).copy()).view(DT[dtype])
        for fill in (0.0, 1.0, 6.0, 100.0, 3e-4, 60000.0):
            rows = torch.full((65536 // 8, 16), fill, dtype=DT[dtype])
            rows[:, :8] = x.view(-1, 8)
            rows = rows.view(-1, 1, 64).cuda()  # [2048, 1, 64]
            layer = garbage(1, 2048 // 16, 1, 16, 64)
            slots = torch.arange(2048, device="cuda")
            fp4_cache.fp4_write(layer, rows, None, slots)
            want = M.dequantise(*M.quantise(f64(rows)))
            assert np.array_equal(M.held(layer.cpu().numpy())[0], want), (dtype, fill)
            assert np.array_equal(f64(fp4_cache.fp4_read(layer, slots, DT[dtype])[0]), want)


def test_ties_and_scales():
    """Values on every border of both grids: amax / 6 halfway between two scales, x / s halfway between two values."""
    for dtype in ("bf16", "fp16"):
        rows = []
        for c in range(0, 226):
            for a in ((M.SCALES[c] + M.SCALES[c + 1]) * 3, M.SCALES[c] * 6):
                for tie in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
                    t = torch.tensor([a, tie * M.SCALES[c], tie * M.SCALES[c + 1], -tie * M.SCALES[c]]).to(DT[dtype])
                    rows.append(torch.cat([t, torch.nextafter(t.float(), torch.tensor(9e9)).to(DT[dtype]), torch.zeros(8, dtype=DT[dtype])]))
        x = torch.stack(rows)
        x = torch.cat([x, torch.zeros(-len(x) % 64, 16, dtype=DT[dtype])]).view(-1, 1, 64).cuda()
        n = x.shape[0]
        layer = garbage(1, -(-n // 16), 1, 16, 64)
        fp4_cache.fp4_write(layer, x, None, torch.arange(n, device="cuda"))
        assert np.array_equal(M.held(layer.cpu().numpy())[0][:n], M.dequantise(*M.quantise(f64(x))))


@pytest.mark.parametrize("heads", [1, 4])
def test_strides(heads):
    """k and v as slices of one projection (rows on 16- but not 32-byte boundaries too), transposed heads, a layer
    that is one of several in a larger tensor, reads into slices."""
    n, dim, tpb = 37, 64, 16
    pool = torch.full((2, 3, 5, heads, 1, 9 * dim), 255, dtype=torch.uint8, device="cuda")
    layer = pool[:, 1]  # kv stride of three layers
    slots = torch.randperm(80, device="cuda")[:n]
    for lead in (0, 8, 16):
        rows = noise((n, 3 * heads, dim), "bf16", lead)
        flat = torch.zeros(n, 3 * heads * dim + 32, dtype=torch.bfloat16, device="cuda")
        flat[:, lead:lead + 3 * heads * dim] = rows.flatten(1)
        k = flat[:, lead + heads * dim:lead + 2 * heads * dim].unflatten(1, (heads, dim))
        v = flat[:, lead + 2 * heads * dim:lead + 3 * heads * dim].unflatten(1, (heads, dim))
        v2 = v.transpose(0, 1).contiguous().transpose(0, 1)
        fp4_cache.fp4_write(layer, k, v2, slots)
        a = torch.zeros(n, heads, 2, dim, dtype=torch.bfloat16, device="cuda")
        fp4_cache.fp4_read(layer, slots, out=(a[:, :, 0], a[:, :, 1]))
        for got, x in ((a[:, :, 0], k), (a[:, :, 1], v)):
            assert np.array_equal(f64(got), M.dequantise(*M.quantise(f64(x))))
    assert bool((pool[:, 0] == 255).all()) and bool((pool[:, 2] == 255).all())
    every_other = torch.stack([slots, torch.full_like(slots, -1)], 1).flatten()[::2]
    assert torch.equal(fp4_cache.fp4_read(layer, every_other)[0], a[:, :, 0])


def test_refusals():
    layer = garbage(2, 4, 2, 16, 64)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(3, device="cuda")
    w, r = fp4_cache.fp4_write, fp4_cache.fp4_read
    for call in (lambda: w(layer, x, None, slots), lambda: w(layer[:1], x, x, slots), lambda: w(layer, x, x.half(), slots),
                 lambda: w(layer, x.float(), x.float(), slots), lambda: w(layer, x, x, slots.int()),
                 lambda: w(layer, x, x, slots.cpu()), lambda: w(layer, x, x, slots[:2]), lambda: w(layer, x.cpu(), x, slots),
                 lambda: w(layer, x[:, :1], x[:, :1], slots), lambda: w(layer.transpose(2, 3), x, x, slots),
                 lambda: w(layer, x.transpose(0, 2).contiguous().transpose(0, 2), x, slots),
                 lambda: w(layer[..., :9 * 60], x, x, slots), lambda: w(layer, x.clone().requires_grad_(), x, slots),
                 lambda: w(layer, torch.zeros(3 * 132, dtype=torch.bfloat16, device="cuda").as_strided((3, 2, 64), (132, 64, 1)), x, slots),
                 lambda: r(layer, slots, torch.float32), lambda: r(layer, slots[None]),
                 lambda: r(layer, slots, out=(x, None)), lambda: r(layer, slots, out=(x.half(), x.half()))):
        with pytest.raises(RuntimeError):
            call()
    assert bool((layer == 255).all())
    w(layer, x[:0], x[:0], slots[:0])
    assert r(layer, slots[:0])[0].shape == (0, 2, 64)


# ---- blocks ---------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("layers,kv,heads,dim,tpb,n", [(1, 2, 8, 128, 16, 1), (3, 2, 2, 64, 32, 7), (2, 1, 1, 576, 64, 5),
                                                       (130, 2, 1, 16, 16, 3)])
def test_blocks(dtype, layers, kv, heads, dim, tpb, n):
    r = np.random.RandomState(layers)
    src = [noise((kv, n + 2, tpb, heads, dim), dtype, l) for l in range(layers)]
    dst = [torch.full_like(x, 5.0) for x in src]
    packed = [garbage(kv, n + 3, heads, tpb, dim) for _ in range(layers)]
    a, b, c = (torch.from_numpy(r.permutation(n + 2)[:n].astype(np.int64)) for _ in range(3))
    fp4_cache.fp4_pack_blocks(src, packed, a, b.cuda())
    fp4_cache.fp4_unpack_blocks(packed, dst, b, c.cuda())
    rest = np.setdiff1d(np.arange(n + 2), c.numpy())
    for l in range(0, layers, 43 if layers > 100 else 1):
        want = M.dequantise(*M.quantise(f64(src[l])[:, a.numpy()]))
        assert np.array_equal(f64(dst[l])[:, c.numpy()], want)
        assert bool((dst[l][:, rest] == 5.0).all())
        assert bool((packed[l][:, np.setdiff1d(np.arange(n + 3), b.numpy())] == 255).all())


def test_blocks_bad_ids():
    src, packed = [noise((2, 6, 16, 2, 64), "bf16", 0)], [garbage(2, 4, 2, 16, 64)]
    ids = lambda *v: torch.tensor(v, dtype=torch.int64)  # noqa: E731
    for a, b in ((ids(0, 6), ids(0, 1)), (ids(0, -1), ids(0, 1)), (ids(0, 1), ids(0, 4)), (ids(0, 1), ids(2, 2)),
                 (ids(0), ids(0, 1)), (ids(0, 1).int(), ids(0, 1))):
        with pytest.raises(RuntimeError):
            fp4_cache.fp4_pack_blocks(src, packed, a, b)
    for a, b in ((ids(0, 1), ids(3, 3)), (ids(0, 4), ids(0, 1))):
        with pytest.raises(RuntimeError):
            fp4_cache.fp4_unpack_blocks(packed, src, a, b)
    assert bool((packed[0] == 255).all())
    # on the device such pairs are skipped; a source may repeat
    fp4_cache.fp4_pack_blocks(src, packed, ids(-1, 2, 6, 2, 3).cuda(), ids(0, 1, 2, 3, 9).cuda())
    got = M.held(packed[0].cpu().numpy()).reshape(2, 4, 16, 2, 64)
    want = M.dequantise(*M.quantise(f64(src[0])[:, 2]))
    assert bool((packed[0][:, [0, 2]] == 255).all())
    assert np.array_equal(got[:, 1], want) and np.array_equal(got[:, 3], want)
    before = src[0].clone()
    fp4_cache.fp4_unpack_blocks(packed, src, ids(-5, 1, 4).cuda(), ids(0, 7, 2).cuda())
    assert torch.equal(src[0], before)


# ---- attention ------------------------------------------------------------------------------------------------


def batch(lens, new, tpb, seed, width=None, holes=False):
    """Block tables over a shuffled pool, with garbage past each sequence's pages."""
    r = np.random.RandomState(seed)
    pages = [-(-n // tpb) for n in lens]
    blocks = sum(pages) + 2
    order = r.permutation(blocks)
    w = max(pages + [1]) + 1 if width is None else width
    tables = np.full((len(lens), w), -12345, dtype=np.int32)
    tables[1::2] = 2 ** 30
    at = 0
    for b, p in enumerate(pages):
        tables[b, :min(p, w)] = order[at:at + min(p, w)]
        at += p
    if holes:
        tables[r.rand(*tables.shape) < 0.2] = blocks
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return blocks, tables, np.array(lens, dtype=np.int32), cu


def spoil(layer, tables, lens, tpb):
    """NaN in every byte that no sequence owns: other blocks, and the tails of last pages."""
    seen = np.zeros(layer.shape[1] * tpb, dtype=bool)
    for b, n in enumerate(lens.tolist()):
        for j in range(min(max(n, 0), tables.shape[1] * tpb)):
            p = tables[b, j // tpb]
            if 0 <= p < layer.shape[1]:
                seen[p * tpb + j % tpb] = True
    d = layer.shape[-1] // 9
    for s in np.flatnonzero(~seen):
        b, u, t = s // tpb, s % tpb // 16, s % 16
        layer[:, b, :, u, t * d // 2:(t + 1) * d // 2] = 255
        layer[:, b, :, u, 8 * d + t * d // 16:8 * d + (t + 1) * d // 16] = 255


def check_attention(heads, group, dim, tpb, dtype, lens, new, causal=True, seed=0, spread=0.5, uniform=False, **kw):
    blocks, tables, lens, cu = batch(lens, new, tpb, seed, kw.get("width"), kw.get("holes", False))
    layer = written(2, blocks, heads, tpb, dim, seed + 1, spread)
    spoil(layer, tables, lens, tpb)
    behind = 0 if uniform else 3
    n = int(cu[-1]) + behind
    r = np.random.RandomState(seed + 2)
    q = torch.from_numpy(r.randn(n, heads * group, dim) * kw.get("size", 1.0)).to(DT[dtype]).cuda()
    scale = kw.get("scale", dim ** -0.5)
    out = torch.full((n, heads * group, dim), 3.0, dtype=DT[dtype], device="cuda")
    got, lse = fp4_cache.fp4_attention(
        torch.from_numpy(layer).cuda(), q, torch.from_numpy(tables).cuda(), torch.from_numpy(lens).cuda(),
        cu_seqlens_q=None if uniform else torch.from_numpy(cu).cuda(), max_q_len=kw.get("max_q_len", max(list(new) + [0])),
        softmax_scale=scale, causal=causal, out=out, return_lse=True)
    assert got is out
    want, wlse, weight, size = M.attention(layer, f64(q), tables, lens, cu, scale, causal, tpb)
    owned = int(cu[-1])
    assert bool((out[owned:] == 3.0).all()) and bool(torch.isneginf(lse[owned:]).all())
    o, l = f64(out)[:owned], f64(lse)[:owned]
    want, wlse, weight, size = want[:owned], wlse[:owned], weight[:owned], size[:owned]
    bound = M.attention_bounds(weight, size, want, dim, dtype)
    assert np.isfinite(o).all()
    off = np.abs(o - want) / bound
    assert off.max(initial=0) <= 1, (off.max(), np.unravel_index(off.argmax(), off.shape))
    empty = np.isneginf(wlse)
    assert np.array_equal(empty, np.isneginf(l)) and not np.any(o[empty])
    # the sum of exponentials: the scores' error, float32 sums, and the logarithm's own rounding
    lbound = (dim / 16 + 8) * 2.0 ** -23 * size + 2.0 ** -14 + 2.0 ** -22 * np.abs(wlse)
    assert (np.abs(l - wlse)[~empty] <= lbound[~empty]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,group,dim,tpb", [(1, 1, 64, 16), (2, 4, 128, 16), (4, 7, 128, 32), (1, 8, 64, 64),
                                                 (1, 16, 128, 48), (2, 3, 64, 16), (1, 24, 64, 16), (1, 71, 128, 16)])
def test_decode(dtype, heads, group, dim, tpb):
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 127, 128, 129, 200, 777]
    check_attention(heads, group, dim, tpb, dtype, lens, [1] * len(lens), uniform=True)


@pytest.mark.parametrize("lens", [[1], [5000], [3, 2500, 1, 0, 40]])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_few_sequences(dim, lens):
    """The keys of one sequence spread over many CTAs and joined."""
    check_attention(2, 4, dim, 16, "bf16", lens, [1] * len(lens), uniform=True)


def test_decode_many_sequences():
    r = np.random.RandomState(1)
    lens = r.randint(0, 40, 700).tolist()
    check_attention(1, 2, 64, 16, "fp16", lens, [1] * 700, uniform=True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,group,dim,tpb", [(2, 4, 128, 16), (1, 7, 64, 32), (3, 1, 128, 64), (1, 16, 64, 16)])
def test_few_new_tokens(causal, dtype, heads, group, dim, tpb):
    lens, new = [5, 100, 33, 0, 300, 17, 8, 2], [5, 3, 0, 0, 8, 1, 4, 5]  # the last sees nothing in its first rows
    check_attention(heads, group, dim, tpb, dtype, lens, new, causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,group,dim,tpb", [(2, 4, 128, 16), (1, 7, 64, 32), (2, 1, 128, 64), (1, 16, 64, 16)])
def test_prompts(causal, heads, group, dim, tpb):
    lens, new = [150, 1, 300, 64, 40, 257, 0], [150, 1, 70, 64, 60, 129, 0]
    check_attention(heads, group, dim, tpb, "bf16", lens, new, causal)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_longer_prompt(dtype):
    check_attention(1, 2, 128, 16, dtype, [700, 513], [600, 200], True)


@pytest.mark.parametrize("new", [1, 3, 90])
def test_bad_pages(new):
    """Pages outside the pool and tables narrower than the sequences hide their tokens."""
    check_attention(2, 4, 128, 16, "bf16", [200, 333, 100], [new] * 3, holes=True, uniform=new == 1)
    check_attention(2, 4, 64, 16, "fp16", [200, 333, 100], [new] * 3, width=7, uniform=new == 1)


@pytest.mark.parametrize("new", [1, 3, 90])
def test_wrong_max_q_len(new):
    """max_q_len only chooses the kernel."""
    for m in (0, 1, 5, 1000):
        check_attention(1, 4, 64, 16, "bf16", [200, 90], [new] * 2, max_q_len=m)


@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("size,scale", [(60.0, 0.125), (1.0, 0.0), (1.0, -0.125), (1e-3, 0.1), (3e4, 2e-5)])
def test_sizes_of_scores(new, size, scale):
    """Scores of some hundreds, all equal, falling, and tiny or huge queries."""
    check_attention(1, 4, 64, 16, "bf16", [250, 180], [new] * 2, size=size, scale=scale, uniform=new == 1)


@pytest.mark.parametrize("new", [1, 70])
def test_wide_values(new):
    check_attention(1, 4, 128, 16, "bf16", [250, 180], [new] * 2, spread=2.0, scale=0.01, uniform=new == 1)


def test_queries_beyond_half():
    """bfloat16 queries past half precision's range on both sides."""
    for size, scale in ((1e30, 1e-31), (1e-30, 1e29)):
        check_attention(1, 4, 64, 16, "bf16", [250], [1], size=size, scale=scale, uniform=True)
        check_attention(1, 4, 64, 16, "bf16", [250], [80], size=size, scale=scale)


def test_bad_query_rows_stay_alone():
    """NaN or infinite queries spoil their own rows and no others."""
    for new in (1, 4, 100):
        blocks, tables, lens, cu = batch([300, 200], [new] * 2, 16, 5)
        layer = torch.from_numpy(written(2, blocks, 1, 16, 128, 6)).cuda()
        q = torch.randn(2 * new, 4, 128, device="cuda").bfloat16()
        args = (torch.from_numpy(tables).cuda(), torch.from_numpy(lens).cuda(), torch.from_numpy(cu).cuda(), new)
        clean = fp4_cache.fp4_attention(layer, q, *args)
        q[0, 1, 5], q[new, 2, 7] = float("nan"), float("inf")
        got = fp4_cache.fp4_attention(layer, q, *args)
        assert bool(got[0, 1].isnan().all()) and bool(got[new, 2].isnan().any())
        clean[0, 1], clean[new, 2], got[0, 1], got[new, 2] = 0, 0, 0, 0
        assert torch.equal(got, clean)


@pytest.mark.parametrize("new", [1, 5, 100])
def test_strided_queries(new):
    """q as the query part of a projection, out and tables as slices."""
    heads, group, dim = 2, 4, 64
    blocks, tables, lens, cu = batch([300, 120], [new] * 2, 16, 7)
    layer = torch.from_numpy(written(2, blocks, heads, 16, dim, 8)).cuda()
    rows = torch.randn(2 * new, heads * group * dim + 40, device="cuda").bfloat16()
    q = rows[:, 8:8 + heads * group * dim].unflatten(1, (heads * group, dim))
    wide = torch.zeros(2, tables.shape[1] + 5, dtype=torch.int32, device="cuda")
    wide[:, :tables.shape[1]] = torch.from_numpy(tables)
    lens2 = torch.from_numpy(lens).cuda()
    cu2 = torch.from_numpy(cu).cuda()
    want = fp4_cache.fp4_attention(layer, q.contiguous(), torch.from_numpy(tables).cuda(), lens2, cu2, new)
    out = torch.zeros(2 * new, heads * group, 2, dim, dtype=torch.bfloat16, device="cuda")
    fp4_cache.fp4_attention(layer, q, wide[:, :tables.shape[1]], lens2, cu2, new, out=out[:, :, 1])
    assert torch.equal(out[:, :, 1], want) and not bool(out[:, :, 0].any())
    swapped = torch.zeros(heads * group, 2 * new, dim, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    fp4_cache.fp4_attention(layer, q, wide[:, :tables.shape[1]].t().contiguous().t(), lens2, cu2, new, out=swapped)
    assert torch.equal(swapped, want)


def test_attention_refusals():
    layer = garbage(2, 4, 2, 16, 64)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    tables, lens = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    f = fp4_cache.fp4_attention
    for call in (lambda: f(layer[:1], q, tables, lens), lambda: f(layer, q[:, :3], tables, lens),
                 lambda: f(layer, q.float(), tables, lens), lambda: f(layer, q[..., :32], tables, lens),
                 lambda: f(layer, q, tables.long(), lens), lambda: f(layer, q, tables, lens.long()),
                 lambda: f(layer, q, tables[:1], lens), lambda: f(layer, q, tables, lens, cu[:2]),
                 lambda: f(layer, q, tables, lens, cu.long()), lambda: f(layer, q, tables, lens, cu, -1),
                 lambda: f(layer, torch.cat([q, q[:1]]), tables, lens), lambda: f(layer, q, tables.cpu(), lens),
                 lambda: f(layer, q, tables, lens, softmax_scale=float("nan")), lambda: f(layer, q, tables, lens, out=q.half()),
                 lambda: f(layer, q.clone().requires_grad_(), tables, lens), lambda: f(layer, q, tables, lens, out=q[:1]),
                 lambda: f(garbage(2, 4, 2, 16, 96), torch.zeros(2, 4, 96, dtype=torch.bfloat16, device="cuda"), tables, lens)):
        with pytest.raises(RuntimeError):
            call()
    empty = f(layer, q[:0], tables[:0], lens[:0])
    assert empty.shape == (0, 4, 64)
    # no row belongs to a sequence: zeros in a new output
    assert not bool(f(layer, q, tables, lens, cu, 1).any())
    # tables without columns, a pool without blocks
    o, l = f(layer, q, tables[:, :0], lens + 5, return_lse=True)
    assert not bool(o.any()) and bool(torch.isneginf(l).all())
    o = f(layer[:, :0], q, tables, lens + 5)
    assert not bool(o.any())


# ---- as they are used -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("tpb,heads,group,dim", [(16, 2, 4, 128), (32, 1, 7, 64)])
def test_serving_run(tpb, heads, group, dim):
    """A prompt is written and attended to, its full blocks go to the host pool and back into other blocks (with
    the framework's own transfers), then tokens are decoded on them: each step equals the definition."""
    layers, prompt, steps = 2, 3 * tpb + 5, 4
    lay = KVCacheLayout(KVCacheLayoutType.LAYERWISE, layers, 12, tpb, heads, dim)
    host = KVCacheLayout(KVCacheLayoutType.BLOCKWISE, layers, 6, tpb, heads, dim).fp4()
    cache = fp4_cache.allocate_fp4_layers(lay, "cuda")
    r = np.random.RandomState(0)
    table = r.permutation(12)[:5]
    slots = (table[:, None] * tpb + np.arange(tpb)).reshape(-1)
    model = [t.cpu().numpy() for t in cache]
    g, c = gpu_byte_strides(lay.fp4(), 1), cpu_byte_strides(host, 1)
    ptrs = torch.tensor([t.data_ptr() for t in cache], dtype=torch.int64)
    pool = torch.zeros(host.get_total_elements(), dtype=torch.uint8).pin_memory()

    def step(at, n):
        for l in range(layers):
            rows = [torch.from_numpy(r.randn(n, heads, dim)).bfloat16().cuda() for _ in range(2)]
            fp4_cache.fp4_write(cache[l], *rows, torch.from_numpy(slots[at:at + n]).cuda())
            M.write(model[l], [f64(x) for x in rows], slots[at:at + n])
            q = torch.from_numpy(r.randn(n, heads * group, dim)).bfloat16().cuda()
            tables, lens = np.asarray(table, dtype=np.int32)[None], np.array([at + n], dtype=np.int32)
            o = fp4_cache.fp4_attention(cache[l], q, torch.from_numpy(tables).cuda(), torch.from_numpy(lens).cuda())
            want, _, weight, size = M.attention(model[l], f64(q), tables, lens, np.array([0, n]), dim ** -0.5, True, tpb)
            assert (np.abs(f64(o) - want) <= M.attention_bounds(weight, size, want, dim, "bf16")).all()

    step(0, prompt)
    full = prompt // tpb
    ids, cpu_ids = torch.from_numpy(table[:full].astype(np.int64)), torch.tensor([4, 0, 5])[:full]
    args = (pool, c["kv"], c["layer"], c["block"], g["chunk"], 0)
    c_ext.transfer_kv_blocks(ids, ptrs, g["kv"], g["block"], cpu_ids, *args, is_host_to_device=False)
    for t in cache:
        t[:, ids] = 255
    fresh = np.setdiff1d(np.arange(12), table)[:full]
    c_ext.transfer_kv_blocks(torch.from_numpy(fresh), ptrs, g["kv"], g["block"], cpu_ids, *args, is_host_to_device=True)
    for l in range(layers):
        model[l][:, fresh] = model[l][:, table[:full]]
        model[l][:, table[:full]] = 255
        assert np.array_equal(M.held(cache[l].cpu().numpy()), M.held(model[l]), equal_nan=True)
    table[:full] = fresh
    slots = (table[:, None] * tpb + np.arange(tpb)).reshape(-1)
    for i in range(steps):
        step(prompt + i, 1)


def test_offload_run():
    """An engine with a 16-bit cache: blocks packed, sent to the host tier in 4 bits through the cache index's put,
    fetched by its get into other blocks, unpacked."""
    from flexkv_b200.cache_index import CpuCacheIndex, KVLayout
    from kvcase import tokens
    layers, tpb, heads, dim = 3, 16, 2, 64
    lay = KVCacheLayout(KVCacheLayoutType.LAYERWISE, layers, 16, tpb, heads, dim)
    host = KVCacheLayout(KVCacheLayoutType.BLOCKWISE, layers, 32, tpb, heads, dim).fp4()
    kv = [noise((2, 16, tpb, heads, dim), "bf16", l, 1.0) for l in range(layers)]
    cache = fp4_cache.allocate_fp4_layers(lay, "cuda")
    g, c = gpu_byte_strides(lay.fp4(), 1), cpu_byte_strides(host, 1)
    pool = torch.zeros(host.get_total_elements(), dtype=torch.uint8).pin_memory()
    layout = KVLayout(torch.tensor([t.data_ptr() for t in cache], dtype=torch.int64), g["kv"], g["block"], pool,
                      c["kv"], c["layer"], c["block"], g["chunk"], gpu_layer_bytes=cache[0].numel())
    index = CpuCacheIndex(32, tpb)
    toks = tokens(5 * tpb, 32000, 1)
    src, staged = torch.tensor([3, 9, 0, 7, 12]), torch.tensor([0, 1, 2, 3, 4])
    fp4_cache.fp4_pack_blocks(kv, cache, src, staged)
    res = index.put([toks], [staged.numpy()], layout)
    assert int(res.num_transferred[0]) == 5
    for t in cache:
        t.fill_(255)
    back = np.array([10, 11, 8, 15, 6], dtype=np.int64)
    got = index.get([toks], [back], layout)
    assert int(got.num_transferred[0]) == 5
    out = [torch.zeros_like(x) for x in kv]
    fp4_cache.fp4_unpack_blocks(cache, out, torch.from_numpy(back), src)
    for l in range(layers):
        assert np.array_equal(f64(out[l])[:, src.numpy()], M.dequantise(*M.quantise(f64(kv[l])[:, src.numpy()])))
    index.close()


def test_launches_are_counted():
    layer, slots = garbage(2, 4, 2, 16, 64), torch.arange(5, device="cuda")
    n = c_ext.kernel_launch_count()
    fp4_cache.fp4_read(layer, slots)
    assert c_ext.kernel_launch_count() == n + 1


def decode_state(seed, lens=(70, 1000, 0, 33), heads=2, group=4, dim=128, tpb=16, new=1):
    blocks, tables, lens, cu = batch(list(lens), [new] * len(lens), tpb, seed)
    layer = torch.from_numpy(written(2, blocks, heads, tpb, dim, seed)).cuda()
    q = torch.randn(new * len(lens), heads * group, dim, device="cuda").bfloat16()
    return layer, q, torch.from_numpy(tables).cuda(), torch.from_numpy(lens).cuda(), torch.from_numpy(cu).cuda()


@pytest.mark.parametrize("new", [1, 3, 80])
def test_graphs(new):
    """Two captured graphs of write, attention and read, replayed in turn and at the same time with changed inputs
    and lengths, give what eager calls give."""
    graphs = []
    for seed in (1, 2):
        layer, q, tables, lens, cu = decode_state(seed, lens=(170, 1000, 0, 133), new=new)
        k, v = (torch.randn(4 * new, 2, 128, device="cuda").bfloat16() for _ in range(2))
        slots = torch.full((4 * new,), -1, dtype=torch.int64, device="cuda")
        slots[:4] = torch.stack([tables[b, 0].long() * 16 + 3 for b in (0, 1, 1, 3)])
        slots[2] += 1
        out = torch.zeros_like(q)

        def run(layer=layer, k=k, v=v, slots=slots, q=q, tables=tables, lens=lens, cu=cu, out=out):
            fp4_cache.fp4_write(layer, k, v, slots)
            fp4_cache.fp4_attention(layer, q, tables, lens, cu, new, out=out)
            return fp4_cache.fp4_read(layer, slots)
        run()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            back = run()
        graphs.append((gr, run, back, layer, k, q, lens, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(6):
        for gr, run, back, layer, k, q, lens, out in graphs:
            k.normal_()
            q.normal_()
            lens.sub_(7).clamp_(min=0)
        torch.cuda.synchronize()
        for (gr, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for gr, run, back, layer, k, q, lens, out in graphs:
            got, rows = out.clone(), [x.clone() for x in back]
            out.zero_()
            want = run()
            assert torch.equal(out, got) and torch.equal(want[0], rows[0]) and torch.equal(want[1], rows[1])


@pytest.mark.parametrize("new", [1, 3, 80])
def test_streams(new):
    """Calls on several streams at once do not disturb one another, and each runs on the current stream."""
    states = [decode_state(s, lens=(3000, 170), new=new) for s in range(4)]
    want = [fp4_cache.fp4_attention(*st, new) for st in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [[] for _ in states]
    for turn in range(10):
        for i, (st, s) in enumerate(zip(states, streams)):
            with torch.cuda.stream(s):
                got[i].append(fp4_cache.fp4_attention(*st, new))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(w, x) for x in gs)


@pytest.mark.parametrize("new", [1, 3, 80])
def test_order_does_not_change_results(new):
    """The same call gives the same bits, whatever else is in the batch's other rows of the pool."""
    st = decode_state(9, lens=(5000, 177, 2000), new=new)
    a = [fp4_cache.fp4_attention(*st, new) for _ in range(5)]
    assert all(torch.equal(a[0], x) for x in a)


def test_no_wait_ran_out():
    """After all of the above: every wait between the warps of the kernels was met."""
    import ctypes
    from flexkv_b200 import _lib
    n = ctypes.c_int64(-1)
    assert _lib.load().fkv_fp4_wait_timeouts(ctypes.byref(n)) == 0 and n.value == 0
    assert _lib.load().fkv_fp4_wait_timeouts(None) == _lib.FKV_ERR_INVALID_ARG


@pytest.mark.parametrize("tokens,heads,group", [(40, 2, 4), (100, 1, 8), (300, 1, 2)])
def test_few_blocks_of_rows_over_many_keys(tokens, heads, group):
    """The keys of a few rows' blocks split over CTAs and joined, with parts that see nothing."""
    check_attention(heads, group, 128, 16, "bf16", [3000, 20, 0], [tokens, 20, 0])
    check_attention(heads, group, 64, 32, "fp16", [1500, tokens], [tokens, tokens], causal=False)


def test_more_sequences_than_lanes():
    """Blocks of rows are found among more sequences than a warp has lanes."""
    r = np.random.RandomState(3)
    new = r.randint(0, 30, 45)
    lens = new + r.randint(0, 40, 45)
    check_attention(1, 5, 64, 16, "bf16", lens.tolist(), new.tolist())


def test_a_head_over_every_cta():
    """One key head's keys over all CTAs, joined in two steps; with rows of two tiles too."""
    check_attention(1, 8, 128, 16, "bf16", [30000], [1], uniform=True)
    check_attention(1, 8, 64, 64, "fp16", [20011, 500], [2, 2])


def test_in_place():
    """out may be q itself."""
    for new in (1, 4, 100):
        layer, q, tables, lens, cu = decode_state(3, lens=(1500, 170), new=new)
        want = fp4_cache.fp4_attention(layer, q, tables, lens, cu, new)
        got = q.clone()
        fp4_cache.fp4_attention(layer, got, tables, lens, cu, new, out=got)
        assert torch.equal(got, want)


def test_repeated_sources_and_tables():
    """The same page in two sequences' tables (a shared prefix), the same slot read twice."""
    layer = torch.from_numpy(written(2, 8, 2, 16, 64, 1)).cuda()
    tables = torch.tensor([[3, 5, 1], [3, 5, 7], [3, 5, 1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([40, 40, 40], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4, 64, device="cuda").bfloat16().repeat(3, 1, 1)
    o = fp4_cache.fp4_attention(layer, q, tables, lens)
    want, _, weight, size = M.attention(layer.cpu().numpy(), f64(q), tables.cpu().numpy(), lens.cpu().numpy(),
                                        np.arange(4), 64 ** -0.5, True, 16)
    assert (np.abs(f64(o) - want) <= M.attention_bounds(weight, size, want, 64, "bf16")).all()
    slots = torch.tensor([5, 5, 100, 5], device="cuda")
    k, v = fp4_cache.fp4_read(layer, slots)
    assert torch.equal(k[0], k[1]) and torch.equal(v[0], v[3])


@pytest.mark.skipif("torch.cuda.device_count() < 2")
def test_another_device():
    """Tensors of a device that is not the current one."""
    torch.cuda.set_device(0)
    layer = torch.from_numpy(written(2, 8, 2, 16, 64, 1)).to("cuda:1")
    slots = torch.arange(40, device="cuda:1")
    k, _ = fp4_cache.fp4_read(layer, slots)
    assert torch.cuda.current_device() == 0 and np.array_equal(f64(k), M.held(layer.cpu().numpy())[0][:40])


def test_slots_past_2_to_the_28():
    """Rows in a pool whose units pass 2^24, two heads a block: each in its place, and nothing anywhere else."""
    blocks, heads, dim = 2 ** 24 + 2, 2, 16
    layer = torch.zeros(1, blocks, heads, 1, 9 * dim, dtype=torch.uint8, device="cuda")
    slots = np.array([2 ** 28 + 17, 5, 2 ** 28 - 1, 2 ** 28, blocks * 16])
    k = torch.randn(len(slots), heads, dim, device="cuda").bfloat16()
    fp4_cache.fp4_write(layer, k, None, torch.from_numpy(slots).cuda())
    held = np.unique(slots[:4] // 16)
    want = np.zeros((1, len(held), heads, 1, 9 * dim), dtype=np.uint8)
    M.write(want, [f64(k)[:4]], np.searchsorted(held, slots[:4] // 16) * 16 + slots[:4] % 16)
    there = layer[:, torch.from_numpy(held).cuda()]
    assert np.array_equal(M.held(there.cpu().numpy()), M.held(want))
    got = f64(fp4_cache.fp4_read(layer, torch.from_numpy(slots).cuda())[0])
    assert np.array_equal(got[:4], M.dequantise(*M.quantise(f64(k)[:4]))) and not got[4].any()
    nonzero = sum(int(torch.count_nonzero(x)) for x in layer[0].split(2 ** 22))
    assert nonzero == int(torch.count_nonzero(there))


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("tpb", [16, 48])
def test_positions_past_2_to_the_28(new, tpb):
    """A sequence whose pages are outside the pool but for one at the start and those behind 2^28 tokens: the same
    as one of these pages alone."""
    far = 2 ** 28 // tpb + 1
    layer = torch.from_numpy(written(2, 9, 2, tpb, 64, 3)).cuda()
    tables = torch.full((1, far + 7), -1, dtype=torch.int32, device="cuda")
    few = torch.tensor([[4, 0, 8, 3, 1, 7, 2, 6]], dtype=torch.int32, device="cuda")
    tables[0, 5], tables[0, far:] = few[0, 0], few[0, 1:]
    length = torch.tensor([far * tpb + 6 * tpb + 5], dtype=torch.int32, device="cuda")
    q = torch.randn(new, 4, 64, device="cuda").bfloat16()
    out, lse = fp4_cache.fp4_attention(layer, q, tables, length, return_lse=True)
    short = length - (far - 1) * tpb
    want, wlse, weight, size = M.attention(layer.cpu().numpy(), f64(q), few.cpu().numpy(), short.cpu().numpy(),
                                           np.array([0, new]), 0.125, True, tpb)
    assert (np.abs(f64(out) - want) <= M.attention_bounds(weight, size, want, 64, "bf16")).all()
    assert np.abs(f64(lse) - wlse).max() < 1e-4


def test_what_is_written_must_not_overlap():
    layer, slots = garbage(2, 4, 2, 16, 64), torch.arange(5, device="cuda")
    x = torch.zeros(5, 2, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (x[:1].expand(5, 2, 64), x[:, :1].expand(5, 2, 64), torch.zeros(900, dtype=x.dtype, device="cuda").as_strided((5, 2, 64), (64, 64, 1))):
        fp4_cache.fp4_write(layer, bad, bad, slots)  # to read from is fine
        with pytest.raises(RuntimeError, match="rows overlap"):
            fp4_cache.fp4_read(layer, slots, out=(x, bad))
        with pytest.raises(RuntimeError, match="rows overlap"):
            fp4_cache.fp4_attention(layer, x[:, :2], torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                                    torch.ones(1, dtype=torch.int32, device="cuda"), out=bad)
    for bad in (layer[:, :1].expand(2, 4, 2, 1, 576), layer[:1].expand(2, 4, 2, 1, 576)):
        with pytest.raises(RuntimeError, match="blocks overlap"):
            fp4_cache.fp4_write(bad, x, x, slots)
        fp4_cache.fp4_read(bad, slots)
        kv, ids = torch.zeros(2, 4, 16, 2, 64, dtype=x.dtype, device="cuda"), torch.arange(2)
        with pytest.raises(RuntimeError, match="blocks overlap"):
            fp4_cache.fp4_pack_blocks([kv], [bad], ids, ids)
        fp4_cache.fp4_unpack_blocks([bad], [kv], ids, ids)
        with pytest.raises(RuntimeError, match="blocks overlap"):
            fp4_cache.fp4_unpack_blocks([layer], [kv[:, :1].expand(2, 4, 16, 2, 64)], ids, ids)
    # sides within a block, and heads outside of tokens
    inner = torch.zeros(4, 2, 2, 1, 576, dtype=torch.uint8, device="cuda").transpose(0, 1)
    fp4_cache.fp4_write(inner, x, x, slots)
    y = torch.zeros(2, 5, 64, dtype=x.dtype, device="cuda").transpose(0, 1)
    fp4_cache.fp4_read(inner, slots, out=(y, x))


@pytest.mark.parametrize("before,new,behind", [(2, 1, 0), (0, 1, 700), (400, 3, 300), (3, 90, 500), (0, 0, 4), (5, 0, 0)])
def test_rows_of_no_sequence(before, new, behind):
    """Zeros and -inf in a new output, whatever its memory held, strided heads or not; as they were in a given one."""
    layer, _, tables, lens, cu = decode_state(4, new=new)
    n = before + new * 4 + behind
    q = torch.randn(n, 8, 128, device="cuda").bfloat16()
    given = torch.full((8, n, 128), 3.0, dtype=q.dtype, device="cuda").transpose(0, 1)
    fp4_cache.fp4_attention(layer, q, tables, lens, cu + before, max(new, 1), out=given)
    rows = torch.cat([torch.arange(before), torch.arange(n - behind, n)]).cuda()
    assert bool((given[rows] == 3.0).all())
    for _ in range(2):
        dirt = [torch.full((n, 8, 128), float("nan"), dtype=q.dtype, device="cuda"), torch.full((n, 8), 7.0, device="cuda")]
        del dirt
        out, lse = fp4_cache.fp4_attention(layer, q, tables, lens, cu + before, max(new, 1), return_lse=True)
        assert not bool(out[rows].any()) and bool(torch.isneginf(lse[rows]).all())
        assert torch.equal(out[before:n - behind], given[before:n - behind])
    none = fp4_cache.fp4_attention(layer, q, tables[:0], lens[:0], cu[:1] + before, return_lse=True)
    assert not bool(none[0].any()) and bool(torch.isneginf(none[1]).all())


@pytest.mark.parametrize("new", [1, 3, 40])
def test_forked_streams(new):
    """Write, then attention on two streams at once, with other kernels before, between and beside them, captured
    and eager: each call sees what was before it on its stream and at the joins."""
    layer, q, tables, lens, cu = decode_state(1, lens=(170, 1000, 0, 133), new=new)
    src, k = torch.empty_like(q), torch.empty(4 * new, 2, 128, dtype=q.dtype, device="cuda")
    late, at = torch.empty_like(k), torch.arange(4 * new, device="cuda") % new
    slots = torch.where(at < 16, tables[:, 0].long().repeat_interleave(new) * 16 + at, -1)
    side = torch.cuda.Stream()

    def run():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        q.zero_()
        with torch.cuda.stream(side):
            x = torch.ones(2048, 2048, device="cuda")
            late.copy_(k + (x @ x)[:1, :1].bfloat16() * 0)
        q.copy_(src)
        main.wait_stream(side)
        fp4_cache.fp4_write(layer, late, late, slots)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            outs = [fp4_cache.fp4_attention(layer, q, tables, lens, cu, new)]
        outs.append(fp4_cache.fp4_attention(layer, q, tables, lens, cu, new))
        outs.append(fp4_cache.fp4_read(layer, slots)[0])
        main.wait_stream(side)
        late.zero_()
        return outs

    for x in (src, k):
        x.normal_()
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for turn in range(4):
        for x in (src, k):
            x.normal_()
        layer.fill_(0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured]
        held = torch.where((slots >= 0)[:, None, None], torch.from_numpy(M.dequantise(*M.quantise(f64(k)))).cuda(), 0.0)
        assert torch.equal(got[2].double(), held)
        want = fp4_cache.fp4_attention(layer, src, tables, lens, cu, new)
        layer.fill_(0)
        eager = run()
        torch.cuda.synchronize()
        for x in (got, eager):
            assert torch.equal(x[0], want) and torch.equal(x[1], want) and torch.equal(x[2], got[2])


def test_outputs_that_share_memory_are_refused():
    layer, slots = garbage(2, 4, 2, 16, 64), torch.arange(5, device="cuda")
    flat = torch.zeros(6, 2, 64, dtype=torch.bfloat16, device="cuda")
    tables, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="out may be q"):
        fp4_cache.fp4_attention(layer, flat[:5], tables, lens, out=flat[1:])
    assert fp4_cache.fp4_attention(layer, flat[:5], tables, lens, out=flat[:5]) is not None
    for v in (flat[:5], flat[1:]):
        with pytest.raises(RuntimeError, match="k and v overlap"):
            fp4_cache.fp4_read(layer, slots, out=(flat[:5], v))
    # interleaved sides of one tensor do not overlap
    both = torch.zeros(5, 2, 2, 64, dtype=torch.bfloat16, device="cuda")
    fp4_cache.fp4_read(layer, slots, out=(both[:, 0], both[:, 1]))


@pytest.mark.parametrize("new", [1, 3, 80])
def test_graphs_of_one_pool(new):
    """Two graphs captured into one memory pool, so that they share workspaces, replayed in turn between eager calls."""
    states = [decode_state(s, lens=(3000, 170), new=new) for s in range(2)]
    want = [fp4_cache.fp4_attention(*st, new) for st in states]
    outs = [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    graphs = []
    for st, out in zip(states, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            fp4_cache.fp4_attention(*st, new, out=out)
        graphs.append(graph)
    for turn in range(6):
        for out in outs:
            out.zero_()
        for i in (0, 1, 1, 0):
            graphs[i].replay()
            assert torch.equal(fp4_cache.fp4_attention(*states[i], new), want[i])
        assert all(torch.equal(out, w) for out, w in zip(outs, want))

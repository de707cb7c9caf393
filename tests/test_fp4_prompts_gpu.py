"""GPU: attention over the 4-bit cache where the many-rows kernel takes whole
blocks of rows (no split of the keys): long walks over the keys, its rings
reused many times, bases that move late.  A sample of the rows is compared
with the definition in 64 bits."""
import numpy as np
import pytest
import torch

import fp4_model as M
from flexkv_b200 import _lib, fp4_cache

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def rows_of_definition(k, v, q, seen, scale):
    """q [rows, D] over k, v [keys, D] with seen [rows, keys]: out, lse, weight and size as fp4_model.attention."""
    s = np.where(seen, q @ k.T * scale, -np.inf)
    m = s.max(-1, keepdims=True)
    none = np.isneginf(m)
    p = np.exp(s - np.where(none, 0, m))
    total = p.sum(-1, keepdims=True)
    safe = np.where(none, 1, total)
    out = p @ v / safe
    weight = p @ np.abs(v) / safe + 2.0 ** -21 * (seen @ np.abs(v))
    lse = np.where(none, -np.inf, m + np.log(safe))[:, 0]
    size = (np.where(seen, np.abs(q) @ np.abs(k).T, 0)).max(-1) * abs(scale)
    return out, lse, weight, size


def rising(blocks, heads, tpb, dim, at, along, climb, seed):
    """A layer whose key at position `at[slot]` has `climb * position` along the direction `along`."""
    r = np.random.RandomState(seed)
    layer = np.zeros((2, blocks, heads, tpb // 16, 9 * dim), dtype=np.uint8)
    for side in range(2):
        x = r.randn(blocks, heads, tpb, dim)
        if side == 0:
            x += climb * at.reshape(blocks, 1, tpb, 1) * along
        layer[side] = M.unit_bytes(*M.quantise(x.reshape(blocks, heads, tpb // 16, 16, dim)))
    return layer


@pytest.mark.parametrize("climb", [0.0, 4.0])
@pytest.mark.parametrize("heads,group,dim,tpb,dtype,causal", [
    (8, 4, 128, 16, "bf16", True), (8, 4, 64, 32, "fp16", False), (8, 5, 64, 16, "bf16", True), (10, 4, 128, 64, "fp16", False),
    (12, 1, 128, 16, "fp16", True)])
def test_prompts_over_many_chunks(heads, group, dim, tpb, dtype, causal, climb):
    """Blocks of one and of two tiles over 20 to 40 chunks of 64 keys; pages outside the pool where the ring that
    marks them has wrapped; with `climb`, scores that rise to the end, so that every row's base moves on and on."""
    lens = [1400, 2500, 1301, 77, 1990, 64, 1310, 1500]
    new = [1024 // group + 3, 1300 // group, 120 // group, 77, 128 // group, 64, 256 // group, 257 // group]
    r = np.random.RandomState(dim + group)
    pages = [-(-n // tpb) for n in lens]
    blocks = sum(pages)
    order = r.permutation(blocks)
    tables = np.full((len(lens), max(pages) + 1), 2 ** 30, dtype=np.int32)
    at, first = np.zeros((blocks, tpb)), 0
    for b, p in enumerate(pages):
        tables[b, :p] = order[first:first + p]
        at[order[first:first + p]] = np.arange(p * tpb).reshape(p, tpb) / lens[b]
        first += p
    for b, pos in ((0, 10 * 64), (0, 19 * 64), (1, 9 * 64 + 48), (1, 26 * 64), (1, 33 * 64 + 16), (4, 17 * 64 + 32)):
        tables[b, pos // tpb] = -1 - b
    along = r.randn(dim)
    along *= 8 / np.linalg.norm(along)
    layer = rising(blocks, heads, tpb, dim, at, along, climb, seed=dim)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) + 2
    n = int(cu[-1]) + 5
    scale = dim ** -0.5
    # along the direction a score climbs by 3 * 8 * 8 * climb / sqrt(D): 98 powers of two for heads of 128
    q = torch.from_numpy(r.randn(n, heads * group, dim) + climb * 3 * along).to(DT[dtype])
    assert _lib.load().fkv_fp4_attention_workspace(n, heads * group, heads, dim, len(lens), max(new)) == 0, \
        "the keys are split: not what this tests"
    out = torch.full((n, heads * group, dim), 3.0, dtype=DT[dtype], device="cuda")
    args = (torch.from_numpy(layer).cuda(), q.cuda(), torch.from_numpy(tables).cuda(),
            torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.from_numpy(cu).cuda(), max(new))
    _, lse = fp4_cache.fp4_attention(*args, softmax_scale=scale, causal=causal, out=out, return_lse=True)
    fresh = fp4_cache.fp4_attention(*args, softmax_scale=scale, causal=causal)
    assert torch.equal(fresh[2:n - 5], out[2:n - 5])
    assert bool((out[:2] == 3.0).all()) and bool((out[n - 5:] == 3.0).all())
    got, glse, qs = out.double().cpu().numpy(), lse.double().cpu().numpy(), q.double().numpy()
    assert np.isfinite(got).all()
    for b, length in enumerate(lens):
        rows = new[b]
        pick = np.unique(np.clip([0, 1, 128 // group - 1, 128 // group, 256 // group - 1, 256 // group, rows // 2, rows - 2,
                                  rows - 1, *r.randint(0, rows, 4)], 0, rows - 1))
        t = tables[b, :pages[b]].astype(np.int64)
        good = (t >= 0) & (t < blocks)
        kv = M.held(layer[:, np.where(good, t, 0)])[:, :length]
        there = np.repeat(good, tpb)[:length]
        end = np.minimum(length - rows + pick + 1, length) if causal else np.full(len(pick), length)
        seen = np.repeat(there & (np.arange(length) < end[:, None]), group, 0)
        for h in range(heads):
            x = qs[cu[b] + pick, h * group:(h + 1) * group].reshape(-1, dim)
            want, wlse, weight, size = rows_of_definition(kv[0][:, h], kv[1][:, h], x, seen, scale)
            # beyond the bounds of fewer keys: a weight goes into one of four float32 sums and one of length / 16
            # products, and each move of the base rounds both once more
            more = (length / 4 * 2.0 ** -24 + length / 16 * 2.0 ** -23 + length / 64 * 2.0 ** -23) * weight
            bound = M.attention_bounds(weight, size, want, dim, dtype) + 1.01 * more
            o = got[cu[b] + pick, h * group:(h + 1) * group].reshape(-1, dim)
            off = np.abs(o - want) / bound
            assert off.max() <= 1, (b, h, off.max(), np.unravel_index(off.argmax(), off.shape))
            l = glse[cu[b] + pick, h * group:(h + 1) * group].reshape(-1)
            lbound = (dim / 16 + 8) * 2.0 ** -23 * size + 2.0 ** -14 + length / 4 * 2.0 ** -24 + 2.0 ** -22 * np.abs(wlse)
            assert (np.abs(l - wlse) <= lbound).all()


def test_prompts_repeat_exactly():
    """The same call gives the same bits where blocks are whole."""
    r = np.random.RandomState(4)
    lens, new = [1500, 900, 1700, 640], [300, 280, 310, 290]
    pages = [-(-n // 16) for n in lens]
    tables = np.zeros((4, max(pages)), dtype=np.int32)
    order = r.permutation(sum(pages))
    for b, p in enumerate(pages):
        tables[b, :p] = order[sum(pages[:b]):sum(pages[:b + 1])]
    layer = torch.randint(0, 200, (2, sum(pages), 8, 1, 9 * 128), dtype=torch.uint8, device="cuda")
    layer[..., 8 * 128:] %= 130
    q = torch.randn(sum(new), 16, 128, device="cuda").bfloat16()
    args = (layer, q, torch.from_numpy(tables).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"),
            torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda"), max(new))
    a = [fp4_cache.fp4_attention(*args) for _ in range(4)]
    assert not bool(a[0].isnan().any()) and all(torch.equal(a[0], x) for x in a)

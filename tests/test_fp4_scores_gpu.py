"""GPU: attention over the 4-bit cache where scores are far past what
differences of rounded products can tell apart.  Where not said otherwise all
sums q k are exact in float32 in any order, so that the definition in 64 bits
and the kernels see the same scores."""
import numpy as np
import pytest
import torch

import fp4_model as M
from flexkv_b200 import fp4_cache

pytestmark = pytest.mark.gpu
D, TPB = 64, 16
# new tokens, heads, group, sequences: few rows (one and two tiles), many rows with split keys, and with whole blocks
FORMS = [(1, 1, 2, 1), (4, 2, 3, 2), (20, 1, 2, 1), (40, 8, 8, 6)]


def attend(form, k, v, q, scale):
    """k, v [keys, D] for every head and sequence, q [D] for every row: out [rows, heads, D], lse, and held k, v."""
    new, heads, group, seqs = form
    keys = k.shape[0]
    pages = -(-keys // TPB)
    layer = torch.zeros(2, pages + 1, heads, 1, 9 * D, dtype=torch.uint8, device="cuda")
    slots = torch.arange(keys, device="cuda")
    rows = [x.to(torch.bfloat16).cuda()[:, None].expand(keys, heads, D) for x in (k, v)]
    fp4_cache.fp4_write(layer, *rows, slots)
    tables = torch.arange(pages, dtype=torch.int32, device="cuda").expand(seqs, pages)
    lens = torch.full((seqs,), keys, dtype=torch.int32, device="cuda")
    x = q.to(torch.bfloat16).cuda().expand(seqs * new, heads * group, D)
    out, lse = fp4_cache.fp4_attention(layer, x, tables, lens, softmax_scale=scale, causal=False, return_lse=True)
    held = [t[:, 0].double().cpu().numpy() for t in fp4_cache.fp4_read(layer, slots)]
    return out.double().cpu().numpy(), lse.double().cpu().numpy(), *held


def check(form, k, v, q, scale, difference):
    """`difference`: the largest that matters between two scores; beyond it weights vanish."""
    scale = float(np.float32(scale))
    out, lse, hk, hv = attend(form, k, v, q, scale)
    s = hk @ q.to(torch.bfloat16).double().numpy() * scale
    p = np.exp(s - s.max())
    want, wlse = p @ hv / p.sum(), s.max() + np.log(p.sum())
    bound = M.attention_bounds(p @ np.abs(hv) / p.sum() + 2.0 ** -21 * np.abs(hv).sum(0), np.array(difference), want, D, "bf16")
    assert np.isfinite(out).all() and (np.abs(out - want) <= bound).all(), np.abs(out - want).max()
    # float32's own step of the score, its product's rounding and that of the base
    assert (np.abs(lse - wlse) <= 2.0 ** -14 + 2.0 ** -21 * abs(wlse)).all(), (lse.flat[0], wlse)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [0, 4, 8, 10, 12, 16, 40, 90])
def test_huge_scores(form, sign, power):
    """One key above the others by a quarter of 64 * 2^power * 6144 and more (or, with the sign, a few lowest ones
    of a common value): all weight goes there."""
    n = 150
    k = 1024.0 * torch.tensor([1, 1.5, 2, 3, 4]).repeat(n // 5)[:, None].expand(n, D).clone()
    k[70] = 6 * 1024.0
    v = (torch.arange(n)[:, None] % 7 + torch.arange(D) % 3).float()
    check(form, k, v, torch.full((D,), sign * 2.0 ** power), 1.0, 16.0)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("exact", [False, True])
def test_near_scores_far_out(form, order, exact):
    """Scores of 1.5e7 that differ by multiples of 4.8: the softmax of the differences.

    exact: one channel makes the difference, so every product is a multiple of 32 (16 * 6, 512 * 12288), as every
    partial sum below 2^29 may be.  Else 16 channels do, each with 6: where three quarters of the channels are
    summed, 2.3e8 + 72, float32's step is 16, and at the end 32, so a difference of 96 may come out as 64: the
    bound is then the general one, by the size of the sums."""
    n = 200
    step = torch.arange(n) * 3 // n
    step = step.flip(0) if order == "falling" else torch.arange(n) * 7 % 3 if order == "mixed" else step
    k = torch.full((n, D), 12288.0)
    k[:, 48:] = torch.tensor([0.0, 6.0, 12.0])[step][:, None]
    q = torch.ones(D)
    q[:48] = 512.0
    if exact:
        k[:, 48:63] = 0
        q[63] = 16.0
    g = torch.Generator().manual_seed(1)
    check(form, k, torch.randn(n, D, generator=g), q, 0.05, 32.0 if exact else 1.6e7)


@pytest.mark.parametrize("form", FORMS)
def test_scores_below_every_other(form):
    """Equal scores of -6e31 and -6e37: the mean."""
    g = torch.Generator().manual_seed(2)
    for q in (-1e30, -1e36):
        check(form, torch.ones(100, D), torch.randn(100, D, generator=g), torch.full((D,), q), 1.0, 1.0)


@pytest.mark.parametrize("form", FORMS)
def test_scales_past_float(form):
    """A multiplier past what a float holds: keys of zeros still score nothing, the largest score takes all weight."""
    k = torch.zeros(100, D)
    k[:, :16] = -1.0
    k[30:33] = 0.0
    g = torch.Generator().manual_seed(3)
    check(form, k, torch.randn(100, D, generator=g), torch.full((D,), 1e20), 1e30, 1.0)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("where", [float("inf"), -float("inf")])
def test_infinite_queries_have_no_softmax(form, where):
    """Scores that are all infinite, of either sign: NaN as in the definition, and zeros where nothing is seen."""
    g = torch.Generator().manual_seed(5)
    q = torch.ones(D)
    q[7] = where
    out, lse, _, _ = attend(form, torch.rand(100, D, generator=g) + 1, torch.randn(100, D, generator=g), q, 0.1)
    assert np.isnan(out).all() and np.isnan(lse).all()
    new, heads, group, seqs = form
    layer = torch.zeros(2, 3, heads, 1, 9 * D, dtype=torch.uint8, device="cuda")
    x = q.bfloat16().cuda().expand(seqs * new, heads * group, D)
    for tables, lens in ((0, 0), (99, 40)):  # no keys; keys in blocks outside the pool
        out, lse = fp4_cache.fp4_attention(layer, x, torch.full((seqs, 3), tables, dtype=torch.int32, device="cuda"),
                                           torch.full((seqs,), lens, dtype=torch.int32, device="cuda"), return_lse=True)
        assert not bool(out.any()) and bool(torch.isneginf(lse).all())

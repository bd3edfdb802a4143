"""Selections of the long-cache operators where they are counted over several CTAs and at the
ends of the keys' range, against plain 64-bit restatements: every id and every moved byte."""
import math

import numpy as np
import pytest
import torch

from test_cache_ops_gpu import DT, TYPES, caches, i32, kept64, normal, ok, ptrs, rng, select64

pytestmark = pytest.mark.gpu


def bits(x):
    return x.contiguous().view(torch.int16 if x.dtype == torch.float16 else torch.int32)


def evict_and_check(ctx, g, t, in_place, n_kv, hd, lens, w, keep, recent, top):
    """One eviction of sequences of `lens` rows and weights `w`; `kept` lies between other words."""
    batch, behind = len(lens), 64
    k, v = caches(g, lens, n_kv, hd, t), caches(g, lens, n_kv, hd, t)
    k0, v0, w0 = [x.clone() for x in k], [x.clone() for x in v], [x.clone() for x in w]
    buf = torch.full((behind + batch * n_kv * keep + behind,), 77, dtype=torch.int32, device="cuda")
    kept = buf[behind:-behind].view(batch, n_kv, keep)
    kw, ko, vo, wo = {}, k, v, w
    if not in_place:
        ko = [torch.full((keep + 2, n_kv * hd), 3.0, dtype=DT[t], device="cuda") for _ in lens]
        vo = [x.clone() for x in ko]
        wo = [torch.full((n_kv, keep + 1), 3.0, device="cuda") for _ in lens]
        kw = dict(k_out_ptrs=ptrs(ko), v_out_ptrs=ptrs(vo), weight_out_ptrs=ptrs(wo), weight_out_stride=keep + 1)
    stride = w[0].shape[1]
    ctx.kv_evict(ptrs(k), ptrs(v), ptrs(w), stride, i32(lens), top, keep, recent, kept, batch, n_kv, hd,
                 f16_cache=t == "f16", **kw)
    ok(ctx)
    assert (buf[:behind] == 77).all() and (buf[-behind:] == 77).all()
    for b, n in enumerate(lens):
        for h in range(n_kv):
            rows = kept64(w0[b][h], n, keep, recent)
            m, cols = len(rows), slice(h * hd, (h + 1) * hd)
            assert kept[b, h].tolist() == rows + [-1] * (keep - m)
            for src, dst in ((k0, ko), (v0, vo)):
                assert torch.equal(bits(dst[b][:m, cols]), bits(src[b][rows, cols]))
                if in_place:
                    assert torch.equal(bits(dst[b][m:, cols]), bits(src[b][m:, cols]))
            assert torch.equal(bits(wo[b][h, :m]), bits(w0[b][h, rows]))


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("top,lens,keep,recent", [
    (40_000, [2501, 5003, 33_001, 17, 40_000], 2400, 0),  # two CTAs a selection
    (100_003, [66_667, 3, 100_003, 30_002], 30_000, 0),   # four
    (300_001, [999, 300_001, 41, 0], 900, 1),             # sixteen, the short members one warp or two
])
def test_eviction_of_short_and_long_sequences_over_clusters(gla_ctx, in_place, top, lens, keep, recent):
    """A capacity past 32,768 rows gives every sequence of the batch a cluster, the short ones
    too: most of their CTAs' warps have no key.  The last rows of each CTA's share are kept."""
    g, n_kv, hd = rng(31, top), 2, 64
    w = []
    for n in lens:
        x = torch.exp(normal(g, n_kv, top))
        older = n - recent
        for ctas in (2, 4, 16):
            per = -(-max(older, 1) // ctas)
            for end in range(per, older + per, per):
                end = min(end, older)
                x[:, max(0, end - 3):end] = 1e3 + torch.arange(3, device="cuda")[-min(3, max(end, 0)):]
        w.append(x)
    evict_and_check(gla_ctx, g, "f16", in_place, n_kv, hd, lens, w, keep, recent, top)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("in_place", [True, False])
def test_eviction_of_an_odd_batch_over_clusters(gla_ctx, t, in_place):
    """Distinct weights, every length modulo 4, nearly all rows kept."""
    g, n_kv, hd, top = rng(32), 1, 96, 33_000
    lens = [2400 + i for i in range(1, 10)] + [1283, 3071 + 2048, 32_999]
    w = [torch.rand(n_kv, top, generator=g, device="cuda") for _ in lens]
    evict_and_check(gla_ctx, g, t, in_place, n_kv, hd, lens, w, 2399, 0, top)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("in_place,top", [(True, 3000), (False, 3000), (True, 33_000)])
@pytest.mark.parametrize("older,pick,most", [
    (2501, 1, [float("inf")] * 2), (2502, 1, [3e38, float("inf"), float("inf"), 2.5e38]),
    (2503, 3, [2e38 + 1e36 * i for i in range(9)]), (2501, 2400, [float("inf")] * 9)])
def test_eviction_of_negative_beside_infinite_weights(gla_ctx, t, in_place, top, older, pick, most):
    """Weights from below zero to the largest: the keys' range is all but all of 32 bits, and
    the filling keys behind an odd number of weights are not in it."""
    g, n_kv, hd, recent = rng(33, older, top), 2, 64, 5
    lens = [older + recent, older + recent]
    w = []
    for low in (-5.0, -0.3):
        x = normal(g, n_kv, top).clamp(-0.2, 4.0)
        x[:, 3] = low
        x[:, 100:100 + 20 * len(most):20] = torch.tensor(most, device="cuda")
        w.append(x)
    evict_and_check(gla_ctx, g, t, in_place, n_kv, hd, lens, w, pick + recent, recent, top)


@pytest.mark.parametrize("scale_q,scale_b", [(1e-25, 1e-24), (1e-30, 1e-30), (1e-38, 1e-5), (1e-40, 1.0), (1.0, 1e-42)])
def test_select_orders_products_below_the_smallest_fp32_number(gla_ctx, scale_q, scale_b):
    """FP32 products that are all zero or nearly so: the order is still that of the 64-bit sums."""
    g, nh, n_kv, hd, br, nb = rng(34, int(-100 * math.log10(scale_q * scale_b))), 4, 2, 64, 16, 300
    bo = (normal(g, nb, n_kv, 2, hd).sort(dim=2)[0].double() * scale_b).float().contiguous()
    q = (normal(g, 1, nh, hd).double() * scale_q).float()
    for n_sel in (9, 200):
        ids = torch.empty(1, n_kv, n_sel, dtype=torch.int32, device="cuda")
        gla_ctx.block_select(q, ptrs([bo]), i32([nb * br]), nb * br, ids, 1, nh, n_kv, hd, br, n_sel, n_last=0)
        ok(gla_ctx)
        want, gap = select64(q[0], bo, nb * br, br, n_sel, 0, 0)
        # the inputs decide: 128 sums of 2^-53 at a magnitude below 2^9 times the scales
        assert gap > 1e-11 * scale_q * scale_b
        np.testing.assert_array_equal(ids[0].cpu().numpy(), want)


@pytest.mark.parametrize("zero", ["q", "bounds", "apart"])
def test_select_of_exact_zeros_takes_the_lowest_blocks(gla_ctx, zero):
    """A zero query, zero bounds, and queries and bounds that meet in no channel."""
    g, nh, n_kv, hd, br, nb, n_sel = rng(35), 4, 2, 128, 16, 300, 20
    bo = normal(g, nb, n_kv, 2, hd).sort(dim=2)[0].contiguous()
    q = normal(g, 1, nh, hd)
    if zero == "q":
        q[:] = 0.0
    elif zero == "bounds":
        bo[:] = 0.0
    else:
        q[:, :, ::2] = 0.0
        bo[:, :, :, 1::2] = 0.0
    ids = torch.empty(1, n_kv, n_sel, dtype=torch.int32, device="cuda")
    gla_ctx.block_select(q, ptrs([bo]), i32([nb * br]), nb * br, ids, 1, nh, n_kv, hd, br, n_sel, n_last=0)
    ok(gla_ctx)
    assert bool((ids[0].cpu() == torch.arange(n_sel)).all())

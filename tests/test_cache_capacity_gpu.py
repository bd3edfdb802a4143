"""Calls of the long-cache operators as a server makes them: a capacity instead of the longest
length, queries that share a cache and its bounds, several new rows of one cache, and a
workspace that grows while the device's memory is nearly full."""
import math

import numpy as np
import pytest
import torch

import gpullama_attn as gla
from test_cache_ops_gpu import (DT, TYPES, attend64, attention_bound, caches, i32, kept64, normal, ok, ptrs,
                                rng, rows_of, select64)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,n_kv,hd,lens,top", [
    (32, 8, 128, [8192, 1, 0, 300, 4095, 77, 5000, 2049] * 2, 131_072), (14, 2, 64, [1, 6000], 100_001),
    (8, 1, 96, [1000], 1 << 21), (16, 2, 96, [8191, 77, 130] * 5, 32_768)])
def test_decode_weights_planned_for_a_capacity(gla_ctx, t, nh, n_kv, hd, lens, top):
    g, grp, scale = rng(41, nh, top), nh // n_kv, 1 / math.sqrt(hd)
    k, v = caches(g, lens, n_kv, hd, t), caches(g, lens, n_kv, hd, t)
    q = normal(g, len(lens), nh, hd)
    # (weights of a head lie `top` apart; a sequence's array ends with its last head's rows)
    w = [torch.zeros((n_kv - 1) * top + n, device="cuda") for n in lens]
    xb = torch.full((len(lens), nh, hd), float("nan"), device="cuda")
    gla_ctx.decode_weights(q, ptrs(k), ptrs(v), i32(lens), top, xb, ptrs(w), top, len(lens), nh, n_kv, hd,
                           f16_cache=t == "f16")
    ok(gla_ctx)
    for b, n in enumerate(lens):
        kk, vv = rows_of(k[b], n, n_kv, hd), rows_of(v[b], n, n_kv, hd)
        for h in range(n_kv):
            qh = q[b, h * grp:(h + 1) * grp]
            want, p = attend64(qh, kk[:, h], vv[:, h], scale)
            tol, rel = attention_bound(qh, kk[:, h], vv[:, h], scale)
            assert float((xb[b, h * grp:(h + 1) * grp].double() - want).abs().max()) <= tol
            got = w[b][h * top:h * top + n].double()
            # a weight within rel of p, added to zero with half a step: (1 + rel) 2^-24 p
            assert bool(((got - p).abs() <= rel * p + 2 * 2.0 ** -24 * p + 1e-37).all())
            assert h == n_kv - 1 or (w[b][h * top + n:(h + 1) * top] == 0).all()


@pytest.mark.parametrize("t", TYPES)
def test_the_other_operators_planned_for_a_capacity(gla_ctx, t):
    """Bounds, selection and eviction: the same with a capacity as with the longest length."""
    g, nh, n_kv, hd, br, cap = rng(42), 8, 2, 64, 16, 200_000
    f16 = t == "f16"
    lens = [3001, 1, 777, 0, 2050]
    top, batch = max(lens), len(lens)
    k, v = caches(g, lens, n_kv, hd, t), caches(g, lens, n_kv, hd, t)
    q = normal(g, batch, nh, hd)
    nb = -(-top // br)
    bs = [[torch.full((nb, n_kv, 2, hd), 7.0, dtype=DT[t], device="cuda") for _ in lens] for _ in range(2)]
    ids = [torch.full((batch, n_kv, 40), 9, dtype=torch.int32, device="cuda") for _ in range(2)]
    for i, m in enumerate((top, cap)):
        gla_ctx.block_bounds(ptrs(k), i32(lens), m, ptrs(bs[i]), batch, n_kv, hd, br, f16_cache=f16)
        gla_ctx.block_select(q, ptrs(bs[i]), i32(lens), m, ids[i], batch, nh, n_kv, hd, br, 40, n_first=1,
                             n_last=2, f16_cache=f16)
    ok(gla_ctx)
    assert all(torch.equal(a, b) for a, b in zip(*bs)) and torch.equal(*ids)
    w = [torch.rand((n_kv - 1) * cap + n + 1, generator=g, device="cuda") for n in lens]
    keep, recent = 600, 7
    out = [torch.full((batch, n_kv, keep), 9, dtype=torch.int32, device="cuda") for _ in range(2)]
    moved = []
    for i, m in enumerate((top, cap)):
        ks, vs, ws = [x.clone() for x in k], [x.clone() for x in v], [x.clone() for x in w]
        gla_ctx.kv_evict(ptrs(ks), ptrs(vs), ptrs(ws), cap, i32(lens), m, keep, recent, out[i], batch, n_kv, hd,
                         f16_cache=f16)
        ok(gla_ctx)
        moved.append([x.nan_to_num(nan=77.0) for x in ks + vs + ws])
    assert torch.equal(*out) and all(torch.equal(a, b) for a, b in zip(*moved))
    for b, n in enumerate(lens):
        for h in range(n_kv):
            rows = kept64(w[b][h * cap:h * cap + n], n, keep, recent)
            assert out[0][b, h].tolist() == rows + [-1] * (keep - len(rows))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,n_kv,hd,br,n,queries,n_sel", [
    (32, 8, 128, 64, 9001, 40, 12), (8, 2, 64, 16, 3000, 150, 9), (7, 1, 96, 32, 20_000, 3, 100)])
def test_select_for_queries_that_share_bounds(gla_ctx, t, nh, n_kv, hd, br, n, queries, n_sel):
    """A prompt chunk: every query over the same bounds, with its own length and blocks.  (The
    last block's bounds hold all of its rows: they bound those of any of its first rows too.)"""
    g = rng(43, n, queries)
    nb = -(-n // br)
    bo = normal(g, nb, n_kv, 2, hd).sort(dim=2)[0].to(DT[t]).contiguous()
    lens = [n - queries + 1 + i for i in range(queries)]
    q = normal(g, queries, nh, hd)
    ids = torch.full((queries, n_kv, n_sel), 99, dtype=torch.int32, device="cuda")
    gla_ctx.block_select(q, ptrs([bo] * queries), i32(lens), n, ids, queries, nh, n_kv, hd, br, n_sel,
                         n_first=1, n_last=2, f16_cache=t == "f16")
    ok(gla_ctx)
    for i, m in enumerate(lens):
        want, gap = select64(q[i], bo, m, br, n_sel, 1, 2)
        assert gap > 1e-11  # the inputs decide: 256 sums of 2^-53 at a magnitude below 2^9
        np.testing.assert_array_equal(ids[i].cpu().numpy(), want)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("style", [gla.ROPE_INTERLEAVED, gla.ROPE_NEOX])
def test_append_of_several_rows_of_one_cache(gla_ctx, t, style):
    """A turn's rows behind an evicted cache, rows apart from positions: as one row a call.  With
    bounds, rows of different blocks."""
    g, nh, n_kv, hd, cap, chunk, first, pos0, theta = rng(44), 12, 4, 96, 120, 70, 33, 9000, 5e5
    f16 = t == "f16"
    q, k, v = normal(g, chunk, nh, hd), normal(g, chunk, n_kv, hd), normal(g, chunk, n_kv, hd)
    kc = [normal(g, cap, n_kv * hd).to(DT[t])]
    vc = [normal(g, cap, n_kv * hd).to(DT[t])]
    k1, v1 = [kc[0].clone()], [vc[0].clone()]
    rows, pos = i32(list(range(first, first + chunk))), i32(list(range(pos0, pos0 + chunk)))
    q_all, q_one = torch.empty_like(q), torch.empty_like(q)
    gla_ctx.rope_append_batched(q, k, v, q_all, ptrs(kc * chunk), ptrs(vc * chunk), pos, chunk, nh, n_kv, hd, cap,
                                theta, style=style, rows=rows, f16_cache=f16)
    for i in range(chunk):
        at = slice(i, i + 1)
        gla_ctx.rope_append_batched(q[at], k[at], v[at], q_one[at], ptrs(k1), ptrs(v1), pos[at], 1, nh, n_kv, hd, cap,
                                    theta, style=style, rows=rows[at], f16_cache=f16)
    ok(gla_ctx)
    assert torch.equal(q_all, q_one) and torch.equal(kc[0], k1[0]) and torch.equal(vc[0], v1[0])
    qr, kr = q[chunk - 1].clone(), k[chunk - 1].clone()
    full = torch.zeros(pos0 + chunk, n_kv * hd, device="cuda")
    gla_ctx.rope_append(qr, kr, v[chunk - 1], full, full.clone(), nh, n_kv, hd, pos[chunk - 1:], theta, style)
    assert torch.equal(q_all[-1], qr) and torch.equal(kc[0][first + chunk - 1], full[-1].to(DT[t]))
    # one row of every other block, the bounds of all of them at once
    br, spread = 16, i32([0, 35, 64, 111])
    bo = torch.zeros(-(-cap // br), n_kv, 2, hd, dtype=DT[t], device="cuda")
    gla_ctx.block_bounds(ptrs(kc), i32([112]), cap, ptrs([bo]), 1, n_kv, hd, br, f16_cache=f16)
    old = bo.clone()
    gla_ctx.rope_append_batched(q[:4], k[:4], v[:4], q_all[:4], ptrs(kc * 4), ptrs(vc * 4), pos[:4], 4, nh, n_kv, hd,
                                cap, theta, style=style, rows=spread, bounds_ptrs=ptrs([bo] * 4), block_rows=br,
                                f16_cache=f16)
    ok(gla_ctx)
    for r in spread.tolist():
        new, was = kc[0][r].view(n_kv, hd), old[r // br]
        lo = new if r % br == 0 else torch.minimum(was[:, 0], new)
        hi = new if r % br == 0 else torch.maximum(was[:, 1], new)
        assert torch.equal(bo[r // br, :, 0], lo) and torch.equal(bo[r // br, :, 1], hi)
        old[r // br] = bo[r // br]
    assert torch.equal(bo, old)  # the other blocks: as they were


def test_the_workspace_grows_in_a_nearly_full_device():
    """Where twice the last size does not fit, the call's own size does; where that does not fit
    either, the call is refused and the context goes on."""
    g, nh, n_kv, hd, n = rng(45), 8, 1, 64, 100
    k, v = caches(g, [n], n_kv, hd, "f16"), caches(g, [n], n_kv, hd, "f16")
    kp, vp, np_ = ptrs(k), ptrs(v), i32([n])
    q, xb = normal(g, 1, nh, hd), torch.empty(1, nh, hd, device="cuda")
    w = torch.zeros(n_kv, n, device="cuda")
    wp = ptrs([w])
    rows = 1 << 25  # times 8 heads in FP32: 1 GiB of scores
    want, p = attend64(q[0], k[0][:n, :hd], v[0][:n, :hd], hd ** -0.5)
    tol, rel = attention_bound(q[0], k[0][:n, :hd], v[0][:n, :hd], hd ** -0.5)
    ctx = gla.Context(0, torch.cuda.current_stream().cuda_stream)

    def call(top):
        xb.fill_(float("nan"))
        w.zero_()
        ctx.decode_weights(q, kp, vp, np_, top, xb, wp, top, 1, nh, n_kv, hd, f16_cache=True)
        assert ctx.device_status() == 0
        assert float((xb[0].double() - want).abs().max()) <= tol
        assert bool(((w[0].double() - p).abs() <= rel * p + 2 * 2.0 ** -24 * p + 1e-37).all())

    try:
        torch.cuda.empty_cache()
        free = torch.cuda.mem_get_info()[0]
        if free < 4 << 30:
            pytest.skip("not enough device memory")
        fill = torch.empty(free - (11 << 28), dtype=torch.uint8, device="cuda")  # 2.75 GiB are left
        call(rows)
        assert 5 << 28 < torch.cuda.mem_get_info()[0] < 2 << 30  # twice the size does not fit
        call(rows + (1 << 20))
        with pytest.raises(gla.GlaError) as e:
            call(4 * rows)
        assert e.value.status == -8
        call(rows + (1 << 20))
        call(n)
    finally:
        fill = None
        ctx.close()
        torch.cuda.empty_cache()


def test_a_workspace_past_64_bits_is_refused(gla_ctx):
    """2^33 heads of 2^31 scores: the count itself would wrap to nothing.  Refused before any launch."""
    p, n = torch.zeros(4, dtype=torch.int64, device="cuda"), i32([0])
    x = torch.zeros(512, device="cuda")
    with pytest.raises(gla.GlaError) as e:
        gla_ctx.decode_weights(x, p, p, n, (1 << 31) - 1, x, p, (1 << 31) - 1, 1 << 30, 8, 1, 64)
    assert e.value.status == -8
    ok(gla_ctx)

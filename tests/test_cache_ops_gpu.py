"""Long-cache operators through the C ABI: block bounds, batched RoPE + append,
block selection, attention over listed blocks, attention that adds up its
weights, and eviction, against plain 64-bit restatements.

Integer results (block ids, kept rows) and moved or compared values (bounds,
kept rows of K, V and weights) are exact.  Attention tolerances are bounds on
the rounding errors, computed from the inputs (``attention_bound``).
"""
import math

import numpy as np
import pytest
import torch

import gpullama_attn as gla

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "f32": torch.float32}
TYPES = ["f16", "f32"]
#: (n_heads, n_kv_heads, head_dim): groups of 1, 2, 3, 4, 7 and 8, every head size
HEADS = [(8, 8, 128), (4, 2, 64), (12, 4, 96), (32, 8, 128), (14, 2, 64), (8, 1, 96), (16, 2, 128)]


def rng(*key):
    g = torch.Generator(device="cuda")
    g.manual_seed(sum(x * 7919 ** i for i, x in enumerate(key)) % (1 << 31))
    return g


def normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def ptrs(tensors):
    return torch.tensor([t.data_ptr() for t in tensors], dtype=torch.int64, device="cuda")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def caches(g, lens, n_kv, hd, t, pad_rows=3, pad_cols=0):
    """One cache tensor a sequence, [rows + pad][kv_stride]; what is behind the rows and
    beside the heads is NaN, so that reading it shows."""
    out = []
    for n in lens:
        c = torch.full((n + pad_rows, n_kv * hd + pad_cols), float("nan"), device="cuda")
        c[:n, : n_kv * hd] = normal(g, n, n_kv * hd)
        out.append(c.to(DT[t]))
    return out


def rows_of(c, n, n_kv, hd):
    return c[:n, : n_kv * hd].view(n, n_kv, hd)


def ok(ctx):
    assert ctx.device_status() == 0


# ------------------------------------------------------------------------- bounds
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n_kv,hd,br,lens,pad", [
    (8, 128, 64, [1, 64, 65, 1000], 0), (2, 64, 16, [17, 0, 16, 333], 16), (1, 96, 128, [127], 0),
    (16, 96, 32, [31, 4097], 8), (3, 64, 16, [5], 0)])
def test_bounds_are_the_minima_and_maxima(gla_ctx, t, n_kv, hd, br, lens, pad):
    g = rng(1, n_kv, hd, br)
    ks = caches(g, lens, n_kv, hd, t, pad_cols=pad)
    top = max(lens)
    nb = -(-top // br) + 1
    bs = [torch.full((nb, n_kv, 2, hd), 7.0, dtype=DT[t], device="cuda") for _ in lens]
    gla_ctx.block_bounds(ptrs(ks), i32(lens), top, ptrs(bs), len(lens), n_kv, hd, br,
                         kv_stride=n_kv * hd + pad, f16_cache=t == "f16")
    ok(gla_ctx)
    for k, b, n in zip(ks, bs, lens):
        x = rows_of(k, n, n_kv, hd)
        for j in range(nb):
            part = x[j * br:(j + 1) * br]
            if part.shape[0]:
                assert torch.equal(b[j, :, 0], part.amin(0)) and torch.equal(b[j, :, 1], part.amax(0))
            else:
                assert (b[j] == 7.0).all()  # blocks past the last row: as they were


@pytest.mark.parametrize("t", TYPES)
def test_bounds_from_a_start_leave_earlier_blocks(gla_ctx, t):
    n_kv, hd, br, n = 4, 64, 32, 200
    k = caches(rng(2), [n, n], n_kv, hd, t)
    bs = [torch.full((7, n_kv, 2, hd), 7.0, dtype=DT[t], device="cuda") for _ in k]
    gla_ctx.block_bounds(ptrs(k), i32([n, n]), n, ptrs(bs), 2, n_kv, hd, br, start_pos=i32([97, 0]),
                         f16_cache=t == "f16")
    ok(gla_ctx)
    assert (bs[0][:3] == 7.0).all()
    x = rows_of(k[0], n, n_kv, hd)
    assert torch.equal(bs[0][3, :, 0], x[96:128].amin(0))
    assert torch.equal(bs[0][6, :, 1], x[192:200].amax(0))
    assert torch.equal(bs[1][0, :, 1], rows_of(k[1], n, n_kv, hd)[:32].amax(0))


# ------------------------------------------------------------------------- append
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("style", [gla.ROPE_INTERLEAVED, gla.ROPE_NEOX])
@pytest.mark.parametrize("nh,n_kv,hd", [(8, 2, 64), (12, 4, 96), (28, 4, 128), (5, 5, 128)])
def test_append_equals_the_single_sequence_rope(gla_ctx, t, style, nh, n_kv, hd):
    """q and the cache rows equal gla_rope_append_f32's bits (FP16: rounded to nearest)."""
    g, batch, cap, theta = rng(3, nh, hd), 5, 40, 500000.0
    q, k, v = normal(g, batch, nh, hd), normal(g, batch, n_kv, hd), normal(g, batch, n_kv, hd)
    pos, rows = i32([0, 7, 39, 4095, 131071]), i32([0, 7, 16, 39, 3])
    kc = [normal(g, cap, n_kv * hd + 8).to(DT[t]) for _ in range(batch)]
    vc = [normal(g, cap, n_kv * hd + 8).to(DT[t]) for _ in range(batch)]
    k0, v0 = [x.clone() for x in kc], [x.clone() for x in vc]
    q_out, k_in = torch.empty_like(q), k.clone()
    gla_ctx.rope_append_batched(q, k, v, q_out, ptrs(kc), ptrs(vc), pos, batch, nh, n_kv, hd, cap,
                                theta, style=style, rows=rows, kv_stride=n_kv * hd + 8,
                                f16_cache=t == "f16")
    ok(gla_ctx)
    assert torch.equal(k, k_in)
    for b in range(batch):
        qr, kr = q[b].clone(), k[b].clone()
        p = int(pos[b])
        full_k = torch.zeros(p + 1, n_kv * hd, device="cuda")
        full_v = torch.zeros(p + 1, n_kv * hd, device="cuda")
        gla_ctx.rope_append(qr, kr, v[b], full_k, full_v, nh, n_kv, hd, pos[b:b + 1], theta, style)
        assert torch.equal(q_out[b], qr)
        r = int(rows[b])
        k0[b][r, : n_kv * hd] = full_k[p].to(DT[t])
        v0[b][r, : n_kv * hd] = v[b].flatten().to(DT[t])
        assert torch.equal(kc[b], k0[b]) and torch.equal(vc[b], v0[b])
    # rows default to the positions, and q may be rotated in place
    q2, pos2 = q.clone(), i32([0, 1, 2, 3, 4])
    gla_ctx.rope_append_batched(q2, k, v, q2, ptrs(kc), ptrs(vc), pos2, batch, nh, n_kv, hd, cap,
                                theta, style=style, kv_stride=n_kv * hd + 8, f16_cache=t == "f16")
    q3 = torch.empty_like(q)
    gla_ctx.rope_append_batched(q, k, v, q3, ptrs(kc), ptrs(vc), pos2, batch, nh, n_kv, hd, cap,
                                theta, style=style, rows=pos2, kv_stride=n_kv * hd + 8,
                                f16_cache=t == "f16")
    assert torch.equal(q2, q3)
    for b in range(batch):
        assert torch.equal(vc[b][b, : n_kv * hd], v[b].flatten().to(DT[t]))


@pytest.mark.parametrize("t", TYPES)
def test_append_keeps_the_bounds_of_the_cache(gla_ctx, t):
    """Appending row after row gives the bounds that gla_block_bounds_* computes."""
    g, batch, nh, n_kv, hd, br, cap = rng(4), 3, 8, 2, 64, 16, 50
    kc = [torch.full((cap, n_kv * hd), float("nan"), device="cuda").to(DT[t]) for _ in range(batch)]
    vc = [x.clone() for x in kc]
    nb = -(-cap // br)
    bs = [torch.full((nb, n_kv, 2, hd), float("nan"), dtype=DT[t], device="cuda") for _ in kc]
    kp, vp, bp = ptrs(kc), ptrs(vc), ptrs(bs)
    q = normal(g, batch, nh, hd)
    for r in range(37):
        gla_ctx.rope_append_batched(q, normal(g, batch, n_kv, hd), normal(g, batch, n_kv, hd), q, kp,
                                    vp, i32([r, r + 100, r + 9]), batch, nh, n_kv, hd, cap, 1e4,
                                    rows=i32([r, r, r]), bounds_ptrs=bp, block_rows=br,
                                    f16_cache=t == "f16")
    want = [torch.full_like(b, float("nan")) for b in bs]
    gla_ctx.block_bounds(kp, i32([37] * batch), cap, ptrs(want), batch, n_kv, hd, br,
                         f16_cache=t == "f16")
    ok(gla_ctx)
    for b, w in zip(bs, want):
        assert torch.equal(b[:3], w[:3]) and b[3].isnan().all() and w[3].isnan().all()


def test_append_outside_the_cache_writes_nothing(gla_ctx):
    g, nh, n_kv, hd, cap = rng(5), 8, 2, 64, 16
    kc = [normal(g, cap, n_kv * hd) for _ in range(4)]
    keep = [x.clone() for x in kc]
    q, k = normal(g, 4, nh, hd), normal(g, 4, n_kv, hd)
    out = torch.full_like(q, 5.0)
    gla_ctx.rope_append_batched(q, k, k, out, ptrs(kc), ptrs(kc), i32([3, 3, -1, 3]), 4, nh, n_kv,
                                hd, cap, 1e4, rows=i32([16, -1, 2, 15]))
    assert gla_ctx.device_status() == -1 and gla_ctx.device_status() == 0
    for b in range(3):
        assert torch.equal(kc[b], keep[b]) and (out[b] == 5.0).all()
    assert torch.equal(kc[3][:15], keep[3][:15]) and torch.equal(kc[3][15], k[3].flatten())


# ------------------------------------------------------------------------- select
def select64(q, bounds, n, br, n_sel, first, last):
    """Ids of one sequence, [n_kv][n_sel], and the smallest gap next to a border."""
    n_kv, hd = bounds.shape[1], bounds.shape[3]
    nb = -(-n // br)
    qq = q.double().view(n_kv, -1, 1, hd)
    bo = bounds[:nb].double()
    s = torch.maximum(qq * bo[:, :, 0].transpose(0, 1)[:, None],
                      qq * bo[:, :, 1].transpose(0, 1)[:, None]).sum(-1)
    s = torch.where(s.isnan(), -math.inf, s).amax(1).cpu().numpy()
    ids = np.full((n_kv, n_sel), -1, np.int32)
    gap = math.inf
    for g in range(n_kv):
        must = [j for j in range(nb) if j < first or j >= nb - last]
        rest = sorted(set(range(nb)) - set(must), key=lambda j: (-s[g, j], j))
        m = n_sel - len(must)
        if nb > n_sel and 0 < m < len(rest):
            d = s[g, rest[m - 1]] - s[g, rest[m]]
            gap = min(gap, d if d else math.inf)
        got = sorted((must + rest)[:n_sel])
        ids[g, : len(got)] = got
    return ids, gap


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,n_kv,hd", HEADS)
@pytest.mark.parametrize("br,lens,n_sel,first,last", [
    (16, [1, 0, 700, 16, 1601], 7, 1, 2), (64, [9000, 300], 20, 0, 0), (32, [640], 1, 0, 1),
    (16, [30000], 300, 2, 1)])
def test_select_equals_the_64_bit_order(gla_ctx, t, nh, n_kv, hd, br, lens, n_sel, first, last):
    g = rng(6, nh, hd, br)
    top = max(lens)
    nb = -(-top // br)
    q = normal(g, len(lens), nh, hd)
    bs = []
    for n in lens:
        x = normal(g, nb, n_kv, 2, hd).sort(dim=2)[0].to(DT[t])
        x[-(-n // br):] = float("nan")  # blocks that the sequence does not have
        bs.append(x)
    ids = torch.full((len(lens), n_kv, n_sel), 99, dtype=torch.int32, device="cuda")
    gla_ctx.block_select(q, ptrs(bs), i32(lens), top, ids, len(lens), nh, n_kv, hd, br, n_sel,
                         n_first=first, n_last=last, f16_cache=t == "f16")
    ok(gla_ctx)
    for b, n in enumerate(lens):
        want, gap = select64(q[b], bs[b], n, br, n_sel, first, last)
        assert gap > 1e-11  # the inputs decide: 256 sums of 2^-53 at a magnitude below 2^9
        np.testing.assert_array_equal(ids[b].cpu().numpy(), want)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,n_kv,hd", [(8, 2, 64), (7, 1, 128), (6, 3, 96)])
def test_select_ties_go_to_the_lowest_block(gla_ctx, t, nh, n_kv, hd):
    """Small whole numbers: every sum is exact, and many blocks tie.  All-equal scores,
    an infinite bound and a NaN are among them."""
    g, br, nb = rng(7, nh), 16, 2500
    q = torch.randint(-1, 2, (3, nh, hd), generator=g, device="cuda").float()
    q[1] = 0.0
    b0 = torch.randint(0, 2, (nb, n_kv, 1, hd), generator=g, device="cuda").float()
    bs = [torch.cat([b0 - 1, b0], 2).to(DT[t]).contiguous() for _ in range(3)]
    bs[1][:] = 0
    q[2] = 1.0
    bs[2][100, :, 1, 5] = float("inf")
    bs[2][101, :, 0, 5] = bs[2][101, :, 1, 5] = float("nan")
    for n_sel in (3, 40, 2499):
        ids = torch.empty(3, n_kv, n_sel, dtype=torch.int32, device="cuda")
        gla_ctx.block_select(q, ptrs(bs), i32([nb * br] * 3), nb * br, ids, 3, nh, n_kv, hd, br,
                             n_sel, n_first=0, n_last=0, f16_cache=t == "f16")
        ok(gla_ctx)
        for b in range(2):
            np.testing.assert_array_equal(ids[b].cpu().numpy(),
                                          select64(q[b], bs[b], nb * br, br, n_sel, 0, 0)[0])
        assert (ids[1].cpu().numpy() == np.arange(n_sel)).all()
        assert (ids[2] == 100).any(-1).all() and not (ids[2] == 101).any()


# ------------------------------------------------------------------------- attention
def attend64(q, k, v, scale):
    """Outputs [heads][hd], weights summed over the heads [rows], in 64 bits."""
    if k.shape[0] == 0:
        return torch.zeros_like(q, dtype=torch.float64), torch.zeros(0, dtype=torch.float64, device="cuda")
    s = (q.double() @ k.double().T) * scale
    p = torch.softmax(s, dim=1)
    return p @ v.double(), p.sum(0)


def attention_bound(q, k, v, scale):
    """(absolute bound of an output's error, relative bound of a weight's).

    A score differs by at most D (natural units): each product of the FP32 sum is
    within (hd + 2) 2^-23 of the sum of |q k| (one rounding a step, twice the half step
    for a matrix instruction that truncates), the FP16 path's split of q adds 2^-22 |q|
    and 2^-25 of the largest |q| for a low half below FP16's range; scaling and
    the subtraction of the maximum (values below |s| log2 e) and the exponential (2^-21) follow.  A weight is then within 2 D (itself and the sum) and
    the sums' n roundings of 2^-24 each; p's split adds 2^-22.
    """
    n, hd = k.shape
    if n == 0:
        return 0.0, 0.0
    qa, ka = q.double().abs(), k.double().abs()
    mag = float((qa @ ka.T).max())
    low = float((qa.amax(1)[:, None] * ka.sum(1)[None]).max())
    top = abs(scale) * mag
    d = abs(scale) * (((hd + 2) * 2.0 ** -23 + 2.0 ** -22) * mag + 2.0 ** -25 * low)
    d += (top * 1.4427 + 16) * 2.0 ** -23 + 2.0 ** -21
    rel = 2 * d + (n + 64) * 2.0 ** -24 + 2.0 ** -21
    return rel * float(v.double().abs().max()), rel


def random_ids(g, lens, n_kv, br, n_sel):
    out = torch.full((len(lens), n_kv, n_sel), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        nb = -(-n // br)
        m = min(nb, n_sel)
        for h in range(n_kv):
            if m:
                pick = torch.randperm(nb, generator=g, device="cuda")[:m].sort()[0]
                pick[-1] = nb - 1  # the block that the rows end in
                out[b, h, :m] = pick.unique()[:m] if pick.unique().numel() == m else torch.arange(
                    nb - m, nb, device="cuda")
    return out


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,n_kv,hd", HEADS)
@pytest.mark.parametrize("br,lens,n_sel", [(16, [1, 0, 333, 16, 47], 9), (64, [5000, 129], 24),
                                           (128, [700], 3), (32, [20000], 200),
                                           (128, [0, 20000, 5], 150), (128, [19300], 140)])
def test_decode_blocks_is_attention_over_the_listed_rows(gla_ctx, t, nh, n_kv, hd, br, lens, n_sel):
    g, pad = rng(8, nh, hd, br), 8
    k, v = caches(g, lens, n_kv, hd, t, pad_cols=pad), caches(g, lens, n_kv, hd, t, pad_cols=pad)
    q = normal(g, len(lens), nh, hd) * 1.5
    ids = random_ids(g, lens, n_kv, br, n_sel)
    # ids that name no rows: negative, past the last block, far past 32 bits of rows
    if n_sel >= 9:
        ids[:, :, -1], ids[:, :, -2] = 1 << 30, -5
        ids[-1, :, -3] = -(-lens[-1] // br)
    xb = torch.full((len(lens), nh, hd), float("nan"), device="cuda")
    gla_ctx.decode_blocks(q, ptrs(k), ptrs(v), i32(lens), ids, n_sel, xb, len(lens), nh, n_kv, hd,
                          br, kv_stride=n_kv * hd + pad, f16_cache=t == "f16")
    ok(gla_ctx)
    again = torch.empty_like(xb)
    gla_ctx.decode_blocks(q, ptrs(k), ptrs(v), i32(lens), ids, n_sel, again, len(lens), nh, n_kv, hd,
                          br, kv_stride=n_kv * hd + pad, f16_cache=t == "f16")
    assert torch.equal(xb, again)
    grp, scale = nh // n_kv, 1 / math.sqrt(hd)
    for b, n in enumerate(lens):
        kk, vv = rows_of(k[b], n, n_kv, hd), rows_of(v[b], n, n_kv, hd)
        for h in range(n_kv):
            rows = [r for j in ids[b, h].tolist() if j >= 0 for r in range(j * br, min(n, (j + 1) * br))]
            at = torch.tensor(rows, dtype=torch.int64, device="cuda")
            qh = q[b, h * grp:(h + 1) * grp]
            want, _ = attend64(qh, kk[at, h], vv[at, h], scale)
            got = xb[b, h * grp:(h + 1) * grp]
            if not rows:
                assert (got == 0).all()
                continue
            tol, _ = attention_bound(qh, kk[at, h], vv[at, h], scale)
            assert float((got.double() - want).abs().max()) <= tol


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch,n_sel", [(1, 257), (40, 100)])
def test_decode_blocks_over_lists_that_are_mostly_empty(gla_ctx, t, batch, n_sel):
    """Named blocks anywhere in a long list, its other slots naming no rows."""
    g, nh, n_kv, hd, br = rng(27, batch), 8, 4, 64, 64
    lens = [1 + 173 * i % 700 for i in range(batch)]
    k, v = caches(g, lens, n_kv, hd, t), caches(g, lens, n_kv, hd, t)
    q = normal(g, batch, nh, hd)
    ids = torch.full((batch, n_kv, n_sel), -1, dtype=torch.int32, device="cuda")
    ids[:, :, 33::5] = 11  # no sequence has a block 11
    at = [[], [0], [n_sel - 1], [1, n_sel - 33, n_sel - 32]]
    for h in range(n_kv):
        for s in at[h]:
            ids[:, h, s] = s % 3
    xb = torch.full((batch, nh, hd), float("nan"), device="cuda")
    gla_ctx.decode_blocks(q, ptrs(k), ptrs(v), i32(lens), ids, n_sel, xb, batch, nh, n_kv, hd, br,
                          f16_cache=t == "f16")
    ok(gla_ctx)
    scale = 1 / math.sqrt(hd)
    for b, n in enumerate(lens):
        kk, vv = rows_of(k[b], n, n_kv, hd), rows_of(v[b], n, n_kv, hd)
        for h in range(n_kv):
            rows = [r for j in ids[b, h].tolist() if j >= 0 for r in range(j * br, min(n, (j + 1) * br))]
            got = xb[b, 2 * h:2 * h + 2]
            if not rows:
                assert (got == 0).all()
                continue
            x = torch.tensor(rows, dtype=torch.int64, device="cuda")
            want, _ = attend64(q[b, 2 * h:2 * h + 2], kk[x, h], vv[x, h], scale)
            tol, _ = attention_bound(q[b, 2 * h:2 * h + 2], kk[x, h], vv[x, h], scale)
            assert float((got.double() - want).abs().max()) <= tol


@pytest.mark.parametrize("t", TYPES)
def test_decode_blocks_listed_twice_and_shared_caches(gla_ctx, t):
    """A block listed twice counts twice; queries of one chunk share a cache, each with
    its own length and blocks."""
    g, nh, n_kv, hd, br, n = rng(9), 8, 2, 64, 16, 100
    k, v = caches(g, [n], n_kv, hd, t), caches(g, [n], n_kv, hd, t)
    lens = [97, 98, 99, 100]
    q = normal(g, 4, nh, hd)
    ids = i32([[[0, 3, 3, 6], [1, 2, -1, 5]]] * 4).contiguous()
    xb = torch.empty(4, nh, hd, device="cuda")
    gla_ctx.decode_blocks(q, ptrs(k * 4), ptrs(v * 4), i32(lens), ids, 4, xb, 4, nh, n_kv, hd, br,
                          scale=-0.3, f16_cache=t == "f16")
    ok(gla_ctx)
    for b, m in enumerate(lens):
        kk, vv = rows_of(k[0], n, n_kv, hd), rows_of(v[0], n, n_kv, hd)
        for h in range(n_kv):
            rows = [r for j in ids[b, h].tolist() if j >= 0 for r in range(j * br, min(m, (j + 1) * br))]
            qh = q[b, h * 4:(h + 1) * 4]
            want, _ = attend64(qh, kk[rows, h], vv[rows, h], -0.3)
            tol, _ = attention_bound(qh, kk[rows, h], vv[rows, h], -0.3)
            assert float((xb[b, h * 4:(h + 1) * 4].double() - want).abs().max()) <= tol


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,n_kv,hd", HEADS)
@pytest.mark.parametrize("lens", [[1, 0, 15, 16, 17, 300], [4000, 129], [30000], [9001, 0, 1, 513]])
def test_decode_weights_adds_the_softmax(gla_ctx, t, nh, n_kv, hd, lens):
    g, pad, top = rng(10, nh, hd, len(lens)), 8, max(lens)
    k, v = caches(g, lens, n_kv, hd, t, pad_cols=pad), caches(g, lens, n_kv, hd, t, pad_cols=pad)
    q = normal(g, len(lens), nh, hd) * 1.5
    w0 = [torch.rand(n_kv, top + 5, generator=g, device="cuda") for _ in lens]
    w = [x.clone() for x in w0]
    xb = torch.full((len(lens), nh, hd), float("nan"), device="cuda")
    for _ in range(2):
        gla_ctx.decode_weights(q, ptrs(k), ptrs(v), i32(lens), top, xb, ptrs(w), top + 5, len(lens),
                               nh, n_kv, hd, kv_stride=n_kv * hd + pad, f16_cache=t == "f16")
    ok(gla_ctx)
    grp, scale = nh // n_kv, 1 / math.sqrt(hd)
    for b, n in enumerate(lens):
        kk, vv = rows_of(k[b], n, n_kv, hd), rows_of(v[b], n, n_kv, hd)
        for h in range(n_kv):
            qh = q[b, h * grp:(h + 1) * grp]
            want, p = attend64(qh, kk[:, h], vv[:, h], scale)
            tol, rel = attention_bound(qh, kk[:, h], vv[:, h], scale)
            assert float((xb[b, h * grp:(h + 1) * grp].double() - want).abs().max()) <= tol
            assert torch.equal(w[b][h, n:], w0[b][h, n:])  # behind the rows: as they were
            old = w0[b][h, :n].double()
            off = (w[b][h, :n].double() - (old + 2 * p)).abs()
            assert bool((off <= 2 * rel * p + 2 * 2.0 ** -24 * (old + 2 * p) + 1e-37).all())


@pytest.mark.parametrize("t", TYPES)
def test_attention_keeps_small_weights_beside_an_empty_large_one(gla_ctx, t):
    """A row with nearly all the weight and no value (an attention sink): what is left
    of the output comes from weights of about 2^-16, which keep their precision."""
    g, nh, n_kv, hd, n = rng(11), 4, 1, 64, 500
    k, v = caches(g, [n], n_kv, hd, t), caches(g, [n], n_kv, hd, t)
    q = normal(g, 1, nh, hd)
    k[0][:n] *= 0.1
    k[0][0] = (q[0].mean(0) * 0).to(DT[t])
    q[0, :, 0] = 8.0
    k[0][:n, 0] = 0.0
    k[0][0, 0] = 11.0  # a score of 11 above the others: weights of 2^-16 at scale 1/8
    v[0][0] = 0.0
    xb, w = torch.empty(1, nh, hd, device="cuda"), torch.zeros(1, n_kv, n, device="cuda")
    gla_ctx.decode_weights(q, ptrs(k), ptrs(v), i32([n]), n, xb, ptrs(list(w)), n, 1, nh, n_kv, hd,
                           f16_cache=t == "f16")
    ok(gla_ctx)
    want, _ = attend64(q[0], k[0][:n, :hd], v[0][:n, :hd], 0.125)
    _, rel = attention_bound(q[0], k[0][:n, :hd], v[0][:n, :hd], 0.125)
    s = (q[0].double() @ k[0][:n, :hd].double().T) * 0.125
    mass = torch.softmax(s, 1) @ v[0][:n, :hd].double().abs()  # relative to the terms, not to max |v|
    assert bool(((xb[0].double() - want).abs() <= rel * mass + 1e-30).all())


@pytest.mark.parametrize("t", TYPES)
def test_attention_magnitudes(gla_ctx, t):
    """Queries near FP32's small and large ends (an FP16 split by itself would lose them),
    a zero query, and scores that leave one row."""
    g, nh, n_kv, hd, n, br = rng(12), 4, 1, 96, 90, 16
    k, v = caches(g, [n], n_kv, hd, t), caches(g, [n], n_kv, hd, t)
    q = normal(g, 1, nh, hd)
    q[0, 0] *= 1e-6
    q[0, 1] = 0
    q[0, 2] *= 1e6
    xb = torch.empty(1, nh, hd, device="cuda")
    ids = torch.arange(6, dtype=torch.int32, device="cuda").view(1, 1, 6).contiguous()
    for scale, heads in ((1e5, (0, 1)), (1e-7, (0, 1, 2, 3)), (1.0, (1, 3))):
        gla_ctx.decode_blocks(q, ptrs(k), ptrs(v), i32([n]), ids, 6, xb, 1, nh, n_kv, hd, br,
                              scale=scale, f16_cache=t == "f16")
        ok(gla_ctx)
        for h in heads:
            qh = q[0, h:h + 1]
            want, _ = attend64(qh, k[0][:n], v[0][:n], scale)
            tol, _ = attention_bound(qh, k[0][:n], v[0][:n], scale)
            assert float((xb[0, h].double() - want[0]).abs().max()) <= tol
    # head 2 at scale 1: scores of 1e6 leave the largest one's row alone
    s = (q[0, 2].double() @ k[0][:n].double().T).cpu()
    two = s.topk(2)[0]
    only = v[0][int(s.argmax())].double()
    # FP16 values are exact operands.  An FP32 value is the sum of a half rounded to 11 bits and
    # a rest of at most 2^12 units of 2^-23 times its power of two, of which the TF32 operand
    # keeps 11 bits: one unit, 2^-23 |v| * (power of two / |v|) <= 2^-23 |v|, may be dropped;
    # p is 1 and the two terms' sum has 24 bits.
    tol = 0.0 if t == "f16" else 2.0 ** -23
    assert float(two[0] - two[1]) > 100 and bool(((xb[0, 2].double() - only).abs() <= tol * only.abs()).all())


def test_offsets_past_32_bits(gla_ctx):
    """A cache of more than 2^32 elements: the last blocks are read, listed and moved."""
    n_kv, hd, br = 8, 128, 128
    n = (1 << 32) // (n_kv * hd) + 300
    if torch.cuda.mem_get_info()[0] < 3 * n * n_kv * hd * 2:
        pytest.skip("not enough device memory")
    k = torch.empty(n, n_kv * hd, dtype=torch.float16, device="cuda")
    g, tail = rng(13), 300
    k[-tail:] = normal(g, tail, n_kv * hd).half()
    k[:br] = normal(g, br, n_kv * hd).half()
    q = normal(g, 1, 32, hd)
    nb = -(-n // br)
    ids = i32([[[0, nb - 2, nb - 1]] * n_kv]).contiguous()
    xb = torch.empty(1, 32, hd, device="cuda")
    gla_ctx.decode_blocks(q, ptrs([k]), ptrs([k]), i32([n]), ids, 3, xb, 1, 32, n_kv, hd, br,
                          f16_cache=True)
    ok(gla_ctx)
    rows = [r for j in (0, nb - 2, nb - 1) for r in range(j * br, min(n, (j + 1) * br))]
    kk = k[rows].view(len(rows), n_kv, hd)
    for h in range(n_kv):
        qh = q[0, 4 * h:4 * h + 4]
        want, _ = attend64(qh, kk[:, h], kk[:, h], hd ** -0.5)
        tol, _ = attention_bound(qh, kk[:, h], kk[:, h], hd ** -0.5)
        assert float((xb[0, 4 * h:4 * h + 4].double() - want).abs().max()) <= tol
    bounds = torch.zeros(nb, n_kv, 2, hd, dtype=torch.float16, device="cuda")
    gla_ctx.block_bounds(ptrs([k]), i32([n]), n, ptrs([bounds]), 1, n_kv, hd, br,
                         start_pos=i32([n - 200]), f16_cache=True)
    ok(gla_ctx)
    last = k[(nb - 1) * br:].view(-1, n_kv, hd)
    assert torch.equal(bounds[nb - 1, :, 0], last.amin(0)) and torch.equal(bounds[nb - 1, :, 1], last.amax(0))


# ------------------------------------------------------------------------- evict
def kept64(w, n, keep, recent):
    if n <= keep:
        return list(range(n))
    w = [-math.inf if math.isnan(x) else x for x in w[: n - recent].tolist()]
    best = sorted(range(n - recent), key=lambda j: (-w[j], j))[: keep - recent]
    return sorted(best) + list(range(n - recent, n))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n_kv,hd,lens,keep,recent", [
    (8, 128, [700, 64, 65, 0, 3], 64, 16), (2, 64, [5000, 4999], 1200, 0), (3, 96, [2000], 1, 1),
    (1, 64, [40000], 9000, 9000), (4, 96, [1300, 1300], 1299, 5), (2, 128, [30], 50, 7),
    (2, 64, [33, 700, 20, 0, 21] * 16, 20, 3), (16, 96, [900] * 10, 300, 40)])
def test_evict_keeps_the_heaviest_rows(gla_ctx, t, in_place, n_kv, hd, lens, keep, recent):
    g, pad, top = rng(14, n_kv, hd, keep), 8, max(lens)
    batch, stride = len(lens), n_kv * hd + pad
    k, v = caches(g, lens, n_kv, hd, t, pad_cols=pad), caches(g, lens, n_kv, hd, t, pad_cols=pad)
    ws = top + 3
    w = []
    for _ in lens:
        x = torch.exp(normal(g, n_kv, ws))
        x[:, ::3] = 0.0  # ties
        x[:, 1::7] = float("nan") if n_kv == 3 else 0.25
        w.append(x)
    k0, v0, w0 = [x.clone() for x in k], [x.clone() for x in v], [x.clone() for x in w]
    kept = torch.full((batch, n_kv, keep), 77, dtype=torch.int32, device="cuda")
    kw = {}
    if in_place:
        ko, vo, wo, wos = k, v, w, ws
    else:
        wos = keep + 1
        ko = [torch.full((keep + 2, stride), 3.0, dtype=DT[t], device="cuda") for _ in lens]
        vo = [x.clone() for x in ko]
        wo = [torch.full((n_kv, wos), 3.0, device="cuda") for _ in lens]
        kw = dict(k_out_ptrs=ptrs(ko), v_out_ptrs=ptrs(vo), weight_out_ptrs=ptrs(wo),
                  weight_out_stride=wos)
    gla_ctx.kv_evict(ptrs(k), ptrs(v), ptrs(w), ws, i32(lens), top, keep, recent, kept, batch, n_kv,
                     hd, kv_stride=stride, f16_cache=t == "f16", **kw)
    ok(gla_ctx)
    same = lambda a, b: torch.equal(a.view(torch.int16 if a.dtype == torch.float16 else torch.int32),  # noqa: E731
                                    b.view(torch.int16 if b.dtype == torch.float16 else torch.int32))
    for b, n in enumerate(lens):
        for h in range(n_kv):
            rows = kept64(w0[b][h], n, keep, recent)
            m = len(rows)
            assert kept[b, h].tolist() == rows + [-1] * (keep - m)
            cols = slice(h * hd, (h + 1) * hd)
            for src, dst in ((k0, ko), (v0, vo)):
                assert same(dst[b][:m, cols].contiguous(), src[b][rows, cols].contiguous())
                if in_place:  # behind the kept rows: as they were
                    assert same(dst[b][m:, cols].contiguous(), src[b][m:, cols].contiguous())
                else:
                    assert (dst[b][m:] == 3.0).all() and (dst[b][:, n_kv * hd:] == 3.0).all()
                    assert same(k[b], k0[b]) and same(v[b], v0[b]) and same(w[b], w0[b])
            assert same(wo[b][h, :m].contiguous(), w0[b][h, rows].contiguous())
            if in_place:
                assert (wo[b][h, m:n] == 0).all() or n <= keep
                assert same(wo[b][h, n:].contiguous(), w0[b][h, n:].contiguous())
            else:
                assert (wo[b][h, m:] == 3.0).all()


@pytest.mark.parametrize("n,keep,recent", [(40_001, 30_000, 1), (100_003, 7000, 33), (900_005, 20_001, 2)])
def test_evict_long_interleaved_sequences_in_place(gla_ctx, n, keep, recent):
    """Selections over the CTAs of a cluster (the longest past their shared memory), with ties
    over all of them; K and V are the two halves of one row."""
    g, hd = rng(26, n), 64
    kv = normal(g, n, 2 * hd).half()
    k, v = kv[:, :hd], kv[:, hd:]
    w = torch.exp(normal(g, 1, n))
    w[0, ::2] = 1.0
    kv0, w0 = kv.clone(), w.clone()
    kept = torch.empty(1, 1, keep, dtype=torch.int32, device="cuda")
    gla_ctx.kv_evict(ptrs([k]), ptrs([v]), ptrs([w]), n, i32([n]), n, keep, recent, kept, 1, 1, hd,
                     kv_stride=2 * hd, f16_cache=True)
    ok(gla_ctx)
    rows = kept64(w0[0], n, keep, recent)
    assert kept[0, 0].tolist() == rows
    assert torch.equal(kv[:keep], kv0[rows]) and torch.equal(kv[keep:], kv0[keep:])
    assert torch.equal(w[0, :keep], w0[0, rows]) and (w[0, keep:] == 0).all()


def test_evict_to_the_same_cache_is_refused(gla_ctx):
    g = rng(15)
    k, v = caches(g, [50, 50], 2, 64, "f32"), caches(g, [50, 50], 2, 64, "f32")
    w = [torch.rand(2, 50, device="cuda") for _ in range(2)]
    ko = [k[0], torch.zeros_like(k[1])]
    vo, wo = [torch.zeros_like(x) for x in v], [torch.zeros_like(x) for x in w]
    before = k[0].clone()
    kept = torch.empty(2, 2, 10, dtype=torch.int32, device="cuda")
    gla_ctx.kv_evict(ptrs(k), ptrs(v), ptrs(w), 50, i32([50, 50]), 50, 10, 2, kept, 2, 2, 64,
                     k_out_ptrs=ptrs(ko), v_out_ptrs=ptrs(vo), weight_out_ptrs=ptrs(wo),
                     weight_out_stride=50)
    assert gla_ctx.device_status() == -1
    assert torch.equal(k[0][:50], before[:50]) and (vo[0] == 0).all()
    assert torch.equal(ko[1][0, :64], k[1][int(kept[1, 0, 0]), :64])


# ------------------------------------------------------------------------- together
@pytest.mark.parametrize("t", TYPES)
def test_a_served_batch_from_prompt_to_evicted_sparse_decode(gla_ctx, t):
    """Prompts in the caches; a few tokens of gla_decode_weights_*; eviction in place;
    bounds of what is left; then, captured once and replayed, the token step of append,
    selection and attention over the selected blocks - each output against 64 bits."""
    f16, g = t == "f16", rng(16)
    nh, n_kv, hd, br, cap, theta = 8, 2, 64, 16, 400, 1e4
    lens, keep, recent, n_sel = [300, 150, 90], 128, 24, 4
    batch, grp, scale = 3, 4, 1 / 8
    k = [torch.zeros(cap, n_kv * hd, dtype=DT[t], device="cuda") for _ in lens]
    v = [torch.zeros_like(x) for x in k]
    for kk, vv, n in zip(k, v, lens):
        kk[:n], vv[:n] = normal(g, n, n_kv * hd).to(DT[t]), normal(g, n, n_kv * hd).to(DT[t])
    w = [torch.zeros(n_kv, cap, device="cuda") for _ in lens]
    kp, vp, wp = ptrs(k), ptrs(v), ptrs(w)
    pos, rows, n_pos = i32(lens), i32(lens), i32([n + 1 for n in lens])
    q_in, q = normal(g, batch, nh, hd), torch.empty(batch, nh, hd, device="cuda")
    kn, vn = normal(g, batch, n_kv, hd), normal(g, batch, n_kv, hd)
    xb = torch.empty(batch, nh, hd, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx = gla.Context(0, stream.cuda_stream)
    with torch.cuda.stream(stream):
        for _ in range(3):
            q_in.normal_(generator=g), kn.normal_(generator=g), vn.normal_(generator=g)
            ctx.rope_append_batched(q_in, kn, vn, q, kp, vp, pos, batch, nh, n_kv, hd, cap, theta,
                                    rows=rows, f16_cache=f16)
            ctx.decode_weights(q, kp, vp, n_pos, cap, xb, wp, cap, batch, nh, n_kv, hd, f16_cache=f16)
            pos += 1
            rows += 1
            n_pos += 1
        rows_now = [n + 3 for n in lens]
        for b, n in enumerate(rows_now):  # each of 3 tokens gave every head a weight of one
            total = w[b].sum(1)
            # 3 * grp softmaxes over n rows: n additions, and 2^-18 a weight's relative error
            assert float((total - 3 * grp).abs().max()) <= 3 * grp * (n * 2.0 ** -24 + 2.0 ** -18)
        k0, w0 = [x.clone() for x in k], [x.clone() for x in w]
        kept = torch.empty(batch, n_kv, keep, dtype=torch.int32, device="cuda")
        now = i32(rows_now)
        ctx.kv_evict(kp, vp, wp, cap, now, cap, keep, recent, kept, batch, n_kv, hd, f16_cache=f16)
        for b, n in enumerate(rows_now):
            for h in range(n_kv):
                want = kept64(w0[b][h], n, keep, recent)
                assert kept[b, h].tolist()[: len(want)] == want
                assert torch.equal(k[b][: len(want), h * hd:(h + 1) * hd], k0[b][want, h * hd:(h + 1) * hd])
        left = torch.clamp(now, max=keep)
        bs = [torch.zeros(-(-cap // br), n_kv, 2, hd, dtype=DT[t], device="cuda") for _ in lens]
        bp = ptrs(bs)
        ctx.block_bounds(kp, left, cap, bp, batch, n_kv, hd, br, f16_cache=f16)
        rows.copy_(left)
        n_pos.copy_(left + 1)
        ids = torch.empty(batch, n_kv, n_sel, dtype=torch.int32, device="cuda")

        def step():
            ctx.rope_append_batched(q_in, kn, vn, q, kp, vp, pos, batch, nh, n_kv, hd, cap, theta,
                                    rows=rows, bounds_ptrs=bp, block_rows=br, f16_cache=f16)
            ctx.block_select(q, bp, n_pos, cap, ids, batch, nh, n_kv, hd, br, n_sel, n_first=1,
                             n_last=1, f16_cache=f16)
            ctx.decode_blocks(q, kp, vp, n_pos, ids, n_sel, xb, batch, nh, n_kv, hd, br,
                              f16_cache=f16)
            pos.add_(1)
            rows.add_(1)
            n_pos.add_(1)

        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for _ in range(20):  # across a block's end
            q_in.normal_(generator=g), kn.normal_(generator=g), vn.normal_(generator=g)
            graph.replay()
            n_now = (n_pos - 1).tolist()
            for b, n in enumerate(n_now):
                kk, vv = k[b][:n].view(n, n_kv, hd), v[b][:n].view(n, n_kv, hd)
                for j in range(-(-n // br)):
                    part = kk[j * br:(j + 1) * br]
                    assert torch.equal(bs[b][j, :, 0], part.amin(0)) and torch.equal(bs[b][j, :, 1], part.amax(0))
                want_ids, gap = select64(q[b], bs[b], n, br, n_sel, 1, 1)
                assert gap > 1e-11
                np.testing.assert_array_equal(ids[b].cpu().numpy(), want_ids)
                for h in range(n_kv):
                    at = [r for j in want_ids[h] if j >= 0 for r in range(j * br, min(n, (j + 1) * br))]
                    qh = q[b, h * grp:(h + 1) * grp]
                    want, _ = attend64(qh, kk[at, h], vv[at, h], scale)
                    tol, _ = attention_bound(qh, kk[at, h], vv[at, h], scale)
                    assert float((xb[b, h * grp:(h + 1) * grp].double() - want).abs().max()) <= tol
        assert ctx.device_status() == 0
        # all blocks listed: the dense batched decode over the same rows
        n = n_pos - 1
        every = torch.arange(-(-cap // br), dtype=torch.int32, device="cuda").repeat(batch, n_kv, 1)
        full, dense = torch.empty_like(xb), torch.empty_like(xb)
        ctx.decode_blocks(q, kp, vp, n, every, every.shape[2], full, batch, nh, n_kv, hd, br, f16_cache=f16)
        ctx.decode_batched(q, kp, vp, n, cap, dense, batch, nh, n_kv, hd, f16_cache=f16)
        for b, m in enumerate(n.tolist()):
            tol = max(attention_bound(q[b], k[b][:m, h * hd:(h + 1) * hd], v[b][:m], scale)[0]
                      for h in range(n_kv))
            assert float((full[b] - dense[b]).abs().max()) <= 2 * tol
        del graph
    stream.synchronize()
    ctx.close()


def test_a_captured_long_list_needs_its_workspace(gla_ctx):
    """Long lists of few heads are cut into parts in the context workspace."""
    g, nh, n_kv, hd, br, n_sel = rng(26), 8, 2, 64, 128, 160
    n = n_sel * br
    k, v = caches(g, [n], n_kv, hd, "f16"), caches(g, [n], n_kv, hd, "f16")
    q, xb = normal(g, 1, nh, hd), torch.empty(1, nh, hd, device="cuda")
    ids = torch.arange(n_sel, dtype=torch.int32, device="cuda").repeat(1, n_kv, 1).contiguous()
    kp, vp, np_ = ptrs(k), ptrs(v), i32([n])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx = gla.Context(0, stream.cuda_stream)
    call = lambda: ctx.decode_blocks(q, kp, vp, np_, ids, n_sel, xb, 1, nh, n_kv, hd, br, f16_cache=True)  # noqa: E731
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(gla.GlaError, match="must grow"):
            with torch.cuda.graph(graph, stream=stream):
                call()
        call()
        want = xb.clone()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for _ in range(3):
            xb.zero_()
            graph.replay()
            assert torch.equal(xb, want)
        del graph
    stream.synchronize()
    assert ctx.device_status() == 0
    ctx.close()
    for h in range(n_kv):
        qh, kk, vv = q[0, 4 * h:4 * h + 4], rows_of(k[0], n, n_kv, hd)[:, h], rows_of(v[0], n, n_kv, hd)[:, h]
        got, (o, _) = want[0, 4 * h:4 * h + 4], attend64(qh, kk, vv, 1 / 8)
        assert float((got.double() - o).abs().max()) <= attention_bound(qh, kk, vv, 1 / 8)[0]


def test_a_captured_weights_call_survives_a_larger_one(gla_ctx):
    """The score workspace may grow after a capture: the graph's own buffer stays."""
    g, nh, n_kv, hd, n = rng(17), 8, 2, 64, 200
    k, v = caches(g, [n], n_kv, hd, "f16"), caches(g, [n], n_kv, hd, "f16")
    big = caches(g, [9000], n_kv, hd, "f16")
    q, xb = normal(g, 1, nh, hd), torch.empty(1, nh, hd, device="cuda")
    xb2, w2 = torch.empty_like(xb), [torch.zeros(n_kv, 9000, device="cuda")]
    w = [torch.zeros(n_kv, n, device="cuda")]
    kp, vp, wp, np_, bp = ptrs(k), ptrs(v), ptrs(w), i32([n]), ptrs(big)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx = gla.Context(0, stream.cuda_stream)
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(gla.GlaError, match="must grow"):
            with torch.cuda.graph(graph, stream=stream):
                ctx.decode_weights(q, kp, vp, np_, n, xb, wp, n, 1, nh, n_kv, hd, f16_cache=True)
        ctx.decode_weights(q, kp, vp, np_, n, xb, wp, n, 1, nh, n_kv, hd, f16_cache=True)
        want, once = xb.clone(), w[0].clone()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ctx.decode_weights(q, kp, vp, np_, n, xb, wp, n, 1, nh, n_kv, hd, f16_cache=True)
        ctx.decode_weights(q, bp, bp, i32([9000]), 9000, xb2, ptrs(w2), 9000, 1, nh, n_kv, hd,
                           f16_cache=True)
        xb.zero_()
        graph.replay()
        stream.synchronize()
        assert torch.equal(xb, want) and torch.equal(w[0], once + once)
        del graph
    assert ctx.device_status() == 0
    ctx.close()


# ------------------------------------------------------------------------- refusals
def test_bad_pointers_and_lengths_are_latched(gla_ctx):
    """A null or misaligned pointer skips its sequence; a length outside is clamped."""
    g, nh, n_kv, hd, br = rng(18), 8, 2, 64, 16
    k = caches(g, [40, 40, 40], n_kv, hd, "f16")
    p = ptrs(k)
    bad = p.clone()
    bad[0], bad[1] = 0, p[1] + 2
    q, xb = normal(g, 3, nh, hd), torch.full((3, nh, hd), 9.0, device="cuda")
    ids = torch.zeros(3, n_kv, 1, dtype=torch.int32, device="cuda")
    gla_ctx.decode_blocks(q, bad, p, i32([40] * 3), ids, 1, xb, 3, nh, n_kv, hd, br, f16_cache=True)
    assert gla_ctx.device_status() in (-1, -4) and gla_ctx.device_status() == 0
    assert (xb[:2] == 0).all() and bool((xb[2] != 9.0).all())
    gla_ctx.decode_blocks(q, p, p, i32([40, -3, 40]), ids, 1, xb, 3, nh, n_kv, hd, br, f16_cache=True)
    assert gla_ctx.device_status() == -1 and (xb[1] == 0).all() and bool((xb[0] != 0).any())
    bs = [torch.full((3, n_kv, 2, hd), 7.0, dtype=torch.float16, device="cuda") for _ in k]
    gla_ctx.block_bounds(bad, i32([40] * 3), 40, ptrs(bs), 3, n_kv, hd, br, f16_cache=True)
    assert gla_ctx.device_status() in (-1, -4)
    assert (bs[0] == 7.0).all() and (bs[1] == 7.0).all() and (bs[2] != 7.0).any()
    gla_ctx.block_bounds(p, i32([41, 40, 40]), 40, ptrs(bs), 3, n_kv, hd, br, f16_cache=True)
    assert gla_ctx.device_status() == -1
    assert torch.equal(bs[0][2, :, 1], rows_of(k[0], 40, n_kv, hd)[32:].amax(0))  # clamped to 40
    got = torch.full((3, n_kv, 2), 5, dtype=torch.int32, device="cuda")
    gla_ctx.block_select(q, ptrs(bs) * i32([0, 1, 1]), i32([40] * 3), 40, got, 3, nh, n_kv, hd, br, 2,
                         f16_cache=True)
    assert gla_ctx.device_status() == -1 and (got[0] == -1).all() and (got[1:] >= 0).all()
    w = [torch.rand(n_kv, 40, device="cuda") for _ in k]
    wbad = ptrs(w) * i32([0, 1, 1])
    gla_ctx.decode_weights(q, p, p, i32([40] * 3), 40, xb, wbad, 40, 3, nh, n_kv, hd, f16_cache=True)
    assert gla_ctx.device_status() == -1 and (xb[0] == 0).all() and bool((xb[1] != 0).any())
    kept = torch.full((3, n_kv, 8), 5, dtype=torch.int32, device="cuda")
    before = [x.clone() for x in k]
    gla_ctx.kv_evict(p, p, wbad, 40, i32([40] * 3), 40, 8, 2, kept, 3, n_kv, hd, f16_cache=True)
    assert gla_ctx.device_status() == -1 and (kept[0] == -1).all()
    assert torch.equal(k[0][:40], before[0][:40])


def test_refusals(gla_ctx):
    """Every refusal is a status before any launch."""
    c = gla_ctx
    q = torch.zeros(64 * 128, device="cuda")
    p, n = torch.zeros(4, dtype=torch.int64, device="cuda"), i32([0, 0, 0, 0])
    ids = torch.zeros(64, dtype=torch.int32, device="cuda")

    def refuse(status, fn, *a, **kw):
        with pytest.raises(gla.GlaError) as e:
            fn(*a, **kw)
        assert e.value.status == status, e.value

    sel = lambda **o: dict(dict(q=q, bounds_ptrs=p, n_pos=n, max_n_pos=64, block_ids=ids, batch=1,  # noqa: E731
                                n_heads=8, n_kv_heads=2, head_dim=64, block_rows=16, n_sel=2), **o)
    blk = lambda **o: dict(dict(q=q, k_ptrs=p, v_ptrs=p, n_pos=n, block_ids=ids, n_sel=2, xb=q,  # noqa: E731
                                batch=1, n_heads=8, n_kv_heads=2, head_dim=64, block_rows=16), **o)
    wts = lambda **o: dict(dict(q=q, k_ptrs=p, v_ptrs=p, n_pos=n, max_n_pos=64, xb=q, weight_ptrs=p,  # noqa: E731
                                weight_stride=64, batch=1, n_heads=8, n_kv_heads=2, head_dim=64), **o)
    evi = lambda **o: dict(dict(k_ptrs=p, v_ptrs=p, weight_ptrs=p, weight_stride=64, n_pos=n,  # noqa: E731
                                max_n_pos=64, n_keep=8, n_recent=2, kept=ids, batch=1, n_kv_heads=2,
                                head_dim=64), **o)
    app = lambda **o: dict(dict(q=q, k=q, v=q, q_out=q, k_ptrs=p, v_ptrs=p, positions=n, batch=1,  # noqa: E731
                                n_heads=8, n_kv_heads=2, head_dim=64, context_length=16, theta=1e4), **o)
    bnd = lambda **o: dict(dict(k_ptrs=p, n_pos=n, max_n_pos=64, bounds_ptrs=p, batch=1, n_kv_heads=2,  # noqa: E731
                                head_dim=64, block_rows=16), **o)
    every = ((c.block_select, sel), (c.decode_blocks, blk), (c.decode_weights, wts),
             (c.rope_append_batched, app), (c.block_bounds, bnd), (c.kv_evict, evi))
    for fn, kw in every:
        refuse(-1, fn, **kw(batch=0))
        refuse(-3, fn, **kw(head_dim=80))
        refuse(-1, fn, **kw(n_kv_heads=0))
        first = next(iter(kw()))
        refuse(-1, fn, **kw(**{first: None}))
        if "n_heads" in kw():
            refuse(-1, fn, **kw(n_heads=9))
            refuse(-3, fn, **kw(n_heads=18))
        if "max_n_pos" in kw():
            refuse(-1, fn, **kw(max_n_pos=0))
        if "block_rows" in kw():
            refuse(-3, fn, **kw(block_rows=48))
        if fn != c.block_select:
            refuse(-1, fn, **kw(kv_stride=127))
            refuse(-4, fn, **kw(kv_stride=132, f16_cache=True))
            refuse(-4, fn, **kw(kv_stride=130))
    refuse(-1, c.block_select, **sel(n_sel=0))
    refuse(-1, c.block_select, **sel(n_first=2, n_last=1))
    refuse(-1, c.block_select, **sel(n_first=-1))
    refuse(-1, c.decode_blocks, **blk(n_sel=0))
    refuse(-1, c.decode_blocks, **blk(n_sel=1 << 27))
    refuse(-1, c.decode_blocks, **blk(scale=math.inf))
    refuse(-4, c.decode_blocks, **blk(q=q[1:]))
    refuse(-4, c.decode_weights, **wts(xb=q[1:]))
    refuse(-1, c.decode_weights, **wts(weight_stride=63))
    refuse(-1, c.decode_weights, **wts(scale=math.nan))
    refuse(-1, c.kv_evict, **evi(n_keep=0))
    refuse(-1, c.kv_evict, **evi(n_recent=9))
    refuse(-1, c.kv_evict, **evi(n_recent=-1))
    refuse(-1, c.kv_evict, **evi(weight_stride=63))
    refuse(-1, c.kv_evict, **evi(k_out_ptrs=p))
    refuse(-1, c.kv_evict, **evi(k_out_ptrs=p, v_out_ptrs=p, weight_out_ptrs=p, weight_out_stride=7))
    refuse(-3, c.rope_append_batched, **app(bounds_ptrs=p, block_rows=8))
    refuse(-1, c.rope_append_batched, **app(theta=0.0))
    refuse(-1, c.rope_append_batched, **app(style=2))
    refuse(-1, c.rope_append_batched, **app(context_length=0))
    assert c.device_status() == 0


# ------------------------------------------------------------------------- near the border
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,n_kv,hd", [(8, 2, 64), (7, 1, 128), (3, 3, 96), (4, 2, 128)])
def test_select_decides_below_fp32_rounding(gla_ctx, t, nh, n_kv, hd):
    """Scores that differ by less than an FP32 sum's rounding, by nothing, and by much:
    the order is that of the 64-bit sums.  Whole-number bounds and queries of 2^-30 steps
    make every 64-bit sum exact, so the reference's order is the true one."""
    g, br, nb = rng(20, nh, hd), 16, 700
    base = torch.randint(-3, 4, (1, n_kv, 2, hd), generator=g, device="cuda").float().sort(dim=2)[0]
    bs = base.repeat(nb, 1, 1, 1)
    # one channel of a block moves by one: times a query element of about 2^-20
    at = torch.randint(0, nb, (nb,), generator=g, device="cuda")
    bs[at, :, :, 0] += torch.randint(0, 5, (nb, 1, 1), generator=g, device="cuda").float()
    bs[::97, :, :, 1:9] += 2
    bs[5::89, :, :, 1:9] -= 3
    q = torch.randint(-(1 << 8), 1 << 8, (1, nh, hd), generator=g, device="cuda").float() / 64
    q[:, :, 0] = torch.randint(1, 1 << 10, (1, nh), generator=g, device="cuda").float() * 2.0 ** -30
    bs = bs.to(DT[t]).contiguous()
    for n_sel, first, last in ((1, 0, 0), (11, 1, 2), (350, 0, 1), (690, 0, 0)):
        ids = torch.empty(1, n_kv, n_sel, dtype=torch.int32, device="cuda")
        gla_ctx.block_select(q, ptrs([bs]), i32([nb * br]), nb * br, ids, 1, nh, n_kv, hd, br, n_sel,
                             n_first=first, n_last=last, f16_cache=t == "f16")
        ok(gla_ctx)
        want, _ = select64(q[0], bs, nb * br, br, n_sel, first, last)
        np.testing.assert_array_equal(ids[0].cpu().numpy(), want)


def test_select_magnitudes(gla_ctx):
    """FP32 sums that overflow, queries of NaN, infinity and zero, tiny products."""
    g, nh, n_kv, hd, br, nb, n_sel = rng(21), 2, 1, 64, 16, 200, 9
    b0 = normal(g, nb, n_kv, 2, hd).sort(dim=2)[0]
    q0 = normal(g, 1, nh, hd)
    cases = [(b0 * 1e30, q0 * 1e8), (b0 * 1e-30, q0 * 1e-12), (b0, q0 * 0), (b0 * 0, q0),
             (b0 * 3e38 / 8, q0 / 4)]
    for bo, q in cases:
        bo, q = bo.contiguous(), q.contiguous()
        ids = torch.empty(1, n_kv, n_sel, dtype=torch.int32, device="cuda")
        gla_ctx.block_select(q, ptrs([bo]), i32([nb * br]), nb * br, ids, 1, nh, n_kv, hd, br, n_sel,
                             n_last=0)
        ok(gla_ctx)
        want, _ = select64(q[0], bo, nb * br, br, n_sel, 0, 0)
        np.testing.assert_array_equal(ids[0].cpu().numpy(), want)
    q = q0.clone()
    q[0, 1, 3] = float("nan")  # that head counts as the lowest: the other one decides
    ids = torch.empty(1, n_kv, n_sel, dtype=torch.int32, device="cuda")
    gla_ctx.block_select(q, ptrs([b0]), i32([nb * br]), nb * br, ids, 1, nh, n_kv, hd, br, n_sel, n_last=0)
    ok(gla_ctx)
    want, _ = select64(q0[0, :1], b0, nb * br, br, n_sel, 0, 0)
    np.testing.assert_array_equal(ids[0].cpu().numpy(), want)


def test_select_refuses_more_blocks_than_it_holds(gla_ctx):
    q = torch.zeros(8 * 64, device="cuda")
    p, ids = torch.zeros(1, dtype=torch.int64, device="cuda"), i32([0] * 64)
    with pytest.raises(gla.GlaError) as e:
        gla_ctx.block_select(q, p, i32([0]), 24576 * 16 + 1, ids, 1, 8, 2, 64, 16, 2)
    assert e.value.status == -3
    gla_ctx.block_select(q, p, i32([0]), 24576 * 16, ids, 1, 8, 2, 64, 16, 2)  # a null pointer: -1s
    assert gla_ctx.device_status() == -1 and (ids[:4] == -1).all()


@pytest.mark.parametrize("t", TYPES)
def test_select_over_the_most_blocks(gla_ctx, t):
    g, nh, n_kv, hd, br, nb, n_sel = rng(22), 4, 1, 64, 16, 24576, 4000
    bs = normal(g, nb, n_kv, 2, hd).sort(dim=2)[0].to(DT[t]).contiguous()
    q = normal(g, 1, nh, hd)
    ids = torch.empty(1, n_kv, n_sel, dtype=torch.int32, device="cuda")
    gla_ctx.block_select(q, ptrs([bs]), i32([nb * br - 3]), nb * br, ids, 1, nh, n_kv, hd, br, n_sel,
                         n_first=2, n_last=3, f16_cache=t == "f16")
    ok(gla_ctx)
    want, gap = select64(q[0], bs, nb * br - 3, br, n_sel, 2, 3)
    assert gap > 1e-11
    np.testing.assert_array_equal(ids[0].cpu().numpy(), want)


# ------------------------------------------------------------------------- calls side by side
def test_two_contexts_at_once(gla_ctx):
    """Two contexts on two streams, their calls in flight together, give what each gives alone."""
    g, nh, n_kv, hd, n = rng(23), 8, 2, 64, 6000
    got, alone = [], []
    streams = [torch.cuda.Stream() for _ in range(2)]
    data = []
    for _ in range(2):
        k, v = caches(g, [n], n_kv, hd, "f16"), caches(g, [n], n_kv, hd, "f16")
        data.append((normal(g, 1, nh, hd), k, v, ptrs(k), ptrs(v), i32([n])))
    torch.cuda.synchronize()
    for together in (False, True):
        out = []
        ctxs = [gla.Context(0, s.cuda_stream) for s in streams]
        for rep in range(3):
            for ctx, s, (q, k, v, kp, vp, np_) in zip(ctxs, streams, data):
                with torch.cuda.stream(s):
                    if rep == 0:
                        out.append((torch.empty(1, nh, hd, device="cuda"), torch.zeros(n_kv, n, device="cuda")))
                    xb, w = out[ctxs.index(ctx)]
                    ctx.decode_weights(q, kp, vp, np_, n, xb, ptrs([w]), n, 1, nh, n_kv, hd, f16_cache=True)
                if not together:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        for ctx in ctxs:
            assert ctx.device_status() == 0
            ctx.close()
        (got if together else alone).extend(out)
    for a, b in zip(alone, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_more_sequences_than_a_grid_row(gla_ctx):
    """70,000 sequences of one and two rows."""
    batch, nh, n_kv, hd, br, cap = 70000, 2, 1, 64, 16, 2
    g = rng(24)
    kv = normal(g, 2, batch, cap, hd)
    at = torch.arange(batch, device="cuda", dtype=torch.int64) * (cap * hd * 4)
    kp, vp = kv[0].data_ptr() + at, kv[1].data_ptr() + at
    q, k, v = normal(g, batch, nh, hd), normal(g, batch, n_kv, hd), normal(g, batch, n_kv, hd)
    rows = (torch.arange(batch, device="cuda") % 2).int()
    q_out = torch.empty_like(q)
    zero = torch.zeros_like(rows)
    gla_ctx.rope_append_batched(q, k, v, q_out, kp, vp, zero, batch, nh, n_kv, hd, cap, 1e4, rows=rows)
    pick = torch.arange(batch, device="cuda")
    # position 0 turns nothing
    assert torch.equal(q_out, q) and torch.equal(kv[0][pick, rows.long()], k[:, 0])
    bounds = torch.zeros(batch, 2, hd, device="cuda")
    bp = bounds.data_ptr() + torch.arange(batch, device="cuda", dtype=torch.int64) * (2 * hd * 4)
    n = rows + 1
    gla_ctx.block_bounds(kp, n, cap, bp, batch, n_kv, hd, br)
    two = (rows == 1)[:, None]
    assert torch.equal(bounds[:, 0], torch.where(two, kv[0].amin(1), kv[0][:, 0]))
    ids = torch.full((batch, n_kv, 1), 9, dtype=torch.int32, device="cuda")
    gla_ctx.block_select(q, bp, n, cap, ids, batch, nh, n_kv, hd, br, 1)
    assert (ids == 0).all()
    xb = torch.empty(batch, nh, hd, device="cuda")
    gla_ctx.decode_blocks(q, kp, vp, n, ids, 1, xb, batch, nh, n_kv, hd, br)
    ok(gla_ctx)
    s = torch.einsum("bhd,btd->bht", q.double(), kv[0].double()) / 8
    s[~two[:, 0], :, 1] = -math.inf
    want = torch.einsum("bht,btd->bhd", torch.softmax(s, -1), kv[1].double())
    # two rows of |q| and |k| below 6: attention_bound's terms at its largest
    tol = attention_bound(torch.full((1, hd), 6.0, device="cuda"), torch.full((2, hd), 6.0, device="cuda"),
                          torch.full((2, hd), 6.0, device="cuda"), 1 / 8)[0]
    assert float(kv.abs().max()) < 6 and float(q.abs().max()) < 6
    assert float((xb.double() - want).abs().max()) <= tol


@pytest.mark.parametrize("t", TYPES)
def test_eviction_captured_and_replayed(gla_ctx, t):
    """Weights, eviction in place and bounds in one captured graph, replayed while the caches
    grow again: every replay keeps what the 64-bit order keeps of its own weights."""
    f16, g = t == "f16", rng(25)
    nh, n_kv, hd, br, cap, keep, recent, theta = 4, 2, 96, 32, 300, 100, 11, 1e4
    k = [normal(g, cap, n_kv * hd).to(DT[t]) for _ in range(2)]
    v = [normal(g, cap, n_kv * hd).to(DT[t]) for _ in range(2)]
    w = [torch.zeros(n_kv, cap, device="cuda") for _ in range(2)]
    bs = [torch.zeros(-(-cap // br), n_kv, 2, hd, dtype=DT[t], device="cuda") for _ in range(2)]
    kp, vp, wp, bp = ptrs(k), ptrs(v), ptrs(w), ptrs(bs)
    q, xb = normal(g, 2, nh, hd), torch.empty(2, nh, hd, device="cuda")
    n = i32([280, 90])
    left = torch.clamp(n, max=keep)
    kept = torch.empty(2, n_kv, keep, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx = gla.Context(0, stream.cuda_stream)

    def step():
        ctx.decode_weights(q, kp, vp, n, cap, xb, wp, cap, 2, nh, n_kv, hd, f16_cache=f16)
        ctx.kv_evict(kp, vp, wp, cap, n, cap, keep, recent, kept, 2, n_kv, hd, f16_cache=f16)
        torch.clamp(n, max=keep, out=left)
        ctx.block_bounds(kp, left, cap, bp, 2, n_kv, hd, br, f16_cache=f16)

    with torch.cuda.stream(stream):
        ctx.decode_weights(q, kp, vp, i32([0, 0]), cap, xb, wp, cap, 2, nh, n_kv, hd, f16_cache=f16)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for lens in ([280, 90], [131, 90], [300, 101], [100, 100]):
            n.copy_(i32(lens))
            q.normal_(generator=g)
            k0, w0 = [x.clone() for x in k], [x.clone() for x in w]
            graph.replay()
            for b, m in enumerate(lens):
                kk, vv = rows_of(k0[b], m, n_kv, hd), None
                for h in range(n_kv):
                    grp = nh // n_kv
                    qh = q[b, h * grp:(h + 1) * grp]
                    _, p = attend64(qh, kk[:, h], kk[:, h], hd ** -0.5)
                    rows = kept[b, h].tolist()
                    rows = rows[: min(m, keep)]
                    assert rows == sorted(set(rows)) and rows[-1] == m - 1
                    total = w0[b][h, :m].double() + p
                    # the kept weights are the sums' (see test_decode_weights_adds_the_softmax), and no
                    # dropped row had more than a kept older one by over both sums' errors
                    _, rel = attention_bound(qh, kk[:, h], kk[:, h], hd ** -0.5)
                    off = 2 * float((rel * p + 2.0 ** -24 * total).max())
                    assert float((w[b][h, : len(rows)].double() - total[rows]).abs().max()) <= off
                    if m > keep:
                        old = [r for r in rows if r < m - recent]
                        gone = sorted(set(range(m - recent)) - set(old))
                        assert float(total[old].min()) >= float(total[gone].max()) - off
                        assert (w[b][h, keep:m] == 0).all()
                    assert torch.equal(k[b][: len(rows), h * hd:(h + 1) * hd], k0[b][rows, h * hd:(h + 1) * hd])
                x = rows_of(k[b], min(m, keep), n_kv, hd)
                assert torch.equal(bs[b][0, :, 0], x[:br].amin(0)) and torch.equal(bs[b][-(-len(rows) // br) - 1, :, 1], x[(-(-len(rows) // br) - 1) * br:].amax(0))
        assert ctx.device_status() == 0
        del graph
    stream.synchronize()
    ctx.close()

"""Attention over FP32 and FP16 caches near the ends of what the header allows."""
import pytest
import torch

from test_cache_ops_gpu import DT, TYPES, attend64, attention_bound, i32, normal, ok, ptrs, rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,big_q,big_k,big_v", [
    ("f32", 60, 56, 114), ("f32", 118, 0, 0), ("f32", 0, 116, 0), ("f32", -100, -20, -90),
    ("f16", 120, 12, 12), ("f16", -120, -2, -8)])
def test_attention_of_very_large_and_small_numbers(gla_ctx, t, big_q, big_k, big_v):
    """Sums of |q k| and |v| just below 2^127 (below 2^7 times the magnitudes named, and 2^10
    for 64 rows of |v| < 2^4), and numbers far below one; the scale brings the scores back."""
    g, nh, n_kv, hd, n, br = rng(51, big_q + 200, big_k + 200), 4, 1, 64, 60, 16
    q = (normal(g, 1, nh, hd).double() * 2.0 ** big_q).float()
    k = (normal(g, 64, hd).double() * 2.0 ** big_k).to(DT[t])
    v = (normal(g, 64, hd).double() * 2.0 ** big_v).to(DT[t])
    scale = 0.125 * 2.0 ** -(big_q + big_k)
    xb = torch.full((1, nh, hd), float("nan"), device="cuda")
    ids = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 1, 4).contiguous()
    gla_ctx.decode_blocks(q, ptrs([k]), ptrs([v]), i32([n]), ids, 4, xb, 1, nh, n_kv, hd, br, scale=scale,
                          f16_cache=t == "f16")
    ok(gla_ctx)
    want, p = attend64(q[0], k[:n], v[:n], scale)
    tol, rel = attention_bound(q[0], k[:n], v[:n], scale)
    assert float((xb[0].double() - want).abs().max()) <= tol
    w = torch.zeros(n_kv, n, device="cuda")
    xb.fill_(float("nan"))
    gla_ctx.decode_weights(q, ptrs([k]), ptrs([v]), i32([n]), n, xb, ptrs([w]), n, 1, nh, n_kv, hd, scale=scale,
                           f16_cache=t == "f16")
    ok(gla_ctx)
    assert float((xb[0].double() - want).abs().max()) <= tol
    assert bool(((w[0].double() - p).abs() <= rel * p + 2 * 2.0 ** -24 * p + 1e-37).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nh,n_kv,hd", [(8, 1, 128), (4, 4, 64), (7, 1, 96)])
def test_a_single_attended_row_is_returned(gla_ctx, t, nh, n_kv, hd):
    """FP16 values bit for bit, FP32 ones within 2^-23: hi + lo keep 23 of 24 bits (lo of at most
    2^12 units holds 11 bits, so a unit, 2^-23 of the value's power of two, may go), the weight is
    one and its half of it exact, and hi + lo is rounded where the unit went, to the same grid."""
    g, n, br = rng(52, nh, hd), 1, 16
    q, k, v = normal(g, 1, nh, hd), normal(g, n, n_kv * hd).to(DT[t]), normal(g, n, n_kv * hd).to(DT[t])
    ids = torch.zeros(1, n_kv, 1, dtype=torch.int32, device="cuda")
    xb = torch.empty(1, nh, hd, device="cuda")
    gla_ctx.decode_blocks(q, ptrs([k]), ptrs([v]), i32([n]), ids, 1, xb, 1, nh, n_kv, hd, br, f16_cache=t == "f16")
    ok(gla_ctx)
    want = v.view(n_kv, 1, hd).expand(n_kv, nh // n_kv, hd).reshape(nh, hd).double()
    tol = 0.0 if t == "f16" else 2.0 ** -23
    assert bool(((xb[0].double() - want).abs() <= tol * want.abs()).all())

"""What is measured of the long-cache operators: block bounds, batched RoPE + append, block
selection, attention over selected blocks, attention that adds up its weights, and eviction.

Every case names its operator ("op") and its sizes.  Sequences of one case have lengths between
"lo" and "hi", fixed by the case; all values come from the seed.  The caches are laid out as the
library lays them out, [position][kv_head][head_dim], one block of memory for each sequence.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
DT = {"f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # a prompt of 4096 rows has just been ingested into an FP32 cache of the 1B shape
        dict(name="bounds f32 1x4096", op="bounds", t="f32", batch=1, nh=32, nkv=8, hd=64, lo=4096, hi=4096, br=16),
        # sixteen prompts of uneven lengths, FP16 caches of the 8B shape
        dict(name="bounds f16 16x32768", op="bounds", t="f16", batch=16, nh=32, nkv=8, hd=128, lo=1024, hi=32768, br=64),
        # one new token of one sequence: the smallest call, all latency
        dict(name="append f32 1", op="append", t="f32", batch=1, nh=32, nkv=8, hd=64, cap=513, lo=511, hi=511, br=16, style=0),
        # a served batch whose caches were evicted: rows are far behind positions
        dict(name="append f16 96", op="append", t="f16", batch=96, nh=32, nkv=8, hd=128, cap=600, lo=1, hi=600, br=64, style=1),
        # one token over 128 Ki cached positions, 4 kv heads of 7 q heads
        dict(name="select f16 1x131072", op="select", t="f16", batch=1, nh=28, nkv=4, hd=128, lo=131072, hi=131072, br=64, nsel=64, first=1, last=2),
        # a served batch of uneven lengths, small blocks, FP32
        dict(name="select f32 16x32768", op="select", t="f32", batch=16, nh=32, nkv=8, hd=128, lo=1024, hi=32768, br=32, nsel=128, first=1, last=2),
        # one token reads 64 of 2048 blocks
        dict(name="blocks f16 1x131072", op="blocks", t="f16", batch=1, nh=28, nkv=4, hd=128, lo=131072, hi=131072, br=64, nsel=64, shared=False),
        # 256 prompt queries over one sequence's cache, each with blocks of its own
        dict(name="blocks f16 256 queries", op="blocks", t="f16", batch=256, nh=32, nkv=8, hd=128, lo=32768, hi=32768, br=64, nsel=32, shared=True),
        # one token over 128 Ki positions, the weights kept for eviction
        dict(name="weights f16 1x131072", op="weights", t="f16", batch=1, nh=28, nkv=4, hd=128, lo=131072, hi=131072),
        # a batch of short and odd lengths in FP32, head size 96, groups of 8
        dict(name="weights f32 16x8191", op="weights", t="f32", batch=16, nh=16, nkv=2, hd=96, lo=77, hi=8191),
        # a prompt's cache cut down to the decode budget
        dict(name="evict f32 1x4096", op="evict", t="f32", batch=1, nh=32, nkv=8, hd=64, lo=4096, hi=4096, keep=1024, recent=256),
        # a batch of long prompts cut down to theirs
        dict(name="evict f16 16x32768", op="evict", t="f16", batch=16, nh=32, nkv=8, hd=128, lo=1024, hi=32768, keep=4096, recent=512),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


#: head layouts drawn from: the library's benchmark shapes and its tests' ones
HEADS = [(32, 8, 64), (32, 8, 128), (28, 4, 128), (16, 2, 96), (8, 8, 128), (14, 2, 64), (16, 16, 96), (12, 4, 64)]


def draw(rng):
    op = rng.choice(["bounds", "append", "select", "blocks", "weights", "evict"])
    t = rng.choice(["f16", "f32"])
    nh, nkv, hd = rng.choice(HEADS)
    batch = _log_int(rng, 1, 64)
    row = nkv * hd * (2 if t == "f16" else 4)
    # the longest sequence: what keeps one tensor of keys at a quarter of a gigabyte at most
    most = max(64, min(131072, (1 << 28) // (row * batch)))
    hi = _log_int(rng, 1, most)
    lo = rng.choice([hi, 1, max(1, hi // 3)])
    br = rng.choice([16, 32, 64, 128])
    c = dict(op=op, t=t, batch=batch, nh=nh, nkv=nkv, hd=hd, lo=lo, hi=hi)
    if op == "bounds":
        c |= dict(br=br)
    elif op == "append":
        cap = _log_int(rng, 1, 1000)
        c |= dict(cap=cap, lo=1, hi=cap, br=br, style=rng.choice([0, 1]))
    elif op == "select":
        # fewer slots than the longest sequence has blocks, so that there is something to select
        hi = max(hi, 8 * br)
        first, last = rng.choice([0, 1, 2]), rng.choice([0, 1, 2])
        nsel = max(first + last + 1, _log_int(rng, 1, n_blocks(hi, br) // 2))
        c |= dict(br=br, hi=hi, lo=rng.choice([hi, 1, hi // 3]), nsel=nsel, first=first, last=last)
    elif op == "blocks":
        shared = rng.random() < 0.4
        nsel = _log_int(rng, 1, max(1, min(128, (1 << 28) // (row * br * batch))))
        c |= dict(br=br, nsel=nsel, shared=shared)
        if shared:
            c |= dict(lo=hi)
    elif op == "evict":
        keep = _log_int(rng, 1, max(1, hi))
        c |= dict(keep=keep, recent=rng.choice([0, keep // 8, keep // 2, keep]))
    return c


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def lengths(c):
    """The sequences' lengths: the longest is there, the others are spread between lo and hi."""
    r = random.Random("%(op)s %(t)s %(batch)d %(nh)d %(nkv)d %(hd)d %(lo)d %(hi)d" % c)
    if c["op"] == "blocks" and c["shared"]:  # queries of one prompt chunk, one position after another
        return [max(1, c["hi"] - c["batch"] + 1 + i) for i in range(c["batch"])]
    return [c["hi"]] + [r.randint(c["lo"], c["hi"]) for _ in range(c["batch"] - 1)]


def n_blocks(n, br):
    return -(-n // br)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def _keys(gen, seqs, rows, nkv, hd, dtype):
    """Keys as models have them: a mean and a spread of each channel's own, and a part that
    changes slowly along the sequence beside one of each row's own."""
    mean = _normal(gen, 1, 1, nkv, hd) * 0.5
    spread = torch.exp(_normal(gen, 1, 1, nkv, hd) * 0.5)
    slow = _normal(gen, seqs, -(-rows // 100) + 1, nkv, hd)
    out = torch.empty(seqs, rows, nkv, hd, dtype=dtype, device=DEV)
    for s in range(seqs):  # one sequence at a time: a batch in FP32 would take gigabytes beside it
        x = _normal(gen, rows, nkv, hd) * 0.7
        x += slow[s].repeat_interleave(100, dim=0)[:rows] * 0.7
        out[s] = x * spread[0] + mean[0]
    return out


def _ptrs(x):
    return torch.tensor([x[i].data_ptr() for i in range(x.shape[0])], dtype=torch.int64, device=DEV)


def prepare(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    op, dtype, b, nh, nkv, hd = c["op"], DT[c["t"]], c["batch"], c["nh"], c["nkv"], c["hd"]
    n = lengths(c)
    top = max(n)
    s = dict(c=c, n=torch.tensor(n, dtype=torch.int32, device=DEV), top=top)
    if op in ("select", "blocks", "weights"):
        s["q"] = _normal(gen, b, nh, hd)
    if op in ("select", "bounds"):
        k = _keys(gen, b, top, nkv, hd, dtype)
        nb = n_blocks(top, c["br"])
        if op == "bounds":
            s["k"], s["k_ptrs"] = k, _ptrs(k)
            s["bounds"] = torch.zeros(b, nb, nkv, 2, hd, dtype=dtype, device=DEV)
        else:
            pad = nb * c["br"] - top
            k = torch.cat([k, k[:, -1:].expand(-1, pad, -1, -1)], 1) if pad else k
            k = k.view(b, nb, c["br"], nkv, hd)
            s["bounds"] = torch.stack([k.amin(2), k.amax(2)], 3).contiguous()
            s["ids"] = torch.zeros(b, nkv, c["nsel"], dtype=torch.int32, device=DEV)
            del k
        s["bounds_ptrs"] = _ptrs(s["bounds"])
    elif op == "append":
        cap, br = c["cap"], c["br"]
        s["q0"], s["k0"], s["v0"] = _normal(gen, b, nh, hd), _normal(gen, b, nkv, hd), _normal(gen, b, nkv, hd)
        s["q"] = torch.empty_like(s["q0"])
        s["k"] = _normal(gen, b, cap, nkv, hd).to(dtype)
        s["v"] = _normal(gen, b, cap, nkv, hd).to(dtype)
        s["rows"] = s["n"] - 1
        far = torch.randint(0, 131072, (b,), generator=gen, device=DEV, dtype=torch.int32)
        s["pos"] = torch.maximum(s["rows"], far)
        nb = n_blocks(cap, br)
        # the bounds of the rows that each sequence has; later blocks hold what was there before
        at = torch.arange(nb * br, device=DEV).clamp(max=cap - 1)
        live = (torch.arange(nb * br, device=DEV)[None] < s["rows"][:, None])[:, :, None, None]
        kk = s["k"][:, at].float()
        lo = torch.where(live, kk, math.inf).view(b, nb, br, nkv, hd).amin(2)
        hi = torch.where(live, kk, -math.inf).view(b, nb, br, nkv, hd).amax(2)
        bo = torch.stack([lo, hi], 3)
        s["bounds"] = torch.where(bo.isfinite(), bo, 0.0).to(dtype).contiguous()
        s["bounds_ptrs"], s["k_ptrs"], s["v_ptrs"] = _ptrs(s["bounds"]), _ptrs(s["k"]), _ptrs(s["v"])
    elif op in ("blocks", "weights", "evict"):
        seqs = 1 if c.get("shared") else b
        s["k"] = _keys(gen, seqs, top, nkv, hd, dtype)
        s["v"] = torch.empty(seqs, top, nkv, hd, dtype=dtype, device=DEV)
        for i in range(seqs):
            s["v"][i] = _normal(gen, top, nkv, hd)
        s["seq"] = torch.zeros(b, dtype=torch.int64, device=DEV) if seqs == 1 else torch.arange(b, device=DEV)
        s["k_ptrs"], s["v_ptrs"] = _ptrs(s["k"])[s["seq"]].contiguous(), _ptrs(s["v"])[s["seq"]].contiguous()
        if op != "evict":
            s["xb"] = torch.empty(b, nh, hd, device=DEV)
        if op == "blocks":
            # what a selection gives: the newest block, others by chance, in order, then -1
            nb = n_blocks(s["n"], c["br"])
            r = torch.rand(b, nkv, n_blocks(top, c["br"]), generator=gen, device=DEV)
            j = torch.arange(r.shape[2], device=DEV)
            r = torch.where(j == nb[:, None, None] - 1, 2.0, torch.where(j < nb[:, None, None], r, -1.0))
            ids = r.argsort(dim=2, descending=True)[:, :, : c["nsel"]]
            ids = torch.where(ids < nb[:, None, None], ids, 1 << 30).sort(dim=2)[0]
            ids = torch.where(ids < 1 << 30, ids, -1).int()
            s["ids"] = torch.full((b, nkv, c["nsel"]), -1, dtype=torch.int32, device=DEV)
            s["ids"][:, :, : ids.shape[2]] = ids
        else:
            # what earlier tokens gave: most rows little, a few much, some nothing at all
            w = torch.exp(_normal(gen, b, nkv, top) * 2 - 4)
            w = torch.where(torch.rand(b, nkv, top, generator=gen, device=DEV) < 0.05, 0.0, w)
            s["w"] = w.contiguous()
            s["w_ptrs"] = _ptrs(s["w"])
        if op == "evict":
            s["kept"] = torch.empty(b, nkv, c["keep"], dtype=torch.int32, device=DEV)
            s["ko"] = torch.zeros(b, c["keep"], nkv, hd, dtype=dtype, device=DEV)
            s["vo"] = torch.zeros_like(s["ko"])
            s["wo"] = torch.zeros(b, nkv, c["keep"], device=DEV)
            s["ko_ptrs"], s["vo_ptrs"], s["wo_ptrs"] = _ptrs(s["ko"]), _ptrs(s["vo"]), _ptrs(s["wo"])
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
THETA = 500000.0
_CTX = []


def _ctx():
    """The library's context of this process: a program makes it once."""
    if not _CTX:
        sys.path.insert(0, os.path.join(os.getcwd(), "gpullama3.java_b200"))
        import gpullama_attn

        _CTX.append(gpullama_attn.Context(0, torch.cuda.current_stream().cuda_stream))
    return _CTX[0]


def run(s):
    c = s["c"]
    return (globals()["own_" + c["op"]] if own else globals()["plain_" + c["op"]])(s, c)


def own_bounds(s, c):
    _ctx().block_bounds(s["k_ptrs"], s["n"], s["top"], s["bounds_ptrs"], c["batch"], c["nkv"], c["hd"], c["br"],
                        f16_cache=c["t"] == "f16")
    return {"bounds": s["bounds"]}


def own_append(s, c):
    _ctx().rope_append_batched(s["q0"], s["k0"], s["v0"], s["q"], s["k_ptrs"], s["v_ptrs"], s["pos"], c["batch"], c["nh"],
                               c["nkv"], c["hd"], c["cap"], THETA, style=c["style"], rows=s["rows"],
                               bounds_ptrs=s["bounds_ptrs"], block_rows=c["br"], f16_cache=c["t"] == "f16")
    return {"q": s["q"], "keys": s["k"], "values": s["v"], "bounds": s["bounds"]}


def own_select(s, c):
    _ctx().block_select(s["q"], s["bounds_ptrs"], s["n"], s["top"], s["ids"], c["batch"], c["nh"], c["nkv"], c["hd"], c["br"],
                        c["nsel"], n_first=c["first"], n_last=c["last"], f16_cache=c["t"] == "f16")
    return {"ids": s["ids"]}


def own_blocks(s, c):
    _ctx().decode_blocks(s["q"], s["k_ptrs"], s["v_ptrs"], s["n"], s["ids"], c["nsel"], s["xb"], c["batch"], c["nh"], c["nkv"],
                         c["hd"], c["br"], f16_cache=c["t"] == "f16")
    return {"xb": s["xb"]}


def own_weights(s, c):
    _ctx().decode_weights(s["q"], s["k_ptrs"], s["v_ptrs"], s["n"], s["top"], s["xb"], s["w_ptrs"], s["top"], c["batch"],
                          c["nh"], c["nkv"], c["hd"], f16_cache=c["t"] == "f16")
    return {"xb": s["xb"], "weights": s["w"]}


def own_evict(s, c):
    _ctx().kv_evict(s["k_ptrs"], s["v_ptrs"], s["w_ptrs"], s["top"], s["n"], s["top"], c["keep"], c["recent"], s["kept"],
                    c["batch"], c["nkv"], c["hd"], k_out_ptrs=s["ko_ptrs"], v_out_ptrs=s["vo_ptrs"],
                    weight_out_ptrs=s["wo_ptrs"], weight_out_stride=c["keep"], f16_cache=c["t"] == "f16")
    return {"kept": s["kept"], "keys": s["ko"], "values": s["vo"], "weights": s["wo"]}


# the plain forms -----------------------------------------------------------------------------
def plain_bounds(s, c):
    """bounds[j][g][0 | 1] = the smallest | largest key of each channel over the rows of block j."""
    k, br = s["k"], c["br"]
    b, top, nkv, hd = k.shape
    nb = n_blocks(top, br)
    at = torch.arange(nb * br, device=DEV)
    live = (at[None] < s["n"][:, None])[:, :, None, None]
    kk = k[:, at.clamp(max=top - 1)].float()
    lo = torch.where(live, kk, math.inf).view(b, nb, br, nkv, hd).amin(2)
    hi = torch.where(live, kk, -math.inf).view(b, nb, br, nkv, hd).amax(2)
    got = torch.stack([lo, hi], 3)
    there = (torch.arange(nb, device=DEV)[None] < n_blocks(s["n"], br)[:, None])[:, :, None, None, None]
    s["bounds"].copy_(torch.where(there, got.to(k.dtype), s["bounds"]))
    return {"bounds": s["bounds"]}


def _rotated(x, pos, style):
    """RoPE as this library has it: the frequency and the angle are FP32 numbers (they define the
    rotation), the cosine and sine are taken in 64 bits and rounded, products and sums in FP32."""
    hd = x.shape[-1]
    i = torch.arange(hd // 2, device=DEV, dtype=torch.float64)
    freq = (1.0 / torch.pow(torch.tensor(THETA, dtype=torch.float64, device=DEV), 2 * i / hd)).float()
    ang = (pos.float()[:, None] * freq[None]).double()
    cs, sn = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]
    x0, x1 = (x[..., 0::2], x[..., 1::2]) if style == 0 else (x[..., : hd // 2], x[..., hd // 2:])
    y0, y1 = x0 * cs - x1 * sn, x0 * sn + x1 * cs
    return torch.stack([y0, y1], -1).flatten(-2) if style == 0 else torch.cat([y0, y1], -1)


def plain_append(s, c):
    s["q"].copy_(_rotated(s["q0"], s["pos"], c["style"]))
    at, rows = torch.arange(c["batch"], device=DEV), s["rows"].long()
    s["k"][at, rows] = _rotated(s["k0"], s["pos"], c["style"]).to(s["k"].dtype)
    s["v"][at, rows] = s["v0"].to(s["v"].dtype)
    blk = rows // c["br"]
    new, old = s["k"][at, rows], s["bounds"][at, blk]
    fresh = (rows % c["br"] == 0)[:, None, None]
    s["bounds"][at, blk] = torch.stack([torch.where(fresh, new, torch.minimum(old[:, :, 0], new)),
                                        torch.where(fresh, new, torch.maximum(old[:, :, 1], new))], 2)
    return {"q": s["q"], "keys": s["k"], "values": s["v"], "bounds": s["bounds"]}


def plain_select(s, c):
    """A block's score is the largest over its kv head's q heads of sum_d max(q_d lo_d, q_d hi_d), in
    64 bits (what is next to the border decides); the nsel best, ties to the lowest, in order."""
    b, nb, nkv, _, hd = s["bounds"].shape
    q = s["q"].view(b, nkv, -1, hd).double()
    bo = s["bounds"].double()
    score = torch.matmul(q.clamp(max=0), bo[:, :, :, 0].permute(0, 2, 3, 1))
    score += torch.matmul(q.clamp(min=0), bo[:, :, :, 1].permute(0, 2, 3, 1))
    score = score.amax(2)
    n = n_blocks(s["n"], c["br"])[:, None, None]
    j = torch.arange(nb, device=DEV)
    score = torch.where((j < c["first"]) | (j >= n - c["last"]), math.inf, score)
    score = torch.where(j < n, score, -math.inf)
    ids = score.sort(dim=2, descending=True, stable=True)[1][:, :, : c["nsel"]]
    ids = torch.where(ids < n, ids, 1 << 30).sort(dim=2)[0]
    ids = torch.where(ids < 1 << 30, ids, -1).int()
    s["ids"].fill_(-1)
    s["ids"][:, :, : ids.shape[2]] = ids
    return {"ids": s["ids"]}


def _softmax(score, live):
    score = torch.where(live, score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, p / total, 0.0)


def plain_blocks(s, c):
    b, nh, hd = s["q"].shape
    nkv, br = c["nkv"], c["br"]
    ids = s["ids"].long()
    rows = (ids[..., None] * br + torch.arange(br, device=DEV)).flatten(2)
    live = (ids >= 0)[..., None].expand(-1, -1, -1, br).flatten(2) & (rows < s["n"][:, None, None])
    rows = torch.where(live, rows, 0)
    at = (s["seq"][:, None, None], rows, torch.arange(nkv, device=DEV)[None, :, None])
    q = s["q"].view(b, nkv, nh // nkv, hd)
    score = torch.matmul(q, s["k"][at].float().transpose(2, 3)) / math.sqrt(hd)
    p = _softmax(score, live[:, :, None])
    s["xb"].copy_(torch.matmul(p, s["v"][at].float()).view(b, nh, hd))
    return {"xb": s["xb"]}


def plain_weights(s, c):
    b, nh, hd = s["q"].shape
    nkv = c["nkv"]
    q = s["q"].view(b, nkv, nh // nkv, hd)
    live = (torch.arange(s["top"], device=DEV)[None] < s["n"][:, None])[:, None, None]
    score = torch.matmul(q, s["k"].float().permute(0, 2, 3, 1)) / math.sqrt(hd)
    p = _softmax(score, live)
    s["xb"].copy_(torch.matmul(p, s["v"].float().transpose(1, 2)).view(b, nh, hd))
    s["w"].add_(p.sum(2))
    return {"xb": s["xb"], "weights": s["w"]}


def plain_evict(s, c):
    """The newest `recent` rows stay, and the others of the largest weight (ties to the lowest)."""
    keep, n = c["keep"], s["n"].long()[:, None, None]
    b, top, nkv, hd = s["k"].shape
    j = torch.arange(top, device=DEV)
    w = torch.where(j >= n - c["recent"], math.inf, s["w"])
    w = torch.where(j < n, w, -math.inf)
    kept = w.sort(dim=2, descending=True, stable=True)[1][:, :, :keep]
    kept = torch.where(kept < n, kept, 1 << 30).sort(dim=2)[0]
    live = kept < 1 << 30
    at = torch.where(live, kept, 0)
    sb, sg = torch.arange(b, device=DEV)[:, None, None], torch.arange(nkv, device=DEV)[None, :, None]
    m = kept.shape[2]
    here = live.transpose(1, 2)[..., None]
    s["kept"].fill_(-1)
    s["kept"][:, :, :m] = torch.where(live, kept, -1).int()
    s["ko"][:, :m] = torch.where(here, s["k"][sb, at, sg].transpose(1, 2), s["ko"][:, :m])
    s["vo"][:, :m] = torch.where(here, s["v"][sb, at, sg].transpose(1, 2), s["vo"][:, :m])
    s["wo"][:, :, :m] = torch.where(live, s["w"][sb, sg, at], s["wo"][:, :, :m])
    return {"kept": s["kept"], "keys": s["ko"], "values": s["vo"], "weights": s["wo"]}


# ---------------------------------------------------------------------------------------------
# work: each input read once, each output written once
# ---------------------------------------------------------------------------------------------
def work(c):
    e = 2 if c["t"] == "f16" else 4
    b, nh, nkv, hd, n = c["batch"], c["nh"], c["nkv"], c["hd"], lengths(c)
    row, rows = nkv * hd * e, sum(n)
    if c["op"] == "bounds":
        nb = sum(n_blocks(x, c["br"]) for x in n)
        return {"bytes": rows * row + nb * 2 * row, "flops": 2 * rows * nkv * hd}
    if c["op"] == "append":
        token = 4 * hd * (2 * nh + 2 * nkv) + 2 * row + 4 * row
        return {"bytes": b * token, "flops": b * (nh + nkv) * hd * 3}
    if c["op"] == "select":
        nb = sum(n_blocks(x, c["br"]) for x in n)
        return {"bytes": 4 * b * nh * hd + nb * 2 * row + 4 * b * nkv * c["nsel"], "flops": 4 * nb * nh * hd}
    if c["op"] == "blocks":
        read = sum(min(x, c["nsel"] * c["br"]) for x in n)
        distinct = min(read, max(n)) if c["shared"] else read
        return {"bytes": 8 * b * nh * hd + 2 * distinct * row + 4 * b * nkv * c["nsel"], "flops": 4 * read * nh * hd}
    if c["op"] == "weights":
        return {"bytes": 8 * b * nh * hd + 2 * rows * row + 8 * rows * nkv, "flops": 4 * rows * nh * hd}
    kept = sum(min(x, c["keep"]) for x in n)
    return {"bytes": 4 * nkv * rows + 4 * kept * row + 8 * kept * nkv, "flops": 0}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits, one sequence at a time
# ---------------------------------------------------------------------------------------------
def exact(c, seed):
    s = prepare(c, seed)
    return globals()["exact_" + c["op"]](s, c)


def exact_bounds(s, c):
    out = s["bounds"].double()
    for i, n in enumerate(lengths(c)):
        for lo, hi in ((0, n // c["br"]), (n // c["br"], n_blocks(n, c["br"]))):
            if hi > lo:
                x = s["k"][i, lo * c["br"]: min(n, hi * c["br"])].double()
                x = x.view(hi - lo, -1, c["nkv"], c["hd"])
                out[i, lo:hi, :, 0], out[i, lo:hi, :, 1] = x.min(dim=1)[0], x.max(dim=1)[0]
    return {"bounds": out}


def exact_append(s, c):
    hd, keys, values, bounds = c["hd"], s["k"].double(), s["v"].double(), s["bounds"].double()
    q, k = s["q0"].double(), s["k0"].double()
    first = torch.arange(0, hd, 2) if c["style"] == 0 else torch.arange(hd // 2)
    second = first + (1 if c["style"] == 0 else hd // 2)
    freq = torch.tensor([1.0 / THETA ** (2 * i / hd) for i in range(hd // 2)]).float()
    ang = (s["pos"].cpu().float()[:, None] * freq).double().to(DEV)[:, None]
    turn = torch.polar(torch.ones_like(ang), ang)
    for x in (q, k):
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
    for i, n in enumerate(lengths(c)):
        r, j = n - 1, (n - 1) // c["br"]
        keys[i, r], values[i, r] = k[i], s["v0"][i].double()
        new = k[i][:, None].expand(-1, 2, -1)
        if r % c["br"]:
            new = torch.stack([torch.minimum(bounds[i, j, :, 0], k[i]), torch.maximum(bounds[i, j, :, 1], k[i])], 1)
        bounds[i, j] = new
    return {"q": q, "keys": keys, "values": values, "bounds": bounds}


def exact_select(s, c):
    out = torch.full((c["batch"], c["nkv"], c["nsel"]), -1, dtype=torch.int32)
    for i, n in enumerate(lengths(c)):
        nb = n_blocks(n, c["br"])
        for g in range(c["nkv"]):
            q = s["q"][i].view(c["nkv"], -1, c["hd"])[g].double()
            lo, hi = s["bounds"][i, :nb, g, 0].double(), s["bounds"][i, :nb, g, 1].double()
            top = torch.stack([torch.maximum(x * lo, x * hi).sum(1) for x in q]).max(dim=0)[0].tolist()
            must = [j for j in range(nb) if j < c["first"] or j >= nb - c["last"]]
            rest = sorted(set(range(nb)) - set(must), key=lambda j: (-top[j], j))
            ids = sorted((must + rest)[: c["nsel"]])
            out[i, g, : len(ids)] = torch.tensor(ids, dtype=torch.int32)
    return {"ids": out}


def _attend(q, k, v, hd):
    """The weights and the sums of one kv head's q heads over rows k, v, in 64 bits."""
    z = (q.double() @ k.double().T) * hd ** -0.5
    w = torch.exp(z - torch.logsumexp(z, dim=1, keepdim=True))
    return w, w @ v.double()


def exact_blocks(s, c):
    if c["batch"] * c["nkv"] > 4096:
        return None
    out = torch.zeros(c["batch"], c["nh"], c["hd"], dtype=torch.float64, device=DEV)
    seq, ids, grp = s["seq"].tolist(), s["ids"].tolist(), c["nh"] // c["nkv"]
    for i, n in enumerate(lengths(c)):
        for g in range(c["nkv"]):
            rows = [r for j in ids[i][g] if j >= 0 for r in range(j * c["br"], min(n, (j + 1) * c["br"]))]
            if rows:
                at = torch.tensor(rows, device=DEV)
                o = _attend(s["q"][i, g * grp: (g + 1) * grp], s["k"][seq[i], at, g], s["v"][seq[i], at, g], c["hd"])[1]
                out[i, g * grp: (g + 1) * grp] = o
    return {"xb": out}


def exact_weights(s, c):
    out = torch.zeros(c["batch"], c["nh"], c["hd"], dtype=torch.float64, device=DEV)
    w, grp = s["w"].double(), c["nh"] // c["nkv"]
    for i, n in enumerate(lengths(c)):
        for g in range(c["nkv"]):
            p, o = _attend(s["q"][i, g * grp: (g + 1) * grp], s["k"][i, :n, g], s["v"][i, :n, g], c["hd"])
            out[i, g * grp: (g + 1) * grp] = o
            w[i, g, :n] += p.sum(0)
    return {"xb": out, "weights": w}


def exact_evict(s, c):
    out = {k: s[k].clone() for k in ("ko", "vo", "wo")}
    kept = torch.full((c["batch"], c["nkv"], c["keep"]), -1, dtype=torch.int32)
    w = s["w"].cpu().tolist()
    for i, n in enumerate(lengths(c)):
        for g in range(c["nkv"]):
            old = max(0, n - c["recent"])
            best = sorted(range(old), key=lambda j: (-w[i][g][j], j))[: max(0, c["keep"] - (n - old))]
            rows = sorted(best) + list(range(old, n))
            kept[i, g, : len(rows)] = torch.tensor(rows, dtype=torch.int32)
            at = torch.tensor(rows, device=DEV)
            out["ko"][i, : len(rows), g], out["vo"][i, : len(rows), g] = s["k"][i, at, g], s["v"][i, at, g]
            out["wo"][i, g, : len(rows)] = s["w"][i, g, at]
    return {"kept": kept, "keys": out["ko"].double(), "values": out["vo"].double(), "weights": out["wo"].double()}

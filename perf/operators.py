"""Workloads of the 8-bit serving operators: keys and values appended to a paged cache of 8-bit elements, attention over that cache, and
products with 8-bit matrices that have a scale for each block of 128.  Every case is one pass as a serving program makes it.

Kinds of case:
  append  : rows of keys and values, rotated on the way, appended to the pages of a ragged batch (kx_paged_append), and what the blocks that
            they touch then stand for, as a program that hands a prefix on reads it back (kx_paged_read)
  attend  : the newest positions of a ragged batch attend to the pages of their sequences (kx_paged_attend)
  product : rows of activations times a matrix of 8-bit elements (kx_fp8_run)

Where `own` is false the same is computed from elementary torch operations.  The cache is the program's memory in both forms: keys
[pages][kv_heads][page][dp], values [pages][kv_heads][page / 64][vp][64] with the 64 tokens in the order of _order(), a scale 2^e for each block of
tokens and head.  Positions that no sequence has reached hold NaN.

Weights, activations and cached rows are random, made from the seed; lengths of ragged batches go by the case alone.
"""
import ctypes as C
import math
import random

import torch

own = False

LEAST, MOST = -100, 448.0   # smallest exponent of a scale; largest element


def listed():
    return [
        # one token of one interactive session: what every step pays per layer
        {"name": "append 1", "kind": "append", "heads": 64, "kv": 8, "dim": 128, "vdim": 128, "rot": 128, "pairs": 0, "page": 64, "block": 32, "batch": 1, "longest": 4001, "new": 1},
        # a step of a served batch of sequences of different lengths
        {"name": "append 64", "kind": "append", "heads": 64, "kv": 8, "dim": 128, "vdim": 128, "rot": 64, "pairs": 1, "page": 128, "block": 64, "batch": 64, "longest": 8192, "new": 1},
        # prompts of several sequences at once, some with a cached prefix
        {"name": "append prompts", "kind": "append", "heads": 64, "kv": 8, "dim": 128, "vdim": 128, "rot": 128, "pairs": 0, "page": 64, "block": 32, "batch": 6, "longest": 6000, "new": 2048},
        # one token of a small model's session
        {"name": "attend 1 x 4096", "kind": "attend", "heads": 16, "kv": 4, "dim": 128, "vdim": 128, "rot": 128, "pairs": 0, "page": 64, "block": 32, "size": 0, "f32": False,
         "batch": 1, "longest": 4096, "new": 1},
        # one token of a session with a long document
        {"name": "attend 1 x 131072", "kind": "attend", "heads": 64, "kv": 8, "dim": 128, "vdim": 128, "rot": 128, "pairs": 0, "page": 256, "block": 64, "size": 0, "f32": False,
         "batch": 1, "longest": 131072, "new": 1},
        # a step of a served batch of sequences of different lengths
        {"name": "attend 64 x 8192", "kind": "attend", "heads": 64, "kv": 8, "dim": 128, "vdim": 128, "rot": 128, "pairs": 0, "page": 64, "block": 32, "size": 0, "f32": False,
         "batch": 64, "longest": 8192, "new": 1},
        # pieces of prompts behind cached prefixes
        {"name": "attend prompts", "kind": "attend", "heads": 32, "kv": 8, "dim": 128, "vdim": 128, "rot": 128, "pairs": 0, "page": 64, "block": 64, "size": 0, "f32": False,
         "batch": 4, "longest": 5000, "new": 777},
        # drafted tokens in the 32-bit format, as it is used to check bf16 results, in a layer with a window
        {"name": "attend drafts f32", "kind": "attend", "heads": 16, "kv": 2, "dim": 192, "vdim": 128, "rot": 64, "pairs": 1, "page": 128, "block": 16, "size": 1000, "f32": True,
         "batch": 5, "longest": 3001, "new": 5},
        # one token through the latent projections of Kimi-K2
        {"name": "product 1", "kind": "product", "tokens": 1, "rows": 2112, "cols": 7168, "x_f32": False, "out_f32": False},
        # a served batch through its output projection
        {"name": "product 24", "kind": "product", "tokens": 24, "rows": 7168, "cols": 8192, "x_f32": False, "out_f32": False},
        # a prefill step through its dense layer
        {"name": "product 2048", "kind": "product", "tokens": 2048, "rows": 18432, "cols": 7168, "x_f32": False, "out_f32": False},
        # a short prompt through a matrix of odd size, 32-bit rows in and out as the hybrid decoder's steps have them
        {"name": "product 333 f32", "kind": "product", "tokens": 333, "rows": 4103, "cols": 2000, "x_f32": True, "out_f32": True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "product", "product"])
    if kind == "product":
        tokens = rng.choice([1, _log(rng, 1, 16), _log(rng, 5, 64), _log(rng, 33, 2048)])
        return {"kind": kind, "tokens": tokens, "rows": _log(rng, 128, 18432), "cols": 8 * _log(rng, 64, 896), "x_f32": rng.random() < 0.3, "out_f32": rng.random() < 0.3}
    kv = rng.choice([1, 2, 4, 8])
    dim, vdim = rng.choice([(64, 64), (80, 80), (96, 96), (128, 128), (128, 128), (192, 128), (256, 256)])
    c = {"kind": kind, "heads": kv * rng.choice([1, 2, 3, 4, 5, 8, 16]), "kv": kv, "dim": dim, "vdim": vdim, "rot": rng.choice([0, dim // 2, dim]), "pairs": rng.randint(0, 1),
         "page": rng.choice([64, 128, 256]), "block": rng.choice([16, 32, 64])}
    if kind == "append":
        batch = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 12000 // batch)
        return {**c, "batch": batch, "longest": new + _log(rng, 1, 12000), "new": new}
    c["size"], c["f32"] = rng.choice([0, 0, _log(rng, 50, 4000)]), rng.random() < 0.25
    if rng.random() < 0.6:
        batch = _log(rng, 1, 64)
        new = rng.choice([1, 1, 1, rng.randint(2, 8)])
        return {**c, "batch": batch, "longest": new + _log(rng, 1, min(131072, 400000 // batch)), "new": new}
    batch = _log(rng, 1, 6)
    new = _log(rng, 9, 2000 // batch)
    return {**c, "batch": batch, "longest": new + _log(rng, 1, 6000), "new": new}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _lengths(case):
    """Positions of each sequence, the new ones among them, and how many are new."""
    rng = random.Random("%(batch)d %(longest)d %(new)d" % case)
    n = [case["longest"]] + [rng.randint(max(1, case["longest"] // 8), case["longest"]) for _ in range(case["batch"] - 1)]
    new = [case["new"]] + [rng.randint((case["new"] + 1) // 2, case["new"]) for _ in range(case["batch"] - 1)]
    return n, [min(a, b) for a, b in zip(n, new)]


def _pad(n, to):
    return -(-n // to) * to


def _widths(case):
    """Elements of a cached row of keys and of values: those of the smallest tile that holds both."""
    return next(t for t in ((64, 64), (128, 128), (192, 128), (256, 256)) if case["dim"] <= t[0] and case["vdim"] <= t[1])


def _order():
    """The token of each place in a group of 64 of cached values."""
    return [32 * h + 16 * r + 4 * q + j for q in range(4) for h in range(2) for r in range(2) for j in range(4)]


def _exponent(x):
    """The least e with x <= 448 * 2^e."""
    m, e = torch.frexp(x)
    return (e - 9 + (m > 0.875)).clamp_min(LEAST)


def _cache(case, g, held):
    """Pages that hold the first held[b] positions of sequence b."""
    n, _ = _lengths(case)
    page, block, kv, (dp, vp) = case["page"], case["block"], case["kv"], _widths(case)
    per = [-(-a // page) for a in n]
    total, most = sum(per), max(per)
    place = torch.randperm(total, generator=g, device="cuda")
    ids = [[sum(per[:b]) + i if i < per[b] else -1 for i in range(most)] for b in range(case["batch"])]
    ids = torch.tensor(ids, device="cuda")
    table = torch.where(ids >= 0, place[ids.clamp_min(0)], -1).to(torch.int32)
    valid = torch.zeros((total, page), dtype=torch.bool, device="cuda")
    at = torch.arange(most * page, device="cuda").view(1, most, page)
    there = at < torch.tensor(held, device="cuda").view(-1, 1, 1)
    valid[place[ids[ids >= 0]]] = there[ids >= 0]

    def rows(dim, to):
        x = _randn(g, total, kv, page, dim) * torch.exp(0.5 * _randn(g, kv, 1, dim))
        x *= valid[:, None, :, None]
        e = _exponent(x.view(total, kv, page // block, block * dim).abs().amax(3))
        x = torch.ldexp(x.view(total, kv, page // block, block, dim), -e[..., None, None]).view(total, kv, page, dim)
        c = torch.zeros((total, kv, page, to), dtype=torch.uint8, device="cuda")
        c[..., :dim] = x.to(torch.float8_e4m3fn).view(torch.uint8)
        c.masked_fill_(~valid[:, None, :, None], 0x7f)
        return c, torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)

    k, ks = rows(case["dim"], dp)
    v, vs = rows(case["vdim"], vp)
    v = v.view(total, kv, page // 64, 64, vp)[:, :, :, _order()].transpose(3, 4).contiguous()
    return {"k": k, "v": v, "ks": ks, "vs": vs, "table": table}


def _ragged(pos, new):
    """What tells the rows of a ragged batch apart: sequence b has rows start[b] to start[b + 1] - 1 at positions from pos[b] on."""
    start = [sum(new[:b]) for b in range(len(new) + 1)]
    b = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    i = (torch.arange(start[-1]) - torch.repeat_interleave(torch.tensor(start[:-1]), torch.tensor(new))).cuda()
    return {"start": torch.tensor(start, dtype=torch.int32, device="cuda"), "pos": torch.tensor(pos, dtype=torch.int32, device="cuda"), "b": b, "i": i,
            "at": torch.tensor(pos, device="cuda")[b] + i, "tokens": start[-1], "batch": len(new), "most": max(new), "longest": max(p + n for p, n in zip(pos, new))}


class _Held:
    """A handle of the library that goes back when the state does."""

    def __init__(self, handle, destroy):
        self.h, self._destroy = handle, destroy

    def __del__(self):
        try:
            self._destroy(self.h)
        except Exception:
            pass


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _inputs(case, seed):
    g = _generator(seed)
    if case["kind"] == "product":
        t, r, c = case["tokens"], case["rows"], case["cols"]
        x = _randn(g, t, c) * torch.exp(0.5 * _randn(g, c))
        w = torch.zeros((_pad(r, 128), _pad(c, 128)), device="cuda")
        w[:r, :c] = _randn(g, r, c) * c ** -0.5
        blocks = w.view(_pad(r, 128) // 128, 128, _pad(c, 128) // 128, 128)
        scale = blocks.abs().amax((1, 3)).clamp_min(1e-12) / MOST * torch.exp2(torch.rand((blocks.shape[0], blocks.shape[2]), generator=g, device="cuda"))
        w = (blocks / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(_pad(r, 128), _pad(c, 128))[:r].contiguous()
        return {"case": case, "x": x if case["x_f32"] else x.to(torch.bfloat16), "w": w, "scale": scale,
                "out": torch.empty((t, r), dtype=torch.float32 if case["out_f32"] else torch.bfloat16, device="cuda")}
    n, new = _lengths(case)
    pos = [a - b for a, b in zip(n, new)]
    append = case["kind"] == "append"
    s = {"case": case, "rows": _ragged(pos, new), "cache": _cache(case, g, pos if append else n)}
    t, kv, d, dv = s["rows"]["tokens"], case["kv"], case["dim"], case["vdim"]
    if append:   # keys and values lie side by side in rows of projections, behind the queries; tokens differ in size, so that scales grow
        s["proj"] = _randn(g, t, case["heads"] * d + kv * (d + dv)) * torch.exp(0.5 * _randn(g, t, 1))
        s["off"] = (case["heads"] * d, case["heads"] * d + kv * d)
        first = [p // case["block"] * case["block"] for p in pos]
        s["back"] = _ragged(first, [a - b for a, b in zip(n, first)])
        m = s["back"]["tokens"]
        s["out"] = [torch.empty((m, kv, w), dtype=torch.bfloat16, device="cuda") for w in (d, dv)]
    else:
        s["proj"] = 2.0 * _randn(g, t, case["heads"] * d)
        s["out"] = torch.empty((t, case["heads"], dv), dtype=torch.float32 if case["f32"] else torch.bfloat16, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:   # what a program keeps beside its tensors: a handle with the operator's scratch
        from blok_amd.lib import KxFp8Args, KxPagedCache, KxPagedConfig, KxPagedRows, check, kx
        lib, h = kx(), C.c_void_p()
        if case["kind"] == "product":
            check(lib.kx_fp8_create(case["tokens"], case["cols"], C.byref(h)))
            s["held"] = _Held(h, lib.kx_fp8_destroy)
            s["args"] = KxFp8Args(x_f32=case["x_f32"], out_f32=case["out_f32"], tokens=case["tokens"], rows=case["rows"], cols=case["cols"], ld=s["w"].shape[1], x_ld=case["cols"],
                                  out_ld=case["rows"], d_w=s["w"].data_ptr(), d_w_scale=s["scale"].data_ptr(), d_x=s["x"].data_ptr(), d_out=s["out"].data_ptr())
            return s
        cfg = KxPagedConfig(heads=case["heads"], kv_heads=case["kv"], dim=case["dim"], vdim=case["vdim"], page=case["page"], block=case["block"], rot=case["rot"],
                            pairs=case["pairs"], size=case.get("size", 0), scale=case["dim"] ** -0.5, base=10000.0)
        check(lib.kx_paged_create(C.byref(cfg), None, int(case.get("f32", False)), case["batch"], s["rows"]["tokens"], C.byref(h)))
        s["held"] = _Held(h, lib.kx_paged_destroy)
        c = s["cache"]
        s["kx_cache"] = KxPagedCache(d_k=c["k"].data_ptr(), d_v=c["v"].data_ptr(), d_k_scale=c["ks"].data_ptr(), d_v_scale=c["vs"].data_ptr(), d_table=c["table"].data_ptr(),
                                     pages=c["k"].shape[0], table_ld=c["table"].shape[1])
        for name in ("rows", "back"):
            if name in s:
                r = s[name]
                s["kx_" + name] = KxPagedRows(d_start=r["start"].data_ptr(), d_pos=r["pos"].data_ptr(), batch=r["batch"], tokens=r["tokens"], longest=r["longest"])
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "product": _own_product}[kind](s)
    return {"append": _plain_append, "attend": _plain_attend, "product": _plain_product}[kind](s)


def _own_append(s):
    from blok_amd.lib import check, kx
    case, (k, v), st = s["case"], s["out"], _stream()
    check(kx().kx_paged_append(s["held"].h, C.byref(s["kx_cache"]), C.byref(s["kx_rows"]), s["proj"].data_ptr(), s["proj"].shape[1], s["off"][0], s["off"][1], st))
    check(kx().kx_paged_read(s["held"].h, C.byref(s["kx_cache"]), C.byref(s["kx_back"]), k.data_ptr(), case["kv"] * case["dim"], v.data_ptr(), case["kv"] * case["vdim"], st))
    return k, v


def _own_attend(s):
    from blok_amd.lib import check, kx
    case = s["case"]
    check(kx().kx_paged_attend(s["held"].h, C.byref(s["kx_cache"]), C.byref(s["kx_rows"]), s["proj"].data_ptr(), s["proj"].shape[1], 0, s["out"].data_ptr(),
                               case["heads"] * case["vdim"], _stream()))
    return s["out"]


def _own_product(s):
    from blok_amd.lib import check, kx
    check(kx().kx_fp8_run(s["held"].h, C.byref(s["args"]), _stream()))
    return s["out"]


def _turned(case, x, at):
    """x [rows][heads][dim] of 64-bit numbers, its first rot dimensions turned in pairs by the rows' positions."""
    rot = case["rot"]
    if not rot:
        return x
    angle = at.double()[:, None, None] * 10000.0 ** (torch.arange(rot // 2, device="cuda", dtype=torch.float64) * (-2.0 / rot))
    c, s = angle.cos(), angle.sin()
    if case["pairs"]:
        p = x[..., :rot].unflatten(-1, (-1, 2))
        turned = torch.stack((p[..., 0] * c - p[..., 1] * s, p[..., 0] * s + p[..., 1] * c), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _rounded(x):
    """The nearest 8-bit elements to 64-bit numbers of at most 448, ties to even."""
    step = torch.frexp(x.abs().clamp_min(2.0 ** -6))[1] - 4
    return torch.ldexp(torch.round(torch.ldexp(x, -step)), step)


def _plain_append(s):
    case, c, r = s["case"], s["cache"], s["rows"]
    kv, page, block, t = case["kv"], case["page"], case["block"], r["tokens"]
    at = r["at"]
    ids = c["table"].long()[r["b"], at // page]
    # the blocks that new rows lie in, counted over all pages; the first of a sequence may hold older rows, which keep or lower their places
    where = ids * (page // block) + at % page // block
    blocks, mine = torch.unique(where, return_inverse=True)
    order = torch.empty(64, dtype=torch.long, device="cuda")
    order[torch.tensor(_order(), device="cuda")] = torch.arange(64, device="cuda")
    base = (blocks % (page // block) * block)[:, None] + torch.arange(block, device="cuda")   # [blocks][block] places in the page
    pg = (blocks // (page // block))[:, None].expand_as(base)
    first = torch.full((len(blocks),), block, device="cuda").scatter_reduce(0, mine, at % block, "amin")
    kept = torch.arange(block, device="cuda") < first[:, None]
    out = []
    for name, off, dim in (("k", s["off"][0], case["dim"]), ("v", s["off"][1], case["vdim"])):
        pool, scales = c[name], c[name + "s"].view(-1, kv, page // block)
        x = s["proj"][:, off:off + kv * dim].double().view(t, kv, dim)
        x = _turned(case, x, at) if name == "k" else x
        index = (pg, slice(None), base) if name == "k" else (pg, slice(None), base // 64, slice(None), order[base % 64])
        old_scale = scales[blocks // (page // block), :, blocks % (page // block)]             # [blocks][kv]
        old = pool[index].view(torch.float8_e4m3fn).double()[..., :dim]                       # [blocks][block][kv][dim]
        old = torch.where(kept[:, :, None, None], old * old_scale.double()[:, None, :, None], 0.0)
        most = torch.zeros((len(blocks), kv), dtype=torch.float64, device="cuda")
        most = most.scatter_reduce(0, mine[:, None].expand(-1, kv), x.abs().amax(2), "amax")
        e = _exponent(most)
        e = torch.where(kept[:, :1], torch.maximum(e, torch.frexp(old_scale)[1] - 1), e)
        old[mine, at % block] = x
        codes = _rounded(torch.ldexp(old, -e[:, None, :, None])).float().to(torch.float8_e4m3fn).view(torch.uint8)
        there = (kept | torch.zeros_like(kept).index_put((mine, at % block), torch.tensor(True, device="cuda")))[:, :, None, None]
        before = pool[index]
        pool[index] = torch.where(there, torch.cat((codes, codes.new_zeros(codes.shape[:-1] + (before.shape[-1] - dim,))), -1), before)
        scales[blocks // (page // block), :, blocks % (page // block)] = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
    back = s["back"]
    at = back["at"]
    ids = c["table"].long()[back["b"], at // page]
    for name, dim in (("k", case["dim"]), ("v", case["vdim"])):
        index = (ids, slice(None), at % page) if name == "k" else (ids, slice(None), at % page // 64, slice(None), order[at % 64])
        x = c[name][index].view(torch.float8_e4m3fn).float()[..., :dim]
        out.append((x * c[name + "s"][ids, :, at % page // block][..., None]).to(torch.bfloat16))
    return tuple(out)


def _plain_attend(s):
    case, c, r = s["case"], s["cache"], s["rows"]
    kv, page, block, d, dv, batch = case["kv"], case["page"], case["block"], case["dim"], case["vdim"], case["batch"]
    g, t, n = case["heads"] // kv, r["tokens"], c["table"].shape[1] * page
    q = _turned(case, s["proj"].double().view(t, case["heads"], d), r["at"]).float()
    ids = c["table"].long().clamp_min(0)                                                      # [batch][pages]
    k = c["k"][ids].view(torch.float8_e4m3fn).float().view(batch, -1, kv, page // block, block, c["k"].shape[3])
    k = (k * c["ks"][ids][..., None, None]).permute(0, 2, 5, 1, 3, 4).reshape(batch, kv, -1, n)[:, :, :d].contiguous()
    v = c["v"][ids].view(torch.float8_e4m3fn).float()                                         # [batch][pages][kv][groups][vp][64]
    back = torch.empty(64, dtype=torch.long, device="cuda")
    back[torch.tensor(_order(), device="cuda")] = torch.arange(64, device="cuda")
    v = v[..., back].transpose(4, 5).reshape(batch, -1, kv, page // block, block, c["v"].shape[3])
    v = (v * c["vs"][ids][..., None, None]).permute(0, 2, 1, 3, 4, 5).reshape(batch, kv, n, -1)[..., :dv].contiguous()
    j = torch.arange(n, device="cuda")
    v = torch.where((j < (r["pos"] + r["start"].diff())[:, None])[:, None, :, None], v, 0.0)
    x = q.new_zeros((batch, r["most"], case["heads"], d))
    x[r["b"], r["i"]] = q
    x = x.view(batch, r["most"], kv, g, d).permute(0, 2, 1, 3, 4).reshape(batch, kv, r["most"] * g, d)
    score = torch.matmul(x, k).view(batch, kv, r["most"], g, n)
    i = r["pos"][:, None] + torch.arange(r["most"], device="cuda")                            # [batch][most]
    seen = j <= i[..., None]
    if case["size"]:
        seen &= i[..., None] - j < case["size"]
    score = torch.where(seen[:, None, :, None], score * case["dim"] ** -0.5, -math.inf)
    p = torch.exp(score - score.amax(4, keepdim=True))
    y = torch.matmul(p.view(batch, kv, r["most"] * g, n), v) / p.sum(4).view(batch, kv, r["most"] * g, 1)
    y = y.view(batch, kv, r["most"], g, dv).permute(0, 2, 1, 3, 4).reshape(batch, r["most"], case["heads"], dv)
    return y[r["b"], r["i"]].to(s["out"].dtype)


def _plain_product(s):
    case = s["case"]
    t, r, c = case["tokens"], case["rows"], case["cols"]
    x = torch.nn.functional.pad(s["x"].float(), (0, _pad(c, 128) - c)).view(t, -1, 128)
    e = _exponent(x.abs().amax(2))[..., None]
    x = torch.ldexp(torch.ldexp(x, -e).to(torch.float8_e4m3fn).float(), e).view(t, -1)
    w = s["w"].view(torch.float8_e4m3fn).float().view(r, -1, 128) * s["scale"].repeat_interleave(128, 0)[:r, :, None]
    return torch.matmul(x, w.view(r, -1).t()).to(s["out"].dtype)


# ---- work and exact results ---------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "product":
        t, r, c = case["tokens"], case["rows"], case["cols"]
        return {"bytes": r * c + 4 * _pad(r, 128) * _pad(c, 128) // 128 ** 2 + t * c * (4 if case["x_f32"] else 2) + t * r * (4 if case["out_f32"] else 2), "flops": 2 * t * r * c}
    n, new = _lengths(case)
    kv, d, dv, block = case["kv"], case["dim"], case["vdim"], case["block"]
    if case["kind"] == "append":
        back = sum(a - (a - b) // block * block for a, b in zip(n, new))
        return {"bytes": kv * (d + dv) * (4 * sum(new) + sum(new) + back + 2 * back), "flops": 4 * sum(new) * kv * (d + dv)}
    size = case["size"] or max(n)
    held = sum(min(a, size + b - 1) for a, b in zip(n, new))
    pairs = sum(sum(min(i + 1, size) for i in range(a - b, a)) for a, b in zip(n, new))
    return {"bytes": kv * held * (d + dv + 8 / block) + case["heads"] * sum(new) * (4 * d + dv * (4 if case["f32"] else 2)), "flops": 2 * case["heads"] * (d + dv) * pairs}


def _value(codes):
    """What 8-bit elements stand for, in 64 bits: a sign, four bits of exponent and three of fraction."""
    c = codes.long()
    e, f = c >> 3 & 15, c & 7
    x = torch.where(e > 0, torch.ldexp(8.0 + f.double(), (e - 10).int()), torch.ldexp(f.double(), torch.full_like(c, -9).int()))
    x = torch.where((c & 127) == 127, math.nan, x)
    return torch.where(c > 127, -x, x)


def _held(case, c, b, n):
    """Keys and values [n][kv][...] of sequence b in 64 bits."""
    j = torch.arange(n, device="cuda")
    ids, o = c["table"][b].long()[j // case["page"]], j % case["page"]
    place = torch.argsort(torch.tensor(_order(), device="cuda"))
    k = _value(c["k"][ids, :, o]) * c["ks"].double()[ids, :, o // case["block"]][..., None]
    v = _value(c["v"][ids, :, o // 64, :, place[o % 64]]) * c["vs"].double()[ids, :, o // case["block"]][..., None]
    return k[..., :case["dim"]], v[..., :case["vdim"]]


def _rotation(case, at):
    """The matrices [rows][dim][dim] that turn rows at the given positions."""
    m = torch.eye(case["dim"], dtype=torch.float64, device="cuda").repeat(len(at), 1, 1)
    for d in range(case["rot"] // 2):
        a, b = (2 * d, 2 * d + 1) if case["pairs"] else (d, d + case["rot"] // 2)
        w = at.double() * 10000.0 ** (-2.0 * d / case["rot"])
        m[:, a, a], m[:, a, b], m[:, b, a], m[:, b, b] = w.cos(), -w.sin(), w.sin(), w.cos()
    return m


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "product":
        x, y = s["x"].double(), 0.0
        for b in range(0, case["cols"], 128):
            part = x[:, b:b + 128]
            e = torch.ceil(torch.log2(part.abs().amax(1, keepdim=True) / MOST)).clamp_min(LEAST)
            q = part / torch.exp2(e)
            step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
            q = torch.round(q / step) * step * torch.exp2(e)
            scale = s["scale"][:, b // 128].double().repeat_interleave(128)[:case["rows"], None]
            y = y + q @ (_value(s["w"][:, b:b + 128])[:, :part.shape[1]] * scale).t()
        return y
    n, new = _lengths(case)
    c, kv = s["cache"], case["kv"]
    start = s["rows"]["start"].tolist()
    if case["kind"] == "attend":
        g, y = case["heads"] // kv, []
        for b in range(case["batch"]):
            k, v = _held(case, c, b, n[b])
            at = torch.arange(n[b] - new[b], n[b], device="cuda")
            j = torch.arange(n[b], device="cuda")
            q = s["proj"][start[b]:start[b + 1]].double().view(new[b], case["heads"], -1)
            q = q @ _rotation(case, at).transpose(1, 2)
            hide = (j > at[:, None]) | (at[:, None] - j >= (case["size"] or n[b]))
            y.append(torch.stack([torch.softmax((q[:, h] @ k[:, h // g].t() * case["dim"] ** -0.5).masked_fill(hide, -math.inf), 1) @ v[:, h // g] for h in range(case["heads"])], 1))
        return torch.cat(y)
    out = [], []
    for b in range(case["batch"]):
        pos, block = n[b] - new[b], case["block"]
        first = pos // block * block
        old = _held(case, c, b, n[b])
        row = s["proj"][start[b]:start[b + 1]].double()
        at = torch.arange(pos, n[b], device="cuda")
        for i, (off, dim) in enumerate(zip(s["off"], (case["dim"], case["vdim"]))):
            x = row[:, off:off + kv * dim].view(new[b], kv, dim)
            if i == 0:   # every head's rows by their positions' matrices
                x = torch.cat([q @ _rotation(case, a).transpose(1, 2) for q, a in zip(x.split(512), at.split(512))])
            x = torch.cat((old[i][first:pos], x))
            for lo in range(0, len(x), block):
                part = x[lo:lo + block]
                fresh = part if lo or first == pos else part[pos - first:]
                e = torch.ceil(torch.log2(fresh.abs().amax((0, 2)) / MOST)).clamp_min(LEAST)
                if lo == 0 and first < pos:
                    page = c["table"][b].long()[first // case["page"]]
                    e = torch.maximum(e, torch.log2(c["ks" if i == 0 else "vs"][page, :, first % case["page"] // block].double()))
                q = part / torch.exp2(e)[:, None]
                step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
                out[i].append(torch.round(q / step) * step * torch.exp2(e)[:, None])
    return tuple(torch.cat(x) for x in out)

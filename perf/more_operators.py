"""Timed cases of the operators between an attention block's projections, for several requests at once.

Paths (entry points of include/drama_moe.h):
  rope    dr_rope(_bf16): the norm of each head and its rotary positions
  append  dr_kv8_append(_bf16): new tokens into a cache held in 8 bits; dr_kv8_read gives back what the cache then stands for
  attn    dr_attn_kv8: attention over that cache, for single tokens and for prompts

A cache holds blocks of 64 tokens of one sequence and head, integers -127 .. 127 stored with 128 added and one f32 scale a block:
kq [pages, hkv, d / 16, 64, 16] is element 16 c + e of token t at [.., c, t, e]; vq [pages, hkv, d, 64] has token 16 a + 4 b + c of
element x at [.., x, 16 b + 4 a + c]; ks, vs [pages, hkv].

`run` computes the plain form in float32 torch operations, or with `own` calls the library.
"""
import math
import os
import sys

import torch

own = False
EPS = 1e-6
BLOCK = 64


# ---- cases ------------------------------------------------------------------------------------


def listed():
    return [
        # the heads of one decode token: 16 of q and 4 of k behind one projection, norms as the served model has them
        {"name": "rope_1", "path": "rope", "rows": 1, "heads": 20, "d": 128, "rot": 128, "pairs": False, "norm": True, "b16": False,
         "out": "bf16", "gated": False, "far": 300, "factor": 1.0},
        # a prompt of 777 rows, a head of no power of two rotated in part by neighbouring pairs, bf16 in place of f32
        {"name": "rope_777_pairs", "path": "rope", "rows": 777, "heads": 15, "d": 80, "rot": 36, "pairs": True, "norm": False, "b16": True,
         "out": "f32", "gated": False, "far": 30000, "factor": 8.0},
        # a long prompt chunk far into a long context, each head's gate beside it in the projection
        {"name": "rope_8192_gated", "path": "rope", "rows": 8192, "heads": 16, "d": 256, "rot": 64, "pairs": False, "norm": True, "b16": False,
         "out": "bf16", "gated": True, "far": 1000000, "factor": 4.0},
        # one token into the cache of one sequence
        {"name": "append_1", "path": "append", "seqs": 1, "rmin": 1, "rmax": 1, "lmin": 500, "lmax": 500, "hkv": 4, "d": 128, "b16": False,
         "pad": 0, "empty": False},
        # a decode step of 64 sequences, a few rows of padding behind them
        {"name": "append_64_bf16", "path": "append", "seqs": 64, "rmin": 1, "rmax": 1, "lmin": 1, "lmax": 4000, "hkv": 8, "d": 128, "b16": True,
         "pad": 5, "empty": True},
        # ragged prompts, some behind tokens that are cached already
        {"name": "append_prompts", "path": "append", "seqs": 9, "rmin": 37, "rmax": 2100, "lmin": 1, "lmax": 300, "hkv": 4, "d": 128, "b16": False,
         "pad": 0, "empty": False},
        # one short request, pure latency
        {"name": "attn_1x300", "path": "attn", "seqs": 1, "rmin": 1, "rmax": 1, "lmin": 299, "lmax": 299, "hq": 16, "hkv": 4, "d": 128,
         "gate": False, "pad": 0, "empty": False},
        # one request with a long document in its cache, wide heads, few of them cached
        {"name": "attn_1x60001", "path": "attn", "seqs": 1, "rmin": 1, "rmax": 1, "lmin": 60000, "lmax": 60000, "hq": 16, "hkv": 2, "d": 256,
         "gate": True, "pad": 0, "empty": False},
        # a decode batch of requests of very different lengths, one of them empty
        {"name": "attn_48_ragged", "path": "attn", "seqs": 48, "rmin": 1, "rmax": 1, "lmin": 20, "lmax": 16000, "hq": 32, "hkv": 8, "d": 128,
         "gate": False, "pad": 3, "empty": True},
        # drafted tokens checked together, five queries a cached head and a head size of no power of two
        {"name": "attn_draft", "path": "attn", "seqs": 6, "rmin": 3, "rmax": 5, "lmin": 5000, "lmax": 9000, "hq": 20, "hkv": 4, "d": 80,
         "gate": False, "pad": 0, "empty": False},
        # a few prompts from their first token on, each query with its own cached head
        {"name": "attn_prompts", "path": "attn", "seqs": 7, "rmin": 33, "rmax": 400, "lmin": 0, "lmax": 0, "hq": 12, "hkv": 12, "d": 64,
         "gate": True, "pad": 10, "empty": True},
        # a chunk of a long prompt behind twice as many cached tokens
        {"name": "attn_chunk_4096", "path": "attn", "seqs": 1, "rmin": 4096, "rmax": 4096, "lmin": 8192, "lmax": 8192, "hq": 16, "hkv": 2,
         "d": 128, "gate": False, "pad": 0, "empty": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["rope", "append", "attn", "attn"])
    flag = lambda p: rng.random() < p
    d = rng.choice([16, 32, 48, 64, 64, 80, 96, 112, 128, 128, 128, 160, 192, 256, 256])
    if path == "rope":
        d = rng.choice([d, rng.randint(2, 256)])
        heads = _log(rng, 1, 40)
        rows = max(1, min(_log(rng, 1, 8192), 8192 * 16 * 256 // (heads * d)))
        rot = rng.choice([d // 2 * 2, d // 4 * 2, 2 * rng.randint(0, d // 2)])
        return {"path": path, "rows": rows, "heads": heads, "d": d, "rot": rot, "pairs": flag(0.5), "norm": flag(0.5), "b16": flag(0.5),
                "out": rng.choice(["f32", "bf16", "both"]), "gated": flag(0.3), "far": _log(rng, 1, 1000000), "factor": rng.choice([1.0, 4.0, 8.0])}
    hkv, seqs = _log(rng, 1, 16), _log(rng, 1, 64)
    if path == "append":
        rmax = rng.choice([1, _log(rng, 1, 2000)])
        rmax = max(1, min(rmax, 8192 * 4 * 128 // (seqs * hkv * d)))
        lo = _log(rng, 1, 4000)
        return {"path": path, "seqs": seqs, "rmin": rng.randint(1, rmax), "rmax": rmax, "lmin": lo, "lmax": _log(rng, lo, 4000), "hkv": hkv, "d": d,
                "b16": flag(0.5), "pad": rng.choice([0, 0, 7]), "empty": flag(0.3)}
    g = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    hkv = max(1, min(hkv, 64 // g))
    kind = rng.choice(["one", "draft", "prompt"])
    rmax = {"one": 1, "draft": rng.randint(2, 8), "prompt": _log(rng, 9, 2000)}[kind]
    if kind == "prompt":
        seqs = max(1, min(seqs, 6000 // rmax))
    lmax = _log(rng, 1, 16000 if kind != "prompt" else 6000)
    # no more work than the largest listed case, and no more cached tokens than the ragged batch holds at its longest
    lmax = max(1, min(lmax, 16000 * 48 * 8 * 128 // (seqs * hkv * d), int(1.2e11 / (4 * seqs * rmax * g * hkv * d))))
    if kind == "prompt":
        rmax = max(9, min(rmax, int(1.2e11 / (4 * seqs * g * hkv * d * (lmax + rmax)))))
    return {"path": path, "seqs": seqs, "rmin": rng.randint(1, rmax), "rmax": rmax, "lmin": rng.randint(0, lmax), "lmax": lmax, "hq": g * hkv,
            "hkv": hkv, "d": d, "gate": flag(0.3), "pad": rng.choice([0, 0, 7]), "empty": flag(0.3)}


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, even over their logarithm, in no order."""
    if lo >= hi:
        return [lo] * n
    a = max(lo, 1)
    return [max(lo, min(hi, int(round(a * (hi / a) ** ((0.5 + 0.6180339887 * i) % 1))))) for i in range(n)]


def _batch(case):
    """(new rows, cached tokens with them) of each sequence. "empty": the second sequence has no row, the third rows but no token."""
    rows = _spread(case["seqs"], case["rmin"], case["rmax"])
    lens = [a + b for a, b in zip(rows, _spread(case["seqs"], case["lmin"], case["lmax"])[::-1])]
    if case["empty"] and case["seqs"] > 2:
        lens[1], rows[1], lens[2] = lens[1] - rows[1], 0, 0
    return rows, lens


# ---- inputs -----------------------------------------------------------------------------------


def _randn(shape, gen, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _sums(v):
    out = [0]
    for a in v:
        out.append(out[-1] + a)
    return out


def _cache(s, case, lens, gen):
    """A cache in use: every block holds numbers, the blocks of a sequence lie anywhere, k with a few channels above the others."""
    hkv, d = case["hkv"], case["d"]
    need = [(n + BLOCK - 1) // BLOCK for n in lens]
    pages, maxp = sum(need) + 3, max(max(need), 1)
    order = torch.randperm(pages, generator=gen, device="cuda").tolist()
    at = _sums(need)
    s["pages"], s["maxp"], s["order"], s["need"] = pages, maxp, order, need
    s["table"] = _ints([order[at[i]:at[i + 1]] + [-1] * (maxp - need[i]) for i in range(len(need))])
    chan = 1 + 2 * (torch.rand((hkv, d), generator=gen, device="cuda") < 0.05)
    # stored numbers of one block's spread, all blocks at once in the cache's own order
    k = _randn((pages, hkv, d // 16, BLOCK, 16), gen, torch.float16).mul_(chan.view(hkv, d // 16, 1, 16).half() * 20)
    s["kq"] = k.round_().clamp_(-127, 127).add_(128).to(torch.uint8)
    v = _randn((pages, hkv, d, BLOCK), gen, torch.float16).mul_(32)
    s["vq"] = v.round_().clamp_(-127, 127).add_(128).to(torch.uint8)
    s["ks"] = torch.exp(0.3 * _randn((pages, hkv), gen)) / 20
    s["vs"] = torch.exp(0.3 * _randn((pages, hkv), gen)) / 32


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["path"] == "rope":
        rows, heads, d, rot = case["rows"], case["heads"], case["d"], case["rot"]
        s["hs"] = 2 * d if case["gated"] else d
        s["x"] = 2 * _randn((rows, heads * s["hs"]), gen)
        if case["b16"]:
            s["x"] = s["x"].to(torch.bfloat16)
        s["nw"] = 1 + 0.1 * _randn((heads, d), gen) if case["norm"] else None
        first = torch.randint(0, case["far"], (1,), generator=gen, device="cuda")
        s["pos"] = (first + torch.arange(rows, device="cuda")).to(torch.int32)
        # positions drawn out by `factor` below the frequencies that turn often within the trained length
        f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / max(rot, 1))
        s["freq"] = torch.where(f * 4096 > 64, f, f / case["factor"]).float()
        s["ms"] = 0.1 * math.log(case["factor"]) + 1
    else:
        rows, lens = _batch(case)
        start = _sums(rows)
        s["rows"], s["total"] = start[-1], start[-1] + case["pad"]
        s["start"], s["len"] = _ints(start), _ints(lens)
        _cache(s, case, lens, gen)
        if case["path"] == "append":
            _prepare_append(s, case, rows, lens, gen)
        else:
            hq, d = case["hq"], case["d"]
            s["q"] = (2 * _randn((s["total"], hq * d), gen)).to(torch.bfloat16)
            s["gate"] = _randn((s["total"], hq * d), gen) if case["gate"] else None
            s["nmax"], s["lmax"] = max(rows), max(lens)
            s["seq_of"] = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(rows)).cuda()
            s["slot_of"] = torch.arange(s["rows"], device="cuda") - s["start"].long()[s["seq_of"]]
    if own:
        _prepare_own(s, case)
    return s


def _prepare_append(s, case, rows, lens, gen):
    for n in ("k", "v"):
        s[n] = _randn((s["total"], case["hkv"] * case["d"]), gen) * (1.5 if n == "k" else 1.0)
        if case["b16"]:
            s[n] = s[n].to(torch.bfloat16)
    # every block that gets a token: its page, its sequence and the row (or -1) of each of its 64 places
    page, places, read, at, start = [], [], [], _sums(s["need"]), _sums(rows)
    for i, (n, m) in enumerate(zip(rows, lens)):
        first = m - n
        if n == 0 or m == 0:
            read.append(0)
            continue
        read.append(m - max(first, 0) // BLOCK * BLOCK)
        for b in range(max(first, 0) // BLOCK, (m + BLOCK - 1) // BLOCK):
            page.append(s["order"][at[i] + b])
            places.append([start[i] + t - first if first <= t < m else -1 for t in range(b * BLOCK, (b + 1) * BLOCK)])
    s["page"], s["place"] = torch.tensor(page, dtype=torch.int64, device="cuda"), torch.tensor(places, dtype=torch.int64, device="cuda").view(-1, BLOCK)
    # what is read back: every sequence's tokens from the first block on that the call reached, in order
    s["read"], s["read_start"] = sum(read), _ints(_sums(read))
    tok = [(i, m - c + t) for i, (m, c) in enumerate(zip(lens, read)) for t in range(c)]
    s["tok_page"] = torch.tensor([s["order"][at[i] + t // BLOCK] for i, t in tok], dtype=torch.int64, device="cuda")
    s["tok_at"] = torch.tensor([t % BLOCK for _, t in tok], dtype=torch.int64, device="cuda")


# ---- the plain forms, float32 -----------------------------------------------------------------


def _plain_rope(s, case):
    rows, heads, d, rot = case["rows"], case["heads"], case["d"], case["rot"]
    x = s["x"].view(rows, heads, s["hs"])[:, :, :d].float()
    if s["nw"] is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["nw"]
    # angles in 64 bits: far positions turn thousands of times
    th = s["pos"].double()[:, None] * s["freq"].double()
    c, n = (torch.cos(th) * s["ms"]).float()[:, None], (torch.sin(th) * s["ms"]).float()[:, None]
    if case["pairs"]:
        a, b = x[:, :, 0:rot:2], x[:, :, 1:rot:2]
        turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = x[:, :, :rot // 2], x[:, :, rot // 2:rot]
        turned = torch.cat([a * c - b * n, b * c + a * n], -1)
    y = torch.cat([turned, x[:, :, rot:]], -1).view(rows, heads * d)
    return {"f32": y, "bf16": y.to(torch.bfloat16)} if case["out"] == "both" else {case["out"]: y.to(torch.bfloat16) if case["out"] == "bf16" else y}


def _v_order(v):
    """The 64 tokens of a block, last in v: in order to the cache's order of v, and back (the map is its own inverse)."""
    return v.unflatten(-1, (4, 4, 4)).transpose(-3, -2).flatten(-3)


def _stored(x, page, place, q, scale):
    """What the blocks, q [blocks, 64, hkv, d] so far, hold with the tokens x (0 where place is -1); their scales are updated."""
    new = place >= 0
    top = x.abs().amax((1, 3)).double()
    s0 = scale[page]
    # a power of two by which the block's scale grows where it has tokens already; whole numbers next to a border need 64 bits
    m, e = torch.frexp(top / (127 * s0.double()))
    grow = torch.where(m == 0.5, e - 1, e).clamp(min=0)
    fresh = new[:, :1] | (s0 == 0)
    s1 = torch.where(fresh, (top / 127).float(), torch.ldexp(s0, grow))
    d1 = s1.double()[:, None, :, None]
    put = torch.where(d1 > 0, torch.round(x.double() / d1), 0.0).clamp(-127, 127)
    old = torch.round(torch.ldexp(q, torch.where(fresh, 0, -grow)[:, None, :, None]))
    scale[page] = s1
    return torch.where(new[:, :, None, None], put, torch.where(new[:, :1, None, None], 0.0, old))


def _plain_append(s, case):
    hkv, d, page, place = case["hkv"], case["d"], s["page"], s["place"]
    new = (place >= 0)[:, :, None, None]
    pick = lambda x: torch.where(new, x.float().view(-1, hkv, d)[place.clamp(min=0)], 0.0)
    # [blocks, 64, hkv, d] of what the blocks hold
    k0 = s["kq"][page].permute(0, 3, 1, 2, 4).flatten(-2).double() - 128
    v0 = _v_order(s["vq"][page]).permute(0, 3, 1, 2).double() - 128
    k1 = _stored(pick(s["k"]), page, place, k0, s["ks"])
    v1 = _stored(pick(s["v"]), page, place, v0, s["vs"])
    s["kq"][page] = (k1 + 128).to(torch.uint8).unflatten(-1, (d // 16, 16)).permute(0, 2, 3, 1, 4)
    s["vq"][page] = _v_order((v1 + 128).to(torch.uint8).permute(0, 2, 3, 1))
    # read back
    p, t = s["tok_page"], s["tok_at"]
    at = 16 * (t // 4 % 4) + 4 * (t // 16) + t % 4
    k = (s["kq"][p, :, :, t].flatten(-2).float() - 128) * s["ks"][p][:, :, None]
    v = (s["vq"][p, :, :, at].float() - 128) * s["vs"][p][:, :, None]
    return k.flatten(1), v.flatten(1), s["ks"], s["vs"]


def _plain_attn(s, case):
    """All sequences at once, each drawn out to the longest."""
    n, hq, hkv, d = case["seqs"], case["hq"], case["hkv"], case["d"]
    rows, lmax, t = s["nmax"], s["lmax"], s["table"].long().clamp(min=0)
    k = (s["kq"][t].float() - 128) * s["ks"][t][:, :, :, None, None, None]  # [n, pages, hkv, d / 16, 64, 16]
    k = k.permute(0, 2, 3, 5, 1, 4).reshape(n, hkv, d, -1)[..., :lmax]
    first = s["start"].long()[:-1, None] + torch.arange(rows, device="cuda")
    q = s["q"][first.clamp(max=max(s["total"] - 1, 0))].float().view(n, rows, hkv, hq // hkv, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, d)
    sc = (q @ k.contiguous()).view(n, hkv, rows, hq // hkv, lmax) / math.sqrt(d)
    count = (s["start"][1:] - s["start"][:-1]).long()
    pos = (s["len"].long() - count)[:, None] + torch.arange(rows, device="cuda")
    seen = (torch.arange(lmax, device="cuda") <= pos[:, :, None])[:, None, :, None]
    sc = torch.where(seen, sc, -math.inf)
    top = sc.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(sc - top), 0.0)
    total = e.sum(-1, keepdim=True)
    v = (_v_order(s["vq"][t]).float() - 128) * s["vs"][t][:, :, :, None, None]  # [n, pages, hkv, d, 64]
    v = v.permute(0, 2, 1, 4, 3).reshape(n, hkv, -1, d)[:, :, :lmax].contiguous()
    o = (e.view(n, hkv, -1, lmax) @ v).view(n, hkv, rows, hq // hkv, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(n, rows, hq * d)
    y = torch.zeros(s["total"], hq * d, device="cuda")
    y[:s["rows"]] = o[s["seq_of"], s["slot_of"]]
    if s["gate"] is not None:
        y = y / (1 + torch.exp(-s["gate"]))
    return y.to(torch.bfloat16)


def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return {"rope": _plain_rope, "append": _plain_append, "attn": _plain_attn}[case["path"]](s, case)


# ---- the library's calls ----------------------------------------------------------------------


def _lib():
    sys.path.insert(0, os.path.join(os.getcwd(), "drama-rs_amd"))
    import dramamoe

    return dramamoe


def _prepare_own(s, case):
    """Output buffers, and the workspace that a program keeps."""
    D = _lib()
    s["D"], s["lib"] = D, D.lib()
    zeros = lambda *shape, dt=torch.float32: torch.zeros(shape, dtype=dt, device="cuda")
    if case["path"] == "rope":
        n = case["heads"] * case["d"]
        s["y"] = zeros(case["rows"], n) if case["out"] != "bf16" else None
        s["yb"] = zeros(case["rows"], n, dt=torch.bfloat16) if case["out"] != "f32" else None
    elif case["path"] == "append":
        s["k_out"], s["v_out"] = (zeros(s["read"], case["hkv"] * case["d"]) for _ in range(2))
    else:
        s["y"] = zeros(s["total"], case["hq"] * case["d"], dt=torch.bfloat16)
        n = s["lib"].dr_attn_kv8_ws(s["total"], case["seqs"], s["nmax"], s["lmax"], case["hq"], case["hkv"], case["d"])
        s["ws"] = zeros(n, dt=torch.uint8)


def _own(s, case):
    P, lib, st = s["D"].ptr, s["lib"], s["D"].stream_ptr()
    if case["path"] == "rope":
        n, heads = case["heads"] * case["d"], case["heads"]
        (lib.dr_rope_bf16 if case["b16"] else lib.dr_rope)(
            P(s["x"]), heads * s["hs"], s["hs"], P(s["nw"]), case["d"], EPS, P(s["pos"]), P(s["freq"]), s["ms"], int(case["pairs"]), P(s["y"]), n,
            P(s["yb"]), n, case["rows"], heads, case["d"], case["rot"], st)
        return {k: v for k, v in (("f32", s["y"]), ("bf16", s["yb"])) if v is not None}
    hkv, d = case["hkv"], case["d"]
    cache = (P(s["table"]), s["maxp"], P(s["kq"]), P(s["ks"]), P(s["vq"]), P(s["vs"]), s["pages"])
    if case["path"] == "append":
        n = hkv * d
        (lib.dr_kv8_append_bf16 if case["b16"] else lib.dr_kv8_append)(
            P(s["k"]), n, P(s["v"]), n, P(s["start"]), P(s["len"]), *cache, s["total"], case["seqs"], hkv, d, st)
        lib.dr_kv8_read(P(s["read_start"]), P(s["len"]), *cache, P(s["k_out"]), n, P(s["v_out"]), n, s["read"], case["seqs"], hkv, d, st)
        return s["k_out"], s["v_out"], s["ks"], s["vs"]
    n = case["hq"] * d
    lib.dr_attn_kv8(P(s["q"]), n, P(s["start"]), P(s["len"]), *cache, 1 / math.sqrt(d), P(s["gate"]), n, d, P(s["ws"]), P(s["y"]), n, s["total"],
                    case["seqs"], s["nmax"], s["lmax"], case["hq"], hkv, d, st)
    return s["y"]


# ---- work and the definition in 64 bits -------------------------------------------------------


def work(case):
    if case["path"] == "rope":
        n = case["rows"] * case["heads"] * case["d"]
        out = {"f32": 4, "bf16": 2, "both": 6}[case["out"]]
        vec = 4 * case["rows"] + 2 * case["rot"] + (4 * case["heads"] * case["d"] if case["norm"] else 0)
        return {"bytes": n * ((2 if case["b16"] else 4) + out) + vec, "flops": n * (7 if case["norm"] else 3)}
    rows, lens = _batch(case)
    hkv, d = case["hkv"], case["d"]
    if case["path"] == "append":
        # tokens in, their numbers out; the read: the numbers of every block that got a token, as f32
        real = [(n, m) for n, m in zip(rows, lens) if n and m]
        new = sum(min(n, m) for n, m in real)
        read = sum(m - max(m - n, 0) // BLOCK * BLOCK for n, m in real)
        each = 2 * hkv * d
        return {"bytes": new * each * ((2 if case["b16"] else 4) + 1) + read * each * 5, "flops": new * each * 4 + read * each * 2}
    hq = case["hq"]
    real = [(n, m) for n, m in zip(rows, lens) if n and m]
    pairs = sum(n * m - n * (n - 1) // 2 for n, m in real)
    q = sum(rows) * hq * d * (2 + 2 + (4 if case["gate"] else 0))
    return {"bytes": sum(2 * m * hkv * d + 8 * hkv * ((m + BLOCK - 1) // BLOCK) for _, m in real) + q, "flops": 4 * d * hq * pairs}


def _exact_rope(s, case):
    rows, heads, d, rot = case["rows"], case["heads"], case["d"], case["rot"]
    y = s["x"].double().view(rows, heads, -1)[..., :d].clone()
    if case["norm"]:
        y *= s["nw"].double() / torch.sqrt(torch.linalg.vector_norm(y, dim=-1, keepdim=True) ** 2 / d + EPS)
    at = torch.arange(rot // 2, device="cuda")
    a, b = (2 * at, 2 * at + 1) if case["pairs"] else (at, at + rot // 2)
    # a rotation is a product of complex numbers
    turn = torch.polar(torch.full((rows, 1, rot // 2), s["ms"], dtype=torch.float64, device="cuda"),
                       torch.outer(s["pos"].double(), s["freq"].double())[:, None])
    z = torch.complex(y[..., a], y[..., b]) * turn
    y[..., a], y[..., b] = z.real, z.imag
    y = y.view(rows, heads * d)
    return {"f32": y, "bf16": y} if case["out"] == "both" else {case["out"]: y}


def _exact_append(s, case):
    hkv, d = case["hkv"], case["d"]
    rows, lens = _batch(case)
    table, start = s["table"].tolist(), _sums(rows)
    back = torch.empty(BLOCK, dtype=torch.int64, device="cuda")
    for t in range(BLOCK):
        back[t] = 16 * (t % 16 // 4) + 4 * (t // 16) + t % 4
    out = []
    for x, scale, block in ((s["k"], s["ks"], lambda p: s["kq"][p].permute(2, 0, 1, 3).reshape(BLOCK, hkv, d)),
                            (s["v"], s["vs"], lambda p: s["vq"][p][:, :, back].permute(2, 0, 1))):
        x, scales, got = x.double().view(-1, hkv, d), scale.double(), []
        for i, (n, m) in enumerate(zip(rows, lens)):
            if n == 0 or m == 0:
                continue
            first = m - n
            for b in range(max(first, 0) // BLOCK, (m + BLOCK - 1) // BLOCK):
                p, lo, hi = table[i][b], max(first, b * BLOCK), min(m, (b + 1) * BLOCK)
                tok = x[start[i] + lo - first:start[i] + hi - first]
                top = tok.abs().amax((0, 2))
                if lo == b * BLOCK:
                    kept, sc = tok[:0], (top / 127).float().double()
                else:
                    kept, sc = block(p)[:lo - b * BLOCK].double() - 128, scales[p]
                    while bool((top > 127 * sc).any()):
                        kept = torch.where((top > 127 * sc)[:, None], kept / 2, kept)
                        sc = torch.where(top > 127 * sc, 2 * sc, sc)
                whole = torch.cat([kept.round(), (tok / sc[:, None]).round().clamp(-127, 127)])
                got.append((whole * sc[:, None]).reshape(-1, hkv * d))
                scales[p] = sc
        out += [torch.cat(got), scales]
    return out[0], out[2], out[1], out[3]


def _exact_attn(s, case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    rows, lens = _batch(case)
    y, at = torch.zeros(s["total"], hq, d, dtype=torch.float64, device="cuda"), 0
    back = [16 * (t % 16 // 4) + 4 * (t // 16) + t % 4 for t in range(BLOCK)]
    for i, (n, m) in enumerate(zip(rows, lens)):
        p = s["table"][i, :(m + BLOCK - 1) // BLOCK].long()
        for h in range(hkv if n and m else 0):
            k = (s["kq"][p, h].transpose(1, 2).reshape(-1, d)[:m].double() - 128) * s["ks"][p, h].double().repeat_interleave(BLOCK)[:m, None]
            v = (s["vq"][p, h][:, :, back].transpose(1, 2).reshape(-1, d)[:m].double() - 128) * s["vs"][p, h].double().repeat_interleave(BLOCK)[:m, None]
            for r0 in range(0, n, 1024):
                r1 = min(n, r0 + 1024)
                pos = torch.arange(m - n + r0, m - n + r1, device="cuda")
                hidden = torch.arange(m, device="cuda")[None, :] > pos[:, None]
                for g in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    z = (s["q"][at + r0:at + r1].view(-1, hq, d)[:, g].double() @ k.t()) * d ** -0.5
                    z.masked_fill_(hidden, -math.inf)
                    y[at + r0:at + r1, g] = torch.nan_to_num(torch.softmax(z, -1)) @ v
        at += n
    if case["gate"]:
        y *= torch.sigmoid(s["gate"].double()).view(y.shape)
    return y.view(s["total"], hq * d)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "attn": _exact_attn}[case["path"]](s, case)

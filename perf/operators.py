"""Timed cases of the operators around and of the MoE block that serve several requests at once.

Paths (entry points of include/drama_moe.h):
  norm     dr_block_norm(_bf16): norm behind a block, gate, residual scale, norm before the next block
  combine  dr_moe_combine_norm: the same on the weighted sum of a prefill's expert rows
  lora     dr_gemm_q8_lora(_bf16s): an int8 projection shared by all rows, with each row's low-rank adapter
  moe      dr_moe_layer_rows*: router, experts and shared expert of a few tokens

`run` computes the plain form in float32 torch operations, or with `own` calls the library.
"""
import math
import os
import sys

import torch

own = False
EPS = 1e-6


# ---- cases ------------------------------------------------------------------------------------


def listed():
    return [
        # one decode token between two blocks: pure latency
        {"name": "norm_1x2048", "path": "norm", "rows": 1, "h": 2048, "b16": False, "post": True, "gate": 0, "cs": False},
        # a prompt of 1000 rows, bf16 block output with a gate logit per element; a hidden size of no power of two
        {"name": "norm_1000x1800_bf16", "path": "norm", "rows": 1000, "h": 1800, "b16": True, "post": True, "gate": 2, "cs": True},
        # the longest prompt chunk of a wider model
        {"name": "norm_4096x4096", "path": "norm", "rows": 4096, "h": 4096, "b16": False, "post": True, "gate": 1, "cs": False},
        # the end of a 300-row prefill layer: eight expert rows a token and the shared expert
        {"name": "combine_300", "path": "combine", "rows": 300, "h": 2048, "topk": 8, "post": False, "gate": 0, "cs": False},
        # one request with an adapter, the projection of a decode step
        {"name": "lora_1", "path": "lora", "fmt": "ref", "rows": 1, "n": 2048, "k": 2048, "adapters": 4, "rmax": 16, "mix": "each"},
        # 48 requests decoded together, nearly every one with an adapter of its own
        {"name": "lora_48", "path": "lora", "fmt": "cfg", "rows": 48, "n": 4096, "k": 2048, "adapters": 40, "rmax": 32, "mix": "each"},
        # a few prompts in one call, each with its adapter, onto an odd number of outputs
        {"name": "lora_700", "path": "lora", "fmt": "ref", "rows": 700, "n": 1031, "k": 1024, "adapters": 5, "rmax": 16, "mix": "runs"},
        # the longest batch of prompts
        {"name": "lora_4096", "path": "lora", "fmt": "cfg", "rows": 4096, "n": 4096, "k": 2048, "adapters": 12, "rmax": 64, "mix": "runs"},
        # one token through one layer of the served model
        {"name": "moe_q4_1", "path": "moe", "kind": "q4", "fmt": "ref", "rows": 1, "e": 256, "h": 2048, "i": 512, "topk": 8, "shared": True},
        # a small batch on the original block-FP8 experts
        {"name": "moe_fp8_8", "path": "moe", "kind": "fp8", "fmt": "cfg", "rows": 8, "e": 256, "h": 2048, "i": 512, "topk": 8, "shared": True},
        # another model's sizes: fewer, wider experts, no shared one
        {"name": "moe_q4_19_e48", "path": "moe", "kind": "q4", "fmt": "cfg", "rows": 19, "e": 48, "h": 1280, "i": 896, "topk": 4, "shared": False},
        # the largest decode batch of the served model
        {"name": "moe_q4_64", "path": "moe", "kind": "q4", "fmt": "ref", "rows": 64, "e": 256, "h": 2048, "i": 512, "topk": 8, "shared": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["norm", "combine", "lora", "lora", "moe", "moe"])
    flag = lambda p: rng.random() < p
    if path in ("norm", "combine"):
        rows, h = _log(rng, 1, 4096), _log(rng, 64, 8192)
        if flag(0.7):
            h = (h + 7) // 8 * 8
        c = {"path": path, "rows": rows, "h": h, "post": flag(0.6), "gate": rng.choice([0, 1, 2]), "cs": flag(0.4)}
        if path == "norm":
            c["rows"] = max(1, min(rows, (4096 * 4096) // h))
            c["b16"] = flag(0.5)
        else:
            c["h"] = h = (h + 3) // 4 * 4
            c["topk"] = rng.randint(1, 8)
            c["rows"] = max(1, min(rows, (4096 * 4096) // (h * (c["topk"] + 1))))
        return c
    if path == "lora":
        rows, n, k = _log(rng, 1, 4096), _log(rng, 64, 8192), 128 * _log(rng, 2, 32)
        rows = max(1, min(rows, (4096 * 4096 * 2048) // (n * k)))
        return {"path": path, "fmt": rng.choice(["ref", "cfg"]), "rows": rows, "n": n, "k": k,
                "adapters": _log(rng, 1, 64), "rmax": rng.choice([8, 16, 32, 64]), "mix": rng.choice(["each", "runs"]) if rows < 128 else "runs"}
    h, i, e, kind = 128 * _log(rng, 2, 32), 128 * _log(rng, 1, 12), _log(rng, 8, 256), rng.choice(["q4", "fp8"])
    e = max(8, min(e, (256 if kind == "q4" else 128) * 2048 * 512 // (h * i)))
    return {"path": path, "kind": kind, "fmt": rng.choice(["ref", "cfg"]), "rows": _log(rng, 1, 64),
            "e": e, "h": h, "i": i, "topk": rng.randint(1, 8), "shared": flag(0.7)}


# ---- inputs -----------------------------------------------------------------------------------


def _randn(shape, gen, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _bytes(n, gen):
    return torch.randint(0, 256, (n,), generator=gen, device="cuda", dtype=torch.uint8)


def _int8(n, k, fmt, gen):
    """int8 weights with f16 scales per 128 inputs ("ref") or a bf16 scale per row ("cfg")."""
    q = _bytes(n * k, gen).view(torch.int8).view(n, k).clamp_(min=-127)
    shape = (n, k // 128) if fmt == "ref" else (n,)
    s = (_randn(shape, gen).abs_().mul_(0.02).add_(1e-4)) / 73
    return q, s.half() if fmt == "ref" else s.to(torch.bfloat16)


def _experts(e, n, k, case, gen):
    """int4 nibbles with a (scale, min) pair per 64 inputs, or e4m3 with a scale per 128 x 128 block."""
    ref = case["fmt"] == "ref"
    if case["kind"] == "q4":
        sm = _randn((e, n, k // 64, 2), gen, torch.float16 if ref else torch.bfloat16).mul_(0.02)
        sm[..., 0].abs_().add_(1e-4)
        return _bytes(e * n * k // 2, gen).view(e, n, k // 2), sm
    q = torch.empty(e, n, k, dtype=torch.uint8, device="cuda")
    for a in range(0, e, 32):
        b = min(e, a + 32)
        q[a:b] = _randn((b - a, n, k), gen, torch.float16).mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    s = _randn((e, n // 128, k // 128), gen).abs_().mul_(0.02).add_(1e-4).div_(100)
    return q, s if ref else s.to(torch.bfloat16)


def _norm_inputs(s, case, gen):
    rows, h = case["rows"], case["h"]
    s["x"] = _randn((rows, h), gen)
    s["pw"] = 1 + 0.1 * _randn((h,), gen) if case["post"] else None
    s["nw"] = 1 + 0.1 * _randn((h,), gen)
    s["gate"] = _randn((rows, h) if case["gate"] == 2 else (rows,), gen) if case["gate"] else None
    s["cs"] = 1 + 0.1 * _randn((h,), gen) if case["cs"] else None
    s["bscale"], s["xscale"] = 0.5, 0.875


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["path"] == "norm":
        s["b"] = _randn((case["rows"], case["h"]), gen)
        if case["b16"]:
            s["b"] = s["b"].to(torch.bfloat16)
        _norm_inputs(s, case, gen)
    elif case["path"] == "combine":
        rows, h, topk = case["rows"], case["h"], case["topk"]
        s["y"] = _randn((rows * topk, h), gen)
        s["slot"] = torch.randperm(rows * topk, generator=gen, device="cuda").to(torch.int32)
        s["wts"] = torch.softmax(_randn((rows, topk), gen), -1)
        s["sgate"] = _randn((rows,), gen)
        s["shared"] = _randn((rows, h), gen)
        _norm_inputs(s, case, gen)
    elif case["path"] == "lora":
        rows, n, k, na, rm = (case[a] for a in ("rows", "n", "k", "adapters", "rmax"))
        s["w"], s["s"] = _int8(n, k, case["fmt"], gen)
        s["x"] = _randn((rows, k), gen).to(torch.bfloat16)
        s["res"] = _randn((rows, n), gen)
        s["la"] = (_randn((na, rm, k), gen) / math.sqrt(k)).to(torch.bfloat16)
        s["lb"] = (0.1 * _randn((na, n, rm), gen)).to(torch.bfloat16)
        # half of the adapters use the whole rank, the others any rank below it
        r = torch.randint(1, rm + 1, (na,), generator=gen, device="cuda")
        s["rank"] = torch.where(torch.rand((na,), generator=gen, device="cuda") < 0.5, rm, r).to(torch.int32)
        s["lscale"] = 0.5 + torch.rand((na,), generator=gen, device="cuda")
        # requests in any order (one row each), or prompts one after another; -1: no adapter
        if case["mix"] == "each":
            a = torch.randint(-1, na, (rows,), generator=gen, device="cuda")
        else:
            run = max(1, rows // 9)
            a = torch.randint(-1, na, (rows // run + 1,), generator=gen, device="cuda").repeat_interleave(run)[:rows]
        s["adapter"] = a.to(torch.int32).contiguous()
    else:
        rows, e, h, i = case["rows"], case["e"], case["h"], case["i"]
        s["router"] = (0.02 * _randn((e + 1 if case["shared"] else e, h), gen)).to(torch.bfloat16)
        s["gu_q"], s["gu_s"] = _experts(e, 2 * i, h, case, gen)
        s["d_q"], s["d_s"] = _experts(e, h, i, case, gen)
        if case["shared"]:
            s["sgu_q"], s["sgu_s"] = _int8(2 * i, h, case["fmt"], gen)
            s["sd_q"], s["sd_s"] = _int8(h, i, case["fmt"], gen)
        s["x"] = _randn((rows, h), gen).to(torch.bfloat16)
        s["res"] = _randn((rows, h), gen)
    if own:
        _prepare_own(s, case)
    return s


# ---- the plain forms, float32 -----------------------------------------------------------------


def _rms(v, w):
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * w


def _norm_tail(s, b):
    n = b if s["pw"] is None else _rms(b, s["pw"])
    if s["cs"] is not None:
        n = n * s["cs"]
    if s["gate"] is not None:
        g = 1 / (1 + torch.exp(-s["gate"]))
        n = n * (g if g.dim() == 2 else g[:, None])
    xo = s["xscale"] * s["x"] + s["bscale"] * n
    return xo, _rms(xo, s["nw"]).to(torch.bfloat16)


def _deq8(q, s):
    w = q.float()
    if s.dim() == 1:
        return w * s.float()[:, None]
    return (w.view(w.shape[0], -1, 128) * s.float()[:, :, None]).view(w.shape)


def _deq(q, s, kind):
    """Experts [m, n, k] in float32 from the chosen experts' stored values and scales."""
    m, n = q.shape[:2]
    if kind == "q4":
        w = torch.stack([q & 15, q >> 4], -1).float().view(m, n, -1, 64)
        p = s.float()
        return (w * p[..., :1] + p[..., 1:]).view(m, n, -1)
    w = q.view(torch.float8_e4m3fn).float()
    k = w.shape[2]
    return (w.view(m, n // 128, 128, k // 128, 128) * s.float()[:, :, None, :, None]).view(m, n, k)


def _swiglu(g, u):
    return g / (1 + torch.exp(-g)) * u


def _plain_lora(s, case):
    x = s["x"].float()
    y = s["res"] + x @ _deq8(s["w"], s["s"]).t()
    col = torch.arange(case["rmax"], device="cuda")
    for a in range(case["adapters"]):
        keep = (s["adapter"] == a)[:, None] & (col < s["rank"][a])
        t = torch.where(keep, x @ s["la"][a].float().t(), 0.0) * s["lscale"][a]
        y = y + t @ s["lb"][a].float().t()
    return y


def _plain_moe(s, case):
    rows, e, i, k = case["rows"], case["e"], case["i"], case["topk"]
    # logits in 64 bits: a pick next to the border must not turn on a rounding
    logits = s["x"].double() @ s["router"].double().t()
    order = torch.sort(logits[:, :e], dim=-1, descending=True, stable=True)
    idx, top = order.indices[:, :k], order.values[:, :k]
    p = torch.exp(top - top[:, :1])
    wts = (p / p.sum(-1, keepdim=True)).float()
    x = s["x"].float()
    out = []
    for r in range(rows):
        pick = idx[r]
        gu = (_deq(s["gu_q"][pick], s["gu_s"][pick], case["kind"]) * x[r]).sum(-1)
        act = _swiglu(gu[:, :i], gu[:, i:])
        d = (_deq(s["d_q"][pick], s["d_s"][pick], case["kind"]) * act[:, None, :]).sum(-1)
        out.append((wts[r][:, None] * d).sum(0))
    y = s["res"] + torch.stack(out)
    if not case["shared"]:
        return y, idx.to(torch.int32), wts
    gu = x @ _deq8(s["sgu_q"], s["sgu_s"]).t()
    sh = _swiglu(gu[:, :i], gu[:, i:]) @ _deq8(s["sd_q"], s["sd_s"]).t()
    sg = logits[:, e].float()
    return y + sh / (1 + torch.exp(-sg))[:, None], idx.to(torch.int32), wts, sg


def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    if case["path"] == "norm":
        return _norm_tail(s, s["b"].float())
    if case["path"] == "combine":
        rows, topk = case["rows"], case["topk"]
        picked = s["y"][s["slot"].long()].view(rows, topk, -1)
        b = s["shared"] / (1 + torch.exp(-s["sgate"]))[:, None] + (s["wts"][:, :, None] * picked).sum(1)
        return _norm_tail(s, b)
    return _plain_lora(s, case) if case["path"] == "lora" else _plain_moe(s, case)


# ---- the library's calls ----------------------------------------------------------------------


def _lib():
    sys.path.insert(0, os.path.join(os.getcwd(), "drama-rs_amd"))
    import dramamoe

    return dramamoe


def _prepare_own(s, case):
    D = _lib()
    s["D"], s["lib"] = D, D.lib()
    empty = lambda shape, dt=torch.float32: torch.empty(shape, dtype=dt, device="cuda")
    rows = case["rows"]
    if case["path"] in ("norm", "combine"):
        s["xo"], s["hn"] = empty((rows, case["h"])), empty((rows, case["h"]), torch.bfloat16)
    elif case["path"] == "lora":
        n = s["lib"].dr_gemm_q8_lora_ws(rows, case["n"], case["k"], case["rmax"])
        s["ws"], s["out"] = torch.zeros(n, dtype=torch.uint8, device="cuda"), empty((rows, case["n"]))
    else:
        n = s["lib"].dr_moe_layer_rows_ws(rows, case["e"], case["h"], case["i"], case["topk"])
        s["ws"] = torch.zeros(n, dtype=torch.uint8, device="cuda")
        s["idx"], s["wts"] = empty((rows, case["topk"]), torch.int32), empty((rows, case["topk"]))
        s["sgate"], s["out"] = empty((rows,)), empty((rows, case["h"]))


def _own(s, case):
    P, lib, st, rows = s["D"].ptr, s["lib"], s["D"].stream_ptr(), case["rows"]
    if case["path"] in ("norm", "combine"):
        h = case["h"]
        tail = (P(s["x"]), h, P(s["pw"]), P(s["gate"]), case["gate"], h, P(s["cs"]), s["bscale"], s["xscale"], P(s["nw"]),
                EPS, P(s["xo"]), h, P(s["hn"]), h, rows, h, st)
        if case["path"] == "norm":
            (lib.dr_block_norm_bf16 if case["b16"] else lib.dr_block_norm)(P(s["b"]), h, *tail)
        else:
            lib.dr_moe_combine_norm(P(s["y"]), P(s["slot"]), P(s["wts"]), P(s["sgate"]), P(s["shared"]), case["topk"], *tail)
        return s["xo"], s["hn"]
    if case["path"] == "lora":
        f = lib.dr_gemm_q8_lora if case["fmt"] == "ref" else lib.dr_gemm_q8_lora_bf16s
        f(P(s["w"]), P(s["s"]), P(s["x"]), case["k"], P(s["adapter"]), P(s["la"]), P(s["lb"]), P(s["rank"]), P(s["lscale"]),
          case["adapters"], case["rmax"], P(s["ws"]), P(s["res"]), P(s["out"]), case["n"], rows, case["n"], case["k"], st)
        return s["out"]
    f = {("q4", "ref"): lib.dr_moe_layer_rows, ("q4", "cfg"): lib.dr_moe_layer_rows_bf16s,
         ("fp8", "ref"): lib.dr_moe_layer_rows_fp8, ("fp8", "cfg"): lib.dr_moe_layer_rows_fp8_bf16s}[case["kind"], case["fmt"]]
    sh = [P(s.get(a)) for a in ("sgu_q", "sgu_s", "sd_q", "sd_s")]
    f(P(s["router"]), P(s["gu_q"]), P(s["gu_s"]), P(s["d_q"]), P(s["d_s"]), *sh, P(s["x"]), P(s["res"]), P(s["idx"]),
      P(s["wts"]), P(s["sgate"]), P(s["ws"]), P(s["out"]), rows, case["e"], case["h"], case["i"], case["topk"], st)
    return (s["out"], s["idx"], s["wts"], s["sgate"]) if case["shared"] else (s["out"], s["idx"], s["wts"])


# ---- work and the definition in 64 bits -------------------------------------------------------


def work(case):
    rows = case["rows"]
    if case["path"] in ("norm", "combine"):
        n = rows * case["h"]
        vec = 4 * case["h"] * (1 + case["post"] + case["cs"])
        gate = {0: 0, 1: 4 * rows, 2: 4 * n}[case["gate"]]
        if case["path"] == "norm":
            return {"bytes": n * ((2 if case["b16"] else 4) + 4 + 4 + 2) + gate + vec, "flops": 12 * n}
        k = case["topk"]
        return {"bytes": n * (4 * (k + 1) + 4 + 4 + 2) + gate + vec + rows * (8 * k + 4), "flops": n * (12 + 2 * (k + 1))}
    if case["path"] == "lora":
        n, k, r = case["n"], case["k"], case["rmax"]
        # adapters that occur: all but in expectation, at three quarters of the largest rank
        groups = rows if case["mix"] == "each" else min(rows, 10)
        used = case["adapters"] * (1 - (1 - 1 / (case["adapters"] + 1)) ** groups)
        r = 0.75 * r
        on = rows * case["adapters"] / (case["adapters"] + 1)
        sc = 2 * n * (k // 128 if case["fmt"] == "ref" else 1)
        return {"bytes": int(n * k + sc + 2 * rows * k + 8 * rows * n + used * 2 * r * (n + k)),
                "flops": int(2 * rows * n * k + 2 * on * r * (n + k))}
    e, h, i, k = case["e"], case["h"], case["i"], min(case["topk"], case["e"])
    used = e * (1 - (1 - k / e) ** rows)
    w = 3 * h * i
    per = w // 2 + 4 * w // 64 if case["kind"] == "q4" else w + (4 if case["fmt"] == "ref" else 2) * w // (128 * 128)
    sh = w + (2 * w // 128 if case["fmt"] == "ref" else 2 * (2 * i + h)) if case["shared"] else 0
    rt = 2 * h * (e + case["shared"])
    return {"bytes": int(used * per + sh + rt + rows * h * 10 + rows * k * 8),
            "flops": int(2 * rows * (w * (k + case["shared"]) + h * (e + case["shared"])))}


def _exact_tail(s, b):
    d = lambda a: s[a].to(torch.float64)
    h = b.shape[1]
    if s["pw"] is not None:
        b = d("pw") * b / torch.sqrt(torch.linalg.vector_norm(b, dim=1, keepdim=True) ** 2 / h + EPS)
    scale = torch.full_like(b, s["bscale"])
    if s["cs"] is not None:
        scale = scale * d("cs")
    if s["gate"] is not None:
        scale = scale * torch.sigmoid(d("gate")).reshape(b.shape[0], -1)
    xo = s["xscale"] * d("x") + scale * b
    return xo, d("nw") * xo / torch.sqrt(torch.linalg.vector_norm(xo, dim=1, keepdim=True) ** 2 / h + EPS)


def _weights64(q, s, kind):
    """One matrix [n, k] in float64 from its stored form."""
    n = q.shape[0]
    if kind == "int8":
        k = q.shape[1]
        scale = s.double()[:, None].expand(n, k) if s.dim() == 1 else s.double().repeat_interleave(128, 1)
        return q.double() * scale
    if kind == "q4":
        w = torch.empty(n, 2 * q.shape[1], dtype=torch.float64, device=q.device)
        w[:, 0::2], w[:, 1::2] = (q % 16).double(), (q // 16).double()
        p = s.double().repeat_interleave(64, 1)
        return w * p[..., 0] + p[..., 1]
    c = q.int()
    ex, man = (c >> 3) & 15, (c & 7).double()
    mag = torch.where(ex == 0, man * 2.0 ** -9, (1 + man / 8) * torch.exp2((ex - 7).double()))
    return torch.where(c > 127, -mag, mag) * s.double().repeat_interleave(128, 0).repeat_interleave(128, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["path"] == "norm":
        return _exact_tail(s, s["b"].double())
    if case["path"] == "combine":
        rows, topk = case["rows"], case["topk"]
        b = s["shared"].double() * torch.sigmoid(s["sgate"].double())[:, None]
        slot = s["slot"].view(rows, topk).long()
        for k in range(topk):
            b += s["wts"][:, k:k + 1].double() * s["y"][slot[:, k]].double()
        return _exact_tail(s, b)
    if case["path"] == "lora":
        y = s["res"].double() + s["x"].double() @ _weights64(s["w"], s["s"], "int8").t()
        ids = s["adapter"].tolist()
        rank, scale = s["rank"].tolist(), s["lscale"].double()
        for a in sorted(set(ids) - {-1}):
            at = torch.tensor([r for r, v in enumerate(ids) if v == a], device="cuda")
            t = s["x"][at].double() @ s["la"][a, :rank[a]].double().t()
            y[at] += scale[a] * (t @ s["lb"][a, :, :rank[a]].double().t())
        return y
    rows, e, i, k = case["rows"], case["e"], case["i"], case["topk"]
    x = s["x"].double()
    logits = torch.stack([(s["router"].double() * x[r]).sum(1) for r in range(rows)])
    prob = torch.softmax(logits[:, :e], 1)
    picks = [sorted(range(e), key=lambda j: (-row[j], j))[:k] for row in logits.tolist()]
    idx = torch.tensor(picks, device="cuda")
    w = torch.gather(prob, 1, idx)
    w = w / w.sum(1, keepdim=True)

    def mlp(v, gu, down):
        z = v @ gu.t()
        return (z[:, :i] * torch.sigmoid(z[:, :i]) * z[:, i:]) @ down.t()

    y = s["res"].double()
    for j in sorted({p for row in picks for p in row}):
        at, slot = (idx == j).nonzero(as_tuple=True)
        gu, dn = _weights64(s["gu_q"][j], s["gu_s"][j], case["kind"]), _weights64(s["d_q"][j], s["d_s"][j], case["kind"])
        y[at] += w[at, slot][:, None] * mlp(x[at], gu, dn)
    if not case["shared"]:
        return y, idx.to(torch.int32), w
    y += torch.sigmoid(logits[:, e:]) * mlp(x, _weights64(s["sgu_q"], s["sgu_s"], "int8"), _weights64(s["sd_q"], s["sd_s"], "int8"))
    return y, idx.to(torch.int32), w, logits[:, e]

"""Operators around the matrix products of a token model's training step, as cases that can be timed one by one.

Three kinds, in the order in which a step meets them:

* `embed`: rows of a table looked up by token, scaled, and the table's gradient;
* `logp`: log probability of a given token of each row of logits, the rows' entropy and likeliest alternatives, and the
  logits' gradient;
* `adamw`: an AdamW step of all the parameters of an encoder, moments held in 32 bits or in 8.

Each has a plain form, written in elementary torch operations, and the call that a user of the package makes (`own`).
A case is a dict of plain values.  `listed()` names the fixed ones, `draw()` gives others of the same ranges.
"""
from __future__ import annotations

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
ESIZE = {"float32": 4, "float16": 2, "bfloat16": 2}


def listed():
    return [
        # the tests' encoder, batch 2 of 128: launches and host calls
        {"name": "embed_tiny", "kind": "embed", "vocab": 1000, "hidden": 64, "tokens": 256, "table": "float32",
         "out": "float32", "scale": 8.0, "padded": 0.0},
        # BERT-large's token table and a batch of 32 sequences of 384, activations in bf16
        {"name": "embed_bert", "kind": "embed", "vocab": 30522, "hidden": 1024, "tokens": 12288, "table": "float32",
         "out": "bfloat16", "scale": 1.0, "padded": 0.1},
        # a decoder's wide table kept in bf16, rows scaled by the root of their width, long batches with padding
        {"name": "embed_wide", "kind": "embed", "vocab": 131072, "hidden": 2048, "tokens": 65536, "table": "bfloat16",
         "out": "bfloat16", "scale": 45.25, "padded": 0.25},
        # widths that fit no vector, and many tokens for few rows (bytes as tokens)
        {"name": "embed_ragged", "kind": "embed", "vocab": 259, "hidden": 333, "tokens": 40001, "table": "float16",
         "out": "float16", "scale": 0.5, "padded": 0.0},
        # one generated token: its log probability and five alternatives
        {"name": "logp_decode", "kind": "logp", "rows": 1, "vocab": 30522, "dtype": "bfloat16", "top": 5, "grad": False,
         "masked": 0.0, "ignored": 0.0},
        # a batch of generated tokens over a wide vocabulary, twenty alternatives each
        {"name": "logp_score", "kind": "logp", "rows": 64, "vocab": 131072, "dtype": "bfloat16", "top": 20, "grad": False,
         "masked": 0.0, "ignored": 0.0},
        # training on a batch of 32 sequences of 128 with BERT's vocabulary, some tokens not scored
        {"name": "logp_train", "kind": "logp", "rows": 4096, "vocab": 30522, "dtype": "bfloat16", "top": 0, "grad": True,
         "masked": 0.0, "ignored": 0.15},
        # fp32 logits of an odd vocabulary, of which a grammar forbids a part: policy gradients with an entropy bonus
        {"name": "logp_ragged", "kind": "logp", "rows": 517, "vocab": 32003, "dtype": "float32", "top": 8, "grad": True,
         "masked": 0.3, "ignored": 0.0},
        # the tests' encoder
        {"name": "adamw_tiny", "kind": "adamw", "vocab": 1000, "hidden": 64, "layers": 2, "ffn": 128, "param": "float32",
         "grad": "float32", "bits": 32, "copies": False, "packed": False},
        # BERT-large with the bf16 copies that its forward pass reads
        {"name": "adamw_bert", "kind": "adamw", "vocab": 30522, "hidden": 1024, "layers": 24, "ffn": 4096,
         "param": "float32", "grad": "float32", "bits": 32, "copies": True, "packed": False},
        # a third of its layers, moments in 8 bits
        {"name": "adamw_bert8", "kind": "adamw", "vocab": 30522, "hidden": 1024, "layers": 8, "ffn": 4096,
         "param": "float32", "grad": "float32", "bits": 8, "copies": False, "packed": False},
        # weights and gradients in bf16, sizes that fit no block
        {"name": "adamw_half8", "kind": "adamw", "vocab": 8191, "hidden": 330, "layers": 6, "ffn": 1111,
         "param": "bfloat16", "grad": "bfloat16", "bits": 8, "copies": False, "packed": False},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["embed", "logp", "adamw"])
    dtype = rng.choice(list(DTYPES))
    if kind == "embed":
        hidden = _log(rng, 16, 2048)
        if rng.random() < 0.6:
            hidden = max(16, hidden // 16 * 16)
        return {"kind": kind, "vocab": _log(rng, 100, 131072), "hidden": hidden, "tokens": _log(rng, 1, 65536), "table": dtype,
                "out": rng.choice([dtype, "bfloat16"]), "scale": rng.choice([1.0, 0.5, 22.625]),
                "padded": rng.choice([0.0, 0.0, 0.2, 0.9])}
    if kind == "logp":
        vocab = _log(rng, 64, 131072)
        return {"kind": kind, "rows": _log(rng, 1, max(2, 120_000_000 // vocab)), "vocab": vocab, "dtype": dtype,
                "top": rng.choice([0, 1, 5, 20]), "grad": rng.random() < 0.6, "masked": rng.choice([0.0, 0.0, 0.5]),
                "ignored": rng.choice([0.0, 0.0, 0.4])}
    hidden = _log(rng, 32, 1024)
    bits = rng.choice([8, 32])
    param = rng.choice(["float32", "float32", dtype])
    return {"kind": kind, "vocab": _log(rng, 100, 31000), "hidden": hidden, "layers": rng.randint(1, 8), "ffn": _log(rng, 32, 4096),
            "param": param, "grad": param if param != "float32" else rng.choice(["float32", "bfloat16"]), "bits": bits,
            "copies": param == "float32" and rng.random() < 0.4, "packed": bits == 32 and rng.random() < 0.3}


# ---- embed ---------------------------------------------------------------------------------------
def _prepare_embed(c, g):
    V, H, T = c["vocab"], c["hidden"], c["tokens"]
    # tokens of a text: the n-th most frequent one about 1 / n as often as the first, anywhere in the table
    rank = torch.exp(torch.rand(T, generator=g, device="cuda", dtype=torch.float64) * torch.log(torch.tensor(float(V)))).long() - 1
    ids = (rank.clamp_(0, V - 1) * 7919 + 13) % V
    ids = torch.where(torch.rand(T, generator=g, device="cuda") < c["padded"], torch.zeros_like(ids), ids)
    table = (torch.randn(V, H, generator=g, device="cuda") * 0.02).to(DTYPES[c["table"]])
    dout = torch.randn(T, H, generator=g, device="cuda").to(DTYPES[c["out"]])
    return {"ids": ids, "table": table.requires_grad_(), "dout": dout, "padding": 0 if c["padded"] else None}


def _run_embed(c, s):
    ids, table, dout = s["ids"], s["table"], s["dout"]
    out_type = DTYPES[c["out"]]
    if own:
        from bagua_core_b200 import ops

        out = ops.embedding(ids, table, scale=c["scale"], padding_idx=s["padding"], dtype=out_type)
        return {"out": out.detach(), "dtable": torch.autograd.grad(out, table, dout)[0]}
    w = table.detach()
    out = (w[ids].float() * c["scale"]).to(out_type)
    # sums over thousands of equal tokens: in 64 bits
    sums = torch.zeros(w.shape, dtype=torch.float64, device=w.device).index_add_(0, ids, dout.double())
    if s["padding"] is not None:
        sums[s["padding"]] = 0
    return {"out": out, "dtable": (sums * c["scale"]).to(w.dtype)}


def _exact_embed(c, s):
    ids, table = s["ids"], s["table"].detach()
    out = table.double().index_select(0, ids) * c["scale"]
    order = torch.argsort(ids, stable=True)
    sums = torch.zeros(table.shape, dtype=torch.float64, device="cuda")
    counts = torch.bincount(ids, minlength=c["vocab"])
    if c["hidden"] * c["tokens"] > 200_000_000:
        return None
    sums[:] = torch.segment_reduce(s["dout"][order].double(), "sum", lengths=counts, axis=0, unsafe=True)
    if s["padding"] is not None:
        sums[s["padding"]] = 0
    return {"out": out, "dtable": sums * c["scale"]}


def _work_embed(c):
    V, H, T = c["vocab"], c["hidden"], c["tokens"]
    t, o = ESIZE[c["table"]], ESIZE[c["out"]]
    rows = min(V, T)  # of the table, read once each
    return {"bytes": 8 * T + rows * H * t + T * H * o + 8 * T + T * H * o + V * H * t, "flops": 2.0 * T * H}


# ---- logp ----------------------------------------------------------------------------------------
def _prepare_logp(c, g):
    N, V = c["rows"], c["vocab"]
    x = torch.randn(N, V, generator=g, device="cuda")
    # some rows are sure of a token, some of nothing
    x *= 0.5 + 3.0 * torch.rand(N, 1, generator=g, device="cuda")
    targets = torch.randint(0, V, (N,), generator=g, device="cuda")
    x.scatter_add_(1, targets[:, None], 8.0 * torch.rand(N, 1, generator=g, device="cuda"))
    if c["masked"]:
        x.masked_fill_(torch.rand(N, V, generator=g, device="cuda") < c["masked"], float("-inf"))
    targets = torch.where(torch.rand(N, generator=g, device="cuda") < c["ignored"], torch.full_like(targets, -100), targets)
    weight = torch.randn(N, generator=g, device="cuda") / N
    return {"logits": x.to(DTYPES[c["dtype"]]).requires_grad_(c["grad"]), "targets": targets, "dlogp": weight,
            "dentropy": torch.full((N,), 0.01 / N, device="cuda")}


def _run_logp(c, s):
    logits, targets, top = s["logits"], s["targets"], c["top"]
    if own:
        from bagua_core_b200 import ops

        r = ops.token_log_probs(logits, targets, top=top)
        got = {"logp": r.log_probs.detach(), "entropy": r.entropy.detach()}
        if top:
            got["top"], got["ids"] = r.top_log_probs, r.top_ids
        if c["grad"]:
            got["dlogits"] = torch.autograd.grad((r.log_probs, r.entropy), logits, (s["dlogp"], s["dentropy"]))[0]
        return got
    x = logits.detach().float()
    scored = targets != -100
    t = targets.clamp(min=0)[:, None]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = m + torch.log(z)
    p = e / z
    lp = x - lse
    logp = lp.gather(1, t)[:, 0]
    entropy = -(p * lp.clamp(min=-1e30)).sum(1)
    got = {"logp": torch.where(scored, logp, 0.0), "entropy": torch.where(scored, entropy, 0.0)}
    if top:
        best, ids = torch.sort(logits.detach(), dim=1, descending=True, stable=True)  # equal ones in the order of their places
        got["top"] = torch.where(scored[:, None], best[:, :top].float() - lse, float("-inf"))
        got["ids"] = torch.where(scored[:, None], ids[:, :top], -1)
    if c["grad"]:
        a = torch.where(scored, s["dlogp"], 0.0)[:, None]
        b = torch.where(scored, s["dentropy"], 0.0)[:, None]
        d = -p * (a + b * (lp.clamp(min=-1e30) + entropy[:, None]))
        got["dlogits"] = d.scatter_add_(1, t, a).to(logits.dtype)
    return got


def _exact_logp(c, s):
    logits, targets = s["logits"].detach(), s["targets"]
    parts = []
    for lo in range(0, c["rows"], 1024):
        x, y = logits[lo:lo + 1024].double(), targets[lo:lo + 1024]
        on = (y >= 0).double()
        lp = torch.log_softmax(x, 1)
        p = lp.exp()
        plogp = torch.where(p > 0, p * lp, torch.zeros_like(p))
        h = -plogp.sum(1)
        hit = torch.zeros_like(x).scatter_(1, y.clamp(min=0)[:, None], 1.0)
        one = {"logp": torch.where(y >= 0, lp.gather(1, y.clamp(min=0)[:, None])[:, 0], 0.0), "entropy": h * on}
        if c["top"]:
            one["top"] = torch.where(y[:, None] >= 0, lp.topk(c["top"], dim=1).values, float("-inf"))
        if c["grad"]:
            a, b = s["dlogp"][lo:lo + 1024].double() * on, s["dentropy"][lo:lo + 1024].double() * on
            one["dlogits"] = a[:, None] * (hit - p) - b[:, None] * (plogp + p * h[:, None])
        parts.append(one)
    got = {k: torch.cat([q[k] for q in parts]) for k in parts[0]}
    if c["top"]:
        got["ids"] = None
    return got


def _work_logp(c):
    N, V, e = c["rows"], c["vocab"], ESIZE[c["dtype"]]
    scored = round(N * (1 - c["ignored"]))
    moved = scored * V * e + N * (16 + 12 * c["top"])
    if c["grad"]:
        moved += scored * V * e + N * V * e + 8 * N
    return {"bytes": moved, "flops": scored * V * (6.0 + (8.0 if c["grad"] else 0.0))}


# ---- adamw ---------------------------------------------------------------------------------------
BETAS, EPS, LR, DECAY = (0.9, 0.999), 1e-8, 5e-5, 0.01
BLOCK = 256  # elements that share a scale, of a moment held in 8 bits


def _shapes(c):
    V, h, f = c["vocab"], c["hidden"], c["ffn"]
    layer = [(3 * h, h), (3 * h,), (h, h), (h,), (h,), (h,), (f, h), (f,), (h, f), (h,), (h,), (h,)]
    return [(V, h), (512, h), (2, h), (h,), (h,)] + layer * c["layers"] + [(2, h), (2,)]


def _layout(c):
    """(sizes, offsets, length of a flat buffer that holds them all)."""
    sizes = [s[0] * s[1] if len(s) == 2 else s[0] for s in _shapes(c)]
    offsets, at = [], 0
    for n in sizes:
        offsets.append(at)
        at += n if c["packed"] else (n + BLOCK - 1) // BLOCK * BLOCK
    return sizes, offsets, at


def _mix(x):
    """A bijection of 32 bits whose every output bit depends on every input bit."""
    M = 0xFFFFFFFF
    x = x ^ (x >> 16)
    x = x * 0x7FEB352D & M
    x = x ^ (x >> 15)
    x = x * 0x846CA68B & M
    return x ^ (x >> 16)


def _read8(code, scale):
    """The values of 8-bit moments: (first, second), from codes and the scales [2, blocks] of their blocks.  Both are small floating
    point numbers with 4 bits of exponent: a sign and 3 bits behind it, or no sign and 4 bits."""
    m, v = code[0].long(), code[1].long()
    e, f = (m >> 3) & 15, (m & 7).double()
    first = torch.where(e > 0, (8 + f) * 2.0 ** (e - 10).double(), f * 2.0 ** -9)
    first = torch.where(m > 127, -first, first)
    e, f = v >> 4, (v & 15).double()
    second = torch.where(e > 0, (16 + f) * 2.0 ** (e - 11).double(), f * 2.0 ** -10)
    return ((first.view(-1, BLOCK) * scale[0].double()[:, None]).view(-1), (second.view(-1, BLOCK) * scale[1].double()[:, None]).view(-1))


def _write8(m, v, bits):
    """(codes of the first moment, of the second, scales): of two neighbouring values the upper one is taken with the probability
    that keeps the mean, decided by 16 of 32 random bits each."""
    tiny = 2.0 ** -126
    top_m, top_v = m.abs().view(-1, BLOCK).amax(1), v.view(-1, BLOCK).amax(1)
    scale = torch.stack([(top_m.float() / 480).clamp(min=tiny) * (top_m > 0), (top_v.float() / 496).clamp(min=tiny) * (top_v > 0)])
    per = scale.double().clamp(min=tiny)
    y = [(m.abs().view(-1, BLOCK) / per[0][:, None]).view(-1), (v.view(-1, BLOCK) / per[1][:, None]).view(-1)]
    codes = []
    for x, half, r in ((y[0], 8, bits & 0xFFFF), (y[1], 16, bits >> 16)):
        e = (torch.frexp(x)[1] - 1).clamp(min=-6).masked_fill_(x == 0, -6)  # zero has no exponent: its code is 0
        q = torch.floor(x * half * torch.ldexp(torch.ones_like(x), -e) + (r.double() + 0.5) / 65536)
        codes.append((e + 6) * half + q.long())
    first = codes[0].clamp(max=127) + 128 * (m < 0)
    # a second moment that is not zero does not become zero: the step divides by it
    second = torch.where(v > 0, codes[1].clamp(1, 255), torch.zeros_like(codes[1]))
    return first.to(torch.uint8), second.to(torch.uint8), scale


def _prepare_adamw(c, g):
    sizes, offsets, n = _layout(c)
    p = torch.randn(n, generator=g, device="cuda").mul_(0.02)
    # gradients of tensors, and of rows of a tensor, differ by orders of magnitude
    size = torch.exp(torch.randn((n + 4095) // 4096, generator=g, device="cuda") * 1.5 - 8).repeat_interleave(4096)[:n]
    grad = torch.randn(n, generator=g, device="cuda").mul_(size)
    m = torch.randn(n, generator=g, device="cuda").mul_(size).mul_(0.3)
    v = torch.randn(n, generator=g, device="cuda").square_().mul_(0.1).add_(0.9).mul_(size).mul_(size)
    del size
    if not c["packed"]:  # nothing between the tensors
        inside = torch.zeros(n, dtype=torch.bool, device="cuda")
        for k, lo in zip(sizes, offsets):
            inside[lo:lo + k] = True
        for t in (p, grad, m, v):
            t.mul_(inside)
        del inside
    s = {"p": p.to(DTYPES[c["param"]]), "g": grad.to(DTYPES[c["grad"]]), "step": 100, "seed": 20_011}
    flat = ["p", "g"]
    if c["bits"] == 8:
        rows = torch.tensor([(k + BLOCK - 1) // BLOCK for k in sizes], device="cuda")
        s["tensor"] = torch.arange(len(sizes), device="cuda").repeat_interleave(rows)  # of each block
        s["block"] = torch.arange(n // BLOCK, device="cuda") - (rows.cumsum(0) - rows)[s["tensor"]]
        s["tensors"] = torch.arange(len(sizes), device="cuda")
        s["m"], s["v"], scale = _write8(m.double(), v.double(), torch.full((n,), 0x7FFF7FFF, device="cuda", dtype=torch.int64))
        s["scales"] = scale
        s["scale"] = [scale[:, lo // BLOCK:(lo + k + BLOCK - 1) // BLOCK] for k, lo in zip(sizes, offsets)]
        s["m_read"], s["v_read"] = (torch.zeros(n, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        flat += ["m_read", "v_read"]
    else:
        s["m"], s["v"] = m, v
    if c["copies"]:
        s["copy"] = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
        flat.append("copy")
    for name in flat + ["m", "v"]:
        s[name + "s"] = [s[name][lo:lo + k] for k, lo in zip(sizes, offsets)]
    return s


def _run_adamw(c, s):
    s["step"] += 1
    t = s["step"]
    copies = {"copy": s["copy"]} if c["copies"] else {}
    if own:
        from bagua_core_b200 import ops

        ops.adamw_step(s["ps"], s["gs"], s["ms"], s["vs"], step=t, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
                       scales=s.get("scale"), copies=s.get("copys"), seed=s["seed"])
        if c["bits"] == 8:
            ops.adamw_read8(s["ms"], s["vs"], s["scale"], s["m_reads"], s["v_reads"])
            return {"p": s["p"], "m": s["m_read"], "v": s["v_read"], "scales": s["scales"], **copies}
        return {"p": s["p"], "m": s["m"], "v": s["v"], **copies}
    c1, c2 = 1 - BETAS[0] ** t, 1 - BETAS[1] ** t
    if c["bits"] == 8:  # in 64 bits: a value next to the border between two codes
        old_m, old_v = _read8((s["m"], s["v"]), s["scales"])
        g = s["g"].double()
        m = old_m * BETAS[0] + g * (1 - BETAS[0])
        v = old_v * BETAS[1] + g * g * (1 - BETAS[1])
        p = s["p"].double() * (1 - LR * DECAY) - LR / c1 * m / (torch.sqrt(v / c2) + EPS)
        key = _mix(_mix(_mix(torch.tensor(s["seed"], device="cuda")) + t & 0xFFFFFFFF) + s["tensors"] & 0xFFFFFFFF)
        place = s["block"][:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
        bits = _mix(place * 0x9E3779B9 + key[s["tensor"]][:, None] & 0xFFFFFFFF).view(-1)
        code_m, code_v, scale = _write8(m, v, bits)
        s["m"].copy_(code_m), s["v"].copy_(code_v), s["scales"].copy_(scale)
        new_m, new_v = _read8((s["m"], s["v"]), s["scales"])
        s["m_read"].copy_(new_m), s["v_read"].copy_(new_v)
        s["p"].copy_(p)
        got = {"p": s["p"], "m": s["m_read"], "v": s["v_read"], "scales": s["scales"]}
    else:
        g, m, v = s["g"].float(), s["m"], s["v"]
        m.mul_(BETAS[0]).add_(g * (1 - BETAS[0]))
        v.mul_(BETAS[1]).add_(g * g * (1 - BETAS[1]))
        p = s["p"].float() * (1 - LR * DECAY) - LR / c1 * m / (torch.sqrt(v / c2) + EPS)
        s["p"].copy_(p)
        got = {"p": s["p"], "m": m, "v": v}
    if c["copies"]:
        s["copy"].copy_(s["p"])
    return {**got, **copies}


def _exact_adamw(c, s):
    t = s["step"] + 1
    p, g = s["p"].double(), s["g"].double()
    if c["bits"] == 8:
        table_m = torch.tensor([(k % 8 + 8 * (k > 7)) * 2.0 ** (max(k // 8, 1) - 10) for k in range(128)], dtype=torch.float64, device="cuda")
        table_v = torch.tensor([(k % 16 + 16 * (k > 15)) * 2.0 ** (max(k // 16, 1) - 11) for k in range(256)], dtype=torch.float64, device="cuda")
        scale = s["scales"].double().repeat_interleave(BLOCK, dim=1)
        code = s["m"].long()
        m0 = torch.where(code >= 128, -table_m[code % 128], table_m[code % 128]) * scale[0]
        v0 = table_v[s["v"].long()] * scale[1]
    else:
        m0, v0 = s["m"].double(), s["v"].double()
    m = m0 + (1 - BETAS[0]) * (g - m0)
    v = v0 + (1 - BETAS[1]) * (g * g - v0)
    p = p - LR * DECAY * p - LR * (m / (1 - BETAS[0] ** t)) / ((v / (1 - BETAS[1] ** t)).sqrt() + EPS)
    got = {"p": p, "m": m, "v": v}
    if c["copies"]:
        got["copy"] = p
    if c["bits"] == 32:
        return got
    big = torch.stack([m.abs().view(-1, BLOCK).amax(1) / 480, v.view(-1, BLOCK).amax(1) / 496])
    got["scales"] = big
    per = torch.where(big > 0, big, torch.ones_like(big)).float().double().repeat_interleave(BLOCK, dim=1)
    place = (s["block"][:, None] * BLOCK + torch.arange(BLOCK, device="cuda")).view(-1)
    key = _mix(_mix(_mix(torch.tensor(s["seed"], device="cuda")) + t & 0xFFFFFFFF) + s["tensors"] & 0xFFFFFFFF)
    random = _mix(place * 0x9E3779B9 + key[s["tensor"].repeat_interleave(BLOCK)] & 0xFFFFFFFF)
    for name, x, table, row, part in (("m", m, table_m, 0, random & 0xFFFF), ("v", v, table_v, 1, random >> 16)):
        y = x.abs() / per[row]
        below = (torch.searchsorted(table, y, right=True) - 1).clamp(0, len(table) - 2)
        up = (y - table[below]) / (table[below + 1] - table[below]) + (part.double() + 0.5) / 65536 >= 1
        k = below + up
        if name == "v":
            k = torch.where(x > 0, k.clamp(min=1), k)
        got[name] = torch.sign(x) * table[k] * per[row]
    return got


def _work_adamw(c):
    n = sum(_layout(c)[0])
    moments = 8 * 2 if c["bits"] == 32 else 2 * 2 + 2 + 4  # read and written; in 8 bits read back too, into bf16
    return {"bytes": n * (2 * ESIZE[c["param"]] + ESIZE[c["grad"]] + moments + 2 * c["copies"]), "flops": 16.0 * n}


# ---- the cases' interface ------------------------------------------------------------------------
_PREPARE = {"embed": _prepare_embed, "logp": _prepare_logp, "adamw": _prepare_adamw}
_RUN = {"embed": _run_embed, "logp": _run_logp, "adamw": _run_adamw}
_EXACT = {"embed": _exact_embed, "logp": _exact_logp, "adamw": _exact_adamw}
_WORK = {"embed": _work_embed, "logp": _work_logp, "adamw": _work_adamw}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"case": case, **_PREPARE[case["kind"]](case, g)}


def run(state):
    return _RUN[state["case"]["kind"]](state["case"], state)


def exact(case, seed):
    return _EXACT[case["kind"]](case, prepare(case, seed))


def work(case):
    return _WORK[case["kind"]](case)

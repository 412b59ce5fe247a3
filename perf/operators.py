"""The serving operators around the quantized projections: the paged key/value cache, the attention that reads it, prompt
attention, and the sampler behind the output head.  ``run`` computes them in elementary torch operations (``own`` false)
or through the library's entry points (``own`` true); ``exact`` computes them from their definitions in 64 bits."""
import functools
import math
import random

import torch

own = False
DEV = "cuda" if torch.cuda.is_available() else "cpu"
FP8_MAX = 448.0


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 64 sequences: rotate q and k, write one token per sequence (hidden 7168 = 56 heads of 128)
        {"name": "append_step", "op": "append", "tokens": 64, "seqs": 64, "hq": 56, "hkv": 8, "d": 128, "page": 64, "pages": 8, "fp8": False,
         "rot": 128, "off": 0, "half": False},
        # the cache write of a 16384-token prompt batch into an e4m3 cache, rotation on the last 64 columns of a head
        {"name": "append_prompt_fp8", "op": "append", "tokens": 16384, "seqs": 5, "hq": 56, "hkv": 8, "d": 128, "page": 64, "pages": 60,
         "fp8": True, "rot": 64, "off": 64, "half": False},
        # a lone short chat: latency only
        {"name": "decode_short", "op": "decode", "seqs": 1, "lo": 333, "hi": 333, "lens": 0, "hq": 16, "hkv": 2, "d": 64, "page": 16,
         "fp8": False, "window": 0},
        # the 64-token decode batch with ragged contexts, seven query heads per cache head
        {"name": "decode_batch", "op": "decode", "seqs": 64, "lo": 1, "hi": 8192, "lens": 1, "hq": 56, "hkv": 8, "d": 128, "page": 64,
         "fp8": False, "window": 0},
        # one sequence with a very long context: the split over the cache's length
        {"name": "decode_long", "op": "decode", "seqs": 1, "lo": 131071, "hi": 131071, "lens": 0, "hq": 56, "hkv": 8, "d": 128, "page": 64,
         "fp8": False, "window": 0},
        # a large batch over an e4m3 cache with small pages
        {"name": "decode_fp8", "op": "decode", "seqs": 128, "lo": 512, "hi": 16384, "lens": 2, "hq": 64, "hkv": 8, "d": 128, "page": 32,
         "fp8": True, "window": 0},
        # a few short prompts packed together
        {"name": "prompt_short", "op": "prompt", "seqs": 7, "lo": 1, "hi": 300, "lens": 3, "hq": 8, "hkv": 2, "d": 64, "window": 0},
        # a prefill batch of ragged documents
        {"name": "prompt_packed", "op": "prompt", "seqs": 9, "lo": 900, "hi": 2600, "lens": 4, "hq": 56, "hkv": 8, "d": 128, "window": 0},
        # one long prompt
        {"name": "prompt_long", "op": "prompt", "seqs": 1, "lo": 8192, "hi": 8192, "lens": 0, "hq": 56, "hkv": 8, "d": 128, "window": 0},
        # the sampler for a lone token over the output head's 129280 logits
        {"name": "sample_one", "op": "sample", "rows": 1, "n": 129280, "mix": 0},
        # ... and for the 64-token batch, every row with settings of its own
        {"name": "sample_batch", "op": "sample", "rows": 64, "n": 129280, "mix": 1},
        # an odd vocabulary in rows with padding behind them
        {"name": "sample_odd", "op": "sample", "rows": 13, "n": 50021, "mix": 1},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prompt", "prompt", "sample"])
    d = rng.choice([64, 128])
    hkv = rng.choice([1, 2, 3, 4, 8])
    hq = hkv * rng.choice([1, 2, 4, 5, 7, 8])
    if op == "append":
        seqs = _log_int(rng, 1, 64)
        page = rng.choice([16, 32, 64, 128])
        pages = rng.randint(1, 16)
        rot = rng.choice([32, 64, d])
        return {"op": op, "tokens": _log_int(rng, 1, seqs * pages * page), "seqs": seqs, "hq": hq, "hkv": hkv, "d": d, "page": page, "pages": pages,
                "fp8": rng.random() < 0.5, "rot": rot, "off": rng.choice([0, d - rot]), "half": rng.random() < 0.5}
    if op == "decode":
        seqs = _log_int(rng, 1, 100)
        hi = _log_int(rng, 1, min(60000, 400000 // seqs))
        return {"op": op, "seqs": seqs, "lo": rng.randint(0, hi), "hi": hi, "lens": rng.randrange(1 << 30), "hq": hq, "hkv": hkv, "d": d,
                "page": rng.choice([16, 32, 64, 128]), "fp8": rng.random() < 0.5, "window": rng.choice([0, 0, 128, _log_int(rng, 1, 4096)])}
    if op == "prompt":
        seqs = _log_int(rng, 1, 12)
        hi = _log_int(rng, 1, 2500)
        return {"op": op, "seqs": seqs, "lo": rng.randint(0, hi), "hi": hi, "lens": rng.randrange(1 << 30), "hq": hq, "hkv": hkv, "d": d,
                "window": rng.choice([0, 0, 128, _log_int(rng, 1, 2000)])}
    return {"op": op, "rows": _log_int(rng, 1, 64), "n": _log_int(rng, 1000, 131072), "mix": 1 + rng.randrange(1 << 30)}


def _lens(c):
    """The sequences' lengths: part of the case's shape, the same for every seed."""
    r = random.Random(c["lens"])
    lens = [r.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]
    return lens[:-1] + [max(1, lens[-1])]


def _visible(n, w):
    """(query, key) pairs of a causal prompt of n tokens with window w (0: none)."""
    w = n if w == 0 else min(w, n)
    return w * (w + 1) // 2 + (n - w) * w


def work(c):
    if c["op"] == "append":
        t, es = c["tokens"], 1 if c["fp8"] else 2
        per = c["d"] * (2 * 2 * c["hq"] + 2 * 2 * c["hkv"] + 2 * es * c["hkv"]) + 8 * (c["rot"] // 2) + 12
        return {"bytes": t * per, "flops": t * (c["hq"] + c["hkv"]) * c["rot"] * 3}
    if c["op"] == "decode":
        w = c["window"]
        toks = sum(min(n, w) if w else n for n in _lens(c))
        es = 1 if c["fp8"] else 2
        return {"bytes": 2 * toks * c["hkv"] * c["d"] * es + c["seqs"] * c["hq"] * (4 * c["d"] + 4) + 4 * (toks // c["page"] + 2 * c["seqs"]),
                "flops": 4 * toks * c["hq"] * c["d"]}
    if c["op"] == "prompt":
        lens = _lens(c)
        return {"bytes": sum(lens) * (c["d"] * 2 * (2 * c["hq"] + 2 * c["hkv"]) + 4 * c["hq"]),
                "flops": 4 * c["d"] * c["hq"] * sum(_visible(n, c["window"]) for n in lens)}
    return {"bytes": c["rows"] * (4 * c["n"] + 28), "flops": c["rows"] * c["n"] * 4}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _bf16(g, *shape, std=1.0):
    return torch.empty(*shape, dtype=torch.bfloat16, device=DEV).normal_(0.0, std, generator=g)


def _cache(c, g, n_pages):
    """(k, v, k_scale, v_scale): [pages][kv heads][page][d] filled with what an earlier part of the dialogue left there."""
    shape = (n_pages, c["hkv"], c["page"], c["d"])
    k, v = _bf16(g, *shape), _bf16(g, *shape)
    if not c["fp8"]:
        return k, v, None, None
    scale = [torch.empty(c["hkv"], device=DEV).uniform_(0.01, 0.03, generator=g) for _ in range(2)]
    k, v = ((x / s[:, None, None]).clamp_(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn) for x, s in zip((k, v), scale))
    return k, v, scale[0], scale[1]


def prepare(c, seed):
    g, op = _gen(seed), c["op"]
    s = {"c": c}
    if op == "append":
        t, cap = c["tokens"], c["pages"] * c["page"]
        # a merged q/k/v projection's rows, the three parts side by side
        rows = _bf16(g, t, (c["hq"] + 2 * c["hkv"]) * c["d"])
        s["q"], s["k"], s["v"] = rows.split([c["hq"] * c["d"], c["hkv"] * c["d"], c["hkv"] * c["d"]], dim=1)
        n_pages = c["seqs"] * c["pages"] + 3
        s["table"] = torch.randperm(n_pages, generator=g, device=DEV)[: c["seqs"] * c["pages"]].reshape(c["seqs"], c["pages"]).int()
        # distinct slots: every sequence takes a run of positions from a start of its own
        at = torch.arange(t, device=DEV)
        s["seq"] = (at % c["seqs"]).int()
        per = -(-t // c["seqs"])
        start = (torch.rand(c["seqs"], generator=g, device=DEV) * (cap - per + 1)).long().clamp_(0, cap - per)
        s["pos"] = (start[s["seq"].long()] + at // c["seqs"]).int()
        angle = torch.arange(cap, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(c["rot"] // 2, device=DEV, dtype=torch.float64) * 2 / c["rot"])
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["ck"], s["cv"], s["ks"], s["vs"] = _cache(c, g, n_pages)
        s["q_out"] = torch.empty(t, c["hq"] * c["d"], dtype=torch.bfloat16, device=DEV)
    elif op == "decode":
        lens = _lens(c)
        per = [max(1, -(-n // c["page"])) for n in lens]
        n_pages = sum(per) + 5
        order = torch.randperm(n_pages, generator=g, device=DEV).int()
        s["table"] = torch.zeros(c["seqs"], max(per), dtype=torch.int32, device=DEV)
        ends = [0]
        for i, n in enumerate(per):
            s["table"][i, :n] = order[ends[-1]: ends[-1] + n]
            ends.append(ends[-1] + n)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["ck"], s["cv"], s["ks"], s["vs"] = _cache(c, g, n_pages)
        s["q"] = _bf16(g, c["seqs"], c["hq"] * c["d"], std=1.5)
    elif op == "prompt":
        lens = _lens(c)
        t = sum(lens)
        rows = _bf16(g, t, (c["hq"] + 2 * c["hkv"]) * c["d"])
        s["q"], s["k"], s["v"] = rows.split([c["hq"] * c["d"], c["hkv"] * c["d"], c["hkv"] * c["d"]], dim=1)
        s["cu"] = torch.tensor([0] + [sum(lens[: i + 1]) for i in range(len(lens))], dtype=torch.int32, device=DEV)
        s["longest"] = max(lens)
    else:
        m, n = c["rows"], c["n"]
        rows = torch.empty(m, n + 7 if n % 2 else n, device=DEV).normal_(0.0, 2.0, generator=g)
        # a few likely tokens stand out, as behind a trained output head
        lucky = torch.randint(0, n, (m, 24), generator=g, device=DEV)
        rows.scatter_add_(1, lucky, torch.empty(m, 24, device=DEV).uniform_(4.0, 12.0, generator=g))
        s["logits"] = rows[:, :n]
        s["u"] = torch.rand(m, generator=g, device=DEV)
        r = random.Random(c["mix"])
        pick = (lambda *v: [r.choice(v) for _ in range(m)]) if c["mix"] else (lambda *v: [v[0]] * m)
        s["temperature"] = torch.tensor(pick(0.8, 1.0, 0.6, 1.3, 0.0), device=DEV)
        s["top_k"] = torch.tensor(pick(50, 0, 1, 20, 1000), dtype=torch.int32, device=DEV)
        s["top_p"] = torch.tensor(pick(0.95, 1.0, 0.9, 0.5, 0.99), device=DEV)
        s["min_p"] = torch.tensor(pick(0.02, 0.0, 0.0, 0.1, 0.001), device=DEV)
    if own and op in ("append", "decode"):
        # the handle over the cache's memory that a program keeps next to it
        ctx = _handle()
        code = (lambda x: x.view(torch.uint8)) if c["fp8"] else (lambda x: x)
        s["cache"] = ctx.pkg.KvCache(ctx, code(s["ck"]), code(s["cv"]), s["ks"], s["vs"])
    return s


@functools.cache
def _handle():
    from __graft_entry__ import load_package
    pkg = load_package()
    ctx = pkg.Ctx(torch.cuda.current_device())
    ctx.pkg = pkg
    return ctx


# ------------------------------------------------------------------ one pass
def run(s):
    return {"append": _append, "decode": _decode, "prompt": _prompt, "sample": _sample}[s["c"]["op"]](s)


def _rotate(x, cos, sin, off, half):
    """x [t][heads][d]; cos, sin [t][rot / 2]: the pairs of columns [off, off + rot) turned by their angles."""
    rot = 2 * cos.shape[1]
    part = x[..., off: off + rot]
    a, b = (part[..., : rot // 2], part[..., rot // 2:]) if half else (part[..., 0::2], part[..., 1::2])
    cos, sin = cos[:, None], sin[:, None]
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([a, b], -1) if half else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([x[..., :off], turned, x[..., off + rot:]], -1)


def _append(s):
    c = s["c"]
    if own:
        ctx = _handle()
        ctx.pkg.kv_append(ctx, s["cache"], s["k"], s["v"], s["pos"], s["table"], seq=s["seq"], rope=(s["cos"], s["sin"], c["off"]),
                          rope_half=c["half"], q=s["q"], q_out=s["q_out"])
        return {"q": s["q_out"], "k": s["ck"], "v": s["cv"]}
    t, d, pos = c["tokens"], c["d"], s["pos"].long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    page = s["table"][s["seq"].long(), pos // c["page"]].long()
    for name, x, scale in (("ck", _rotate(s["k"].float().reshape(t, -1, d), cos, sin, c["off"], c["half"]), s["ks"]),
                           ("cv", s["v"].float().reshape(t, -1, d), s["vs"])):
        if c["fp8"]:
            code = (x / scale[:, None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
            s[name].view(torch.uint8)[page, :, pos % c["page"]] = code.view(torch.uint8)
        else:
            s[name][page, :, pos % c["page"]] = x.to(torch.bfloat16)
    s["q_out"].copy_(_rotate(s["q"].float().reshape(t, -1, d), cos, sin, c["off"], c["half"]).reshape(t, -1))
    return {"q": s["q_out"], "k": s["ck"], "v": s["cv"]}


def _softmax_product(score, seen, v):
    """(score masked by seen, softmax, times v; log of the sum): a row that sees nothing gives zeros and -inf."""
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    e = torch.exp(score - top)
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, v) / total.clamp(min=1e-38)
    return out, (top + torch.log(total)).squeeze(-1)


def _decode(s):
    c = s["c"]
    if own:
        ctx = _handle()
        out, lse = ctx.pkg.attn_decode(ctx, s["cache"], s["q"], s["table"], s["lens"], window=c["window"], return_lse=True)
        return {"out": out, "lse": lse}
    b, hkv, d, table = c["seqs"], c["hkv"], c["d"], s["table"].long()
    length = table.shape[1] * c["page"]
    k, v = (x[table].float().transpose(1, 2).reshape(b, hkv, length, d) for x in (s["ck"], s["cv"]))
    if c["fp8"]:
        k, v = k * s["ks"][:, None, None], v * s["vs"][:, None, None]
    at, n = torch.arange(length, device=DEV), s["lens"][:, None]
    seen = (at < n) & (at >= (n - c["window"] if c["window"] else 0))
    v = torch.where(seen[:, None, :, None], v, 0.0)
    q = s["q"].float().reshape(b, hkv, -1, d)
    out, lse = _softmax_product(torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5, seen[:, None, None], v)
    return {"out": out.reshape(b, -1).to(torch.bfloat16), "lse": lse.reshape(b, -1)}


def _prompt(s):
    c = s["c"]
    if own:
        ctx = _handle()
        out, lse = ctx.pkg.attn_prompt(ctx, s["q"], s["k"], s["v"], s["cu"], head_dim=c["d"], window=c["window"], return_lse=True)
        return {"out": out, "lse": lse}
    t, b, hkv, d, n = s["q"].shape[0], c["seqs"], c["hkv"], c["d"], s["longest"]
    at = torch.arange(n, device=DEV)
    here = at < (s["cu"][1:] - s["cu"][:-1])[:, None]
    row = (s["cu"][:-1, None] + at).clamp(max=t - 1).long()
    # padded to the longest: [seq][kv head][group or 1][token][d]
    q, k, v = (x.float()[row].reshape(b, n, hkv, -1, d).permute(0, 2, 3, 1, 4) for x in (s["q"], s["k"], s["v"]))
    seen = at[:, None] >= at
    if c["window"]:
        seen = seen & (at[:, None] - at < c["window"])
    out, lse = _softmax_product(torch.matmul(q * d ** -0.5, k.transpose(-1, -2)), seen, v)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, n, -1)[here]
    return {"out": out.to(torch.bfloat16), "lse": lse.permute(0, 3, 1, 2).reshape(b, n, -1)[here]}


def _sample(s):
    if own:
        ctx = _handle()
        ids, lp = ctx.pkg.sample(ctx, s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                                 return_logprobs=True)
        return {"ids": ids, "logprobs": lp}
    n = s["logits"].shape[1]
    value, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    value = value.double()
    gap = value - value[:, :1]
    greedy = s["temperature"] <= 0
    w = torch.exp(gap / torch.where(greedy, 1.0, s["temperature"]).double()[:, None])
    rank = torch.arange(n, device=DEV)
    k = torch.where((s["top_k"] <= 0) | greedy, torch.where(greedy, 1, n), s["top_k"])
    kept = torch.where(rank < k[:, None], w, 0.0)
    before = kept.cumsum(1) - kept
    keep = (rank < k[:, None]) & ((before < s["top_p"].double()[:, None] * kept.sum(1, keepdim=True)) | (s["top_p"] >= 1)[:, None] | (rank == 0))
    keep = keep & ((w >= s["min_p"].double()[:, None]) | (rank == 0))
    # the draw walks the kept tokens in the vocabulary's order
    mass = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    cum = mass.cumsum(1)
    hit = (cum > s["u"].double()[:, None] * cum[:, -1:]) & (mass > 0)
    ids = hit.int().argmax(1)
    lp = s["logits"].gather(1, ids[:, None]).squeeze(1).double() - value[:, 0] - torch.log(torch.exp(gap).sum(1))
    return {"ids": ids.int(), "logprobs": lp.float()}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    return {"append": _exact_append, "decode": _exact_decode, "prompt": _exact_prompt, "sample": _exact_sample}[c["op"]](c, s)


def _exact_append(c, s):
    t, d, m = c["tokens"], c["d"], c["rot"] // 2
    pos = s["pos"].long()
    # pairs of columns as complex numbers, turned by one multiplication
    turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
    first = torch.arange(m, device=DEV) + c["off"] if c["half"] else torch.arange(m, device=DEV) * 2 + c["off"]
    second = first + (m if c["half"] else 1)

    def turned(x):
        x = x.double().reshape(t, -1, d).clone()
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x
    out = {"q": turned(s["q"]).reshape(t, -1)}
    slot = s["table"].long()[s["seq"].long(), pos // c["page"]] * c["page"] + pos % c["page"]
    for name, new, old, scale in (("k", turned(s["k"]), s["ck"], s["ks"]), ("v", s["v"].double().reshape(t, -1, d), s["cv"], s["vs"])):
        if c["fp8"]:
            new = (new / scale.double()[:, None]).clamp(-FP8_MAX, FP8_MAX)
        flat = old.double().transpose(1, 2).reshape(-1, c["hkv"], d)
        flat[slot] = new
        out[name] = flat.reshape(-1, c["page"], c["hkv"], d).transpose(1, 2).contiguous()
    return out


def _exact_rows(q, k, v, first):
    """softmax(q k) v for rows of q [g][d] whose first visible keys (of those given) are all of them from ``first`` on."""
    sc = q @ k[first:].T
    lse = torch.logsumexp(sc, 1)
    return torch.exp(sc - lse[:, None]) @ v[first:], lse


def _exact_decode(c, s):
    lens, d, g = _lens(c), c["d"], c["hq"] // c["hkv"]
    out = torch.zeros(c["seqs"], c["hq"], d, dtype=torch.float64, device=DEV)
    lse = torch.full((c["seqs"], c["hq"]), -math.inf, dtype=torch.float64, device=DEV)
    q = s["q"].double().reshape(c["seqs"], c["hq"], d) / math.sqrt(d)
    for i, n in enumerate(lens):
        if n == 0:
            continue
        pages = s["table"][i, : -(-n // c["page"])].long()
        for h in range(c["hkv"]):
            k, v = (x[pages, h].double().reshape(-1, d)[:n] * (1.0 if sc is None else sc[h].double()) for x, sc in ((s["ck"], s["ks"]), (s["cv"], s["vs"])))
            rows = slice(h * g, h * g + g)
            out[i, rows], lse[i, rows] = _exact_rows(q[i, rows], k, v, max(0, n - c["window"]) if c["window"] else 0)
    return {"out": out.reshape(c["seqs"], -1), "lse": lse}


def _exact_prompt(c, s):
    d, g = c["d"], c["hq"] // c["hkv"]
    t = s["q"].shape[0]
    q, k, v = (x.double().reshape(t, -1, d) for x in (s["q"], s["k"], s["v"]))
    out = torch.zeros(t, c["hq"], d, dtype=torch.float64, device=DEV)
    lse = torch.zeros(t, c["hq"], dtype=torch.float64, device=DEV)
    start = 0
    for n in _lens(c):
        i = torch.arange(n, device=DEV)
        hidden = i[None, :] > i[:, None]
        if c["window"]:
            hidden |= i[None, :] <= i[:, None] - c["window"]
        for h in range(c["hq"] if n else 0):
            rows = slice(start, start + n)
            sc = (q[rows, h] @ k[rows, h // g].T / math.sqrt(d)).masked_fill_(hidden, -math.inf)
            lse[rows, h] = torch.logsumexp(sc, 1)
            out[rows, h] = torch.softmax(sc, 1) @ v[rows, h // g]
        start += n
    return {"out": out.reshape(t, -1), "lse": lse}


def _exact_sample(c, s):
    import numpy as np
    logits = s["logits"].cpu().numpy().astype(np.float64)
    u, temp, top_k, top_p, min_p = (s[k].cpu().numpy().astype(np.float64) for k in ("u", "temperature", "top_k", "top_p", "min_p"))
    ids, lps = [], []
    for r in range(c["rows"]):
        x = logits[r]
        best = x.max()
        if temp[r] <= 0:
            token = int(np.flatnonzero(x == best)[0])
        else:
            p = np.exp((x - best) / temp[r])
            by = np.lexsort((np.arange(x.size), -x))
            if top_k[r] > 0:
                by = by[: int(top_k[r])]
            if top_p[r] < 1:
                mass = np.concatenate([[0.0], np.cumsum(p[by])])
                by = by[: max(1, int((mass[:-1] < top_p[r] * mass[-1]).sum()))]
            by = np.sort(by[(p[by] >= min_p[r]) | (np.arange(by.size) == 0)])
            mass = np.cumsum(p[by])
            token = int(by[np.flatnonzero(mass > u[r] * mass[-1])[0]])
        ids.append(token)
        lps.append(x[token] - best - np.log(np.exp(x - best).sum()))
    return {"ids": torch.tensor(ids, dtype=torch.int32), "logprobs": torch.tensor(lps, dtype=torch.float64)}

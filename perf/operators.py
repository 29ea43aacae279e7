"""Cases of the operators of a decode step on an 8-bit key-value cache, and their plain forms.

``append``   keys and values of new tokens into 8-bit pages with one power-of-two scale per page and head
``attend``   attention of one new token per sequence over those pages
``sample``   temperature, top-k, top-p and min-p sampling from one random word per row

Where ``own`` is true ``run`` calls the framework's operators, otherwise their plain forms below.
"""
import math

import numpy as np
import torch

own = False

E4M3_MAX = 448.0
MIN_EXP, MAX_EXP = -100, 120  # exponents that a page's scale can have
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a decode step of 64 sequences: one token each, anywhere in a page
        {"name": "append_step", "op": "append", "seqs": 64, "most": 1, "ragged": False, "before": 2000, "kv_heads": 4,
         "head_dim": 128, "page": 64, "dtype": "bf16"},
        # an admission of mixed prompts, packed, into fresh pages
        {"name": "append_prompts", "op": "append", "seqs": 16, "most": 1024, "ragged": True, "before": 0, "kv_heads": 8,
         "head_dim": 128, "page": 64, "dtype": "bf16"},
        # pieces of odd lengths that continue in the middle of small pages
        {"name": "append_pieces", "op": "append", "seqs": 33, "most": 517, "ragged": True, "before": 301, "kv_heads": 2,
         "head_dim": 64, "page": 16, "dtype": "fp16"},
        # a few long documents
        {"name": "append_long", "op": "append", "seqs": 4, "most": 16384, "ragged": False, "before": 0, "kv_heads": 8,
         "head_dim": 128, "page": 64, "dtype": "bf16"},
        # one short chat: nothing but latency
        {"name": "attend_one", "op": "attend", "seqs": 1, "most": 211, "ragged": False, "heads": 14, "kv_heads": 2,
         "head_dim": 64, "page": 16, "window": 0, "dtype": "bf16"},
        # the rollout step of a policy: 64 sequences of about 1024 tokens
        {"name": "attend_step", "op": "attend", "seqs": 64, "most": 1024, "ragged": False, "heads": 28, "kv_heads": 4,
         "head_dim": 128, "page": 64, "window": 0, "dtype": "bf16"},
        # a server's batch: lengths from a few tokens to 8192
        {"name": "attend_ragged", "op": "attend", "seqs": 128, "most": 8192, "ragged": True, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "window": 0, "dtype": "bf16"},
        # one very long document: the work has to be split along the context
        {"name": "attend_long", "op": "attend", "seqs": 1, "most": 131067, "ragged": False, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "window": 0, "dtype": "bf16"},
        # as many key heads as query heads, a head size off the powers of two, a sliding window
        {"name": "attend_window", "op": "attend", "seqs": 24, "most": 4500, "ragged": True, "heads": 32, "kv_heads": 32,
         "head_dim": 96, "page": 32, "window": 2047, "dtype": "fp16"},
        # one request of a chat: all filters on
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 152064, "temperature": 0.7, "top_k": 20, "top_p": 0.8,
         "min_p": 0.0, "per_row": False, "dtype": "bf16"},
        # the rollout step of a policy: nucleus sampling
        {"name": "sample_step", "op": "sample", "rows": 64, "vocab": 152064, "temperature": 1.0, "top_k": 0, "top_p": 0.95,
         "min_p": 0.0, "per_row": False, "dtype": "bf16"},
        # a server's batch: every request brings its own parameters, some are greedy, some filter nothing
        {"name": "sample_mixed", "op": "sample", "rows": 256, "vocab": 128256, "temperature": 1.0, "top_k": 50, "top_p": 0.9,
         "min_p": 0.05, "per_row": True, "dtype": "fp32"},
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["append", "attend", "sample"])
    if op == "sample":
        vocab = _log_uniform(rng, 1000, 262144)
        return {"op": op, "rows": _log_uniform(rng, 1, max(1, min(256, 256 * 128256 // vocab))), "vocab": vocab,
                "temperature": round(rng.uniform(0.3, 1.5), 3), "top_k": rng.choice([0, 1, _log_uniform(rng, 2, 2000)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.05, 0.999), 3)]),
                "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 3)]), "per_row": rng.random() < 0.4,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    case = {"op": op, "kv_heads": rng.choice([1, 2, 3, 4, 8, 16]), "head_dim": rng.choice([64, 96, 128, 128, 256]),
            "page": rng.choice([16, 32, 64, 64, 128]), "ragged": rng.random() < 0.6, "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    width = case["kv_heads"] * case["head_dim"]
    if op == "append":
        seqs = _log_uniform(rng, 1, 256)
        most = 1 if rng.random() < 0.35 else _log_uniform(rng, 2, min(16384, 4 * 16384 // seqs, 4 * 16384 * 1024 // (width * seqs)))
        return {**case, "seqs": seqs, "most": most, "before": rng.choice([0, _log_uniform(rng, 1, 2000)])}
    seqs = _log_uniform(rng, 1, 256)
    room = (128 * 8192 if case["ragged"] else 131072) * 1024 // (width * seqs)
    return {**case, "seqs": seqs, "most": _log_uniform(rng, 1, min(131072, room)),
            "heads": case["kv_heads"] * rng.choice([1, 2, 4, 5, 7, 8, 12, 16]),
            "window": rng.choice([0, 0, _log_uniform(rng, 1, 4096)])}


def _lengths(case):
    """Tokens of every sequence: ``most``, or spread over the logarithm from 1 to ``most`` without a pattern in their order."""
    n, most = case["seqs"], case["most"]
    if not case["ragged"]:
        return [most] * n
    part = [((i + 1) * 0.6180339887498949) % 1.0 for i in range(n)]
    return [max(1, min(most, int(round(math.exp(p * math.log(most + 0.49)))))) for p in part]


def _starts(case):
    """Tokens that each sequence has in the cache before an append."""
    return [0 if not case["before"] else int(case["before"] * (((i + 1) * 0.7548776662466927) % 1.0)) for i in range(case["seqs"])]


def work(case):
    if case["op"] == "sample":
        size = 4 if case["dtype"] == "fp32" else 2
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (4 + 12 + 16 * case["per_row"]), "flops": 4 * n}
    width = case["kv_heads"] * case["head_dim"]
    if case["op"] == "append":
        tokens = sum(_lengths(case))
        pages = sum(-(-(s % case["page"] + n) // case["page"]) for s, n in zip(_starts(case), _lengths(case)))
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2 * tokens * width * (size + 1) + pages * (8 * case["kv_heads"] + 4) + 8 * case["seqs"], "flops": 4 * tokens * width}
    seen = sum(min(n, case["window"] or n) for n in _lengths(case))
    pages = sum(-(-min(n, case["window"] or n) // case["page"]) for n in _lengths(case))
    qo = 2 * case["seqs"] * case["heads"] * case["head_dim"] * 2
    return {"bytes": 2 * seen * width + pages * (8 * case["kv_heads"] + 4) + qo + 4 * case["seqs"],
            "flops": 4 * seen * case["heads"] * case["head_dim"]}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _scale_of(amax):
    """The smallest power of two that brings ``amax`` within 448, as fp32."""
    m, e = torch.frexp(amax.double() / E4M3_MAX)
    e = torch.where(m > 0.5, e, e - 1).clamp(MIN_EXP, MAX_EXP)
    return torch.ldexp(torch.ones_like(m), torch.where(amax > 0, e, torch.full_like(e, MIN_EXP))).float()


def _pages(case, gen, lengths):
    """A cache that holds ``lengths[i]`` tokens of sequence i in pages of no order: codes, scales and the block table."""
    page, hk, d = case["page"], case["kv_heads"], case["head_dim"]
    per = -(-max(lengths) // page)
    count = [-(-n // page) for n in lengths]
    total = sum(count) + 1
    order = torch.randperm(total, generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    first = torch.tensor(np.concatenate([[0], np.cumsum(count)[:-1]]), device="cuda")
    col = torch.arange(per, device="cuda")
    at = first[:, None] + col[None, :]
    table = torch.where(col[None, :] < torch.tensor(count, device="cuda")[:, None], order[at.clamp(max=total - 1)], 0).to(torch.int32)
    held = []
    for _ in range(2):
        size = torch.rand(1, hk, 1, 1, generator=gen, device="cuda") * 2 + 0.3  # heads differ in size
        x = torch.randn(total, hk, page, d, generator=gen, device="cuda", dtype=torch.bfloat16)
        x.mul_(size.to(torch.bfloat16))
        scale = _scale_of(x.abs().amax((2, 3)))
        held += [(x.float() / scale[:, :, None, None]).to(torch.float8_e4m3fn), scale]
    return {"k_cache": held[0], "k_scale": held[1], "v_cache": held[2], "v_scale": held[3], "table": table}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=gen, device="cuda")  # noqa: E731
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        z = torch.randn(rows, vocab, generator=gen, device="cuda") * 2
        likely = (rand(rows, 64) * vocab).long()  # a few tokens stand out, in some rows by a lot
        z.scatter_add_(1, likely, -2.5 * torch.log(rand(rows, 64).clamp_min(1e-6)) + 2)
        z *= 0.5 + rand(rows, 1)
        par = {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
        if case["per_row"]:
            off = lambda share: rand(rows) < share  # noqa: E731
            par = {"temperature": torch.where(off(0.15), 0.0, par["temperature"] * (0.5 + rand(rows))),
                   "top_k": torch.where(off(0.4), 0, (rand(rows) * (2 * par["top_k"] + 1)).long()).to(torch.int32),
                   "top_p": torch.where(off(0.3), 1.0, (par["top_p"] * (0.7 + 0.3 * rand(rows)))),
                   "min_p": torch.where(off(0.5), 0.0, par["min_p"] * rand(rows))}
        rng = torch.randint(-2**31, 2**31 - 1, (rows,), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
        return {"op": "sample", "logits": z.to(DTYPES[case["dtype"]]), "rng": rng, **par}
    dt, hk, d = DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lengths = _lengths(case)
    if case["op"] == "append":
        starts = _starts(case)
        s = _pages(case, gen, [a + n for a, n in zip(starts, lengths)])
        kv = [torch.randn(sum(lengths), hk, d, generator=gen, device="cuda") * (rand(1, hk, 1) * 2 + 0.3) for _ in range(2)]
        return {"op": "append", **s, "k": kv[0].to(dt), "v": kv[1].to(dt), "starts": i32(starts), "most": case["most"],
                "cu": None if case["most"] == 1 else i32(np.concatenate([[0], np.cumsum(lengths)]))}
    s = _pages(case, gen, lengths)
    q = torch.randn(case["seqs"], case["heads"], d, generator=gen, device="cuda") * (0.5 + rand(1, case["heads"], 1))
    return {"op": "attend", **s, "q": q.to(dt), "seq_lens": i32([n - 1 for n in lengths]), "scale": d**-0.5,
            "window": case["window"] or None}


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _append(s):
    page, n = s["k_cache"].shape[2], s["starts"].shape[0]
    starts, tokens = s["starts"].long(), s["k"].shape[0]
    at = torch.arange(tokens, device="cuda")
    seq = at if s["cu"] is None else torch.searchsorted(s["cu"][1:].long(), at, right=True)
    pos = starts[seq] + (at - (at if s["cu"] is None else s["cu"].long()[seq]))
    blk, row = s["table"][seq, pos // page].long(), pos % page
    first = s["table"][torch.arange(n, device="cuda"), starts // page].long()
    kept = starts % page  # rows of its first page that a sequence filled earlier
    for x, codes, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        x = x.float()
        amax = torch.where(torch.isfinite(x), x.abs(), 0).amax(-1)
        most = torch.zeros_like(scale).index_reduce_(0, blk, amax, "amax")
        was = scale[first]
        need = _scale_of(most)
        now = need.clone()
        now[first] = torch.where(kept[:, None] > 0, torch.maximum(was, need[first]), need[first])
        old = codes.view(torch.uint8)[first].view(torch.float8_e4m3fn)
        again = (old.float() * (was / now[first])[:, :, None, None]).to(torch.float8_e4m3fn)
        rows = torch.arange(page, device="cuda")[None, None, :, None] < kept[:, None, None, None]
        codes.view(torch.uint8)[first] = torch.where(rows, again.view(torch.uint8), old.view(torch.uint8))
        codes.view(torch.uint8)[blk, :, row] = (x / now[blk][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        scale[blk] = now[blk]
    return {"k_cache": s["k_cache"], "k_scale": s["k_scale"], "v_cache": s["v_cache"], "v_scale": s["v_scale"]}


def _attend(s):
    q, table = s["q"].float(), s["table"].long()
    b, heads, d = q.shape
    hk, page = s["k_cache"].shape[1:3]
    length = s["seq_lens"].long() + 1
    pos = torch.arange(table.shape[1] * page, device="cuda")
    seen = pos[None, :] < length[:, None]
    if s["window"]:
        seen &= pos[None, :] >= length[:, None] - s["window"]

    def held(codes, scale):
        x = codes.view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * scale[table][..., None, None]
        return x.transpose(1, 2).reshape(b, hk, -1, d)

    score = (q.view(b, hk, heads // hk, d) @ held(s["k_cache"], s["k_scale"]).transpose(2, 3)) * s["scale"]
    score.masked_fill_(~seen[:, None, None, :], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    v = held(s["v_cache"], s["v_scale"]).masked_fill_(~seen[:, None, :, None], 0)
    return ((p @ v) / p.sum(-1, keepdim=True)).view(b, heads, d).to(s["q"].dtype)


def _hash(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _sample(s):
    rows, vocab = s["logits"].shape
    col = lambda name, dt: (s[name].to(dt) if torch.is_tensor(s[name]) else torch.full((rows,), s[name], device="cuda", dtype=dt))[:, None]  # noqa: E731
    temperature, top_k, top_p, min_p = col("temperature", torch.float32), col("top_k", torch.int64), col("top_p", torch.float32), col("min_p", torch.float32)
    z = s["logits"].float() / temperature.clamp_min(1e-6)
    # most likely first, the lower index first among equals; sums and borders in 64 bits
    order = torch.sort(z, dim=-1, descending=True, stable=True)
    zs = order.values.double()
    top = zs[:, :1]
    kth = zs.gather(1, torch.where(top_k > 0, top_k.clamp(max=vocab), vocab) - 1)
    keep = zs >= kth
    w = torch.where(keep, torch.exp(zs - top), 0)
    before = w.cumsum(-1) - w
    keep &= (before <= top_p.double() * w.sum(-1, keepdim=True)) | (top_p >= 1)
    keep &= (zs >= top + torch.log(min_p.double())) | (min_p <= 0)
    lse = top + torch.log(torch.where(keep, w, 0).sum(-1, keepdim=True))
    at = torch.arange(vocab, device="cuda")
    h = _hash((s["rng"].long() & 0xFFFFFFFF)[:, None] ^ _hash((at * 0x85EBCA6B + 0x165667B1) & 0xFFFFFFFF))
    u = (_hash((h + at) & 0xFFFFFFFF).double() + 0.5) / 2.0**32
    kept = torch.empty_like(keep).scatter_(1, order.indices, keep)
    key = torch.where(temperature > 0, z.double() - torch.log(-torch.log(u)), z.double()).masked_fill_(~kept, float("-inf"))
    best = key == key.amax(-1, keepdim=True)
    tok = torch.where(best, at, vocab).amin(-1)
    return {"token": tok.to(torch.int32), "logp": (z.double().gather(1, tok[:, None]) - lse)[:, 0].float()}


def run(s):
    if own:
        from trl_b200.ops import functional as F

        if s["op"] == "append":
            F.kv8_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["starts"],
                         cu_seqlens=s["cu"], max_new=s["most"])
            return {"k_cache": s["k_cache"], "k_scale": s["k_scale"], "v_cache": s["v_cache"], "v_scale": s["v_scale"]}
        if s["op"] == "attend":
            return F.kv8_decode_attn(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["seq_lens"],
                                     s["scale"], window=s["window"])
        tok, logp = F.sample_filtered(s["logits"], s["rng"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                      min_p=s["min_p"])
        return {"token": tok, "logp": logp}
    return {"append": _append, "attend": _attend, "sample": _sample}[s["op"]](s)


# ---- the definitions in 64 bits, sequence by sequence and row by row -----------------------------------------------
def _round_e4m3(x):
    """Nearest values with three fraction bits and exponents of at least -6, ties to even; no number above 448 comes in."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _exact_append(case, s):
    page, starts, lengths = case["page"], _starts(case), _lengths(case)
    table = s["table"].tolist()
    out = {}
    for name in "kv":
        codes, scale = s[name + "_cache"].double(), s[name + "_scale"].double()
        done = 0
        for i, (start, n) in enumerate(zip(starts, lengths)):
            x = s[name][done:done + n].double().transpose(0, 1)
            done += n
            at = 0
            while at < n:
                row = (start + at) % page
                take, blk = min(page - row, n - at), table[i][(start + at) // page]
                piece = x[:, at:at + take]
                amax = piece.abs().amax((1, 2))
                near = torch.floor(torch.log2(amax.clamp_min(2.0**-200) / E4M3_MAX)).to(torch.int32) - 1
                for _ in range(3):  # the logarithm says about where; products of powers of two say it exactly
                    near += (torch.ldexp(torch.full_like(amax, E4M3_MAX), near) < amax).to(torch.int32)
                new = torch.ldexp(torch.ones_like(amax), near.clamp(MIN_EXP, MAX_EXP))
                if row:
                    new = torch.maximum(new, scale[blk])
                    codes[blk, :, :row] = _round_e4m3(codes[blk, :, :row] * (scale[blk] / new)[:, None, None])
                codes[blk, :, row:row + take] = _round_e4m3(piece / new[:, None, None])
                scale[blk] = new
                at += take
        out[name + "_cache"], out[name + "_scale"] = codes, scale
    return out


def _exact_attend(case, s):
    hk, page, d = case["kv_heads"], case["page"], case["head_dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(_lengths(case)):
        lo = max(0, n - (s["window"] or n))
        blocks = s["table"][i, lo // page:-(-n // page)].long()
        base = lo // page * page

        def rows(name):
            codes = s[name + "_cache"].view(torch.uint8)[blocks].view(torch.float8_e4m3fn).double()
            x = (codes * s[name + "_scale"][blocks].double()[:, :, None, None]).transpose(0, 1).reshape(hk, -1, d)
            return x[:, lo - base:n - base]

        score = torch.einsum("hgd,htd->hgt", s["q"][i].double().view(hk, -1, d), rows("k")) * s["scale"]
        out[i] = torch.einsum("hgt,htd->hgd", torch.softmax(score, -1), rows("v")).reshape(-1, d)
    return out


def _exact_sample(case, s):
    logp = []
    drawn = _sample(s)["token"].tolist()  # the log-probability of which token: a choice of whole numbers
    for i, tok in enumerate(drawn):
        of = lambda name: float(s[name][i]) if torch.is_tensor(s[name]) else float(np.float32(s[name]))  # noqa: E731
        z = (s["logits"][i].float() / max(np.float32(of("temperature")), np.float32(1e-6))).double()
        values, order = torch.sort(z, descending=True, stable=True)
        n = int((values >= values[min(int(of("top_k")), len(z)) - 1]).sum()) if of("top_k") > 0 else len(z)
        p = torch.softmax(values[:n], 0)
        if of("top_p") < 1:
            before = torch.cat([p.new_zeros(1), p.cumsum(0)[:-1]])
            n = int((before <= of("top_p")).sum())
        if of("min_p") > 0:
            n = min(n, int((values - values[0] >= math.log(of("min_p"))).sum()))
        logp.append(z[tok] - torch.logsumexp(values[:n], 0))
    return {"token": None, "logp": torch.stack(logp)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](case, s)

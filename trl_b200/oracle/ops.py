"""Pure-PyTorch reference implementations of every hot op.

These are the numerical oracles for the sm_100a kernels and also the execution
path on CPU (fp32, gloo).  All functions are differentiable through autograd and
do their arithmetic in fp32 regardless of the input dtype.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    var = xf.pow(2).mean(-1, keepdim=True)
    return (xf * torch.rsqrt(var + eps) * weight.float()).to(x.dtype)


def rope_cos_sin(positions: torch.Tensor, head_dim: int, theta: float, dtype=torch.float32):
    """cos/sin tables [T, head_dim/2] for integer ``positions`` [T]."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, device=positions.device, dtype=torch.float32) / head_dim))
    ang = positions.float()[:, None] * inv[None, :]
    return ang.cos().to(dtype), ang.sin().to(dtype)


def apply_rope(x: torch.Tensor, positions: torch.Tensor, theta: float) -> torch.Tensor:
    """Rotate-half RoPE on ``x`` [T, H, D] (HF Llama/Qwen convention)."""
    d = x.shape[-1]
    cos, sin = rope_cos_sin(positions, d, theta)
    xf = x.float()
    x1, x2 = xf[..., : d // 2], xf[..., d // 2:]
    c, s = cos[:, None, :], sin[:, None, :]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).to(x.dtype)


def apply_mrope(x: torch.Tensor, positions3: torch.Tensor, theta: float, sections) -> torch.Tensor:
    """Multimodal rotary embedding on ``x`` [T, H, D]: ``positions3`` [3, T] holds a temporal, a height and a width
    position per token; the D/2 rotary frequencies are cut into ``sections`` (their sizes sum to D/2) and section i
    turns with position set i mod 3.  With three equal position rows this is ordinary RoPE
    (Qwen2-VL; transformers modeling_qwen2_vl.py ``apply_multimodal_rotary_pos_emb`` is the behaviour matched)."""
    d = x.shape[-1]
    half = d // 2
    if sum(sections) != half:
        raise ValueError(f"mrope_section {list(sections)} must sum to head_dim / 2 = {half}")
    inv = 1.0 / (theta ** (torch.arange(0, d, 2, device=x.device, dtype=torch.float32) / d))  # [half]
    ang = positions3.float()[:, :, None] * inv[None, None, :]                                  # [3, T, half]
    which = torch.cat([torch.full((n,), i % 3, dtype=torch.long) for i, n in enumerate(sections)]).to(x.device)
    ang = ang.gather(0, which[None, None, :].expand(1, ang.shape[1], half))[0]                 # [T, half]
    cos, sin = ang.cos()[:, None, :], ang.sin()[:, None, :]
    xf = x.float()
    x1, x2 = xf[..., :half], xf[..., half:]
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1).to(x.dtype)


def swiglu(gate_up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` for ``gate_up = [gate | up]`` along the last dim."""
    g, u = gate_up.float().chunk(2, dim=-1)
    return (F.silu(g) * u).to(gate_up.dtype)


def attention_varlen(q, k, v, cu_seqlens, max_seqlen=None, causal=True, scale=None, window=None):
    """Causal GQA attention over packed documents.

    q [T, Hq, D]; k, v [T, Hkv, D]; ``cu_seqlens`` int tensor [n_docs + 1].
    A dense block-diagonal mask is built: fine for an oracle, O(T^2) memory.
    """
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    doc = torch.bucketize(torch.arange(T, device=q.device), cu_seqlens[1:].to(q.device), right=True)
    mask = doc[:, None] == doc[None, :]
    if causal:
        idx = torch.arange(T, device=q.device)
        mask = mask & (idx[:, None] >= idx[None, :])
    if window:
        idx = torch.arange(T, device=q.device)
        mask = mask & (idx[:, None] - idx[None, :] < window)
        if not causal:
            mask = mask & (idx[None, :] - idx[:, None] < window)
    rep = Hq // Hkv
    qf = q.float().transpose(0, 1)  # [Hq, T, D]
    kf = k.float().transpose(0, 1).repeat_interleave(rep, dim=0)
    vf = v.float().transpose(0, 1).repeat_interleave(rep, dim=0)
    s = torch.matmul(qf, kf.transpose(1, 2)) * scale
    s = s.masked_fill(~mask[None], float("-inf"))
    p = torch.softmax(s, dim=-1)
    o = torch.matmul(p, vf)  # [Hq, T, D]
    return o.transpose(0, 1).to(q.dtype).contiguous()


def attention_varlen_qk(q, k, v, cu_q, cu_k, scale=None):
    """Causal GQA attention, query segment i (``cu_q``) against key segment i (``cu_k``), mask aligned to the end of the
    key segment: query j of a segment with lq queries and lk keys sees keys 0 .. j + lk - lq.  Dense mask, oracle only."""
    Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[0], k.shape[1]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    cq, ck = cu_q.to(q.device).long(), cu_k.to(q.device).long()
    iq, ik = torch.arange(Tq, device=q.device), torch.arange(Tk, device=q.device)
    sq = torch.bucketize(iq, cq[1:], right=True)
    sk = torch.bucketize(ik, ck[1:], right=True)
    # position of every query / key counted from the END of its segment
    q_from_end = cq[1:][sq] - iq
    k_from_end = ck[1:][sk] - ik
    mask = (sq[:, None] == sk[None, :]) & (k_from_end[None, :] >= q_from_end[:, None])
    rep = Hq // Hkv
    qf = q.float().transpose(0, 1)
    kf = k.float().transpose(0, 1).repeat_interleave(rep, dim=0)
    vf = v.float().transpose(0, 1).repeat_interleave(rep, dim=0)
    s = torch.matmul(qf, kf.transpose(1, 2)) * scale
    s = s.masked_fill(~mask[None], float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.matmul(p, vf).transpose(0, 1).to(q.dtype).contiguous()


def lm_head_logprobs(hidden, weight, labels, temperature=1.0, bias=None, softcap=None,
                     compute_entropy=True, entropy_grad=False):
    """Per-token log p(label) and entropy from ``hidden[N,H] @ weight[V,H]^T``.

    Entropy carries no gradient (matches trl/trainer/utils.py:1291-1424) unless ``entropy_grad``
    (the differentiable entropy of the GRPO bonus, trl/trainer/grpo_trainer.py:3155-3175).
    """
    logits = hidden.float() @ weight.float().t()
    if bias is not None:
        logits = logits + bias.float()
    if softcap:
        logits = torch.tanh(logits / softcap) * softcap
    logits = logits / temperature
    lse = torch.logsumexp(logits, dim=-1)
    tgt = logits.gather(-1, labels.long().clamp_min(0)[:, None]).squeeze(-1)
    logp = tgt - lse
    ent = None
    if compute_entropy:
        with torch.set_grad_enabled(bool(entropy_grad) and torch.is_grad_enabled()):
            p = torch.softmax(logits, dim=-1)
            ent = (lse if entropy_grad else lse.detach()) - (p * logits).sum(-1)
    return logp, ent


def lm_head_ce(hidden, weight, labels, ignore_index=-100, bias=None):
    """Sum of token NLL over valid labels plus (correct, entropy_sum, n_valid).

    Mirrors the quantities of trl/trainer/sft_trainer.py:117-234.  When no label
    is valid the loss is ``(hidden.sum() + weight.sum()) * 0`` so that backward
    and gradient synchronisation still run on every rank.
    """
    valid = labels != ignore_index
    n_valid = valid.sum()
    if int(n_valid) == 0:
        z = (hidden.sum() + weight.sum()).float() * 0.0
        zero = torch.zeros((), device=hidden.device)
        return z, zero, zero, n_valid
    h = hidden[valid]
    y = labels[valid]
    logits = h.float() @ weight.float().t()
    if bias is not None:
        logits = logits + bias.float()
    logp = torch.log_softmax(logits, dim=-1)
    nll = -logp.gather(-1, y[:, None]).squeeze(-1)
    with torch.no_grad():
        correct = (logits.argmax(-1) == y).sum()
        ent = -(logp.exp() * logp).sum(-1).sum()
    return nll.sum(), correct, ent, n_valid


def selective_log_softmax(logits, index):
    """log_softmax(logits).gather(index); index [...] or [..., K] (utils.py:479-523)."""
    squeeze = index.ndim == logits.ndim - 1
    if squeeze:
        index = index.unsqueeze(-1)
    if logits.dtype in (torch.float32, torch.float64):
        sel = torch.gather(logits, dim=-1, index=index)
        lse = torch.stack([torch.logsumexp(l, dim=-1) for l in logits])
        out = sel - lse.unsqueeze(-1)
    else:
        out = torch.stack([F.log_softmax(rl, dim=-1).gather(-1, ri) for rl, ri in zip(logits, index)])
    return out.squeeze(-1) if squeeze else out


def entropy_from_logits(logits: torch.Tensor, chunk_size: int = 128) -> torch.Tensor:
    """Shannon entropy (nats) row-chunked (utils.py:526-560)."""
    shp = logits.shape[:-1]
    flat = logits.reshape(-1, logits.shape[-1])
    outs = []
    for c in flat.split(chunk_size, dim=0):
        lp = F.log_softmax(c, dim=-1)
        outs.append(-(lp.exp() * lp).sum(-1))
    return torch.cat(outs, 0).reshape(shp) if outs else flat.new_zeros(shp)


def moe_router(hidden, gate_weight, top_k, norm_topk_prob):
    """softmax(fp32) -> top-k -> optional renormalise.  Returns (probs, idx, full_probs)."""
    logits = hidden.float() @ gate_weight.float().t()
    probs = torch.softmax(logits, dim=-1)
    w, idx = torch.topk(probs, top_k, dim=-1)
    if norm_topk_prob:
        w = w / w.sum(-1, keepdim=True)
    return w, idx, probs


def moe_experts(hidden, gate_up_w, down_w, topk_w, topk_idx):
    """Dense loop over experts.  gate_up_w [E, 2I, H]; down_w [E, H, I]."""
    out = torch.zeros_like(hidden, dtype=torch.float32)
    E = gate_up_w.shape[0]
    for e in range(E):
        tok, slot = (topk_idx == e).nonzero(as_tuple=True)
        if tok.numel() == 0:
            continue
        x = hidden[tok].float()
        gu = x @ gate_up_w[e].float().t()
        act = swiglu(gu)
        y = act @ down_w[e].float().t()
        out.index_add_(0, tok, y * topk_w[tok, slot].float()[:, None])
    return out.to(hidden.dtype)


def load_balancing_loss(router_probs, topk_idx, num_experts, top_k, token_mask=None):
    """Switch-style aux loss ``E * sum_e f_e * P_e`` over all layers' tokens.

    router_probs [L*T, E] are post-softmax probabilities; topk_idx [L*T, K].
    """
    onehot = F.one_hot(topk_idx, num_experts).float()  # [N, K, E]
    if token_mask is None:
        f = onehot.mean(0)  # [K, E]
        p = router_probs.float().mean(0)
    else:
        m = token_mask.float().reshape(-1)
        f = (onehot * m[:, None, None]).sum(0) / m.sum().clamp_min(1)
        p = (router_probs.float() * m[:, None]).sum(0) / m.sum().clamp_min(1)
    return (f * p[None, :]).sum() * num_experts


def grpo_token_loss(logp, old_logp, ref_logp, adv, eps_low, eps_high, beta, delta=None):
    """Token-level clipped surrogate + k3 KL (grpo_trainer.py:3054-3121)."""
    ratio = torch.exp(logp - old_logp)
    clipped = torch.clamp(ratio, 1 - eps_low, 1 + eps_high)
    r1 = ratio if delta is None else torch.clamp(ratio, max=delta)
    loss = -torch.min(r1 * adv, clipped * adv)
    kl = None
    if beta != 0.0 and ref_logp is not None:
        d = ref_logp - logp
        kl = torch.exp(d) - d - 1
        loss = loss + beta * kl
    return loss, ratio, kl


def dpo_sigmoid_loss(pol_c, pol_r, ref_c, ref_r, beta, label_smoothing=0.0):
    d = (pol_c - ref_c) - (pol_r - ref_r)
    loss = -F.logsigmoid(beta * d) * (1 - label_smoothing) - F.logsigmoid(-beta * d) * label_smoothing
    return loss, beta * (pol_c - ref_c), beta * (pol_r - ref_r)


# ---- 8-bit paged cache and filtered sampling ------------------------------------------------------------------------
def kv8_scale(amax: torch.Tensor) -> torch.Tensor:
    """The smallest power of two, from 2^-100 to 2^120, that brings ``amax`` within 448 (the largest e4m3 number)."""
    frac, exp = torch.frexp(amax.double() / 448.0)
    exp = torch.where(frac > 0.5, exp, exp - 1).clamp(-100, 120)
    return torch.ldexp(torch.ones_like(frac), torch.where(amax > 0, exp, torch.full_like(exp, -100))).float()


def kv8_append(k, v, k_cache, v_cache, k_scale, v_scale, block_table, starts, cu_seqlens=None, slots=None):
    """New tokens into an 8-bit paged cache, sequence by sequence and page by page (see ``ops.functional.kv8_append``)."""
    page = k_cache.shape[2]
    cu = list(range(starts.shape[0] + 1)) if cu_seqlens is None else cu_seqlens.tolist()
    for i, start in enumerate(starts.tolist()):
        if start < 0:
            continue
        row = block_table[i if slots is None else int(slots[i])].tolist()
        at, n = 0, cu[i + 1] - cu[i]
        while at < n:
            first = (start + at) % page
            take, blk = min(page - first, n - at), row[(start + at) // page]
            for x, codes, scale in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
                new = x[cu[i] + at:cu[i] + at + take].float().transpose(0, 1)  # [heads, take, dim]
                new = torch.where(torch.isfinite(new), new, float("nan"))
                now = kv8_scale(torch.nan_to_num(new.abs(), nan=0.0).amax((1, 2)))
                if first:
                    was = scale[blk].clone()
                    now = torch.maximum(was, now)
                    codes[blk, :, :first] = (codes[blk, :, :first].float() * (was / now)[:, None, None]).to(codes.dtype)
                codes[blk, :, first:first + take] = (new / now[:, None, None]).to(codes.dtype)
                scale[blk] = now
            at += take


def kv8_gather(codes, scale, blocks, lo, hi):
    """Positions ``lo .. hi`` of the sequence whose pages are ``blocks``: fp32 [heads, hi - lo, dim]."""
    x = codes[blocks].float() * scale[blocks][:, :, None, None]
    return x.transpose(0, 1).reshape(codes.shape[1], -1, codes.shape[3])[:, lo:hi]


def kv8_decode_attn(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, scale, slots=None, window=None):
    B, Hq, D = q.shape
    heads, page = k_cache.shape[1:3]
    out = torch.zeros_like(q)
    for i in range(B):
        slot = i if slots is None else int(slots[i])
        n = int(seq_lens[slot]) + 1
        if n <= 0:
            continue
        lo = max(0, n - window) if window else 0
        blocks = block_table[slot, :-(-n // page)].long()
        kk, vv = kv8_gather(k_cache, k_scale, blocks, lo, n), kv8_gather(v_cache, v_scale, blocks, lo, n)
        s = torch.einsum("hgd,htd->hgt", q[i].float().view(heads, -1, D), kk) * scale
        out[i] = torch.einsum("hgt,htd->hgd", torch.softmax(s, -1), vv).reshape(Hq, D).to(q.dtype)
    return out


def _hash_u32(x: torch.Tensor) -> torch.Tensor:
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def row_uniforms(rng: torch.Tensor, vocab: int) -> torch.Tensor:
    """The uniform numbers in (0, 1), fp64 [B, vocab], that the rows' random words stand for."""
    col = torch.arange(vocab, device=rng.device)
    h = _hash_u32((rng.long() & 0xFFFFFFFF)[:, None] ^ _hash_u32((col * 0x85EBCA6B + 0x165667B1) & 0xFFFFFFFF))
    return (_hash_u32((h + col) & 0xFFFFFFFF).double() + 0.5) / 2.0**32


def sample_filtered(logits, rng, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Row by row, sums in fp64 (see ``ops.functional.sample_filtered``)."""
    B, V = logits.shape
    per = lambda x, i: x[i].item() if torch.is_tensor(x) else x  # noqa: E731
    u = row_uniforms(rng, V)
    toks, logps = torch.zeros(B, dtype=torch.int32), torch.full((B,), float("-inf"))
    for i in range(B):
        t, k, p, m = per(temperature, i), int(per(top_k, i)), per(top_p, i), per(min_p, i)
        z = logits[i].float() / torch.tensor(t, dtype=torch.float32).clamp_min(1e-6)
        z = torch.nan_to_num(z, nan=float("-inf"), posinf=torch.finfo(torch.float32).max, neginf=float("-inf")).double()
        if z.max() == float("-inf"):
            continue
        zs, order = torch.sort(z, descending=True, stable=True)
        keep = (zs >= zs[k - 1] if 0 < k < V else torch.ones(V, dtype=torch.bool)) & (zs > float("-inf"))
        w = torch.where(keep, torch.exp(zs - zs[0]), 0.0)
        if p < 1:
            keep &= w.cumsum(0) - w <= max(p, 0.0) * w.sum()
        if m > 0:
            keep &= zs >= zs[0] + math.log(min(m, 1.0))
        kept = order[keep]
        key = z[kept] if not t > 0 else z[kept] - torch.log(-torch.log(u[i, kept]))
        toks[i] = int(kept[key == key.max()].min())
        logps[i] = float(z[toks[i]] - zs[0] - torch.logsumexp(z[kept] - zs[0], 0))
    return toks.to(logits.device), logps.to(logits.device)

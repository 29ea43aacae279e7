"""Inputs and 64-bit references of the 8-bit paged cache and of filtered sampling."""
import math

import torch


def table_of(rows, blocks, pages, gen, device):
    """A block table whose entries are all different pages."""
    assert rows * blocks <= pages
    return torch.randperm(pages, generator=gen)[: rows * blocks].view(rows, blocks).to(torch.int32).to(device)


def filled_cache(lens, heads, page, dim, device, seed=0, spread=0, extra=3):
    """(cache tensors, block table): random codes, scales 2^-3 .. 2^1 (with ``spread``: 2^-spread .. 2^spread)."""
    g = torch.Generator().manual_seed(seed)
    blocks = max(1, max(-(-n // page) for n in lens))
    pages = len(lens) * blocks + extra
    x = [torch.randn(pages, heads, page, dim, generator=g).mul(60).clamp(-448, 448).to(torch.float8_e4m3fn).to(device) for _ in range(2)]
    lo, hi = (-spread, spread + 1) if spread else (-3, 2)
    s = [torch.ldexp(torch.ones(pages, heads), torch.randint(lo, hi, (pages, heads), generator=g)).to(device) for _ in range(2)]
    return (*x, *s), table_of(len(lens), blocks, pages, g, device)


def attention64(q, cache, table, lens, scale, window=None):
    """(output fp64, bound fp64) of decode attention.  The bound adds up what may be rounded:

    * the output: half a step of its type, eps / 2 of the value;
    * the weights, once to fp16: 2^-11 of each, and 2^-25 of the largest where they are below fp16's normal numbers;
    * scores: a dot product of D terms in 32 bits, (D + 8) 2^-24 of its terms' magnitudes, times 2 for the softmax's quotient;
    * sums, exponentials and scale factors in 32 bits: 2^-18 covers sums of 10^5 such terms' errors of 2^-22 at random signs.
    """
    k8, v8, ks, vs = cache
    B, Hq, D = q.shape
    heads, page = k8.shape[1:3]
    out, tol = torch.zeros(B, Hq, D, dtype=torch.float64), torch.zeros(B, Hq, D, dtype=torch.float64)
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        lo = max(0, n - window) if window else 0
        pages = table[b, : -(-n // page)].long()
        take = lambda c, s: (c[pages].double() * s[pages].double()[:, :, None, None]).transpose(0, 1).reshape(heads, -1, D)[:, lo:n]  # noqa: E731
        k, v = take(k8, ks), take(v8, vs)
        sv = vs[pages].double().repeat_interleave(page, 0).t()[:, lo:n]
        qq = q[b].double().view(heads, Hq // heads, D)
        s = torch.einsum("hgd,htd->hgt", qq, k) * scale
        ds = 2 * (D + 8) * 2.0**-24 * (torch.einsum("hgd,htd->hgt", qq.abs(), k.abs()) * abs(scale)).amax(-1, keepdim=True)
        p = torch.softmax(s, -1)
        o = torch.einsum("hgt,htd->hgd", p, v)
        mags = torch.einsum("hgt,htd->hgd", p, v.abs())
        # the largest weight is that of p * v_scale; what is below 2^-14 of it is off by up to 2^-25 of it
        top = (s + torch.log(sv)[:, None]).argmax(-1)
        small = (n - lo) * 2.0**-25 * 448 * sv.gather(1, top)[..., None] * p.gather(2, top[..., None])
        t = torch.finfo(q.dtype).eps / 2 * o.abs() + (2.0**-11 + 2.0**-18 + ds) * mags + small
        out[b], tol[b] = o.reshape(Hq, D), t.reshape(Hq, D)
    return out, tol


MASS_TOL = 2.0**-18  # relative error of a sum of fp32 exponentials: arguments down to -32 are off by 2^-19, the function by 2^-22


def check_sample(logits, rng, tok, logp, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Every row's token is the draw of the definition and its log-probability right, in 64 bits.

    Only what lies within the 32-bit errors of a border may fall either way: a token whose key is within 2^-21 (|z| + 32) of
    the largest (z, its noise and their sum are rounded to 24 bits), and tokens at the edge of top-p within MASS_TOL."""
    from trl_b200.oracle.ops import row_uniforms

    B, V = logits.shape
    logits, rng, tok, logp = logits.cpu(), rng.cpu(), tok.cpu(), logp.cpu()
    per = lambda x, i: x[i].item() if torch.is_tensor(x) else x  # noqa: E731
    u = row_uniforms(rng, V)
    for i in range(B):
        T, k, p, m = per(temperature, i), int(per(top_k, i)), per(top_p, i), per(min_p, i)
        z32 = logits[i].float() / max(torch.tensor(T, dtype=torch.float32), torch.tensor(1e-6))
        z = torch.nan_to_num(z32, nan=-math.inf, posinf=torch.finfo(torch.float32).max, neginf=-math.inf).double()
        t = int(tok[i])
        if z.max() == -math.inf:
            assert t == 0 and logp[i] == -math.inf, i
            continue
        zs, order = torch.sort(z, descending=True, stable=True)
        base = zs > -math.inf
        if 0 < k < V:
            base = base & (zs >= zs[k - 1])
        w = torch.where(base, torch.exp(zs - zs[0]), 0.0)
        before = w.cumsum(0) - w
        floor = zs[0] + (math.log(min(m, 1.0)) if m > 0 else -math.inf)

        def kept(sign):
            keep = base & (zs >= floor)
            if p < 1:
                keep = keep & ((before <= (max(p, 0.0) + sign * MASS_TOL) * w.sum()) | (torch.arange(V) == 0))
            return order[keep]

        least, most = kept(-1), kept(1)
        assert t in most.tolist(), (i, t)
        key = z if not T > 0 else z - torch.log(-torch.log(u[i]))
        slack = 2.0**-21 * (float(z[least].abs().max()) + 32) if T > 0 else 0.0
        if len(least) == len(most) and T > 0 and key[least].sort().values[-2:].diff().numel() and float(key[least].sort().values[-2:].diff()) > slack:
            assert t == int(least[key[least].argmax()]), i
        assert key[t] >= key[least].max() - slack, (i, t, float(key[t]), float(key[least].max()))
        if not T > 0:
            assert t == int((z == z.max()).nonzero()[0]), i
        off = MASS_TOL + 2.0**-23 * (abs(float(z[t] - z.max())) + 32)
        # differences first: beside 3e38 a logarithm of a count is nothing, even in 64 bits
        hi, lo = (float(z[t] - zs[0] - torch.logsumexp(z[x] - zs[0], 0)) for x in (least, most))
        assert lo - off <= float(logp[i]) <= hi + off, (i, lo, float(logp[i]), hi)

"""8-bit paged cache, its decode attention and filtered sampling on the GPU against 64-bit references."""
import math

import pytest
import torch

from kv8_util import attention64, check_sample, filled_cache, table_of
from trl_b200.ops import functional as F

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _same_cache(a, b):
    for x, y in zip(a, b):
        x, y = x.float().cpu(), y.float().cpu()
        assert torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(x.nan_to_num(), y.nan_to_num())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("page, dim, heads", [(16, 64, 1), (64, 128, 4), (32, 96, 3), (128, 256, 2)])
def test_append_equals_the_definition(dtype, page, dim, heads):
    """Codes and scales are whole decisions: equal, over several calls that fill pages from the middle and behind."""
    g = torch.Generator().manual_seed(page + dim)
    blocks = 6
    table = table_of(5, blocks, 5 * blocks + 2, g, "cuda")
    cache, ref = F.kv8_alloc(5 * blocks + 2, heads, page, dim, "cuda"), F.kv8_alloc(5 * blocks + 2, heads, page, dim)
    at = [0, 3, page - 1, page, 0]
    for lens in ([2 * page + 5, 1, 2, page, 0], [1] * 5, [page, 2 * page + 1, 1, 7, page - 1], [1] * 5):
        starts = _i32([-1 if i == 4 and lens[4] == 1 else a for i, a in enumerate(at)])
        k, v = (torch.randn(sum(lens), heads, dim, generator=g) * 2.0 ** torch.randint(-6, 7, (sum(lens), 1, 1), generator=g) for _ in range(2))
        k[0, 0, :4] = torch.tensor([math.inf, math.nan, -math.inf, 0.0])
        k, v = k.to(dtype).cuda(), v.to(dtype).cuda()
        cu = None if lens == [1] * 5 else _i32([sum(lens[:i]) for i in range(6)])
        F.kv8_append(k, v, *cache, table, starts, cu_seqlens=cu, max_new=max(lens))
        F.kv8_append(k.cpu(), v.cpu(), *ref, table.cpu(), starts.cpu(), cu_seqlens=None if cu is None else cu.cpu())
        _same_cache(cache, ref)
        at = [a + n for a, n in zip(at, lens)]


def test_append_slots_strides_and_streams():
    """Rows of the block table by slot, keys and values as parts of one projection, a side stream."""
    g = torch.Generator().manual_seed(3)
    heads, page, dim = 2, 16, 64
    table = table_of(4, 3, 20, g, "cuda")
    qkv = torch.randn(30, 5 * heads * dim, generator=g).bfloat16().cuda()
    k, v = qkv[:, 2 * dim:4 * dim].view(30, heads, dim), qkv[:, 4 * dim:6 * dim].view(30, heads, dim)
    slots, starts, cu = _i32([3, 1]), _i32([5, 0]), _i32([0, 10, 30])
    cache, ref = F.kv8_alloc(20, heads, page, dim, "cuda"), F.kv8_alloc(20, heads, page, dim)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        F.kv8_append(k, v, *cache, table, starts, cu_seqlens=cu, slots=slots)
    torch.cuda.current_stream().wait_stream(side)
    F.kv8_append(k.cpu(), v.cpu(), *ref, table.cpu(), starts.cpu(), cu_seqlens=cu.cpu(), slots=slots.cpu())
    _same_cache(cache, ref)


def test_pages_that_do_not_exist_are_reported_and_left_out():
    from trl_b200.ops import cuda as K

    K.check_status()
    cache, _ = filled_cache([16], 1, 16, 64, "cuda")
    was = [t.clone() for t in cache]
    k = torch.ones(1, 1, 64, device="cuda").bfloat16()
    for table, start in ((_i32([[99]]), 0), (_i32([[-1]]), 0), (_i32([[0]]), 16)):
        F.kv8_append(k, k, *cache, table, _i32([start]))
        with pytest.raises(RuntimeError, match="code=3"):
            K.check_status()
    F.kv8_append(k, k, *cache, _i32([[0]]), _i32([0]), slots=_i32([1]))
    with pytest.raises(RuntimeError, match="code=3"):
        K.check_status()
    _same_cache(cache, was)
    # attention: a missing page's tokens count for nothing
    q = torch.randn(1, 1, 64, device="cuda").bfloat16()
    out = F.kv8_decode_attn(q, *cache, _i32([[99, 0]]), _i32([31]), 0.1)
    with pytest.raises(RuntimeError, match="code=3"):
        K.check_status()
    want, tol = attention64(q.cpu(), [t.cpu() for t in cache], torch.zeros(1, 1, dtype=torch.int32), [16], 0.1)
    assert ((out.cpu().double() - want).abs() <= tol).all()


CASES = [  # lengths, heads, key heads, dim, page, window
    ([1], 1, 1, 64, 16, None), ([1, 2, 15, 16, 17, 31, 33], 8, 1, 128, 16, None), ([211], 14, 2, 64, 16, None),
    ([300, 0, 64, 65, 1, 129], 28, 4, 128, 64, None), ([77, 500], 12, 1, 128, 32, None), ([40, 41, 97], 16, 1, 96, 32, None),
    ([70, 1000, 3], 6, 6, 96, 32, None), ([130, 17, 260], 10, 2, 256, 128, None), ([90], 40, 2, 64, 64, None),
    ([5000, 1, 33], 32, 8, 128, 64, None), ([700, 20, 64, 1], 8, 2, 128, 64, 64), ([700, 20, 129, 1], 4, 4, 64, 16, 1),
    ([333] * 40, 4, 2, 128, 64, 100), ([20000], 8, 8, 128, 64, None), ([9, 0, 0, 4], 3, 1, 64, 16, None)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens, Hq, Hk, D, page, window", CASES)
def test_attention_matches_64_bits(lens, Hq, Hk, D, page, window, dtype):
    cache, table = filled_cache(lens, Hk, page, D, "cuda", seed=len(lens) + D)
    g = torch.Generator().manual_seed(7)
    q = (torch.randn(len(lens), Hq, D, generator=g) * torch.rand(len(lens), Hq, 1, generator=g)).to(dtype).cuda()
    scale = 0.02 / math.sqrt(D)  # codes of size 60
    out = F.kv8_decode_attn(q, *cache, table, _i32([n - 1 for n in lens]), scale, window=window)
    want, tol = attention64(q.cpu(), [t.cpu() for t in cache], table.cpu(), lens, scale, window)
    err = (out.cpu().double() - want).abs()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-30)).max())


def test_attention_of_pages_with_very_different_scales():
    """Scales from 2^-40 to 2^40 within a row: the weights stay within fp16 because the scale is part of the exponent."""
    lens = [500, 64, 1000]
    cache, table = filled_cache(lens, 2, 16, 128, "cuda", spread=40)
    cache = (cache[0], cache[1], torch.full_like(cache[2], 0.01).copy_(torch.ones_like(cache[2]) * 2**-7), cache[3])
    q = torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    out = F.kv8_decode_attn(q, *cache, table, _i32([n - 1 for n in lens]), 0.05)
    want, tol = attention64(q.cpu(), [t.cpu() for t in cache], table.cpu(), lens, 0.05)
    assert ((out.cpu().double() - want).abs() <= tol).all()


def test_attention_ignores_what_is_out_of_sight():
    """NaN and the largest codes before a window, behind the newest token and in other pages change nothing."""
    lens, window = [100, 37], 30
    cache, table = filled_cache(lens, 2, 16, 64, "cuda")
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    want = F.kv8_decode_attn(q, *cache, table, _i32([99, 36]), 0.01, window=window)
    for code in (0x7F, 0xFE, 0x7E):
        seen = torch.zeros(cache[0].shape[0], 16, dtype=torch.bool)
        for b, n in enumerate(lens):
            for t in range(max(0, n - window), n):
                seen[int(table[b, t // 16]), t % 16] = True
        spoiled = []
        for c in cache[:2]:
            u = c.clone().view(torch.uint8)
            u[(~seen)[:, None, :, None].expand_as(u)] = code
            spoiled.append(u.view(torch.float8_e4m3fn))
        assert torch.equal(F.kv8_decode_attn(q, *spoiled, *cache[2:], table, _i32([99, 36]), 0.01, window=window), want)


def test_attention_slots_strides_out_and_repeats():
    lens = [50, 0, 333, 64]
    cache, table = filled_cache(lens, 2, 16, 64, "cuda")
    big = torch.randn(3, 9, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    q, slots = big[:, 2:8], [2, 0, 2]
    want, tol = attention64(q.cpu(), [t.cpu() for t in cache], table.cpu()[slots], [lens[s] for s in slots], 0.01)
    out = torch.full((4, 6, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    got = F.kv8_decode_attn(q, *cache, table, _i32([n - 1 for n in lens]), 0.01, slots=_i32(slots), out=out[:3])
    assert got.data_ptr() == out.data_ptr() and (out[3] == 7).all()
    assert ((got.cpu().double() - want).abs() <= tol).all()
    again = F.kv8_decode_attn(q, *cache, table, _i32([n - 1 for n in lens]), 0.01, slots=_i32(slots))
    assert torch.equal(again, got) and torch.equal(got[0], F.kv8_decode_attn(q[:1], *cache, table, _i32([n - 1 for n in lens]), 0.01, slots=_i32([2]))[0]) is not None


def test_two_streams_and_two_graphs_do_not_share_scratch():
    lens = [9000, 8000]
    cache, table = filled_cache(lens, 4, 64, 128, "cuda")
    seq = _i32([n - 1 for n in lens])
    qs = [torch.randn(2, 16, 128, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in range(2)]
    want = [F.kv8_decode_attn(q, *cache, table, seq, 0.01).clone() for q in qs]
    streams, outs, graphs = [torch.cuda.Stream() for _ in range(2)], [torch.empty_like(q) for q in qs], []
    for q, o in zip(qs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            F.kv8_decode_attn(q, *cache, table, seq, 0.01, out=o)
        graphs.append(g)
    for _ in range(20):
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_many_sequences():
    lens = [1 + (i * 7919) % 90 for i in range(1500)]
    cache, table = filled_cache(lens, 1, 16, 64, "cuda")
    q = torch.randn(1500, 2, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    out = F.kv8_decode_attn(q, *cache, table, _i32([n - 1 for n in lens]), 0.01)
    want, tol = attention64(q.cpu(), [t.cpu() for t in cache], table.cpu(), lens, 0.01)
    assert ((out.cpu().double() - want).abs() <= tol).all()


# ---- sampling ------------------------------------------------------------------------------------------------------
def _logits(rows, vocab, dtype, seed=0, sharp=2.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, vocab, generator=g) * sharp
    z.scatter_add_(1, torch.randint(0, vocab, (rows, min(vocab, 20)), generator=g), torch.rand(rows, min(vocab, 20), generator=g) * 8)
    rng = torch.randint(-2**31, 2**31 - 1, (rows,), generator=g).to(torch.int32)
    return z.to(dtype).cuda(), rng.cuda()


@pytest.mark.parametrize("kw", [
    {}, {"temperature": 0.0}, {"top_k": 1}, {"top_k": 20, "top_p": 0.8}, {"top_p": 0.95}, {"top_p": 0.3, "temperature": 0.5},
    {"min_p": 0.05}, {"top_k": 300, "min_p": 0.01, "top_p": 0.99}, {"top_p": 0.999, "temperature": 1.5}, {"top_k": 6000},
    {"top_k": 6000, "top_p": 0.9, "temperature": 1.3}, {"top_p": 0.0}, {"temperature": 0.0, "top_k": 5, "top_p": 0.5}])
@pytest.mark.parametrize("rows, vocab, dtype", [(3, 32000, torch.bfloat16), (1, 152064, torch.float32), (40, 5003, torch.float16)])
def test_sampling_matches_64_bits(rows, vocab, dtype, kw):
    logits, rng = _logits(rows, vocab, dtype, seed=rows)
    tok, logp = F.sample_filtered(logits, rng, **kw)
    check_sample(logits, rng, tok, logp, **kw)
    again = F.sample_filtered(logits, rng, **kw)
    assert torch.equal(tok, again[0]) and torch.equal(logp, again[1])


@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 9, 17, 1000])
def test_sampling_of_small_vocabularies(vocab):
    logits, rng = _logits(150, vocab, torch.float32)
    for kw in ({}, {"top_k": 2}, {"top_p": 0.6}, {"top_k": 3, "top_p": 0.9, "min_p": 0.1}):
        check_sample(logits, rng, *F.sample_filtered(logits, rng, **kw), **kw)


def test_sampling_parameters_per_row_and_strides():
    logits, rng = _logits(64, 4099, torch.float32)
    wide = torch.empty(64, 4200, device="cuda")
    view = wide[:, 33:33 + 4099]
    view.copy_(logits)
    g = torch.Generator().manual_seed(5)
    kw = {"temperature": torch.where(torch.rand(64, generator=g) < 0.2, 0.0, torch.rand(64, generator=g) * 2),
          "top_k": torch.randint(0, 80, (64,), generator=g).to(torch.int32), "top_p": torch.rand(64, generator=g) * 1.2,
          "min_p": torch.rand(64, generator=g) * 0.2 * (torch.rand(64, generator=g) < 0.5)}
    tok, logp = F.sample_filtered(view, rng, **{k: v.cuda() for k, v in kw.items()})
    check_sample(logits, rng, tok, logp, **kw)


@pytest.mark.parametrize("fill", ["equal", "two values", "grid", "nearly equal"])
def test_sampling_of_many_equals(fill):
    """More equal tokens at the border than a list holds: the lower columns stay."""
    rows, vocab = 6, 40000
    z = torch.zeros(rows, vocab)
    g = torch.Generator().manual_seed(0)
    if fill == "two values":
        z[:, ::3] = 1.0
    elif fill == "grid":
        z = torch.randint(0, 4, (rows, vocab), generator=g).float()
    elif fill == "nearly equal":
        z = 1 + torch.rand(rows, vocab, generator=g) * 2**-10
    rng = torch.arange(rows, dtype=torch.int32).cuda()
    for kw in ({"top_p": 0.5}, {"top_p": 0.9}, {"top_k": 10}, {"top_k": 20000, "top_p": 0.7}, {"top_k": 39999}, {"top_p": 0.1, "temperature": 2.0}):
        tok, logp = F.sample_filtered(z.cuda(), rng, **kw)
        check_sample(z, rng, tok, logp, **kw)


def test_sampling_of_spoiled_rows():
    inf, nan = math.inf, math.nan
    z = torch.full((8, 70000), -inf)
    z[1, 69999] = -3.0
    z[2, 5], z[2, 7] = nan, 1.0
    z[3, 11] = inf
    z[3, 12], z[4, 100:200] = 3.0, torch.arange(100.0)
    z[5] = nan
    z[6, :60000] = -1000.0
    z[6, 60000] = 1000.0
    z[7] = torch.linspace(-3e38, 3e38, 70000)
    rng = torch.arange(8, dtype=torch.int32).cuda()
    for kw in ({}, {"top_k": 50}, {"top_p": 0.5}, {"top_k": 5000, "top_p": 0.99}, {"temperature": 0.0}, {"min_p": 0.5}, {"temperature": 1e-30}):
        tok, logp = F.sample_filtered(z.cuda(), rng, **kw)
        check_sample(z, rng, tok, logp, **kw)


def test_sampling_frequencies():
    """Draws of 20000 words from one row follow its probabilities within five standard deviations."""
    p = torch.tensor([0.02, 0.5, 0.08, 0.3, 0.1])
    logits = torch.full((20000, 3000), -math.inf, device="cuda")
    logits[:, 100:105] = p.log().cuda()
    rng = torch.arange(20000, dtype=torch.int32, device="cuda")
    tok, _ = F.sample_filtered(logits, rng)
    freq = torch.bincount(tok.long().cpu(), minlength=105)[100:].float() / 20000
    assert ((freq - p).abs() <= 5 * (p * (1 - p) / 20000).sqrt()).all()


def test_a_decode_loop_of_all_three_operators():
    """Prompts, then steps of append, attention and sampling, eager and from a captured graph, against the definitions."""
    g = torch.Generator().manual_seed(11)
    heads, Hq, D, page, V, steps = 2, 6, 64, 16, 500, 20
    lens = [37, 5, 64]
    B, blocks = 3, 8
    table = table_of(B, blocks, 30, g, "cuda")
    head_w = (torch.randn(V, Hq * D, generator=g) * 0.3).bfloat16().cuda()
    emb = torch.randn(V, (Hq + 2 * heads) * D, generator=g).bfloat16().cuda()
    kv = [torch.randn(sum(lens), heads, D, generator=g).bfloat16().cuda() for _ in range(2)]
    words = torch.randint(-2**31, 2**31 - 1, (steps, B), generator=g).to(torch.int32).cuda()

    def rollout(use_graph):
        cache = F.kv8_alloc(30, heads, page, D, "cuda")
        F.kv8_append(*kv, *cache, table, _i32([0] * B), cu_seqlens=_i32([0, 37, 42, 106]), max_new=64)
        pos, tok, word = _i32(lens), torch.zeros(B, dtype=torch.int64, device="cuda"), words[0].clone()
        kept = []

        def step():
            x = emb[tok]
            q, k, v = x[:, :Hq * D].view(B, Hq, D), x[:, Hq * D:(Hq + heads) * D].view(B, heads, D), x[:, (Hq + heads) * D:].view(B, heads, D)
            F.kv8_append(k, v, *cache, table, pos)
            o = F.kv8_decode_attn(q, *cache, table, pos, D**-0.5)
            logits = (o.view(B, -1) @ head_w.t()) * 0.2
            t, lp = F.sample_filtered(logits, word, temperature=0.9, top_k=40, top_p=0.9)
            tok.copy_(t)
            pos.add_(1)
            return q, o, logits, t, lp

        if use_graph:
            side = torch.cuda.Stream()
            state = [t.clone() for t in (pos, tok, *cache)]
            with torch.cuda.stream(side):
                step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                res = step()
            for t, o in zip((pos, tok, *cache), state):
                t.view(torch.uint8).copy_(o.view(torch.uint8)) if t.dtype == torch.float8_e4m3fn else t.copy_(o)
        for i in range(steps):
            word.copy_(words[i])
            if use_graph:
                graph.replay()
            else:
                res = step()
            kept.append([t.clone() for t in res])
            if not use_graph:
                want, tol = attention64(res[0].cpu(), [t.cpu() for t in cache], table.cpu(), [n + i + 1 for n in lens], D**-0.5)
                assert ((res[1].cpu().double() - want).abs() <= tol).all()
                check_sample(res[2], word, res[3], res[4], temperature=0.9, top_k=40, top_p=0.9)
        return kept, cache

    a, ca = rollout(False)
    b, cb = rollout(True)
    for x, y in zip(a, b):
        assert torch.equal(x[3], y[3]) and torch.equal(x[1], y[1])
    _same_cache(ca, cb)


def test_fused_rope_append_equals_its_parts():
    """RoPE and append of a decode step in one kernel against the bf16 cache's kernel followed by the append."""
    from trl_b200.ops import cuda as K

    g = torch.Generator().manual_seed(2)
    for D, page, Hq, Hk in ((128, 64, 4, 2), (64, 16, 3, 1)):
        B, half = 5, D // 2
        pos = _i32([0, 17, -1, 40, 63])
        qkv = torch.randn(B, (Hq + 2 * Hk) * D, generator=g).bfloat16().cuda()
        table = table_of(B, 4, 4 * B + 1, g, "cuda")
        theta = 10000.0
        # the rotation in 64 bits, rounded where the kernel rounds
        ang = pos.cpu().double()[:, None] * theta ** (-torch.arange(half).double() * 2 / D)
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        x = qkv.cpu().double().view(B, Hq + 2 * Hk, D)[:, :Hq + Hk]
        rot = torch.cat([x[..., :half] * c - x[..., half:] * s, x[..., half:] * c + x[..., :half] * s], -1)
        for f32 in (False, True):
            cache = F.kv8_alloc(4 * B + 1, Hk, page, D, "cuda")
            q = torch.full((B, Hq, D), 9.0, dtype=torch.bfloat16, device="cuda")
            src = qkv.float() if f32 else qkv
            K.kv8_rope_append(src, None, None, None, 1e-6, pos, None, table, q, *cache, Hq, theta)
            live = (pos >= 0).cpu()
            # bf16's half step and the error of an fp32 angle of at most 64 (2^-18 of the pair's size)
            size = x.abs().amax()
            assert ((q.cpu().double() - rot[:, :Hq]).abs() <= 2.0**-8 * rot[:, :Hq].abs() + 2.0**-18 * size)[live].all()
            assert (q.cpu()[~live] == 9).all() and (not f32 or (src == 0).all())
            for i in live.nonzero().flatten().tolist():
                blk, row = int(table[i, int(pos[i]) // page]), int(pos[i]) % page
                for codes, scale, want in ((cache[0], cache[2], rot[i, Hq:]), (cache[1], cache[3], qkv.cpu().double().view(B, -1, D)[i, Hq + Hk:])):
                    held = codes[blk, :, row].cpu().double() * scale[blk].cpu().double()[:, None]
                    t = 2.0**-4 * want.abs() * (1 + 2.0**-7) + 2.0**-8 * want.abs() + 2.0**-18 * size + 2.0**-10 * scale[blk].cpu().double()[:, None]
                    assert ((held - want).abs() <= t).all()


@pytest.mark.parametrize("vocab, dtype", [(200003, torch.float32), (400000, torch.bfloat16)])
@pytest.mark.parametrize("kw", [{}, {"top_k": 70}, {"top_p": 0.9}, {"top_k": 900, "top_p": 0.5, "min_p": 0.001}, {"min_p": 0.1}])
def test_sampling_of_rows_beyond_shared_memory(vocab, dtype, kw):
    logits, rng = _logits(2, vocab, dtype, seed=7)
    check_sample(logits, rng, *F.sample_filtered(logits, rng, **kw), **kw)


@pytest.mark.parametrize("count", [1, 31, 63, 64, 65, 128, 129, 511, 512, 513, 1024, 1025, 2047, 2048, 2049, 5000])
def test_sampling_of_lists_of_all_lengths(count):
    """``count`` tokens, evenly spaced from likely to unlikely, among others that are out of reach."""
    g = torch.Generator().manual_seed(count)
    rows, vocab = 5, 20011
    z = torch.full((rows, vocab), -60.0)
    for i in range(rows):
        at = torch.randperm(vocab, generator=g)[:count]
        z[i, at] = -torch.arange(count) * (0.5, 0.05, 0.003, 12.0 / count, 0.0)[i]
    rng = torch.randint(-2**31, 2**31 - 1, (rows,), generator=g).to(torch.int32).cuda()
    for kw in ({"top_p": 0.9}, {"top_p": 0.999}, {"top_k": max(1, count // 2)}, {"top_k": min(count + 1, 512), "top_p": 0.7},
               {"top_p": 0.97, "min_p": 0.02}, {"top_p": 0.4, "min_p": 1e-4}):
        check_sample(z, rng, *F.sample_filtered(z.cuda(), rng, **kw), **kw)


def test_sampling_on_two_streams_and_replayed():
    logits, rng = _logits(9, 33000, torch.bfloat16)
    other, rng2 = _logits(9, 33000, torch.bfloat16, seed=1)
    kw = {"top_p": 0.9, "top_k": 400}
    want, want2 = F.sample_filtered(logits, rng, **kw), F.sample_filtered(other, rng2, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        a = F.sample_filtered(logits, rng, **kw)
        with torch.cuda.stream(side):
            b = F.sample_filtered(other, rng2, **kw)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip((*a, *b), (*want, *want2)))
    z, words = logits.clone(), rng.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = F.sample_filtered(z, words, **kw)
    for x, r, w in ((logits, rng, want), (other, rng2, want2), (logits, rng, want)):
        z.copy_(x)
        words.copy_(r)
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(c, w))


@pytest.mark.parametrize("D, Hq, Hk", [(64, 8, 2), (128, 4, 4), (256, 8, 1)])
def test_attention_repeats_itself(D, Hq, Hk):
    """The same call gives the same bits, whatever runs beside it."""
    lens = [1, 700, 4097, 63, 0, 129]
    cache, table = filled_cache(lens, Hk, 32, D, "cuda", seed=D)
    q = torch.randn(len(lens), Hq, D, device="cuda").to(torch.bfloat16)
    at = _i32([n - 1 for n in lens])
    first = F.kv8_decode_attn(q, *cache, table, at, D**-0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        with torch.cuda.stream(side):
            beside = F.kv8_decode_attn(q, *cache, table, at, D**-0.5)
        assert torch.equal(first, F.kv8_decode_attn(q, *cache, table, at, D**-0.5))
    torch.cuda.synchronize()
    assert torch.equal(first, beside)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sampling_of_more_rows_than_are_held(dtype):
    """Rows that start at odd places, of all kinds of parameters, some with infinities and NaN."""
    rows, vocab = 330, 4099
    logits, rng = _logits(rows, vocab, torch.float32, seed=3, sharp=1.5)
    g = torch.Generator().manual_seed(9)
    logits[::11, :2000] = -math.inf
    logits[5::37, 17] = math.nan
    logits[6::41, 400] = math.inf
    logits[7::53] = -math.inf
    logits[8::59] = 0.25
    logits = logits.to(dtype)
    kw = {"temperature": torch.where(torch.rand(rows, generator=g) < 0.1, 0.0, 0.2 + torch.rand(rows, generator=g) * 2),
          "top_k": torch.where(torch.rand(rows, generator=g) < 0.5, 0, torch.randint(0, 1500, (rows,), generator=g)).to(torch.int32),
          "top_p": 0.2 + torch.rand(rows, generator=g), "min_p": torch.rand(rows, generator=g) * 0.1 * (torch.rand(rows, generator=g) < 0.5)}
    tok, logp = F.sample_filtered(logits, rng, **{k: v.cuda() for k, v in kw.items()})
    check_sample(logits, rng, tok, logp, **kw)
    few = F.sample_filtered(logits[40:60], rng[40:60], **{k: v[40:60].cuda() for k, v in kw.items()})
    assert torch.equal(tok[40:60], few[0])  # a row's draw does not depend on how many there are


@pytest.mark.parametrize("D, Hq, Hk, page, dtype", [(64, 14, 2, 16, torch.bfloat16), (128, 34, 2, 64, torch.float16), (96, 5, 5, 32, torch.bfloat16), (256, 8, 1, 16, torch.bfloat16)])
@pytest.mark.parametrize("room", [64, 600, 1600])
def test_attention_of_few_rows_whatever_the_table_has_room_for(D, Hq, Hk, page, dtype, room):
    """The room in the block table decides how the work is dealt, not what comes out."""
    lens = [0, 1, 17, 63]
    cache, narrow = filled_cache(lens, Hk, page, D, "cuda", seed=room)
    table = torch.zeros(len(lens), room // page, dtype=torch.int32, device="cuda")
    table[:, :narrow.shape[1]] = narrow
    q = torch.randn(len(lens), Hq, D, device="cuda").to(dtype)
    slots = _i32([3, 1, 0, 2])
    at = _i32([n - 1 for n in lens])
    for window in (None, 5, 2**31 - 1):
        out = F.kv8_decode_attn(q, *cache, table, at, D**-0.5, slots=slots, window=window)
        order = [lens[i] for i in slots.tolist()]
        want, tol = attention64(q.cpu(), [x.cpu() for x in cache], table[slots.long()].cpu(), order, D**-0.5, window)
        assert ((out.cpu().double() - want).abs() <= tol).all()
        assert (out[2] == 0).all()

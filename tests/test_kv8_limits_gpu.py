"""The 8-bit paged cache, its decode attention and filtered sampling at the limits of their numbers (B200)."""
import math

import pytest
import torch

from kv8_util import attention64, check_sample, filled_cache
from trl_b200.ops import functional as F

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cpu(cache):
    return [t.cpu() for t in cache]


# rows that a block takes alone; that a warp takes whole; that a block's warps share; that several blocks share
SHAPES = [("a block a row", [60, 17, 200, 33], 4, 2, 64, 16), ("a warp a row", [20 + i % 30 for i in range(700)], 8, 4, 64, 16),
          ("a block's warps", [9000, 8500, 9100, 9050] * 3, 8, 4, 128, 64), ("blocks", [120000, 90001, 50], 8, 1, 128, 64)]


# ---- attention -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name, lens, Hq, Hk, D, page", SHAPES, ids=[s[0] for s in SHAPES])
@pytest.mark.parametrize("what", ["nan query", "inf query", "-inf query", "nan key", "nan value"])
def test_attention_keeps_nan_that_is_in_sight(name, lens, Hq, Hk, D, page, what):
    """NaN comes out wherever the formula gives it, however a row is dealt to warps, and nowhere else."""
    cache, table = filled_cache(lens, Hk, page, D, "cuda", seed=3, extra=0)
    B, G = len(lens), Hq // Hk
    q = torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    bad = torch.zeros(B, Hq, D, dtype=torch.bool)
    row, head = 1, Hq - 1
    if what.endswith("query"):
        if what != "nan query":  # scores of one sign: all +inf (NaN by inf - inf) or all -inf (0 / 0)
            pages = table[row, : -(-lens[row] // page)].long()
            u = cache[0].view(torch.uint8)
            u[pages, head // G, :, 5] = torch.tensor([1.0]).to(torch.float8_e4m3fn).view(torch.uint8).item()
        q[row, head, 5] = float(what.split()[0])
        bad[row, head] = True
    else:
        at = lens[row] - 3
        u = cache[0 if what == "nan key" else 1].view(torch.uint8)
        u[int(table[row, at // page]), head // G, at % page, 7] = 0x7F
        heads = slice(head // G * G, head // G * G + G)
        bad[row, heads] = True
        if what == "nan value":
            bad[row, heads] = False
            bad[row, heads, 7] = True
    some = [0, 1, 2, B - 1] if B > 3 else list(range(B))
    out = F.kv8_decode_attn(q, *cache, table, _i32([n - 1 for n in lens]), 0.01).cpu()
    assert torch.equal(torch.isnan(out), bad)
    clean, c8 = q.clone(), [t.clone() for t in cache]
    clean[~torch.isfinite(clean)] = 0
    for c in c8[:2]:
        u = c.view(torch.uint8)
        u[(u & 0x7F) == 0x7F] = 0
    want, tol = attention64(clean[some].cpu(), _cpu(c8), table[some].cpu(), [lens[i] for i in some], 0.01)
    err = (out[some].double() - want).abs()
    assert (err <= tol)[~bad[some]].all()


@pytest.mark.parametrize("name, lens, Hq, Hk, D, page", SHAPES, ids=[s[0] for s in SHAPES])
def test_attention_of_scores_far_below_zero(name, lens, Hq, Hk, D, page):
    """All scores of a row equal and about -2^120: the softmax is uniform, the output the values' mean.

    Its error: the output's half step, weights and sums 2^-11 of the magnitudes' mean.  One scale for all values: in 32 bits
    scores of this size have steps of 2^97, beside which the logarithm of a page's scale is nothing."""
    cache, table = filled_cache(lens, Hk, page, D, "cuda", seed=4, extra=0)
    cache[0].view(torch.uint8).fill_(torch.tensor([1.0]).to(torch.float8_e4m3fn).view(torch.uint8).item())
    cache[2].fill_(2.0**114)
    cache[3].fill_(0.5)
    q = torch.full((len(lens), Hq, D), -1.0, device="cuda", dtype=torch.bfloat16)
    out = F.kv8_decode_attn(q, *cache, table, _i32([n - 1 for n in lens]), 1.0).cpu()
    for b in {0, 1, len(lens) - 1}:
        pages = table[b, : -(-lens[b] // page)].long()
        v = (cache[1][pages].double() * cache[3][pages].double()[:, :, None, None]).transpose(0, 1).reshape(Hk, -1, D)[:, : lens[b]].cpu()
        want, mags = (x.repeat_interleave(Hq // Hk, 0) for x in (v.mean(1), v.abs().mean(1)))
        assert ((out[b].double() - want).abs() <= torch.finfo(torch.bfloat16).eps / 2 * want.abs() + 2.0**-10 * mags).all()


@pytest.mark.parametrize("B, n, drop", [(1000, 8000, 20), (1000, 8000, 26), (900, 3000, 28), (3, 600, 24), (2, 600, 27)])
def test_attention_keeps_many_small_weights_beside_a_large_one(B, n, drop):
    """One token of value 0 has nearly all the weight, the others 2^-drop of it each: their sum is the output.  With many
    sequences (of the same pages) a warp takes a whole row.

    A weight is rounded to fp16 once, 2^-11 of it, and where it is below fp16's normal numbers by up to 2^-32 of the largest (the
    largest stands at 2^7 or above, the smallest step of fp16 is 2^-24, its half 2^-25)."""
    Hk, G, D, page = 2, 4, 128, 64
    cache, table = filled_cache([n], Hk, page, D, "cuda", seed=5, extra=0)
    cache[2].fill_(1.0)
    cache[3].fill_(2.0**-3)
    first, row = int(table[0, 0]), 7
    u = cache[0].view(torch.uint8)
    u.fill_(0)
    u[first, :, row, 0] = torch.tensor([1.0]).to(torch.float8_e4m3fn).view(torch.uint8).item()
    cache[1].view(torch.uint8).bitwise_and_(0x7F)  # values of one sign: no cancellation
    cache[1].view(torch.uint8)[first, :, row] = 0  # the value of the heavy token
    q = torch.zeros(B, Hk * G, D, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 1.0
    out = F.kv8_decode_attn(q, *cache, table.expand(B, -1).contiguous(), _i32([n - 1] * B), drop * math.log(2)).cpu().double()
    v = (cache[1].double() * 2.0**-3)[table[0].long()].transpose(0, 1).reshape(Hk, -1, D)[:, :n].cpu()
    den = 1 + (n - 1) * 2.0**-drop
    want = (v.sum(1) * 2.0**-drop / den).repeat_interleave(G, 0)[None]
    mags = (v.sum(1) / den).repeat_interleave(G, 0)[None]
    tol = torch.finfo(q.dtype).eps / 2 * want + (2.0**-11 * 2.0**-drop + 2.0**-32 + 2.0**-18 * 2.0**-drop) * mags
    assert ((out - want).abs() <= tol).all(), float(((out - want).abs() / tol).max())
    assert (want > 8 * tol).all()  # what is lost would be seen


@pytest.mark.parametrize("Hq, Hk, page", [(9, 1, 16), (24, 2, 64), (40, 2, 128)])
def test_attention_of_wide_heads_in_several_tiles(Hq, Hk, page):
    """Head dim 256 with more than eight query heads a key head: their pages are read by several tiles."""
    lens = [1, 700, 64, 2100, 0, 33]
    cache, table = filled_cache(lens, Hk, page, 256, "cuda", seed=Hq)
    q = torch.randn(len(lens), Hq, 256, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    for window in (None, 50):
        out = F.kv8_decode_attn(q, *cache, table, _i32([n - 1 for n in lens]), 0.002, window=window)
        want, tol = attention64(q.cpu(), _cpu(cache), table.cpu(), lens, 0.002, window)
        assert ((out.cpu().double() - want).abs() <= tol).all() and (out[4] == 0).all()


def test_a_sequence_alone_has_the_output_that_it_has_in_a_batch():
    """Within the bound of each: the work is dealt otherwise, so the bits may differ."""
    lens = [50, 0, 333, 64]
    cache, table = filled_cache(lens, 2, 16, 64, "cuda")
    big = torch.randn(3, 9, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    q, slots, seq = big[:, 2:8], [2, 0, 2], _i32([n - 1 for n in lens])
    want, tol = attention64(q.cpu(), _cpu(cache), table.cpu()[slots], [lens[s] for s in slots], 0.01)
    for i, slot in enumerate(slots):
        out = F.kv8_decode_attn(q[i:i + 1], *cache, table, seq, 0.01, slots=_i32([slot]))
        assert ((out.cpu().double() - want[i:i + 1]).abs() <= tol[i:i + 1]).all()


# ---- RoPE and append -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("D, page, Hq, Hk", [(128, 64, 4, 2), (64, 16, 3, 1), (64, 128, 2, 2), (96, 32, 5, 1)])
def test_rope_append_brings_earlier_rows_to_a_grown_scale(D, page, Hq, Hk, f32):
    """Codes and scales are those of the definition's append of the rotated row: earlier rows of the page at the new scale, later
    ones and other pages as they were.  The first query heads have the keys' values, so they show the keys as they were rotated
    and rounded; those are held to 64 bits.  Far positions, with and without a shift of them."""
    from trl_b200.ops import cuda as K
    from trl_b200.oracle import ops as R

    g = torch.Generator().manual_seed(D + page)
    B, blocks, half, theta = 6, 70, D // 2, 1e4
    lens = [(blocks - 3) * page + page // 2, 5, 0, 40 * page + 1, -1, 17 * page + page - 1]
    cache, table = filled_cache([max(1, n + 1) for n in lens], Hk, page, D, "cuda", seed=page)
    for c, s in zip(cache[:2], cache[2:]):
        c.view(torch.uint8)[(c.view(torch.uint8) & 0x7F) == 0x7F] = 0x55
        s.copy_(torch.ldexp(torch.ones(s.shape), torch.randint(-9, 0, s.shape, generator=g)))
    for delta in (None, torch.tensor([3, 900, 0, -2, 7, 11], dtype=torch.int32)):
        # sizes from 2^-6 to 2^9: scales of 2^-9 .. 2^-1, for magnitudes up to 224, grow in some pages and stay in others
        x = torch.randn(B, Hq + 2 * Hk, D, generator=g) * 2.0 ** torch.randint(-6, 10, (B, 1, 1), generator=g)
        x[:, :Hk] = x[:, Hq:Hq + Hk]
        x = x.bfloat16()
        got, was = [t.clone() for t in cache], _cpu(cache)
        q = torch.full((B, Hq, D), 9.0, dtype=torch.bfloat16, device="cuda")
        src = x.view(B, -1).cuda()
        K.kv8_rope_append(src.float() if f32 else src, None, None, None, 1e-6, _i32(lens), None, table, q, *got, Hq, theta,
                          pos_delta=None if delta is None else delta.cuda())
        K.check_status()
        got, q = _cpu(got), q.cpu()
        # an angle is off by what its exponent of up to 13.3 is in 32 bits (three roundings of 2^-24 of it) and 2^-22: below 2^-18.5
        pos = torch.tensor(lens).double() + (0 if delta is None else delta.double())
        ang = pos[:, None, None] * theta ** (-torch.arange(half).double() * 2 / D)
        y = x[:, :Hq].double()
        lo, hi, size = y[..., :half], y[..., half:], (y[..., :half].square() + y[..., half:].square()).sqrt().repeat(1, 1, 2)
        want = torch.cat([lo * ang.cos() - hi * ang.sin(), hi * ang.cos() + lo * ang.sin()], -1)
        tol = torch.finfo(q.dtype).eps / 2 * want.abs() + size * (ang.abs().repeat(1, 1, 2) * 2.0**-18.5 + 2.0**-20)
        live = torch.tensor(lens) >= 0
        assert ((q.double() - want).abs() <= tol)[live].all() and (q[~live] == 9).all()
        grown = 0
        for i, n in enumerate(lens):
            if n < 0:
                continue
            page_id, row = int(table[i, n // page]), n % page
            for which, new in ((0, q[i, :Hk].float()), (1, x[i, Hq + Hk:].float())):
                codes, scale, c0, s0 = got[which][page_id], got[2 + which][page_id], was[which][page_id], was[2 + which][page_id]
                need = R.kv8_scale(new.abs().amax(-1))
                now = torch.maximum(s0, need) if row else need
                assert torch.equal(scale, now)
                again = (c0[:, :row].float() * (s0 / now)[:, None, None]).to(c0.dtype)
                assert torch.equal(codes[:, :row].view(torch.uint8), again.view(torch.uint8))
                assert torch.equal(codes[:, row].view(torch.uint8), (new / now[:, None]).to(c0.dtype).view(torch.uint8))
                assert torch.equal(codes[:, row + 1:].view(torch.uint8), c0[:, row + 1:].view(torch.uint8))
                grown += int(row > 0 and bool((now > s0).any()))
        assert grown > 0
        rest = sorted(set(range(cache[0].shape[0])) - {int(table[i, n // page]) for i, n in enumerate(lens) if n >= 0})
        for a, b in zip(got, was):
            a, b = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (a, b))
            assert torch.equal(a[rest], b[rest])


@pytest.mark.parametrize("f32", [False, True])
def test_rope_append_reports_slots_that_the_table_does_not_have(f32):
    """They are treated as idle: their sums are cleared, nothing is written for them, the other rows are as ever."""
    from trl_b200.ops import cuda as K

    K.check_status()
    D, Hq, Hk, page = 64, 2, 1, 16
    cache, table = filled_cache([40] * 3, Hk, page, D, "cuda", seed=6)
    x = torch.randn(4, (Hq + 2 * Hk) * D, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    seq, delta = _i32([17, 5, 20]), _i32([0, 3, 0])
    got, want = ([t.clone() for t in cache] for _ in range(2))
    q, ref = (torch.full((4, Hq, D), 9.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    src = x.float() if f32 else x
    K.kv8_rope_append(src, None, None, None, 1e-6, seq, _i32([3, 1, -1, 2**31 - 1]), table, q, *got, Hq, 1e4, pos_delta=delta)
    with pytest.raises(RuntimeError, match="code=3"):
        K.check_status()
    K.kv8_rope_append(x[1:2], None, None, None, 1e-6, seq, _i32([1]), table, ref[1:2], *want, Hq, 1e4, pos_delta=delta)
    K.check_status()
    assert torch.equal(q, ref) and (not f32 or bool((src == 0).all()))
    for a, b in zip(got, want):
        assert torch.equal(*(t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (a, b)))


# ---- sampling ------------------------------------------------------------------------------------------------------
def _neighbours(rows, vocab, seed, levels=8):
    """fp32 logits on a few levels, each up to three steps of fp32 above its level: many quotients by a temperature are equal
    where the logits are not."""
    g = torch.Generator().manual_seed(seed)
    base = (torch.randint(0, levels, (rows, vocab), generator=g) * 0.37 + 1.03 + torch.rand(rows, 1, generator=g))
    z = (base.view(torch.int32) + torch.randint(0, 4, (rows, vocab), generator=g).to(torch.int32)).view(torch.float32)
    rng = torch.randint(-2**31, 2**31 - 1, (rows,), generator=g).to(torch.int32)
    return z, rng


# rows in the shared memory of a cluster; more rows than are held; rows longer than shared memory
@pytest.mark.parametrize("rows, vocab", [(40, 3001), (330, 4099), (6, 40000), (2, 200003)])
@pytest.mark.parametrize("kw", [{"temperature": 0.0}, {"temperature": 0.0, "top_p": 0.9}, {"temperature": 0.0, "top_k": 7, "min_p": 0.3},
                                {"temperature": 0.7, "top_k": 20}, {"temperature": 0.7, "top_k": 300, "top_p": 0.8}, {"temperature": 0.3, "top_k": 1000},
                                {"temperature": 0.7, "top_p": 0.3}, {"temperature": 1.3, "top_p": 0.9}, {"temperature": 0.05, "top_p": 0.7},
                                {"temperature": 0.7, "min_p": 1.0}, {"temperature": 0.9, "min_p": 0.4, "top_p": 0.6}])
def test_sampling_compares_quotients(rows, vocab, kw):
    """Logits whose quotients by the temperature are equal are equals, whichever of them is larger."""
    z, rng = _neighbours(rows, vocab, rows + vocab)
    tok, logp = F.sample_filtered(z.cuda(), rng.cuda(), **kw)
    check_sample(z, rng, tok, logp, **kw)


def test_sampling_compares_quotients_by_temperatures_of_rows():
    rows, vocab = 300, 700
    z, rng = _neighbours(rows, vocab, 1, levels=3)
    g = torch.Generator().manual_seed(2)
    kw = {"temperature": torch.where(torch.rand(rows, generator=g) < 0.3, 0.0, 0.1 + 2 * torch.rand(rows, generator=g)),
          "top_k": torch.randint(0, 400, (rows,), generator=g).to(torch.int32), "top_p": 0.2 + torch.rand(rows, generator=g)}
    tok, logp = F.sample_filtered(z.cuda(), rng.cuda(), **{k: v.cuda() for k, v in kw.items()})
    check_sample(z, rng, tok, logp, **kw)


@pytest.mark.parametrize("kw", [{}, {"top_k": 2}, {"top_p": 0.9}, {"min_p": 0.1}, {"temperature": 0.0}])
def test_sampling_of_quotients_that_are_not_finite(kw):
    """Finite logits whose quotients are infinite, and temperatures without bound."""
    z = torch.full((6, 1000), -3.0e38)
    z[1, 5], z[2, 9], z[2, 700] = -1.0e37, 3.0e38, 3.2e38
    z[3] = torch.linspace(-1e-38, 1e-38, 1000)
    z[4, 17], z[5, :] = 4.0, torch.linspace(-30, 30, 1000)
    rng = torch.arange(6, dtype=torch.int32)
    for t in (0.5, 0.25, 4e4, 1e20, math.inf):
        par = {"temperature": t, **kw}
        tok, logp = F.sample_filtered(z.cuda(), rng.cuda(), **par)
        check_sample(z, rng, tok, logp, **par)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [6, 700])
def test_sampling_of_infinite_logits(dtype, rows):
    """+inf stands for fp32's largest number, beside the largest of a narrower type too, however many rows there are."""
    vocab = 1500
    g = torch.Generator().manual_seed(rows)
    top = torch.finfo(dtype).max
    z = (torch.randn(rows, vocab, generator=g) * 2).to(dtype)
    z[0::6, 7], z[0::6, 3] = math.inf, top
    z[1::6, 3], z[1::6, 4] = top, torch.nextafter(torch.tensor(top, dtype=dtype), torch.tensor(0.0, dtype=dtype))
    z[2::6, 100], z[2::6, 90], z[2::6, 110] = math.inf, math.inf, top
    z[3::6, 11], z[3::6, 12] = math.nan, top
    rng = torch.randint(-2**31, 2**31 - 1, (rows,), generator=g).to(torch.int32)
    for kw in ({}, {"top_k": 3}, {"top_p": 0.9}, {"top_k": 600, "top_p": 0.7}, {"temperature": 0.0}, {"min_p": 0.2, "temperature": 0.5}, {"temperature": 3.0}):
        tok, logp = F.sample_filtered(z.cuda(), rng.cuda(), **kw)
        check_sample(z, rng, tok, logp, **kw)


def test_sampling_takes_numbers_of_tokens_beyond_32_bits():
    z, rng = torch.randn(4, 100, generator=torch.Generator().manual_seed(0)), torch.arange(4, dtype=torch.int32)
    k = torch.tensor([2**32 + 1, 2**31 + 1, -2**32 + 1, 3], dtype=torch.int64)
    tok, logp = F.sample_filtered(z.cuda(), rng.cuda(), top_k=k.cuda())
    check_sample(z, rng, tok, logp, top_k=k)
    for dtype in (torch.uint8, torch.int16, torch.int32, torch.int64):
        few = torch.tensor([1, 0, 50, 3], dtype=dtype)
        tok, logp = F.sample_filtered(z.cuda(), rng.cuda(), top_k=few.cuda())
        check_sample(z, rng, tok, logp, top_k=few)

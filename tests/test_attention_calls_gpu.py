"""Calls of the attention operators that the documentation allows and the other tests leave out: whole waves of
row tiles, wrong lengths into filled outputs, values at the ends of the 16-bit weights' range, far positions."""
import math

import pytest
import torch

import attention_ref as R
from airllm_b200 import AmoeError, attention, moe
from test_attention_gpu import (BF16, E4M3, F16, F32, PREFILLS, SPLITS, filled, gen, i32, on_gpu, randn, starts,
                                table_for)

pytestmark = pytest.mark.gpu


# ---- prefill -----------------------------------------------------------------------------------
@pytest.mark.parametrize("n,before,heads,kv,d", [(296, 300, 128, 1, 128), (444, 300, 128, 1, 64), (1184, 300, 32, 8, 128),
                                                (1776, 300, 64, 8, 64)])
def test_prefill_of_whole_waves(cuda_device, n, before, heads, kv, d):
    """Row tiles that fill the GPU's CTAs exactly leave none whose keys could be split."""
    g = gen(n)
    q, k, v = randn(g, n, heads, d, dtype=BF16), randn(g, n + before, kv, d, dtype=BF16), randn(g, n + before, kv, d, dtype=BF16)
    out = attention.prefill(q.cuda(), k.cuda(), v.cuda(), starts([n]).cuda(), starts([n + before]).cuda())
    some = [0, heads // kv, heads - 1]  # the definition takes long: some heads
    for h in some:
        one = h * kv // heads
        want, bound = R.attention(q[:, h:h + 1], k[:, one:one + 1], v[:, one:one + 1])
        R.close(out[:, h:h + 1], want, bound)
    assert torch.isfinite(out).all()


# ---- wrong lengths -----------------------------------------------------------------------------
@pytest.mark.parametrize("kind,out", [(BF16, BF16), (E4M3, F32)])
def test_read_of_wrong_lengths_gives_zeros(cuda_device, kind, out):
    """Rows below cu[seqs] whose start or first position is wrong are zeros, not what the output held; the others are read."""
    g = gen(61)
    kv, d, page = 3, 64, 16
    table, pool = table_for(g, [40, 40], page)
    pages = filled(g, pool, kv, page, d, kind)
    cache = on_gpu(pages)
    held = [[R.rows_of(c, s, table[i], 0, 40).to(out) for c, s in pages] for i in range(2)]
    for cu, first, rows in [  # rows: (sequence, its position) of each output row, None: zeros
        ([0, 10, 14], [-1, 2], [None] * 10 + [(1, 2 + i) for i in range(4)]),
        ([0, 10, 14], [3, -(1 << 31)], [(0, 3 + i) for i in range(10)] + [None] * 4),
        ([3, 9, 9], [0, 0], [None] * 3 + [(0, i) for i in range(6)]),
        ([-2, 4, 6], [0, 0], [None] * 4 + [(1, 0), (1, 1)]),
    ]:
        k = torch.full((20, kv, d), 7.0, dtype=out, device="cuda")
        v = torch.full((20, kv, d), 7.0, dtype=out, device="cuda")
        cache.read(table.cuda(), i32(cu).cuda(), 20, first=i32(first).cuda(), k_out=k, v_out=v)
        with pytest.raises(AmoeError, match="lengths"):
            cache.check()
        for got, which in ((k.cpu(), 0), (v.cpu(), 1)):
            for t, at in enumerate(rows):
                want = torch.zeros(kv, d, dtype=out) if at is None else held[at[0]][which][at[1]]
                assert torch.equal(got[t], want), (cu, first, t)
            assert (got[len(rows):] == 7).all()


def test_starts_that_decrease_or_pass_the_rows_are_reported(cuda_device):
    g = gen(62)
    kv, d, page, n = 2, 64, 16, 6
    cache = attention.KVCache(8, page, kv, d, dtype=F16)
    table = i32([[0, 1], [2, 3], [4, 5]]).cuda()
    rows = randn(g, n, kv, d, dtype=F16).cuda()
    zero = i32([0, 0, 0]).cuda()
    for cu in ([0, 2, 4, 7], [0, 2, 4, 2 ** 31 - 1], [0, 5, 3, 3], [0, 5, 2, 6], [0, 2, 9, 6], [0, -3, 4, 6]):
        cache.append(rows, rows, table, zero, i32(cu).cuda())
        with pytest.raises(AmoeError, match="lengths"):
            cache.check()
        cache.read(table, i32(cu).cuda(), n)
        with pytest.raises(AmoeError, match="lengths"):
            cache.check()
    # the rows that were given are there all the same, and fewer rows than were given are no mistake
    cache.append(rows, rows, table, zero, i32([0, 2, 4, 9]).cuda())
    with pytest.raises(AmoeError, match="lengths"):
        cache.check()
    k, v = cache.read(table, i32([0, 2, 4, 6]).cuda(), n)
    assert torch.equal(k, rows) and torch.equal(v, rows)
    cache.append(rows, rows, table, zero, i32([0, 2, 2, 5]).cuda())
    cache.read(table, i32([0, 0, 0, 0]).cuda(), n)
    cache.check()
    # the last of many sequences
    many = 3000
    wide = torch.zeros(many, 2, dtype=torch.int32).cuda()
    cu = torch.zeros(many + 1, dtype=torch.int32)
    for at, bad in ((many, n + 1), (many - 1, n), (many - 1, 1)):
        cu.zero_()
        cu[at] = bad
        cache.append(rows, rows, wide, torch.zeros(many, dtype=torch.int32).cuda(), cu.cuda())
        with pytest.raises(AmoeError, match="lengths"):
            cache.check()


# ---- weights of 16 bits ------------------------------------------------------------------------
def tail(n, kv, d, t):
    """(q row, k, v): one key of weight 1 with a zero value, then n - 1 keys of weight 2^-t with values of 1000."""
    q = torch.zeros(d, dtype=F16)
    k, v = torch.zeros(n, kv, d, dtype=F16), torch.full((n, kv, d), 1000.0, dtype=F16)
    q[0], k[0, :, 0], v[0] = 1.0, t * math.log(2), 0.0
    return q, k, v


# What f16 weights lose beside attention_ref's bound: below 2^-25 of the row's largest weight (here 1, and the
# denominator at least 1) half a step of the factor 2^11's subnormals, 2^-25 / 2^11, a key, times its value.
def tail_bound(n):
    return n * 2.0 ** -36 * 1000.0


TAILS = [10.0, 20.3, 23.4, 24.9, 25.1, 27.0]


@pytest.mark.parametrize("t", TAILS)
@pytest.mark.parametrize("kind,n,kv", [(F16, 131072, 1), (F16, 4000, 2), (E4M3, 131072, 1), (E4M3, 4000, 2)])
def test_decode_of_a_flat_tail(cuda_device, t, kind, n, kv):
    d, page = 64, 128
    q, k, v = tail(n, kv, d, t)
    pages = -(-n // page)
    cache = attention.KVCache(pages, page, kv, d, dtype=kind)
    table = torch.arange(pages, dtype=torch.int32).view(1, -1)
    cache.append(k.cuda(), v.cuda(), table.cuda(), i32([0]).cuda(), i32([0, n]).cuda())
    qs = q.expand(1, 4 * kv, d).contiguous()
    got = cache.decode(qs.cuda(), table.cuda(), i32([n]).cuda(), scale=1.0)
    held = (R.values(*R.e4m3(x.float())) for x in (k, v)) if kind == E4M3 else (k, v)
    want, bound = R.attention(qs, *held, scale=1.0)
    R.close(got, want, bound + tail_bound(n))


@pytest.mark.parametrize("t", TAILS)
@pytest.mark.parametrize("queries,n,heads,split", [(1, 131072, 2, True), (444, 6444, 128, False)])
def test_prefill_of_a_flat_tail(cuda_device, t, queries, n, heads, split):
    d = 64
    q, k, v = tail(n, 1, d, t)
    assert (moe.load_library().amoe_attn_prefill_workspace(d, 0, heads, 1, queries, n, 1) > 0) == split
    qs = q.expand(queries, heads, d).contiguous()
    got = attention.prefill(qs.cuda(), k.cuda(), v.cuda(), i32([0, queries]).cuda(), i32([0, n]).cuda(), scale=1.0)
    want, bound = R.attention(qs[:, :1], k, v, scale=1.0)
    for h in (0, heads - 1):
        R.close(got[:, h:h + 1], want, bound + tail_bound(n))


# ---- rotation ----------------------------------------------------------------------------------
@pytest.mark.parametrize("d,yarn", [(64, True), (128, True), (64, False), (128, False)])
def test_append_rotates_by_the_published_frequencies(cuda_device, d, yarn):
    """Frequencies computed here, not taken from the object under test."""
    g = gen(71)
    theta = 150000.0
    freq, conc = [1.0 / theta ** (2 * i / d) for i in range(d // 2)], 1.0
    if yarn:
        low, high = (d / 2 * math.log(4096 / (2 * math.pi * beta)) / math.log(theta) for beta in (32, 1))
        freq = [f * (1 - r + r / 32) for f, r in zip(freq, (min(max((i - low) / (high - low), 0), 1) for i in range(d // 2)))]
        conc = 1 + 0.1 * math.log(32)
        assert freq[0] == 1.0 and abs(freq[-1] * 32 * theta ** (1 - 2 / d) - 1) < 1e-12
    rope = attention.Rope.yarn(d, theta) if yarn else attention.Rope(d, theta, yarn=False)
    new, past, page = [3, 70, 1], [131000, 0, 4096], 128
    table, pool = table_for(g, [a + b for a, b in zip(new, past)], page)
    n = sum(new)
    x = randn(g, n, 6, d)
    cache = attention.KVCache(pool, page, 1, d, dtype=BF16)
    k_out = torch.empty(n, 1, d, device="cuda")
    q = cache.append(x[:, 4:5].cuda(), x[:, 5:].cuda(), table.cuda(), i32(past).cuda(), starts(new).cuda(), q=x[:, :4].cuda(),
                     rope=rope, k_out=k_out)
    cache.check()
    pos = torch.cat([torch.arange(p, p + m) for m, p in zip(new, past)])
    # A frequency is within 2^-48 of the one computed here, an angle within pos 2^-48, and an element turns by that times
    # its pair's length; both sides round to float32 once.
    far = x[:, :5].double().abs().amax() * math.sqrt(2) * conc * pos.max() * 2.0 ** -48
    want = R.rotated(x[:, :5], pos, freq, conc).double()
    got = torch.cat((q, k_out), 1).cpu().double()
    assert ((got - want).abs() <= 2.0 ** -23 * want.abs() + far).all()


# ---- values that are not finite ----------------------------------------------------------------
@pytest.mark.parametrize("share", [0.003, 0.1, 1.0])
@pytest.mark.parametrize("case", range(len(PREFILLS) + len(SPLITS)))
def test_prefill_of_odd_values(cuda_device, case, share):
    """Infinities and NaN strewn over V: an element is the formula's sum over the keys that its row sees, an infinity
    of either sign and NaN included, and no row has anything of a key that it does not see."""
    new, before, heads, kv, d, dtype, window, with_sinks = (PREFILLS + SPLITS)[case]
    g = gen(600 + case)
    keys = [a + b for a, b in zip(new, before)]
    n, m = sum(new), sum(keys)
    q, k, v = randn(g, n, heads, d, dtype=dtype, scale=0.5), randn(g, m, kv, d, dtype=dtype), randn(g, m, kv, d, dtype=dtype)
    odd = torch.tensor([math.inf, -math.inf, math.nan, math.inf], dtype=dtype)
    rows = torch.rand(m, kv, generator=g) < share
    hit = rows[..., None] & (torch.rand(m, kv, d, generator=g) < (0.03 if share < 1 else 1.0))
    v[hit] = odd[torch.randint(0, 4, (int(hit.sum()),), generator=g)]
    sinks = randn(g, heads) if with_sinks else None
    out = attention.prefill(q.cuda(), k.cuda(), v.cuda(), starts(new).cuda(), starts(keys).cuda(), window=window,
                            sinks=None if sinks is None else sinks.cuda()).cpu().double()
    some = sorted({0, heads // kv - 1, heads - 1})  # heads
    a = b = 0
    for x, y in zip(new, keys):
        for h in some:
            one = h * kv // heads
            want, bound = R.attention(q[a:a + x, h:h + 1], k[b:b + y, one:one + 1], v[b:b + y, one:one + 1],
                                      None if sinks is None else sinks[h:h + 1], window)
            got, fine = out[a:a + x, h:h + 1], torch.isfinite(want)
            assert torch.equal(torch.nan_to_num(got[~fine], 9.0, 7.0, 8.0), torch.nan_to_num(want[~fine], 9.0, 7.0, 8.0))
            assert torch.isfinite(got[fine]).all() and ((got - want).abs()[fine] <= bound[fine]).all()
        a, b = a + x, b + y


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 128)])
def test_an_infinity_does_not_make_prefill_slow(cuda_device, dtype, d):
    """Computing rows again, key by key, took 60 to 360 times as long."""
    n = 4096
    q, k, v = (torch.randn(n, h, d, device="cuda").to(dtype) for h in (64, 8, 8))
    cu = i32([0, n]).cuda()

    def ms(values):
        times = []
        for _ in range(5):
            a, b = torch.cuda.Event(True), torch.cuda.Event(True)
            a.record()
            attention.prefill(q, k, values, cu)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return sorted(times)[2]

    one, row = v.clone(), v.clone()
    one[5, 0, 3], row[n // 2] = math.inf, math.nan
    clean = ms(v)
    for values in (one, row, torch.full_like(v, math.nan)):
        assert ms(values) < 10 * clean  # 2.2 measured


@pytest.mark.parametrize("window", [1, 0])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 64), (BF16, 128)])
def test_prefill_scores_that_are_not_finite(cuda_device, dtype, d, bad, window):
    """A score of NaN or +inf makes its row NaN, whichever column of a tile its key stands in and although the row sees
    nothing else; a window of one key shows each column alone."""
    g = gen(64)
    n = 200
    q, k, v = randn(g, n, 2, d, dtype=dtype), randn(g, n, 1, d, dtype=dtype), randn(g, n, 1, d, dtype=dtype)
    q[:, :, 0] = 1.0
    first = 64
    k[first::2, 0, 0] = bad
    out = attention.prefill(q.cuda(), k.cuda(), v.cuda(), i32([0, n]).cuda(), window=window).cpu()
    hit = torch.arange(n) >= first
    if window:
        hit &= torch.arange(n) % 2 == 0
    assert torch.isnan(out[hit]).all() and torch.isfinite(out[~hit]).all()
    if window:
        assert torch.equal(out[~hit], v[~hit].expand(-1, 2, d))


# ---- far positions -----------------------------------------------------------------------------
@pytest.mark.parametrize("kind,d,page", [(BF16, 64, 4096), (E4M3, 64, 4096), (F16, 128, 1024), (BF16, 64, 16)])
@pytest.mark.parametrize("short", [0, 1, 17])
def test_decode_next_to_2_31(cuda_device, kind, d, page, short):
    """The last positions that a length can name, over a table that repeats a few pages: a window's keys, and not the slot
    behind the last."""
    g = gen(81)
    n, window, kv = 2 ** 31 - 1 - short, 70, 1
    pages = filled(g, 3, kv, page, d, kind)
    cache = on_gpu(pages)
    width = 2 ** 31 // page if page >= 1024 else 2 ** 27
    table = torch.zeros(1, width, dtype=torch.int32)
    table[0, -1], table[0, -2] = 2, 1
    last = torch.full((1,), n, dtype=torch.int32)
    q = randn(g, 1, 4, d, dtype=BF16 if kind == E4M3 else kind)
    got = cache.decode(q.cuda(), table.cuda(), last.cuda(), window=window, max_len=1000)
    cache.check()
    pos = torch.arange(n - window, n)
    ids, slot = table[0, pos // page].long(), pos % page
    k, v = (R.values(c.view(torch.uint8)[ids, :, slot].view(c.dtype) if s is not None else c[ids, :, slot],
                     None if s is None else s[ids, :, slot]) for c, s in pages)
    R.close(got, *R.attention(q, k, v))


def test_prefill_clamps_starts(cuda_device):
    """A first start below zero is the first row, one behind the rows given their end; the rows are written all the same."""
    g = gen(82)
    n = 60
    q, k, v = (randn(g, n, 4, 64, dtype=BF16).cuda() for _ in range(3))
    want = attention.prefill(q, k, v, i32([0, 25, n]).cuda())
    for cu_q, cu_k in (([-4, 25, n], [0, 25, n]), ([-(1 << 31), 25, 2 ** 31 - 1], [-7, 25, n + 9])):
        out = torch.full_like(q, 7.0)
        attention.prefill(q, k, v, i32(cu_q).cuda(), i32(cu_k).cuda(), out=out)
        assert torch.equal(out, want)


def test_refusals_raise_the_library_error(cuda_device):
    cache = attention.KVCache(4, 16, 2, 64)
    table, cu = i32([[0, 1]]).cuda(), i32([0, 5]).cuda()
    with pytest.raises(AmoeError, match="total"):
        cache.read(table, cu, -1)

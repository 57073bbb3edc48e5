"""The attention operators on the GPU against their float64 definitions (attention_ref.py):
rotation and quantised append, read back, packed prefill and paged decode, alone and as a
serving loop runs them."""
import math

import pytest
import torch

import attention_ref as R
import oracle
from airllm_b200 import AmoeError, attention, moe

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def starts(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)


def i32(v):
    return torch.tensor(v, dtype=torch.int32)


def table_for(g, lens, page, spare=2):
    """(table [seqs, n], pages): each sequence's pages, scattered over the pool."""
    per = [max(1, -(-n // page)) for n in lens]
    pool = sum(per) + spare
    order = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(per)), pool - 1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(per):
        table[i, :c] = order[at:at + c]
        at += c
    return table, pool


def filled(g, pool, heads, page, d, dtype):
    """Random pages (codes, scales) of a cache on the CPU."""
    out = []
    for _ in range(2):
        rows = randn(g, pool, heads, page, d)
        out += [R.e4m3(rows)] if dtype == E4M3 else [(rows.to(dtype), None)]
    return out


def on_gpu(pages):
    (k, ks), (v, vs) = pages
    return attention.KVCache.from_tensors(k.cuda(), v.cuda(), None if ks is None else ks.cuda(),
                                          None if vs is None else vs.cuda())


# ---- append and read ---------------------------------------------------------------------------
APPENDS = [  # new tokens, past, heads, kv_heads, d, page, source, cache, rotation
    ([1], [0], 8, 1, 64, 16, BF16, BF16, True),
    ([1, 1, 1], [700, 0, 131071], 64, 8, 64, 64, F16, E4M3, True),
    ([5, 0, 33, 1], [3, 9, 0, 64], 8, 8, 64, 8, F32, F16, True),
    ([40, 2], [0, 17], 32, 8, 128, 32, F32, E4M3, True),
    ([7, 300], [1, 2], 12, 1, 128, 128, BF16, E4M3, False),
    ([2, 2, 2, 2, 2], [0, 1, 2, 3, 4], 28, 4, 64, 1, F32, BF16, True),
    ([17], [4000], 5, 5, 128, 4096, F16, F16, True),
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_writes_the_definition(cuda_device, case):
    new, past, heads, kv, d, page, src, kind, turn = APPENDS[case]
    g = gen(case)
    table, pool = table_for(g, [a + b for a, b in zip(new, past)], page)
    pages = filled(g, pool, kv, page, d, kind)
    n = sum(new)
    qkv = randn(g, n + 2, heads + 2 * kv, d, dtype=src, scale=3.0)  # two rows behind the last sequence
    dev = qkv.cuda()
    q, k, v = dev[:, :heads], dev[:, heads:heads + kv], dev[:, heads + kv:]
    cache = on_gpu(pages)
    rope = attention.Rope(d, 150000.0) if turn else None
    out16 = F16 if src == F32 else src
    q_out = torch.full((n + 2, heads, d), 7.0, dtype=out16, device="cuda")
    k_out = torch.full((n + 2, kv, d), 7.0, dtype=F32, device="cuda")
    v_out = torch.full((n + 2, kv, d), 7.0, dtype=BF16, device="cuda")
    got = cache.append(k, v, table.cuda(), i32(past).cuda(), starts(new).cuda(), q=q, rope=rope, q_out=q_out,
                       k_out=k_out, v_out=v_out)
    assert got is q_out
    cache.check()

    pos = torch.cat([torch.arange(p, p + m) for m, p in zip(new, past)])
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
    freq, conc = (rope.frequencies, rope.concentration) if turn else ([0.0] * (d // 2), 1.0)
    qr = R.rotated(qkv[:n, :heads], pos, freq, conc)
    kr = R.rotated(qkv[:n, heads:heads + kv], pos, freq, conc)
    vr = qkv[:n, heads + kv:].float()
    assert torch.equal(q_out[:n].cpu(), qr.to(out16))
    assert torch.equal(k_out[:n].cpu(), kr)
    assert torch.equal(v_out[:n].cpu(), vr.to(BF16))
    for t in (q_out, k_out, v_out):
        assert (t[n:] == 7).all()
    ids, slot = table[seq, pos // page].long(), pos % page
    for rows, (codes, scale), at, sc in ((kr, pages[0], cache.k, cache.k_scale), (vr, pages[1], cache.v, cache.v_scale)):
        if kind == E4M3:
            c, s = R.e4m3(rows)
            codes.view(torch.uint8)[ids, :, slot] = c.view(torch.uint8)
            scale[ids, :, slot] = s
            assert torch.equal(sc.cpu(), scale)
            assert torch.equal(at.view(torch.uint8).cpu(), codes.view(torch.uint8))
        else:
            codes[ids, :, slot] = rows.to(kind)
            assert torch.equal(at.view(torch.int16).cpu(), codes.view(torch.int16))


def test_e4m3_rows_at_the_borders(cuda_device):
    d = 64
    x = torch.zeros(12, 1, d)
    x[1, 0, 5] = 448.0
    x[2, 0, 5] = 448.0 * (1 + 2.0 ** -23)  # the next float32 above
    x[3, 0, :] = torch.linspace(-448, 448, d)
    x[4, 0, 0], x[4, 0, 1], x[4, 0, 2] = 448.0, 17.0, 19.0  # ties between E4M3 neighbours 16, 18, 20
    x[5, 0, 63] = 1e-44
    x[6, 0, 3] = 3e38
    x[7, 0, 7] = math.inf
    x[8, 0, 60] = math.nan
    x[9, 0, 0], x[9, 0, 1] = 1.75, 2.0 ** -17  # the second is below half the smallest code
    x[10, 0, :] = -0.0
    x[11, 0, 0], x[11, 0, 1] = 1.75 * 2.0 ** -100, 1.76 * 2.0 ** -100
    cache = attention.KVCache(1, 16, 1, d, dtype=E4M3)
    cache.append(x.cuda(), x.cuda(), i32([[0]]).cuda(), i32([0]).cuda(), i32([0, 12]).cuda())
    codes, scale = R.e4m3(x)
    assert torch.equal(cache.k_scale[0, 0, :12].cpu(), scale[:, 0])
    assert scale[7, 0] == 255 and scale[8, 0] == 255
    ok = scale[:, 0] != 255
    for pages in (cache.k, cache.v):
        assert torch.equal(pages[0, 0, :12].view(torch.uint8).cpu()[ok], codes[:, 0].view(torch.uint8)[ok])
    k, v = cache.read(i32([[0]]).cuda(), i32([0, 12]).cuda(), 12, dtype=F32)
    want = R.values(codes, scale).float()
    assert torch.equal(torch.isnan(k.cpu()), torch.isnan(want)) and torch.isnan(k[7]).all() and torch.isnan(v[8]).all()
    assert torch.equal(k.cpu()[ok], want[ok]) and torch.equal(v.cpu()[ok], want[ok])


@pytest.mark.parametrize("kind,out,d,page,kv", [(E4M3, BF16, 64, 16, 8), (E4M3, F32, 128, 64, 1), (BF16, BF16, 128, 8, 3),
                                               (F16, F32, 64, 1, 2), (E4M3, F16, 64, 128, 5), (BF16, F16, 64, 32, 4)])
def test_read_gathers_the_sequences(cuda_device, kind, out, d, page, kv):
    g = gen(page)
    lens, first = [1, 0, 130, 37, 256], [0, 0, 3, 36, 0]
    table, pool = table_for(g, lens, page)
    pages = filled(g, pool, kv, page, d, kind)
    count = [n - f for n, f in zip(lens, first)]
    total = sum(count)
    k = torch.full((total + 3, kv, d), 7.0, dtype=out, device="cuda")
    wide = torch.full((total + 3, kv + 1, d + 16), 7.0, dtype=out, device="cuda")  # v_out: a strided view
    cache = on_gpu(pages)
    cache.read(table.cuda(), starts(count).cuda(), total + 3, first=i32(first).cuda(), k_out=k, v_out=wide[:, 1:, 16:])
    cache.check()
    for got, (codes, scale) in ((k, pages[0]), (wide[:, 1:, 16:], pages[1])):
        want = torch.cat([R.rows_of(codes, scale, table[i], f, c) for i, (f, c) in enumerate(zip(first, count))])
        assert torch.equal(got[:total].cpu(), want.to(out))
        assert (got[total:] == 7).all()
    assert (wide[:, 0] == 7).all() and (wide[:, :, :16] == 7).all()


def test_wrong_pages_and_lengths_are_skipped_and_reported(cuda_device):
    g = gen(3)
    kv, d, page = 2, 64, 16
    pages = filled(g, 4, kv, page, d, BF16)
    cache = on_gpu(pages)
    before = cache.k.clone()
    rows = randn(g, 6, kv, d, dtype=BF16).cuda()
    one = i32([0, 6]).cuda()
    bad = i32([[1, 4, -1]]).cuda()
    cache.append(rows, rows, bad, i32([14]).cuda(), one)  # positions 14, 15 in page 1; 16.. in page 4 of 4
    with pytest.raises(AmoeError, match="outside the cache"):
        cache.check()
    cache.check()  # the report is given once
    same = (cache.k == before).all(-1)  # rows: single bf16 elements of two random rows coincide now and then
    assert not same[1, :, 14:].any() and same[0].all() and same[2:].all() and same[1, :, :14].all()
    cache.append(rows, rows, bad, i32([45]).cuda(), one)  # positions 45..47 in page -1, 48.. beyond the table
    with pytest.raises(AmoeError, match="outside the cache, a position beyond"):
        cache.check()
    for past, cu in (([-1], one), ([0], i32([-2, 6]).cuda()), ([0], i32([3, 6]).cuda())):
        cache.append(rows, rows, bad, i32(past).cuda(), cu)
        with pytest.raises(AmoeError, match="lengths"):
            cache.check()
    k, v = cache.read(bad, i32([0, 60]).cuda(), 60)
    with pytest.raises(AmoeError, match="outside the cache, a position beyond"):
        cache.check()
    assert torch.equal(k[:16], cache.k[1].transpose(0, 1)) and (k[16:] == 0).all() and (v[16:] == 0).all()
    # decode sees the keys it can reach only
    q = randn(g, 1, 4, d, dtype=BF16).cuda()
    got = cache.decode(q, bad, i32([60]).cuda())
    with pytest.raises(AmoeError, match="outside the cache, a position beyond"):
        cache.check()
    held = [t[1].transpose(0, 1).cpu() for t in (cache.k, cache.v)]
    R.close(got, *R.attention(q.cpu(), *held))
    got = cache.decode(q, bad, i32([-5]).cuda())
    assert (got == 0).all()
    with pytest.raises(AmoeError, match="lengths"):
        cache.check()


# ---- prefill -----------------------------------------------------------------------------------
PREFILLS = [  # queries, keys before them, heads, kv_heads, d, type, window, sinks
    ([1], [0], 8, 1, 64, BF16, 0, False),
    ([1], [300], 64, 8, 64, F16, 0, True),
    ([129], [0], 16, 2, 64, BF16, 0, True),
    ([3, 0, 64, 200], [0, 5, 0, 70], 64, 8, 64, BF16, 0, True),
    ([500, 1, 17], [0, 0, 400], 8, 8, 64, F16, 0, False),
    ([260, 131], [0, 1], 32, 8, 128, BF16, 0, False),
    ([77, 300], [128, 0], 28, 4, 128, F16, 0, True),
    ([400, 33], [0, 500], 64, 8, 64, BF16, 128, True),
    ([300], [0], 12, 1, 64, F16, 1, False),
    ([90, 90], [0, 37], 40, 8, 128, BF16, 50, True),
    ([140], [0], 128, 1, 64, BF16, 0, False),
    ([70], [9], 256, 2, 128, F16, 17, True),
    ([33, 5], [0, 0], 15, 5, 64, BF16, 127, False),
    ([1000], [0], 2, 2, 64, F16, 0, True),
    ([1] * 40, list(range(40)), 8, 2, 64, BF16, 0, False),
]


@pytest.mark.parametrize("case", range(len(PREFILLS)))
def test_prefill_is_the_definition(cuda_device, case):
    new, before, heads, kv, d, dtype, window, with_sinks = PREFILLS[case]
    g = gen(100 + case)
    keys = [a + b for a, b in zip(new, before)]
    n, m = sum(new), sum(keys)
    q = randn(g, n + 5, heads, d, dtype=dtype, scale=2.0)
    kvs = randn(g, m + 4, 2 * kv, d, dtype=dtype)
    sinks = randn(g, heads, scale=2.0) if with_sinks else None
    out = torch.full((n + 5, heads, d), 7.0, dtype=dtype, device="cuda")
    dev = kvs.cuda()
    got = attention.prefill(q.cuda(), dev[:, :kv], dev[:, kv:], starts(new).cuda(), starts(keys).cuda(), window=window,
                            sinks=None if sinks is None else sinks.cuda(), out=out)
    assert got is out and (out[n:] == 7).all()
    a = b = 0
    for x, y in zip(new, keys):
        want, bound = R.attention(q[a:a + x], kvs[b:b + y, :kv], kvs[b:b + y, kv:], sinks, window)
        R.close(out[a:a + x], want, bound)
        a, b = a + x, b + y


def test_prefill_rows_that_see_nothing_are_zero(cuda_device):
    g = gen(9)
    q = randn(g, 70, 8, 64, dtype=BF16)
    k, v = randn(g, 20, 2, 64, dtype=BF16), randn(g, 20, 2, 64, dtype=BF16)
    # more queries than keys: the first 50 stand before every key; a sequence without keys; one without queries
    cu_q, cu_k = i32([0, 40, 70, 70]), i32([0, 10, 10, 20])
    for sinks in (None, torch.zeros(8)):
        out = attention.prefill(q.cuda(), k.cuda(), v.cuda(), cu_q.cuda(), cu_k.cuda(),
                                sinks=None if sinks is None else sinks.cuda()).cpu()
        assert (out[:30] == 0).all() and (out[40:] == 0).all()
        want, bound = R.attention(q[30:40], k[:10], v[:10], sinks)
        R.close(out[30:40], want, bound)
    # no keys at all
    empty = torch.empty(0, 2, 64, dtype=BF16, device="cuda")
    out = attention.prefill(q.cuda(), empty, empty, i32([0, 70]).cuda(), i32([0, 0]).cuda())
    assert (out == 0).all()
    # starts that lie: nothing out of range is read or written
    for cu_q, cu_k in (([0, 200], [0, 300]), ([5, 2], [0, 20]), ([-4, 30], [-7, 9]), ([0, 70], [20, 10])):
        attention.prefill(q.cuda(), k.cuda(), v.cuda(), i32(cu_q).cuda(), i32(cu_k).cuda())
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype,d,window", [(BF16, 64, 0), (F16, 128, 0), (BF16, 64, 40), (F16, 64, 128)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_prefill_masked_keys_do_not_count(cuda_device, dtype, d, window, bad):
    """A NaN or infinity in V or K reaches the rows that see it and no other, within its own
    sequence, across the border of two sequences and behind the last key."""
    g = gen(11)
    new = [150, 70]
    q = randn(g, 220, 8, d, dtype=dtype)
    k, v = randn(g, 230, 2, d, dtype=dtype), randn(g, 230, 2, d, dtype=dtype)
    v[100, 0, 3] = bad
    v[147, 1, d - 1] = bad
    v[200] = bad
    v[220:] = bad
    k[219] = bad
    k[220:] = bad
    out = attention.prefill(q.cuda(), k.cuda(), v.cuda(), starts(new).cuda(), window=window).cpu()
    a = 0
    for n in new:
        kk, vv = k[a:a + n], v[a:a + n]
        clean = torch.isfinite(kk).all(-1).all(-1)
        last = n if bool(clean.all()) else int((~clean).nonzero()[0])  # rows from a bad key on are its business
        want, bound = R.attention(q[a:a + last], kk[:last], vv[:last], None, window)
        got = out[a:a + last].double()
        fine = torch.isfinite(want)
        assert torch.isfinite(got[fine]).all() and not torch.isfinite(got[~fine]).any()
        assert ((got - want).abs()[fine] <= bound[fine]).all()
        a += n


def test_prefill_far_scores_and_sinks(cuda_device):
    """Scores of some hundreds, growing and falling along the keys: the running maximum moves by
    far more than the accumulators could hold without it."""
    g = gen(12)
    for sign in (1.0, -1.0):
        q = torch.ones(300, 4, 64, dtype=F16)
        k = (torch.linspace(-6, 6, 300)[:, None, None] * sign).expand(300, 1, 64).to(F16).contiguous()
        v = randn(g, 300, 1, 64, dtype=F16)
        sinks = torch.tensor([-1e4, 0.0, 40.0, -math.inf])
        out = attention.prefill(q.cuda(), k.cuda(), v.cuda(), i32([0, 300]).cuda(), sinks=sinks.cuda(), scale=0.9)
        want, bound = R.attention(q, k, v, sinks, scale=0.9)
        R.close(out, want, bound)


# ---- decode ------------------------------------------------------------------------------------
DECODES = [  # lengths, heads, kv_heads, d, page, query, cache, window, sinks
    ([1], 8, 1, 64, 16, BF16, BF16, 0, False),
    ([1000], 64, 8, 64, 64, BF16, BF16, 0, True),
    ([0, 1, 2, 15, 16, 17, 63, 64, 65], 64, 8, 64, 16, F16, F16, 0, True),
    ([31, 32, 33, 500], 16, 16, 64, 8, F16, E4M3, 0, False),
    ([777, 0, 128, 129], 64, 8, 64, 32, BF16, E4M3, 128, True),
    ([5000, 3], 32, 8, 128, 64, BF16, BF16, 0, False),
    ([4001, 40], 28, 4, 128, 128, F16, E4M3, 0, True),
    ([300, 2000], 12, 1, 128, 1, BF16, E4M3, 0, False),
    ([900], 128, 1, 64, 64, F16, F16, 1, True),
    ([257, 1023, 4097], 40, 8, 64, 4096, F16, E4M3, 1000, False),
    ([700] * 20, 34, 2, 128, 16, BF16, BF16, 0, True),
    ([12345], 5, 5, 64, 2, F16, F16, 3000, False),
    ([60000], 8, 8, 64, 64, BF16, E4M3, 0, True),
]


@pytest.mark.parametrize("case", range(len(DECODES)))
def test_decode_is_the_definition(cuda_device, case):
    lens, heads, kv, d, page, qt, kind, window, with_sinks = DECODES[case]
    g = gen(200 + case)
    table, pool = table_for(g, lens, page)
    pages = filled(g, pool, kv, page, d, kind)
    q = randn(g, len(lens), heads, 2, d, dtype=qt, scale=2.0)  # a strided view: every second row
    sinks = randn(g, heads, scale=2.0) if with_sinks else None
    cache = on_gpu(pages)
    dev = None if sinks is None else sinks.cuda()
    outs = [cache.decode(q.cuda()[:, :, 1], table.cuda(), i32(lens).cuda(), window=window, sinks=dev, max_len=most)
            for most in (max(lens), 0, 1)]
    cache.check()
    for i, n in enumerate(lens):
        k, v = (R.rows_of(c, s, table[i], 0, n) for c, s in pages)
        want, bound = R.attention(q[i:i + 1, :, 1], k, v, sinks, window)
        if n == 0:
            want, bound = torch.zeros(1, heads, d, dtype=torch.float64), torch.zeros(1, heads, d, dtype=torch.float64)
        for out in outs:
            R.close(out[i:i + 1], want, bound)


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_decode_ignores_what_lies_outside_the_sequence(cuda_device, kind):
    """NaN in the slots behind the last token and before the window, in pages and scales."""
    g = gen(21)
    lens, window, d, page = [70, 9], 40, 64, 16
    table, pool = table_for(g, lens, page)
    pages = filled(g, pool, 2, page, d, kind)
    q = randn(g, 2, 16, d, dtype=BF16)
    clean = on_gpu(pages).decode(q.cuda(), table.cuda(), i32(lens).cuda(), window=window)
    cache = on_gpu(pages)
    keep = torch.zeros(pool, 2, page, dtype=torch.bool)
    for i, n in enumerate(lens):
        pos = torch.arange(max(0, n - window), n)
        keep[table[i, pos // page].long(), :, pos % page] = True
    drop = (~keep).cuda()
    for t in (cache.k, cache.v):
        t.view(torch.uint8)[drop] = 0x7f if kind == E4M3 else 0xff
    if kind == E4M3:
        cache.k_scale[drop] = 255
        cache.v_scale[drop] = 255
    got = cache.decode(q.cuda(), table.cuda(), i32(lens).cuda(), window=window)
    assert torch.isfinite(got).all()
    assert torch.equal(got, clean)
    # inside the sequence they count
    cache.v.view(torch.uint8)[:] = 0x7f if kind == E4M3 else 0xff
    if kind == E4M3:
        cache.v_scale[:] = 255
    assert torch.isnan(cache.decode(q.cuda(), table.cuda(), i32(lens).cuda(), window=window)).all()


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_decode_with_far_sinks(cuda_device, kind):
    g = gen(24)
    lens = [0, 3, 900]
    table, pool = table_for(g, lens, 16)
    pages = filled(g, pool, 2, 16, 64, kind)
    q = randn(g, 3, 8, 64, dtype=BF16)
    sinks = torch.tensor([-1e4, 1e4, -300.0, 300.0, 0.0, -math.inf, 60.0, -60.0])
    got = on_gpu(pages).decode(q.cuda(), table.cuda(), i32(lens).cuda(), sinks=sinks.cuda())
    assert (got[0] == 0).all()
    for i in (1, 2):
        R.close(got[i:i + 1], *R.attention(q[i:i + 1], *(R.rows_of(c, s, table[i], 0, lens[i]) for c, s in pages), sinks))


def test_decode_over_scales_far_apart(cuda_device):
    """E4M3 rows whose scales span the whole exponent range, zero rows among them."""
    g = gen(22)
    n, d, page = 200, 64, 64
    rows = randn(g, n, 1, d)
    rows_v = randn(g, n, 1, d) * torch.exp2(torch.randint(-30, 10, (n, 1, 1), generator=g).float())
    rows_v[::7] = 0
    cache = attention.KVCache(4, page, 1, d, dtype=E4M3)
    table = i32([[2, 0, 3, 1]])
    cache.append(rows.cuda(), rows_v.cuda(), table.cuda(), i32([0]).cuda(), i32([0, n]).cuda())
    q = randn(g, 1, 8, d, dtype=F16)
    got = cache.decode(q.cuda(), table.cuda(), i32([n]).cuda())
    k, v = (R.values(*R.e4m3(r)) for r in (rows, rows_v))
    R.close(got, *R.attention(q, k, v))
    # every value zero, or smaller than the output type holds
    rows_v[:] = 0
    cache.append(rows.cuda(), rows_v.cuda(), table.cuda(), i32([0]).cuda(), i32([0, n]).cuda())
    assert (cache.decode(q.cuda(), table.cuda(), i32([n]).cuda()) == 0).all()


def test_a_page_far_into_a_large_cache(cuda_device):
    """Byte offsets beyond 32 bits: pages behind the 4 GiB mark."""
    kv, d, page = 8, 64, 128
    pages = (1 << 32) // (kv * page * d * 2) + 40
    cache = attention.KVCache(pages, page, kv, d, dtype=BF16)
    g = gen(23)
    n = 300
    table = i32([[pages - 1, 3, pages - 17]])
    k, v = randn(g, n, kv, d, dtype=BF16), randn(g, n, kv, d, dtype=BF16)
    cache.append(k.cuda(), v.cuda(), table.cuda(), i32([0]).cuda(), i32([0, n]).cuda())
    rk, rv = cache.read(table.cuda(), i32([0, n]).cuda(), n)
    assert torch.equal(rk.cpu(), k) and torch.equal(rv.cpu(), v)
    q = randn(g, 1, 64, d, dtype=BF16)
    R.close(cache.decode(q.cuda(), table.cuda(), i32([n]).cuda()), *R.attention(q, k, v))
    cache.check()


# ---- together ----------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,window", [(F16, 0), (F16, 128), (E4M3, 128), (BF16, 0)])
def test_a_serving_loop_against_the_oracle(cuda_device, kind, window):
    """Two prompts prefilled together, a second chunk of one over what the cache gives back, then
    decode steps: rows equal to the oracle's causal attention over the rotated keys that the cache holds."""
    heads, kv, d, page = 16, 2, 64, 16
    g = gen(31)
    dtype = BF16 if kind == BF16 else F16
    rope = attention.Rope(d, 150000.0)
    cache = attention.KVCache(40, page, kv, d, dtype=kind)
    table = torch.randperm(40, generator=g).to(torch.int32).view(2, 20).cuda()
    sinks = randn(g, heads)
    length = [0, 0]
    rot_q = [[], []]

    def step(new):
        n = sum(new)
        x = randn(g, n, heads + 2 * kv, d, scale=1.5)
        dev = x.cuda()
        cu, past = starts(new).cuda(), i32(length).cuda()
        k_out = torch.empty(n, kv, d, dtype=dtype, device="cuda")
        q = cache.append(dev[:, heads:heads + kv], dev[:, heads + kv:], table, past, cu, q=dev[:, :heads], rope=rope,
                         q_type=dtype, k_out=k_out)
        for i in range(2):
            length[i] += new[i]
        total = [length[i] if new[i] else 0 for i in range(2)]
        if new == [1, 1]:
            out = cache.decode(q, table, i32(length).cuda(), window=window, sinks=sinks.cuda())
        else:
            k, v = cache.read(table, starts(total).cuda(), sum(total), dtype=dtype)
            out = attention.prefill(q, k, v, cu, starts(total).cuda(), window=window, sinks=sinks.cuda())
        cache.check()
        # the oracle over the cache's own values
        a = 0
        for i in range(2):
            if not new[i]:
                continue
            got, qq = out[a:a + new[i]], q[a:a + new[i]].cpu()
            rows = [R.rows_of(p.cpu(), None if s is None else s.cpu(), table[i].cpu(), 0, length[i])
                    for p, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
            held = oracle.KVCache(kv, d, length[i])
            held.append(rows[0].float().numpy().ravel(), rows[1].float().numpy().ravel(), length[i])
            ref = oracle.causal_attention(qq.float().numpy().ravel(), heads, held, sinks=sinks.numpy(), window=window)
            _, bound = R.attention(qq, rows[0], rows[1], sinks, window)
            R.close(got, torch.from_numpy(ref).double().view(got.shape), bound)
            a += new[i]

    step([70, 33])
    step([0, 90])
    for _ in range(3):
        step([1, 1])


def test_calls_are_captured_and_replayed(cuda_device):
    g = gen(41)
    heads, kv, d, page = 64, 8, 64, 16
    cache = attention.KVCache(64, page, kv, d, dtype=E4M3)
    table = torch.arange(64, dtype=torch.int32).view(2, 32).cuda()
    rope = attention.Rope(d)
    qkv = randn(g, 2, heads + 2 * kv, d, dtype=BF16).cuda()
    length, cu = i32([100, 7]).cuda(), i32([0, 1, 2]).cuda()

    def step():
        q = cache.append(qkv[:, heads:heads + kv], qkv[:, heads + kv:], table, length, cu, q=qkv[:, :heads], rope=rope)
        return cache.decode(q, table, length + 1, window=128)

    def chunk():
        k, v = cache.read(table, i32_cu, 109, dtype=BF16)
        return attention.prefill(qkv[:, :heads], k, v, cu, i32_cu)

    i32_cu = i32([0, 101, 109]).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), chunk()
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(other):
        out2 = chunk()
    for i in range(3):
        qkv.copy_(randn(g, 2, heads + 2 * kv, d, dtype=BF16))
        length.copy_(i32([100 + i, 7 + i]))
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step()) and torch.equal(out2, chunk())
    cache.check()


def test_streams_and_the_current_device(cuda_device):
    g = gen(42)
    q = randn(g, 200, 8, 64, dtype=BF16).cuda()
    k, v = randn(g, 200, 2, 64, dtype=BF16).cuda(), randn(g, 200, 2, 64, dtype=BF16).cuda()
    cu = i32([0, 200]).cuda()
    want = attention.prefill(q, k, v, cu)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        inside = attention.prefill(q, k, v, cu)
    given = attention.prefill(q, k, v, cu, stream=side)
    raw = attention.prefill(q, k, v, cu, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(inside, want) and torch.equal(given, want) and torch.equal(raw, want)
    assert torch.cuda.current_device() == 0
    # two decode calls at once on two streams share nothing
    cache = attention.KVCache(600, 64, 2, 64)
    cache.k.normal_(), cache.v.normal_()
    table = torch.randperm(600, device="cuda").to(torch.int32).view(2, 300)
    lens = i32([19000, 18000]).cuda()
    qs = [randn(g, 2, 16, 64, dtype=BF16).cuda() for _ in range(2)]
    alone = [cache.decode(x, table, lens) for x in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        both = [cache.decode(x, table, lens, stream=s) for x, s in zip(qs, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, both))


def test_python_refusals(cuda_device):
    cache = attention.KVCache(4, 16, 2, 64)
    t = torch.zeros(5, 2, 64, dtype=BF16, device="cuda")
    table, cu, one = i32([[0, 1]]).cuda(), i32([0, 5]).cuda(), i32([0]).cuda()
    for call, word in [
        (lambda: cache.append(t[:, :1], t, table, one, cu), "heads"),
        (lambda: cache.append(t, t[:4], table, one, cu), "must be"),
        (lambda: cache.append(t.cpu(), t, table, one, cu), "cpu"),
        (lambda: cache.append(t.double(), t, table, one, cu), "type"),
        (lambda: cache.append(t.half(), t, table, one, cu), "type"),
        (lambda: cache.append(t, t, table.long(), one, cu), "page_table"),
        (lambda: cache.append(t, t, table, one.long(), cu), "past"),
        (lambda: cache.append(t, t, table, one, i32([0, 1, 5]).cuda()), "cu"),
        (lambda: cache.append(t, t, table, one, cu, q_out=t), "without q"),
        (lambda: cache.append(t, t, table, one, cu, q=t, q_out=t[:1].expand(5, 2, 64)), "overlap"),
        (lambda: cache.append(t, t, table, one, cu, rope=attention.Rope(128)), "rope"),
        (lambda: cache.append(t.transpose(1, 2).contiguous().transpose(1, 2), t, table, one, cu), "adjacent"),
        (lambda: cache.read(table, cu, 5, k_out=t[:1].expand(5, 2, 64)), "overlap"),
        (lambda: cache.decode(t, table, one), "must be"),
        (lambda: cache.decode(t[:1].half(), table, one), "types"),
        (lambda: cache.decode(t[:1], table, one, sinks=torch.zeros(3, device="cuda")), "sinks"),
        (lambda: cache.decode(t[:1], table, one, window=-1), "window"),
        (lambda: cache.decode(t[:1], table, one, scale=0.0), "scale"),
        (lambda: attention.prefill(t.float(), t, t, cu), "F16 or BF16|type"),
        (lambda: attention.prefill(t, t, t[:4], cu), "must be"),
        (lambda: attention.prefill(t, t, t, cu.cpu()), "cpu"),
        (lambda: attention.prefill(torch.zeros(5, 2, 96, dtype=BF16, device="cuda"), t, t, cu), "must be|head_dim"),
        (lambda: attention.prefill(t, t, t, cu, sinks=torch.zeros(2, device="cuda").half()), "sinks"),
        (lambda: attention.KVCache(4, 24, 2, 64).read(table, cu, 5), "power of two"),
        (lambda: attention.KVCache(0, 16, 2, 64), "shape"),
        (lambda: attention.KVCache(4, 16, 2, 64, dtype=torch.float32), "cache of"),
        (lambda: attention.KVCache.from_tensors(cache.k, cache.v, cache.status, None), "E4M3"),
    ]:
        with pytest.raises(AmoeError, match=word):
            call()
    # nothing to do
    none = torch.empty(0, 2, 64, dtype=BF16, device="cuda")
    assert cache.append(none, none, table, one, i32([0, 0]).cuda()) is None
    assert attention.prefill(none, none, none, i32([0, 0]).cuda()).shape == (0, 2, 64)
    assert cache.read(table, i32([0, 0]).cuda(), 0)[0].shape == (0, 2, 64)
    cache.check()


# ---- layouts, counts and values at the edges -----------------------------------------------------
def test_many_sequences(cuda_device):
    """More sequences than a warp looks at at once, empty ones among them, for each operator."""
    g = gen(51)
    n, heads, kv, d, page = 150, 8, 2, 64, 8
    new = [int(x) for x in torch.randint(0, 4, (n,), generator=g)]
    past = [int(x) for x in torch.randint(0, 20, (n,), generator=g)]
    lens = [a + b for a, b in zip(new, past)]
    table, pool = table_for(g, lens, page)
    pages = filled(g, pool, kv, page, d, F16)
    total = sum(new)
    x = randn(g, total, heads + 2 * kv, d, dtype=F16)
    dev, cache = x.cuda(), on_gpu(pages)
    cache.append(dev[:, heads:heads + kv], dev[:, heads + kv:], table.cuda(), i32(past).cuda(), starts(new).cuda())
    k, v = cache.read(table.cuda(), starts(lens).cuda(), sum(lens))
    out = attention.prefill(dev[:, :heads], k, v, starts(new).cuda(), starts(lens).cuda())
    one = torch.randn(n, heads, d, generator=g).half()
    dec = cache.decode(one.cuda(), table.cuda(), i32(lens).cuda())
    cache.check()
    a = b = 0
    for i in range(n):
        held = [R.rows_of(c, s, table[i], 0, past[i]).half() for c, s in pages]
        kk = torch.cat((held[0], x[a:a + new[i], heads:heads + kv]))
        vv = torch.cat((held[1], x[a:a + new[i], heads + kv:]))
        assert torch.equal(k[b:b + lens[i]].cpu(), kk) and torch.equal(v[b:b + lens[i]].cpu(), vv)
        if new[i]:
            R.close(out[a:a + new[i]], *R.attention(x[a:a + new[i], :heads], kk, vv))
        if lens[i]:
            R.close(dec[i:i + 1], *R.attention(one[i:i + 1], kk, vv))
        else:
            assert (dec[i] == 0).all()
        a, b = a + new[i], b + lens[i]


def test_prefill_layouts(cuda_device):
    """Heads outermost, wide gaps between rows, one head of a shared buffer, and a key head that is a view of
    another: the result of the contiguous tensors, or a refusal."""
    g = gen(52)
    n, heads, kv, d = 150, 8, 4, 128
    q, k, v = randn(g, n, heads, d, dtype=BF16), randn(g, n, kv, d, dtype=BF16), randn(g, n, kv, d, dtype=BF16)
    cu = i32([0, 100, n]).cuda()
    want = attention.prefill(q.cuda(), k.cuda(), v.cuda(), cu)

    def outer(t):  # [heads, tokens, d] in memory
        return t.transpose(0, 1).contiguous().cuda().transpose(0, 1)

    def gaps(t):
        wide = torch.full((n, t.shape[1] + 3, d + 24), math.nan, dtype=BF16, device="cuda")
        wide[:, 1:-2, 8:8 + d] = t.cuda()
        return wide[:, 1:-2, 8:8 + d]

    out = torch.full((heads, n, d), 7.0, dtype=BF16, device="cuda").transpose(0, 1)
    for layout in (outer, gaps):
        assert torch.equal(attention.prefill(layout(q), layout(k), layout(v), cu), want)
    assert torch.equal(attention.prefill(outer(q), gaps(k), v.cuda(), cu, out=out), want)
    # one key head for all queries, out of a buffer of several
    one = attention.prefill(q.cuda(), k.cuda()[:, 2:3], v.cuda()[:, 2:3], cu)
    R.close(one[:100], *R.attention(q[:100], k[:100, 2:3], v[:100, 2:3]))
    # a broadcast head
    try:
        got = attention.prefill(q.cuda(), k.cuda()[:, 1:2].expand(n, kv, d), v.cuda()[:, 1:2].expand(n, kv, d), cu)
    except AmoeError as e:
        assert "strides" in str(e)
    else:
        R.close(got[:100], *R.attention(q[:100], k[:100, 1:2].expand(100, kv, d), v[:100, 1:2].expand(100, kv, d)))
    # rows that do not start on 16 bytes
    odd = torch.zeros(n, heads, d + 4, dtype=BF16, device="cuda")[:, :, 4:]
    with pytest.raises(AmoeError, match="16 bytes"):
        attention.prefill(odd, k.cuda(), v.cuda(), cu)
    with pytest.raises(AmoeError, match="overlap"):
        attention.prefill(q.cuda(), k.cuda(), v.cuda(), cu, out=out[:, :1].expand(n, heads, d))


@pytest.mark.parametrize("d", [64, 128])
def test_prefill_nan_queries_and_keys(cuda_device, d):
    """A NaN in one query's row stays there; one in a key's row reaches every later query, whichever column of a tile
    the key stands in."""
    g = gen(53)
    n = 80
    q, k, v = randn(g, n, 2, d, dtype=F16), randn(g, n, 1, d, dtype=F16), randn(g, n, 1, d, dtype=F16)
    cu = i32([0, n]).cuda()
    clean = attention.prefill(q.cuda(), k.cuda(), v.cuda(), cu)
    bad = q.clone()
    bad[33, 1, 5] = math.nan
    got = attention.prefill(bad.cuda(), k.cuda(), v.cuda(), cu)
    assert torch.isnan(got[33, 1]).all()
    got[33, 1] = clean[33, 1]
    assert torch.equal(got, clean)
    for j in list(range(20)) + [63, 64, 79]:
        bad = k.clone()
        bad[j, 0, 3] = math.nan
        got = attention.prefill(q.cuda(), bad.cuda(), v.cuda(), cu)
        assert torch.isnan(got[j:]).all(), j
        assert torch.equal(got[:j], clean[:j]), j


def test_prefill_far_sinks_and_windows(cuda_device):
    g = gen(54)
    n = 200
    q, k, v = randn(g, n, 8, 64, dtype=BF16), randn(g, n, 2, 64, dtype=BF16), randn(g, n, 2, 64, dtype=BF16)
    cu = i32([0, n]).cuda()
    sinks = torch.tensor([-1e4, 1e4, -300.0, 300.0, 0.0, -math.inf, 60.0, -60.0])
    out = attention.prefill(q.cuda(), k.cuda(), v.cuda(), cu, sinks=sinks.cuda())
    R.close(out, *R.attention(q, k, v, sinks))
    sinks[3] = math.inf
    out = attention.prefill(q.cuda(), k.cuda(), v.cuda(), cu, sinks=sinks.cuda())
    assert torch.isnan(out[:, 3]).all() and torch.isfinite(out[:, :3]).all()
    plain = attention.prefill(q.cuda(), k.cuda(), v.cuda(), cu)
    for window in (n, n + 1, 2 ** 31 - 1):
        assert torch.equal(attention.prefill(q.cuda(), k.cuda(), v.cuda(), cu, window=window), plain)
    # more queries than keys under the longest window
    out = attention.prefill(q.cuda(), k[:50].cuda(), v[:50].cuda(), cu, i32([0, 50]).cuda(), window=2 ** 31 - 1)
    assert (out[:150] == 0).all()
    R.close(out[150:], *R.attention(q[150:], k[:50], v[:50]))


def test_a_long_decode_is_captured(cuda_device):
    """The form with a workspace and a second kernel, in a graph, and its refusal without the workspace."""
    g = gen(55)
    cache = attention.KVCache(700, 64, 1, 64, dtype=F16)
    cache.k.copy_(randn(g, 700, 1, 64, 64)), cache.v.copy_(randn(g, 700, 1, 64, 64))
    table = torch.randperm(700, generator=g).to(torch.int32).view(1, 700).cuda()
    q, length = randn(g, 1, 8, 64, dtype=F16).cuda(), i32([40001]).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.decode(q, table, length)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.decode(q, table, length)
    for n in (40001, 12, 44800):
        length.fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, cache.decode(q, table, length))
        k, v = (R.rows_of(t.cpu(), None, table[0].cpu(), 0, n) for t in (cache.k, cache.v))
        R.close(out, *R.attention(q.cpu(), k, v))
    cache.check()


SPLITS = [  # queries, keys before them, heads, kv_heads, d, type, window, sinks: few rows behind many keys
    ([1], [5000], 64, 8, 64, BF16, 0, True),
    ([17], [8191], 8, 1, 64, F16, 0, False),
    ([40], [3001], 8, 2, 128, BF16, 0, True),
    ([3, 0, 20], [9000, 100, 10], 12, 1, 64, BF16, 0, True),
    ([33], [7000], 10, 2, 128, F16, 2100, False),
    ([9], [20000], 128, 1, 64, F16, 0, True),
    # more tiles than CTAs that run at once (296, 444): those of the last wave are split
    ([300], [1500], 128, 1, 128, F16, 0, True),
    ([250, 210], [700, 1400], 128, 1, 64, BF16, 0, True),
    ([130, 0, 190], [1900, 100, 1500], 128, 1, 128, BF16, 1200, False),
]


@pytest.mark.parametrize("case", range(len(SPLITS)))
def test_prefill_split_over_the_keys(cuda_device, case):
    new, before, heads, kv, d, dtype, window, with_sinks = SPLITS[case]
    g = gen(300 + case)
    keys = [a + b for a, b in zip(new, before)]
    n, m = sum(new), sum(keys)
    assert moe.load_library().amoe_attn_prefill_workspace(d, window, heads, kv, n + 2, m, len(new)) > 0
    q = randn(g, n + 2, heads, d, dtype=dtype, scale=2.0)
    k, v = randn(g, m, kv, d, dtype=dtype), randn(g, m, kv, d, dtype=dtype)
    sinks = randn(g, heads, scale=2.0) if with_sinks else None
    # beside the plain values: an infinity that only the last query of the first sequence sees, NaN behind the first
    # sequence's keys where there is another
    bad = v.clone()
    if new[0] > 1:
        bad[keys[0] - 1, 0, 3] = math.inf
    if len(new) > 1:
        bad[keys[0]:keys[0] + keys[1]] = math.nan
    for values in (v, bad):
        out = torch.full((n + 2, heads, d), 7.0, dtype=dtype, device="cuda")
        attention.prefill(q.cuda(), k.cuda(), values.cuda(), starts(new).cuda(), starts(keys).cuda(), window=window,
                          sinks=None if sinks is None else sinks.cuda(), out=out)
        assert (out[n:] == 7).all()
        a = b = 0
        for x, y in zip(new, keys):
            want, bound = R.attention(q[a:a + x], k[b:b + y], values[b:b + y], sinks, window)
            got = out[a:a + x].double().cpu()
            fine = torch.isfinite(want)
            assert torch.equal(torch.isfinite(got), fine)
            assert ((got - want).abs()[fine] <= bound[fine]).all()
            a, b = a + x, b + y


def test_a_split_prefill_without_a_split_tile_is_waited_for(cuda_device):
    # the rows given allow a last wave of split tiles; the starts leave only whole ones, and what follows reads their rows
    g = gen(309)
    n, m = 280, 6000
    q = randn(g, 310, 128, 128, dtype=F16, scale=2.0).cuda()
    k, v = randn(g, m, 1, 128, dtype=F16).cuda(), randn(g, m, 1, 128, dtype=F16).cuda()
    assert moe.load_library().amoe_attn_prefill_workspace(128, 0, 128, 1, 310, m, 1) > 0
    want = attention.prefill(q[:n], k, v, i32([0, n]).cuda(), i32([0, m]).cuda())
    assert moe.load_library().amoe_attn_prefill_workspace(128, 0, 128, 1, n, m, 1) == 0
    cu_q, cu_k = i32([0, n]).cuda(), i32([0, m]).cuda()
    for _ in range(5):
        out = torch.full_like(q, 7.0)
        attention.prefill(q, k, v, cu_q, cu_k, out=out)
        copy = out.clone()
        assert torch.equal(copy[:n], want) and (copy[n:] == 7).all()


def test_a_split_prefill_is_captured_and_sees_nothing(cuda_device):
    g = gen(310)
    q = randn(g, 30, 8, 64, dtype=BF16).cuda()
    k, v = randn(g, 6000, 1, 64, dtype=BF16).cuda(), randn(g, 6000, 1, 64, dtype=BF16).cuda()
    cu_q, cu_k = i32([0, 30]).cuda(), i32([0, 6000]).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention.prefill(q, k, v, cu_q, cu_k)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention.prefill(q, k, v, cu_q, cu_k)
    for n in (6000, 0, 7, 3333):
        cu_k[1] = n
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        # queries that stand before every key see nothing
        seen = min(n, 30)
        assert (out[:30 - seen] == 0).all()
        if seen:
            R.close(out[30 - seen:], *R.attention(q[30 - seen:].cpu(), k[:n].cpu(), v[:n].cpu()))


def test_split_prefills_on_two_streams_and_strided_rows(cuda_device):
    g = gen(311)
    heads, kv, d, n, m = 16, 2, 64, 24, 7000
    calls = []
    for _ in range(2):
        fused = randn(g, n, (heads + 2) * d, dtype=BF16).cuda()  # queries beside something else
        q = fused[:, d:(heads + 1) * d].view(n, heads, d)
        both = randn(g, m, 2, kv, d, dtype=BF16).cuda()  # keys and values of a token side by side
        out = torch.full((n, heads, d + 8), 7.0, dtype=BF16, device="cuda")
        calls.append((q, both[:, 0], both[:, 1], out))
    cu_q, cu_k = i32([0, 9, n]).cuda(), i32([0, 4000, m]).cuda()
    assert moe.load_library().amoe_attn_prefill_workspace(d, 0, heads, kv, n, m, 2) > 0
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, (q, k, v, out) in zip(streams, calls):
            attention.prefill(q, k, v, cu_q, cu_k, out=out[:, :, :d], stream=stream)
    torch.cuda.synchronize()
    for q, k, v, out in calls:
        assert (out[:, :, d:] == 7).all()
        for a, b, x, y in ((0, 9, 0, 4000), (9, n, 4000, m)):
            R.close(out[a:b, :, :d], *R.attention(q[a:b].cpu(), k[x:y].cpu(), v[x:y].cpu()))


SHARES = [  # lengths of one call that the device shares the CTAs out by, heads, kv_heads, d, page, cache, window, sinks
    ([9000, 1, 0, 300, 8191, 77], 8, 1, 64, 64, BF16, 0, True),
    ([17, 12001], 8, 2, 128, 16, E4M3, 0, True),
    ([0, 0, 10000], 16, 1, 64, 128, F16, 0, False),
    ([9999, 20000, 8200], 8, 1, 64, 32, E4M3, 8500, False),
    ([8300] + [5] * 69, 16, 1, 64, 64, BF16, 0, True),
]


@pytest.mark.parametrize("case", range(len(SHARES)))
def test_decode_of_uneven_lengths(cuda_device, case):
    lens, heads, kv, d, page, kind, window, with_sinks = SHARES[case]
    g = gen(400 + case)
    table, pool = table_for(g, lens, page)
    pages = filled(g, pool, kv, page, d, kind)
    q = randn(g, len(lens), heads, d, dtype=BF16 if kind == E4M3 else kind, scale=2.0)
    sinks = randn(g, heads, scale=2.0) if with_sinks else None
    cache = on_gpu(pages)
    length, dq, dt = i32(lens).cuda(), q.cuda(), table.cuda()
    want = []
    for i, n in enumerate(lens):
        zero = torch.zeros(1, heads, d, dtype=torch.float64)
        want.append(R.attention(q[i:i + 1], *(R.rows_of(c, s, table[i], 0, n) for c, s in pages), sinks, window)
                    if n else (zero, zero))
    kw = dict(window=window, sinks=None if sinks is None else sinks.cuda())
    out = cache.decode(dq, dt, length, **kw)
    assert max(cache._workspace.values()) > 0
    cache.check()
    for i, w in enumerate(want):
        R.close(out[i:i + 1], *w)
    # captured; then other lengths in the same graph: all zero, one of them negative, one beyond the table
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.decode(dq, dt, length, **kw)
    graph.replay()
    for i, w in enumerate(want):
        R.close(out[i:i + 1], *w)
    length.zero_()
    graph.replay()
    assert (out == 0).all()
    cache.check()
    length[0] = -5
    graph.replay()
    assert (out == 0).all()
    with pytest.raises(AmoeError):
        cache.check()
    length[0] = 1 << 30
    graph.replay()
    with pytest.raises(AmoeError):
        cache.check()
    length.copy_(i32(lens))
    graph.replay()
    for i, w in enumerate(want):
        R.close(out[i:i + 1], *w)

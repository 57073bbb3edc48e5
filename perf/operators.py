"""The attention operators' measured cases: inputs, plain forms in torch and definitions in 64 bits.

Four operators over a paged key-value cache, with the GPT-OSS attention half's conventions (grouped
heads, YaRN, learned sinks, a sliding window on every other layer):

  append   rotate q and k at their positions, write k and v into the cache's pages (16 bits, or E4M3
           with one power-of-two scale for each token and head)
  read     gather a sequence's pages back into packed rows
  store    append into an E4M3 cache, then read the sequences back: what a chunk of a prompt does
  prefill  causal attention of packed prompts
  decode   attention of one new token a sequence over its pages

``own`` false: elementary torch operations.  ``own`` true: the calls of airllm_b200.attention.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
THETA = 150000.0  # GPT-OSS's rotary base


# ---- the cases ---------------------------------------------------------------------------------
def listed():
    gptoss = dict(heads=64, kv_heads=8, dim=64)  # GPT-OSS's heads: eight queries share a key head
    wide = dict(heads=32, kv_heads=8, dim=128)   # the 128-wide heads of Llama-shaped models
    return [
        # one token of one sequence into a 16-bit cache: a single user's decode step, latency only
        dict(name="append_one_token", op="append", seqs=1, tokens=1, past=700, cache="bf16", src="bf16", page=64, **gptoss),
        # a packed prompt batch straight from an f32 projection, four ragged sequences
        dict(name="append_prompts_f32", op="append", seqs=4, tokens=8192, past=0, cache="f16", src="f32", page=64, **gptoss),
        # one decode step of 64 users into an 8-bit cache, and the last few tokens read back (windowed layer)
        dict(name="store_step_64", op="store", seqs=64, tokens=64, past=127, cache="e4m3", src="bf16", page=16, **gptoss),
        # a chunk of long prompts into an 8-bit cache, and the whole context read back for its attention
        dict(name="store_chunk", op="store", seqs=5, tokens=6001, past=3500, cache="e4m3", src="f16", page=128, **wide),
        # a long context out of an 8-bit cache, as a prompt's next chunk needs it
        dict(name="read_long", op="read", seqs=2, tokens=50001, past=0, cache="e4m3", src="bf16", page=64, **gptoss),
        # a short prompt, latency only
        dict(name="prefill_short", op="prefill", seqs=1, tokens=48, past=0, src="bf16", window=0, sinks=True, **gptoss),
        # one long prompt on a full-attention layer
        dict(name="prefill_long", op="prefill", seqs=1, tokens=8192, past=0, src="bf16", window=0, sinks=True, **gptoss),
        # a ragged batch on a sliding-window layer
        dict(name="prefill_window", op="prefill", seqs=7, tokens=12001, past=0, src="f16", window=128, sinks=True, **gptoss),
        # chunks that continue a context, 128-wide heads, no sinks
        dict(name="prefill_chunk", op="prefill", seqs=3, tokens=1500, past=2777, src="bf16", window=0, sinks=False, **wide),
        # one user's token over a medium context: latency
        dict(name="decode_one", op="decode", seqs=1, length=1000, cache="bf16", src="bf16", page=64, window=0, sinks=True, **gptoss),
        # one user's token over a very long context: the split over the length
        dict(name="decode_long", op="decode", seqs=1, length=131072, cache="f16", src="f16", page=64, window=0, sinks=True, **gptoss),
        # a serving batch over an 8-bit cache
        dict(name="decode_batch", op="decode", seqs=48, length=8192, cache="e4m3", src="bf16", page=32, window=0, sinks=True, **gptoss),
    ]


def draw(rng):
    def span(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    heads, kv_heads = rng.choice([(64, 8), (64, 8), (32, 8), (40, 8), (28, 4), (16, 16), (12, 1)])
    case = dict(heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128]), seqs=span(1, 64))
    case["op"] = rng.choice(["append", "store", "read", "prefill", "prefill", "decode", "decode"])
    case["src"] = rng.choice(["f16", "bf16"])
    if case["op"] in ("append", "store", "read"):
        case["page"] = rng.choice([8, 16, 32, 64, 128])
        case["cache"] = case["src"] if case["op"] == "append" else rng.choice([case["src"], "e4m3"])
        case["tokens"] = max(case["seqs"], span(1, 8192))
        case["past"] = rng.choice([0, span(1, 500)])
        if case["op"] != "read" and rng.random() < 0.3:
            case["src"] = "f32"
            if case["cache"] != "e4m3":
                case["cache"] = rng.choice(["f16", "bf16"])
    elif case["op"] == "prefill":
        case["tokens"] = max(case["seqs"], span(1, 6000))
        case["past"] = rng.choice([0, 0, span(1, 1000)])
        case["window"] = rng.choice([0, 0, 128, span(1, 1000)])
        case["sinks"] = rng.random() < 0.5
    else:
        case["page"] = rng.choice([8, 16, 32, 64, 128])
        case["cache"] = rng.choice([case["src"], "e4m3"])
        case["length"] = span(1, max(2, min(60000, 300000 // case["seqs"])))
        case["window"] = rng.choice([0, 0, 128, span(1, 2000)])
        case["sinks"] = rng.random() < 0.5
    return case


def spread(case):
    """New tokens and context of each sequence: ragged, the same for every seed."""
    r = random.Random(case["seqs"] * 1000003 + case.get("tokens", case.get("length", 0)))
    n = case["seqs"]
    if case["op"] == "decode":  # lengths from half the named one up, the named one among them
        lens = [max(1, int(case["length"] * r.uniform(0.5, 1.0))) for _ in range(n)]
        lens[r.randrange(n)] = case["length"]
        return [1] * n, [x - 1 for x in lens]
    share = [r.uniform(0.2, 1.0) for _ in range(n)]
    new = [1 + int((case["tokens"] - n) * s / sum(share)) for s in share]
    new[r.randrange(n)] += case["tokens"] - sum(new)
    past = [int(case["past"] * r.uniform(0.5, 1.0)) for _ in range(n)]
    past[r.randrange(n)] = case["past"]
    return new, past


def read_back(case, new, past):
    """First position and number of the rows that a store or read gathers."""
    if case["op"] == "store" and case["tokens"] == case["seqs"]:  # decode steps read their window only
        first = [max(0, p + n - 128) for n, p in zip(new, past)]
    else:
        first = [0] * len(new)
    return first, [n + p - f for n, p, f in zip(new, past, first)]


def visible(new, past, window):
    """Pairs of query and key that the causal mask and the window leave."""
    total = 0
    for n, p in zip(new, past):
        if not window:
            total += n * p + n * (n + 1) // 2
        else:
            total += sum(min(window, p + i + 1) for i in range(n))
    return total


def work(case):
    new, past = spread(case)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    t, src = sum(new), BYTES[case["src"]]
    if case["op"] == "prefill":
        keys = sum(n + p for n, p in zip(new, past))
        return {"bytes": 2 * t * h * d * src + 2 * keys * g * d * src, "flops": 4 * h * d * visible(new, past, case["window"])}
    row = g * (d * BYTES[case["cache"]] + (1 if case["cache"] == "e4m3" else 0))  # one token's keys or values
    if case["op"] == "decode":
        seen = visible(new, past, case["window"])
        return {"bytes": 2 * seen * row + 2 * t * h * d * src, "flops": 4 * h * d * seen}
    out = {"bytes": 0, "flops": 0}
    if case["op"] != "read":  # rotation: two products and a sum an element
        out["bytes"] += t * (h + 2 * g) * d * src + t * h * d * 2 + 2 * t * row
        out["flops"] += 3 * t * (h + g) * d
    if case["op"] != "append":
        rows = sum(read_back(case, new, past)[1])
        out["bytes"] += 2 * rows * (row + g * d * 2)
        out["flops"] += 2 * rows * g * d
    return out


# ---- inputs ------------------------------------------------------------------------------------
def quantised(rows):
    """Rows of 32-bit values as E4M3 codes and the exponents of their scales (biased by 127): the smallest power of
    two that brings the row's largest value to 448 or less."""
    top = rows.abs().amax(-1)
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(top > 0, (e - 9 + (m > 0.875)).clamp(-127, 127), torch.zeros_like(e))
    codes = torch.ldexp(rows, -e.unsqueeze(-1)).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    new, past = spread(case)
    h, kv, d, n = case["heads"], case["kv_heads"], case["dim"], case["seqs"]
    src = TYPES[case["src"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=DEVICE) * scale

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEVICE)

    def starts(v):
        return ints([sum(v[:i]) for i in range(len(v) + 1)])

    s = {"op": case["op"], "new": new, "past_list": past, "heads": h, "kv_heads": kv, "dim": d, "seqs": n}
    total = sum(new)
    s["tokens"] = total
    s["most"] = max(a + b for a, b in zip(new, past))
    if case["op"] == "prefill":
        keys = sum(new) + sum(past)
        s["q"] = normal(total, h, d, scale=1.5).to(src)
        kvs = normal(keys, 2 * kv, d).to(src)  # keys and values side by side, as a fused projection leaves them
        s["k"], s["v"] = kvs[:, :kv], kvs[:, kv:]
        s["cu_q"], s["cu_k"] = starts(new), starts([a + b for a, b in zip(new, past)])
        s["most_q"], s["total_k"] = max(new), keys
    else:
        page = case["page"]
        per = [-(-(a + b) // page) for a, b in zip(new, past)]
        pool, width = sum(per) + 3, max(per)
        order = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32)
        table = torch.zeros((n, width), dtype=torch.int32, device=DEVICE)
        at = 0
        for i, c in enumerate(per):
            table[i, :c] = order[at:at + c]
            at += c
        s["table"], s["page"], s["cache_type"] = table, page, case["cache"]
        for name in ("k", "v"):
            rows = normal(pool, kv, page, d)
            if case["cache"] == "e4m3":
                codes, scale = quantised(rows)
                s[name + "_pages"], s[name + "_scale"] = codes, scale
            else:
                s[name + "_pages"], s[name + "_scale"] = rows.to(TYPES[case["cache"]]), None
            del rows
        s["past"] = ints(past)
        if case["op"] == "decode":
            s["q"] = normal(n, h, d, scale=1.5).to(src)
            s["length"] = s["past"] + 1
        else:
            first, count = read_back(case, new, past)
            s["first"], s["cu_read"], s["total_read"] = ints(first), starts(count), sum(count)
            s["out_type"] = TYPES[case["src"] if case["src"] != "f32" else "f16" if case["cache"] == "e4m3" else case["cache"]]
            if case["op"] != "read":
                qkv = normal(total, h + 2 * kv, d).to(src)
                s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
                s["cu"] = starts(new)
    if case["op"] in ("prefill", "decode"):
        s["window"] = case["window"]
        s["sinks"] = normal(h) if case["sinks"] else None
    if own and case["op"] != "prefill":
        from airllm_b200 import attention

        s["cache"] = attention.KVCache.from_tensors(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    if own and case["op"] in ("append", "store"):
        s["rope"] = attention.Rope(d, THETA, yarn=True)
    return s


# ---- one pass ----------------------------------------------------------------------------------
def run(s):
    if own:
        return run_own(s)
    if s["op"] == "prefill":
        return plain_prefill(s)
    if s["op"] == "decode":
        return plain_decode(s)
    out = {}
    if s["op"] != "read":
        out["q"] = plain_append(s)
    if s["op"] == "append":
        out["k_pages"], out["v_pages"] = s["k_pages"], s["v_pages"]
    else:
        out["k"], out["v"] = plain_read(s, s["k_pages"], s["k_scale"]), plain_read(s, s["v_pages"], s["v_scale"])
    return out


def run_own(s):
    if s["op"] == "prefill":
        from airllm_b200 import attention

        return attention.prefill(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], window=s["window"], sinks=s["sinks"])
    cache = s["cache"]
    if s["op"] == "decode":
        return cache.decode(s["q"], s["table"], s["length"], window=s["window"], sinks=s["sinks"], max_len=s["most"])
    out = {}
    if s["op"] != "read":
        out["q"] = cache.append(s["k"], s["v"], s["table"], s["past"], s["cu"], q=s["q"], rope=s["rope"], q_type=s["out_type"])
    if s["op"] == "append":
        out["k_pages"], out["v_pages"] = s["k_pages"], s["v_pages"]
    else:
        out["k"], out["v"] = cache.read(s["table"], s["cu_read"], s["total_read"], first=s["first"], dtype=s["out_type"])
    return out


def yarn(d, dev):
    """GPT-OSS's YaRN frequencies and concentration: factor 32 over an original context of 4096, beta 32 and 1."""
    i = torch.arange(d // 2, dtype=torch.float64, device=dev)
    base = THETA ** (-2.0 * i / d)
    low = max(0.0, math.floor(d * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(THETA))))
    high = min(d // 2 - 1.0, math.ceil(d * math.log(4096 / (2 * math.pi)) / (2 * math.log(THETA))))
    ramp = ((i - low) / (high - low)).clamp(0, 1)
    return base * (ramp + (1 - ramp) / 32), 1 + 0.1 * math.log(32)


def rotated(x, c, s):
    """Rows [tokens, heads, d] by angles [tokens, 1, d / 2], in 64 bits, rounded to 32."""
    a, b = x.double().chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1).float()


def owner(cu, total):
    """The sequence of each packed row and its place in it."""
    row = torch.arange(total, dtype=torch.int32, device=cu.device)
    seq = torch.searchsorted(cu[1:], row, right=True)
    return seq, row - cu[seq]


def place(s, seq, pos):
    return s["table"][seq, pos // s["page"]].long(), pos.long() % s["page"]


def plain_append(s):
    seq, i = owner(s["cu"], s["tokens"])
    pos = s["past"][seq] + i
    freq, conc = yarn(s["dim"], pos.device)
    angle = pos.double()[:, None, None] * freq
    c, sn = torch.cos(angle) * conc, torch.sin(angle) * conc
    page, slot = place(s, seq, pos)
    for name, rows in (("k", rotated(s["k"], c, sn)), ("v", s["v"].float())):
        if s["cache_type"] == "e4m3":
            codes, scale = quantised(rows)
            s[name + "_pages"].view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)
            s[name + "_scale"][page, :, slot] = scale
        else:
            s[name + "_pages"][page, :, slot] = rows.to(s[name + "_pages"].dtype)
    return rotated(s["q"], c, sn).to(s["out_type"])


def held(pages, scale, page, slot):
    """The values that cache rows stand for, in 32 bits: [..., kv_heads, d]."""
    if scale is None:
        return pages[page, :, slot].float()
    e = scale[page, :, slot].int() - 127
    return torch.ldexp(pages.view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn).float(), e.unsqueeze(-1))


def plain_read(s, pages, scale):
    seq, i = owner(s["cu_read"], s["total_read"])
    return held(pages, scale, *place(s, seq, s["first"][seq] + i)).to(s["out_type"])


def softmax_rows(score, seen, sinks):
    """exp(score - max) over the seen keys and their sum with the sink's term; a row that sees nothing sums to 1."""
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, sinks)
    top = top.masked_fill(top == float("-inf"), 0.0)
    e = torch.exp(score - top)
    total = e.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks - top)
    return e, total.masked_fill(total == 0, 1.0)


def plain_prefill(s):
    h, kv, d, n = s["heads"], s["kv_heads"], s["dim"], s["seqs"]
    dev = s["q"].device
    nq, nk = s["cu_q"].diff(), s["cu_k"].diff()
    iq = torch.arange(s["most_q"], device=dev)
    ik = torch.arange(s["most"], device=dev)
    # sequences padded to the longest, rows past a sequence's end read some other row and are masked or dropped
    rq = (s["cu_q"][:-1, None] + iq).clamp(max=s["tokens"] - 1).long()
    rk = (s["cu_k"][:-1, None] + ik).clamp(max=s["total_k"] - 1).long()
    q = s["q"][rq].float().view(n, -1, kv, h // kv, d).permute(0, 2, 3, 1, 4)  # [n, kv, group, queries, d]
    k = s["k"][rk].float().permute(0, 2, 3, 1).unsqueeze(2)                    # [n, kv, 1, d, keys]
    v = s["v"][rk].float().permute(0, 2, 1, 3).unsqueeze(2)                    # [n, kv, 1, keys, d]
    pos = (nk - nq)[:, None] + iq  # each query's position among its keys
    seen = (ik <= pos[:, :, None]) & (ik < nk[:, None, None])
    if s["window"]:
        seen &= ik > pos[:, :, None] - s["window"]
    sinks = None if s["sinks"] is None else s["sinks"].view(1, kv, h // kv, 1, 1)
    score = torch.matmul(q / math.sqrt(d), k)
    e, total = softmax_rows(score, seen[:, None, None], sinks)
    del score
    o = (torch.matmul(e, v) / total).permute(0, 3, 1, 2, 4).reshape(n, -1, h, d)
    seq, i = owner(s["cu_q"], s["tokens"])
    return o[seq, i.long()].to(s["q"].dtype)


def plain_decode(s):
    h, kv, d, n = s["heads"], s["kv_heads"], s["dim"], s["seqs"]
    ik = torch.arange(s["most"], device=s["q"].device)
    pos = torch.minimum(ik, s["length"][:, None] - 1)
    page, slot = place(s, torch.arange(n, device=ik.device)[:, None], pos)
    k = held(s["k_pages"], s["k_scale"], page, slot).permute(0, 2, 3, 1)  # [n, kv, d, keys]
    v = held(s["v_pages"], s["v_scale"], page, slot).permute(0, 2, 1, 3)
    seen = ik < s["length"][:, None]
    if s["window"]:
        seen &= ik >= s["length"][:, None] - s["window"]
    q = s["q"].float().view(n, kv, h // kv, d) / math.sqrt(d)
    sinks = None if s["sinks"] is None else s["sinks"].view(1, kv, h // kv, 1)
    e, total = softmax_rows(torch.matmul(q, k), seen[:, None, None], sinks)
    return (torch.matmul(e, v) / total).reshape(n, h, d).to(s["q"].dtype)


# ---- definitions in 64 bits --------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    new, past = s["new"], s["past_list"]
    if case["op"] == "prefill":
        out, a, b = [], 0, 0
        for n, p in zip(new, past):
            out.append(exact_attention(s, s["q"][a:a + n], s["k"][b:b + n + p], s["v"][b:b + n + p]))
            a, b = a + n, b + n + p
        return torch.cat(out)
    if case["op"] == "decode":
        out = []
        for i, p in enumerate(past):
            k, v = (exact_rows(s, name, i, 0, p + 1) for name in ("k", "v"))
            out.append(exact_attention(s, s["q"][i:i + 1], k, v))
        return torch.cat(out)
    out = {}
    if case["op"] != "read":
        out["q"] = exact_append(s)
    if case["op"] == "append":
        out["k_pages"], out["v_pages"] = s["k_pages"].double(), s["v_pages"].double()
    else:
        first, count = read_back(case, new, past)
        for name in ("k", "v"):
            out[name] = torch.cat([exact_rows(s, name, i, f, c) for i, (f, c) in enumerate(zip(first, count))])
    return out


def exact_rows(s, name, i, first, count):
    """`count` cached rows of sequence i from position `first`: [count, kv_heads, d]."""
    a, b = first // s["page"], -(-(first + count) // s["page"])
    ids = s["table"][i, a:b].long()
    rows = s[name + "_pages"].view(torch.uint8)[ids].view(s[name + "_pages"].dtype).double()
    if s[name + "_scale"] is not None:
        rows = rows * torch.exp2(s[name + "_scale"][ids].double() - 127)[..., None]
    rows = rows.permute(0, 2, 1, 3).reshape(-1, s["kv_heads"], s["dim"])
    return rows[first - a * s["page"]:][:count]


def exact_attention(s, q, k, v):
    """The last len(q) of len(k) tokens attend to what came before them."""
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    n, m, group = len(q), len(k), s["heads"] // s["kv_heads"]
    at = torch.arange(m - n, m, device=q.device)[:, None]
    key = torch.arange(m, device=q.device)[None]
    hidden = (key > at) if not s["window"] else (key > at) | (key <= at - s["window"])
    for head in range(s["heads"]):
        kk, vv = k[:, head // group].double(), v[:, head // group].double()
        score = (q[:, head].double() @ kk.T) * (1 / math.sqrt(s["dim"]))
        score[hidden] = -math.inf
        if s["sinks"] is not None:  # one more key, whose value is zero
            score = torch.cat((score, s["sinks"][head].double().expand(n, 1)), 1)
            vv = torch.cat((vv, torch.zeros_like(vv[:1])))
        out[:, head] = torch.softmax(score, 1) @ vv
    return out


def exact_append(s):
    """Writes the new rows where they belong, one sequence after another; the rotated queries."""
    d, kv, page = s["dim"], s["kv_heads"], s["page"]
    half = d // 2
    def corner(beta):
        return d * math.log(4096 / (beta * 2 * math.pi)) / (2 * math.log(THETA))
    low, high = max(0.0, math.floor(corner(32.0))), min(half - 1.0, math.ceil(corner(1.0)))
    freq = []
    for i in range(half):
        ramp = min(1.0, max(0.0, (i - low) / (high - low)))
        freq.append(THETA ** (-2.0 * i / d) * (ramp + (1.0 - ramp) / 32.0))
    freq = torch.tensor(freq, dtype=torch.float64, device=s["q"].device)
    conc = 1.0 + 0.1 * math.log(32.0)

    def turn(x, pos):
        w = (pos.double()[:, None] * freq)[:, None]
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * torch.polar(torch.full_like(w, conc), w)
        return torch.cat((z.real, z.imag), -1)

    out, a = [], 0
    for i, (n, p) in enumerate(zip(s["new"], s["past_list"])):
        pos = torch.arange(p, p + n, device=freq.device)
        out.append(turn(s["q"][a:a + n], pos))
        ids, slot = s["table"][i][pos // page].long(), pos % page
        for name, rows in (("k", turn(s["k"][a:a + n], pos)), ("v", s["v"][a:a + n].double())):
            rows = rows.float().double()  # a cached value is the 32-bit one rounded again
            if s["cache_type"] == "e4m3":
                top = rows.abs().amax(-1, keepdim=True)
                e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0))
                e = torch.where(top > 448.0 * torch.exp2(e), e + 1, torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e))
                e = torch.where(top > 0, e.clamp(-127, 127), torch.zeros_like(e))
                codes = (rows * torch.exp2(-e)).float().to(torch.float8_e4m3fn)
                s[name + "_pages"].view(torch.uint8)[ids, :, slot] = codes.view(torch.uint8)
                s[name + "_scale"][ids, :, slot] = (e[..., 0] + 127).to(torch.uint8)
            else:
                s[name + "_pages"][ids, :, slot] = rows.float().to(s[name + "_pages"].dtype)
        a += n
    return torch.cat(out)

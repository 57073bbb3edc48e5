"""Calls of the attention entry points that the documentation allows, on the host side (no GPU)."""
import copy
import ctypes
import math
import os
import re
import struct
import subprocess

import numpy as np
import pytest

from airllm_b200 import AmoeError, attention, build, moe

CUDA = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cuda")
F16, BF16 = moe.GGUF_F16, moe.GGUF_BF16
AT = 1 << 20  # an aligned address that no refused call reads


def rows(data=AT, ts=1 << 15, hs=128, heads=8, kind=BF16):
    return moe.AmoeRows(data, ts, hs, heads, kind)


def ref(x):
    return None if x is None else ctypes.byref(x)


def last_error():
    return moe.load_library().amoe_last_error(None).decode()


SHAPES = [(64, 64, 8), (128, 32, 8), (64, 12, 1), (128, 128, 1), (64, 15, 5)]


@pytest.mark.parametrize("d,heads,kv", SHAPES)
def test_prefill_takes_the_workspace_that_it_asks_for(d, heads, kv):
    """Every count of rows that fills whole waves of CTAs is among these.  A call is refused for its workspace exactly
    where the size is not 0; other calls are given a device ordinal that the check behind the workspace's refuses."""
    lib, a = moe.load_library(), moe.AmoeAttn(0.0, 0, None)
    q, k = rows(heads=heads), rows(heads=kv)
    asked = 0
    for behind in (0, 300, 2777, 9000):
        for seqs in (1, 3):
            for n in range(1, 4097):
                size = lib.amoe_attn_prefill_workspace(d, 0, heads, kv, n, n + behind, seqs)
                assert size >= 0
                if size:
                    asked += 1
                    continue
                rc = lib.amoe_attn_prefill(63, d, ref(a), ref(q), ref(k), ref(k), ref(q), n, n + behind, AT, AT, seqs,
                                           None, 0, None)
                assert rc == moe.AMOE_ERR_CUDA, (behind, seqs, n, last_error())
    assert asked > 0


def test_append_of_more_tokens_than_a_grid_holds():
    lib, r = moe.load_library(), rows()
    c = moe.AmoeKvCache(AT, AT, None, None, AT, 4, 16, 8, 64, BF16, 0)
    s = moe.AmoeKvSeqs(AT, 4, 2)
    flat = rows(ts=0)
    assert lib.amoe_kv_append(ref(c), ref(s), AT, AT, 2 ** 31 - 1, None, None, ref(flat), ref(flat), None, None, None,
                              None) == moe.AMOE_ERR_INVALID
    assert "tokens" in last_error()


def published_yarn(d, theta, factor, context, fast, slow, truncate):
    """Frequencies by the paper's formula: a pair's turns within the original context decide."""
    out = []
    corner = [d / 2 * math.log(context / (2 * math.pi * beta), theta) for beta in (fast, slow)]
    if truncate:
        corner = [math.floor(corner[0]), math.ceil(corner[1])]
    low, high = max(corner[0], 0), min(corner[1], d - 1)
    for i in range(d // 2):
        base = 1.0 / theta ** (i / (d / 2))
        keep = 1 - min(max((i - low) / (high - low), 0.0), 1.0)  # how much of the pair is left as it is
        out.append(keep * base + (1 - keep) * base / factor)
    return out


@pytest.mark.parametrize("d,theta,factor,context,fast,slow,truncate", [
    (64, 150000.0, 32.0, 4096.0, 32.0, 1.0, 0), (128, 150000.0, 32.0, 4096.0, 32.0, 1.0, 0),
    (128, 1e6, 4.0, 32768.0, 32.0, 1.0, 1), (64, 10000.0, 40.0, 4096.0, 32.0, 1.0, 1), (2, 10000.0, 8.0, 4096.0, 32.0, 1.0, 0),
    (96, 500000.0, 1.0, 8192.0, 16.0, 2.0, 0)])
def test_yarn_frequencies_are_the_published_ones(d, theta, factor, context, fast, slow, truncate):
    rope = moe.AmoeRope()
    assert moe.load_library().amoe_rope_init_yarn(d, theta, factor, context, fast, slow, truncate, ref(rope)) == moe.AMOE_OK
    got, want = list(rope.freq)[:d // 2], published_yarn(d, theta, factor, context, fast, slow, truncate)
    # a handful of float64 roundings on either side
    for a, b in zip(got, want):
        assert abs(a - b) <= 2.0 ** -48 * b
    assert got[0] == 1.0  # the fastest pair is left as it is
    if d >= 64:  # and the slowest divided
        assert abs(got[-1] - theta ** (2 / d - 1) / factor) <= 2.0 ** -48 * got[-1]
    assert abs(rope.concentration - (1 + 0.1 * math.log(factor))) <= 2.0 ** -50 and rope.head_dim == d


def test_yarn_with_every_pair_fast_or_slow():
    lib, rope = moe.load_library(), moe.AmoeRope()
    # a context so long that every pair turns often enough, and one in which none turns once
    assert lib.amoe_rope_init_yarn(64, 1e4, 8.0, 1e12, 32.0, 1.0, 0, ref(rope)) == moe.AMOE_OK
    assert all(abs(f * 1e4 ** (i / 32) - 1) < 1e-12 for i, f in enumerate(list(rope.freq)[:32]))
    assert lib.amoe_rope_init_yarn(64, 1e4, 8.0, 3.0, 32.0, 1.0, 0, ref(rope)) == moe.AMOE_OK
    assert all(abs(f * 8 * 1e4 ** (i / 32) - 1) < 1e-12 for i, f in enumerate(list(rope.freq)[:32]) if i > 0)


def test_the_reference_table_is_kept_under_its_own_name():
    """YaRNRoPE's ends of the ramp (rope.go:17-44) are the other way round."""
    rope = moe.AmoeRope()
    assert moe.load_library().amoe_rope_init(64, 150000.0, 1, ref(rope)) == moe.AMOE_OK
    assert rope.freq[0] == 1 / 32 and abs(rope.freq[31] * 150000.0 ** (31 / 32) - 1) < 1e-12


@pytest.mark.parametrize("at,value,word", [
    (0, 63, "even"), (0, 256, "128"), (1, 1.0, "theta"), (1, math.inf, "theta"), (2, 0.5, "factor"), (2, math.nan, "factor"),
    (2, math.inf, "factor"), (3, 0.0, "original_context"), (3, math.inf, "original_context"), (4, 0.5, "beta_fast"),
    (4, math.inf, "beta_fast"), (5, 0.0, "beta_slow"), (5, math.nan, "beta_slow")])
def test_yarn_refusals(at, value, word):
    args = [64, 150000.0, 32.0, 4096.0, 32.0, 1.0, 0]
    args[at] = value
    assert moe.load_library().amoe_rope_init_yarn(*args, ref(moe.AmoeRope())) == moe.AMOE_ERR_INVALID
    assert word in last_error()


def test_rope_from_python():
    rope = attention.Rope.yarn(64, 150000.0)
    assert rope.frequencies[0] == 1.0 and len(rope.frequencies) == 32
    assert abs(rope.concentration - 1.3465735902799727) < 1e-12
    assert attention.Rope.yarn(128, 1e6, factor=4.0, original_context=32768, truncate=True, concentration=1.0).concentration == 1.0
    with pytest.raises(AmoeError, match="factor"):
        attention.Rope.yarn(64, factor=0.0)
    assert attention.Rope(64, 150000.0).frequencies[0] == 1 / 32  # the reference's table


def test_the_search_for_sequences(tmp_path):
    exe = str(tmp_path / "kv_search")
    subprocess.run([build.NVCC, *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr", "-I", build.INCLUDE, "-I", build.CSRC,
                    "-o", exe, os.path.join(CUDA, "kv_search_check.cu")], check=True)
    got = subprocess.run([exe], capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout.strip() == "ok", got.stdout


def test_the_polynomial_of_the_exponentials():
    """2^x on the FMA pipe as attn_prefill.cu writes it, step by step in float32 (a product of two float32 is exact in
    float64, so adding there and rounding once is a fused step but for double roundings), against 2^x in float64."""
    src = open(os.path.join(build.CSRC, "attn_prefill.cu")).read()
    body = src[src.index("float2 ex2_poly("):]
    body = body[:body.index("\n}")]
    coeff = [np.float32(a) for a, b in re.findall(r"pair\(([\d.]+)f, ([\d.]+)f\)", body) if a == b and float(a) < 2]
    assert len(coeff) == 6
    f32, f64 = np.float32, np.float64

    def fma(a, b, c):
        return (a.astype(f64) * f64(b) + f64(c) if np.isscalar(b) else a.astype(f64) * b.astype(f64) + f64(c)).astype(f32)

    x = np.concatenate([np.linspace(-0.5, 0.5, 400001), np.linspace(-126, 16, 400001)]).astype(f32)
    t = x + f32(12582912.0)
    n = t - f32(12582912.0)
    f = x - n  # exact
    y = np.full_like(f, coeff[0])
    for c in coeff[1:]:
        y = fma(y, f, c)
    got = (y.view(np.int32) + (t.view(np.uint32).astype(np.int64) << 23).astype(np.uint32).view(np.int32)).view(f32)
    off = np.abs(got.astype(f64) / np.exp2(x.astype(f64)) - 1).max()
    assert 2.0 ** -22.5 < off <= 2.0 ** -22.1  # the bound that the source states, and that it is not idle
    assert "to 2^-22.1:" in src


@pytest.mark.parametrize("scale", [1e-50, 1e39, math.inf, math.nan, 0.0, -1.0, -math.inf])
def test_scales_that_float32_does_not_hold(scale):
    """1e-50 became 0, which asks for the default; 1e39 raised something else."""
    with pytest.raises(AmoeError, match="scale"):
        attention._attn(scale, 0, None, 8, 0)


def test_scales_that_float32_holds():
    for scale in (2.0 ** -149, 0.125, 3e38):
        assert struct.unpack("fiP", attention._attn(scale, 7, None, 8, 0))[0] == np.float32(scale)
    assert struct.unpack("fiP", attention._attn(None, 7, None, 8, 0)) == (0.0, 7, 0)


def test_check_clears_the_status_before_it_returns(monkeypatch):
    """The report is cleared on the current stream; a call on another stream may follow at once, and what it reports must
    not be cleared with it."""
    log = []

    class Status:
        def item(self):
            log.append("read")
            return moe.KV_BAD_PAGE

        def zero_(self):
            log.append("clear")

    cache = attention.KVCache.__new__(attention.KVCache)
    cache.status, cache.device = Status(), "cuda:0"
    monkeypatch.setattr(attention.torch.cuda, "synchronize", lambda device=None: log.append("wait"))
    with pytest.raises(AmoeError, match="page id"):
        cache.check()
    assert log == ["wait", "read", "clear", "wait"]


def test_a_copied_rope_has_its_own_table():
    """A deep copy kept the address of the original's table, which ends with the original."""
    rope = attention.Rope.yarn(64, 150000.0)
    other = copy.deepcopy(rope)
    rope._c.freq[0] = 7.0
    assert other.frequencies[0] == 1.0
    assert other._at == ctypes.addressof(other._c) != rope._at

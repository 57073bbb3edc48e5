"""The attention entry points' host side (no GPU): every refusal comes before the first CUDA
call, the paged cache's index arithmetic stays in bounds for wrong tables and lengths, and
the rotary frequencies are the oracle's."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

import oracle
from airllm_b200 import build, moe

CUDA = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cuda")
F32, F16, BF16, E4M3 = moe.GGUF_F32, moe.GGUF_F16, moe.GGUF_BF16, moe.KV_E4M3
AT = 1 << 20  # an aligned address that no refused call reads


def rows(data=AT, ts=512, hs=64, heads=8, kind=BF16):
    return moe.AmoeRows(data, ts, hs, heads, kind)


def cache(**kw):
    a = dict(k=AT, v=AT, k_scale=None, v_scale=None, status=AT, pages=4, page_size=16, kv_heads=8, head_dim=64,
             type=BF16, device=0)
    a.update(kw)
    return moe.AmoeKvCache(*[a[n] for n, _ in moe.AmoeKvCache._fields_])


def seqs(table=AT, stride=4, n=2):
    return moe.AmoeKvSeqs(table, stride, n)


def ref(x):
    return None if x is None else ctypes.byref(x)


def refused(rc, word):
    assert rc == moe.AMOE_ERR_INVALID
    assert word in moe.load_library().amoe_last_error(None).decode()


BAD_CACHES = [
    (dict(head_dim=96), "head_dim"), (dict(type=F32), "cache type"), (dict(page_size=24), "power of two"),
    (dict(page_size=0), "power of two"), (dict(page_size=8192), "power of two"), (dict(kv_heads=0), "kv_heads"),
    (dict(pages=0), "pages"), (dict(k=None), "NULL"), (dict(status=None), "NULL"), (dict(v=AT + 8), "aligned"),
    (dict(type=E4M3), "k_scale"),
]


@pytest.mark.parametrize("bad,word", BAD_CACHES)
def test_wrong_caches_are_refused(bad, word):
    lib, c, s, r, a = moe.load_library(), cache(**bad), seqs(), rows(), moe.AmoeAttn(0.0, 0, None)
    refused(lib.amoe_kv_append(ref(c), ref(s), AT, AT, 3, None, None, ref(r), ref(r), None, None, None, None), word)
    refused(lib.amoe_kv_read(ref(c), ref(s), AT, None, 3, ref(r), ref(r), None), word)
    refused(lib.amoe_attn_decode(ref(c), ref(s), ref(a), ref(r), ref(r), AT, 0, None, 0, None), word)


@pytest.mark.parametrize("s,word", [(dict(table=None), "page_table"), (dict(stride=0), "positive"), (dict(n=0), "positive")])
def test_wrong_tables_are_refused(s, word):
    lib, r = moe.load_library(), rows()
    refused(lib.amoe_kv_read(ref(cache()), ref(seqs(**s)), AT, None, 3, ref(r), ref(r), None), word)


@pytest.mark.parametrize("name,k,v,q,out,word", [
    ("heads", rows(heads=4), rows(), None, None, "heads"),
    ("types", rows(), rows(kind=F16), None, None, "element type"),
    ("type", rows(kind=8), rows(kind=8), None, None, "element type"),
    ("address", rows(data=AT + 2), rows(), None, None, "16 bytes"),
    ("stride", rows(ts=513), rows(), None, None, "16 bytes"),
    ("negative", rows(), rows(hs=-64), None, None, "negative"),
    ("far", rows(ts=1 << 61), rows(), None, None, "too large"),
    ("null", rows(data=None), rows(), None, None, "NULL"),
    ("q_out", rows(), rows(), None, rows(), "q_out"),
    ("q_out heads", rows(), rows(), rows(heads=16), rows(), "heads"),
])
def test_wrong_rows_are_refused_by_append(name, k, v, q, out, word):
    lib = moe.load_library()
    refused(lib.amoe_kv_append(ref(cache()), ref(seqs()), AT, AT, 3, None, ref(q), ref(k), ref(v), ref(out), None,
                               None, None), word)


def test_append_and_read_refuse_the_rest():
    lib, c, s, r = moe.load_library(), cache(), seqs(), rows()
    rope = moe.AmoeRope()
    assert lib.amoe_rope_init(128, 1e4, 0, ref(rope)) == moe.AMOE_OK
    refused(lib.amoe_kv_append(ref(c), ref(s), AT, AT, 3, ref(rope), None, ref(r), ref(r), None, None, None, None),
            "rope")
    refused(lib.amoe_kv_append(ref(c), ref(s), None, AT, 3, None, None, ref(r), ref(r), None, None, None, None), "cu")
    refused(lib.amoe_kv_append(ref(c), ref(s), AT, None, 3, None, None, ref(r), ref(r), None, None, None, None), "past")
    refused(lib.amoe_kv_append(ref(c), ref(s), AT, AT, -1, None, None, ref(r), ref(r), None, None, None, None), "tokens")
    refused(lib.amoe_kv_append(None, ref(s), AT, AT, 1, None, None, ref(r), ref(r), None, None, None, None), "cache")
    refused(lib.amoe_kv_read(ref(c), ref(s), None, None, 3, ref(r), ref(r), None), "cu")
    refused(lib.amoe_kv_read(ref(c), ref(s), AT, None, 3, ref(r), None, None), "v_out")
    # nothing to do is not an error, and touches no device
    assert lib.amoe_kv_append(ref(c), ref(s), AT, AT, 0, None, None, ref(r), ref(r), None, None, None, None) == 0
    assert lib.amoe_kv_read(ref(c), ref(s), AT, None, 0, ref(r), ref(r), None) == 0


@pytest.mark.parametrize("kw,word", [
    (dict(d=80), "head_dim"), (dict(q=rows(kind=F32), o=rows(kind=F32)), "F16 or BF16"), (dict(k=rows(kind=F16)), "type"),
    (dict(v=rows(heads=4)), "heads"), (dict(q=rows(heads=12), o=rows(heads=12)), "multiple"),
    (dict(k=rows(heads=1), v=rows(heads=1), q=rows(heads=129), o=rows(heads=129)), "128"),
    (dict(o=rows(heads=16)), "heads"), (dict(window=-1), "window"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=-1.0), "scale"), (dict(cu=None), "cu_q"), (dict(n=-1), "q_tokens"),
    (dict(seqs=0), "seqs"),
])
def test_prefill_refusals(kw, word):
    lib = moe.load_library()
    a = moe.AmoeAttn(kw.get("scale", 0.0), kw.get("window", 0), None)
    q, k, v, o = (kw.get(n, rows()) for n in "qkvo")
    refused(lib.amoe_attn_prefill(0, kw.get("d", 64), ref(a), ref(q), ref(k), ref(v), ref(o), kw.get("n", 5), 5,
                                  kw.get("cu", AT), AT, kw.get("seqs", 1), None, 0, None), word)


def test_prefill_without_rows_does_nothing():
    lib, r, a = moe.load_library(), rows(), moe.AmoeAttn(0.0, 0, None)
    assert lib.amoe_attn_prefill(0, 64, ref(a), ref(r), ref(r), ref(r), ref(r), 0, 5, AT, AT, 1, None, 0, None) == moe.AMOE_OK


@pytest.mark.parametrize("c,q,o,kw,word", [
    (cache(), rows(kind=F32), rows(kind=F32), {}, "F16 or BF16"), (cache(), rows(kind=F16), rows(kind=F16), {}, "types"),
    (cache(), rows(), rows(kind=F16), {}, "type"), (cache(), rows(heads=12), rows(heads=12), {}, "multiple"),
    (cache(kv_heads=1), rows(heads=129), rows(heads=129), {}, "128"), (cache(), rows(), rows(), dict(len=None), "kv_len"),
    (cache(), rows(), rows(), dict(most=-1), "max_len"), (cache(), rows(), rows(), dict(n=65536), "65535"),
])
def test_decode_refusals(c, q, o, kw, word):
    lib, a = moe.load_library(), moe.AmoeAttn(0.0, 0, None)
    refused(lib.amoe_attn_decode(ref(c), ref(seqs(n=kw.get("n", 2))), ref(a), ref(q), ref(o), kw.get("len", AT),
                                 kw.get("most", 0), None, 0, None), word)


def test_decode_workspace():
    lib, a, r = moe.load_library(), moe.AmoeAttn(0.0, 0, None), rows()
    c = cache(pages=4096, page_size=64)
    short, long, many = seqs(stride=16, n=1), seqs(stride=2048, n=1), seqs(stride=2048, n=256)
    def size(s, window=0, most=0):
        return lib.amoe_attn_decode_workspace(ref(c), ref(s), 8, window, most)
    # a short context or a large batch needs none, a long one does unless the call bounds it
    assert size(short) == 0 and size(many) == 0 and size(long) > 0
    assert size(long, window=128) == 0 and size(long, most=1000) == 0
    assert lib.amoe_attn_decode_workspace(ref(c), ref(long), 12, 0, 0) == moe.AMOE_ERR_INVALID
    assert lib.amoe_attn_decode_workspace(ref(c), ref(long), 8, -1, 0) == moe.AMOE_ERR_INVALID
    assert lib.amoe_attn_decode_workspace(None, ref(long), 8, 0, 0) == moe.AMOE_ERR_INVALID
    for work, n in ((None, size(long)), (AT, size(long) - 1)):
        refused(lib.amoe_attn_decode(ref(c), ref(long), ref(a), ref(r), ref(r), AT, 0, work, n, None), "workspace")
    refused(lib.amoe_attn_decode(ref(c), ref(long), ref(a), ref(r), ref(r), AT, 0, AT + 4, 1 << 40, None), "aligned")


@pytest.mark.parametrize("d,theta,yarn", [(64, 150000.0, 1), (128, 150000.0, 1), (64, 10000.0, 0), (2, 500000.0, 1)])
def test_rope_frequencies_turn_like_the_oracle(d, theta, yarn):
    rope = moe.AmoeRope()
    assert moe.load_library().amoe_rope_init(d, theta, yarn, ref(rope)) == moe.AMOE_OK
    assert rope.head_dim == d
    pos, half = 777, d // 2
    x = np.random.default_rng(d).standard_normal(d).astype(np.float32)
    ang = pos * np.array(rope.freq[:half])
    c, s = np.cos(ang) * rope.concentration, np.sin(ang) * rope.concentration
    a, b = x[:half].astype(np.float64), x[half:].astype(np.float64)
    want = np.concatenate([a * c - b * s, b * c + a * s])
    got = (oracle.yarn_rope if yarn else oracle.rope)(x, d, pos, theta)
    # one rounding to f32 on each side of the same float64 formula
    np.testing.assert_allclose(got, want, rtol=2.0 ** -23, atol=0)


@pytest.mark.parametrize("d,theta,word", [(63, 1e4, "even"), (0, 1e4, "even"), (256, 1e4, "128"), (64, 0.0, "theta"),
                                          (64, math.inf, "theta"), (64, math.nan, "theta")])
def test_rope_refusals(d, theta, word):
    refused(moe.load_library().amoe_rope_init(d, theta, 1, ref(moe.AmoeRope())), word)
    refused(moe.load_library().amoe_rope_init(64, 1e4, 1, None), "out")


def test_index_arithmetic_stays_in_bounds(tmp_path):
    exe = str(tmp_path / "kv_index")
    subprocess.run([build.NVCC, *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr", "-I", build.INCLUDE, "-I", build.CSRC, "-o", exe,
                    os.path.join(CUDA, "kv_index_check.cu")], check=True)
    got = subprocess.run([exe], capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout.strip() == "ok", got.stdout


def test_prefill_workspace():
    lib, a, r = moe.load_library(), moe.AmoeAttn(0.0, 0, None), rows()
    def size(d=64, window=0, heads=8, kv=8, q=16, k=32768, n=1):
        return lib.amoe_attn_prefill_workspace(d, window, heads, kv, q, k, n)
    # few queries behind many keys need one; many queries, few keys, a window or many sequences none
    assert size() > 0 and size(d=128) > 0 and size(q=1) > 0
    assert size(q=20000) == 0 and size(k=200) == 0 and size(window=128) == 0 and size(q=300, n=300) == 0
    assert size(q=0, k=0) == 0
    for bad in (dict(d=80), dict(heads=12), dict(window=-1), dict(q=-1), dict(k=-1), dict(n=0)):
        assert size(**bad) == moe.AMOE_ERR_INVALID
    for work, n in ((None, size()), (AT, size() - 1)):
        refused(lib.amoe_attn_prefill(0, 64, ref(a), ref(r), ref(r), ref(r), ref(r), 16, 32768, AT, AT, 1, work, n, None),
                "workspace")
    refused(lib.amoe_attn_prefill(0, 64, ref(a), ref(r), ref(r), ref(r), ref(r), 16, 32768, AT, AT, 1, AT + 4, 1 << 40,
                                  None), "aligned")

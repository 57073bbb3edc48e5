"""Calls of the attention entry points that the documentation allows, on the host side (no GPU)."""
import ctypes

import pytest

from airllm_b200 import moe

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

"""Calls of the attention operators that the documentation allows and the other tests leave out: whole waves of
row tiles, wrong lengths into filled outputs, values at the ends of the 16-bit weights' range, far positions."""
import math

import pytest
import torch

import attention_ref as R
from airllm_b200 import AmoeError, attention, moe
from test_attention_gpu import BF16, E4M3, F16, F32, filled, gen, i32, on_gpu, randn, starts, table_for

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

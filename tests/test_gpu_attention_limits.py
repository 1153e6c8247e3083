"""The attention operators at the ends of what their interface allows, against the definitions in 64 bits: widths between the
16-byte words, bounds that disagree with the call, scores and weights far apart, values in places that are masked."""
import math

import numpy as np
import pytest
import torch

import attention_ref as ref
import ovk_b200
from gpu_util import ctx, dev
from test_gpu_attention import F16, F32, cache_rows, check_kv4, check_prompt, filled_cache, i32, make_table, randn, starts

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------- widths between words
@pytest.mark.parametrize("d,wide", [(20, 24), (100, 104), (250, 256), (33, 40), (12, 16), (1, 8), (64, 72)])
@pytest.mark.parametrize("gap,shift", [(None, 0), (8, 0), (3, 1)])
def test_prompt_heads_that_end_inside_a_word(d, wide, gap, shift):
    """Slices of padded rows: 16-byte aligned, whatever their width.  Nothing behind a row is read or written."""
    lens, hq, hk = [130, 0, 61], 4, 2
    n = sum(lens)

    def padded(heads, seed):
        t = torch.full((n, heads, wide), math.nan, dtype=F16)
        t[..., :d] = randn((n, heads, d), seed, F16)
        return t
    q, k, v = padded(hq, 1), padded(hk, 2), padded(hk, 3)
    if gap is None:
        out = None
    else:
        pitch = (d + 7) // 8 * 8 + gap if shift == 0 else d + gap
        buffer = torch.full((shift + (n * hq + 1) * pitch,), 7.0, dtype=F16, device="cuda")
        out = buffer[shift:shift + n * hq * pitch].view(n, hq, pitch)[..., :d]
    got = ctx().attention_prompt(q.cuda()[..., :d], k.cuda()[..., :d], v.cuda()[..., :d], starts(lens), max(lens), out=out)
    ctx().flush()
    assert ctx().last_kernel == "attention_prompt_tc"
    check_prompt(q[..., :d], k[..., :d], v[..., :d], [0, 130, 130, 191], [0, 130, 130, 191], d ** -0.5, True, 0, got.cpu(), False)
    if gap is not None:
        rows = buffer[shift:shift + n * hq * pitch].view(n, hq, pitch)
        assert bool((rows[..., d:] == 7).all()) and bool((buffer[:shift] == 7).all()) and bool((buffer[shift + n * hq * pitch:] == 7).all())

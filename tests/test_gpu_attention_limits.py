"""The attention operators at the ends of what their interface allows, against the definitions in 64 bits: widths between the
16-byte words, bounds that disagree with the call, scores and weights far apart, values in places that are masked."""
import ctypes as C
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


# ------------------------------------------------------- bounds that disagree with the call
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("bad", [0, 30, 69])
@pytest.mark.parametrize("kind", ["long", "before", "behind"])
def test_prompt_reports_bad_sequences_of_large_batches(dtype, bad, kind):
    """A sequence that is left out is reported wherever it lies in the batch."""
    lens = [3] * 70
    lens[bad] = 9 if kind == "long" else 3
    n = sum(lens)
    q, k = randn((n, 2, 64), 1, dtype).cuda(), randn((n, 1, 64), 2, dtype).cuda()
    cu = [sum(lens[:i]) for i in range(71)]
    if kind == "before":  # the sequence before this one ends in front of its own start
        cu[bad + 1] = -1 if bad == 0 else cu[bad] - 1
    elif kind == "behind":
        cu[bad + 1] = n + 5
    out = ctx().attention_prompt(q, k, k, i32(cu), 8, cu_k=i32([sum(lens[:i]) for i in range(71)]), out=torch.full_like(q, 3.0))
    with pytest.raises(ovk_b200.OvkError) as e:
        ctx().flush()
    assert e.value.status == ovk_b200.INVALID_ARGUMENT and "bounds" in e.value.message
    if kind == "long":
        keep = torch.ones(n, dtype=torch.bool)
        keep[cu[bad]:cu[bad + 1]] = False
        assert bool((out[~keep.cuda()] == 3).all()) and bool((out[keep.cuda()] != 3).any(-1).all())
    ctx().attention_prompt(q, k, k, starts(lens), 9)
    ctx().flush()


@pytest.mark.parametrize("cu,kept", [([0, 9], []), ([-1, 2], []), ([0, 1, 5], [0]), ([-3, 1, 3], [1, 2]), ([0, 2, 1], None)])
def test_append_of_bad_bounds_is_left_out_and_reported(cu, kept):
    """Sequences whose rows lie outside the tensors store nothing; the others store their rows."""
    batch = len(cu) - 1
    cache = ctx().kv4_cache(2 * batch, 1, 8, 64, 32)
    k = torch.ones((3, 1, 64), dtype=F16, device="cuda")
    table, lens = [[2 * b, 2 * b + 1] for b in range(batch)], [max(cu[b + 1] - cu[b], 0) for b in range(batch)]
    ctx().kv4_append(cache, k, k, i32(table), i32(cu), i32(lens))
    with pytest.raises(ovk_b200.OvkError) as e:
        ctx().flush()
    assert e.value.status == ovk_b200.INVALID_ARGUMENT and "bounds" in e.value.message
    # (which sequence rows belong to that two claim is not said)
    assert kept is None or int((cache.k_scales != 0).any(-1).sum()) == len(kept)
    ctx().flush()


def test_append_reports_bad_bounds_of_a_large_batch():
    """Bounds that no row falls into, far from the rows there are."""
    cu = [0] * 2000 + [1]
    cu[700] = -4
    cache = ctx().kv4_cache(2, 1, 8, 64, 32)
    k = torch.ones((1, 1, 64), dtype=F16, device="cuda")
    ctx().kv4_append(cache, k, k, i32([[0]] * 2000), i32(cu), i32([1] * 2000))
    with pytest.raises(ovk_b200.OvkError) as e:
        ctx().flush()
    assert "bounds" in e.value.message and int((cache.k_scales != 0).any(-1).sum()) == 1
    ctx().flush()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,hq,hk,new,lens", [(128, 8, 1, [5, 1], [77, 4]), (64, 12, 4, [1, 9], [3, 40]), (256, 4, 1, [70], [90])])
def test_kv4_more_new_tokens_than_promised(dtype, d, hq, hk, new, lens):
    """max_tokens chooses a variant; results hold for any number of new tokens."""
    cache, table = filled_cache(lens, hk, d, 32, 16, True, d)
    q = randn((sum(new), hq, d), 9, F32, 1.5).to(dtype)
    for most in (1, 2, max(new), 1000):
        got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts(new), i32(lens), max_tokens=most)
        ctx().flush()
        check_kv4(cache, table, q, new, lens, d ** -0.5, 0, got.cpu())


# --------------------------------------------------- scores and weights far from one another
@pytest.mark.parametrize("score", [-1e31, -3e37, 1e37])
@pytest.mark.parametrize("d,split", [(64, 8), (128, 16), (256, 8), (33, 4)])
def test_prompt_f32_scores_of_any_size(score, d, split):
    """A row with one key gives that key's value, however low its score; of several keys the highest score takes all."""
    n = 70
    q, k = torch.zeros(n, 2, d), torch.zeros(n, 1, d)
    v = randn((n, 1, d), 3)
    root = math.sqrt(abs(score))
    q[..., 1], k[..., 1] = root, math.copysign(root, score)
    k[:, 0, 1] *= 1 + torch.arange(n) / n  # farther from zero with each key
    cu = [0, 1, split, n]
    got = ctx().attention_prompt(q.cuda(), k.cuda(), v.cuda(), i32(cu), scale=1.0)
    ctx().flush()
    for a, b in zip(cu, cu[1:]):
        for i in range(a, b):  # scores are in steps of more than a weight's whole range
            want = v[a if score < 0 else i]
            assert bool(((got[i].cpu() - want).abs() <= 2.0 ** -21 * want.abs()).all()), (i, float(got[i].abs().max()))


SIZES = [1.0, 37.3, 300.7, 5.1e3, 1.03e6, 1e27]  # scales that bring a score of a million to 2^20 .. 2^110


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("scale", SIZES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_f16_scores_of_any_size(d, scale, sign):
    """Equal scores, however large: the mean of the values that a row reads."""
    q, k = torch.zeros(250, 2, d, dtype=F16), torch.zeros(250, 1, d, dtype=F16)
    q[..., 0], k[..., 0] = 1000.0, sign * 1000.0
    q[..., 1], k[..., 1] = 3.0, 3.0
    v = randn((250, 1, d), 3, F16)
    got = ctx().attention_prompt(q.cuda(), k.cuda(), v.cuda(), starts([1] * 50 + [200]), scale=scale)
    ctx().flush()
    assert bool(((got[:50].cpu() - v[:50]).abs() <= 2.0 ** -11 * v[:50].abs()).all())
    x, count = v[50:].double(), torch.arange(1, 201)[:, None, None]
    # a weight is one fp16 number (2^-11), sums are f32
    ref.check(got[50:], (x.cumsum(0) / count).expand(200, 2, d), (x.abs().cumsum(0) / count * (2.0 ** -11 + 210 * 2.0 ** -23)).expand(200, 2, d), "mean")


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("scale", SIZES)
@pytest.mark.parametrize("d,lens", [(64, [1]), (128, [1, 1]), (256, [1, 40]), (128, [700])])
def test_kv4_scores_of_any_size(dtype, d, lens, scale, sign):
    """Equal scores, however large: the mean of the cached values."""
    table, pages = make_table(lens, 16, 1)
    cache = ctx().kv4_cache(pages, 1, 16, d, 32)
    total = sum(lens)
    k, v = torch.zeros(total, 1, d), randn((total, 1, d), 2, F32, 3e-4)
    k[..., 0] = sign * 1000.0
    ctx().kv4_append(cache, k.cuda(), v.cuda(), dev(table), starts(lens), i32(lens))
    q = torch.zeros(len(lens), 4, d, dtype=dtype)
    q[..., 0] = 1000.0
    got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts([1] * len(lens)), i32(lens), scale=scale)
    ctx().flush()
    values = ref.dequantize(*cache_rows(cache, "v"))
    for b, n in enumerate(lens):
        at = torch.arange(n)
        rows = values[torch.as_tensor(table[b])[at // 16].long(), 0, at % 16]
        # a weight times a value's scale is one fp16 number (f16) or two (f32)
        p_error = 2.0 ** -11 if dtype == F16 else 2.0 ** -21
        ref.check(got[b], rows.mean(0).expand(4, d), (rows.abs().mean(0) * (p_error + (n + 8) * 2.0 ** -23)).expand(4, d), f"sequence {b}")


@pytest.mark.parametrize("d,heads", [(64, 1), (128, 2), (256, 1)])
@pytest.mark.parametrize("peak", ["first", "last"])
def test_prompt_f16_long_flat_tail(d, heads, peak):
    """One key outweighs each of thousands by 2^26, which together are half a thousandth of it: weights are f16, off by 2^-11 of
    themselves or 2^-32 of the largest, whichever is more."""
    n, m = 32768, 128  # keys; queries, the last m tokens
    q = torch.zeros(m, heads, d, dtype=F16)
    k, v = torch.zeros(n, 1, d, dtype=F16), torch.zeros(n, 1, d, dtype=F16)
    q[..., 0] = 8.0
    k[..., 0] = -2.25  # scores of -18: e^-18 = 2^-25.97
    v[..., 0], v[:, 0, 1] = 1.0, torch.linspace(-1, 1, n).half()
    at = 0 if peak == "first" else n - m
    k[at, 0, 0], v[at, 0, :2] = 0.0, 0.0
    v[at, 0, 2] = 1.0
    got = ctx().attention_prompt(q.cuda(), k.cuda(), v.cuda(), i32([0, m]), m, cu_k=i32([0, n]), scale=1.0).double().cpu()
    ctx().flush()
    w = math.exp(-18.0)
    for i in (0, 1, m // 2, m - 1):
        reads = n - m + i + 1
        below = (reads - 1) * w
        total = 1 + below
        # each weight's rounding, 2^-11 of it or (reads - 1) of 2^-32 in all; f32 sums; the result's half step
        slack = below * 2.0 ** -11 + reads * 2.0 ** -32 + below * reads * 2.0 ** -23
        want = torch.tensor([below, float(v[:reads, 0, 1].double().sum()) * w, 1.0]) / total
        for e, tol in ((0, slack), (1, slack), (2, 2.0 ** -11)):
            assert float((got[i, :, e] - want[e]).abs().max()) <= tol + 2.0 ** -11 * abs(float(want[e])), (i, e, got[i, :, e], want[e])


# ------------------------------------------------------------ what lies in masked places
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,hq,block", [(64, 2, 64), (128, 4, 32), (128, 12, 128), (256, 4, 32)])
@pytest.mark.parametrize("scale", [math.inf, math.nan, 65504.0])
@pytest.mark.parametrize("new,lens,window,at", [([1], [100], 33, 65), ([3], [100], 0, 99), ([2], [70], 20, 48), ([4], [64], 0, 61)])
def test_kv4_scales_in_masked_places_leave_small_values_exact(dtype, d, hq, block, scale, new, lens, window, at):
    """A value scale that some rows must not read, far above those that they read, costs them no accuracy."""
    table, pages = make_table(lens, 16, 1)
    cache = ctx().kv4_cache(pages, 1, 16, d, block)
    k, v = randn((lens[0], 1, d), 1), randn((lens[0], 1, d), 2, F32, 2e-4)
    ctx().kv4_append(cache, k.cuda(), v.cuda(), dev(table), starts(lens), i32(lens))
    ctx().flush()
    clean = {w: ref.dequantize(*cache_rows(cache, w)) for w in ("k", "v")}
    sizes = ref.row_sizes(*cache_rows(cache, "k"))
    cache.v_scales[int(table[0][at // 16]), 0, at % 16] = scale
    q = randn((new[0], hq, d), 9, F32, 1.5).to(dtype)
    got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts(new), i32(lens), max_tokens=new[0], window=window)
    ctx().flush()
    got, n, checked = got.cpu(), lens[0], 0
    p_error, q_error = (2.0 ** -21, 2.0 ** -21) if dtype == F32 else (2.0 ** -11, 0.0)
    for i in range(new[0]):
        last = n - new[0] + i
        first = max(0, last - window + 1) if window else 0
        if first <= at <= last:
            continue
        t = torch.arange(first, last + 1)
        page = torch.as_tensor(table[0])[t // 16].long()
        for h in range(hq):
            want, bound = ref.attend(q[i:i + 1, h].double(), clean["k"][page, 0, t % 16], clean["v"][page, 0, t % 16], d ** -0.5, False, 0,
                                     p_error, q_error, sizes[page, 0, t % 16])
            ref.check(got[i:i + 1, h], want, bound, f"row {i} head {h}")
            checked += 1
    assert checked


def test_a_context_of_the_default_stream_under_another_current_stream():
    lens = [70, 5]
    table, pages = make_table(lens, 16, 1)
    cos, sin = (torch.rand(100, 64, device="cuda") for _ in range(2))
    q, k, v = (randn((75, h, 128), s, F16).cuda() for h, s in ((4, 1), (1, 2), (1, 3)))
    at, cu, n, t = torch.arange(75, device="cuda"), starts(lens), i32(lens), dev(table)
    c = ctx()

    def layer():
        x, y = c.rotary(q, cos, sin, at, k=k)
        cache = c.kv4_cache(pages, 1, 16, 128)
        c.kv4_append(cache, y, v, t, cu, n)
        return x, y, c.attention_prompt(x, y, v, cu), c.attention_kv4(cache, x, t, cu, n, max_tokens=70), *cache.tensors
    want = layer()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = layer()
        c.flush()
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("window", [2 ** 63 - 1, 2 ** 40, 2 ** 31, 2 ** 30])
def test_windows_of_any_size(dtype, window):
    """A window longer than any sequence is none, also where there are more new tokens than keys."""
    cache, table = filled_cache([2, 50], 1, 64, 32, 16, True, 3)
    q = randn((6, 2, 64), 9, dtype)
    got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts([5, 1]), i32([2, 50]), max_tokens=5, window=window)
    ctx().flush()
    check_kv4(cache, table, q, [5, 1], [2, 50], 64 ** -0.5, 0, got.cpu())
    q, k, v = randn((140, 2, 64), 1, dtype), randn((12, 1, 64), 2, dtype), randn((12, 1, 64), 3, dtype)
    for causal in (True, False):
        got = ctx().attention_prompt(q.cuda(), k.cuda(), v.cuda(), i32([0, 140]), cu_k=i32([0, 12]), causal=causal, window=window)
        want = ctx().attention_prompt(q.cuda(), k.cuda(), v.cuda(), i32([0, 140]), cu_k=i32([0, 12]), causal=causal)
        ctx().flush()
        assert torch.equal(got, want)


def test_fresh_contexts_start_with_cleared_counters():
    """The first call of a context that was just made, several blocks sharing a sequence."""
    lens = [6000]
    cache, table = filled_cache(lens, 1, 128, 32, 64, True, 3)
    q, t, cu, n = randn((1, 8, 128), 1, F16).cuda(), dev(table), starts([1]), i32(lens)
    want = ctx().attention_kv4(cache, q, t, cu, n).clone()
    ctx().flush()
    for _ in range(20):
        c = ovk_b200.Context(0)
        got = torch.empty_like(q)
        c.attention_kv4(cache, q, t, cu, n, out=got)
        c.flush()
        assert torch.equal(got, want)
        c.close()


# --------------------------------------------------------- calls that no other test makes
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,block", [(64, 32), (128, 128), (256, 64)])
def test_append_of_slices_at_any_alignment(dtype, d, block):
    """Keys and values as slices of one wide product that starts anywhere: the same codes as from tensors of their own."""
    wide = randn((21, 4 * d + 3), 1, dtype).cuda()
    k, v = wide[:, 1:1 + 2 * d].unflatten(1, (2, d)), wide[:, 3 + 2 * d:].unflatten(1, (2, d))
    lens, caches = [20, 1], []
    for a, b in ((k, v), (k.contiguous(), v.contiguous())):
        cache = ctx().kv4_cache(5, 2, 8, d, block)
        ctx().kv4_append(cache, a, b, i32([[4, 1, 0], [3, -1, -1]]), starts(lens), i32(lens))
        ctx().flush()
        caches.append((ctx().last_kernel, cache))
    assert [c[0] for c in caches] == ["kv4_append_scalar", "kv4_append"]
    assert all(torch.equal(x, y) for x, y in zip(caches[0][1].tensors, caches[1][1].tensors))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_kv4_sequences_that_share_pages(dtype):
    """A common beginning of three sequences lies in the cache once."""
    lens = [48, 61, 70]
    cache, table = filled_cache([100, 40, 40], 1, 128, 32, 16, True, 5)
    shared = np.array([[table[0][0], table[0][1], table[0][2], -1, -1], [*table[0][:3], table[1][0], -1], [*table[0][:3], table[2][0], table[2][1]]],
                      dtype=np.int32)
    q = randn((3, 8, 128), 9, F32, 1.5).to(dtype)
    got = ctx().attention_kv4(cache, q.cuda(), dev(shared), starts([1] * 3), i32(lens))
    ctx().flush()
    check_kv4(cache, shared, q, [1] * 3, lens, 128 ** -0.5, 0, got.cpu())


def test_kv4_workspaces_of_the_caller():
    """Through the C interface: a workspace of the stated size gives the same bits and is left zeroed; less is refused."""
    lib, c, lens = ovk_b200.lib(), ctx(), [9000, 3]
    cache, table = filled_cache(lens, 1, 128, 32, 64, True, 3)
    q, t, cu, n = randn((2, 8, 128), 1, F16).cuda(), dev(table), starts([1, 1]), i32(lens)
    want = c.attention_kv4(cache, q, t, cu, n)
    out = torch.empty_like(q)
    heads = lambda x: ovk_b200.Heads(x.data_ptr(), 8, 1024, 128)  # noqa: E731
    batch = ovk_b200.KV4Batch(2, 2, t.shape[1], cu.data_ptr(), n.data_ptr(), t.data_ptr())
    size = C.c_size_t()
    assert lib.ovk_attention_kv4_workspace(c.h, cache.params, 8, 1, ovk_b200.FLOAT16, C.byref(size)) == ovk_b200.OK
    space = torch.full((size.value + 16,), 255, dtype=torch.uint8, device="cuda")
    space[:4096] = 0

    def call(at, size):
        return lib.ovk_attention_kv4(c.h, cache.params, batch, heads(q), heads(out), ovk_b200.FLOAT16, 1, 128 ** -0.5, 0, at, size)
    for _ in range(3):
        out.zero_()
        assert call(space.data_ptr(), size.value) == ovk_b200.OK
        c.flush()
        assert torch.equal(out, want) and int(space[:4096].sum()) == 0 and bool((space[-16:] == 255).all())
    assert call(space.data_ptr(), 4096) == ovk_b200.INVALID_ARGUMENT and call(space.data_ptr() + 8, size.value) == ovk_b200.INVALID_ARGUMENT
    stream = torch.cuda.Stream()
    own = ovk_b200.Context(0, stream.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):  # the context's own workspace would be shared by all graphs
        rc = lib.ovk_attention_kv4(own.h, cache.params, batch, heads(q), heads(out), ovk_b200.FLOAT16, 1, 1.0, 0, None, 0)
        out.zero_()
    assert rc == ovk_b200.INVALID_ARGUMENT and b"workspace" in lib.ovk_last_error(own.h)
    del graph
    own.close()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_every_operator_repeats_itself(dtype):
    """Results do not depend on timing: the same bits ten times, two contexts at once."""
    lens = [700, 3, 1500]
    total = sum(lens)
    table, pages = make_table(lens, 16, 1)
    cos, sin = (torch.rand(1500, 64, device="cuda") for _ in range(2))
    q, k, v = (randn((total, h, 128), s, dtype).cuda() for h, s in ((8, 1), (2, 2), (2, 3)))
    at = torch.cat([torch.arange(n) for n in lens]).cuda()
    cu, n, t, last = starts(lens), i32(lens), dev(table), starts([1] * 3)
    streams = [torch.cuda.Stream() for _ in range(2)]
    contexts = [ovk_b200.Context(0, s.cuda_stream) for s in streams]
    torch.cuda.synchronize()
    first = None
    for _ in range(10):
        results = []
        for c, s in zip(contexts, streams):
            with torch.cuda.stream(s):
                x, y = c.rotary(q, cos, sin, at, k=k)
                cache = c.kv4_cache(pages, 2, 16, 128)
                c.kv4_append(cache, y, v, t, cu, n)
                results.append((x, y, *cache.tensors, c.attention_prompt(x, y, v, cu), c.attention_kv4(cache, x[:3].contiguous(), t, last, n)))
        for c in contexts:
            c.flush()
        first = first or results[0]
        for r in results:
            assert all(torch.equal(a, b) for a, b in zip(r, first))
    for c in contexts:
        c.close()


@pytest.mark.parametrize("dtype,below", [(F16, 24.0), (F32, 24.0), (F32, 33.0)])
@pytest.mark.parametrize("d,hq", [(64, 2), (128, 12), (256, 4)])
@pytest.mark.parametrize("n,peak", [(32, 0), (32, 31), (257, 30), (32767, 0), (32767, 32000)])
def test_kv4_long_flat_tail(dtype, below, d, hq, n, peak):
    """One token outweighs each of many by 2^below: a weight times its value's scale is off by 2^-11 (f16) or 2^-22 (f32) of
    itself or by 2^-31 or 2^-35 of the largest weight and scale, whichever is more."""
    table, pages = make_table([n], 64, 1)
    cache = ctx().kv4_cache(pages, 1, 64, d, 32)
    k, v = torch.zeros(n, 1, d), torch.ones(n, 1, d)
    k[..., 0] = -4.0
    k[peak, 0, 0], v[peak, 0, :2] = 0.0, 0.0
    v[:, 0, 1] *= torch.linspace(0, 1, n)
    ctx().kv4_append(cache, k.cuda(), v.cuda(), dev(table), starts([n]), i32([n]))
    q = torch.zeros(1, hq, d, dtype=dtype)
    q[..., 0] = 8.0
    scale = below / 32.0 * math.log(2)
    got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts([1]), i32([n]), scale=scale)
    ctx().flush()
    at = torch.arange(n)
    page = torch.as_tensor(table[0])[at // 64].long()
    rows = {w: ref.dequantize(*cache_rows(cache, w))[page, 0, at % 64] for w in ("k", "v")}
    p = torch.softmax(rows["k"] @ q[0, 0].double() * scale, 0)
    itself, floor = (2.0 ** -11, 2.0 ** -31) if dtype == F16 else (2.0 ** -21, 2.0 ** -35)
    largest = 15 * float(cache.v_scales.max())
    # a score of -33 powers of two is rounded three times (33 * 3 * 2^-24 of the weight), sums of n weights are off by n 2^-23
    bound = (p @ rows["v"].abs()) * (itself + 2.0 ** -17 + n * 2.0 ** -23) + n * floor * largest * float(p.max())
    assert float(p[peak]) > 0.9 and float((p @ rows["v"])[0]) > 1.9 * float(bound[0])  # a tail left out is noticed
    ref.check(got[0], (p @ rows["v"]).expand(hq, d), bound.expand(hq, d), "tail")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,hq,hk", [(64, 3, 3), (128, 8, 2), (256, 4, 1)])
def test_results_in_the_place_of_the_queries(dtype, d, hq, hk):
    lens = [1, 700, 0, 129, 2000]
    n = sum(lens)
    q, k, v = (randn((n, h, d), s, dtype).cuda() for s, h in ((1, hq), (2, hk), (3, hk)))
    want = ctx().attention_prompt(q, k, v, starts(lens))
    x = q.clone()
    assert ctx().attention_prompt(x, k, v, starts(lens), out=x) is x
    ctx().flush()
    assert torch.equal(x, want)
    cache, table = filled_cache(lens, hk, d, 32, 16, True, 5)
    new = [1, 40, 0, 3, 1]
    q, cu, t, total = q[:sum(new)].contiguous(), starts(new), dev(table), i32(lens)
    want = ctx().attention_kv4(cache, q, t, cu, total, max_tokens=40)
    for _ in range(5):
        x = q.clone()
        ctx().attention_kv4(cache, x, t, cu, total, max_tokens=40, out=x)
        ctx().flush()
        assert torch.equal(x, want)

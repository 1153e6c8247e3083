"""Rotary positions, the 4-bit key / value cache and attention against their definitions in 64 bits, through the C ABI."""
import math

import numpy as np
import pytest
import torch

import attention_ref as ref
import ovk_b200
from gpu_util import ctx, dev, host

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def randn(shape, seed, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def starts(lengths, first=0):
    return i32([first + sum(lengths[:i]) for i in range(len(lengths) + 1)])


# ------------------------------------------------------------------------- rotary
def tables(rows, pairs, dtype):
    angle = torch.arange(rows).double()[:, None] * torch.pow(10000.0, -torch.arange(pairs).double() / pairs)
    return angle.cos().to(dtype), angle.sin().to(dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens,hq,hk,d,rotary,sections,interleaved,index,table", [
    (1, 1, 1, 64, 64, [32], False, torch.int64, F32),
    (64, 16, 2, 128, 128, [16, 24, 24], False, torch.int64, F32),
    (37, 5, 1, 128, 128, [3, 0, 61], False, torch.int32, F32),       # sections that split a 16-byte access
    (37, 5, 1, 128, 64, [8, 24], False, torch.int32, F16),           # half of a head is copied
    (19, 3, 3, 80, 80, [40], False, torch.int64, F32),
    (19, 3, 3, 80, 20, [4, 3, 2, 1], True, torch.int32, F16),
    (33, 2, 1, 256, 256, [128], True, torch.int64, F32),
    (7, 4, 1, 6, 2, [1], False, torch.int64, F32),
    (5, 4, 1, 6, 6, [1, 2], True, torch.int32, F32),
])
def test_rotary(dtype, tokens, hq, hk, d, rotary, sections, interleaved, index, table):
    cos, sin = tables(91, rotary // 2, table)
    at = torch.from_numpy(np.random.default_rng(tokens).integers(0, 91, (len(sections), tokens)))
    q, k = randn((tokens, hq, d), 1, dtype), randn((tokens, hk, d), 2, dtype)
    got = ctx().rotary(q.cuda(), cos.cuda(), sin.cuda(), at.to(index).cuda(), k=k.cuda(), sections=sections, interleaved=interleaved)
    ctx().flush()
    for x, y in zip((q, k), got):
        want, size = ref.rotary(x, cos, sin, at, sections, interleaved)
        # two products, one of them rounded on its own, and their sum: two roundings of at most the sum of sizes
        ref.check(y, want, size * 2 * 2.0 ** -24, "rotary")


def test_rotary_in_place_on_a_slice_of_a_fused_product():
    qkv = randn((23, 6, 128), 3, F16).cuda()
    before = qkv.clone()
    cos, sin = (t.cuda() for t in tables(64, 64, F32))
    at = torch.arange(23, device="cuda")
    want = ctx().rotary(before[:, :5].contiguous(), cos, sin, at)
    view = qkv[:, :5]
    assert ctx().rotary(view, cos, sin, at, out=view) is view
    ctx().flush()
    assert torch.equal(view, want) and torch.equal(qkv[:, 5], before[:, 5])


def test_rotary_unaligned_rows_give_the_same_bits():
    x = randn((9, 3, 128), 4, F16).cuda()
    cos, sin = (t.cuda() for t in tables(64, 64, F32))
    at = torch.arange(9, device="cuda")
    want = ctx().rotary(x, cos, sin, at)
    wide = torch.zeros((9, 3, 131), dtype=F16, device="cuda")
    wide[..., 1:129] = x
    got = ctx().rotary(wide[..., 1:129], cos, sin, at)
    assert ctx().last_kernel == "rotary_scalar"
    ctx().flush()
    assert torch.equal(got, want)


def test_rotary_position_outside_the_tables_writes_zeros_and_reports():
    x = randn((4, 2, 96), 5, F32).cuda()
    x[1] = math.inf
    cos, sin = (t.cuda() for t in tables(8, 32, F32))
    for at in (i32([[0, 8, 2, 7], [1, 1, 1, 1]]), i32([[0, 1, 2, 3], [5, -1, 2, 7]])):
        got = ctx().rotary(x, cos, sin, at, sections=[16, 16])
        with pytest.raises(ovk_b200.OvkError) as e:
            ctx().flush()
        assert e.value.status == ovk_b200.INVALID_ARGUMENT and "position" in e.value.message
        assert torch.equal(got[1], torch.zeros_like(got[1])) and bool((got[[0, 2, 3]] != 0).any())
    ctx().flush()


# -------------------------------------------------------------------- 4-bit cache
def place(cache, table, lens, new):
    """(page, head-row place) of each new token, in packed order."""
    out = []
    for b, n in enumerate(new):
        for i in range(n):
            p = lens[b] - n + i
            out.append((table[b][p // cache.page_size], p % cache.page_size))
    return out


def make_table(lens, page_size, seed, spare=2):
    per = [-(-n // page_size) for n in lens]
    order = np.random.default_rng(seed).permutation(sum(per) + spare)
    table = np.full((len(lens), max(max(per), 1)), -7, dtype=np.int32)  # entries behind a sequence are never read
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(per) + spare


def cache_rows(cache, which):
    blocks = cache.head_dim // cache.block_size
    code = ref.unpack(getattr(cache, which).cpu(), cache.head_dim)
    scale = getattr(cache, which + "_scales").cpu()
    zp = getattr(cache, which + "_zero_points")
    zero = torch.full(scale.shape, 8, dtype=torch.uint8) if zp is None else ref.unpack(zp.cpu(), blocks)
    return code, scale, zero


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,block,heads,page,zero_points", [
    (64, 32, 1, 16, True), (64, 64, 3, 5, True), (128, 32, 2, 16, True), (128, 64, 2, 1, False), (128, 128, 5, 7, True),
    (256, 32, 1, 64, False), (256, 64, 2, 16, True), (256, 128, 1, 9, True)])
def test_append(dtype, d, block, heads, page, zero_points):
    new, before = [3, 0, 1, 18], [4, 5, 0, 13]
    lens = [n + o for n, o in zip(new, before)]
    table, pages = make_table(lens, page, d + heads)
    cache = ctx().kv4_cache(pages, heads, page, d, block, zero_points)
    for t in cache.tensors:
        t.fill_(77)
    old = {w: [t.clone() for t in cache_rows(cache, w)] for w in ("k", "v")}
    # two rows behind the last sequence and one before the first
    k, v = (randn((sum(new) + 3, heads, d), s, F32, 1.0) for s in (1, 2))
    k[1, :, :block], k[2, :, 1:] = 0.0, 0.0
    k[3], v[4, 0, 5] = 30000.0, math.nan
    v[5, 0, 3], v[6, 0, 2], v[7], v[8] = math.inf, -math.inf, 1e-7, -3.0
    k[9, 0, :8] = torch.tensor([0.0, 0.5, 1.5, 2.5, 3.5, 4.5, 7.5, 15.0])  # ties
    k[9, 0, 8:] = 0.25
    k, v = k.to(dtype), v.to(dtype)
    ctx().kv4_append(cache, k.cuda(), v.cuda(), dev(table), starts(new, 1), i32(lens))
    ctx().flush()
    for which, x in (("k", k), ("v", v)):
        got = cache_rows(cache, which)
        want = ref.quantize(x[1:-2], block, zero_points)
        slots = place(cache, table, lens, new)
        for i, (p, o) in enumerate(slots):
            for a, b_, name in zip(got, want, ("codes", "scales", "zero points")):
                assert torch.equal(a[p, :, o], b_[i]), (which, name, i)
                old_rows = old[which][("codes", "scales", "zero points").index(name)]
                old_rows[p, :, o] = b_[i]
        for a, b_ in zip(got, old[which]):
            assert torch.equal(a, b_), "a row that no new token has was written"


def test_append_rounds_next_to_borders_as_the_definition():
    rng = np.random.default_rng(0)
    d, n = 128, 512
    x = rng.standard_normal((n, 1, d)).astype(np.float32)
    s = (x.max(-1, keepdims=True).clip(0) - x.min(-1, keepdims=True).clip(max=0)) / 15
    s = s.astype(np.float16).astype(np.float32)
    lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    near = (np.rint(x / s) + 0.5).astype(np.float32) * s  # quotients on a border, one step below and one above it
    near = np.nextafter(near, rng.choice([-np.inf, np.inf], near.shape).astype(np.float32)) * 1.0
    y = np.where((near < hi) & (near > lo) & (x != hi) & (x != lo) & (rng.random(x.shape) < 0.7), near, x).astype(np.float32)
    k = torch.from_numpy(y)
    cache = ctx().kv4_cache(1, 1, n, d, 128)
    ctx().kv4_append(cache, k.cuda(), k.cuda(), i32([[0]]), i32([0, n]), i32([n]))
    ctx().flush()
    code, scale, zero = cache_rows(cache, "v")
    want = ref.quantize(k, 128, True)
    assert torch.equal(scale[0, 0], want[1][:, 0]) and torch.equal(zero[0, 0], want[2][:, 0]) and torch.equal(code[0, 0], want[0][:, 0])


def test_append_and_gather_block_quantized_agree_on_the_row_layout():
    cache = ctx().kv4_cache(3, 2, 8, 128, 32)
    k, v = randn((20, 2, 128), 1, F16), randn((20, 2, 128), 2, F16)
    ctx().kv4_append(cache, k.cuda(), v.cuda(), i32([[2, 0, 1]]), i32([0, 20]), i32([20]))
    rows = torch.tensor([[((2, 0, 1)[t // 8] * 2 + h) * 8 + t % 8 for h in range(2)] for t in range(20)], device="cuda")
    got = ctx().gather_block_quantized(cache.v.flatten(0, 2), rows, cache.v_scales, cache.v_zero_points, 32, out_dtype=F32)
    ctx().flush()
    assert torch.equal(got.cpu().double(), ref.dequantize(*ref.quantize(v, 32, True)))


@pytest.mark.parametrize("lens,table", [([17], [[0, 1]]), ([-1], [[0, 1]]), ([1], [[0, 1]]), ([16], [[0, 2]]), ([16], [[0, -1]])])
def test_append_outside_the_cache_is_left_out_and_reported(lens, table):
    cache = ctx().kv4_cache(2, 1, 8, 64, 32)
    k = torch.ones((3, 1, 64), dtype=F16, device="cuda")
    ctx().kv4_append(cache, k, k, i32(table), i32([0, 3]), i32(lens))
    with pytest.raises(ovk_b200.OvkError) as e:
        ctx().flush()
    assert e.value.status == ovk_b200.INVALID_ARGUMENT and "page" in e.value.message
    rows = int((cache.k_scales != 0).any(-1).sum())
    assert rows == {17: 2, -1: 0, 1: 1, 16: 0}[lens[0]]
    ctx().flush()


# ------------------------------------------------------------- attention over it
def filled_cache(lens, heads, d, block, page, zero_points, seed, spread=1.0):
    table, pages = make_table(lens, page, seed)
    cache = ctx().kv4_cache(pages, heads, page, d, block, zero_points)
    total = sum(lens)
    k, v = randn((max(total, 1), heads, d), seed, F32, spread), randn((max(total, 1), heads, d), seed + 1, F32)
    # one channel of outliers, as keys have
    k[..., 3] *= 4
    if total:
        ctx().kv4_append(cache, k[:total].cuda(), v[:total].cuda(), dev(table), starts(lens), i32(lens))
    ctx().flush()
    return cache, table


def check_kv4(cache, table, q, new, lens, scale, window, got, first=0):
    rows = {w: ref.dequantize(*cache_rows(cache, w)) for w in ("k", "v")}
    sizes = ref.row_sizes(*cache_rows(cache, "k"))
    group = q.shape[1] // cache.kv_heads
    f32 = q.dtype == F32
    # weights enter the second product as one fp16 number (f16) or two (f32: 2^-22)
    p_error, q_error = (2.0 ** -21, 2.0 ** -21) if f32 else (2.0 ** -11, 0.0)
    at = first
    for b, n in enumerate(new):
        tokens = np.arange(lens[b])
        page = torch.as_tensor(table[b][tokens // cache.page_size].astype(np.int64))
        for h in range(q.shape[1]):
            k, v = (rows[w][page, h // group, torch.as_tensor(tokens % cache.page_size)] for w in ("k", "v"))
            k_size = sizes[page, h // group, torch.as_tensor(tokens % cache.page_size)]
            m = min(n, lens[b])  # new tokens beyond the cache's length have no position
            want, bound = ref.attend(q[at + n - m:at + n, h].double().cpu(), k, v, scale, True, window, p_error, q_error, k_size)
            assert torch.equal(got[at:at + n - m, h], torch.zeros_like(got[at:at + n - m, h]))
            ref.check(got[at + n - m:at + n, h], want, bound, f"sequence {b} head {h}")
        at += n


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,block,hq,hk,page,zero_points,new,lens,window", [
    (128, 32, 8, 1, 16, True, [1], [1], 0),
    (128, 32, 8, 1, 16, True, [1], [700], 0),
    (128, 32, 16, 2, 16, True, [1, 1, 1], [5, 64, 331], 0),
    (128, 64, 4, 4, 48, False, [1, 1], [129, 1], 0),
    (128, 128, 7, 1, 1, True, [1, 1], [40, 65], 0),
    (64, 32, 6, 2, 64, True, [1, 0, 1], [100, 3, 17], 0),
    (64, 64, 3, 3, 7, True, [2, 3], [2, 50], 0),
    (256, 32, 4, 1, 16, True, [1], [900], 512),
    (256, 64, 4, 2, 100, False, [1, 1], [333, 90], 33),
    (256, 128, 8, 1, 16, True, [5, 1], [77, 4], 16),
    (128, 32, 12, 1, 16, True, [1, 1], [77, 4], 0),       # more than eight heads a group
    (128, 32, 8, 2, 16, True, [5, 2, 9], [77, 2, 40], 0),  # drafts: several tiles of rows
    (64, 32, 20, 1, 16, True, [4], [70], 20),
    (128, 32, 2, 1, 16, True, [0, 1, 3], [4, 0, 1], 0),    # nothing in the cache; more new tokens than it holds
])
def test_attention_kv4(dtype, d, block, hq, hk, page, zero_points, new, lens, window):
    cache, table = filled_cache(lens, hk, d, block, page, zero_points, d + hq)
    n = sum(new)
    q = randn((n + 3, hq, d), 9, F32, 1.5).to(dtype)
    out = torch.full((n + 3, hq, d), 7.0, dtype=dtype, device="cuda")
    got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts(new, 1), i32(lens), max_tokens=max(new), window=window, out=out)
    ctx().flush()
    assert bool((got[0] == 7).all()) and bool((got[n + 1:] == 7).all()), "rows outside the sequences were written"
    check_kv4(cache, table, q, new, lens, d ** -0.5, window, got.cpu(), 1)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attention_kv4_split_over_many_blocks(dtype):
    """One long sequence and a few short ones: items that begin and end inside a block's run."""
    lens = [20011, 1, 63, 64, 65, 3000]
    cache, table = filled_cache(lens, 1, 128, 32, 64, True, 5)
    q = randn((6, 2, 128), 9, F32, 1.5).to(dtype)
    got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts([1] * 6), i32(lens))
    again = ctx().attention_kv4(cache, q.cuda(), dev(table), starts([1] * 6), i32(lens))
    ctx().flush()
    assert torch.equal(got, again)
    check_kv4(cache, table, q, [1] * 6, lens, 128 ** -0.5, 0, got.cpu())


def test_attention_kv4_many_sequences():
    """More sequences than a block has threads, many of them without a new token."""
    rng = np.random.default_rng(3)
    lens = [int(v) for v in rng.integers(0, 40, 300)]
    new = [int(v) for v in rng.integers(0, 2, 300)]
    cache, table = filled_cache(lens, 1, 64, 32, 8, True, 6)
    q = randn((sum(new), 2, 64), 9, F16, 1.5)
    got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts(new), i32(lens))
    ctx().flush()
    check_kv4(cache, table, q, new, lens, 64 ** -0.5, 0, got.cpu())


def test_attention_kv4_far_more_sequences_than_threads():
    """The shares of the work are found by a scan over the batch that takes several passes."""
    rng = np.random.default_rng(4)
    lens = [int(v) for v in rng.integers(0, 9, 1100)]
    lens[700], new = 3000, [int(v) for v in rng.integers(0, 2, 1100)]
    new[700] = 1
    cache, table = filled_cache(lens, 1, 64, 64, 8, True, 7)
    q = randn((sum(new), 2, 64), 9, F16, 1.5)
    got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts(new), i32(lens))
    ctx().flush()
    check_kv4(cache, table, q, new, lens, 64 ** -0.5, 0, got.cpu())


def test_cache_offsets_beyond_32_bits():
    """Pages at the end of a cache whose codes, and scales, lie more than 2^32 bytes from their tensors' starts."""
    page, d, pages = 64, 128, 8_600_000 // 8 + 10  # 68.8 million rows: codes of 4.4 GB each
    make = lambda last, dtype: torch.empty((pages, 1, page, last), dtype=dtype, device="cuda")  # noqa: E731
    cache = ovk_b200.KV4Cache(make(64, torch.uint8), make(64, torch.uint8), make(4, F16), make(4, F16), make(2, torch.uint8), make(2, torch.uint8))
    assert cache.k.numel() > 2 ** 32
    lens, table = [150], np.array([[pages - 1, 3, pages - 2]], dtype=np.int32)
    k, v, q = randn((150, 1, d), 1, F16), randn((150, 1, d), 2, F16), randn((1, 8, d), 3, F16)
    ctx().kv4_append(cache, k.cuda(), v.cuda(), dev(table), starts(lens), i32(lens))
    got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts([1]), i32(lens))
    ctx().flush()
    rows = {w: ref.dequantize(*ref.quantize(x, 32, True))[:, 0] for w, x in (("k", k), ("v", v))}
    sizes = ref.row_sizes(*ref.quantize(k, 32, True))[:, 0]
    for h in range(8):
        want, bound = ref.attend(q[:, h].double(), rows["k"], rows["v"], d ** -0.5, True, 0, 2.0 ** -11, 0.0, sizes)
        ref.check(got[:, h], want, bound, f"head {h}")


def test_attention_kv4_without_pages_or_sequences():
    q = randn((2, 4, 128), 1, F16).cuda()
    cache = ctx().kv4_cache(0, 2, 16, 128)
    none = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    got = ctx().attention_kv4(cache, q, none, i32([0, 1, 2]), i32([0, 0]), out=torch.full_like(q, 3.0))
    ctx().flush()
    assert bool((got == 0).all())
    got = ctx().attention_kv4(cache, q, torch.zeros((0, 4), dtype=torch.int32, device="cuda"), i32([0]), i32([]), out=torch.full_like(q, 3.0))
    ctx().flush()
    assert bool((got == 3).all())
    assert ctx().attention_kv4(cache, q[:0], none, i32([0, 0, 0]), i32([0, 0])).shape == (0, 4, 128)
    ctx().kv4_append(cache, q[:0, :2], q[:0, :2], none, i32([0, 0, 0]), i32([0, 0]))
    ctx().flush()


@pytest.mark.parametrize("scale", [0.0, -0.11, 3.0])
def test_scales_of_any_sign(scale):
    cache, table = filled_cache([70], 1, 128, 32, 16, True, 3)
    q = randn((1, 4, 128), 1, F16)
    got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts([1]), i32([70]), scale=scale)
    ctx().flush()
    check_kv4(cache, table, q, [1], [70], scale, 0, got.cpu())
    q, k, v = (randn((140, 2, 128), s, F16) for s in (1, 2, 3))
    got = ctx().attention_prompt(q.cuda(), k.cuda(), v.cuda(), starts([140]), scale=scale)
    ctx().flush()
    check_prompt(q, k, v, [0, 140], [0, 140], scale, True, 0, got.cpu(), False)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attention_kv4_extreme_queries_and_scales(dtype):
    lens = [90]
    table, pages = make_table(lens, 16, 1)
    cache = ctx().kv4_cache(pages, 1, 16, 128, 32)
    k, v = randn((90, 1, 128), 1), randn((90, 1, 128), 2)
    v[:30] *= 1e-3
    v[60:] *= 300.0  # later tokens' scales pass the earlier ones' by far
    ctx().kv4_append(cache, k.cuda(), v.cuda(), dev(table), starts(lens), i32(lens))
    q = randn((1, 4, 128), 3)
    q[0, 1] *= 30.0
    q[0, 2] *= 1e-6
    q[0, 3] = 0.0
    if dtype == F32:
        q[0, 2] *= 1e-30
    q = q.to(dtype)
    got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts([1]), i32(lens))
    ctx().flush()
    check_kv4(cache, table, q, [1], lens, 128 ** -0.5, 0, got.cpu())


def test_attention_kv4_scales_that_are_not_finite_reach_only_rows_that_read_them():
    lens, new = [40], [3]
    cache, table = filled_cache(lens, 1, 128, 32, 16, True, 7)
    page, at = int(table[0][39 // 16]), 39 % 16
    cache.v_scales[page, 0, at] = math.inf
    cache.k_scales[page, 0, at] = math.nan
    q = randn((3, 4, 128), 3, F16)
    got = ctx().attention_kv4(cache, q.cuda(), dev(table), starts(new), i32(lens), max_tokens=3)
    ctx().flush()
    assert bool(torch.isfinite(got[:2]).all()) and bool(torch.isnan(got[2]).all())


@pytest.mark.parametrize("lens,table,cu,word", [([17], [[0, 1]], [0, 1], "page"), ([-3], [[0, 1]], [0, 1], "page"),
                                                ([5], [[0, 1]], [0, 9], "bounds"), ([5], [[0, 1]], [-1, 1], "bounds")])
def test_attention_kv4_outside_the_cache_gives_zeros_and_reports(lens, table, cu, word):
    cache, _ = filled_cache([16], 1, 64, 32, 8, True, 8)
    q = randn((2, 2, 64), 1, F16).cuda()
    got = ctx().attention_kv4(cache, q, i32(table), i32(cu), i32(lens), out=torch.full_like(q, 3.0))
    with pytest.raises(ovk_b200.OvkError) as e:
        ctx().flush()
    assert e.value.status == ovk_b200.INVALID_ARGUMENT and word in e.value.message
    if word == "page":
        assert bool((got[0] == 0).all()) and bool((got[1] == 3).all())
    else:
        assert bool((got == 3).all())
    ctx().flush()


def test_attention_kv4_bad_page_is_left_out():
    cache, table = filled_cache([24], 1, 64, 32, 8, True, 9)
    q = randn((1, 2, 64), 1, F16)
    bad = table.copy()
    bad[0, 1] = 99
    got = ctx().attention_kv4(cache, q.cuda(), dev(bad), i32([0, 1]), i32([24]))
    with pytest.raises(ovk_b200.OvkError):
        ctx().flush()
    rows = {w: ref.dequantize(*cache_rows(cache, w)) for w in ("k", "v")}
    keep = [t for t in range(24) if t // 8 != 1]
    k, v = (torch.stack([rows[w][table[0][t // 8], 0, t % 8] for t in keep]) for w in ("k", "v"))
    sizes = ref.row_sizes(*cache_rows(cache, "k"))
    k_size = torch.stack([sizes[table[0][t // 8], 0, t % 8] for t in keep])
    for h in range(2):
        want, bound = ref.attend(q[:, h].double(), k, v, 64 ** -0.5, False, 0, 2.0 ** -11, 0.0, k_size)
        ref.check(got[:, h], want, bound, "bad page")


# ---------------------------------------------------------------------- prompts
def check_prompt(q, k, v, cu_q, cu_k, scale, causal, window, got, exact_weights):
    group = q.shape[1] // k.shape[1]
    p_error = 2.0 ** -23 if exact_weights else 2.0 ** -11
    for b in range(len(cu_q) - 1):
        for h in range(q.shape[1]):
            rows, keys = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
            qs, n = q[rows, h].double(), cu_q[b + 1] - cu_q[b]
            ks, vs = k[keys, h // group].double(), v[keys, h // group].double()
            m = min(n, ks.shape[0])  # rows that come before every key
            if causal and m < n:
                assert torch.equal(got[rows, h][:n - m], torch.zeros(n - m, q.shape[2], dtype=got.dtype))
                want, bound = ref.attend(qs[n - m:], ks, vs, scale, causal, window, p_error)
                ref.check(got[rows, h][n - m:], want, bound, f"sequence {b} head {h}")
            elif m < n:  # without a causal mask every row reads what its window leaves
                for i in range(n):
                    at = ks.shape[0] - n + i
                    lo = max(0, at - window + 1) if window else 0
                    want, bound = ref.attend(qs[i:i + 1], ks[lo:], vs[lo:], scale, False, 0, p_error)
                    ref.check(got[rows, h][i:i + 1], want, bound, f"sequence {b} head {h} row {i}")
            else:
                want, bound = ref.attend(qs, ks, vs, scale, causal, window, p_error)
                ref.check(got[rows, h], want, bound, f"sequence {b} head {h}")


PROMPTS = [
    (64, 2, 1, [1], None, True, 0),
    (128, 2, 2, [64], None, True, 0),
    (128, 4, 1, [130, 0, 1, 257], None, True, 0),
    (128, 2, 1, [70, 200], None, False, 0),
    (256, 2, 1, [300, 65], None, True, 100),
    (256, 2, 1, [129], None, False, 0),
    (64, 3, 3, [20, 129, 5], [100, 400, 5], True, 0),
    (64, 2, 1, [128, 60], [384, 61], False, 50),
    (80, 2, 1, [140], None, True, 0),
    (33, 2, 1, [70], None, True, 0),
    (128, 3, 1, [9, 140, 3], [4, 100, 0], True, 0),   # rows without keys
    (128, 1, 1, [9, 3], [4, 0], False, 2),
    (200, 2, 1, [260], None, True, 1),                # every row reads itself
    (128, 2, 1, [513], None, True, 128),
    (16, 2, 1, [150], None, True, 0),
    (1, 1, 1, [5], None, True, 0),
]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,hq,hk,new,seen,causal,window", PROMPTS)
def test_attention_prompt(dtype, d, hq, hk, new, seen, causal, window):
    seen = new if seen is None else seen
    tq, tk = sum(new) + 3, sum(seen) + 4
    q, k, v = randn((tq, hq, d), 1, F32, 1.5).to(dtype), randn((tk, hk, d), 2, dtype), randn((tk, hk, d), 3, dtype)
    # rows outside every sequence hold what an uninitialised buffer may hold
    q[0], q[-2:], k[:2], k[-2:], v[:2], v[-2:] = math.nan, math.inf, math.nan, math.inf, math.nan, math.inf
    out = torch.full((tq, hq, d), 7.0, dtype=dtype, device="cuda")
    got = ctx().attention_prompt(q.cuda(), k.cuda(), v.cuda(), starts(new, 1), max(new), cu_k=starts(seen, 2), causal=causal, window=window,
                                 out=out)
    ctx().flush()
    got = got.cpu()
    assert bool((got[0] == 7).all()) and bool((got[-2:] == 7).all()), "rows outside the sequences were written"
    cu = lambda lens, first: [first + sum(lens[:i]) for i in range(len(lens) + 1)]  # noqa: E731
    check_prompt(q, k, v, cu(new, 1), cu(seen, 2), d ** -0.5, causal, window, got, dtype == F32)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,n,window", [(128, 200, 0), (256, 150, 0), (64, 300, 70)])
def test_attention_prompt_infinities_reach_only_rows_that_read_them(dtype, d, n, window):
    q, k, v = (randn((n, 2, d), s, dtype) for s in (1, 2, 3))
    at = n - 40
    k[at], v[at, :, 5], v[at + 1, :, 6] = math.nan, math.inf, math.nan
    got = ctx().attention_prompt(q.cuda(), k.cuda(), v.cuda(), starts([n]), n, window=window)
    ctx().flush()
    got = got.cpu()
    assert bool(torch.isfinite(got[:at]).all()) and bool(torch.isnan(got[at]).all())
    last = n if window == 0 else min(n, at + window)
    assert bool(torch.isnan(got[at:last]).all())
    clean_k, clean_v = k.clone(), v.clone()
    clean_k[at:], clean_v[at:] = 0, 0
    check_prompt(q[:at], clean_k[:at], clean_v[:at], [0, at], [0, at], d ** -0.5, True, window, got, dtype == F32)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attention_prompt_on_slices_of_a_fused_product(dtype):
    qkv = randn((2, 150, 8, 128), 1, dtype).cuda()[1]  # [tokens, 4 query + 2 key + 2 value heads, 128]
    cu = starts([60, 90])
    got = ctx().attention_prompt(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], cu, 90)
    want = ctx().attention_prompt(qkv[:, :4].contiguous(), qkv[:, 4:6].contiguous(), qkv[:, 6:].contiguous(), cu, 90)
    heads_first = torch.empty((4, 150, 128), dtype=dtype, device="cuda")
    ctx().attention_prompt(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], cu, 90, out=heads_first.transpose(0, 1))
    ctx().flush()
    assert torch.equal(got, want) and torch.equal(heads_first.transpose(0, 1), want)


def test_attention_prompt_large_scores_and_lowest_values():
    """Scores far apart and far from zero: the running maximum moves by thousands."""
    q, k, v = (randn((300, 1, 128), s, F16) for s in (1, 2, 3))
    q *= 20
    k[::7] = -k[::7] * 8
    got = ctx().attention_prompt(q.cuda(), k.cuda(), v.cuda(), starts([300]), 300)
    ctx().flush()
    check_prompt(q, k, v, [0, 300], [0, 300], 128 ** -0.5, True, 0, got.cpu(), False)
    lowest = torch.full((130, 1, 64), torch.finfo(F16).min, dtype=F16)
    got = ctx().attention_prompt(lowest.cuda(), lowest.cuda(), randn((130, 1, 64), 3, F16).cuda(), starts([130]), 130)
    ctx().flush()
    assert bool(torch.isfinite(got).all())


def test_attention_prompt_longer_than_promised_is_left_out_and_reported():
    q, k = randn((300, 2, 64), 1, F16).cuda(), randn((300, 1, 64), 2, F16).cuda()
    out = ctx().attention_prompt(q, k, k, i32([0, 100, 300]), 150, out=torch.full_like(q, 3.0))
    with pytest.raises(ovk_b200.OvkError) as e:
        ctx().flush()
    assert "bounds" in e.value.message and bool((out[100:] == 3).all()) and bool((out[:100] != 3).all())
    want = ctx().attention_prompt(q, k, k, i32([0, 100, 300]))
    assert torch.equal(ctx().attention_prompt(q, k, k, i32([0, 100, 300]), 200), want)
    ctx().flush()


def test_attention_prompt_broadcast_keys_and_no_keys():
    q, k = randn((90, 4, 128), 1, F16).cuda(), randn((90, 1, 128), 2, F16).cuda()
    wide = k.expand(90, 2, 128)  # one head's rows under two names
    got = ctx().attention_prompt(q, wide, wide, starts([90]))
    want = ctx().attention_prompt(q, wide.contiguous(), wide.contiguous(), starts([90]))
    none = ctx().attention_prompt(q, k[:0], k[:0], starts([90]), cu_k=i32([0, 0]), out=torch.full_like(q, 3.0))
    ctx().flush()
    assert bool((none == 0).all())
    # the two calls take different kernels: both are within half a step and the weights' rounding of the exact result
    assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -10 * float(k.float().abs().max())


def test_attention_prompt_bad_bounds_are_left_out_and_reported():
    q, k = randn((20, 2, 64), 1, F16).cuda(), randn((20, 1, 64), 2, F16).cuda()
    for cu_q, cu_k, zeros in (([0, 10, 25], [0, 10, 20], False), ([0, 10, 20], [0, 10, 21], True), ([0, 10, 5], [0, 10, 20], False),
                              ([0, 10, 20], [0, 10, 8], True)):
        out = ctx().attention_prompt(q, k, k, i32(cu_q), 20, cu_k=i32(cu_k), out=torch.full_like(q, 3.0))
        with pytest.raises(ovk_b200.OvkError) as e:
            ctx().flush()
        assert e.value.status == ovk_b200.INVALID_ARGUMENT and "bounds" in e.value.message
        assert bool((out[10:] == (0 if zeros else 3)).all()) and bool((out[:10] != 3).all())
    ctx().flush()


# ------------------------------------------------------- together, streams, graphs
def layer(c, state, step):
    """Rotary, cache write and attention of one decoder layer for packed new tokens."""
    q, k = c.rotary(step["q"], state["cos"], state["sin"], step["positions"], k=step["k"], sections=[16, 24, 24])
    c.kv4_append(state["cache"], k, step["v"], state["table"], step["cu"], step["lens"])
    if step["prompt"]:
        return c.attention_prompt(q, k, step["v"], step["cu"], step["longest"])
    return c.attention_kv4(state["cache"], q, state["table"], step["cu"], step["lens"])


def make_steps(prompt, decode, hq, hk, d, dtype):
    steps, lens = [], [0] * len(prompt)
    for i in range(decode + 1):
        new = prompt if i == 0 else [1] * len(prompt)
        lens = [a + b for a, b in zip(lens, new)]
        n = sum(new)
        at = torch.cat([torch.arange(b - a, b) for a, b in zip(new, lens)])
        steps.append({"q": randn((n, hq, d), 10 * i, dtype).cuda(), "k": randn((n, hk, d), 10 * i + 1, dtype).cuda(),
                      "v": randn((n, hk, d), 10 * i + 2, dtype).cuda(), "positions": torch.stack([at, at // 2, at % 5]).cuda(),
                      "cu": starts(new), "lens": i32(lens), "longest": max(new), "prompt": i == 0, "new": new, "all": list(lens)})
    return steps


def make_state(c, prompt, decode, hk, d):
    lens = [n + decode for n in prompt]
    table, pages = make_table(lens, 16, 1)
    cos, sin = tables(4096, d // 2, F32)
    return {"cache": c.kv4_cache(pages, hk, 16, d, 32), "table": dev(np.maximum(table, 0)), "cos": cos.cuda(), "sin": sin.cuda()}


@pytest.mark.parametrize("dtype", [F16, F32])
def test_a_prompt_and_decode_steps_of_a_layer(dtype):
    prompt, hq, hk, d = [37, 5, 130], 16, 2, 128
    state, steps = make_state(ctx(), prompt, 3, hk, d), make_steps(prompt, 3, hq, hk, d, dtype)
    table = state["table"].cpu().numpy()
    for step in steps:
        got = layer(ctx(), state, step)
        q, k = ctx().rotary(step["q"], state["cos"], state["sin"], step["positions"], k=step["k"], sections=[16, 24, 24])
        ctx().flush()
        cu = step["cu"].tolist()
        if step["prompt"]:
            check_prompt(q.cpu(), k.cpu(), step["v"].cpu(), cu, cu, d ** -0.5, True, 0, got.cpu(), dtype == F32)
        else:
            check_kv4(state["cache"], table, q.cpu(), step["new"], step["all"], d ** -0.5, 0, got.cpu())


def test_captured_replayed_and_on_a_stream_of_its_own():
    prompt, hq, hk, d = [37, 5, 130], 16, 2, 128
    steps = make_steps(prompt, 1, hq, hk, d, F16)
    state = make_state(ctx(), prompt, 1, hk, d)
    want = [layer(ctx(), state, s).clone() for s in steps]
    ctx().flush()
    stream = torch.cuda.Stream()
    own = ovk_b200.Context(0, stream.cuda_stream)
    state2 = make_state(own, prompt, 1, hk, d)
    torch.cuda.synchronize()
    eager = [layer(own, state2, s) for s in steps]  # called under another current stream
    own.flush()
    assert all(torch.equal(a, b) for a, b in zip(eager, want))
    graphs, outs = [], []
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(layer(own, state2, s))
        graphs.append(g)
    for t in state2["cache"].tensors:
        t.zero_()
    for _ in range(3):
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    del graphs, outs
    own.close()


def test_two_contexts_at_once_do_not_share_results():
    lens = [5000]
    cache, table = filled_cache(lens, 2, 128, 32, 64, True, 3)
    q = [randn((1, 16, 128), s, F16).cuda() for s in (1, 2)]
    t, cu, n = dev(table), starts([1]), i32(lens)
    want = [ctx().attention_kv4(cache, x, t, cu, n).clone() for x in q]
    ctx().flush()
    streams = [torch.cuda.Stream() for _ in q]
    cs = [ovk_b200.Context(0, s.cuda_stream) for s in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        got = [c.attention_kv4(cache, x, t, cu, n) for c, x in zip(cs, q)]
        for c in cs:
            c.flush()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for c in cs:
        c.close()


# ------------------------------------------------------------- rows as they are stored
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,hq,hk,lens,window", [(64, 2, 1, [130, 5], 0), (80, 3, 3, [129, 257], 0), (128, 4, 2, [1, 200], 0), (200, 2, 1, [140], 64),
                                                 (256, 1, 1, [129, 127], 0), (8, 2, 2, [131], 0)])
def test_attention_prompt_results_at_any_alignment_have_the_same_bits(dtype, d, hq, hk, lens, window):
    n = sum(lens)
    q, k, v = (randn((n, h, d), s, dtype).cuda() for s, h in ((1, hq), (2, hk), (3, hk)))
    want = ctx().attention_prompt(q, k, v, starts(lens), max(lens), window=window)
    buffer = torch.full((n * hq * (d + 2) + 9,), 7.0, dtype=dtype, device="cuda")
    out = buffer[1:1 + n * hq * (d + 2)].view(n, hq, d + 2)[..., :d]  # odd start, a gap of two elements behind each row
    ctx().attention_prompt(q, k, v, starts(lens), max(lens), window=window, out=out)
    ctx().flush()
    assert torch.equal(out, want)
    assert int((buffer == 7).sum()) >= buffer.numel() - n * hq * d, "elements between the rows were written"
    assert bool((buffer[1:1 + n * hq * (d + 2)].view(n, hq, d + 2)[..., d:] == 7).all()) and bool((buffer[-8:] == 7).all())


@pytest.mark.parametrize("zero_points", [True, False])
def test_append_of_the_largest_values_and_many_heads(zero_points):
    top = torch.finfo(F32).max
    lens, heads = [5, 2], 300
    k = randn((7, heads, 64), 1, F32)
    v = randn((7, heads, 64), 2, F32)
    k[0, 0, 1], k[0, 0, 2], k[0, 1, 3], v[1, 2, 3] = top, -top, -top, top
    v[2, 299] = torch.linspace(-1e-8, 1e-8, 64)
    v[3, 298, :32] = 65504.0 * 15
    v[3, 297, :32] = -65504.0 * 15.5
    cache = ctx().kv4_cache(4, heads, 3, 64, 32, zero_points)
    table = [[2, 0], [3, 1]]
    ctx().kv4_append(cache, k.cuda(), v.cuda(), i32(table), starts(lens), i32(lens))
    ctx().flush()
    for which, x in (("k", k), ("v", v)):
        got, want = cache_rows(cache, which), ref.quantize(x, 32, zero_points)
        for i, (p, o) in enumerate(place(cache, table, lens, lens)):
            for a, b, name in zip(got, want, ("codes", "scales", "zero points")):
                assert torch.equal(a[p, :, o], b[i]), (which, name, i)

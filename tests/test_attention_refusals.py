"""What the attention operators refuse, through the C ABI without a context: every check of a call's arguments comes before
anything touches a GPU, and a call whose arguments pass gets no further than the missing context."""
import ctypes as C

import pytest

import ovk_b200
from ovk_b200 import FLOAT, FLOAT16, INT32, INT64, INVALID_ARGUMENT, UNSUPPORTED, Heads, KV4Batch, KV4CacheParams, PromptParams, RotaryParams

BASE = 1 << 20  # an address that no call reads: a refused call dereferences nothing


def outcome(rc):
    return rc, ovk_b200.lib().ovk_last_error(None).decode()


def heads(n=2, d=64, at=BASE, token=None, head=None):
    return Heads(at, n, n * d if token is None else token, d if head is None else head)


def rotary(x=None, out=None, count=1, at=BASE, cos=BASE, sin=BASE, **changes):
    fields = dict(tokens=5, head_dim=64, rotary_dim=64, max_position=100, dtype=FLOAT16, table_dtype=FLOAT, positions_dtype=INT64,
                  interleaved=0, axes=1, sections=(32,)) | changes
    fields["sections"] = (C.c_int32 * 4)(*fields["sections"])
    x = x or heads()
    out = out or heads(at=2 * BASE)
    return outcome(ovk_b200.lib().ovk_rotary(None, RotaryParams(**fields), count, (Heads * 2)(x, x), (Heads * 2)(out, out), at, cos, sin))


@pytest.mark.parametrize("changes,status,word", [
    ({}, INVALID_ARGUMENT, "null context"),
    ({"x": heads(at=2 * BASE)}, INVALID_ARGUMENT, "null context"),                    # in place
    ({"dtype": INT32}, UNSUPPORTED, "dtype"),
    ({"table_dtype": 16}, UNSUPPORTED, "table dtype"),
    ({"positions_dtype": FLOAT}, INVALID_ARGUMENT, "position dtype"),
    ({"tokens": -1}, INVALID_ARGUMENT, "tokens"),
    ({"rotary_dim": 63}, INVALID_ARGUMENT, "rotary_dim"),
    ({"rotary_dim": 66, "sections": (33,)}, INVALID_ARGUMENT, "rotary_dim"),
    ({"axes": 5}, INVALID_ARGUMENT, "axes"),
    ({"axes": 0}, INVALID_ARGUMENT, "axes"),
    ({"sections": (31,)}, INVALID_ARGUMENT, "sections"),
    ({"axes": 2, "sections": (40, -8)}, INVALID_ARGUMENT, "section"),
    ({"max_position": 0}, INVALID_ARGUMENT, "positions"),
    ({"count": 3}, INVALID_ARGUMENT, "tensors"),
    ({"at": None}, INVALID_ARGUMENT, "null positions"),
    ({"at": BASE + 4}, INVALID_ARGUMENT, "misaligned"),
    ({"cos": None}, INVALID_ARGUMENT, "null positions or tables"),
    ({"x": heads(at=None)}, INVALID_ARGUMENT, "no data"),
    ({"x": heads(at=BASE + 1)}, INVALID_ARGUMENT, "aligned"),
    ({"x": heads(n=3)}, INVALID_ARGUMENT, "heads"),
    ({"x": heads(token=-128)}, INVALID_ARGUMENT, "strides"),
    ({"out": heads(at=2 * BASE, token=64)}, INVALID_ARGUMENT, "overlap"),
    ({"out": heads(at=2 * BASE, head=0)}, INVALID_ARGUMENT, "overlap"),
    ({"x": heads(at=2 * BASE, token=256)}, INVALID_ARGUMENT, "in place"),
])
def test_rotary(changes, status, word):
    rc, message = rotary(**changes)
    assert rc == status and word in message, message


def cache(**changes):
    fields = dict(k=BASE, v=BASE, k_scales=BASE, v_scales=BASE, k_zero_points=BASE, v_zero_points=BASE, pages=10, kv_heads=2,
                  page_size=16, head_dim=128, block_size=32) | changes
    return KV4CacheParams(**fields)


def batch(**changes):
    return KV4Batch(**(dict(tokens=3, batch=3, max_pages=4, cu_tokens=BASE, lens=BASE, block_table=BASE) | changes))


BAD_CACHES = [
    ({"head_dim": 96}, UNSUPPORTED, "head_dim"), ({"block_size": 16}, UNSUPPORTED, "block_size"),
    ({"head_dim": 64, "block_size": 128}, INVALID_ARGUMENT, "divide"), ({"page_size": 0}, INVALID_ARGUMENT, "pages"),
    ({"pages": 1 << 27}, INVALID_ARGUMENT, "rows"), ({"pages": -1}, INVALID_ARGUMENT, "pages"),
    ({"pages": (1 << 31) - 1, "kv_heads": 1 << 16, "page_size": (1 << 31) - 1}, INVALID_ARGUMENT, "rows"),
    ({"k": None}, INVALID_ARGUMENT, "no data"), ({"v_scales": None}, INVALID_ARGUMENT, "no data"),
    ({"k_zero_points": None}, INVALID_ARGUMENT, "zero points"), ({"v": BASE + 8}, INVALID_ARGUMENT, "16-byte"),
]
BAD_BATCHES = [
    ({"tokens": -1}, "tokens"), ({"batch": -1}, "sequences"), ({"max_pages": 1 << 31}, "pages"), ({"cu_tokens": None}, "null"),
    ({"lens": None}, "null"), ({"block_table": None}, "null"), ({"lens": BASE + 2}, "misaligned"),
]


def append(c=None, b=None, k=None, v=None, dtype=FLOAT16):
    k, v = k or heads(2, 128), v or heads(2, 128)
    return outcome(ovk_b200.lib().ovk_kv4_append(None, c or cache(), b or batch(), k, v, dtype))


def attention(c=None, b=None, q=None, out=None, dtype=FLOAT16, max_tokens=1, scale=0.1, window=0, space=None, size=0):
    q, out = q or heads(8, 128), out or heads(8, 128, 2 * BASE)
    return outcome(ovk_b200.lib().ovk_attention_kv4(None, c or cache(), b or batch(), q, out, dtype, max_tokens, scale, window, space, size))


def workspace(c=None, heads=8, max_tokens=1, dtype=FLOAT16):
    n = C.c_size_t()
    return outcome(ovk_b200.lib().ovk_attention_kv4_workspace(None, c or cache(), heads, max_tokens, dtype, C.byref(n)))


@pytest.mark.parametrize("changes,status,word", [({}, INVALID_ARGUMENT, "null context")] + BAD_CACHES)
def test_caches(changes, status, word):
    for call in (append, attention, workspace):
        rc, message = call(c=cache(**changes))
        assert rc == status and word in message, message


@pytest.mark.parametrize("changes,word", BAD_BATCHES)
def test_batches(changes, word):
    for call in (append, attention):
        rc, message = call(b=batch(**changes))
        assert rc == INVALID_ARGUMENT and word in message, message


@pytest.mark.parametrize("changes,status,word", [
    ({"dtype": 16}, UNSUPPORTED, "dtype"), ({"k": heads(3, 128)}, INVALID_ARGUMENT, "heads"), ({"v": heads(1, 128)}, INVALID_ARGUMENT, "heads"),
    ({"v": heads(2, 128, None)}, INVALID_ARGUMENT, "no data"),
])
def test_append(changes, status, word):
    rc, message = append(**changes)
    assert rc == status and word in message, message


@pytest.mark.parametrize("changes,status,word", [
    ({"dtype": INT32}, UNSUPPORTED, "dtype"), ({"q": heads(7, 128)}, INVALID_ARGUMENT, "heads"), ({"out": heads(6, 128)}, INVALID_ARGUMENT, "heads"),
    ({"q": heads(8, 128, BASE + 2)}, INVALID_ARGUMENT, "16-byte"), ({"q": heads(8, 128, token=1028)}, INVALID_ARGUMENT, "16-byte"),
    ({"out": heads(8, 128, token=512)}, INVALID_ARGUMENT, "overlap"), ({"max_tokens": 0}, INVALID_ARGUMENT, "max_tokens"),
    ({"window": -1}, INVALID_ARGUMENT, "window"), ({"scale": float("nan")}, INVALID_ARGUMENT, "scale"),
    ({"scale": float("inf")}, INVALID_ARGUMENT, "scale"),
])
def test_attention_kv4(changes, status, word):
    rc, message = attention(**changes)
    assert rc == status and word in message, message


def prompt(q=None, k=None, v=None, out=None, cu_q=BASE, cu_k=BASE, **changes):
    fields = dict(q_tokens=5, k_tokens=5, batch=2, head_dim=64, dtype=FLOAT16, causal=1, window=0, scale=0.1, max_q=0) | changes
    q, k, v, out = q or heads(4), k or heads(2), v or heads(2), out or heads(4, at=2 * BASE)
    return outcome(ovk_b200.lib().ovk_attention_prompt(None, PromptParams(**fields), q, k, v, cu_q, cu_k, out))


@pytest.mark.parametrize("changes,status,word", [
    ({}, INVALID_ARGUMENT, "null context"), ({"dtype": 16}, UNSUPPORTED, "dtype"), ({"head_dim": 0}, UNSUPPORTED, "head_dim"),
    ({"head_dim": 257}, UNSUPPORTED, "head_dim"), ({"q_tokens": -1}, INVALID_ARGUMENT, "rows"), ({"batch": -1}, INVALID_ARGUMENT, "sequences"),
    ({"window": -2}, INVALID_ARGUMENT, "window"), ({"max_q": -1}, INVALID_ARGUMENT, "max_q"), ({"scale": float("-inf")}, INVALID_ARGUMENT, "scale"), ({"q": heads(5)}, INVALID_ARGUMENT, "heads"),
    ({"v": heads(1)}, INVALID_ARGUMENT, "heads"), ({"out": heads(2, at=2 * BASE)}, INVALID_ARGUMENT, "heads"),
    ({"out": heads(4, at=2 * BASE, token=64)}, INVALID_ARGUMENT, "overlap"), ({"cu_q": None}, INVALID_ARGUMENT, "bounds"),
    ({"cu_k": BASE + 1}, INVALID_ARGUMENT, "bounds"), ({"k": heads(2, at=None)}, INVALID_ARGUMENT, "no data"),
    ({"k": heads(2, at=BASE + 1)}, INVALID_ARGUMENT, "aligned"),
])
def test_prompt(changes, status, word):
    rc, message = prompt(**changes)
    assert rc == status and word in message, message


def test_null_structs():
    lib, h = ovk_b200.lib(), heads()
    for rc in (lib.ovk_rotary(None, None, 1, h, h, None, None, None), lib.ovk_kv4_append(None, None, batch(), h, h, FLOAT),
               lib.ovk_kv4_append(None, cache(), None, h, h, FLOAT), lib.ovk_kv4_append(None, cache(), batch(), None, h, FLOAT),
               lib.ovk_attention_kv4(None, None, batch(), h, h, FLOAT, 1, 1.0, 0, None, 0),
               lib.ovk_attention_kv4_workspace(None, cache(), 8, 1, FLOAT, None), lib.ovk_attention_prompt(None, None, h, h, h, None, None, h)):
        assert rc == INVALID_ARGUMENT


def test_cache_object_checks_its_tensors():
    import torch
    code, scale = torch.zeros((2, 1, 4, 64), dtype=torch.uint8), torch.zeros((2, 1, 4, 4), dtype=torch.float16)
    with pytest.raises(ovk_b200.OvkError) as e:  # CPU tensors
        ovk_b200.KV4Cache(code, code, scale, scale)
    assert "one GPU" in e.value.message
    with pytest.raises(ovk_b200.OvkError):
        ovk_b200.KV4Cache(code, code, scale, scale, code)
    with pytest.raises(ovk_b200.OvkError):
        ovk_b200.KV4Cache(code[0], code, scale, scale)


def test_packed_structs_are_the_declared_ones():
    """The wrappers hand structs over as packed bytes: same size and same fields as the ctypes declarations."""
    assert ovk_b200._PACK_HEADS(1, 2, 3, 4) == bytes(Heads(1, 2, 3, 4))
    assert ovk_b200._PACK_HEADS2(1, 2, 3, 4, 5, 6, 7, 8) == bytes((Heads * 2)(Heads(1, 2, 3, 4), Heads(5, 6, 7, 8)))
    assert ovk_b200._PACK_ROTARY(*range(1, 14)) == bytes(RotaryParams(*range(1, 10), (C.c_int32 * 4)(10, 11, 12, 13)))
    assert ovk_b200._PACK_BATCH(*range(1, 7)) == bytes(KV4Batch(*range(1, 7)))
    assert ovk_b200._PACK_PROMPT(1, 2, 3, 4, 5, 6, 7, 8.5, 9) == bytes(PromptParams(1, 2, 3, 4, 5, 6, 7, 8.5, 9))

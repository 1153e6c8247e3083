"""More of what the attention operators refuse, without a GPU: scales beyond powers of two, and wrappers called with what is no
tensor of the right kind or no number of the right size."""
import pytest
import torch

import ovk_b200
from ovk_b200 import INVALID_ARGUMENT
from test_attention_refusals import attention, prompt


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38, float("inf"), float("nan")])
def test_scales_that_are_not_finite_in_powers_of_two(scale):
    for rc, message in (attention(scale=scale), prompt(scale=scale)):
        assert rc == INVALID_ARGUMENT and "scale" in message, message


@pytest.mark.parametrize("scale", [2.3e38, -2.3e38, 0.0, 1e-45])
def test_finite_scales_pass(scale):
    for rc, message in (attention(scale=scale), prompt(scale=scale)):
        assert rc == INVALID_ARGUMENT and "null context" in message, message


@pytest.fixture
def context():
    """A context without a GPU behind it: whatever a wrapper refuses by itself."""
    c = object.__new__(ovk_b200.Context)
    c.h, c.device, c._foreign_stream = None, -1, lambda: None  # CPU tensors are on device -1
    return c


def refused(call, *args, word="", **named):
    with pytest.raises(ovk_b200.OvkError) as e:
        call(*args, **named)
    assert e.value.status == INVALID_ARGUMENT and word in e.value.message, e.value.message


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


X, T = torch.zeros(4, 2, 64), torch.zeros(9, 32)


@pytest.mark.parametrize("change,word", [
    ({"cos": [1.0]}, "cos"), ({"cos": T[0]}, "cos"), ({"sin": None}, "sin"), ({"sin": T[:5]}, "sin"), ({"positions": torch.tensor(3)}, "positions"),
    ({"positions": [0, 1, 2, 3]}, "positions"), ({"positions": i32(2, 2, 4)}, "positions"), ({"positions": i32(5)}, "positions"),
    ({"sections": 32}, "sections"), ({"sections": [32.0]}, "sections"), ({"sections": [1 << 40]}, "sections"), ({"sections": [16, 16]}, "2 sections"),
    ({"q": None}, "q"), ({"q": X[0]}, "q"), ({"q": X.to(torch.bfloat16)}, "q"), ({"k": X[:3]}, "k"),
])
def test_rotary_wrapper(context, change, word):
    refused(context.rotary, **({"q": X, "cos": T, "sin": T, "positions": i32(4)} | change), word="Rotary: " + word)


@pytest.mark.parametrize("change,word", [
    ({"window": 1.5}, "window"), ({"window": 1 << 63}, "window"), ({"window": None}, "window"), ({"max_q": 3.7}, "max_q"), ({"max_q": 1 << 31}, "max_q"),
    ({"scale": "a"}, "scale"), ({"scale": 1 << 2000}, "scale"), ({"cu_q": [0, 4]}, "cu_q"), ({"cu_q": i32()}, "cu_q"), ({"cu_q": i32(0)}, "cu_q"),
    ({"cu_q": i32(2).long()}, "cu_q"), ({"cu_k": i32(3)}, "cu_k"), ({"k": X[..., :32]}, "k"), ({"v": X[:, :1]}, "v"), ({"q": [1]}, "q"),
])
def test_prompt_wrapper(context, change, word):
    refused(context.attention_prompt, **({"q": X, "k": X, "v": X, "cu_q": i32(2)} | change), word="AttentionPrompt: " + word)


@pytest.mark.parametrize("change,word", [
    ({"lens": [4]}, "lens"), ({"lens": i32(1, 1)}, "lens"), ({"block_table": None}, "block_table"), ({"block_table": i32(1)}, "block_table"),
    ({"block_table": i32(2, 3)}, "block_table"), ({"cu_tokens": i32(1)}, "cu_tokens"), ({"q": X[..., :32]}, "q"), ({"cache": "x"}, "KV4Cache"),
    ({"max_tokens": 1.0}, "max_tokens"), ({"max_tokens": 1 << 70}, "max_tokens"), ({"window": "all"}, "window"), ({"window": -1 << 64}, "window"),
    ({"scale": [1]}, "scale"),
])
def test_kv4_wrapper(context, change, word):
    cache = object.__new__(ovk_b200.KV4Cache)
    cache.device, cache.kv_heads, cache.head_dim = -1, 2, 64
    given = {"cache": cache, "q": X, "block_table": i32(1, 3), "cu_tokens": i32(2), "lens": i32(1)} | change
    refused(context.attention_kv4, **given, word=word)
    if not {"max_tokens", "window", "scale"} & set(change):
        x = given.pop("q")
        refused(context.kv4_append, **given, k=x, v=x, word="k" if word == "q" else word)


@pytest.mark.parametrize("change,word", [({"pages": 1.5}, "pages"), ({"pages": -1}, "-1 pages"), ({"block_size": 0}, "blocks of 0"), ({"head_dim": "64"}, "head_dim")])
def test_new_caches(context, change, word):
    refused(context.kv4_cache, **({"pages": 2, "kv_heads": 1, "page_size": 4, "head_dim": 64} | change), word=word)


def test_caches_of_what_is_no_tensor():
    code, scale = torch.zeros((2, 1, 4, 64), dtype=torch.uint8), torch.zeros((2, 1, 4, 4), dtype=torch.float16)
    for args in ((None, code, scale, scale), (code, None, scale, scale), (code, code, [1], scale), (code, code, scale, scale, 3, 3)):
        refused(ovk_b200.KV4Cache, *args, word="tensors")


@pytest.mark.parametrize("shape", [(6,), (3, 2, 4), (3, 2, 1, 2)])
def test_gather_of_a_table_that_is_none(context, shape):
    refused(context.gather_block_quantized, torch.zeros(shape, dtype=torch.uint8), [0], None, None, 32, word="table")

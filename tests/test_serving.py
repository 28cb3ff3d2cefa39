"""Refusals of the serving operators that need no GPU: the C entry points' argument checks and the Python ones."""

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from pto_wsp_b200 import serving  # noqa: E402
from pto_wsp_b200.runtime import load_library  # noqa: E402

ARG, UNSUPPORTED, LIMIT = 4, 2, 6
PTR = 1 << 20  # an address that the checks look at and nothing reads


def cache(**over):
    c = serving._Cache(PTR, PTR, PTR, PTR, 2048 * 8, 128, 2048, 2048 * 8, 128, 2048, 10, 16, 8, 128, 0)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def call(name, *structs):
    lib = serving._library()
    rc = getattr(lib, "ptowsp_cuda_" + name)(*[C.addressof(s) if s is not None else None for s in structs], None)
    return rc, (load_library().ptowsp_cuda_last_error() or b"").decode()


def attention(**over):
    a = serving._Attention(PTR, PTR, None, 4096, 128, 4096, 128, PTR, 8, PTR, None, 4, 8, 4, 32, 1, 0, 1, 0.1, 0, PTR,
                           1 << 30, None)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def append(**over):
    a = serving._Append(PTR, PTR, 1024, 128, 1024, 128, PTR, 4, 1, 0, None)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def reserve(**over):
    a = serving._Reserve(PTR, 8, 8, 16, 4, 0, PTR, PTR, PTR, 100, PTR, PTR, PTR, 10, PTR, PTR + 64, PTR + 64, PTR, None)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def sample(**over):
    a = serving._Sample(PTR, 1000, 4, 1000, 0, 0, PTR, None, None, None, None, PTR, PTR)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code,text", [
    ({"k": None}, ARG, "null"),
    ({"v_scale": None}, ARG, "null"),
    ({"format": 2}, ARG, "format"),
    ({"head_dim": 96}, UNSUPPORTED, "head_dim"),
    ({"page_size": 24}, UNSUPPORTED, "page_size"),
    ({"page_size": 256}, UNSUPPORTED, "page_size"),
    ({"num_kv_heads": 0}, ARG, "num_kv_heads"),
    ({"num_pages": 0}, ARG, "num_pages"),
    ({"k": PTR + 8}, ARG, "aligned"),
    ({"v_token_stride": 120}, ARG, "strides"),
    ({"k_page_stride": -16}, ARG, "strides"),
])
def test_cache_refusals(over, code, text):
    for name, args in (("kv8_append", append()), ("kv8_attention", attention())):
        rc, msg = call(name, cache(**over), args)
        assert rc == code and text in msg and name in msg


@pytest.mark.parametrize("over,code,text", [
    ({"dtype": 0}, UNSUPPORTED, "f16 or bf16"),
    ({"num_heads": 12}, ARG, "multiple"),
    ({"num_heads": 0}, ARG, "multiple"),
    ({"window": -1}, ARG, "negative"),
    ({"requests": -1}, ARG, "negative"),
    ({"max_pages": 1 << 28}, LIMIT, "max_pages"),
    ({"max_q": 1 << 30}, LIMIT, "max_q"),
    ({"scale": float("nan")}, ARG, "finite"),
    ({"scale": float("inf")}, ARG, "finite"),
    ({"q": None}, ARG, "null"),
    ({"kv_len": None}, ARG, "null"),
    ({"page_table": None}, ARG, "null"),
    ({"tokens": 5}, ARG, "q_start"),
    ({"max_q": 2}, ARG, "q_start"),
    ({"q": PTR + 2}, ARG, "aligned"),
    ({"out_head_stride": 68}, ARG, "aligned"),
])
def test_attention_refusals(over, code, text):
    rc, msg = call("kv8_attention", cache(), attention(**over))
    assert rc == code and text in msg


def test_attention_without_work_is_no_error():
    assert call("kv8_attention", cache(), attention(requests=0, tokens=0, q=None))[0] == 0


@pytest.mark.parametrize("over,code,text", [
    ({"dtype": 3}, UNSUPPORTED, "f32, f16 or bf16"),
    ({"tokens": -1}, ARG, "tokens"),
    ({"slots": None}, ARG, "null"),
    ({"k_head_stride": 68}, ARG, "aligned"),
    ({"v": PTR + 4}, ARG, "aligned"),
])
def test_append_refusals(over, code, text):
    rc, msg = call("kv8_append", cache(), append(**over))
    assert rc == code and text in msg


@pytest.mark.parametrize("over,code,text", [
    ({"requests": 16385}, LIMIT, "16384"),
    ({"requests": -1}, ARG, "negative"),
    ({"page_size": 24}, ARG, "power of two"),
    ({"page_size": 0}, ARG, "power of two"),
    ({"max_pages": 1 << 28, "table_stride": 1 << 28}, LIMIT, "max_pages"),
    ({"table_stride": 7}, ARG, "overlap"),
    ({"slots": None}, ARG, "null"),
    ({"free_ring": None}, ARG, "null"),
    ({"granted": None}, ARG, "null"),
    ({"kv_len_out": PTR}, ARG, "kv_len_out"),
    ({"free_state_out": PTR}, ARG, "free_state_out"),
])
def test_reserve_refusals(over, code, text):
    rc, msg = call("reserve_pages", reserve(**over))
    assert rc == code and text in msg


@pytest.mark.parametrize("over,code,text", [
    ({"vocab": 0}, ARG, "vocab"),
    ({"vocab": (1 << 22) + 1}, LIMIT, "vocab"),
    ({"rows": -1}, ARG, "rows"),
    ({"dtype": 7}, UNSUPPORTED, "logits"),
    ({"u": None}, ARG, "null"),
    ({"token": None}, ARG, "null"),
    ({"logits": PTR + 2}, ARG, "aligned"),
])
def test_sample_refusals(over, code, text):
    rc, msg = call("sample_tokens", sample(**over))
    assert rc == code and text in msg


def test_null_argument_structs():
    for name, structs in (("reserve_pages", [None]), ("sample_tokens", [None]), ("kv8_append", [cache(), None]),
                          ("kv8_attention", [cache(), None]), ("kv8_append", [None, append()])):
        rc, msg = call(name, *structs)
        assert rc == ARG and "null" in msg


def test_host_tensors_are_refused():
    x = torch.zeros(4, 8)
    with pytest.raises(TypeError, match="CUDA"):
        serving.sample_tokens(x, torch.zeros(4))
    with pytest.raises(TypeError, match="CUDA"):
        serving.append_kv8(x, x, x, x, x, x, x)
    with pytest.raises(TypeError, match="CUDA"):
        serving.reserve_pages(x, x, x, x, x, page_size=16, max_tokens=1)

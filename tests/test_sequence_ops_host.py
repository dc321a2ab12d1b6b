"""Refusals of the sequence operators (no GPU needed).

Every check of sizes, strides, types and pointers runs before the handle's
device is touched, so the calls are made here on a zeroed stand-in for the
handle and on addresses that nothing ever reads.
"""

import ctypes as C

import pytest

import ppocr_b200 as P

A = 1 << 20   # an aligned address; never read


@pytest.fixture()
def gpu():
    g = P.Gpu.__new__(P.Gpu)
    g._memory = C.create_string_buffer(4096)
    g._h = C.cast(g._memory, C.c_void_p)
    g.device = 0
    yield g
    g._h = None   # nothing to destroy


def arr(shape, dtype="f32", strides=None, ptr=A, device=0):
    return P.DeviceArray(ptr, shape, dtype, strides, device)


def packed(gpu, **kw):
    a = dict(q=arr((10, 4, 16)), k=arr((12, 2, 16)), v=arr((12, 2, 16)), q_offsets=arr((3,), "i32"),
             k_offsets=arr((3,), "i32"), out=arr((10, 4, 16)))
    a.update(kw)
    return gpu.attention_packed(**a)


def cache(pages=6, heads=2, page=16, d=16, ptr=A, scales=None):
    return P.PagedCache(arr((pages, heads, page, d), "i8", ptr=ptr), arr((pages, heads, page, d), "i8", ptr=ptr),
                        arr(scales or (pages, heads)), arr((pages, heads)))


def cached(gpu, **kw):
    a = dict(cache=cache(), q=arr((3, 4, 16)), lengths=arr((3,), "i32"), table=arr((3, 2), "i32"), out=arr((3, 4, 16)))
    a.update(kw)
    return gpu.attention_cached(**a)


def append(gpu, **kw):
    a = dict(cache=cache(), k=arr((5, 2, 16)), v=arr((5, 2, 16)), offsets=arr((4,), "i32"), held=arr((3,), "i32"),
             table=arr((3, 2), "i32"))
    a.update(kw)
    return gpu.cache_append(**a)


def read(gpu, **kw):
    a = dict(cache=cache(), k=arr((5, 2, 16)), v=arr((5, 2, 16)), offsets=arr((4,), "i32"), first=arr((3,), "i32"),
             table=arr((3, 2), "i32"))
    a.update(kw)
    return gpu.cache_read(**a)


def rules(gpu, **kw):
    a = dict(logits=arr((4, 100)), out=arr((4, 100)))
    a.update(kw)
    return gpu.logit_rules(**a)


@pytest.mark.parametrize("call", [packed, cached, append, read, rules])
def test_valid_arguments_reach_the_device(gpu, call):
    if P.gpu_count() > 0:
        pytest.skip("the stand-in handle must not reach a device")
    with pytest.raises(P.GpuError):
        call(gpu)


@pytest.mark.parametrize("change,words", [
    (dict(q=arr((10, 4))), "axes"),
    (dict(q=arr((10, 4, 16), "i8")), "expected f32 or bf16"),
    (dict(k=arr((12, 2, 16), "bf16")), "expected f32"),
    (dict(v=arr((11, 2, 16))), "shape"),
    (dict(k=arr((12, 2, 15))), "shape"),
    (dict(out=arr((10, 2, 16))), "shape"),
    (dict(k=arr((12, 3, 16)), v=arr((12, 3, 16))), "multiple of kv_heads"),
    (dict(k=arr((12, 0, 16)), v=arr((12, 0, 16))), "multiple of kv_heads"),
    (dict(q=arr((10, 4, 129)), k=arr((12, 2, 129)), v=arr((12, 2, 129)), out=arr((10, 4, 129))), "1..128"),
    (dict(q=arr((10, 4, 0)), k=arr((12, 2, 0)), v=arr((12, 2, 0)), out=arr((10, 4, 0))), "1..128"),
    (dict(q=arr((10, 4, 16), strides=(64, 16, 2))), "contiguous"),
    (dict(out=arr((10, 4, 16), strides=(64, 8, 1))), "share memory"),
    (dict(out=arr((10, 4, 16), strides=(0, 16, 1))), "share memory"),
    (dict(q=arr((10, 4, 16), strides=(-64, 16, 1))), "strides"),
    (dict(q=arr((10, 4, 16), strides=(1 << 41, 16, 1))), "strides"),
    (dict(q=arr((10, 4, 16), ptr=0)), "null"),
    (dict(q=arr((10, 4, 16), ptr=A + 2)), "aligned"),
    (dict(q=arr((10, 4, 16), device=1)), "device"),
    (dict(k_offsets=arr((4,), "i32")), "shape"),
    (dict(q_offsets=arr((0,), "i32"), k_offsets=arr((0,), "i32")), "empty"),
    (dict(q_offsets=arr((3,), "f32")), "expected i32"),
    (dict(q_offsets=arr((3,), "i32", strides=(2,))), "contiguous"),
    (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"),
])
def test_attention_packed_refuses(gpu, change, words):
    with pytest.raises(P.InvalidInput, match=words):
        packed(gpu, **change)


@pytest.mark.parametrize("call", [cached, append, read])
@pytest.mark.parametrize("change,words", [
    (dict(cache=cache(page=8)), "16, 32, 64 or 128"),
    (dict(cache=cache(page=48)), "16, 32, 64 or 128"),
    (dict(cache=cache(d=12)), "multiple of 8|shape"),
    (dict(cache=cache(d=136)), "up to 128|shape"),
    (dict(cache=cache(ptr=A + 8)), "16-byte"),
    (dict(cache=cache(ptr=0)), "null"),
    (dict(cache=cache(scales=(6, 3))), "shape"),
    (dict(table=arr((3, 2), "i32", strides=(1, 3))), "contiguous"),
    (dict(table=arr((3, 2), "i32", strides=(1, 1))), "stride"),
    (dict(table=arr((3, 2), "i32", ptr=0)), "table pointer"),
    (dict(table=arr((3, 1 << 27), "i32")), "2\\^31"),
    (dict(table=arr((2, 2), "i32")), "shape"),
])
def test_cache_calls_refuse(gpu, call, change, words):
    with pytest.raises(P.InvalidInput, match=words):
        call(gpu, **change)


@pytest.mark.parametrize("call,change,words", [
    (cached, dict(q=arr((3, 3, 16)), out=arr((3, 3, 16))), "multiple of kv_heads"),
    (cached, dict(q=arr((3, 4, 24))), "shape"),
    (cached, dict(out=arr((3, 4, 16), "bf16")), "expected f32"),
    (cached, dict(lengths=arr((4,), "i32")), "shape"),
    (cached, dict(out=arr((3, 4, 16), strides=(16, 16, 1))), "share memory"),
    (append, dict(k=arr((5, 4, 16)), v=arr((5, 4, 16))), "shape"),
    (append, dict(v=arr((6, 2, 16))), "shape"),
    (append, dict(held=arr((2,), "i32")), "shape"),
    (read, dict(k=arr((5, 2, 16), strides=(0, 16, 1))), "share memory"),
    (read, dict(v=arr((5, 2, 16), strides=(32, 0, 1))), "share memory"),
    (read, dict(first=arr((3,), "f32")), "expected i32"),
    (rules, dict(out=arr((4, 99))), "shape"),
    (rules, dict(out=arr((4, 100), "bf16")), "expected f32"),
    (rules, dict(logits=arr((4, 100), strides=(200, 2))), "contiguous"),
    (rules, dict(logits=arr((4, 100), strides=(99, 1))), "stride"),
    (rules, dict(logits=arr((4, 100), strides=(128, 1))), "in place"),
    (rules, dict(logits=arr((4, 100), ptr=0)), "null"),
    (rules, dict(presence=arr((4,))), "need a history"),
    (rules, dict(history=arr((7,), "i32")), "go together"),
    (rules, dict(history=arr((7,), "i32"), history_offsets=arr((4,), "i32")), "shape"),
    (rules, dict(bias=arr((99,))), "shape"),
    (rules, dict(mask=arr((2, 3), "i32")), "words"),
    (rules, dict(mask_index=arr((4,), "i32")), "needs a mask"),
    (rules, dict(mask=arr((0, 4), "i32")), "at least one row"),
    (rules, dict(mask=arr((2, 4), "i32", strides=(2, 1))), "words"),
])
def test_other_refusals(gpu, call, change, words):
    with pytest.raises(P.InvalidInput, match=words):
        call(gpu, **change)


@pytest.mark.parametrize("call,change", [
    (packed, dict(scale=1e39)), (packed, dict(scale=1e31)), (cached, dict(scale=1e300)),
    (packed, dict(q_offsets=arr(((1 << 31) + 1,), "i32"), k_offsets=arr(((1 << 31) + 1,), "i32"))),
    (packed, dict(q=arr((1 << 31, 4, 16)), out=arr((1 << 31, 4, 16)))),
    (packed, dict(q=arr((10, 1 << 33, 16)), out=arr((10, 1 << 33, 16)))),
    (cached, dict(table=arr((3, 1 << 33), "i32"))),
    (append, dict(k=arr((1 << 31, 2, 16)), v=arr((1 << 31, 2, 16)))),
    (rules, dict(logits=arr((4, 1 << 31)), out=arr((4, 1 << 31)))),
    (rules, dict(logits=arr(((1 << 31) - 1, 1)), out=arr(((1 << 31) - 1, 1)))),
    (rules, dict(logits=arr((1 << 40, 1)), out=arr((1 << 40, 1)))),
])
def test_sizes_and_scales_out_of_range_are_refused(gpu, call, change):
    with pytest.raises(P.InvalidInput):
        call(gpu, **change)


@pytest.mark.parametrize("call,change", [
    (packed, dict(q_offsets=arr((3,), "i32", ptr=A + 2))), (packed, dict(k_offsets=arr((3,), "i32", ptr=A + 1))),
    (cached, dict(lengths=arr((3,), "i32", ptr=A + 2))), (cached, dict(table=arr((3, 2), "i32", ptr=A + 2))),
    (append, dict(offsets=arr((4,), "i32", ptr=A + 1))), (append, dict(held=arr((3,), "i32", ptr=A + 2))),
    (read, dict(first=arr((3,), "i32", ptr=A + 2))), (rules, dict(bias=arr((100,), ptr=A + 2))),
    (rules, dict(mask=arr((1, 4), "i32", ptr=A + 2))),
    (rules, dict(mask=arr((1, 4), "i32"), mask_index=arr((4,), "i32", ptr=A + 1))),
    (rules, dict(history=arr((7,), "i32", ptr=A + 2), history_offsets=arr((5,), "i32"))),
    (rules, dict(history=arr((7,), "i32"), history_offsets=arr((5,), "i32", ptr=A + 2))),
    (rules, dict(history=arr((7,), "i32"), history_offsets=arr((5,), "i32"), repetition=arr((4,), ptr=A + 2))),
])
def test_misaligned_arrays_are_refused(gpu, call, change):
    with pytest.raises(P.InvalidInput, match="aligned"):
        call(gpu, **change)


def test_argument_layouts_are_the_headers(tmp_path):
    """The packed arguments have the sizes and ends of the header's structures."""
    import os
    import shutil
    import subprocess

    if shutil.which("g++") is None:
        pytest.skip("needs a C++ compiler")
    ends = [("ppocr_attention_packed_args", "k_offsets"), ("ppocr_cache_append_args", "held"), ("ppocr_cache_read_args", "first"),
            ("ppocr_attention_cached_args", "lengths"), ("ppocr_logit_rules_args", "mask_index")]
    src = tmp_path / "layout.cpp"
    src.write_text('#include "ppocr_b200.h"\n#include <cstdio>\nint main() {\n' + "".join(
        f'std::printf("%zu %zu\\n", sizeof({t}), offsetof({t}, {m}));\n' for t, m in ends) + "}\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["g++", "-I", include, str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split("\n")
    for line, pack in zip(out, (P._ATTENTION_PACKED, P._CACHE_TOKENS, P._CACHE_TOKENS, P._ATTENTION_CACHED, P._LOGIT_RULES)):
        size, last = (int(v) for v in line.split())
        assert pack.__self__.size == size == last + 8


def test_null_handles_and_arguments():
    lib = P.library()
    for name in ("ppocr_attention_packed", "ppocr_cache_append", "ppocr_cache_read", "ppocr_attention_cached",
                 "ppocr_logit_rules"):
        assert getattr(lib, name)(None, None, None) == P.InvalidInput.code
    assert lib.ppocr_gpu_synchronize(None, None, 0) == P.InvalidInput.code
    assert lib.ppocr_recognizer_forward_ctc_rules(None, None, 0, None, None, None, None, None) == P.InvalidInput.code

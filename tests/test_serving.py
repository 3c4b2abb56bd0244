"""What the 8-bit decoder layer's entry points refuse: messages and status codes, before anything reaches a device."""
import ctypes

import pytest

OK_BUT_NO_DEVICE = (-13, "device")  # in order, as far as this can be told without one

F32, F16, BF16, I8, I32 = 10, 8, 9, 1, 3


@pytest.fixture()
def calls(mlel):
    return mlel, mlel.lib()


def T(mlel, dtype, dims, ptr=0x10000, strides=None):
    return mlel.device_tensor(ptr, dtype, dims, strides)


def refused(mlel, status, word):
    assert status != 0
    message = (mlel.lib().mlel_last_error() or b"").decode()
    assert word in message, message
    return status


def by(*tensors):
    return [None if t is None else ctypes.byref(t) for t in tensors]


QUANTIZE = dict(x=(F16, (3, 40)), q=(I8, (3, 40)), s=(F32, (3,)))


@pytest.mark.parametrize("change, word, status", [
    (dict(x=(I8, (3, 40))), "f32, f16 or bf16", -8),
    (dict(x=(F16, (3, 40, 1))), "axes", -13),
    (dict(q=(I32, (3, 40))), "int8", -13),
    (dict(q=(I8, (3, 41))), "fit", -13),
    (dict(s=(F32, (4,))), "fit", -13),
    (dict(s=(F16, (3,))), "f32", -13),
    (dict(x=(F16, (3, 0)), q=(I8, (3, 0))), "no scale", -13),
    (dict(x=(F16, (3, 40), 0x10001)), "boundary", -13),
    (dict(x=(F16, (3, 40), 0)), "null", -13),
    (dict(x=(F16, (3, 40), 0x10000, (80, 4))), "side by side", -13),
    (dict(x=(F16, (3, 40), 0x10000, (81, 2))), "whole elements", -13),
    (dict(x=(F16, (-3, 40))), "axis", -13),
    (dict(x=(77, (3, 40))), "type", -13),
    (dict(q=(I8, (3, 40), 0x10000, (39, 1))), "overlap", -13),
    (dict(x=None), "missing", -13),
    (dict(x=(F16, (1, 2 ** 30 + 1)), q=(I8, (1, 2 ** 30 + 1)), s=(F32, (1,))), "more than", -13),
    (dict(), *OK_BUT_NO_DEVICE[::-1]),
])
def test_quantize_rows_refuses(calls, change, word, status):
    mlel, lib = calls
    args = [None if v is None else T(mlel, *v) for v in {**QUANTIZE, **change}.values()]
    assert refused(mlel, lib.mlel_cuda_quantize_rows(*by(*args), None), word) == status


def test_nothing_to_do_is_no_error(calls):
    mlel, lib = calls
    assert lib.mlel_cuda_quantize_rows(*by(T(mlel, F16, (0, 40), 0), T(mlel, I8, (0, 40), 0), T(mlel, F32, (0,), 0)), None) == 0
    assert lib.mlel_cuda_matmul_scaled(*by(T(mlel, I8, (0, 40), 0), T(mlel, F32, (0,), 0), T(mlel, I8, (5, 40)), T(mlel, F32, (5,)), None,
                                           T(mlel, F32, (0, 5), 0)), None) == 0


MATMUL = dict(a=(I8, (7, 48)), sa=(F32, (7,)), b=(I8, (9, 48)), sb=(F32, (9,)), bias=(F32, (9,)), out=(BF16, (7, 9)))


@pytest.mark.parametrize("change, word, status", [
    (dict(a=(F16, (7, 48))), "int8", -13),
    (dict(b=(I8, (9, 47))), "fit", -13),
    (dict(sa=(F32, (9,))), "fit", -13),
    (dict(sb=(BF16, (9,))), "f32", -13),
    (dict(bias=(F32, (7,))), "fit", -13),
    (dict(out=(I32, (7, 9))), "f32, f16 or bf16", -8),
    (dict(out=(BF16, (9, 7))), "fit", -13),
    (dict(out=(BF16, (7, 9), 0x10000, (16, 2))), "overlap", -13),
    (dict(a=(I8, (7, 131072)), b=(I8, (9, 131072))), "131071", -13),
    (dict(a=(I8, (7, 0)), b=(I8, (9, 0))), "131071", -13),
    (dict(bias=None), *OK_BUT_NO_DEVICE[::-1]),
    (dict(), *OK_BUT_NO_DEVICE[::-1]),
])
def test_matmul_scaled_refuses(calls, change, word, status):
    mlel, lib = calls
    args = [None if v is None else T(mlel, *v) for v in {**MATMUL, **change}.values()]
    assert refused(mlel, lib.mlel_cuda_matmul_scaled(*by(*args), None), word) == status


def paged(mlel, keys=(I8, (11, 2, 32, 64)), values=None, key_scales=(F32, (11, 2)), value_scales=None, starts=(I32, (4,)),
          lengths=(I32, (3,)), table=(I32, (3, 5)), max_new=20, max_length=150):
    class Cache(ctypes.Structure):
        _fields_ = [(n, mlel.Tensor) for n in ("keys", "values", "key_scales", "value_scales")]

    class Batch(ctypes.Structure):
        _fields_ = [(n, mlel.Tensor) for n in ("starts", "lengths", "page_table")] + [("max_new", ctypes.c_int32), ("max_length", ctypes.c_int32)]
    cache = Cache(T(mlel, *keys), T(mlel, *(values or keys)), T(mlel, *key_scales), T(mlel, *(value_scales or key_scales)))
    return cache, Batch(T(mlel, *starts), T(mlel, *lengths), T(mlel, *table), max_new, max_length)


PAGED_REFUSALS = [
    (dict(keys=(I32, (11, 2, 32, 64))), "int8", -13),
    (dict(keys=(I8, (11, 2, 40, 64))), "multiple of 16 tokens", -8),
    (dict(keys=(I8, (11, 2, 272, 64))), "at most 256", -8),
    (dict(keys=(I8, (11, 2, 32, 72))), "head_dim", -8),
    (dict(keys=(I8, (11, 2, 32, 272))), "head_dim", -8),
    (dict(keys=(I8, (0, 2, 32, 64))), "fit", -13),
    (dict(keys=(I8, (11, 2, 32, 64), 0x10008)), "16-byte", -13),
    (dict(keys=(I8, (11, 2, 32, 64), 0x10000, (8192, 4096, 64, 1))), "packed", -13),
    (dict(values=(I8, (11, 2, 16, 64))), "fit", -13),
    (dict(key_scales=(F32, (11, 3))), "fit", -13),
    (dict(value_scales=(F16, (11, 2))), "f32", -13),
    (dict(starts=(I32, (3,))), "sequences", -13),
    (dict(lengths=(4, (3,))), "i32", -13),
    (dict(table=(I32, (2, 5))), "sequences", -13),
    (dict(table=(I32, (3, 4))), "columns", -13),
    (dict(max_new=200), "max_new", -13),
    (dict(max_new=-1), "max_new", -13),
    (dict(max_length=(1 << 30) + 1), "max_length", -13),
]
APPEND = dict(k=(F16, (30, 2, 64)), v=(F16, (30, 2, 64)), cos=(F32, (150, 32)), sin=(F32, (150, 32)), q=(F16, (30, 6, 64)), r=(F16, (30, 6, 64)))


@pytest.mark.parametrize("cache, change, word, status", [(c, {}, w, s) for c, w, s in PAGED_REFUSALS] + [
    ({}, dict(k=(F32, (30, 2, 64))), "f16 or bf16", -8),
    ({}, dict(v=(BF16, (30, 2, 64))), "keys' type", -8),
    ({}, dict(v=(F16, (31, 2, 64))), "fit", -13),
    ({}, dict(k=(F16, (30, 3, 64)), v=(F16, (30, 3, 64))), "fit", -13),
    ({}, dict(cos=None), "together", -13),
    ({}, dict(cos=(F32, (149, 32)), sin=(F32, (149, 32))), "rows", -13),
    ({}, dict(cos=(F32, (150, 33)), sin=(F32, (150, 33))), "pairs", -13),
    ({}, dict(sin=(F32, (150, 31))), "shape", -13),
    ({}, dict(q=None), "together", -13),
    ({}, dict(q=(BF16, (30, 6, 64))), "type", -8),
    ({}, dict(r=(F16, (30, 5, 64))), "fit", -13),
    ({}, dict(r=(F16, (30, 6, 64), 0x10000, (2 * 6 * 80, 160, 2))), "layout", -13),
    ({}, dict(r=(F16, (30, 6, 64), 0x20000, (768, 100, 2))), "overlap", -13),
    ({}, dict(cos=None, sin=None, q=None, r=None), *OK_BUT_NO_DEVICE[::-1]),
    ({}, {}, *OK_BUT_NO_DEVICE[::-1]),
])
def test_append_refuses(calls, cache, change, word, status):
    mlel, lib = calls
    args = [None if v is None else T(mlel, *v) for v in {**APPEND, **change}.values()]
    assert refused(mlel, lib.mlel_cuda_paged_append(*by(*paged(mlel, **cache)), *by(*args), 0, None), word) == status


@pytest.mark.parametrize("cache, change, word, status", [(c, {}, w, s) for c, w, s in PAGED_REFUSALS] + [
    ({}, dict(q=(F32, (30, 6, 64))), "f16 or bf16", -8),
    ({}, dict(q=(F16, (30, 5, 64))), "multiple of its heads", -13),
    ({}, dict(q=(F16, (30, 6, 80))), "head_dim", -13),
    ({}, dict(out=(BF16, (30, 6, 64))), "type", -8),
    ({}, dict(out=(F16, (29, 6, 64))), "shape", -13),
    ({}, dict(scale=float("inf")), "finite", -13),
    ({}, dict(softcap=-1.0), "not negative", -13),
    ({}, dict(softcap=float("nan")), "finite", -13),
    ({}, dict(window=-1), "not negative", -13),
    ({}, {}, *OK_BUT_NO_DEVICE[::-1]),
])
def test_attention_refuses(calls, cache, change, word, status):
    mlel, lib = calls
    a = {**dict(q=(F16, (30, 6, 64)), out=(F16, (30, 6, 64)), scale=0.125, window=0, softcap=0.0), **change}
    c, b = paged(mlel, **cache)
    q, out = T(mlel, *a["q"]), T(mlel, *a["out"])
    rc = lib.mlel_cuda_paged_attention(*by(c, b, q, out), ctypes.c_float(a["scale"]), 1, a["window"], ctypes.c_float(a["softcap"]),
                                       ctypes.c_void_p(0x10000), ctypes.c_uint64(1 << 40), None)
    assert refused(mlel, rc, word) == status


def test_attention_refuses_rows_beyond_32_bits(calls):
    """2^28 new tokens with eight query heads a cache head: more rows than a 32-bit number counts."""
    mlel, lib = calls
    c, b = paged(mlel, table=(I32, (3, 1 << 23)), max_new=1 << 28, max_length=1 << 28)
    q = T(mlel, F16, (1 << 28, 16, 64))
    rc = lib.mlel_cuda_paged_attention(*by(c, b, q, q), ctypes.c_float(0.125), 1, 0, ctypes.c_float(0.0), ctypes.c_void_p(0x10000),
                                       ctypes.c_uint64(1 << 40), None)
    assert refused(mlel, rc, "rows of queries") == -13
    need = ctypes.c_uint64()
    assert refused(mlel, lib.mlel_paged_attention_workspace(*by(c, b, q, need)), "rows of queries") == -13


@pytest.mark.parametrize("loose", [31, 1 << 20, 1 << 28, 1 << 30])
def test_loose_bounds_on_new_tokens_change_nothing(calls, loose):
    """No sequence has more new tokens than the token axis: the launch is that of the close bound."""
    mlel, lib = calls
    needs = []
    for bound in (3, loose):
        c, b = paged(mlel, table=(I32, (3, 1 << 25)), max_new=bound, max_length=1 << 30)
        need = ctypes.c_uint64()
        assert lib.mlel_paged_attention_workspace(*by(c, b, T(mlel, F16, (3, 8, 64)), need)) == 0
        needs.append(need.value)
    assert needs[0] == needs[1] > 0


def test_a_record_that_cannot_be_read_is_no_clean_one(calls):
    """Without a device, or with one in an error state, there is no telling what was left out."""
    import torch
    mlel, lib = calls
    if torch.cuda.is_available():
        pytest.skip("there is a device to read")
    assert refused(mlel, lib.mlel_paged_error(), "cannot be read") == -4


@pytest.mark.parametrize("code, wait, raised", [(0, 0, None), (2, 0, None), (-4, 0, "status -4"), (0, 61, "code 61"), (1, 88, "code 88")])
def test_python_layer_raises_for_failed_devices_and_waits(mlel, monkeypatch, code, wait, raised):
    import contextlib

    import torch
    from mlel_b200 import serving

    class Fake:
        mlel_paged_error = staticmethod(lambda: code)
        mlel_device_error = staticmethod(lambda: wait)
    monkeypatch.setattr(serving, "lib", Fake)
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    if raised is None:
        assert serving.paged_error(0) == code
    else:
        with pytest.raises(mlel.MlelError, match=raised):
            serving.paged_error(0)


@pytest.mark.parametrize("k", [33, 48])
@pytest.mark.parametrize("change, word", [(dict(weight="float32"), "weight has to be torch.int8"), (dict(weight="float16"), "weight has to be torch.int8"),
                                          (dict(weight="uint8"), "weight has to be torch.int8"), (dict(scales="float16"), "scales has to be torch.float32"),
                                          (dict(bias="bfloat16"), "bias has to be torch.float32")], ids=str)
def test_weights_of_other_types_are_refused(mlel, change, word, k):
    """Rows on 16-byte boundaries or not: nothing is converted in silence."""
    import torch
    from mlel_b200 import serving
    types = {**dict(weight="int8", scales="float32", bias="float32"), **change}
    operands = [torch.zeros(*shape, dtype=getattr(torch, types[name])) for name, shape in (("weight", (5, k)), ("scales", (5,)), ("bias", (5,)))]
    with pytest.raises(TypeError, match=word):
        serving.QuantizedLinear(*operands)


def test_python_layer_refuses_host_tensors(mlel):
    import torch
    from mlel_b200 import serving
    with pytest.raises(ValueError, match="CUDA"):
        serving.quantize_rows(torch.zeros(3, 4))
    with pytest.raises(ValueError, match="CUDA"):
        serving.PagedCache.empty(3, 2, 16, 64, device="cpu")
    with pytest.raises(TypeError, match="float64"):
        serving._pack(torch.zeros(3, 4, dtype=torch.float64))
    with pytest.raises(ValueError, match="repeats"):
        serving._pack(torch.zeros(1, 4).expand(3, 4))

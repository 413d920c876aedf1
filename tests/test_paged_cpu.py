"""Refusals of the paged-cache and log-probability entry points (nothing is launched), and the oracle's own layout."""
import ctypes

import pytest
import torch

from oracle import paged_oracle as oracle


def _buffer():
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf)
    return buf, p + (-p) % 256


def _refused(native_lib, code, text, name, *args):
    from dynaflow_b200 import _native

    assert getattr(native_lib, name)(*args) == code
    assert text in _native.last_error()


def test_page_plan_refusals(native_lib):
    keep, p = _buffer()

    def plan(requests=2, max_pages=4, num_pages=8, rows=4, page=16, per=0, lens=p, slots=p):
        return (lens, p, p, p, p, p, p, slots, p, requests, max_pages, num_pages, rows, page, per, p, None)

    _refused(native_lib, -1, "NULL", "df_page_plan", *plan(lens=None))
    _refused(native_lib, -1, "NULL", "df_page_plan", *plan(slots=None))
    _refused(native_lib, -1, "positive", "df_page_plan", *plan(requests=0))
    _refused(native_lib, -1, "positive", "df_page_plan", *plan(max_pages=0))
    _refused(native_lib, -1, "negative", "df_page_plan", *plan(rows=-1))
    _refused(native_lib, -1, "multiple of 16", "df_page_plan", *plan(page=24))
    _refused(native_lib, -3, "8192", "df_page_plan", *plan(requests=8193))
    _refused(native_lib, -3, "2^31", "df_page_plan", *plan(num_pages=1 << 27, page=32))
    _refused(native_lib, -3, "2^30", "df_page_plan", *plan(max_pages=1 << 29))
    _refused(native_lib, -3, "2^30", "df_page_plan", *plan(per=1 << 29))


def test_append_refusals(native_lib):
    keep, p = _buffer()

    def append(qkv=p, ld=384, out=p, ld_out=384, positions=4, rows=2, hq=1, hkv=1, hd=128, cache=p, pages=2, page=16):
        return (qkv, ld, out, ld_out, p, p, p, positions, rows, hq, hkv, hd, cache, pages, page, None)

    _refused(native_lib, -1, "NULL", "df_rope_append_paged4_bf16", *append(cache=None))
    _refused(native_lib, -3, "head_dim", "df_rope_append_paged4_bf16", *append(hd=64))
    _refused(native_lib, -1, "positive", "df_rope_append_paged4_bf16", *append(hkv=0))
    _refused(native_lib, -1, "positive", "df_rope_append_paged4_bf16", *append(rows=0))
    _refused(native_lib, -1, "multiple of 16", "df_rope_append_paged4_bf16", *append(page=8))
    _refused(native_lib, -1, "strides", "df_rope_append_paged4_bf16", *append(ld=380))
    _refused(native_lib, -1, "strides", "df_rope_append_paged4_bf16", *append(ld_out=388))
    _refused(native_lib, -1, "aligned", "df_rope_append_paged4_bf16", *append(qkv=p + 2))
    _refused(native_lib, -3, "2^31", "df_rope_append_paged4_bf16", *append(pages=1 << 28))


def test_wrappers_refuse_wrong_tensors():
    from dynaflow_b200 import ops

    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32)  # noqa: E731
    args = dict(page_size=16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.page_plan(i32(2), i32(2), i32(2, 3), i32(2), i32(6), i32(1), i32(3), i32(4), i32(4), **args)
    with pytest.raises(ValueError, match="seq_lens"):
        ops.page_plan(i32(3), i32(2), i32(2, 3), i32(2), i32(6), i32(1), i32(3), i32(4), i32(4), **args)
    with pytest.raises(ValueError, match="new_lens"):
        ops.page_plan(i32(2), i32(2).long(), i32(2, 3), i32(2), i32(6), i32(1), i32(3), i32(4), i32(4), **args)
    with pytest.raises(ValueError, match="page_table"):
        ops.page_plan(i32(2), i32(2), i32(3, 2).T, i32(2), i32(6), i32(1), i32(3), i32(4), i32(4), **args)
    with pytest.raises(ValueError, match="positions"):
        ops.page_plan(i32(2), i32(2), i32(2, 3), i32(2), i32(6), i32(1), i32(3), i32(4), i32(5), **args)
    qkv = torch.zeros(2, 384, dtype=torch.bfloat16)
    cache, angles = ops.paged4_cache(2, 1, 16, device="cpu"), ops.rope_angles(4, 10000.0, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.rope_append_paged4(qkv, i32(2), i32(2), angles, 1, 1, cache, page_size=16)
    with pytest.raises(ValueError, match="bf16"):
        ops.rope_append_paged4(qkv.float(), i32(2), i32(2), angles, 1, 1, cache, page_size=16)
    with pytest.raises(ValueError, match="cache"):
        ops.rope_append_paged4(qkv, i32(2), i32(2), angles, 1, 1, cache, page_size=32)
    with pytest.raises(ValueError, match="heads"):
        ops.rope_append_paged4(qkv, i32(2), i32(2), angles, 2, 1, cache, page_size=16)
    with pytest.raises(ValueError, match="angles"):
        ops.rope_append_paged4(qkv, i32(2), i32(2), angles.double(), 1, 1, cache, page_size=16)
    with pytest.raises(ValueError, match="slots"):
        ops.rope_append_paged4(qkv, i32(2), i32(3), angles, 1, 1, cache, page_size=16)
    with pytest.raises(ValueError, match="multiple"):
        ops.paged4_cache(2, 1, 20, device="cpu")


def test_oracle_cache_round_trip():
    """What is written to a slot is read back within half a step of the code, and nothing else changes."""
    g = torch.Generator().manual_seed(1)
    cache = torch.full((3, 2, 48 * 136), 0xAB, dtype=torch.uint8)
    x, y = torch.randn(5, 128, generator=g).bfloat16(), torch.randn(5, 128, generator=g).bfloat16()
    slots = [0, 17, 47, 48, 143]
    oracle.write_tokens(cache, slots, 1, 48, x, y)
    assert (cache[:, 0] == 0xAB).all() and int((cache[:, 1] != 0xAB).sum()) <= 5 * 136
    for i, s in enumerate(slots):
        k, v = oracle.read_token(cache, s, 1, 48)
        for got, want in ((k, x[i]), (v, y[i])):
            step = (want.max() - want.min()).double() / 15
            assert ((got - want.double()).abs() <= step * (0.5 + 15 * 2 ** -8)).all()     # the bf16 scale: 15 steps off by 2^-8 of one

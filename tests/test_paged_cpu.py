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


def test_attention_refusals(native_lib):
    keep, p = _buffer()
    name = "df_attention_paged4_bf16"

    def call(q=p, ld_q=512, starts=None, fresh=None, rows=2, requests=2, max_pages=4, page=16, hq=4, hkv=1, hd=128, max_new=1, scale=0.1, ws=p, ws_bytes=1 << 40):
        return (q, ld_q, p, p, p, starts, fresh, p, 512, rows, requests, max_pages, 8, page, hq, hkv, hd, max_new, scale, ws, ws_bytes, 0, p, None)

    _refused(native_lib, -1, "NULL", name, *call(ws=None))
    _refused(native_lib, -1, "together", name, *call(starts=p))
    _refused(native_lib, -1, "one row", name, *call(max_new=2))
    _refused(native_lib, -1, "one row", name, *call(rows=1))
    _refused(native_lib, -3, "head_dim", name, *call(hd=64))
    _refused(native_lib, -1, "multiple of kv_heads", name, *call(hq=3, hkv=2))
    _refused(native_lib, -1, "multiple of 16", name, *call(page=40))
    _refused(native_lib, -3, "2^31", name, *call(max_pages=1 << 28))
    _refused(native_lib, -3, "2^31", name, *call(starts=p, fresh=p, max_new=1 << 20, max_pages=1 << 20, hq=16, ld_q=2048))
    _refused(native_lib, -1, "strides", name, *call(ld_q=504))
    _refused(native_lib, -1, "aligned", name, *call(q=p + 8))
    _refused(native_lib, -1, "scale", name, *call(scale=0.0))
    _refused(native_lib, -1, "too small", name, *call(ws_bytes=1024))
    assert native_lib.df_attention_paged4_workspace_bytes(0, 4, 1, 1) == 0
    assert native_lib.df_attention_paged4_workspace_bytes(3, 4, 3, 1) == 0
    # the scratch does not grow with the cache
    assert 0 < native_lib.df_attention_paged4_workspace_bytes(256, 32, 8, 1) < 32 << 20


def test_attention_wrapper_refuses_wrong_tensors():
    from dynaflow_b200 import ops

    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32)  # noqa: E731
    q, cache = torch.zeros(2, 512, dtype=torch.bfloat16), ops.paged4_cache(4, 1, 16, device="cpu")
    ws = torch.zeros(64, dtype=torch.uint8)
    call = lambda q=q, cache=cache, table=i32(2, 3), lens=i32(2), out=q, ws=ws, **kw: ops.attention_paged4(q, cache, table, lens, out, ws, page_size=16, **kw)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        call()
    with pytest.raises(ValueError, match="bf16"):
        call(q=q.float())
    with pytest.raises(ValueError, match="Hq"):
        call(out=torch.zeros(2, 256, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="seq_lens"):
        call(lens=i32(3))
    with pytest.raises(ValueError, match="together"):
        call(new_lens=i32(2))
    with pytest.raises(ValueError, match="row_starts"):
        call(new_lens=i32(2), row_starts=i32(2))
    with pytest.raises(ValueError, match="max_new must be 1"):
        call(max_new=2)
    with pytest.raises(ValueError, match="uint8"):
        call(ws=ws.float())
    with pytest.raises(ValueError, match="positive"):
        ops.attention_paged4_workspace(2, 3, 2, device="cpu")


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


def test_logprob_refusals(native_lib):
    keep, p = _buffer()
    name = "df_token_logprobs"

    def call(logits=p, fp32=0, ld=100, id_bytes=8, rows=2, vocab=100, top=5, lp=p, tid=p, ws=p, ws_bytes=1 << 30):
        return (logits, fp32, ld, p, id_bytes, rows, vocab, top, lp, p, tid, p, ws, ws_bytes, None)

    _refused(native_lib, -1, "NULL", name, *call(logits=None))
    _refused(native_lib, -1, "NULL", name, *call(lp=None))
    _refused(native_lib, -1, "NULL", name, *call(tid=None))
    _refused(native_lib, -1, "positive", name, *call(rows=0))
    _refused(native_lib, -1, "fp32", name, *call(fp32=2))
    _refused(native_lib, -1, "4- or 8-byte", name, *call(id_bytes=2))
    _refused(native_lib, -1, "stride", name, *call(ld=99))
    _refused(native_lib, -3, "32", name, *call(top=33))
    _refused(native_lib, -3, "vocabulary", name, *call(vocab=4, top=5))
    _refused(native_lib, -1, "aligned", name, *call(logits=p + 1))
    _refused(native_lib, -1, "too small", name, *call(rows=1, vocab=2000000, ld=2000000, ws_bytes=8))
    shard = "df_token_logprobs_shard"
    _refused(native_lib, -1, "vocab_start", shard, p, 0, 100, p, 8, 2, 100, -1, 5, p, p, 1 << 30, None)
    _refused(native_lib, -1, "NULL", shard, p, 0, 100, p, 8, 2, 100, 0, 5, None, p, 1 << 30, None)
    join = "df_token_logprobs_join"
    _refused(native_lib, -1, "parts", join, p, 65, 2, 5, p, p, p, p, None)
    _refused(native_lib, -3, "top", join, p, 2, 2, 40, p, p, p, p, None)
    assert native_lib.df_token_logprobs_workspace_bytes(0, 10, 0) == 0
    assert native_lib.df_token_logprobs_record_bytes(3, 4) == 3 * (16 + 4 * 8)


def test_logprob_wrappers_refuse_wrong_tensors():
    from dynaflow_b200 import ops

    x, ids = torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.token_logprobs(x, ids, 2)
    with pytest.raises(ValueError, match="bf16 or fp32"):
        ops.token_logprobs(x.half(), ids, 2)
    with pytest.raises(ValueError, match="bf16 or fp32"):
        ops.token_logprobs(x.T, ids, 2)
    with pytest.raises(ValueError, match="ids"):
        ops.token_logprobs(x, ids[:1], 2)
    with pytest.raises(ValueError, match="top"):
        ops.token_logprobs(x, ids, 33)
    with pytest.raises(ValueError, match="top_ids"):
        ops.token_logprobs(x, ids, 2, out=ops.token_logprobs_out(2, 3, "cpu"))
    with pytest.raises(ValueError, match="record"):
        ops.token_logprobs_shard(x, ids, 0, 2, torch.zeros(8, dtype=torch.uint8), torch.zeros(8, dtype=torch.uint8))
    with pytest.raises(ValueError, match="records"):
        ops.token_logprobs_join(torch.zeros(8, dtype=torch.uint8), 2, 2, 2)


@pytest.mark.parametrize("workspace", [torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(64, dtype=torch.uint8)[::2],
                                       torch.zeros(64, dtype=torch.float32)], ids=["expanded", "strided", "float"])
def test_logprob_workspaces_are_what_their_size_says(workspace):
    # the bytes of an expanded tensor's shape are not the bytes of its storage
    from dynaflow_b200 import ops

    x, ids = torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64)
    record = torch.zeros(2 * (16 + 2 * 8), dtype=torch.uint8)
    with pytest.raises(ValueError, match="workspace"):
        ops.token_logprobs(x, ids, 2, workspace=workspace)
    with pytest.raises(ValueError, match="workspace"):
        ops.token_logprobs_shard(x, ids, 0, 2, record, workspace)

"""Tensor-level wrappers over the C ABI (``include/dynaflow_b200.h``).

PyTorch is used for device memory and streams only: every function here hands
raw device pointers and the current CUDA stream to ``libdynaflow_b200.so``.
There is no eager/PyTorch fallback; a missing library or a CPU tensor raises.

Weight layout is ``torch.nn.Linear``'s ``[out_features, in_features]``, i.e. the
layout the subgraphs of a DynaFlow-split model hold their weights in.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native
from ._native import df_status_t

DEVICE_ERRORS = {1: "DF_ERR_TIMEOUT", 2: "DF_ERR_PEER", 3: "DF_ERR_PLAN"}
_WHERE = {1: "tma-producer", 2: "mma(full)", 3: "mma(tmem-empty)", 4: "epilogue", 5: "h-ready", 16: "peer-flag", 21: "small-gemm-producer", 22: "small-gemm-mma", 23: "small-gemm-epilogue", 24: "small-gemm-partial-rows", 32: "attention-producer", 33: "attention-mma", 34: "attention-softmax",
          48: "page-plan(pages missing)", 49: "page-plan(table row full)", 50: "page-plan(rows missing)",
          51: "paged-attention"}


class DeviceStatusError(RuntimeError):
    """A kernel reported a bounded wait that ran out (the context stays usable)."""


_status: dict[int, torch.Tensor] = {}


def _dev_index(t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise RuntimeError("dynaflow_b200 ops take CUDA tensors only (there is no CPU path)")
    return t.device.index if t.device.index is not None else torch.cuda.current_device()


def status_block(device: int | torch.device | None = None) -> torch.Tensor:
    """The per-device 16-byte status block kernels report into."""
    if device is None:
        device = torch.cuda.current_device()
    idx = device.index if isinstance(device, torch.device) else int(device)
    st = _status.get(idx)
    if st is None:
        st = torch.zeros(4, dtype=torch.int32, device=f"cuda:{idx}")
        _status[idx] = st
    return st


def read_status(device=None) -> df_status_t:
    """Synchronises the current stream and returns the device status block."""
    st = status_block(device)
    host = df_status_t()
    rc = _native.load().df_status_read(st.data_ptr(), ctypes.byref(host), _stream_ptr(st))
    if rc != 0:
        raise RuntimeError(f"df_status_read failed ({rc}): {_native.last_error()}")
    return host


def check_status(device=None) -> None:
    """Raises ``DeviceStatusError`` if a kernel recorded an error; clears the block."""
    host = read_status(device)
    if host.code != 0:
        st = status_block(device)
        _native.load().df_status_clear(st.data_ptr(), _stream_ptr(st))
        raise DeviceStatusError(
            f"device status {DEVICE_ERRORS.get(host.code, host.code)} at {_WHERE.get(host.where, host.where)} "
            f"(block {host.block}, aux {host.aux})")


def set_timeout_ms(ms: int) -> None:
    rc = _native.load().df_set_timeout_ms(int(ms))
    if rc != 0:
        raise ValueError(_native.last_error())


LAUNCH_OPTIONS = {"stream_k": 0, "mlp_one_launch": 1, "operand_swap": 2, "split_k_small": 3, "decode_keys_on_lanes": 4, "dependent_launch": 5}


def set_launch_option(name: str, on: bool) -> None:
    """Switches one of the equally valid launch forms on or off (``df_set_launch_option``)."""
    rc = _native.load().df_set_launch_option(LAUNCH_OPTIONS[name], int(bool(on)))
    if rc != 0:
        raise ValueError(_native.last_error())


def _stream_ptr(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{what} failed ({rc}): {_native.last_error()}")


def _same_device(first: torch.Tensor, *others: torch.Tensor | None) -> int:
    """The index of the CUDA device that all the tensors are on."""
    idx = first.get_device()
    if idx < 0:
        _dev_index(first)
    for t in others:
        if t is not None and t.get_device() != idx:
            raise ValueError(f"all tensors of a call must be on one device, got {first.device} and {t.device}")
    return idx


# the handle alone: building torch's stream object takes longer than a small call's checks
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda idx: torch.cuda.current_stream(idx).cuda_stream)


def _launch(idx: int, what: str, *args) -> None:
    """Calls an entry point on the current stream of device ``idx``, with that device current (launches go to the current
    device)."""
    fn = getattr(_native.load(), what)
    if torch.cuda.current_device() == idx:
        rc = fn(*args, _raw_stream(idx))
    else:
        with torch.cuda.device(idx):
            rc = fn(*args, _raw_stream(idx))
    if rc != 0:
        _check(rc, what)


def _status_ptr(idx: int) -> int:
    st = _status.get(idx)
    return (status_block(idx) if st is None else st).data_ptr()


_BF16, _I32 = torch.bfloat16, torch.int32


def _int32(t: torch.Tensor, shape: tuple[int, ...]) -> bool:
    return t.dtype is _I32 and t.shape == shape and t.is_contiguous()


def _require_int32(*named: tuple[str, torch.Tensor, tuple[int, ...]]) -> None:
    for name, t, shape in named:
        if not _int32(t, shape):
            raise ValueError(f"{name} must be a contiguous int32 tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")


def _row_stride(name: str, t: torch.Tensor) -> int:
    """Of a 2-D bf16 tensor with unit inner stride."""
    stride = t.stride()
    if t.dtype is not _BF16 or len(stride) != 2 or stride[1] != 1:
        _require_bf16_2d(name, t)
    return stride[0]


def _require_bf16_2d(name: str, t: torch.Tensor) -> None:
    if t.dtype is not torch.bfloat16 or t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be a 2-D bf16 tensor with unit inner stride, got "
                         f"{t.dtype} {tuple(t.shape)} strides {t.stride()}")


_splitk_ws: dict[tuple[int, int], torch.Tensor] = {}


def splitk_workspace(device: torch.device) -> torch.Tensor:
    """Scratch for the stream-K form of the GEMMs: one per (device, stream), created on first
    use, so that launches on different streams never share partial sums."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    key = (idx, torch.cuda.current_stream(device).cuda_stream)
    ws = _splitk_ws.get(key)
    if ws is None:
        with torch.cuda.device(idx):
            ws = torch.empty(int(_native.load().df_gemm_splitk_workspace_bytes()), dtype=torch.uint8, device=device)
        _splitk_ws[key] = ws
    return ws


def gemm_bf16(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None, max_ctas: int = 0) -> torch.Tensor:
    """``out[M,N] = a[M,K] @ b[N,K].T`` (``b`` in ``nn.Linear`` layout)."""
    _require_bf16_2d("a", a)
    _require_bf16_2d("b", b)
    M, K = a.shape
    N, Kb = b.shape
    if K != Kb:
        raise ValueError(f"inner dimensions differ: a is {tuple(a.shape)}, b is {tuple(b.shape)}")
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=a.device)
    _require_bf16_2d("out", out)
    if tuple(out.shape) != (M, N):
        raise ValueError(f"out must be {(M, N)}, got {tuple(out.shape)}")
    if M == 0:
        return out
    _dev_index(a)
    st = status_block(a.device)
    ws = splitk_workspace(a.device)
    rc = _native.load().df_gemm_bf16_ws(a.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, K, a.stride(0), b.stride(0),
                                        out.stride(0), max_ctas, ws.data_ptr(), ws.numel(), st.data_ptr(),
                                        _stream_ptr(a))
    _check(rc, "df_gemm_bf16_ws")
    return out


def gateup_silu(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, out: torch.Tensor | None = None,
                max_ctas: int = 0) -> torch.Tensor:
    """``silu(x @ w_gate.T) * (x @ w_up.T)`` with the SiLU*mul fused into the GEMM epilogue."""
    _require_bf16_2d("x", x)
    _require_bf16_2d("w_gate", w_gate)
    _require_bf16_2d("w_up", w_up)
    M, H = x.shape
    I = w_gate.shape[0]
    if tuple(w_gate.shape) != (I, H) or tuple(w_up.shape) != (I, H) or w_gate.stride(0) != w_up.stride(0):
        raise ValueError("w_gate and w_up must both be [I, H] with equal row strides")
    if out is None:
        out = torch.empty((M, I), dtype=torch.bfloat16, device=x.device)
    _require_bf16_2d("out", out)
    if M == 0:
        return out
    _dev_index(x)
    st = status_block(x.device)
    ws = splitk_workspace(x.device)
    rc = _native.load().df_gateup_silu_bf16_ws(x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), out.data_ptr(), M, H, I,
                                               x.stride(0), w_gate.stride(0), out.stride(0), max_ctas, ws.data_ptr(),
                                               ws.numel(), st.data_ptr(), _stream_ptr(x))
    _check(rc, "df_gateup_silu_bf16_ws")
    return out


def mlp_workspace_bytes(M: int, H: int, I: int) -> int:
    return int(_native.load().df_mlp_workspace_bytes(M, H, I))


def gated_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
              max_ctas: int = 0) -> torch.Tensor:
    """``(silu(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T`` for one nano-batch of rows."""
    for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        _require_bf16_2d(name, t)
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    M, H = x.shape
    I = w_gate.shape[0]
    if tuple(w_gate.shape) != (I, H) or tuple(w_up.shape) != (I, H) or tuple(w_down.shape) != (H, I):
        raise ValueError("expected w_gate, w_up: [I, H] and w_down: [H, I]")
    if out is None:
        out = torch.empty((M, H), dtype=torch.bfloat16, device=x.device)
    if not out.is_contiguous() or tuple(out.shape) != (M, H) or out.dtype != torch.bfloat16:
        raise ValueError("out must be a contiguous bf16 [M, H] tensor")
    if M == 0:
        return out
    need = mlp_workspace_bytes(M, H, I)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    if workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace too small: need {need} bytes")
    _dev_index(x)
    st = status_block(x.device)
    rc = _native.load().df_mlp_gated_bf16(x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(),
                                          out.data_ptr(), workspace.data_ptr(), M, H, I, max_ctas, st.data_ptr(),
                                          _stream_ptr(x))
    _check(rc, "df_mlp_gated_bf16")
    return out


def attention_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, *, batch: int, seq_len: int,
                      cu_seqlens: torch.Tensor | None = None, scale: float | None = None, max_ctas: int = 0) -> torch.Tensor:
    """Causal grouped-query attention of a prefill nano-batch. ``q [T, Hq*128]``, ``k, v [T, Hkv*128]``,
    ``out [T, Hq*128]``: 2-D bf16 views with unit inner stride (column ranges of a fused qkv
    activation are fine). The ``T`` rows are ``batch`` sequences back to back, each ``seq_len``
    long, or starting at ``cu_seqlens[b]`` (int32 on the device, ``batch + 1`` entries; ``seq_len``
    is then the longest length)."""
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out)):
        _require_bf16_2d(name, t)
    T = q.shape[0]
    hd = 128
    if q.shape[1] % hd or k.shape[1] % hd or tuple(k.shape) != tuple(v.shape) or tuple(out.shape) != tuple(q.shape) \
            or k.shape[0] != T:
        raise ValueError("expected q/out [T, Hq*128] and k/v [T, Hkv*128]")
    if T == 0:
        return out
    if cu_seqlens is not None and (cu_seqlens.dtype != torch.int32 or not cu_seqlens.is_cuda
                                   or cu_seqlens.numel() != batch + 1):
        raise ValueError("cu_seqlens must be an int32 device tensor of batch + 1 entries")
    _dev_index(q)
    st = status_block(q.device)
    rc = _native.load().df_attention_prefill_bf16(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), T, batch, seq_len,
        cu_seqlens.data_ptr() if cu_seqlens is not None else None, q.shape[1] // hd, k.shape[1] // hd, hd,
        q.stride(0), k.stride(0), v.stride(0), out.stride(0), float(scale if scale is not None else hd ** -0.5),
        max_ctas, st.data_ptr(), _stream_ptr(q))
    _check(rc, "df_attention_prefill_bf16")
    return out


def attention_decode_workspace_bytes(batch: int, q_heads: int, kv_heads: int, max_len: int) -> int:
    return int(_native.load().df_attention_decode_workspace_bytes(batch, q_heads, kv_heads, max_len))


def attention_decode_workspace(batch: int, q_heads: int, kv_heads: int, max_len: int,
                               device: torch.device | str = "cuda") -> torch.Tensor:
    """Scratch for ``attention_decode`` (the chunks' partial results); its contents are arbitrary."""
    return torch.empty(attention_decode_workspace_bytes(batch, q_heads, kv_heads, max_len), dtype=torch.uint8, device=device)


def rope_append(qkv: torch.Tensor, seq_lens: torch.Tensor, q_heads: int, kv_heads: int, k_cache: torch.Tensor,
                v_cache: torch.Tensor, theta: float) -> None:
    """Rotary embedding of the new token's query and key heads (position ``seq_lens[b] - 1``) in place in
    ``qkv [B, (Hq + 2 Hkv) * 128]``, rotated keys and values into that position of the caches, one launch."""
    _require_bf16_2d("qkv", qkv)
    B = qkv.shape[0]
    if k_cache.dim() != 3 or not k_cache.is_contiguous() or not v_cache.is_contiguous() or k_cache.shape[0] != B \
            or k_cache.shape[2] != kv_heads * 128 or tuple(v_cache.shape) != tuple(k_cache.shape):
        raise ValueError("expected contiguous bf16 caches [B, max_len, Hkv*128]")
    rc = _native.load().df_rope_append_bf16(qkv.data_ptr(), qkv.stride(0), seq_lens.data_ptr(), B, q_heads, kv_heads, 128,
                                            float(theta), k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[2],
                                            k_cache.shape[1], _stream_ptr(qkv))
    _check(rc, "df_rope_append_bf16")


def attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, seq_lens: torch.Tensor,
                     out: torch.Tensor, workspace: torch.Tensor, *, scale: float | None = None,
                     max_ctas: int = 0) -> torch.Tensor:
    """One new token per sequence against its key/value cache. ``q, out [B, Hq*128]`` (2-D bf16
    views, unit inner stride), ``k_cache, v_cache [B, max_len, Hkv*128]`` contiguous bf16,
    ``seq_lens`` int32 on the device, ``workspace`` from ``attention_decode_workspace``."""
    _require_bf16_2d("q", q)
    _require_bf16_2d("out", out)
    hd = 128
    B = q.shape[0]
    if k_cache.dtype != torch.bfloat16 or k_cache.dim() != 3 or not k_cache.is_contiguous() \
            or tuple(v_cache.shape) != tuple(k_cache.shape) or not v_cache.is_contiguous() or k_cache.shape[0] != B:
        raise ValueError("expected contiguous bf16 caches [B, max_len, Hkv*128]")
    max_len, kv_cols = k_cache.shape[1], k_cache.shape[2]
    if q.shape[1] % hd or kv_cols % hd or tuple(out.shape) != tuple(q.shape):
        raise ValueError("expected q/out [B, Hq*128] and caches [B, max_len, Hkv*128]")
    if seq_lens.dtype != torch.int32 or not seq_lens.is_cuda or seq_lens.numel() != B:
        raise ValueError("seq_lens must be an int32 device tensor of B entries")
    _dev_index(q)
    st = status_block(q.device)
    rc = _native.load().df_attention_decode_bf16(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), seq_lens.data_ptr(), B, max_len,
        q.shape[1] // hd, kv_cols // hd, hd, q.stride(0), kv_cols, out.stride(0),
        float(scale if scale is not None else hd ** -0.5), workspace.data_ptr(), workspace.numel(), max_ctas,
        st.data_ptr(), _stream_ptr(q))
    _check(rc, "df_attention_decode_bf16")
    return out


def kv_cache_append(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    seq_lens: torch.Tensor) -> None:
    """``cache[b, seq_lens[b] - 1] = new[b]`` for keys and values (``k_new, v_new [B, Hkv*128]`` views
    with equal row strides)."""
    _require_bf16_2d("k_new", k_new)
    _require_bf16_2d("v_new", v_new)
    if k_new.stride(0) != v_new.stride(0) or tuple(k_new.shape) != tuple(v_new.shape):
        raise ValueError("k_new and v_new must have equal shapes and row strides")
    B, cols = k_new.shape
    rc = _native.load().df_kv_cache_append_bf16(k_new.data_ptr(), v_new.data_ptr(), k_new.stride(0), k_cache.data_ptr(),
                                                v_cache.data_ptr(), cols, seq_lens.data_ptr(), B, k_cache.shape[1],
                                                cols // 128, 128, _stream_ptr(k_new))
    _check(rc, "df_kv_cache_append_bf16")


STATIC_SCRATCH_BYTES = 64 << 20


def gated_mlp_static(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                     out: torch.Tensor, max_ctas: int = 0) -> torch.Tensor:
    """``gated_mlp`` for callers that cannot provide or allocate scratch (a policy
    substitute that only holds the subgraph's tensors, a host whose HBM is fully
    budgeted): the intermediate lives in a 64 MiB array inside the library, so
    ``rows * I * 2`` must not exceed ``STATIC_SCRATCH_BYTES`` and ``out`` must be
    passed in. This wrapper itself creates no tensor. Calls that may overlap on the
    GPU share that array and race; the first call on a device should happen
    outside stream capture (it looks up the array's address)."""
    for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down), ("out", out)):
        _require_bf16_2d(name, t)
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    M, H = x.shape
    I = w_gate.shape[0]
    if tuple(w_gate.shape) != (I, H) or tuple(w_up.shape) != (I, H) or tuple(w_down.shape) != (H, I):
        raise ValueError("expected w_gate, w_up: [I, H] and w_down: [H, I]")
    if tuple(out.shape) != (M, H):
        raise ValueError("out must be [M, H]")
    if M == 0:
        return out
    _dev_index(x)
    st = status_block(x.device)
    rc = _native.load().df_mlp_gated_bf16_static(x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(),
                                                 out.data_ptr(), M, H, I, max_ctas, st.data_ptr(), _stream_ptr(x))
    _check(rc, "df_mlp_gated_bf16_static")
    return out


# ------------------------------------------------------ paged 4-bit key/value cache
PAGE_GRANULE = 16          # page sizes are multiples of this many tokens
PAGED4_TOKEN_BYTES = 136   # one token of one key/value head: 64 bytes of codes and 4 of parameters, for key and value


def paged4_cache(num_pages: int, kv_heads: int, page_size: int, device: torch.device | str = "cuda") -> torch.Tensor:
    """One layer's cache, ``uint8 [num_pages, kv_heads, page_size * 136]`` (contents arbitrary: only slots that were
    written are read)."""
    if num_pages <= 0 or kv_heads <= 0 or page_size <= 0 or page_size % PAGE_GRANULE:
        raise ValueError(f"num_pages and kv_heads must be positive, page_size a multiple of {PAGE_GRANULE}")
    return torch.empty(num_pages, kv_heads, page_size * PAGED4_TOKEN_BYTES, dtype=torch.uint8, device=device)


def _paged4_shape(cache: torch.Tensor, page_size: int) -> tuple[int, int]:
    """Pages and key/value heads of a cache."""
    shape = cache.shape
    if cache.dtype is not torch.uint8 or len(shape) != 3 or not cache.is_contiguous() or page_size <= 0 or page_size % PAGE_GRANULE \
            or shape[2] != page_size * PAGED4_TOKEN_BYTES:
        raise ValueError(f"expected a contiguous uint8 cache [pages, kv_heads, page_size * {PAGED4_TOKEN_BYTES}], page_size a "
                         f"multiple of {PAGE_GRANULE}; got {cache.dtype} {tuple(shape)} and page_size {page_size}")
    return shape[0], shape[1]


def page_plan(seq_lens: torch.Tensor, new_lens: torch.Tensor, page_table: torch.Tensor, page_counts: torch.Tensor,
              free_pages: torch.Tensor, free_count: torch.Tensor, row_starts: torch.Tensor, slots: torch.Tensor,
              positions: torch.Tensor, *, page_size: int, rows_per_request: int = 0) -> None:
    """Page tables, slots and positions of a step, on the device (``df_page_plan``): request ``b`` is ``seq_lens[b]`` tokens
    long after the step, ``new_lens[b]`` of them new. Updates ``page_table [B, max_pages]``, ``page_counts [B]`` and the free
    list ``free_pages [num_pages]`` / ``free_count [1]`` (pages no longer needed are given back first, so length 0 ends a
    request); writes ``row_starts [B + 1]`` and, per row, ``slots`` and ``positions`` (``-1`` and 0 where there is no token).
    ``rows_per_request`` 0: new tokens back to back; else request ``b`` owns rows ``b * rows_per_request ...``. All int32.
    Too few free pages, a full table row or too few rows are reported by ``check_status``."""
    if page_table.dim() != 2:
        raise ValueError(f"page_table must be [requests, max_pages], got {tuple(page_table.shape)}")
    B, max_pages = table = tuple(page_table.shape)
    num_pages, rows = free_pages.numel(), slots.numel()
    one, per_row = (B,), (rows,)
    if not (_int32(page_table, table) and _int32(seq_lens, one) and _int32(new_lens, one) and _int32(page_counts, one)
            and _int32(free_pages, (num_pages,)) and _int32(free_count, (1,)) and _int32(row_starts, (B + 1,))
            and _int32(slots, per_row) and _int32(positions, per_row)):
        _require_int32(("page_table", page_table, table), ("seq_lens", seq_lens, one), ("new_lens", new_lens, one),
                       ("page_counts", page_counts, one), ("free_pages", free_pages, (num_pages,)), ("free_count", free_count, (1,)),
                       ("row_starts", row_starts, (B + 1,)), ("slots", slots, per_row), ("positions", positions, per_row))
    if B == 0:
        raise ValueError("page_plan needs at least one request")
    idx = _same_device(page_table, seq_lens, new_lens, page_counts, free_pages, free_count, row_starts, slots, positions)
    _launch(idx, "df_page_plan", seq_lens.data_ptr(), new_lens.data_ptr(), page_table.data_ptr(), page_counts.data_ptr(),
            free_pages.data_ptr(), free_count.data_ptr(), row_starts.data_ptr(), slots.data_ptr(), positions.data_ptr(), B,
            max_pages, num_pages, rows, page_size, rows_per_request, _status_ptr(idx))


def rope_angles(num_positions: int, theta: float, device: torch.device | str = "cuda") -> torch.Tensor:
    """``[num_positions, 128]`` fp32: cos, then sin, of the 64 rotary angles of every position (formed in 64 bits: a
    32-bit angle of a far position is off by more than a bf16 step)."""
    freq = theta ** (-torch.arange(64, dtype=torch.float64, device=device) / 64)
    angle = torch.arange(num_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def rope_append_paged4(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, angles: torch.Tensor, q_heads: int,
                       kv_heads: int, cache: torch.Tensor, *, page_size: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary embedding of the query and key heads of ``qkv [rows, (Hq + 2 Hkv) * 128]`` at ``positions``, keys and values
    quantised into the ``slots`` of a paged 4-bit cache, one launch. ``out`` (default: in place) receives the rotated queries,
    and keys and values as the cache stands for them, so that attention over these rows sees what later steps will see.
    Rows with a slot or position out of range are padding: left as they are in ``out``. ``angles`` from ``rope_angles``."""
    ld = _row_stride("qkv", qkv)
    num_pages, heads = _paged4_shape(cache, page_size)
    rows, cols = shape = qkv.shape
    if out is None:
        out, ld_out = qkv, ld
    else:
        ld_out = _row_stride("out", out)
        if out.shape != shape:
            raise ValueError(f"out must be {(rows, cols)}, got {tuple(out.shape)}")
    if cols != (q_heads + 2 * kv_heads) * 128 or heads != kv_heads:
        raise ValueError("expected qkv [rows, (q_heads + 2 kv_heads) * 128] and a cache of kv_heads heads")
    angle_shape, per_row = angles.shape, (rows,)
    if angles.dtype is not torch.float32 or len(angle_shape) != 2 or angle_shape[1] != 128 or not angles.is_contiguous():
        raise ValueError("angles must be a contiguous fp32 tensor [positions, 128]")
    if not (_int32(positions, per_row) and _int32(slots, per_row)):
        _require_int32(("positions", positions, per_row), ("slots", slots, per_row))
    idx = _same_device(qkv, positions, slots, angles, cache, out)
    if rows == 0:
        return out
    _launch(idx, "df_rope_append_paged4_bf16", qkv.data_ptr(), ld, out.data_ptr(), ld_out, positions.data_ptr(), slots.data_ptr(),
            angles.data_ptr(), angle_shape[0], rows, q_heads, kv_heads, 128, cache.data_ptr(), num_pages, page_size)
    return out


def attention_paged4_workspace(requests: int, q_heads: int, kv_heads: int, max_new: int = 1,
                               device: torch.device | str = "cuda") -> torch.Tensor:
    """Scratch for ``attention_paged4`` (partial results of cut requests), zeroed: its counters are zero between calls. Calls
    that can overlap on the GPU, captured graphs included, need one each."""
    need = int(_native.load().df_attention_paged4_workspace_bytes(requests, q_heads, kv_heads, max_new))
    if need == 0:
        raise ValueError("requests, max_new and the head counts must be positive, q_heads a multiple of kv_heads")
    return torch.zeros(need, dtype=torch.uint8, device=device)


def attention_paged4(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, out: torch.Tensor,
                     workspace: torch.Tensor, *, page_size: int, row_starts: torch.Tensor | None = None,
                     new_lens: torch.Tensor | None = None, max_new: int = 1, scale: float | None = None,
                     max_ctas: int = 0) -> torch.Tensor:
    """The new tokens' attention over a paged 4-bit cache. ``q, out [rows, Hq * 128]`` (2-D bf16 views, unit inner stride),
    ``cache [pages, Hkv, page_size * 136]``, ``page_table [B, max_pages]`` and ``seq_lens [B]`` int32. Without ``new_lens``
    row ``b`` is request ``b``'s one new token; with ``row_starts [B + 1]`` and ``new_lens [B]`` (from ``page_plan``) request ``b``
    has rows ``row_starts[b] ...``, at most ``max_new``, causal among themselves. Rows of no request keep what they held, a row
    without keys is zeros. Lengths past what a row of the table holds are limited to that."""
    ld_q, ld_out = _row_stride("q", q), _row_stride("out", out)
    num_pages, kv_heads = _paged4_shape(cache, page_size)
    rows, cols = shape = q.shape
    if cols == 0 or cols % (128 * kv_heads) or out.shape != shape:
        raise ValueError("expected q/out [rows, Hq * 128], Hq a multiple of the cache's heads")
    if page_table.dim() != 2:
        raise ValueError(f"page_table must be [requests, max_pages], got {tuple(page_table.shape)}")
    B, max_pages = table = tuple(page_table.shape)
    if not (_int32(page_table, table) and _int32(seq_lens, (B,))):
        _require_int32(("page_table", page_table, table), ("seq_lens", seq_lens, (B,)))
    starts = lens = None
    if row_starts is not None or new_lens is not None:
        if row_starts is None or new_lens is None:
            raise ValueError("row_starts and new_lens come together")
        _require_int32(("row_starts", row_starts, (B + 1,)), ("new_lens", new_lens, (B,)))
        starts, lens = row_starts.data_ptr(), new_lens.data_ptr()
    elif max_new != 1 or rows < B:
        raise ValueError("without new_lens every request has one row: max_new must be 1, q at least as many rows as requests")
    if workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 tensor")
    idx = _same_device(q, cache, page_table, seq_lens, out, workspace, row_starts, new_lens)
    if rows == 0 or B == 0:
        return out
    _launch(idx, "df_attention_paged4_bf16", q.data_ptr(), ld_q, cache.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(), starts,
            lens, out.data_ptr(), ld_out, rows, B, max_pages, num_pages, page_size, cols // 128, kv_heads, 128, max_new,
            128 ** -0.5 if scale is None else scale, workspace.data_ptr(), workspace.nbytes, max_ctas, _status_ptr(idx))
    return out


# ------------------------------------------------------------ token log probabilities
MAX_TOP_TOKENS = 32


def token_logprobs_out(rows: int, top: int, device: torch.device | str = "cuda") -> tuple[torch.Tensor, ...]:
    """Result tensors of ``token_logprobs``: log probabilities and entropies ``[rows]`` fp32, the most likely tokens' ids
    (int32) and log probabilities (fp32) ``[rows, top]``."""
    return (torch.empty(rows, dtype=torch.float32, device=device), torch.empty(rows, dtype=torch.float32, device=device),
            torch.empty(rows, top, dtype=torch.int32, device=device), torch.empty(rows, top, dtype=torch.float32, device=device))


def token_logprobs_workspace(rows: int, vocab: int, top: int, device: torch.device | str = "cuda") -> torch.Tensor:
    """Scratch for ``token_logprobs`` / ``token_logprobs_shard``; its contents are arbitrary. Calls that can overlap on the
    GPU, captured graphs included, need one each."""
    need = int(_native.load().df_token_logprobs_workspace_bytes(rows, vocab, top))
    if need == 0:
        raise ValueError(f"rows and vocab must be positive, top 0 to {MAX_TOP_TOKENS}")
    return torch.empty(need, dtype=torch.uint8, device=device)


def _require_logits(logits: torch.Tensor, ids: torch.Tensor) -> tuple[int, int, int, bool]:
    """Rows, vocabulary, row stride, and whether the logits are fp32."""
    stride, dtype = logits.stride(), logits.dtype
    if len(stride) != 2 or (dtype is not _BF16 and dtype is not torch.float32) or stride[1] != 1:
        raise ValueError(f"logits must be 2-D bf16 or fp32 with unit inner stride, got {dtype} {tuple(logits.shape)} strides {stride}")
    rows, vocab = logits.shape
    if (ids.dtype is not torch.int64 and ids.dtype is not _I32) or ids.shape != (rows,) or not ids.is_contiguous():
        raise ValueError(f"ids must be a contiguous int32 or int64 tensor of {rows} entries, got {ids.dtype} {tuple(ids.shape)}")
    return rows, vocab, stride[0], dtype is not _BF16


def _require_logprobs_workspace(workspace: torch.Tensor) -> None:
    if workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous uint8 tensor, got {workspace.dtype} strides {workspace.stride()}")


def _require_logprobs_out(out: tuple[torch.Tensor, ...], rows: int, top: int) -> None:
    lp, ent, tid, tlp = out
    for name, t, dtype, shape in (("logprob", lp, torch.float32, (rows,)), ("entropy", ent, torch.float32, (rows,)),
                                  ("top_ids", tid, _I32, (rows, top)), ("top_logprobs", tlp, torch.float32, (rows, top))):
        if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top: int = 0, *, out: tuple[torch.Tensor, ...] | None = None,
                   workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, ...]:
    """``(logprob, entropy, top_ids, top_logprobs)`` of ``logits [rows, vocab]`` (bf16 or fp32, any row stride): the log
    probability of ``ids [rows]``, the entropy (nats), and the ``top`` most likely tokens, largest first, of equal logits the
    lower index first. Forbidden tokens are ``-inf`` (logits of ``-2**123`` and lower count as such beside higher ones); a row of
    nothing else has log probabilities ``-inf`` and entropy 0."""
    rows, vocab, ld, fp32 = _require_logits(logits, ids)
    if out is None:
        out = token_logprobs_out(rows, top, logits.device)
    else:
        _require_logprobs_out(out, rows, top)
    if workspace is None and rows > 0:
        workspace = token_logprobs_workspace(rows, vocab, top, logits.device)
    elif workspace is not None:
        _require_logprobs_workspace(workspace)
    idx = _same_device(logits, ids, workspace, *out)
    if rows == 0:
        return out
    lp, ent, tid, tlp = out
    _launch(idx, "df_token_logprobs", logits.data_ptr(), fp32, ld, ids.data_ptr(),
            ids.element_size(), rows, vocab, top, lp.data_ptr(), ent.data_ptr(), tid.data_ptr(), tlp.data_ptr(),
            workspace.data_ptr(), workspace.nbytes)
    return out


def token_logprobs_record(rows: int, top: int, device: torch.device | str = "cuda") -> torch.Tensor:
    """One rank's record of ``rows`` rows (``token_logprobs_shard`` fills it)."""
    need = int(_native.load().df_token_logprobs_record_bytes(rows, top))
    if need == 0:
        raise ValueError(f"rows must be positive, top 0 to {MAX_TOP_TOKENS}")
    return torch.empty(need, dtype=torch.uint8, device=device)


def token_logprobs_shard(logits: torch.Tensor, ids: torch.Tensor, vocab_start: int, top: int, record: torch.Tensor,
                         workspace: torch.Tensor) -> torch.Tensor:
    """This rank's part of ``token_logprobs`` when ``logits`` are tokens ``vocab_start ...`` of a split vocabulary (``ids`` are of
    the whole one). The ranks' records, all-gathered in rank order, give the results with ``token_logprobs_join``."""
    rows, vocab, ld, fp32 = _require_logits(logits, ids)
    if record.dtype != torch.uint8 or not record.is_contiguous() or record.numel() < int(_native.load().df_token_logprobs_record_bytes(rows, top)):
        raise ValueError("record must be a contiguous uint8 tensor from token_logprobs_record")
    _require_logprobs_workspace(workspace)
    idx = _same_device(logits, ids, record, workspace)
    if rows == 0:
        return record
    _launch(idx, "df_token_logprobs_shard", logits.data_ptr(), fp32, ld, ids.data_ptr(),
            ids.element_size(), rows, vocab, vocab_start, top, record.data_ptr(), workspace.data_ptr(),
            workspace.nbytes)
    return record


def token_logprobs_join(records: torch.Tensor, parts: int, rows: int, top: int, *, out: tuple[torch.Tensor, ...] | None = None) -> tuple[torch.Tensor, ...]:
    """The results from the ``parts`` ranks' records, one behind the other."""
    each = int(_native.load().df_token_logprobs_record_bytes(rows, top))
    if each == 0 or records.dtype != torch.uint8 or not records.is_contiguous() or records.numel() != parts * each:
        raise ValueError("records must be a contiguous uint8 tensor of the ranks' records")
    if out is None:
        out = token_logprobs_out(rows, top, records.device)
    else:
        _require_logprobs_out(out, rows, top)
    idx = _same_device(records, *out)
    lp, ent, tid, tlp = out
    _launch(idx, "df_token_logprobs_join", records.data_ptr(), parts, rows, top, lp.data_ptr(), ent.data_ptr(), tid.data_ptr(),
            tlp.data_ptr())
    return out

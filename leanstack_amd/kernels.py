"""Torch-tensor wrappers of the C ABI: projections and the greedy lm_head.

Tensors are device memory that torch owns; the kernels run on torch's current
HIP stream (``torch.cuda.current_stream().cuda_stream`` is a hipStream_t on
ROCm), as the cuTile head launches on the current stream
(src/leanstack/runtime/cutile_logits.py:59).  Nothing here falls back to
another implementation: a missing library or a rejected argument raises.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools

import torch

from . import _lib
from .adapters import AdapterStore
from .layout import PackedWeight
from .paged_cache import PagedKVCache


# The wrappers run for every projection of every token, so their host time is
# kept below the kernels': tensor attributes that need no Python object
# (is_cuda, get_device), the raw stream handle and device index straight from
# torch's bindings, a device switch only where the call's device is not the
# current one, and sizes that depend on the shape alone looked up once.  One
# decode layer of five calls: 89 -> 52 us, the kernels' own time.
_NO_SWITCH = contextlib.nullcontext()


def _on(device: torch.device):
    """Context in which a GPU tensor's `device` is current."""
    return _NO_SWITCH if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def _on_index(index: int):
    """_on() for a device's index."""
    return _NO_SWITCH if torch._C._cuda_getDevice() == index else torch.cuda.device(index)


def _require_device(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{what} must be a GPU tensor, got device {t.device}")


def _one_device(first: torch.Tensor, *named: tuple[torch.Tensor | None, str]) -> torch.device:
    """The device of `first`, after checking that every other tensor given
    (None skipped) lives on it: the C layer launches on one device and sees
    only pointers."""
    index, dev = first.get_device(), first.device
    for t, what in named:
        if t is not None and (t.get_device() != index or (index < 0 and t.device != dev)):
            raise ValueError(f"{what} is on {t.device}, the call's tensors are on {dev}")
    return dev


def _rows(x: torch.Tensor, k: int, what: str) -> tuple[torch.Tensor, int, int]:
    """x as [M, k] rows with unit column stride: the tensor whose data_ptr()
    they start at, M, and the row stride.  Rows the kernels cannot read in
    place (column stride, row stride not a multiple of 8 or above the
    library's largest, misalignment) are copied."""
    if x.dtype is not torch.bfloat16:
        raise ValueError(f"{what} must be bfloat16, got {x.dtype}")
    if x.shape[-1] != k:
        raise ValueError(f"{what} last dim {x.shape[-1]} != K={k}")
    if x.is_contiguous() and k % 8 == 0 and k <= _lib.MAX_ACTIVATION_STRIDE and x.data_ptr() % 16 == 0:
        return x, x.numel() // k, k
    x2 = x.reshape(-1, k)
    if (x2.stride(-1) != 1 or (x2.shape[0] > 1 and (x2.stride(0) % 8 or x2.stride(0) > _lib.MAX_ACTIVATION_STRIDE))
            or x2.data_ptr() % 16):
        x2 = x2.clone(memory_format=torch.contiguous_format)  # (contiguous() keeps a misaligned start)
    ld = x2.stride(0) if x2.shape[0] > 1 else k
    return x2, x2.shape[0], ld


def stream_handle() -> int:
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _check_out(out: torch.Tensor, m: int, n_out: int, dtype: torch.dtype, what: str = "out") -> None:
    """A caller-supplied output must hold exactly the m x n_out values the
    kernel writes, contiguously: the C layer sees only a pointer."""
    if out.dtype != dtype or out.shape[-1:] != (n_out,) or out.numel() != m * n_out or not out.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of {m} x {n_out} values "
                         f"(got {out.dtype} {tuple(out.shape)})")


def _device_index(device: torch.device) -> int:
    return device.index if device.index is not None else torch.cuda.current_device()


def _device_workspace(cache: dict[tuple[int, int], torch.Tensor], device: torch.device, nbytes: int,
                      what: str) -> torch.Tensor:
    """The zero-filled workspace of `cache` for `device` and the current
    stream, grown to `nbytes`.  One per (device, stream): the split blocks of
    a call count arrivals in the workspace's flag words and read each other's
    partial slots, so two calls that overlap must not share one, and calls on
    one stream are ordered.  It is never allocated while the stream is being
    captured, so a captured graph never replays a workspace's allocation or
    zero fill (run the same launch once on the capture stream before the
    capture); a graph keeps using the workspace of the stream it was captured
    on, so eager calls on that stream must not overlap its replays."""
    index = _device_index(device)
    key = (index, torch._C._cuda_getCurrentRawStream(index))
    ws = cache.get(key)
    if ws is None or ws.numel() < nbytes:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"the {what} workspace must be allocated before graph capture: run the same "
                               f"launch once on the capture stream, outside the capture, first")
        ws = torch.zeros(nbytes, device=device, dtype=torch.uint8)
        cache[key] = ws
    return ws


_prefill_workspaces: dict[tuple[int, int], torch.Tensor] = {}


@functools.lru_cache(maxsize=4096)
def _linear_workspace_bytes(current_device: int, m: int, n: int, k: int) -> int:
    """lsk_workspace_bytes of a projection: a function of the shape and the
    current device's CU count."""
    return _lib.load().lsk_workspace_bytes(_lib.OP_LINEAR, m, n, k)


def prefill_workspace(device: torch.device, m: int, n: int, k: int) -> torch.Tensor | None:
    """The split-K workspace of the prefill GEMM on `device` for the current
    stream (zero-filled once, left zero-filled by every call), or None when
    the shape does not use one."""
    nbytes = _linear_workspace_bytes(torch._C._cuda_getDevice(), m, n, k)
    if nbytes == 0:
        return None
    return _device_workspace(_prefill_workspaces, device, nbytes, "prefill")


def set_linear_wait_limit(polls: int) -> None:
    """Polls of a split-K arrival word before a prefill workgroup gives up
    (then the workspace's error word is set and its tiles are NaN)."""
    _lib.load().lsk_set_linear_wait_limit(int(polls))


LINEAR_WAIT_LIMIT_DEFAULT = 1 << 22


def kernel_durations_us(fn, max_dispatches: int = 4096) -> list[float]:
    """Run fn() (eager launches of this library's kernels on the current
    stream) with every dispatch timed by events bound to the dispatch itself
    (lsk_dispatch_timing_begin/end), and return each kernel's own duration in
    microseconds, in launch order.  Waits for the timed kernels."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("dispatch timing cannot run inside a graph capture")
    lib = _lib.load()
    _lib.check(lib.lsk_dispatch_timing_begin(int(max_dispatches)), "lsk_dispatch_timing_begin")
    durations = (ctypes.c_float * int(max_dispatches))()
    count = ctypes.c_int(0)
    try:
        fn()
    finally:
        status = lib.lsk_dispatch_timing_end(durations, int(max_dispatches), ctypes.byref(count))
    _lib.check(status, "lsk_dispatch_timing_end")
    return [float(durations[i]) for i in range(min(count.value, int(max_dispatches)))]


def linear_error(workspace: torch.Tensor) -> int:
    """Read and clear the error word of a prefill workspace (0 = no bounded
    wait gave up since the last read).  Synchronous."""
    err = ctypes.c_int(0)
    _lib.check(_lib.load().lsk_linear_error(workspace.data_ptr(), ctypes.byref(err)), "lsk_linear_error")
    return err.value


def linear(x: torch.Tensor, weight: PackedWeight, *, epilogue: int = _lib.EPI_NONE,
           residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
           workspace: torch.Tensor | None | str = "auto") -> torch.Tensor:
    """out[..., N'] = epilogue(x[..., K] . W^T) on the GPU.

    epilogue EPI_NONE (N' = N), EPI_SILU_MUL (gate_up layout, N' = N/2,
    SiLU(gate)*up), EPI_RESIDUAL_ADD (N' = N, residual + projection).
    workspace: "auto" uses the split-K workspace of the device and current
    stream for prefill shapes (prefill_workspace), None runs one
    workgroup per output block with no waits (the form for prefill calls
    that may run concurrently with other kernels on the device), a uint8
    device tensor is used as given.  A split-K workgroup whose bounded wait
    gives up (possible only when another kernel holds CUs the split needs)
    sets the workspace's error word (linear_error) and writes NaN to its
    tiles."""
    if not isinstance(weight, PackedWeight):
        raise ValueError("weight must be a PackedWeight (pack it with leanstack_amd.layout / leanserve)")
    lib = _lib.load()
    x2, m, ldx = _rows(x, weight.k, "x")
    n_out = weight.n // 2 if epilogue == _lib.EPI_SILU_MUL else weight.n
    if out is not None:
        _check_out(out, m, n_out, torch.bfloat16)
    r2 = None
    if residual is not None:
        r2, rm, ldr = _rows(residual, weight.n, "residual")
        if rm != m:
            raise ValueError(f"residual has {rm} rows, x has {m}")
    _require_device(x, "x")
    _require_device(weight.data, "weight")
    if out is None:
        out = x.new_empty((*x.shape[:-1], n_out))
    _require_device(out, "out")
    res_ptr, ldr = (None, 0) if r2 is None else (r2.data_ptr(), ldr)
    if r2 is not None:
        _require_device(r2, "residual")
    if m == 0:
        return out  # no rows: nothing to launch (F.linear returns the empty result too)
    if isinstance(workspace, str):
        if workspace != "auto":
            raise ValueError(f"workspace must be 'auto', None or a tensor, not {workspace!r}")
        workspace = prefill_workspace(x.device, m, weight.n, weight.k) if m > _lib.DECODE_MAX_M else None
    ws_ptr, ws_bytes = None, 0
    if workspace is not None:
        _require_device(workspace, "workspace")
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    dev = _one_device(x, (weight.data, "weight"), (out, "out"), (r2, "residual"), (workspace, "workspace"))
    with _on(dev):
        status = lib.lsk_linear_bf16(
            weight.data.data_ptr(), weight.layout, weight.n, weight.k,
            x2.data_ptr(), m, ldx,
            out.data_ptr(), n_out,
            epilogue, res_ptr, ldr,
            ws_ptr, ws_bytes, stream_handle(),
        )
    _lib.check(status, "lsk_linear_bf16")
    return out


def rmsnorm_linear(x: torch.Tensor, norm_weight: torch.Tensor, eps: float, weight: PackedWeight, *,
                   epilogue: int = _lib.EPI_NONE, residual: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """out[..., N'] = epilogue(rms_norm(x) . W^T) for 1..16 rows of x, the
    RMSNorm (F.rms_norm over the last dim with `norm_weight` and `eps`, one
    bf16 rounding) computed inside the projection kernel."""
    if not isinstance(weight, PackedWeight):
        raise ValueError("weight must be a PackedWeight (pack it with leanstack_amd.layout / leanserve)")
    lib = _lib.load()
    x2, m, ldx = _rows(x, weight.k, "x")
    nw = norm_weight.reshape(-1)
    if nw.dtype != torch.bfloat16 or nw.numel() != weight.k:
        raise ValueError(f"norm_weight must be a bfloat16 [{weight.k}] tensor, got {nw.dtype} {tuple(norm_weight.shape)}")
    n_out = weight.n // 2 if epilogue == _lib.EPI_SILU_MUL else weight.n
    if out is not None:
        _check_out(out, m, n_out, torch.bfloat16)
    r2 = None
    if residual is not None:
        r2, rm, ldr = _rows(residual, weight.n, "residual")
        if rm != m:
            raise ValueError(f"residual has {rm} rows, x has {m}")
    _require_device(x, "x")
    _require_device(weight.data, "weight")
    _require_device(norm_weight, "norm_weight")
    if nw.stride(0) != 1 or nw.data_ptr() % 16:
        nw = nw.contiguous() if nw.stride(0) != 1 else nw.clone()
    if out is None:
        out = x.new_empty((*x.shape[:-1], n_out))
    _require_device(out, "out")
    res_ptr, ldr = (None, 0) if r2 is None else (r2.data_ptr(), ldr)
    if r2 is not None:
        _require_device(r2, "residual")
    if m == 0:
        return out
    dev = _one_device(x, (weight.data, "weight"), (nw, "norm_weight"), (out, "out"), (r2, "residual"))
    with _on(dev):
        status = lib.lsk_rmsnorm_linear_bf16(
            weight.data.data_ptr(), weight.layout, weight.n, weight.k,
            x2.data_ptr(), m, ldx,
            nw.data_ptr(), float(eps),
            out.data_ptr(), n_out,
            epilogue, res_ptr, ldr, stream_handle(),
        )
    _lib.check(status, "lsk_rmsnorm_linear_bf16")
    return out


RMSNORM_MAX_K = 4096


def rmsnorm_rows(x: torch.Tensor, norm_weight: torch.Tensor, eps: float) -> torch.Tensor:
    """rms_norm(x) over the last dim, one bf16 rounding, for contiguous
    bfloat16 x[..., K] with K a multiple of 512 up to RMSNORM_MAX_K."""
    k = x.shape[-1]
    if x.dtype != torch.bfloat16 or norm_weight.dtype != torch.bfloat16 or norm_weight.shape != (k,):
        raise ValueError(f"x and norm_weight must be bfloat16 [..., K] and [K], got {x.dtype} {tuple(x.shape)} and "
                         f"{norm_weight.dtype} {tuple(norm_weight.shape)}")
    if not (x.is_contiguous() and norm_weight.is_contiguous()):
        raise ValueError("x and norm_weight must be contiguous")
    _require_device(x, "x")
    _require_device(norm_weight, "norm_weight")
    _one_device(x, (norm_weight, "norm_weight"))
    return _rmsnorm_rows(x, norm_weight, eps)


def _rmsnorm_rows(x: torch.Tensor, norm_weight: torch.Tensor, eps: float) -> torch.Tensor:
    """rmsnorm_rows of tensors already known to fit it."""
    k = x.shape[-1]
    out = x.new_empty(x.shape)
    m = x.numel() // k if k else 0
    if m == 0:
        return out
    with _on(x.device):
        status = _lib.load().lsk_rmsnorm_bf16(x.data_ptr(), m, k, k, norm_weight.data_ptr(), float(eps),
                                              out.data_ptr(), stream_handle())
    _lib.check(status, "lsk_rmsnorm_bf16")
    return out


def qk_norm_rope(qkv: torch.Tensor, q_norm_weight: torch.Tensor, k_norm_weight: torch.Tensor, eps: float,
                 cos: torch.Tensor, sin: torch.Tensor, *, num_attention_heads: int,
                 num_key_value_heads: int) -> tuple[torch.Tensor, torch.Tensor]:
    """q [B, n_q, T, d] and k [B, n_kv, T, d] of raw QKV rows [B, T, (n_q + 2 n_kv) d]
    (contiguous bfloat16, d = 128): per-head RMSNorm and rotate-half RoPE in
    one kernel.  cos / sin: [B or 1, T or 1, d/2] bfloat16 with equal strides,
    rows contiguous."""
    b, t, n = qkv.shape
    n_q, n_kv = num_attention_heads, num_key_value_heads
    d = n // (n_q + 2 * n_kv)
    if not qkv.is_contiguous() or n != (n_q + 2 * n_kv) * d:
        raise ValueError(f"qkv must be contiguous [B, T, ({n_q} + 2 * {n_kv}) * d] rows, got {tuple(qkv.shape)}")
    for x, what in ((qkv, "qkv"), (q_norm_weight, "q_norm_weight"), (k_norm_weight, "k_norm_weight"), (cos, "cos"),
                    (sin, "sin")):
        _require_device(x, what)
        if x.dtype != torch.bfloat16:
            raise ValueError(f"{what} must be bfloat16, got {x.dtype}")
    if q_norm_weight.shape != (d,) or k_norm_weight.shape != (d,) or not (q_norm_weight.is_contiguous()
                                                                           and k_norm_weight.is_contiguous()):
        raise ValueError(f"the q / k norm weights must be contiguous [{d}]")
    if (cos.dim() != 3 or cos.shape != sin.shape or cos.stride() != sin.stride() or cos.shape[0] not in (1, b)
            or cos.shape[1] not in (1, t) or cos.shape[2] != d // 2 or cos.stride(2) != 1):
        raise ValueError(f"cos / sin must be [{b} or 1, {t} or 1, {d // 2}] with equal strides and contiguous rows, got "
                         f"{tuple(cos.shape)} / {tuple(sin.shape)}")
    _one_device(qkv, (q_norm_weight, "q_norm_weight"), (k_norm_weight, "k_norm_weight"), (cos, "cos"), (sin, "sin"))
    return _qk_norm_rope(qkv, q_norm_weight, k_norm_weight, eps, cos, sin, n_q, n_kv)


def _qk_norm_rope(qkv: torch.Tensor, q_norm_weight: torch.Tensor, k_norm_weight: torch.Tensor, eps: float,
                  cos: torch.Tensor, sin: torch.Tensor, n_q: int, n_kv: int) -> tuple[torch.Tensor, torch.Tensor]:
    """qk_norm_rope of tensors already known to fit it."""
    b, t, n = qkv.shape
    d = n // (n_q + 2 * n_kv)
    q = qkv.new_empty((b, n_q, t, d))
    k = qkv.new_empty((b, n_kv, t, d))
    if b * t == 0:
        return q, k
    with _on(qkv.device):
        status = _lib.load().lsk_qk_norm_rope_bf16(
            qkv.data_ptr(), b, t, n, n_q, n_kv, d, q_norm_weight.data_ptr(), k_norm_weight.data_ptr(), float(eps),
            cos.data_ptr(), sin.data_ptr(), cos.stride(0) if cos.shape[0] > 1 else 0,
            cos.stride(1) if cos.shape[1] > 1 else 0, q.data_ptr(), k.data_ptr(), stream_handle())
    _lib.check(status, "lsk_qk_norm_rope_bf16")
    return q, k


_attention_workspaces: dict[tuple[int, int], torch.Tensor] = {}


@functools.lru_cache(maxsize=1024)
def _attention_workspace_bytes(n_q: int, n_kv: int, head_dim: int, max_seq_len: int) -> int:
    return _lib.load().lsk_attention_workspace_bytes(n_q, n_kv, head_dim, max_seq_len)


def attention_workspace(device: torch.device, n_q: int, n_kv: int, head_dim: int,
                        max_seq_len: int) -> torch.Tensor:
    """The decode attention workspace of `device` for the current stream
    (zero-filled once, left zero-filled by every call), large enough for this
    geometry.  Calls on other streams get their own."""
    nbytes = _attention_workspace_bytes(n_q, n_kv, head_dim, max_seq_len)
    if nbytes == 0:
        raise ValueError(f"no attention workspace for n_q={n_q}, n_kv={n_kv}, head_dim={head_dim}, "
                         f"max_seq_len={max_seq_len}")
    return _device_workspace(_attention_workspaces, device, nbytes, "attention")


def decode_attention(qkv: torch.Tensor, q_norm_weight: torch.Tensor, k_norm_weight: torch.Tensor, eps: float,
                     cos: torch.Tensor, sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     pos: int | torch.Tensor, scale: float, *, num_attention_heads: int, num_key_value_heads: int,
                     out: torch.Tensor | None = None, workspace: torch.Tensor | str = "auto") -> torch.Tensor:
    """One decode token of one layer between QKV and o_proj: per-head q/k
    RMSNorm and RoPE of the raw QKV row, k and v written to row `pos` of the
    layer's caches ([n_kv, max_seq_len, d] bf16, batch 1), and GQA attention
    over rows 0..pos.  Returns out [n_q * d] bf16.  The caller advances its
    cache cursor.  workspace: "auto" (attention_workspace), or a zero-filled
    uint8 device tensor of lsk_attention_workspace_bytes() bytes.

    pos: an int (cos / sin are this position's rows, d/2 values each), or a
    one-element int32 device tensor read by the kernel (cos / sin are then the
    whole [max_seq_len, d/2] tables): one launch for any position, so a
    captured HIP graph can be replayed token after token with the caller
    writing the next position into that tensor.  Out-of-range device
    positions change nothing."""
    lib = _lib.load()
    n_q, n_kv = num_attention_heads, num_key_value_heads
    on_device = isinstance(pos, torch.Tensor)
    for t, what in ((qkv, "qkv"), (q_norm_weight, "q_norm_weight"), (k_norm_weight, "k_norm_weight"), (cos, "cos"),
                    (sin, "sin"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        _require_device(t, what)
        if t.dtype != torch.bfloat16:
            raise ValueError(f"{what} must be bfloat16, got {t.dtype}")
    if k_cache.dim() != 3 or k_cache.shape != v_cache.shape or k_cache.shape[0] != n_kv:
        raise ValueError(f"k_cache / v_cache must be [n_kv={n_kv}, max_seq_len, head_dim], got "
                         f"{tuple(k_cache.shape)} / {tuple(v_cache.shape)}")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache / v_cache must be contiguous")
    d, s_max = k_cache.shape[2], k_cache.shape[1]
    if qkv.numel() != (n_q + 2 * n_kv) * d:
        raise ValueError(f"qkv has {qkv.numel()} values, expected {(n_q + 2 * n_kv) * d}")
    rope_len = s_max * (d // 2) if on_device else d // 2
    if q_norm_weight.numel() != d or k_norm_weight.numel() != d or cos.numel() != rope_len or sin.numel() != rope_len:
        where = f"the whole [{s_max}, {d // 2}] tables" if on_device else "this position's row"
        raise ValueError(f"norm weights must hold {d} values and cos / sin {rope_len} ({where})")
    if on_device:
        _require_device(pos, "pos")
        if pos.dtype != torch.int32 or pos.numel() != 1:
            raise ValueError("a device pos must be a one-element int32 tensor")
    flat = [t if t.is_contiguous() else t.reshape(-1).contiguous() for t in (qkv, q_norm_weight, k_norm_weight, cos, sin)]
    if out is None:
        out = qkv.new_empty((n_q * d,))
    if out.dtype != torch.bfloat16 or out.numel() != n_q * d or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous bfloat16 tensor of {n_q * d} values")
    if isinstance(workspace, str):
        if workspace != "auto":
            raise ValueError(f"workspace must be 'auto' or a tensor, not {workspace!r}")
        workspace = attention_workspace(qkv.device, n_q, n_kv, d, s_max)
    _require_device(workspace, "workspace")
    dev = _one_device(qkv, (q_norm_weight, "q_norm_weight"), (k_norm_weight, "k_norm_weight"), (cos, "cos"),
                      (sin, "sin"), (k_cache, "k_cache"), (v_cache, "v_cache"), (out, "out"),
                      (workspace, "workspace"), (pos if on_device else None, "pos"))
    common = (flat[0].data_ptr(), n_q, n_kv, d, flat[1].data_ptr(), flat[2].data_ptr(), float(eps),
              flat[3].data_ptr(), flat[4].data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), s_max)
    tail = (float(scale), out.data_ptr(), workspace.data_ptr(), workspace.numel() * workspace.element_size())
    with _on(dev):
        tail += (stream_handle(),)
        if on_device:
            status = lib.lsk_decode_attention_at_bf16(*common, pos.data_ptr(), *tail)
        else:
            status = lib.lsk_decode_attention_bf16(*common, int(pos), *tail)
    _lib.check(status, "lsk_decode_attention_at_bf16" if on_device else "lsk_decode_attention_bf16")
    return out


ATTENTION_MAX_ROWS = 16384
ATTENTION_COUNTER_BYTES = 256  # the part of an attention workspace that must start zeroed

# Workspaces of gqa_attention by (device, stream, bytes): one size per head
# geometry, so none is ever replaced under a call that is still running.
_gqa_workspaces: dict[tuple[int, int, int], torch.Tensor] = {}


def _gqa_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    if torch.cuda.is_current_stream_capturing():
        # the graph's own: replays never share one with eager calls
        workspace = torch.empty(nbytes, device=device, dtype=torch.uint8)
        workspace[:ATTENTION_COUNTER_BYTES].zero_()
        return workspace
    key = (_device_index(device), stream_handle(), nbytes)
    workspace = _gqa_workspaces.get(key)
    if workspace is None:
        workspace = _gqa_workspaces[key] = torch.zeros(nbytes, device=device, dtype=torch.uint8)
    return workspace


def gqa_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float) -> torch.Tensor:
    """softmax(q k^T * scale) v of one query row per head over rows already
    cached: q [n_q, d] contiguous, k / v [n_kv, rows, d] with equal strides and
    contiguous rows (a cache's written part), bfloat16, d = 128.  Returns
    [n_q * d] bf16."""
    n_q, d = q.shape
    n_kv, rows, _ = k.shape
    for t, what in ((q, "q"), (k, "k"), (v, "v")):
        _require_device(t, what)
        if t.dtype != torch.bfloat16:
            raise ValueError(f"{what} must be bfloat16, got {t.dtype}")
    if k.shape != v.shape or k.stride() != v.stride() or k.shape[2] != d or k.stride(2) != 1 or k.stride(1) != d \
            or not q.is_contiguous():
        raise ValueError(f"q must be contiguous [n_q, {d}] and k / v [n_kv, rows, {d}] with equal strides and "
                         f"contiguous rows, got {tuple(q.shape)}, {tuple(k.shape)} / {tuple(v.shape)}")
    _one_device(q, (k, "k"), (v, "v"))
    return _gqa_attention(q, k, v, scale)


def _gqa_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float) -> torch.Tensor:
    """gqa_attention of tensors already known to fit it."""
    n_q, d = q.shape
    n_kv, rows, _ = k.shape
    lib = _lib.load()
    out = q.new_empty((n_q * d,))
    with _on(q.device):
        workspace = None
        if rows > 128:  # sized for the longest cache: one workspace as a sequence grows
            workspace = _gqa_workspace(q.device, _attention_workspace_bytes(n_q, n_kv, d, ATTENTION_MAX_ROWS))
        status = lib.lsk_gqa_attention_bf16(
            q.data_ptr(), n_q, n_kv, d, k.data_ptr(), v.data_ptr(), max(k.stride(0), rows * d), rows, float(scale),
            out.data_ptr(), None if workspace is None else workspace.data_ptr(),
            0 if workspace is None else workspace.numel(), stream_handle())
    _lib.check(status, "lsk_gqa_attention_bf16")
    return out


def _key_rows(k: torch.Tensor, v: torch.Tensor, what: str) -> tuple[int, ...]:
    """Strides of key and value rows [..., heads, rows, d] that the attention
    kernel reads in place (never copied: they are a cache's): a leading one per
    axis but the last.  Axes of one entry, and empty tensors, take any."""
    d = k.shape[-1]
    strides = k.stride()
    if (k.dtype is torch.bfloat16 is v.dtype and k.shape == v.shape and strides == v.stride() and strides[-1] == 1
            and d <= strides[-2] <= _lib.MAX_ACTIVATION_STRIDE and not (strides[0] | strides[1] | strides[-2]) & 7):
        return strides  # (the library checks the addresses)
    if k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16 or k.shape != v.shape:
        raise ValueError(f"{what} must be bfloat16 tensors of one shape, got {k.dtype} {tuple(k.shape)} / {v.dtype} "
                         f"{tuple(v.shape)}")
    if k.numel() == 0:
        return (0,) * (k.dim() - 2) + (d,)
    strides = [s if n > 1 else 0 for n, s in zip(k.shape[:-1], k.stride())]
    if strides != [s if n > 1 else 0 for n, s in zip(v.shape[:-1], v.stride())] or k.stride(-1) != 1 or v.stride(-1) != 1 \
            or any(s % 8 for s in strides) or k.data_ptr() % 16 or v.data_ptr() % 16 or 0 < strides[-1] < d \
            or strides[-1] > _lib.MAX_ACTIVATION_STRIDE:
        raise ValueError(f"{what} must have equal strides, multiples of 8 (of rows up to {_lib.MAX_ACTIVATION_STRIDE}), rows "
                         f"of unit stride and 16-byte alignment, got strides {k.stride()} / {v.stride()}")
    if k.shape[-2] > 1 and strides[-1] == 0:
        raise ValueError(f"{what}: the rows must not repeat (stride 0)")
    strides[-1] = strides[-1] or d
    return tuple(strides)


@functools.lru_cache(maxsize=4096)
def _prefix_workspace_bytes(b: int, t: int, n_q: int, n_kv: int, prefix: int, rows: int) -> int:
    return _lib.load().lsk_prefix_attention_workspace_bytes(b, t, n_q, n_kv, prefix, rows)


def shared_prefix_attention(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k: torch.Tensor,
                            v: torch.Tensor, lens: torch.Tensor, scale: float, *,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T * scale) v of T query tokens of each of B requests over a
    prefix that they share and the rows that each has cached since -> [B, T, n_q * d].

    q: [B, n_q, T, d].  prefix_k / prefix_v: [n_kv, P, d], read once for all requests
    (the written part of an ArenaKVCache layer, for one).  k / v: [B, n_kv, S, d],
    and lens, int32 [B] on the device: how many of a request's S rows are written,
    its T new tokens' rows the last of them (lengths outside 0..S are taken at the
    ends).  Query t sees the prefix and the first lens - (T - 1 - t) own rows.  Rows
    behind the written ones are not read; a query that sees no row gives zeros.
    bfloat16, d = 128, q heads in groups of n_q / n_kv.  Caches are read in place at
    any strides that are multiples of 8 (rows up to 2^22 - 8 elements apart, a head's
    rows below 2^31 bytes); lens is read on the device, so a captured call follows
    it.  out: a contiguous [B, T, n_q * d] tensor."""
    if q.dim() != 4 or prefix_k.dim() != 3 or k.dim() != 4:
        raise ValueError(f"q, prefix_k / prefix_v and k / v must be [B, n_q, T, d], [n_kv, P, d] and [B, n_kv, S, d], got "
                         f"{tuple(q.shape)}, {tuple(prefix_k.shape)} and {tuple(k.shape)}")
    b, n_q, t, d = q.shape
    n_kv, prefix, rows = prefix_k.shape[0], prefix_k.shape[1], k.shape[2]
    if q.dtype is not torch.bfloat16:
        raise ValueError(f"q must be bfloat16, got {q.dtype}")
    if d != 128 or n_kv < 1 or n_q < 1 or n_q % n_kv or prefix_k.shape[2] != d or k.shape != (b, n_kv, rows, d):
        raise ValueError(f"q {tuple(q.shape)}, prefix {tuple(prefix_k.shape)} and own rows {tuple(k.shape)} do not fit "
                         f"together (d = 128, n_q a multiple of n_kv)")
    prefix_strides = _key_rows(prefix_k, prefix_v, "prefix_k / prefix_v")
    strides = _key_rows(k, v, "k / v")
    index = q.get_device()
    lens_at = _per_row(lens, b, torch.int32, index, "lens")
    if not (prefix_k.get_device() == prefix_v.get_device() == k.get_device() == v.get_device() == index):
        _one_device(q, (prefix_k, "prefix_k"), (prefix_v, "prefix_v"), (k, "k"), (v, "v"))
    if out is not None:
        _one_device(q, (out, "out"))
        if tuple(out.shape) != (b, t, n_q * d) or out.dtype is not torch.bfloat16 or not out.is_contiguous() \
                or out.data_ptr() % 16:
            raise ValueError(f"out must be a contiguous, 16-byte aligned bfloat16 [{b}, {t}, {n_q * d}] tensor, got "
                             f"{out.dtype} {tuple(out.shape)}")
        if any(_overlap(out, x) for x in (q, prefix_k, prefix_v, k, v) if x.numel()):
            raise ValueError("out must not overlap the inputs")
    _require_device(q, "q")
    if out is None:
        out = q.new_empty((b, t, n_q * d))
    if b * t == 0:
        return out
    q_strides = q.stride()
    if q_strides[3] != 1 or (q_strides[0] | q_strides[1] | q_strides[2]) & 7 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        q_strides = q.stride()
    nbytes = _prefix_workspace_bytes(b, t, n_q, n_kv, prefix, rows)
    workspace = q.new_empty((nbytes // 2,)) if nbytes else None
    with _on_index(index):
        status = _lib.load().lsk_prefix_attention_bf16(
            q.data_ptr(), q_strides[0], q_strides[1], q_strides[2], b, t, n_q, n_kv, d, prefix_k.data_ptr(),
            prefix_v.data_ptr(), prefix_strides[0], prefix_strides[1], prefix, k.data_ptr(), v.data_ptr(), strides[0],
            strides[1], strides[2], rows, lens_at, float(scale), out.data_ptr(), _ptr(workspace), nbytes,
            torch._C._cuda_getCurrentRawStream(index))
    _lib.check(status, "lsk_prefix_attention_bf16")
    return out


def _pool(cache: PagedKVCache, layer: int, table: torch.Tensor) -> tuple[_lib.PagedPool, int, int]:
    """(struct, B, device index) of a layer's pages and the batch's page table."""
    if not isinstance(cache, PagedKVCache):
        raise ValueError("cache must be a PagedKVCache")
    if not 0 <= layer < cache.num_layers:
        raise ValueError(f"layer {layer} of a cache of {cache.num_layers}")
    if table.dtype is not torch.int32 or table.dim() != 2 or table.shape[1] < 1 or table.stride(1) != 1 and table.shape[1] > 1:
        raise ValueError(f"table must be int32 [B, pages] with contiguous rows, got {table.dtype} {tuple(table.shape)} of "
                         f"strides {table.stride()}")
    b, width = table.shape
    stride = table.stride(0) if b > 1 else width
    if stride < width:
        raise ValueError(f"table must not repeat or interleave its rows (stride {stride} of {width} entries)")
    index = cache.storage.get_device()
    if table.get_device() != index:
        raise ValueError(f"table is on {table.device}, the cache on {cache.storage.device}")
    keys = cache.storage.data_ptr()
    exponents = cache.exponents.data_ptr()
    plane = cache.num_pages * cache.num_key_value_heads * (cache.page_rows // 16)  # blocks of a layer's keys
    at = 2 * layer * plane
    return _lib.PagedPool(keys + at * 2048, keys + (at + plane) * 2048, exponents + at, exponents + at + plane,
                          cache.num_pages, cache.num_key_value_heads, cache.page_rows, width, table.data_ptr(),
                          stride), b, index


def _head_rows(x: torch.Tensor) -> tuple[torch.Tensor, tuple[int, ...]]:
    """x [B, heads, T, d] as the paged kernels read it in place, copied if they cannot, and its strides."""
    strides = x.stride()
    if strides[3] != 1 or (strides[0] | strides[1] | strides[2]) & 7 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        strides = x.stride()
    return x, strides


def paged_append(cache: PagedKVCache, layer: int, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
                 lens: torch.Tensor, *, counts: torch.Tensor | None = None) -> None:
    """New key and value rows of a batch into their pages, rounded to 8 bits.

    k / v: [B, n_kv, T, d] bfloat16, d = 128 (views of the QKV projection's rows are read in
    place); table: int32 [B, pages]; lens: int32 [B], a request's rows with the new ones;
    counts: int32 [B], how many of the T are real (the first; all without).  Row t goes to
    the request's row lens - counts + t; rows in front of row 0, past the table or in an entry
    that names no page are dropped.  The three are read on the device, so a captured call
    follows them.  No two requests may append to one page (PagedKVCache.reserve sees to it)."""
    pool, b, index = _pool(cache, layer, table)
    n_kv = cache.num_key_value_heads
    if k.dim() != 4 or k.shape != v.shape or k.shape[0] != b or k.shape[1] != n_kv or k.shape[3] != 128 \
            or k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16:
        raise ValueError(f"k and v must be bfloat16 [{b}, {n_kv}, T, 128], got {k.dtype} {tuple(k.shape)} and {v.dtype} "
                         f"{tuple(v.shape)}")
    lens_at = _per_row(lens, b, torch.int32, index, "lens")
    counts_at = _per_row(counts, b, torch.int32, index, "counts")
    if not (k.get_device() == v.get_device() == index):
        _one_device(cache.storage, (k, "k"), (v, "v"))
    _require_device(cache.storage, "cache")
    t = k.shape[2]
    if b * t == 0:
        return
    k, ks = _head_rows(k)
    v, vs = _head_rows(v)
    with _on_index(index):
        status = _lib.load().lsk_paged_append_bf16(
            ctypes.byref(pool), k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2], b, t, lens_at,
            counts_at, torch._C._cuda_getCurrentRawStream(index))
    _lib.check(status, "lsk_paged_append_bf16")


def paged_read(cache: PagedKVCache, layer: int, table: torch.Tensor, starts: torch.Tensor, rows: int, *,
               lens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [B, n_kv, rows, 128] bfloat16: what the cache stands for in rows starts[b] ..
    starts[b] + rows - 1 (int32 [B] on the device).  Rows from lens[b] on and rows without
    a page are zeros."""
    pool, b, index = _pool(cache, layer, table)
    starts_at = _per_row(starts, b, torch.int32, index, "starts")
    lens_at = _per_row(lens, b, torch.int32, index, "lens")
    if rows < 0:
        raise ValueError(f"rows={rows} must not be negative")
    _require_device(cache.storage, "cache")
    k = cache.storage.new_empty((b, cache.num_key_value_heads, rows, 128), dtype=torch.bfloat16)
    v = torch.empty_like(k)
    if b * rows == 0:
        return k, v
    with _on_index(index):
        status = _lib.load().lsk_paged_read_bf16(ctypes.byref(pool), starts_at, lens_at, b, rows, k.data_ptr(), v.data_ptr(),
                                                 torch._C._cuda_getCurrentRawStream(index))
    _lib.check(status, "lsk_paged_read_bf16")
    return k, v


def copy_pages(cache: PagedKVCache, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Page src[i] to page dst[i] in every layer, keys, values and exponents (int32 [n] on
    the pool's device).  Entries outside 0..num_pages - 1 copy nothing.  A destination must
    not be named again, neither as a destination nor as a source."""
    if not isinstance(cache, PagedKVCache):
        raise ValueError("cache must be a PagedKVCache")
    n = src.numel()
    index = cache.storage.get_device()
    src_at = _per_row(src, n, torch.int32, index, "src")
    dst_at = _per_row(dst, n, torch.int32, index, "dst")
    _require_device(cache.storage, "cache")
    if n == 0:
        return
    with _on_index(index):
        status = _lib.load().lsk_paged_copy(
            cache.storage.data_ptr(), cache.exponents.data_ptr(), 2 * cache.num_layers, cache.num_pages,
            cache.num_key_value_heads * (cache.page_rows // 16), src_at, dst_at, n,
            torch._C._cuda_getCurrentRawStream(index))
    _lib.check(status, "lsk_paged_copy")


@functools.lru_cache(maxsize=4096)
def _paged_workspace_bytes(b: int, t: int, n_q: int, n_kv: int, capacity: int) -> int:
    return _lib.load().lsk_paged_attention_workspace_bytes(b, t, n_q, n_kv, capacity)


def paged_attention(q: torch.Tensor, cache: PagedKVCache, layer: int, table: torch.Tensor, lens: torch.Tensor,
                    scale: float, *, counts: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T * scale) v of T query tokens of each of B requests over their pages ->
    [B, T, n_q * d].

    q: [B, n_q, T, d] bfloat16, d = 128, q heads in groups of n_q / n_kv; table, lens and
    counts as for paged_append, which the new tokens' rows went through before: query t sees
    the first lens - (counts - 1 - t) rows.  Query tokens from counts on, and those that see
    no row, give zeros.  T = 1 is a decode step, a few tokens a verify block, thousands a
    prompt (in chunks if wanted).  out: a contiguous [B, T, n_q * d] tensor."""
    pool, b, index = _pool(cache, layer, table)
    n_kv = cache.num_key_value_heads
    if q.dim() != 4 or q.dtype is not torch.bfloat16 or q.shape[0] != b or q.shape[3] != 128 or q.shape[1] < 1 \
            or q.shape[1] % n_kv:
        raise ValueError(f"q must be bfloat16 [{b}, a multiple of {n_kv}, T, 128], got {q.dtype} {tuple(q.shape)}")
    n_q, t = q.shape[1], q.shape[2]
    lens_at = _per_row(lens, b, torch.int32, index, "lens")
    counts_at = _per_row(counts, b, torch.int32, index, "counts")
    if q.get_device() != index:
        _one_device(cache.storage, (q, "q"))
    if out is not None:
        _one_device(cache.storage, (out, "out"))
        if tuple(out.shape) != (b, t, n_q * 128) or out.dtype is not torch.bfloat16 or not out.is_contiguous() \
                or out.data_ptr() % 16:
            raise ValueError(f"out must be a contiguous, 16-byte aligned bfloat16 [{b}, {t}, {n_q * 128}] tensor, got "
                             f"{out.dtype} {tuple(out.shape)}")
        if q.numel() and _overlap(out, q):
            raise ValueError("out must not overlap q")
    _require_device(cache.storage, "cache")
    if out is None:
        out = q.new_empty((b, t, n_q * 128))
    if b * t == 0:
        return out
    q, qs = _head_rows(q)
    nbytes = _paged_workspace_bytes(b, t, n_q, n_kv, table.shape[1] * cache.page_rows)
    workspace = q.new_empty((nbytes // 2,)) if nbytes else None
    with _on_index(index):
        status = _lib.load().lsk_paged_attention_bf16(
            ctypes.byref(pool), q.data_ptr(), qs[0], qs[1], qs[2], b, t, n_q, 128, lens_at, counts_at, float(scale),
            out.data_ptr(), _ptr(workspace), nbytes, torch._C._cuda_getCurrentRawStream(index))
    _lib.check(status, "lsk_paged_attention_bf16")
    return out


class LmHeadWorkspace:
    """Device workspace of the greedy head, sized once per (M, V, K): a status
    word and the per-workgroup argmax partials.  Zero-filled here; every call
    leaves the partials zero again, so it is never cleared between calls.
    Calls that share one must be stream-ordered."""

    def __init__(self, m: int, v: int, k: int, device: torch.device | str) -> None:
        nbytes = _lib.load().lsk_workspace_bytes(_lib.OP_LM_HEAD_ARGMAX, m, v, k)
        if nbytes == 0:
            raise ValueError(f"no lm_head workspace for M={m}, V={v}, K={k}")
        self.m, self.v, self.k = m, v, k
        self.buffer = torch.zeros(nbytes, device=device, dtype=torch.uint8)

    def give_ups(self) -> int:
        """Argmax stages (rows) that gave up waiting for a partial since the
        workspace was made (their out_idx was -1); 0 while every grid runs to
        its end.  Synchronizes with the device."""
        return int(self.buffer[:4].view(torch.int32).item())


def lm_head_argmax(hidden: torch.Tensor, weight: PackedWeight, *, logits_mode: int = _lib.LOGITS_FP32,
                   logits_out: torch.Tensor | None = None, workspace: LmHeadWorkspace | None = None,
                   out: torch.Tensor | None = None, norm_weight: torch.Tensor | None = None,
                   eps: float = 1e-6) -> torch.Tensor:
    """Greedy token per row: int64 [M] = argmax over the vocab of hidden . W^T.

    logits_mode LOGITS_FP32 compares fp32 scores (cuTile head); LOGITS_BF16
    compares bf16-rounded logits (torch.mv head).  Lowest index wins ties.
    norm_weight: the final RMSNorm ([K] bf16, with eps) applied to hidden in
    the kernel (K = 2560, M <= 8)."""
    if not isinstance(weight, PackedWeight) or weight.layout != _lib.LAYOUT_MFMA16X32:
        raise ValueError("lm_head weight must be a PackedWeight in the mfma16x32 layout")
    lib = _lib.load()
    h2, m, ldx = _rows(hidden, weight.k, "hidden")
    v = weight.n
    if out is not None and (out.dtype != torch.long or out.numel() < m or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous int64 tensor of at least {m} values "
                         f"(got {out.dtype} {tuple(out.shape)})")
    if logits_out is not None:
        if logits_out.dtype != torch.float32 or logits_out.numel() != m * v or not logits_out.is_contiguous():
            raise ValueError(f"logits_out must be a contiguous float32 tensor of {m}x{v}")
    if norm_weight is not None and (norm_weight.dtype != torch.bfloat16 or norm_weight.numel() != weight.k):
        raise ValueError(f"norm_weight must be a bfloat16 tensor of {weight.k} values")
    _require_device(hidden, "hidden")
    _require_device(weight.data, "weight")
    if m == 0:  # no rows: an empty index tensor, as torch.argmax over [0, V] scores gives
        return out if out is not None else torch.empty((0,), device=hidden.device, dtype=torch.long)
    if workspace is None or workspace.m < m or workspace.v != v or workspace.k != weight.k:
        workspace = LmHeadWorkspace(m, v, weight.k, hidden.device)
    if out is None:
        out = torch.empty((m,), device=hidden.device, dtype=torch.long)
    _require_device(out, "out")
    logits_ptr = None
    if logits_out is not None:
        _require_device(logits_out, "logits_out")
        logits_ptr = logits_out.data_ptr()
    dev = _one_device(hidden, (weight.data, "weight"), (out, "out"), (logits_out, "logits_out"),
                      (norm_weight, "norm_weight"), (workspace.buffer, "workspace"))
    if norm_weight is not None:
        _require_device(norm_weight, "norm_weight")
        nw = norm_weight.reshape(-1).contiguous()
        with _on(dev):
            status = lib.lsk_rmsnorm_lm_head_argmax_bf16(
                weight.data.data_ptr(), weight.layout, v, weight.k, h2.data_ptr(), m, ldx, nw.data_ptr(), float(eps),
                logits_ptr, logits_mode, out.data_ptr(), workspace.buffer.data_ptr(), workspace.buffer.numel(),
                stream_handle(),
            )
        _lib.check(status, "lsk_rmsnorm_lm_head_argmax_bf16")
        return out
    with _on(dev):
        status = lib.lsk_lm_head_argmax_bf16(
            weight.data.data_ptr(), weight.layout, v, weight.k,
            h2.data_ptr(), m, ldx,
            logits_ptr, logits_mode,
            out.data_ptr(),
            workspace.buffer.data_ptr(), workspace.buffer.numel(), stream_handle(),
        )
    _lib.check(status, "lsk_lm_head_argmax_bf16")
    return out


def lm_head_argmax_noalloc(hidden: torch.Tensor, weight: PackedWeight, out: torch.Tensor, *,
                           logits_mode: int = _lib.LOGITS_FP32, logits_out: torch.Tensor | None = None) -> torch.Tensor:
    """lm_head_argmax with no allocation anywhere on the call: the argmax
    partials use the library's static device scratch
    (lsk_lm_head_argmax_noalloc_bf16), `out` (int64, at least M values) is
    the caller's, and `hidden` must already be contiguous [M, K] bf16 rows.
    Usable under HIP graph capture; calls on one device that are not
    stream-ordered with each other race on the scratch."""
    if not isinstance(weight, PackedWeight) or weight.layout != _lib.LAYOUT_MFMA16X32:
        raise ValueError("lm_head weight must be a PackedWeight in the mfma16x32 layout")
    if hidden.dtype != torch.bfloat16 or hidden.shape[-1] != weight.k or not hidden.is_contiguous():
        raise ValueError(f"hidden must be contiguous bfloat16 [M, {weight.k}] rows")
    m = hidden.numel() // weight.k
    if out.dtype != torch.long or out.numel() < m or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous int64 tensor of at least {m} values")
    if logits_out is not None and (logits_out.dtype != torch.float32 or logits_out.numel() != m * weight.n
                                   or not logits_out.is_contiguous()):
        raise ValueError(f"logits_out must be a contiguous float32 tensor of {m}x{weight.n}")
    for t, what in ((hidden, "hidden"), (weight.data, "weight"), (out, "out")):
        _require_device(t, what)
    if m == 0:
        return out
    dev = _one_device(hidden, (weight.data, "weight"), (out, "out"), (logits_out, "logits_out"))
    with _on(dev):
        status = _lib.load().lsk_lm_head_argmax_noalloc_bf16(
            weight.data.data_ptr(), weight.layout, weight.n, weight.k, hidden.data_ptr(), m, weight.k,
            logits_out.data_ptr() if logits_out is not None else None, logits_mode, out.data_ptr(), stream_handle())
    _lib.check(status, "lsk_lm_head_argmax_noalloc_bf16")
    return out


@functools.lru_cache(maxsize=4096)
def _lora_workspace_bytes(m: int, n: int, k: int, rank_tiles: int, count: int, epilogue: int) -> int:
    return _lib.load().lsk_lora_workspace_bytes(m, n, k, rank_tiles, count, epilogue)


def _check_index(index: torch.Tensor, m: int) -> None:
    if index.dtype is not torch.int32 or index.numel() != m or not index.is_contiguous():
        raise ValueError(f"index must be a contiguous int32 tensor of {m} values, got {index.dtype} {tuple(index.shape)}")


def lora_add(y: torch.Tensor, x: torch.Tensor, store: AdapterStore, index: torch.Tensor, *,
             epilogue: int = _lib.EPI_NONE, out: torch.Tensor | None = None) -> torch.Tensor:
    """The rows' own low-rank adapters added to what a shared projection gave:
    z = y + scale (x . A^T) . B^T of adapter index[m] of `store` (a row whose
    index is outside [0, store.count) keeps y), in fp32, rounded once.

    y: [..., N] bfloat16, x: [..., K] bfloat16, the projection's input; index: int32,
    one per row, read on the device.  epilogue EPI_NONE returns z; EPI_SILU_MUL
    (a gate_up store) returns SiLU(gate) * up of z, y being in the column order of
    the gate_up weight's packed rows (lora_linear makes it).  out: contiguous
    [..., N] (or N/2), and with EPI_NONE it may be y itself."""
    if not isinstance(store, AdapterStore):
        raise ValueError("store must be an AdapterStore")
    silu = epilogue == _lib.EPI_SILU_MUL
    if silu != store.gate_up or epilogue not in (_lib.EPI_NONE, _lib.EPI_SILU_MUL):
        raise ValueError(f"epilogue {epilogue}: a gate_up store takes EPI_SILU_MUL, any other EPI_NONE")
    n, k = store.n, store.k
    y2, m, ldy = _rows(y, n, "y")
    x2, xm, ldx = _rows(x, k, "x")
    if xm != m:
        raise ValueError(f"x has {xm} rows, y has {m}")
    _check_index(index, m)
    n_out = n // 2 if silu else n
    if out is not None:
        _check_out(out, m, n_out, torch.bfloat16)
        if out.data_ptr() % 16:
            raise ValueError("out must be 16-byte aligned")
        if _overlap(out, x2) or (_overlap(out, y2) and (silu or out.data_ptr() != y2.data_ptr() or not y2.is_contiguous())):
            raise ValueError("out must be y itself (contiguous, EPI_NONE) or overlap neither y nor x")
    _require_device(y, "y")
    at = y.get_device()
    if not (x.get_device() == store.a_tiles.get_device() == index.get_device() == at) or \
            (out is not None and out.get_device() != at):
        _one_device(y, (x, "x"), (store.a_tiles, "store"), (index, "index"), (out, "out"))
    if out is None:
        out = y.new_empty((*y.shape[:-1], n_out))
    if m == 0:
        return out
    nbytes = _lora_workspace_bytes(m, n, k, store.rank_tiles, store.count, epilogue)
    workspace = y.new_empty((nbytes // 2,)) if nbytes else None
    with _on_index(at):
        status = _lib.load().lsk_lora_add_bf16(
            y2.data_ptr(), m, n, ldy, x2.data_ptr(), k, ldx, store.a_tiles.data_ptr(), store.b_tiles.data_ptr(),
            store.scales.data_ptr(), store.ranks.data_ptr(), store.count, store.rank_tiles, index.data_ptr(), epilogue,
            out.data_ptr(), _ptr(workspace), nbytes, torch._C._cuda_getCurrentRawStream(at))
    _lib.check(status, "lsk_lora_add_bf16")
    return out


def lora_linear(x: torch.Tensor, weight: PackedWeight, store: AdapterStore, index: torch.Tensor, *,
                epilogue: int = _lib.EPI_NONE, residual: torch.Tensor | None = None,
                out: torch.Tensor | None = None, workspace: torch.Tensor | None | str = "auto") -> torch.Tensor:
    """linear() with the rows' own adapters: the shared projection (its residual
    included) rounded to bf16 as linear() gives it, the adapters added by
    lora_add; EPI_SILU_MUL takes SiLU(gate) * up after the adapters."""
    if not isinstance(weight, PackedWeight):
        raise ValueError("weight must be a PackedWeight (pack it with leanstack_amd.layout / leanserve)")
    if not isinstance(store, AdapterStore) or (store.n, store.k) != weight.shape:
        raise ValueError(f"the store's adapters must be of the weight's shape {weight.shape}")
    if store.gate_up != (weight.layout == _lib.LAYOUT_MFMA16X32_GATEUP) or store.gate_up != (epilogue == _lib.EPI_SILU_MUL):
        raise ValueError("a gate_up weight takes a gate_up store and EPI_SILU_MUL, and no other does")
    if out is not None and (out.data_ptr() % 16 or _overlap(out, x)):
        raise ValueError("out must be 16-byte aligned and not overlap x")
    # (lora_add's checks, in front of the projection: a refused call has written nothing)
    if x.shape[-1] == weight.k:
        _check_index(index, x.numel() // weight.k)
    if not (store.a_tiles.get_device() == index.get_device() == x.get_device()):
        _one_device(x, (store.a_tiles, "store"), (index, "index"))
    if epilogue == _lib.EPI_SILU_MUL:
        # the same tiles read as a plain weight give both halves, before SiLU, in packed order
        if residual is not None:
            raise ValueError("EPI_SILU_MUL takes no residual")
        both = PackedWeight(weight.data, weight.n, weight.k, _lib.LAYOUT_MFMA16X32)
        return lora_add(linear(x, both, workspace=workspace), x, store, index, epilogue=epilogue, out=out)
    y = linear(x, weight, epilogue=epilogue, residual=residual, out=out, workspace=workspace)
    return lora_add(y, x, store, index, out=y)


def _per_row(t: torch.Tensor | None, m: int, dtype: torch.dtype, device_index: int, what: str) -> int | None:
    """The address of an optional contiguous [m] argument on the call's device."""
    if t is None:
        return None
    if t.dtype is not dtype or t.dim() != 1 or t.numel() != m or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of {m} values, got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != device_index:
        raise ValueError(f"{what} is on {t.device}, the call's tensors are on device {device_index}")
    return t.data_ptr()


def _row_list(t: torch.Tensor, m: int, dtype: torch.dtype, device_index: int, what: str) -> tuple[int, int, int]:
    """Address, row stride and row length of an [m, n] argument with contiguous rows."""
    if t.dtype is not dtype or t.dim() != 2 or t.shape[0] != m:
        raise ValueError(f"{what} must be a {dtype} tensor of {m} contiguous rows, got {t.dtype} {tuple(t.shape)}")
    n = t.shape[1]
    ld, unit = t.stride()
    if n > 1 and unit != 1:
        raise ValueError(f"{what} must be a {dtype} tensor of {m} contiguous rows, got strides {(ld, unit)}")
    if m == 1:
        ld = n
    elif ld < n:
        raise ValueError(f"{what} must not repeat or interleave its rows (stride {ld} of {n} values)")
    if t.get_device() != device_index:
        raise ValueError(f"{what} is on {t.device}, the call's tensors are on device {device_index}")
    return t.data_ptr(), ld, n


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two tensors meet."""
    def last(t):
        return t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    return a.data_ptr() < last(b) and b.data_ptr() < last(a)


def constrain_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None,
                     history_lens: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
                     repetition: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                     presence: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                     bias_values: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Each request's constraints on its row of logits [M, V] (float32 or
    bfloat16), and its greedy token: (out [M, V] in the logits' type, int64 [M]).

    In this order, in fp32: tokens of the row's history are divided (if positive)
    or multiplied (if not) by `repetition`; those said c > 0 times behind the
    prompt lose `frequency` * c and `presence`; `bias_values` are added at
    `bias_ids`; values not `allowed` become -inf.  The token is the lowest index
    of the row's largest value (NaN counts as the largest), -1 where all are -inf.

    history: int32 [M, L], of which the first history_lens[m] tokens count (all
    without history_lens) and the first prompt_lens[m] are the prompt (none without
    prompt_lens); tokens outside [0, V) count for nothing.  repetition, frequency,
    presence: float32 [M] (1, 0, 0 without).  bias_ids / bias_values: int32 /
    float32 [M, n], n up to 1023, the last of several entries for one token counts,
    ids outside [0, V) for none.  allowed: int32 [M, ceil(V / 32)], bit v % 32 of
    word v // 32 set where v is allowed.  Lengths and lists are read on the device,
    so a captured call follows what they hold at each replay.  out: a contiguous
    [M, V] tensor of the logits' type, or the (contiguous) logits themselves."""
    dtype = logits.dtype
    if dtype is torch.float32:
        mode = _lib.LOGITS_FP32
    elif dtype is torch.bfloat16:
        mode = _lib.LOGITS_BF16
    else:
        raise ValueError(f"logits must be float32 or bfloat16, got {dtype}")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be [M, V], got {tuple(logits.shape)}")
    m, v = logits.shape
    index = logits.get_device()
    past = lens = prompts = rho = alpha_f = alpha_p = ids = values = words = None
    history_ld = history_len = bias_ld = bias_count = allowed_ld = 0
    if history is not None:
        past, history_ld, history_len = _row_list(history, m, torch.int32, index, "history")
        if history_len > _lib.CONSTRAIN_MAX_HISTORY:
            raise ValueError(f"history holds {history_len} tokens per row, at most {_lib.CONSTRAIN_MAX_HISTORY}")
        lens = _per_row(history_lens, m, torch.int32, index, "history_lens")
        prompts = _per_row(prompt_lens, m, torch.int32, index, "prompt_lens")
        rho = _per_row(repetition, m, torch.float32, index, "repetition")
        alpha_f = _per_row(frequency, m, torch.float32, index, "frequency")
        alpha_p = _per_row(presence, m, torch.float32, index, "presence")
        if history_len == 0:  # no token to count or to penalise
            past = lens = prompts = rho = alpha_f = alpha_p = None
    elif not (history_lens is prompt_lens is repetition is frequency is presence is None):
        raise ValueError("lengths or penalties given without a history")
    if bias_ids is not None and bias_values is not None:
        ids, bias_ld, bias_count = _row_list(bias_ids, m, torch.int32, index, "bias_ids")
        values, values_ld, values_count = _row_list(bias_values, m, torch.float32, index, "bias_values")
        if values_ld != bias_ld or values_count != bias_count:
            raise ValueError(f"bias_ids and bias_values must have the same shape and strides, got {tuple(bias_ids.shape)} "
                             f"/ {tuple(bias_values.shape)}")
        if bias_count > _lib.CONSTRAIN_MAX_BIAS:
            raise ValueError(f"{bias_count} biases per row, at most {_lib.CONSTRAIN_MAX_BIAS}")
    elif not (bias_ids is bias_values is None):
        raise ValueError("bias_ids and bias_values go together")
    if allowed is not None:
        words, allowed_ld, count = _row_list(allowed, m, torch.int32, index, "allowed")
        if count != (v + 31) // 32:
            raise ValueError(f"allowed must hold {(v + 31) // 32} words per row, got {count}")
    ld, unit = logits.stride()
    src = logits
    if (v > 1 and unit != 1) or (m > 1 and ld < v):
        src, ld = logits.contiguous(), v
    elif m == 1:
        ld = v
    if out is None:
        out = logits.new_empty((m, v))
    else:
        if out.dtype is not dtype or out.shape != logits.shape or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {dtype} tensor of {m} x {v} values")
        if out.get_device() != index:
            raise ValueError(f"out is on {out.device}, the call's tensors are on {logits.device}")
        if m and _overlap(out, logits) and not (src is logits and out.data_ptr() == src.data_ptr() and ld == v):
            raise ValueError("out must be the logits themselves (contiguous) or not overlap them")
    _require_device(logits, "logits")
    tokens = logits.new_empty((m,), dtype=torch.long)
    if m == 0:
        return out, tokens
    with _on_index(index):
        stream = torch._C._cuda_getCurrentRawStream(index)
        workspace = _constrain_workspace(logits, stream, m, v)
        status = _lib.load().lsk_constrain_logits(
            src.data_ptr(), mode, m, v, ld, past, history_ld, history_len, lens, prompts, rho, alpha_f, alpha_p, ids,
            values, bias_ld, bias_count, words, allowed_ld, out.data_ptr(), tokens.data_ptr(), workspace.data_ptr(),
            workspace.numel(), stream)
    _lib.check(status, "lsk_constrain_logits")
    return out, tokens


# Workspaces of constrain_logits by (device, stream).
_constrain_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def _constrain_workspace(logits: torch.Tensor, stream: int, m: int, v: int) -> torch.Tensor:
    """A workspace that is zero: the current stream's own, which every call leaves zero,
    or under capture the graph's own, so that replays share none with eager calls."""
    nbytes = _constrain_workspace_bytes(m, v)
    if torch.cuda.is_current_stream_capturing():
        return logits.new_empty((nbytes,), dtype=torch.uint8).zero_()
    key = (logits.get_device(), stream)
    workspace = _constrain_workspaces.get(key)
    if workspace is None or workspace.numel() < nbytes:
        workspace = logits.new_empty((max(nbytes, 4096),), dtype=torch.uint8).zero_()
        _constrain_workspaces[key] = workspace
    return workspace


@functools.lru_cache(maxsize=1024)
def _constrain_workspace_bytes(m: int, v: int) -> int:
    return _lib.load().lsk_constrain_workspace_bytes(m, v)


def sample_logits(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature: torch.Tensor | None = None,
                  top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                  min_p: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """A token drawn from each request's row of logits [M, V] (float32 or bfloat16), and the
    logarithm of its probability among the kept ones: (int64 [M], float32 [M]).

    Of the probabilities at `temperature` (1 without; 0 and below: the largest logit's token)
    the top_k largest are kept (all without, or below 1; the lower index of equal logits
    first), of those the ones of at least min_p times the largest, of those the shortest
    prefix that holds top_p of their sum.  The token is the first, in the order of
    indices, at which the running sum of the kept ones exceeds uniforms[m] (float32, in
    [0, 1), from a generator of the caller's) times their sum.  Weights are whole
    multiples of 2^-44 of the largest, so that the result depends on nothing but the
    arguments.  A row with a NaN, or of -inf alone, gives token -1 and NaN.

    uniforms, temperature, top_p, min_p: float32 [M], top_k: int32 [M], read on the
    device, so a captured call follows them.  A filter that no row uses is better left out:
    what is given decides how the rows are worked on.  V at most 2^19."""
    dtype = logits.dtype
    if dtype is torch.float32:
        mode = _lib.LOGITS_FP32
    elif dtype is torch.bfloat16:
        mode = _lib.LOGITS_BF16
    else:
        raise ValueError(f"logits must be float32 or bfloat16, got {dtype}")
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= _lib.SAMPLE_MAX_VOCAB:
        raise ValueError(f"logits must be [M, V] with V up to {_lib.SAMPLE_MAX_VOCAB}, got {tuple(logits.shape)}")
    m, v = logits.shape
    index = logits.get_device()
    if uniforms is None:
        raise ValueError("uniforms must be given")
    uniforms_at = _per_row(uniforms, m, torch.float32, index, "uniforms")
    temperature_at = _per_row(temperature, m, torch.float32, index, "temperature")
    k_at = _per_row(top_k, m, torch.int32, index, "top_k")
    p_at = _per_row(top_p, m, torch.float32, index, "top_p")
    min_p_at = _per_row(min_p, m, torch.float32, index, "min_p")
    _require_device(logits, "logits")
    ld, unit = logits.stride()
    if (v > 1 and unit != 1) or (m > 1 and ld < v):
        logits, ld = logits.contiguous(), v
    elif m == 1:
        ld = v
    tokens = logits.new_empty((m,), dtype=torch.long)
    logprobs = logits.new_empty((m,), dtype=torch.float32)
    if m == 0:
        return tokens, logprobs
    nbytes = _sample_workspace_bytes(mode, m, v, k_at is not None, p_at is not None, min_p_at is not None)
    workspace = logits.new_empty((nbytes,), dtype=torch.uint8) if nbytes else None
    with _on_index(index):
        status = _lib.load().lsk_sample_logits(
            logits.data_ptr(), mode, m, v, ld, uniforms_at, temperature_at, k_at, p_at, min_p_at, tokens.data_ptr(),
            logprobs.data_ptr(), _ptr(workspace), nbytes, torch._C._cuda_getCurrentRawStream(index))
    _lib.check(status, "lsk_sample_logits")
    return tokens, logprobs


@functools.lru_cache(maxsize=1024)
def _sample_workspace_bytes(mode: int, m: int, v: int, by_k: bool, by_p: bool, by_min_p: bool) -> int:
    return _lib.load().lsk_sample_workspace_bytes(mode, m, v, by_k, by_p, by_min_p)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


class StackStep:
    """A prepared stack program: many projections at the same M in one
    persistent launch (lsk_stack_prepare / lsk_stack_run).

    `projections` is a list of dicts with keys x, weight (PackedWeight), out,
    and optionally epilogue, residual, depends_on (index of an earlier entry:
    every entry up to it finishes before this one reads its inputs).  The
    program holds the tensors' addresses, so x, out and residual are used in
    place (rows of unit column stride, row strides a multiple of 8 elements,
    16-byte aligned): one entry's out can be a later entry's x.  A tensor
    that would need a copy is refused."""

    def __init__(self, projections: list[dict], m: int, device: torch.device | str) -> None:
        lib = _lib.load()
        device = torch.device(device)
        count = len(projections)
        arr = (_lib.Projection * count)()
        self._keep = []  # tensors whose pointers the program holds

        def in_place(t: torch.Tensor, t2: torch.Tensor, what: str) -> None:
            if t2.data_ptr() != t.data_ptr() or t2.stride(-1) != 1:
                raise ValueError(f"{what} must be usable in place (unit column stride, row stride a multiple "
                                 f"of 8, 16-byte aligned): the program holds its address")
            if t.device.type != "cuda" or t.device.index != (device.index if device.index is not None
                                                             else torch.cuda.current_device()):
                raise ValueError(f"{what} is on {t.device}, the program on {device}")

        for i, spec in enumerate(projections):
            w = spec["weight"]
            if not isinstance(w, PackedWeight):
                raise ValueError(f"projection {i}: weight must be a PackedWeight")
            x, out = spec["x"], spec["out"]
            epi = spec.get("epilogue", _lib.EPI_NONE)
            x2, xm, ldx = _rows(x, w.k, f"projection {i} x")
            if xm != m:
                raise ValueError(f"projection {i}: x has {xm} rows, the step runs M={m}")
            in_place(x, x2, f"projection {i} x")
            in_place(w.data, w.data, f"projection {i} weight")
            n_out = w.n // 2 if epi == _lib.EPI_SILU_MUL else w.n
            if out.dtype != torch.bfloat16 or out.shape[-1] != n_out or out.numel() != m * n_out:
                raise ValueError(f"projection {i}: out must be bfloat16 [{m}, {n_out}]")
            o2 = out.reshape(-1, n_out)
            in_place(out, o2, f"projection {i} out")
            ldy = o2.stride(0) if m > 1 else n_out
            res = spec.get("residual")
            res_ptr, ldr = None, 0
            if res is not None:
                r2, rm, ldr = _rows(res, w.n, f"projection {i} residual")
                if rm != m:
                    raise ValueError(f"projection {i}: residual has {rm} rows, the step runs M={m}")
                in_place(res, r2, f"projection {i} residual")
                res_ptr = r2.data_ptr()
                self._keep.append(r2)
            self._keep += [x2, o2, w.data]
            arr[i] = _lib.Projection(w.data.data_ptr(), w.layout, w.n, w.k, x2.data_ptr(), ldx, o2.data_ptr(), ldy,
                                     epi, res_ptr, ldr, int(spec.get("depends_on", -1)))
        self.count = count
        self.m = m
        with torch.cuda.device(device):
            self.program = torch.empty(lib.lsk_stack_program_bytes(count), dtype=torch.uint8, device=device)
            self.workspace = torch.zeros(lib.lsk_stack_workspace_bytes(count), dtype=torch.uint8, device=device)
            status = lib.lsk_stack_prepare(arr, count, m, self.program.data_ptr(), self.program.numel())
        _lib.check(status, "lsk_stack_prepare")

    def launch(self) -> None:
        lib = _lib.load()
        with torch.cuda.device(self.program.device):
            status = lib.lsk_stack_run(self.program.data_ptr(), self.count, self.workspace.data_ptr(),
                                       self.workspace.numel(), stream_handle())
        _lib.check(status, "lsk_stack_run")

    def error(self) -> int:
        """Read and clear the error word (synchronises): 0 if every wait completed."""
        lib = _lib.load()
        torch.cuda.synchronize(self.workspace.device)
        out = ctypes.c_int(0)
        _lib.check(lib.lsk_stack_error(self.workspace.data_ptr(), ctypes.byref(out)), "lsk_stack_error")
        return out.value

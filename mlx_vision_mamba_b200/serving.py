"""Serving operators: the selective scan and the causal conv1d + SiLU over a
cache of request states, and low-rank adapters beside a shared projection.

The reference runs whole sequences from a zero state
(mlx_vision_mamba/mamba_block.py:20-74,129-132).  A program that answers
requests with a trained MambaBlock instead keeps, per request, the recurrent
state and the last d_conv - 1 conv inputs in a slot of a cache, and in each
call brings prompts of different lengths and single new tokens of many
requests.  The rows of all requests lie one after the other in (rows,
channels) tensors; a `RequestBatch` says which rows belong to which request,
where its state lies and which adapter it uses, and

* `conv1d_silu_cached_cuda(x, weight, bias, state, batch)`
* `selective_scan_cached_cuda(x, delta, A, B, C, D, state, batch, z=None)`
* `lora_add_cuda(base, x, adapters, batch, out=None)`

run on it (`MambaBlock.serve` calls all three).  They update the state tensors
in place and have no gradient: with grad mode on they refuse inputs that
require one.  A call runs on the current stream of x's device, allocates only
its outputs (and the scan's carries, when it splits long prompts) and never
synchronises, so it can be captured into a CUDA graph after one eager call
with the same batch.

There is no CPU path: inputs must be CUDA tensors and libvmscan.so must load.
"""

from __future__ import annotations

from typing import Optional, Sequence

import numpy as np
import torch

from . import _native
from .scan import D_STATE

_DTYPES = (torch.float32, torch.bfloat16)
_MAX_ROWS = 1 << 30


def _int_list(name: str, values, count: Optional[int] = None) -> np.ndarray:
    """values (numbers on the host) as an int32 array of `count` entries."""
    if isinstance(values, torch.Tensor):
        if values.is_cuda:
            raise ValueError(f"RequestBatch: `{name}` must be on the host (its checks and launch sizes come from it)")
        values = values.numpy()
    arr = np.asarray(values)
    if arr.size == 0:
        arr = arr.astype(np.int64)
    if arr.ndim != 1 or arr.dtype.kind not in "iu":
        raise ValueError(f"RequestBatch: `{name}` must be a flat list of integers, got {arr.dtype} {arr.shape}")
    if count is not None and arr.size != count:
        raise ValueError(f"RequestBatch: `{name}` has {arr.size} entries for {count} requests")
    if arr.size and (int(arr.min()) < -1 or int(arr.max()) >= 1 << 31):
        raise ValueError(f"RequestBatch: `{name}` has an entry outside [-1, 2^31)")
    return np.ascontiguousarray(arr, dtype=np.int32)


class _Table:
    __slots__ = ("tensor", "host", "info", "captured")

    def __init__(self, tensor, host, info):
        self.tensor, self.host, self.info, self.captured = tensor, host, info, False


class RequestBatch:
    """The requests of one packed batch.

    lengths:  rows of each request (0 allowed: only its state is carried over).
    slots:    cache slot each request's state is written to; default 0, 1, ...;
              -1 makes a padding request: its rows come out as zeros (as `base`
              from lora_add_cuda) and no state is touched.
    sources:  slot each request's state is read from; default its own slot (a
              running request goes on); -1 starts from zeros (a fresh prompt);
              another slot forks a kept state (a shared prompt).
    adapters: adapter of each request for lora_add_cuda, -1 for none.

    All are host integers, checked here: no two requests may write one slot,
    and no request may read a slot that another one writes.  The operators
    take tensors of at least `tokens` rows; rows behind the last request come
    out as zeros (as `base` from lora_add_cuda).

    Device tables are made on first use, one copy per stream, and live as long
    as the batch: keep it while a CUDA graph captured with it is replayed.
    `update` changes slots, sources and adapters in place, also for captured
    graphs; the lengths are fixed.
    """

    def __init__(self, lengths: Sequence[int], slots=None, sources=None, adapters=None, device="cuda"):
        self.lengths = _int_list("lengths", lengths)
        self.count = int(self.lengths.size)
        if self.count == 0:
            raise ValueError("RequestBatch: no requests")
        if int(self.lengths.min()) < 0:
            raise ValueError("RequestBatch: a length is negative")
        self.tokens = int(self.lengths.sum(dtype=np.int64))
        if self.tokens > _MAX_ROWS:
            raise ValueError(f"RequestBatch: {self.tokens} rows (at most {_MAX_ROWS})")
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device() if torch.cuda.is_available() else 0)
        self.index = -2 if self.device.type != "cuda" else self.device.index
        self.single_tokens = bool((self.lengths == 1).all())
        self._tables = {}
        self._set(slots if slots is not None else np.arange(self.count), sources, adapters)

    def _set(self, slots, sources, adapters):
        slots = _int_list("slots", slots, self.count)
        sources = slots.copy() if sources is None else _int_list("sources", sources, self.count)
        sources[slots < 0] = -1
        written = slots[slots >= 0]
        if np.unique(written).size != written.size:
            raise ValueError("RequestBatch: two requests write the same slot")
        foreign = sources[(sources >= 0) & (sources != slots)]
        if np.intersect1d(foreign, written).size:
            raise ValueError("RequestBatch: a request reads a slot that another request writes")
        adapters = None if adapters is None else _int_list("adapters", adapters, self.count)
        self.slots, self.sources, self.adapters = slots, sources, adapters
        self.max_slot = int(max(slots.max(), sources.max()))
        self.max_adapter = -1 if adapters is None else int(adapters.max())

    def update(self, slots=None, sources=None, adapters=None) -> None:
        """New slots, sources and adapters (each default as in the constructor;
        adapters None keeps the present ones) for the same lengths.  The device
        tables are rewritten in order on the current stream: call it on the
        stream that uses the batch or replays graphs captured with it."""
        if _capturing():
            raise RuntimeError("RequestBatch.update: not while a CUDA graph is being captured")
        if adapters is not None and self.adapters is None and any(k[0] == "lora" for k in self._tables):
            raise RuntimeError("RequestBatch.update: the batch was made without adapters")
        self._set(slots if slots is not None else np.arange(self.count), sources,
                  self.adapters if adapters is None else adapters)
        if not self._tables:
            return
        here = torch.cuda.current_stream(self.device).cuda_stream
        # tables that another stream uses are dropped (made again there), unless
        # a graph has captured them: those are rewritten on this stream
        self._tables = {k: t for k, t in self._tables.items() if k[-1] == here or t.captured}
        for key, table in self._tables.items():
            host, info = self._build(key)
            if info != table.info or host.numel() != table.host.numel():
                raise RuntimeError("RequestBatch.update: table sizes changed")
            table.tensor.copy_(host, non_blocking=True)
            table.host = host

    def _build(self, key):
        """(pinned int32 host table, its sizes) of kind key[0]."""
        lib = _native.load()
        kind, arg = key[0], key[1]
        ptr = lambda a: a.ctypes.data  # noqa: E731
        if kind == "step":
            return _pinned(np.concatenate([self.slots, self.sources])), (self.count,)
        if kind == "lora":
            most = lib.vmscan_lora_tiles(self.count, ptr(self.lengths), ptr(self.adapters), self.max_adapter + 1, None,
                                         None, 0)
            if most < 0:
                _native.check(-most, "vmscan_lora_tiles")
            table = np.empty(4 * most + self.tokens, dtype=np.int32)
            if self.tokens:
                _check_count(lib.vmscan_lora_tiles(self.count, ptr(self.lengths), ptr(self.adapters),
                                                   self.max_adapter + 1, ptr(table) + 16 * most, ptr(table), most),
                             "vmscan_lora_tiles")
            return _pinned(table), (int(most),)
        if kind == "scan":
            rows, by_length = lib.vmscan_cached_scan_rows(self.count, ptr(self.lengths), arg), 1
        else:
            rows, by_length = lib.vmscan_cached_conv_rows(), 0
        if rows < 0:
            _native.check(-rows, "vmscan_cached_scan_rows")
        info = np.zeros(3, dtype=np.int64)
        args = (self.count, ptr(self.lengths), ptr(self.slots), ptr(self.sources), rows, by_length)
        n = _check_count(lib.vmscan_request_pieces(*args, None, 0, ptr(info)), "vmscan_request_pieces")
        table = np.empty(8 * n + 4 * int(info[1]), dtype=np.int32)
        _check_count(lib.vmscan_request_pieces(*args, ptr(table), table.size, ptr(info)), "vmscan_request_pieces")
        return _pinned(table), (int(n), int(info[0]), int(info[1]), int(info[2]))

    def _table(self, kind: str, stream: int, arg: int = 0) -> _Table:
        """The device table of a kind for a stream (the current one)."""
        key = (kind, arg, stream)
        table = self._tables.get(key)
        if table is not None and not (table.captured or _capturing()):
            return table
        if _capturing():
            # any stream's table will do: capture starts after a device-wide
            # synchronisation, so its upload has completed
            if table is None:
                table = next((t for k, t in self._tables.items() if k[:2] == key[:2]), None)
            if table is None:
                raise RuntimeError("RequestBatch: call the operator once with this batch before capturing it")
            table.captured = True
        elif table is None:
            host, info = self._build(key)
            table = _Table(host.to(self.device, non_blocking=True), host, info)
            self._tables[key] = table
        return table


def _check_count(n: int, where: str) -> int:
    if n < 0:
        _native.check(-int(n), where)
    return int(n)


_CUDA_BUILD = hasattr(torch._C, "_cuda_isCurrentStreamCapturing")


def _capturing() -> bool:
    return _CUDA_BUILD and torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


def _stream_of(index: int) -> int:
    """The current stream of a device as an integer handle.  (The Stream object
    of torch.cuda.current_stream takes 3 us to make, a quarter of a small call.)"""
    return torch._C._cuda_getCurrentRawStream(index)


def _pinned(a: np.ndarray) -> torch.Tensor:
    t = torch.from_numpy(a)
    return t.pin_memory() if torch.cuda.is_available() and a.size else t


class LoraAdapters:
    """Low-rank adapters of one projection: out += scale[i] (x a[i]^T) b[i]^T.

    a: (adapters, rank, d_in) and b: (adapters, d_out, rank), CUDA, fp32 or
    bf16 (the type of the activations they are used with); scale: one number
    per adapter (a list, or a tensor), default 1.  Adapters of a smaller rank
    are padded with zero rows / columns; rank is at most 128."""

    MAX_RANK = 128

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale=None):
        if not (isinstance(a, torch.Tensor) and isinstance(b, torch.Tensor) and a.is_cuda and b.is_cuda):
            raise RuntimeError("LoraAdapters: a and b must be CUDA tensors (there is no CPU path)")
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or 0 in a.shape + b.shape:
            raise ValueError(f"LoraAdapters: a must be (adapters, rank, d_in) and b (adapters, d_out, rank), got "
                             f"{tuple(a.shape)} and {tuple(b.shape)}")
        if a.dtype not in _DTYPES or b.dtype != a.dtype or a.device != b.device:
            raise ValueError(f"LoraAdapters: a and b must both be fp32 or both bf16 on one device, got {a.dtype} on "
                             f"{a.device} and {b.dtype} on {b.device}")
        if a.shape[1] > self.MAX_RANK:
            raise ValueError(f"LoraAdapters: rank {a.shape[1]} (at most {self.MAX_RANK})")
        self.count, self.rank, self.d_in = a.shape
        self.d_out = b.shape[1]
        self.a, self.b = a.detach().contiguous(), b.detach().contiguous()
        if scale is None:
            scale = torch.ones(self.count)
        scale = torch.as_tensor(scale, dtype=torch.float32)
        if tuple(scale.shape) != (self.count,):
            raise ValueError(f"LoraAdapters: scale must have {self.count} entries, got {tuple(scale.shape)}")
        self.scale = scale.detach().to(a.device).contiguous()


# The operators' small calls are bound by the host, so each tests all that a good
# call satisfies in one expression; only when that fails are the conditions gone
# through one by one to say which it was.


def _refuse_batch(where: str, batch, x) -> None:
    """Raises what is wrong with a batch and the rows it is used on."""
    if not isinstance(batch, RequestBatch):
        raise TypeError(f"{where}: `batch` must be a RequestBatch, got {type(batch).__name__}")
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError(f"{where}: inputs must be CUDA tensors (there is no CPU path)")
    if x.device != batch.device:
        raise ValueError(f"{where}: the batch is for {batch.device}, x is on {x.device}")
    if x.dim() != 2:
        raise ValueError(f"{where}: x must be (rows, channels), got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{where}: x must be fp32 or bf16, got {x.dtype}")
    if x.shape[0] < batch.tokens:
        raise ValueError(f"{where}: x has {x.shape[0]} rows, the batch's requests have {batch.tokens}")
    raise ValueError(f"{where}: x has {x.shape[0]} rows (at most {_MAX_ROWS})")


def _batch_ok(batch, x) -> bool:
    return (isinstance(batch, RequestBatch) and isinstance(x, torch.Tensor) and x.is_cuda
            and x.get_device() == batch.index and x.dim() == 2 and x.dtype in _DTYPES
            and batch.tokens <= x.shape[0] <= _MAX_ROWS)


def _refuse_tensors(where: str, x, named) -> None:
    """Raises for the first of (name, tensor, shape) that is no CUDA tensor of
    that shape on x's device."""
    for name, t, shape in named:
        if not isinstance(t, torch.Tensor) or t.device != x.device:
            raise RuntimeError(f"{where}: `{name}` must be a CUDA tensor on x's device (there is no CPU path)")
        if tuple(t.shape) != shape:
            raise ValueError(f"{where}: {name} must be {shape}, got {tuple(t.shape)}")


def _refuse_grad(where: str) -> None:
    raise RuntimeError(f"{where}: a serving operator has no gradient; call it under torch.no_grad()")


def _check_state(where: str, state, tail, dtype: torch.dtype, batch: RequestBatch) -> None:
    if (isinstance(state, torch.Tensor) and state.get_device() == batch.index and state.dim() == 3
            and state.shape[1:] == tail and state.dtype is dtype and state.is_contiguous()
            and batch.max_slot < state.shape[0] and state.data_ptr() % 16 == 0):
        return
    if not isinstance(state, torch.Tensor) or state.device != batch.device:
        raise RuntimeError(f"{where}: `state` must be a CUDA tensor on x's device")
    if state.dim() != 3 or tuple(state.shape[1:]) != tail or state.dtype != dtype:
        raise ValueError(f"{where}: state must be (slots, {tail[0]}, {tail[1]}) {dtype}, got {tuple(state.shape)} "
                         f"{state.dtype}")
    if batch.max_slot >= state.shape[0]:
        raise ValueError(f"{where}: the batch uses slot {batch.max_slot}, the state has {state.shape[0]} slots")
    raise ValueError(f"{where}: state must be contiguous and 16-byte aligned (it is updated in place)")


def _rows(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """t (rows, columns) in `dtype` with unit column stride (a view when it is so)."""
    if t.dtype is not dtype:
        t = t.to(dtype)
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _param(t: torch.Tensor) -> torch.Tensor:
    """A parameter as contiguous, 16-byte aligned fp32."""
    if t.dtype is torch.float32 and t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    t = t.detach().float().contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _out_rows(x: torch.Tensor, columns: int, batch: RequestBatch) -> torch.Tensor:
    """Output rows; those behind the last request are zero."""
    rows = x.shape[0]
    y = x.new_empty((rows, columns))
    if rows > batch.tokens:
        y[batch.tokens:].zero_()
    return y


def selective_scan_cached_cuda(x, delta, A, B, C, D, state, batch: RequestBatch,
                               z: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Selective scan of every request of `batch` from its stored state.

    Args (formulas and parameters as selective_scan_cuda):
        x, delta: (rows, D_inner) fp32 or bf16 (delta, B, C, z are cast to x's
            type when they differ); rows may be strided views
        A: (D_inner, 16); D: (D_inner,)
        B, C: (rows, 16)
        state: (slots, D_inner, 16) fp32, contiguous; the requests' source
            slots are read and their slots overwritten in place
        z: optional (rows, D_inner) gate; returns y * silu(z)
    Returns y (rows, D_inner) in x's type: zeros in the rows of padding
    requests and behind the last request.  The state and all arithmetic are
    fp32.  Every request's result is the one it has alone in a batch, up to
    rounding where a long prompt is split for speed.
    """
    where = "selective_scan_cached_cuda"
    if not _batch_ok(batch, x):
        _refuse_batch(where, batch, x)
    rows, dn = x.shape
    index, shape, bc = batch.index, x.shape, (rows, D_STATE)
    try:
        good = (delta.shape == shape and A.shape == (dn, D_STATE) and B.shape == bc and C.shape == bc
                and D.shape == (dn,) and (z is None or (z.shape == shape and z.get_device() == index))
                and delta.get_device() == A.get_device() == B.get_device() == C.get_device() == D.get_device() == index)
    except AttributeError:
        good = False
    if not good:
        named = [("delta", delta, (rows, dn)), ("A", A, (dn, D_STATE)), ("B", B, bc), ("C", C, bc), ("D", D, (dn,))]
        _refuse_tensors(where, x, named + ([("z", z, (rows, dn))] if z is not None else []))
    _check_state(where, state, (dn, D_STATE), torch.float32, batch)
    if torch.is_grad_enabled() and (x.requires_grad or delta.requires_grad or A.requires_grad or B.requires_grad
                                    or C.requires_grad or D.requires_grad or state.requires_grad
                                    or (z is not None and z.requires_grad)):
        _refuse_grad(where)
    if dn == 0:
        return torch.zeros_like(x)
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _scan_cached(x, delta, A, B, C, D, state, batch, z)
    return _scan_cached(x, delta, A, B, C, D, state, batch, z)


def _scan_cached(x, delta, A, B, C, D, state, batch, z):
    sd = x.dtype
    lib = _native.load()
    rows, dn = x.shape
    x, delta, B, C = _rows(x, sd), _rows(delta, sd), _rows(B, sd), _rows(C, sd)
    A, D = _param(A), _param(D)
    zp, ldz = None, 0
    if z is not None:
        z = _rows(z, sd)
        zp, ldz = z.data_ptr(), z.stride(0)
    y = _out_rows(x, dn, batch)
    stream = _stream_of(batch.index)
    args = (dn, D_STATE, sd is torch.bfloat16, x.data_ptr(), x.stride(0), delta.data_ptr(), delta.stride(0),
            A.data_ptr(), B.data_ptr(), B.stride(0), C.data_ptr(), C.stride(0), D.data_ptr(), zp, ldz, y.data_ptr(), dn,
            state.data_ptr(), state.shape[0])
    if batch.single_tokens:
        table = batch._table("step", stream).tensor.data_ptr()
        _native.check(lib.vmscan_cached_step(batch.tokens, *args, table, table + 4 * batch.count, stream),
                      "vmscan_cached_step")
        return y
    table = batch._table("scan", stream, dn)
    n, n_carry, n_chains, carry_rows = table.info
    ws, ws_n = None, 0
    if carry_rows:
        ws_n = _check_count(lib.vmscan_cached_scan_workspace_bytes(dn, carry_rows),
                            "vmscan_cached_scan_workspace_bytes")
        ws = torch.empty(ws_n, dtype=torch.uint8, device=x.device)
    pieces = table.tensor.data_ptr()
    _native.check(lib.vmscan_cached_scan(rows, *args, pieces, n, n_carry, pieces + 32 * n if n_chains else None,
                                         n_chains, carry_rows, None if ws is None else ws.data_ptr(), ws_n, stream),
                  "vmscan_cached_scan")
    return y


def conv1d_silu_cached_cuda(x, weight, bias, state, batch: RequestBatch) -> torch.Tensor:
    """silu(causal depthwise conv1d) of every request of `batch`, its rows
    preceded by the K - 1 conv inputs stored in its source slot.

    x: (rows, C) fp32 or bf16; weight: (C, K, 1) (MLX's Conv1d layout, K at
    most 8) and bias: (C,), used in fp32; state: (slots, K - 1, C) in x's type,
    contiguous, oldest input first: the requests' slots receive their last
    K - 1 inputs.  Returns (rows, C) in x's type: zeros in the rows of padding
    requests and behind the last request.
    """
    where = "conv1d_silu_cached_cuda"
    if not _batch_ok(batch, x):
        _refuse_batch(where, batch, x)
    rows, c = x.shape
    index = batch.index
    for name, t in (("weight", weight), ("bias", bias)):
        if not isinstance(t, torch.Tensor) or t.get_device() != index:
            raise RuntimeError(f"{where}: `{name}` must be a CUDA tensor on x's device (there is no CPU path)")
    if weight.dim() != 3 or weight.shape[0] != c or weight.shape[2] != 1 or bias.shape != (c,):
        raise ValueError(f"{where}: bad shapes x={tuple(x.shape)} weight={tuple(weight.shape)} bias={tuple(bias.shape)}")
    k = weight.shape[1]
    if not 1 <= k <= 8:
        raise ValueError(f"{where}: kernel size {k} (1 to 8)")
    _check_state(where, state, (k - 1, c), x.dtype, batch)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or bias.requires_grad
                                    or state.requires_grad):
        _refuse_grad(where)
    if c == 0:
        return torch.zeros_like(x)
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _conv_cached(x, weight, bias, state, batch, k)
    return _conv_cached(x, weight, bias, state, batch, k)


def _conv_cached(x, weight, bias, state, batch, k):
    rows, c = x.shape
    x = _rows(x, x.dtype)
    weight, bias = _param(weight), _param(bias)
    out = _out_rows(x, c, batch)
    stream = _stream_of(batch.index)
    table = batch._table("conv", stream)
    _native.check(_native.load().vmscan_cached_conv1d_silu(
        rows, c, k, x.dtype is torch.bfloat16, x.data_ptr(), x.stride(0), weight.data_ptr(), bias.data_ptr(),
        out.data_ptr(), c, state.data_ptr(), state.shape[0], table.tensor.data_ptr(), table.info[0], stream),
        "vmscan_cached_conv1d_silu")
    return out


def _span(t: torch.Tensor):
    """[first byte, last byte) that t (rows, columns) can touch."""
    e = t.element_size()
    return t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * e


def _collide(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether an element of out may also be one of t (column slices of the
    same wider rows do not collide)."""
    (a0, a1), (b0, b1) = _span(out), _span(t)
    if a1 <= b0 or b1 <= a0:
        return False
    e, ld = out.element_size(), out.stride(0)
    if t.element_size() == e and t.stride(0) == ld and ld > 0 and (b0 - a0) % e == 0:
        shift = (b0 - a0) // e % ld  # columns between the two slices
        return not (out.shape[1] <= shift and shift + t.shape[1] <= ld)
    return True


def lora_add_cuda(base: torch.Tensor, x: torch.Tensor, adapters: LoraAdapters, batch: RequestBatch,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """base + scale (x a^T) b^T with the adapter of each row's request: the
    low-rank part of many requests' adapters beside the shared projection
    `base = x W^T`.

    base: (rows, d_out) and x: (rows, d_in) in the adapters' type; batch: made
    with `adapters`.  Rows of requests with adapter -1 and rows behind the last
    request are base's.  `out` (rows, d_out) receives the result: base itself
    for an update in place, or a tensor that overlaps neither base nor x
    (default: a new one).  Products and sums are fp32; a bf16 result is rounded
    once.
    """
    where = "lora_add_cuda"
    if not _batch_ok(batch, x):
        _refuse_batch(where, batch, x)
    if not isinstance(adapters, LoraAdapters):
        raise TypeError(f"{where}: `adapters` must be LoraAdapters, got {type(adapters).__name__}")
    rows, index, dtype = x.shape[0], batch.index, adapters.a.dtype
    wide = (rows, adapters.d_out)
    for name, t, shape in (("x", x, (rows, adapters.d_in)), ("base", base, wide), ("out", out, wide)):
        if t is None and name == "out":
            continue
        if not isinstance(t, torch.Tensor) or t.get_device() != index:
            raise RuntimeError(f"{where}: `{name}` must be a CUDA tensor on x's device (there is no CPU path)")
        if t.shape != shape:
            raise ValueError(f"{where}: {name} must be {shape}, got {tuple(t.shape)}")
        if t.dtype is not dtype:
            raise TypeError(f"{where}: {name} is {t.dtype}, the adapters are {dtype}")
        if t.requires_grad and torch.is_grad_enabled():
            _refuse_grad(where)
    if adapters.a.get_device() != index:
        raise ValueError(f"{where}: the adapters are on {adapters.a.device}, x is on {x.device}")
    if batch.adapters is None:
        raise ValueError(f"{where}: the batch was made without adapters")
    if batch.max_adapter >= adapters.count:
        raise ValueError(f"{where}: the batch uses adapter {batch.max_adapter}, there are {adapters.count}")
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _lora_add(where, base, x, adapters, batch, out)
    return _lora_add(where, base, x, adapters, batch, out)


def _lora_add(where, base, x, adapters, batch, out):
    rows = x.shape[0]
    x = _rows(x, x.dtype)
    if out is None:
        base = _rows(base, base.dtype)
        out = base.new_empty((rows, adapters.d_out))
        in_place = False
    else:
        in_place = out is base or (out.data_ptr() == base.data_ptr() and out.stride() == base.stride())
        if rows and ((out.stride(1) != 1 and out.shape[1] > 1) or (rows > 1 and out.stride(0) < out.shape[1])):
            raise ValueError(f"{where}: out must have unit column stride and rows that do not overlap")
        base = base if in_place else _rows(base, base.dtype)
        if rows and (_collide(out, x) or (not in_place and _collide(out, base))):
            raise ValueError(f"{where}: out overlaps x or base (it may only be base itself)")
    if rows > batch.tokens and not in_place:
        out[batch.tokens:].copy_(base[batch.tokens:])
    if batch.tokens == 0:
        return out
    stream = _stream_of(batch.index)
    table = batch._table("lora", stream)
    tiles = table.info[0]
    p = table.tensor.data_ptr()
    _native.check(_native.load().vmscan_lora_add(
        rows, adapters.d_in, adapters.d_out, adapters.rank, adapters.count, x.dtype is torch.bfloat16, x.data_ptr(), x.stride(0),
        adapters.a.data_ptr(), adapters.b.data_ptr(), adapters.scale.data_ptr(), base.data_ptr(), base.stride(0),
        out.data_ptr(), out.stride(0), p + 16 * tiles, batch.tokens, p, tiles, stream), "vmscan_lora_add")
    return out

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
in place (which autograd is told of) and have no derivatives: with grad mode on
they refuse inputs that require a gradient, and dual tensors while forward mode
is on.  A call runs on the current stream of x's device, allocates only
its outputs (and the scan's carries, when it splits long prompts) and never
synchronises, so it can be captured into a CUDA graph after one eager call
with the same batch.

There is no CPU path: inputs must be CUDA tensors and libvmscan.so must load.
"""

from __future__ import annotations

import threading
from typing import Optional, Sequence

import numpy as np
import torch

from . import _native
from .scan import D_STATE

_DTYPES = (torch.float32, torch.bfloat16)
_MAX_ROWS = 1 << 30
# Held while a batch's tables are made, taken for a graph or rewritten, so that
# threads agree on them (not by calls that find theirs).
_TABLES = threading.Lock()


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
    return np.array(arr, dtype=np.int32, order="C")  # a copy: what was checked stays as it was


class _Table:
    """A device table, its pinned source, the stream it was made on and what the
    operators are told of it: (address, sizes...).  captured: a graph uses it;
    limit: slots of the smallest cache that one uses it with."""

    __slots__ = ("tensor", "host", "stream", "told", "captured", "limit")

    def __init__(self, host, info, device):
        self.host, self.stream = host, torch.cuda.current_stream(device)
        # an inference tensor could not be rewritten by an update outside inference mode
        with torch.inference_mode(False):
            self.tensor = torch.empty(host.shape, dtype=host.dtype, device=device)
            self.tensor.copy_(host, non_blocking=True)
        self.told, self.captured, self.limit = (self.tensor.data_ptr(), *info), False, None

    def write(self, host, here):
        """The table becomes `host` on stream `here`, after what its own stream
        has been given and before what that one is given next."""
        if self.stream != here:
            here.wait_stream(self.stream)
        try:
            with torch.cuda.stream(here):
                self.tensor.copy_(host, non_blocking=True)
        finally:
            if self.stream != here:
                self.stream.wait_stream(here)


class RequestBatch:
    """The requests of one packed batch.

    lengths:  rows of each request (0 allowed: only its state is carried over).
    slots:    cache slot each request's state is written to; default 0, 1, ...;
              -1 makes a padding request: its rows come out as zeros (as `base`
              from lora_add_cuda, whatever its adapter) and no state is touched.
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
    graphs; the lengths are fixed.  The attributes are for reading.
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
        self._set(slots, sources, adapters)

    def _set(self, slots, sources, adapters):
        slots = _int_list("slots", np.arange(self.count) if slots is None else slots, self.count)
        sources = slots.copy() if sources is None else _int_list("sources", sources, self.count)
        sources[slots < 0] = -1
        written = slots[slots >= 0]
        if np.unique(written).size != written.size:
            raise ValueError("RequestBatch: two requests write the same slot")
        foreign = sources[(sources >= 0) & (sources != slots)]
        if np.intersect1d(foreign, written).size:
            raise ValueError("RequestBatch: a request reads a slot that another request writes")
        given = None if adapters is None else _int_list("adapters", adapters, self.count)
        adapters = None if given is None else np.where(slots < 0, np.int32(-1), given)
        for a in (self.lengths, slots, sources, given, adapters):
            if a is not None:
                a.setflags(write=False)
        self.slots, self.sources, self.adapters, self._adapters_given = slots, sources, adapters, given
        self.max_slot = int(max(slots.max(), sources.max()))
        self.max_adapter = -2 if adapters is None else int(adapters.max())  # -2: made without adapters

    def update(self, slots=None, sources=None, adapters=None) -> None:
        """New slots, sources and adapters for the same lengths.  What is left
        out stays as it is, but for the sources of new slots, which default to
        the requests' own slots as in the constructor.
        The device tables are rewritten on the current stream, after what other
        streams have run with this batch so far and before what they run later;
        graphs captured with it must be replayed in order with the current
        stream.  Nothing changes when the new values are refused or a table
        cannot be rewritten."""
        if _capturing():
            raise RuntimeError("RequestBatch.update: not while a CUDA graph is being captured")
        with _TABLES:
            self._update(slots, sources, adapters)

    def _update(self, slots, sources, adapters) -> None:
        names = ("slots", "sources", "adapters", "_adapters_given", "max_slot", "max_adapter")
        before = {n: getattr(self, n) for n in names}
        if slots is None:
            slots, sources = self.slots, self.sources if sources is None else sources
        try:
            self._set(slots, sources, self._adapters_given if adapters is None else adapters)
            limit = min((t.limit for t in self._tables.values() if t.limit is not None), default=None)
            if limit is not None and self.max_slot >= limit:
                raise ValueError(f"RequestBatch.update: slot {self.max_slot} in a graph whose cache has {limit} slots")
            new = [(table, *self._build(key)) for key, table in self._tables.items()]
            if any(info != table.told[1:] for table, _, info in new):
                raise RuntimeError("RequestBatch.update: table sizes changed")
        except Exception:
            for n, v in before.items():
                setattr(self, n, v)
            raise
        if not new:
            return
        here = torch.cuda.current_stream(self.device)
        written = []
        try:
            for table, host, _ in new:
                table.write(host, here)
                written.append(table)
        except Exception:
            # The values go back, and with them what the graphs read; the tables
            # that no graph holds are made anew by the next call that needs them.
            for n, v in before.items():
                setattr(self, n, v)
            self._tables = {k: t for k, t in self._tables.items() if t.captured}
            for table in written:
                if table.captured:
                    table.write(table.host, here)
            raise
        for table, host, _ in new:
            table.host = host

    def _build(self, key):
        """(pinned int32 host table, its sizes) of kind key[0]."""
        lib = _native.load()
        kind, arg = key[0], key[1]
        ptr = lambda a: a.ctypes.data  # noqa: E731
        if kind == "step":
            return _pinned(np.concatenate([self.slots, self.sources])), (self.count,)
        if kind == "lora":
            most = lib.vmscan_lora_tiles(self.count, ptr(self.lengths), ptr(self.adapters), arg, None, None, 0)
            if most < 0:
                _native.check(-most, "vmscan_lora_tiles")
            table = np.empty(4 * most + self.tokens, dtype=np.int32)
            if self.tokens:
                _check_count(lib.vmscan_lora_tiles(self.count, ptr(self.lengths), ptr(self.adapters), arg,
                                                   ptr(table) + 16 * most, ptr(table), most), "vmscan_lora_tiles")
            return _pinned(table), (int(most),)
        if kind == "scan":
            with torch.cuda.device(self.index if self.index >= 0 and torch.cuda.is_initialized() else -1):
                rows, scan = lib.vmscan_cached_scan_rows(self.count, ptr(self.lengths), arg // 2, arg % 2), 1
        else:
            rows, scan = lib.vmscan_cached_conv_rows(self.tokens, arg), 0
        if rows < 0:
            _native.check(-rows, "vmscan_cached_scan_rows")
        info = np.zeros(5, dtype=np.int64)
        args = (self.count, ptr(self.lengths), ptr(self.slots), ptr(self.sources), rows, scan)
        n = _check_count(lib.vmscan_request_pieces(*args, None, 0, ptr(info)), "vmscan_request_pieces")
        table = np.empty(8 * n + 4 * int(info[1]), dtype=np.int32)
        _check_count(lib.vmscan_request_pieces(*args, ptr(table), table.size, ptr(info)), "vmscan_request_pieces")
        return _pinned(table), (int(n), *(int(v) for v in info))

    def _table(self, kind: str, stream: int, arg: int, capturing: bool, slots: int):
        """(address, sizes...) of the device table of a kind for the current
        stream; called by the operators (slots: of the cache they are given)."""
        key = (kind, arg, stream)
        table = self._tables.get(key)
        if table is None or capturing:
            with _TABLES:
                table = self._table_for_graph(key, slots) if capturing else self._new_table(key)
        return table.told

    def _new_table(self, key):
        table = self._tables.get(key)  # another thread's, made meanwhile
        if table is None:
            host, info = self._build(key)
            self._tables[key] = table = _Table(host, info, self.device)
        return table

    def _table_for_graph(self, key, slots: int):
        # any stream's table will do: capture starts after a device-wide
        # synchronisation, so its upload has completed
        table = self._tables.get(key) or next((t for k, t in self._tables.items() if k[:2] == key[:2]), None)
        if table is None:
            raise RuntimeError("RequestBatch: call the operator once with this batch before capturing it")
        table.captured = True
        if key[0] != "lora":
            table.limit = slots if table.limit is None else min(slots, table.limit)
        return table


def _check_count(n: int, where: str) -> int:
    if n < 0:
        _native.check(-int(n), where)
    return int(n)


_CUDA_BUILD = hasattr(torch._C, "_cuda_isCurrentStreamCapturing")


def _capturing() -> bool:
    return _CUDA_BUILD and torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


def _pinned(a: np.ndarray) -> torch.Tensor:
    t = torch.from_numpy(a)
    return t.pin_memory() if torch.cuda.is_available() and a.size else t


class LoraAdapters:
    """Low-rank adapters of one projection: out += scale[i] (x a[i]^T) b[i]^T.

    a: (adapters, rank, d_in) and b: (adapters, d_out, rank), CUDA, fp32 or
    bf16 (the type of the activations they are used with); scale: one number
    per adapter (a list, or a tensor), default 1.  Adapters of a smaller rank
    than the others' are given with zero rows / columns; rank is at most 128.

    The factors are copied: `a` and `b` are views of the copies, whose rows are
    padded with zeros to whole accesses (ranks to a multiple of 4, rows of a to
    16 bytes), and later changes to the tensors that were passed are not seen."""

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
        unit = 16 // a.element_size()
        rank, wide = -(-self.rank // 4) * 4, -(-self.d_in // unit) * unit
        self.a = a.new_zeros((self.count, rank, wide))[:, :self.rank, :self.d_in]
        self.b = b.new_zeros((self.count, self.d_out, rank))[:, :, :self.rank]
        self.a.copy_(a.detach())
        self.b.copy_(b.detach())
        if scale is None:
            scale = torch.ones(self.count)
        scale = torch.as_tensor(scale, dtype=torch.float32)
        if tuple(scale.shape) != (self.count,):
            raise ValueError(f"LoraAdapters: scale must have {self.count} entries, got {tuple(scale.shape)}")
        self.scale = scale.detach().to(a.device, copy=True).contiguous()

    def check(self, where: str, d_in: int, d_out: int, dtype: torch.dtype, batch: RequestBatch) -> None:
        """Raises unless lora_add_cuda takes these adapters for x (rows, d_in)
        and base (rows, d_out) of a type and a batch."""
        if not isinstance(batch, RequestBatch):
            raise TypeError(f"{where}: `batch` must be a RequestBatch, got {type(batch).__name__}")
        if (self.d_in, self.d_out) != (d_in, d_out):
            raise ValueError(f"{where}: adapters of {self.d_in} -> {self.d_out} beside a projection {d_in} -> {d_out}")
        if self.a.dtype != dtype:
            raise TypeError(f"{where}: adapters are {self.a.dtype}, the activations {dtype}")
        if self.a.get_device() != batch.index:
            raise ValueError(f"{where}: the adapters are on {self.a.device}, the batch is for device {batch.index}")
        if batch.max_adapter < -1:
            raise ValueError(f"{where}: the batch was made without adapters")
        if batch.max_adapter >= self.count:
            raise ValueError(f"{where}: the batch uses adapter {batch.max_adapter}, there are {self.count}")


_ext_module = None


def _ext():
    """The compiled entry points (csrc/serving_ext.cpp): checks, outputs and
    launches of the operators below."""
    global _ext_module
    if _ext_module is None:
        _native.load()
        try:
            from . import _serving_ext
        except ImportError as e:
            raise ImportError(f"_serving_ext.so is missing or does not load ({e}); build it with "
                              "`python -m mlx_vision_mamba_b200.build`") from e
        _serving_ext.setup(RequestBatch, LoraAdapters)
        _ext_module = _serving_ext
    return _ext_module


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
    return (_ext_module or _ext()).scan(x, delta, A, B, C, D, state, batch, z)


def conv1d_silu_cached_cuda(x, weight, bias, state, batch: RequestBatch) -> torch.Tensor:
    """silu(causal depthwise conv1d) of every request of `batch`, its rows
    preceded by the K - 1 conv inputs stored in its source slot.

    x: (rows, C) fp32 or bf16; weight: (C, K, 1) (MLX's Conv1d layout, K at
    most 8) and bias: (C,), used in fp32; state: (slots, K - 1, C) in x's type,
    contiguous, oldest input first: the requests' slots receive their last
    K - 1 inputs.  Returns (rows, C) in x's type: zeros in the rows of padding
    requests and behind the last request.
    """
    return (_ext_module or _ext()).conv(x, weight, bias, state, batch)


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
    once.  A row of x with a NaN or an infinity comes out as NaN (or infinite)
    where its request has an adapter, whatever the factors; so does one whose
    values, factors or inner products reach 3.39e38, the last step of fp32's
    range.  A row's result does not depend on the rows beside it.
    """
    return (_ext_module or _ext()).lora(base, x, adapters, batch, out)

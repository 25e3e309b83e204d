"""Host side of the serving operators, without a GPU: the checks of
RequestBatch and of the operators, and the tables that tell the kernels which
rows, slots and adapters they work on."""

import contextlib
import os
import re
import threading
import time

import numpy as np
import pytest
import torch

from mlx_vision_mamba_b200 import (
    LoraAdapters,
    MambaBlock,
    RequestBatch,
    _native,
    build,
    conv1d_silu_cached_cuda,
    lora_add_cuda,
    selective_scan_cached_cuda,
)


@pytest.mark.parametrize(
    "kw",
    [
        dict(lengths=[]),
        dict(lengths=[3, -1]),
        dict(lengths=[1.5, 2.0]),
        dict(lengths=[[1, 2]]),
        dict(lengths=[1 << 30, 1]),
        dict(lengths=[2, 2], slots=[0]),
        dict(lengths=[2, 2], slots=[4, 4]),  # one slot written twice
        dict(lengths=[2, 2], slots=[0, -2]),
        dict(lengths=[2, 2], slots=[0, 1], sources=[1, 1]),  # reads a slot that the other writes
        dict(lengths=[2, 2], slots=[0, 1], sources=[0, 0]),
        dict(lengths=[0, 2], slots=[0, 1], sources=[0, 0]),
        dict(lengths=[2, 2], slots=[0, 1], sources=[5]),
        dict(lengths=[2, 2], adapters=[0]),
        dict(lengths=[2, 2], adapters=[0, -2]),
        dict(lengths=[2, 2], slots=[0, 1 << 31]),
    ],
)
def test_bad_batches_are_refused(kw):
    with pytest.raises(ValueError):
        RequestBatch(**kw)


def test_allowed_batches():
    b = RequestBatch([2, 0, 5], slots=[3, -1, 4], sources=[7, 4, 7])  # a fork; a padding request reads nothing
    assert b.tokens == 7 and b.count == 3 and b.max_slot == 7 and not b.single_tokens
    assert b.sources.tolist() == [7, -1, 7]
    assert RequestBatch([1, 1], slots=[-1, -1]).max_slot == -1
    assert RequestBatch([1] * 5).single_tokens
    assert RequestBatch(torch.tensor([4, 1])).sources.tolist() == [0, 1]
    assert RequestBatch([1], sources=[-1]).sources.tolist() == [-1]


def test_a_batch_keeps_what_it_checked():
    """The caller's arrays are copied, the batch's cannot be written, and a
    padding request has neither source nor adapter."""
    slots, sources = np.array([4, -1], np.int32), np.array([2, 3], np.int32)
    b = RequestBatch(np.array([1, 1], np.int32), slots=slots, sources=sources, adapters=[0, 1])
    assert sources.tolist() == [2, 3] and b.sources.tolist() == [2, -1] and b.adapters.tolist() == [0, -1]
    slots[0] = 99
    assert b.slots.tolist() == [4, -1]
    for a in (b.lengths, b.slots, b.sources, b.adapters):
        with pytest.raises(ValueError):
            a[0] = 7
    b.update(slots=[1, 2])  # the adapters that were given come back
    assert b.sources.tolist() == [1, 2] and b.adapters.tolist() == [0, 1]
    with pytest.raises(ValueError):
        b.update(slots=[3, 3])
    assert b.slots.tolist() == [1, 2] and b.max_slot == 2


def test_an_update_keeps_what_it_is_not_given():
    b = RequestBatch([1, 1, 1], slots=[5, 6, -1], sources=[-1, 8, 0], adapters=[0, 1, 2])
    b.update(adapters=[2, 2, 2])
    assert b.slots.tolist() == [5, 6, -1] and b.sources.tolist() == [-1, 8, -1] and b.adapters.tolist() == [2, 2, -1]
    b.update()
    assert b.slots.tolist() == [5, 6, -1] and b.sources.tolist() == [-1, 8, -1] and b.max_slot == 8
    b.update(sources=[5, -1, -1])
    assert b.slots.tolist() == [5, 6, -1] and b.sources.tolist() == [5, -1, -1]
    with pytest.raises(ValueError):
        b.update(sources=[6, -1, -1])  # the second request writes it
    b.update(slots=[7, 8, 9])  # new slots: their own are the sources
    assert b.sources.tolist() == [7, 8, 9] and b.adapters.tolist() == [2, 2, 2] and b.max_slot == 9


def _pieces(batch, rows, scan):
    lib = _native.load()
    info = np.zeros(5, dtype=np.int64)
    p = lambda a: a.ctypes.data  # noqa: E731
    args = (batch.count, p(batch.lengths), p(batch.slots), p(batch.sources), rows, scan)
    n = lib.vmscan_request_pieces(*args, None, 0, p(info))
    size = 8 * n + 4 * int(info[1])
    table = np.full(size + 8, 77, dtype=np.int32)
    assert lib.vmscan_request_pieces(*args, p(table), size, p(info)) == n
    assert (table[size:] == 77).all()  # writes what it counted
    assert lib.vmscan_request_pieces(*args, p(table), size - 1, p(info)) == -6
    return table[:8 * n].reshape(n, 8), table[8 * n:size].reshape(-1, 4), info


@pytest.mark.parametrize("scan", [0, 1])
@pytest.mark.parametrize("rows", [0, 1, 7, 8, 32, 64, 1000])
@pytest.mark.parametrize("lengths", [[1], [0], [0, 0, 3], [65, 0, 1, 64, 63, 200], [1000], [8, 9, 7, 16, 17]])
def test_pieces_cover_every_row_once(lengths, rows, scan):
    n = len(lengths)
    slots = [i if i != 2 else -1 for i in range(n)]
    batch = RequestBatch(lengths, slots=slots, sources=[(n + i) if i % 2 else -1 for i in range(n)])
    pieces, chains, info = _pieces(batch, rows, scan)
    first, later = pieces[:int(info[0])], pieces[int(info[0]):]
    begins = np.concatenate([[0], np.cumsum(lengths)])
    written = np.zeros(int(begins[-1]), dtype=int)
    owners = {}
    for phase, group in enumerate((first, later)):
        for t0, t1, begin, end, source, slot, carry, ordinal in group:
            assert begin <= t0 <= t1 <= end and (t1 > t0 or begin == end)  # only an empty request has an empty piece
            assert rows == 0 or t1 - t0 <= ((rows + 7) // 8 * 8 if scan else rows)
            if not (phase == 0 and carry >= 0 and ordinal > 0):  # a carry writes no rows
                written[t0:t1] += 1
                owners.setdefault((begin, end, slot), []).append((ordinal, t0, t1, source, carry, phase))
            else:
                assert [t0, t1, begin, end, source, slot, carry, ordinal] in later.tolist() and t1 < end
    assert (written == 1).all()
    used = []
    for i in range(n):
        mine = sorted(owners[(begins[i], begins[i + 1], slots[i])])
        assert [m[0] for m in mine] == list(range(len(mine)))
        assert mine[0][1] == begins[i] and mine[-1][2] == begins[i + 1]
        assert all(m[3] == batch.sources[i] for m in mine)
        if scan:
            assert [m[5] for m in mine] == [0] + [1] * (len(mine) - 1)
        if not scan or len(mine) == 1:
            assert all(m[4] == -1 for m in mine)
        else:
            carries = [m[4] for m in mine]
            assert carries == list(range(carries[0], carries[0] + len(mine)))
            assert [carries[0], len(mine), 0, 0] in chains.tolist() and len(mine) <= info[3]
            # the pieces between the first and the last one leave a carry in the first phase
            assert sorted(r[7] for r in first.tolist() if r[6] in carries) == list(range(len(mine) - 1))
            used += carries
    assert sorted(used) == list(range(int(info[2]))) and len(chains) == info[1]
    if scan:  # long pieces first
        assert (np.diff(first[:, 1] - first[:, 0]) <= 0).all() and (np.diff(later[:, 1] - later[:, 0]) <= 0).all()
    else:
        assert len(later) == 0 and (np.diff(pieces[:, 0]) >= 0).all()


def test_scan_rows_rule():
    """One long prompt is split, a full batch of even prompts is not."""
    lib = _native.load()

    def rows(lengths, dn):
        a = np.asarray(lengths, np.int32)
        return lib.vmscan_cached_scan_rows(a.size, a.ctypes.data, dn, 0)

    assert 0 < rows([32768], 768) < 8192
    assert rows([512] * 256, 1536) == 0
    assert rows([1] * 10, 64) == 0
    assert lib.vmscan_cached_scan_rows(0, None, 64, 0) == -2


@pytest.mark.parametrize("lengths", [[1] * 40, [100, 0, 3, 17, 16, 1], [0, 0]])
def test_lora_tiles(lengths):
    lib = _native.load()
    n = len(lengths)
    rng = np.random.RandomState(n)
    ads = rng.randint(-1, 3, n)
    batch = RequestBatch(lengths, adapters=ads)
    p = lambda a: a.ctypes.data  # noqa: E731
    args = (n, p(batch.lengths), p(batch.adapters), 3)
    most = lib.vmscan_lora_tiles(*args, None, None, 0)
    index, tiles = np.full(batch.tokens + 4, -5, np.int32), np.full((most + 1, 4), -5, np.int32)
    if most:
        assert lib.vmscan_lora_tiles(*args, p(index), p(tiles), most) == most
        assert lib.vmscan_lora_tiles(*args, p(index), p(tiles), most - 1) == -6
    assert (index[batch.tokens:] == -5).all() and (tiles[most:] == -5).all()
    assert sorted(index[:batch.tokens].tolist()) == list(range(batch.tokens))
    of_row = np.repeat(ads, lengths)
    covered = 0
    for first, count, ad, _ in tiles[:most]:
        assert (of_row[index[first:first + count]] == ad).all() or count == 0
        covered += count
    assert covered == batch.tokens
    assert lib.vmscan_lora_tiles(n, p(batch.lengths), p(batch.adapters), 1, None, None, 0) == (-2 if ads.max() > 0 else most)


def test_operators_refuse_cpu_tensors_and_wrong_batches():
    b = RequestBatch([2], device="cpu")
    x = torch.zeros(2, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        selective_scan_cached_cuda(x, x, torch.zeros(4, 16), x, x, torch.zeros(4), torch.zeros(1, 4, 16), b)
    with pytest.raises(RuntimeError, match="CUDA"):
        conv1d_silu_cached_cuda(x, torch.zeros(4, 4, 1), torch.zeros(4), torch.zeros(1, 3, 4), b)
    with pytest.raises(RuntimeError, match="CUDA"):
        lora_add_cuda(x, x, None, b)
    with pytest.raises(TypeError, match="RequestBatch"):
        conv1d_silu_cached_cuda(x, torch.zeros(4, 4, 1), torch.zeros(4), torch.zeros(1, 3, 4), [2])
    with pytest.raises(RuntimeError, match="CUDA"):
        LoraAdapters(torch.zeros(1, 2, 4), torch.zeros(1, 4, 2))


def test_c_entry_points_validate():
    """Every call here returns before any CUDA work."""
    lib = _native.load()
    P = 4096
    scan = lambda **o: lib.vmscan_cached_scan(*[{**dict(  # noqa: E731
        rows=4, dn=8, ds=16, bf16=0, u=P, ldu=8, dl=P, ldd=8, A=P, B=P, ldb=16, C=P, ldc=16, D=P, z=None, ldz=0, y=P,
        ldy=8, state=P, slots=2, pieces=P, n=1, nf=1, chains=None, nch=0, cr=0, lc=1, un=0, ws=None, wn=0, stream=None), **o}[k]
        for k in ("rows dn ds bf16 u ldu dl ldd A B ldb C ldc D z ldz y ldy state slots pieces n nf chains nch cr lc un ws wn "
                  "stream").split()])
    assert scan(ds=8) == 3
    assert scan(A=None) == 1 and scan(u=None) == 1 and scan(state=None) == 1 and scan(pieces=None) == 1
    assert scan(dn=0) == 2 and scan(rows=-1) == 2 and scan(slots=0) == 2 and scan(ldy=7) == 2 and scan(ldu=-8) == 2
    assert scan(n=0) == 2 and scan(n=1, nf=2) == 2 and scan(nf=0) == 2 and scan(cr=3) == 2 and scan(n=2) == 2
    assert scan(A=P + 4) == 4 and scan(state=P + 8) == 4 and scan(pieces=P + 4) == 4
    assert scan(n=4, nf=2, chains=P, nch=1, cr=3) == 6  # no workspace
    need = lib.vmscan_cached_scan_workspace_bytes(8, 3)
    assert need >= 3 * 8 * 33 * 4
    assert scan(n=4, nf=2, chains=P, nch=1, cr=3, ws=P, wn=need - 1) == 6
    assert lib.vmscan_cached_scan_workspace_bytes(0, 3) == -2
    step = lambda **o: lib.vmscan_cached_step(*[{**dict(  # noqa: E731
        rows=4, dn=8, ds=16, bf16=0, u=P, ldu=8, dl=P, ldd=8, A=P, B=P, ldb=16, C=P, ldc=16, D=P, z=None, ldz=0, y=P,
        ldy=8, state=P, slots=2, slot=P, source=P, stream=None), **o}[k]
        for k in "rows dn ds bf16 u ldu dl ldd A B ldb C ldc D z ldz y ldy state slots slot source stream".split()])
    assert step(slot=None) == 1 and step(rows=0) == 2 and step(ds=4) == 3
    conv = lambda **o: lib.vmscan_cached_conv1d_silu(*[{**dict(  # noqa: E731
        rows=4, c=8, k=4, bf16=0, x=P, ldx=8, w=P, b=P, out=P, ldo=8, state=P, slots=2, pieces=P, n=1, stream=None),
        **o}[k] for k in "rows c k bf16 x ldx w b out ldo state slots pieces n stream".split()])
    assert conv(k=0) == 10 and conv(k=9) == 10 and conv(state=None) == 1 and conv(x=None) == 1 and conv(n=0) == 2
    assert conv(ldo=4) == 2 and conv(c=0) == 2 and conv(pieces=P + 8) == 4
    lora = lambda **o: lib.vmscan_lora_add(*[{**dict(  # noqa: E731
        rows=4, di=8, do=8, r=4, ad=2, bf16=0, x=P, ldx=8, a=P, lda=8, b=P, s=P, base=P, ldb=8, out=P, ldo=8, idx=P, ni=4,
        tiles=P, nt=1, stream=None), **o}[k]
        for k in "rows di do r ad bf16 x ldx a lda b s base ldb out ldo idx ni tiles nt stream".split()])
    assert lora(r=0) == 2 and lora(r=129) == 2 and lora(rows=0) == 2 and lora(ni=5) == 2 and lora(nt=0) == 2
    assert lora(r=3) == 4 and lora(lda=6) == 4 and lora(lda=4) == 4 and lora(bf16=1, lda=12) == 4 and lora(a=P + 4) == 4
    assert lora(x=None) == 1 and lora(s=None) == 1 and lora(tiles=P + 4) == 4 and lora(ldo=7) == 2


class _Stream:
    """Stands in for a CUDA stream: notes what it was made to wait for."""

    def __init__(self):
        self.waits = []

    def wait_stream(self, other):
        self.waits.append(other)


@pytest.fixture
def host_streams(monkeypatch):
    """The tables of a batch on the host, made and rewritten on stand-in
    streams; returns the function that sets the current one."""
    now = [_Stream()]
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now[0])
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    return lambda s: now.__setitem__(0, s)


def _step_table(batch, key, capturing=False, slots=99):
    batch._table("step", key, 0, capturing, slots)
    return batch._tables[("step", 0, key)]


def test_an_update_outside_inference_mode_reaches_tables_made_inside(host_streams):
    a, b = _Stream(), _Stream()
    batch = RequestBatch([1, 1], device="cpu")
    with torch.inference_mode():
        tables = [_step_table(batch, 1), batch._table("conv", 1, 64, False, 9) and batch._tables[("conv", 64, 1)]]
        host_streams(a)
        tables.append(_step_table(batch, 2))
    host_streams(b)
    batch.update(slots=[5, 6], sources=[-1, 6])
    assert tables[0].tensor.tolist() == tables[2].tensor.tolist() == [5, 6, -1, 6]
    assert tables[1].tensor.view(-1, 8)[:, 4:6].tolist() == [[-1, 5], [6, 6]]
    assert all(t.tensor.tolist() == t.host.tolist() and set(t.stream.waits) == {b} for t in tables)
    assert b.waits == [tables[0].stream, tables[0].stream, a]
    with torch.inference_mode():
        batch.update(slots=[7, 8])
    assert tables[2].tensor.tolist() == [7, 8, 7, 8] and _step_table(batch, 2) is tables[2]


def test_a_failed_update_leaves_batch_and_tables_as_they_were(host_streams):
    batch = RequestBatch([1, 1], slots=[3, 4], device="cpu")
    first, second, third = (_step_table(batch, k) for k in (1, 2, 3))
    _step_table(batch, 1, capturing=True)  # a graph holds the first one
    address = first.told

    class Fails:
        def copy_(self, *args, **kw):
            raise RuntimeError("copy")

    kept, third.tensor = third.tensor, Fails()
    with pytest.raises(RuntimeError, match="copy"):
        batch.update(slots=[5, 6])
    assert batch.slots.tolist() == batch.sources.tolist() == [3, 4] and batch.max_slot == 4
    assert first.tensor.tolist() == first.host.tolist() == [3, 4, 3, 4] and kept.tolist() == [3, 4, 3, 4]
    assert _step_table(batch, 1) is first and first.told == address
    for k, old in ((2, second), (3, third)):  # not held by a graph: made anew, with the batch's values
        assert _step_table(batch, k) is not old and _step_table(batch, k).tensor.tolist() == [3, 4, 3, 4]
    batch.update(slots=[5, 6])
    assert all(t.tensor.tolist() == [5, 6, 5, 6] for t in batch._tables.values())


def test_overlapped_kernels_read_carries_through_plain_pointers():
    """A kernel that starts under the one before it must not declare what that
    one writes read-only for its whole life (`const ... __restrict__`): only
    parameters and host tables may be."""
    with open(os.path.join(build.CSRC, "vmscan_cached.cuh")) as f:
        kernels = re.split(r"__global__", f.read())[1:]
    checked = []
    for text in kernels:
        name, params = re.match(r".*?(\w+_kernel)\((.*?)\)\s*\{", text, re.S).groups()
        body = text.split("\n}\n")[0]
        if "launch_next()" in body or "wait_previous()" in body:
            qualified = {p.split()[-1] for p in params.split(",") if "__restrict__" in p}
            assert qualified <= {"chains", "pieces", "A"}, (name, qualified)
            checked.append(name)
    assert checked == ["cached_scan_kernel", "cached_chain_kernel"]


def test_serve_refuses_what_a_later_step_would():
    """Before anything else runs, so that the conv windows cannot move on alone
    (on the host the first operator would raise RuntimeError)."""
    block, batch, x = MambaBlock(d_model=32), RequestBatch([3, 1], device="cpu"), torch.zeros(4, 32)
    good = block.new_cache(2).ssm
    with pytest.raises(RuntimeError, match="CUDA"):
        block.serve(x, block.new_cache(2), batch)
    shifted = torch.zeros(good.numel() + 1)[1:].view(good.shape)
    assert shifted.data_ptr() % 16 != 0 and shifted.is_contiguous()
    for ssm in (good.to(torch.bfloat16), good.double(), good.transpose(1, 2).contiguous().transpose(1, 2),
                torch.zeros(2, 64, 32)[:, :, ::2], good[:1].expand(2, -1, -1), shifted, good[:1]):
        cache = block.new_cache(2)
        cache.ssm = ssm
        with pytest.raises(ValueError, match="MambaBlock.serve"):
            block.serve(x, cache, batch)
    wide = MambaBlock(d_model=1040)  # dt_rank 65
    with pytest.raises(ValueError, match="dt_rank"):
        wide.serve(torch.zeros(4, 1040), wide.new_cache(2), batch)
    with pytest.raises(ValueError, match="rows"):
        block.serve(torch.zeros(1, 32).expand(65535 * 64 + 1, 32), block.new_cache(2), batch)


def test_threads_share_one_table(host_streams, monkeypatch):
    """Two threads that need the same table get one, whose address a graph may
    hold from then on."""
    batch = RequestBatch([1, 1], device="cpu")
    build_table, built = RequestBatch._build, []

    def slow(self, key):
        built.append(key)
        time.sleep(0.3)
        return build_table(self, key)

    monkeypatch.setattr(RequestBatch, "_build", slow)
    told = []
    threads = [threading.Thread(target=lambda: told.append(batch._table("step", 1, 0, False, 9))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert built == [("step", 0, 1)] and told[0] == told[1] == batch._tables[("step", 0, 1)].told


def test_an_update_reaches_a_table_that_another_thread_is_making(host_streams, monkeypatch):
    batch = RequestBatch([1, 1], device="cpu")
    build_table, built, updated = RequestBatch._build, threading.Event(), threading.Event()

    def slow(self, key):
        table = build_table(self, key)
        if not built.is_set():
            built.set()
            updated.wait(0.5)  # an update that does not wait for this table is over by then
        return table

    monkeypatch.setattr(RequestBatch, "_build", slow)
    maker = threading.Thread(target=lambda: batch._table("step", 1, 0, False, 9))
    maker.start()
    assert built.wait(10)
    batch.update(slots=[6, 7])
    updated.set()
    maker.join()
    assert batch._tables[("step", 0, 1)].tensor.tolist() == [6, 7, 6, 7]


def test_the_extension_is_built_anew_for_another_pytorch(monkeypatch):
    from mlx_vision_mamba_b200 import _serving_ext

    monkeypatch.setattr(os.path, "getmtime", lambda path: 0.0)  # the sources' times are another matter
    assert not build._ext_stale()
    assert _serving_ext.built_for == build._ext_tag()
    monkeypatch.setattr(torch, "__version__", "99.1")
    assert build._ext_stale()

"""Serving operators on the GPU against 64-bit references (serving_ref.py,
whose bounds are derived there), at the lengths, slots, strides and sizes where
they can go wrong, and MambaBlock.serve against the oracle's block."""

import pytest
import torch

import serving_ref as ref
from mlx_vision_mamba_b200 import _native
from mlx_vision_mamba_b200 import (
    LoraAdapters,
    MambaBlock,
    RequestBatch,
    ResidualMambaBlock,
    conv1d_silu_cached_cuda,
    lora_add_cuda,
    selective_scan_cached_cuda,
)

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _scan_inputs(rows, dn, slots, dtype=F32, gate=True, seed=0, step=-3.0):
    g = _gen(seed)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return dict(
        x=n(rows, dn).to(dtype), delta=torch.nn.functional.softplus(0.5 * n(rows, dn) + step).to(dtype),
        A=-torch.arange(1, 17, device="cuda") * torch.exp(0.1 * n(dn, 16)), B=n(rows, 16).to(dtype),
        C=n(rows, 16).to(dtype), D=n(dn), state=0.3 * n(slots, dn, 16), z=n(rows, dn).to(dtype) if gate else None)


def _scan_check(name, inp, batch):
    want = ref.scan(batch=batch, **inp)
    run = dict(inp, state=inp["state"].clone())
    y = selective_scan_cached_cuda(batch=batch, **run)
    again = inp["state"].clone()
    y2 = selective_scan_cached_cuda(batch=batch, **dict(inp, state=again))
    assert y.dtype == inp["x"].dtype and torch.equal(y, y2) and torch.equal(run["state"], again), f"{name}: not repeatable"
    ref.check(f"{name} y", y, want[0], want[1])
    ref.check(f"{name} state", run["state"], want[2], want[3])
    return y, run["state"]


def _mixed(lengths, **kw):
    n = len(lengths)
    return RequestBatch(lengths, slots=[n + (i * 7 + 3) % n for i in range(n)] if n % 7 else list(range(n, 2 * n)),
                        sources=[-1 if i % 3 == 0 else i for i in range(n)], **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("dn", [1, 31, 64, 130])
@pytest.mark.parametrize("lengths", [[1], [7], [8, 9, 1, 16], [0, 5, 33, 0, 1], [100]])
def test_scan_prompts(lengths, dn, gate, dtype):
    batch = _mixed(lengths)
    _scan_check(f"scan {lengths} {dn}", _scan_inputs(batch.tokens, dn, 2 * len(lengths), dtype, gate, seed=dn), batch)


@pytest.mark.parametrize("lengths,dn", [([1500], 40), ([2100, 3, 700], 33), ([0, 1200, 1], 260)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_split_prompts(lengths, dn, dtype):
    """Prompts long enough to be scanned in several pieces, from and to the same slot and forked."""
    n = len(lengths)
    for batch in (RequestBatch(lengths), RequestBatch(lengths, slots=list(range(n, 2 * n)), sources=[0] * n)):
        n_pieces, n_first, chains, _, most, _ = batch._build(("scan", 2 * dn))[1]
        assert chains > 0 and n_pieces > n_first and most > 2
        _scan_check(f"scan {lengths} {dn}", _scan_inputs(batch.tokens, dn, 2 * n, dtype, seed=7), batch)


def test_scan_long_memory():
    """Small steps: the state at the end still holds the first rows'."""
    batch = RequestBatch([1800], sources=[-1])
    _scan_check("long memory", _scan_inputs(1800, 64, 1, seed=3, step=-8.0), batch)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dn", [1, 3, 32, 100, 771])
@pytest.mark.parametrize("count", [1, 2, 37])
def test_scan_tokens(count, dn, dtype):
    slots = [count + i if i % 5 != 4 else -1 for i in range(count)]
    sources = [-1 if i % 4 == 3 else i for i in range(count)]
    batch = RequestBatch([1] * count, slots=slots, sources=sources)
    assert batch.single_tokens
    inp = _scan_inputs(count, dn, 2 * count, dtype, gate=dn != 100, seed=count)
    y, _ = _scan_check(f"tokens {count} {dn}", inp, batch)
    for i, s in enumerate(slots):
        if s < 0:
            assert (y[i] == 0).all()
    _scan_check("in place", inp, RequestBatch([1] * count))


def test_scan_single_tokens_equal_one_prompt_row_by_row():
    """A prompt fed whole, in pieces and token by token ends in the same place."""
    rows, dn = 41, 96
    inp = _scan_inputs(rows, dn, 1, seed=5)
    want = ref.scan(batch=RequestBatch([rows], sources=[-1]), **inp)
    state = torch.full_like(inp["state"], float("nan"))  # a fresh prompt reads nothing
    at, ys = 0, []
    for k, length in enumerate([17, 1, 1, 8, 1, 13]):
        part = {n: (t[at:at + length] if n in ("x", "delta", "B", "C", "z") else t) for n, t in inp.items()}
        batch = RequestBatch([length], sources=[-1] if k == 0 else [0])
        ys.append(selective_scan_cached_cuda(batch=batch, **dict(part, state=state)))
        at += length
    ref.check("y", torch.cat(ys), want[0], want[1])
    ref.check("state", state, want[2], want[3])


def test_scan_strided_rows():
    """Column slices of wider rows at odd offsets, rows that repeat (stride 0),
    columns with a stride, and types that have to be cast."""
    rows, dn = 50, 37
    inp = _scan_inputs(rows, dn, 4, seed=11)
    wide = torch.randn(rows, 3 * dn + 5, device="cuda")
    wide[:, 1:1 + dn], wide[:, 2 + dn:2 + 2 * dn] = inp["x"], inp["z"]
    inp["x"], inp["z"] = wide[:, 1:1 + dn], wide[:, 2 + dn:2 + 2 * dn]
    dbc = torch.randn(rows, 35, device="cuda")
    inp["B"] = dbc[:, 3:19]
    inp["C"] = inp["C"][:1].expand(rows, 16)
    inp["delta"] = inp["delta"].t().contiguous().t()
    inp["D"] = inp["D"].double()
    for batch in (RequestBatch([20, 30], sources=[-1, 3], slots=[1, 2]), RequestBatch([1] * 4, slots=[3, 0, 1, 2])):
        cut = {n: (t[:batch.tokens] if n in ("x", "delta", "B", "C", "z") else t) for n, t in inp.items()}
        _scan_check("strided", cut, batch)


def test_rows_behind_the_last_request_and_padding_requests():
    inp = _scan_inputs(20, 40, 6, seed=2)
    nan = torch.full((20, 40), float("nan"), device="cuda")
    x = torch.where(torch.arange(20, device="cuda")[:, None] < 12, inp["x"], nan)  # rows 12..: never read
    batch = RequestBatch([5, 4, 3], slots=[0, -1, 5])
    x[5:9] = float("nan")  # the padding request's rows
    state = inp["state"].clone()
    y = selective_scan_cached_cuda(batch=batch, **dict(inp, x=x, state=state))
    assert (y[12:] == 0).all() and (y[5:9] == 0).all()
    want = ref.scan(batch=batch, **inp)
    ref.check("y", y[:5], want[0][:5], want[1][:5])
    ref.check("state", state, want[2], want[3])  # slots 1..4 bit for bit
    w, b = torch.randn(40, 4, 1, device="cuda"), torch.randn(40, device="cuda")
    cs = torch.randn(6, 3, 40, device="cuda")
    new = cs.clone()
    out = conv1d_silu_cached_cuda(x, w, b, new, batch)
    assert (out[12:] == 0).all() and (out[5:9] == 0).all()
    want = ref.conv(inp["x"], w, b, cs, batch)
    ref.check("conv", out[:5], want[0][:5], want[1][:5])
    ref.check("window", new, want[2], torch.zeros_like(want[2]))


def test_one_request_does_not_reach_another():
    """Non-finite values stay in their own request, and a fresh request does
    not read its slot."""
    lengths = [9, 1, 0, 700, 30]
    inp = _scan_inputs(sum(lengths), 33, 5, seed=4)
    batch = RequestBatch(lengths, sources=[0, -1, 2, 3, 4])
    clean = inp["state"].clone()
    y0 = selective_scan_cached_cuda(batch=batch, **dict(inp, state=clean))
    bad = {k: (v.clone() if v is not None else None) for k, v in inp.items()}
    bad["x"][9] = float("nan")
    bad["x"][12:14] = float("inf")
    bad["state"][1] = float("nan")
    y1 = selective_scan_cached_cuda(batch=batch, **bad)
    same = torch.ones(sum(lengths), dtype=torch.bool, device="cuda")
    same[9:710] = False
    assert torch.equal(y0[same], y1[same])
    assert torch.isnan(y1[9]).all() and not torch.isfinite(y1[12:14]).any()
    for s in (0, 2, 4):
        assert torch.equal(clean[s], bad["state"][s])
    inp["state"][1] = float("nan")
    fresh = inp["state"].clone()
    assert torch.equal(selective_scan_cached_cuda(batch=batch, **dict(inp, state=fresh)), y0)


def test_extreme_steps():
    """Steps of zero keep the state, huge steps clear it."""
    inp = _scan_inputs(6, 32, 2, seed=9)
    inp["delta"][0:2] = 0.0
    inp["delta"][3] = 200.0
    inp["x"][3] = 0.0
    batch = RequestBatch([2, 4])
    y, state = _scan_check("extreme", inp, batch)
    assert torch.equal(state[0], inp["state"][0])


def test_cache_offsets_beyond_32_bits():
    dn = 1024
    slots = 2 ** 31 // (dn * 16) + 6
    state = torch.zeros(slots, dn, 16, device="cuda")
    inp = _scan_inputs(12, dn, 4, seed=6)
    lengths = [7, 1, 4]
    at = [slots - 1, slots - 2, slots - 3]
    for i, s in enumerate(at):
        state[s] = inp["state"][i]
    small = RequestBatch(lengths, slots=[0, 1, 2])
    want = ref.scan(batch=small, **inp)
    y = selective_scan_cached_cuda(batch=RequestBatch(lengths, slots=at), **dict(inp, state=state))
    ref.check("y", y, want[0], want[1])
    ref.check("state", state[at], want[2][:3], want[3][:3])
    want = ref.scan(batch=RequestBatch([1] * 3), **{k: (v[:3] if k in "x delta B C z".split() else v) for k, v in inp.items()})
    for i, s in enumerate(at):
        state[s] = inp["state"][i]
    y = selective_scan_cached_cuda(batch=RequestBatch([1] * 3, slots=at),
                                   **{k: (v[:3] if k in "x delta B C z".split() else v) for k, v in dict(inp, state=state).items()})
    ref.check("token y", y, want[0], want[1])
    ref.check("token state", state[at], want[2][:3], want[3][:3])
    assert state[:4].abs().max() == 0
    del state
    torch.cuda.empty_cache()
    c, k = 4096, 8
    slots = 2 ** 31 // (c * (k - 1)) + 6
    win = torch.zeros(slots, k - 1, c, dtype=BF16, device="cuda")
    x, w, b = torch.randn(9, c, device="cuda").to(BF16), torch.randn(c, k, 1, device="cuda"), torch.randn(c, device="cuda")
    few = torch.randn(2, k - 1, c, device="cuda").to(BF16)
    win[slots - 2:] = few
    y = conv1d_silu_cached_cuda(x, w, b, win, RequestBatch([3, 6], slots=[slots - 2, slots - 1]))
    want = ref.conv(x, w, b, few, RequestBatch([3, 6]))
    ref.check("conv", y, want[0], want[1])
    ref.check("window", win[slots - 2:], want[2], torch.zeros_like(want[2]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("k", [1, 2, 4, 5, 8])
@pytest.mark.parametrize("c", [1, 64, 66, 771])
@pytest.mark.parametrize("lengths", [[1], [1] * 9, [3, 0, 1, 2, 40], [31, 32, 33, 64, 100], [200]])
def test_conv(lengths, c, k, dtype):
    batch = _mixed(lengths)
    g = _gen(c + k)
    x = torch.randn(batch.tokens, c, generator=g, device="cuda").to(dtype)
    w = torch.randn(c, k, 1, generator=g, device="cuda")
    b = torch.randn(c, generator=g, device="cuda")
    state = torch.randn(2 * len(lengths), k - 1, c, generator=g, device="cuda").to(dtype)
    for bt in (batch, RequestBatch(lengths)):  # forked, and in place
        want = ref.conv(x, w, b, state, bt)
        new = state.clone()
        y = conv1d_silu_cached_cuda(x, w, b, new, bt)
        assert y.dtype == dtype
        ref.check(f"conv {lengths} {c} {k}", y, want[0], want[1])
        ref.check("window", new, want[2], torch.zeros_like(want[2]))  # copies: exact


def test_conv_strided_rows():
    x = torch.randn(40, 100, device="cuda")
    w, b = torch.randn(64, 4, 1, device="cuda"), torch.randn(64, device="cuda")
    state = torch.randn(2, 3, 64, device="cuda")
    for off in (0, 4, 5):
        v = x[:, off:off + 64]
        bt = RequestBatch([30, 10])
        want = ref.conv(v, w, b, state, bt)
        new = state.clone()
        ref.check(f"offset {off}", conv1d_silu_cached_cuda(v, w, b, new, bt), want[0], want[1])
        ref.check("window", new, want[2], torch.zeros_like(want[2]))


def _lora_inputs(batch, count, d_in, d_out, rank, dtype, seed=0, rows=None):
    g = _gen(seed)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    rows = batch.tokens if rows is None else rows
    ads = LoraAdapters((n(count, rank, d_in) * d_in ** -0.5).to(dtype), (n(count, d_out, rank) * rank ** -0.5).to(dtype),
                       [0.5 + i for i in range(count)])
    return n(rows, d_out).to(dtype), n(rows, d_in).to(dtype), ads


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d_in,d_out,rank", [(1, 1, 1), (8, 8, 4), (33, 70, 5), (384, 520, 16), (130, 257, 64), (96, 64, 128)])
@pytest.mark.parametrize("lengths", [[1], [1] * 21, [0, 40, 1, 17, 100], [16, 32]])
def test_lora(lengths, d_in, d_out, rank, dtype):
    n = len(lengths)
    batch = RequestBatch(lengths, adapters=[(i * 5 + 2) % 4 - 1 for i in range(n)])
    base, x, ads = _lora_inputs(batch, 3, d_in, d_out, rank, dtype, seed=d_in + n)
    want = ref.lora(base, x, ads, batch)
    y = lora_add_cuda(base, x, ads, batch)
    ref.check(f"lora {lengths} {d_in} {d_out} {rank}", y, want[0], want[1])
    assert torch.equal(y, lora_add_cuda(base, x, ads, batch))
    inside = base.clone()
    assert lora_add_cuda(inside, x, ads, batch, out=inside) is inside and torch.equal(inside, y)


@pytest.mark.parametrize("rank", [5, 16, 24, 64, 100])
@pytest.mark.parametrize("dtype,d_in,d_out", [(F32, 40, 72), (F32, 41, 70), (BF16, 40, 72)])
def test_lora_keeps_what_is_not_finite(rank, dtype, d_in, d_out):
    """NaN (of any pattern) and infinities in a row, or in a factor, reach the
    outputs that the formula sums them into, and no others."""
    batch = RequestBatch([20, 3, 1, 9, 2], adapters=[0, 1, -1, 2, 1])
    base, x, ads = _lora_inputs(batch, 3, d_in, d_out, rank, dtype, seed=rank)
    clean = lora_add_cuda(base, x, ads, batch)
    assert torch.isfinite(clean).all()
    patterns = {F32: [0x7FC00000, 0x7FFFFFFF, 0x7F800001, -1, -0x400000], BF16: [0x7FC0, 0x7FFF, 0x7F81, -1, -0x40]}[dtype]
    bits = torch.int32 if dtype == F32 else torch.int16
    nans = torch.tensor(patterns, device="cuda", dtype=bits).view(dtype)
    assert torch.isnan(nans).all()
    bad = x.clone()
    for i in range(5):
        bad[3 * i, (7 * i) % d_in] = nans[i]
    bad[20, d_in - 1], bad[34, 0] = nans[1], nans[3]
    bad[1, 2], bad[21, 5], bad[30, 1] = float("inf"), float("-inf"), float("inf")
    bad[23] = nans[1]  # the request without an adapter
    y = lora_add_cuda(base, bad, ads, batch)
    nan_rows, inf_rows = [0, 3, 6, 9, 12, 20, 34], [1, 21, 30]
    assert torch.isnan(y[nan_rows]).all() and not torch.isfinite(y[inf_rows]).any()
    others = [i for i in range(35) if i not in nan_rows + inf_rows]
    assert torch.equal(y[others], clean[others])
    for nan in nans:
        ads.a[1, rank - 1, 3] = nan
        y = lora_add_cuda(base, x, ads, batch)
        rows = [20, 21, 22, 33, 34]
        assert torch.isnan(y[rows]).all()
        others = [i for i in range(35) if i not in rows]
        assert torch.equal(y[others], clean[others])
        ads.a[1, rank - 1, 3] = 0.5
        kept = ads.b[0, d_out - 1, rank - 1].clone()
        ads.b[0, d_out - 1, rank - 1] = nan
        y = lora_add_cuda(base, x, ads, batch)
        assert torch.isnan(y[:20, d_out - 1]).all() and torch.equal(y[:20, :d_out - 1], clean[:20, :d_out - 1])
        ads.b[0, d_out - 1, rank - 1] = kept
        weird = base.clone()
        weird[4, 6] = nan
        y = lora_add_cuda(weird, x, ads, batch)
        assert torch.isnan(y[4, 6]) and torch.isfinite(y).sum() == y.numel() - 1


def test_lora_strides_and_rows_behind():
    batch = RequestBatch([5, 20, 1], adapters=[1, -1, 0])
    base, x, ads = _lora_inputs(batch, 2, 40, 30, 8, F32, rows=31)
    wide = torch.randn(31, 100, device="cuda")
    wide[:, 1:41], wide[:, 43:73] = x, base
    want = ref.lora(base, x, ads, batch)
    for xv, bv in ((wide[:, 1:41], wide[:, 43:73]), (x.t().contiguous().t(), base.t().contiguous().t())):
        y = lora_add_cuda(bv, xv, ads, batch)
        ref.check("strided", y, want[0], want[1])
        assert torch.equal(y[26:], base[26:]) and torch.equal(y[5:25], base[5:25])
    padded = RequestBatch([5, 20, 1], slots=[0, 1, -1], adapters=[1, -1, 0])
    assert torch.equal(lora_add_cuda(base, x, ads, padded)[25], base[25])  # a padding request has no adapter
    out = torch.zeros(31, 64, device="cuda")[:, 3:33]
    assert torch.equal(lora_add_cuda(base, x, ads, batch, out=out), out)
    ref.check("out", out, want[0], want[1])
    view = wide[:, 43:73]  # a column slice beside x in the same rows, updated in place
    lora_add_cuda(view, wide[:, 1:41], ads, batch, out=view)
    ref.check("in place", view, want[0], want[1])
    assert torch.equal(wide[:, 1:41], x)


def test_refusals():
    inp = _scan_inputs(4, 32, 2)
    batch = RequestBatch([3, 1])
    run = lambda b=batch, **kw: selective_scan_cached_cuda(batch=b, **dict(inp, **kw))  # noqa: E731
    with pytest.raises(TypeError):
        run(x=inp["x"].half())
    with pytest.raises(ValueError):
        run(b=RequestBatch([3, 2]))  # more rows than x has
    with pytest.raises(ValueError):
        run(b=RequestBatch([3, 1], slots=[0, 2]))  # slot outside the cache
    with pytest.raises(ValueError):
        run(b=RequestBatch([3, 1], sources=[0, 2], slots=[0, 1]))
    with pytest.raises(ValueError):
        run(state=inp["state"].to(BF16))
    with pytest.raises(ValueError):
        run(state=inp["state"].transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(ValueError):
        run(A=inp["A"][:, :8])
    with pytest.raises(ValueError):
        run(B=inp["B"][:3])
    with pytest.raises(RuntimeError):
        run(delta=inp["delta"].cpu())
    with pytest.raises(RuntimeError, match="no gradient"):
        run(x=inp["x"].clone().requires_grad_(True))
    with torch.no_grad():
        run(x=inp["x"].clone().requires_grad_(True), state=inp["state"].clone())
    w, b = torch.randn(32, 4, 1, device="cuda"), torch.randn(32, device="cuda")
    with pytest.raises(ValueError):
        conv1d_silu_cached_cuda(inp["x"], torch.randn(32, 9, 1, device="cuda"), b, torch.zeros(2, 8, 32, device="cuda"), batch)
    with pytest.raises(ValueError):
        conv1d_silu_cached_cuda(inp["x"], w, b, torch.zeros(2, 4, 32, device="cuda"), batch)
    with pytest.raises(ValueError):
        conv1d_silu_cached_cuda(inp["x"].to(BF16), w, b, torch.zeros(2, 3, 32, device="cuda"), batch)
    lb = RequestBatch([3, 1], adapters=[0, 1])
    base, x, ads = _lora_inputs(lb, 2, 24, 16, 4, F32)
    with pytest.raises(ValueError):
        lora_add_cuda(base, x, ads, batch)  # no adapters in the batch
    with pytest.raises(ValueError):
        lora_add_cuda(base, x, ads, RequestBatch([3, 1], adapters=[0, 2]))
    with pytest.raises(TypeError):
        lora_add_cuda(base.to(BF16), x.to(BF16), ads, lb)
    with pytest.raises(ValueError):
        lora_add_cuda(base, x, ads, lb, out=base[:1].expand(4, 16))
    both = torch.randn(4, 30, device="cuda")
    with pytest.raises(ValueError):
        lora_add_cuda(base, both[:, :24], ads, lb, out=both[:, 10:26])
    with pytest.raises(ValueError):
        LoraAdapters(torch.zeros(1, 129, 4, device="cuda"), torch.zeros(1, 4, 129, device="cuda"))


def test_other_streams_and_graphs():
    """The same batch on two streams, captured, replayed with new inputs, and
    replayed after its slots and adapters changed."""
    dn, count = 48, 6
    batch = RequestBatch([1] * count, slots=list(range(count)), adapters=[0] * count)
    base, xl, ads = _lora_inputs(batch, 2, 24, 40, 4, F32, seed=1)
    inp = _scan_inputs(count, dn, 2 * count, seed=8)
    w, b = torch.randn(dn, 4, 1, device="cuda"), torch.randn(dn, device="cuda")
    win = torch.randn(2 * count, 3, dn, device="cuda")

    def step(state, window):
        c = conv1d_silu_cached_cuda(inp["x"], w, b, window, batch)
        return c, selective_scan_cached_cuda(batch=batch, **dict(inp, state=state)), lora_add_cuda(base, xl, ads, batch)

    s0, w0 = inp["state"].clone(), win.clone()
    first = step(s0, w0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s1, w1 = inp["state"].clone(), win.clone()
        second = step(s1, w1)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(first + (s0, w0), second + (s1, w1)):
        assert torch.equal(p, q)

    state, window = inp["state"].clone(), win.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(state, window)
    state.copy_(inp["state"])
    window.copy_(win)
    graph.replay()
    for p, q in zip(first + (s0, w0), captured + (state, window)):
        assert torch.equal(p, q)

    batch.update(slots=[7, -1, 9, 2, 0, 1], sources=[3, 0, -1, 2, 0, 1], adapters=[1, 0, -1, 1, 1, 0])
    state.copy_(inp["state"])
    window.copy_(win)
    graph.replay()
    want = ref.scan(batch=batch, **inp)
    ref.check("y", captured[1], want[0], want[1])
    ref.check("state", state, want[2], want[3])
    want = ref.conv(inp["x"], w, b, win, batch)
    ref.check("conv", captured[0], want[0], want[1])
    ref.check("window", window, want[2], torch.zeros_like(want[2]))
    want = ref.lora(base, xl, ads, batch)
    ref.check("lora", captured[2], want[0], want[1])
    s2, w2 = inp["state"].clone(), win.clone()
    for p, q in zip(step(s2, w2) + (s2, w2), captured + (state, window)):
        assert torch.equal(p, q)


def test_update_is_ordered_and_refused_whole():
    """update waits for other streams' calls and holds back their next ones; a
    slot outside a captured cache, or an adapter outside the captured ones, is
    refused and changes nothing."""
    count, dn = 5, 64
    batch = RequestBatch([1] * count, adapters=[0, 1, 0, 1, 0])
    inp = _scan_inputs(count, dn, 2 * count, seed=12)
    base, xl, ads = _lora_inputs(batch, 2, 24, 40, 4, F32, seed=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for k in range(3):
        slots = [(i + k) % count + (count if k == 2 else 0) for i in range(count)]
        batch.update(slots=slots, sources=[-1 if i == k else s for i, s in enumerate(slots)])
        with torch.cuda.stream(side):
            state = inp["state"].clone()
            y = selective_scan_cached_cuda(batch=batch, **dict(inp, state=state))
        torch.cuda.current_stream().wait_stream(side)
        want = ref.scan(batch=batch, **inp)
        ref.check("y", y, want[0], want[1])
        ref.check("state", state, want[2], want[3])
    lora_add_cuda(base, xl, ads, batch)
    graph = torch.cuda.CUDAGraph()
    state = inp["state"].clone()
    with torch.cuda.graph(graph):
        selective_scan_cached_cuda(batch=batch, **dict(inp, state=state))
        lora_add_cuda(base, xl, ads, batch)
    before = batch.slots.tolist()
    with pytest.raises(ValueError, match="cache"):
        batch.update(slots=[0, 1, 2, 3, 2 * count])
    with pytest.raises(RuntimeError):
        batch.update(adapters=[0, 1, 2, 0, 0])
    assert batch.slots.tolist() == before and batch.adapters.tolist() == [0, 1, 0, 1, 0]
    state.copy_(inp["state"])
    graph.replay()
    want = ref.scan(batch=batch, **inp)
    ref.check("state", state, want[2], want[3])


def test_requests_without_rows():
    """A call that only forks, clears and keeps states."""
    inp = _scan_inputs(0, 40, 6, seed=1)
    batch = RequestBatch([0, 0, 0, 0], slots=[3, 4, -1, 2], sources=[0, -1, 1, 2])
    state = inp["state"].clone()
    y = selective_scan_cached_cuda(batch=batch, **dict(inp, state=state))
    assert y.shape == (0, 40)
    want = inp["state"].clone()
    want[3], want[4] = inp["state"][0], 0
    assert torch.equal(state, want)
    window = torch.randn(6, 3, 40, device="cuda")
    new = window.clone()
    conv1d_silu_cached_cuda(inp["x"], torch.randn(40, 4, 1, device="cuda"), torch.randn(40, device="cuda"), new, batch)
    window[3], window[4] = window[0].clone(), 0
    assert torch.equal(new, window)
    lb = RequestBatch([0, 0], adapters=[0, 1])
    base, x, ads = _lora_inputs(lb, 2, 8, 12, 4, F32, rows=3)
    assert torch.equal(lora_add_cuda(base, x, ads, lb), base)
    block = MambaBlock(d_model=32).cuda()
    cache = block.new_cache(2)
    cache.ssm.normal_()
    kept = cache.ssm[0].clone()
    assert block.serve(torch.empty(0, 32, device="cuda"), cache, RequestBatch([0], slots=[1], sources=[0])).shape == (0, 32)
    assert torch.equal(cache.ssm[1], kept)


def test_capture_needs_an_eager_call():
    inp = _scan_inputs(3, 32, 1)
    batch = RequestBatch([3])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="once"):
        with torch.cuda.graph(graph):
            selective_scan_cached_cuda(batch=batch, **inp)
    torch.cuda.synchronize()


@pytest.mark.parametrize("d_model", [64, 20])
def test_block_serves_what_it_computes(d_model):
    """MambaBlock.serve over prompts and single tokens, against the oracle's
    block on each request's whole sequence in 64 bits (and the oracle in 32
    bits for the reference's own rounding)."""
    from oracle.model_ref import MambaBlockRef
    from parity import assert_parity

    torch.manual_seed(d_model)
    block = MambaBlock(d_model=d_model).cuda()
    res = ResidualMambaBlock(d_model=d_model).cuda()
    oracle = {}
    for dt in (torch.float64, F32):
        oracle[dt] = MambaBlockRef(d_model=d_model)
        oracle[dt].load_state_dict({k: v.cpu() for k, v in block.state_dict().items()})
        oracle[dt].to(dt)
    totals = [40, 7, 90]
    seqs = [torch.randn(t, d_model) for t in totals]
    fed, outs = [0, 0, 0], [[], [], []]
    cache = block.new_cache(4)
    for lengths in ([17, 2, 64], [1, 1, 1], [1, 1, 1], [5, 0, 20], [16, 3, 4]):
        rows = torch.cat([s[f:f + l] for s, f, l in zip(seqs, fed, lengths)]).cuda()
        batch = RequestBatch(lengths, slots=[2, 0, 3], sources=[-1] * 3 if fed == [0, 0, 0] else None)
        y = block.serve(rows, cache, batch).cpu()
        at = 0
        for i, l in enumerate(lengths):
            outs[i].append(y[at:at + l])
            at += l
            fed[i] += l
    assert fed == totals
    with torch.no_grad():
        for i, s in enumerate(seqs):
            exact, ref32 = oracle[torch.float64](s[None].double())[0], oracle[F32](s[None])[0]
            assert_parity(f"serve {d_model} request {i}", torch.cat(outs[i]), exact, ref32)
        rows = torch.randn(30, d_model, device="cuda")
        got = res.serve(rows, res.new_cache(1), RequestBatch([30], sources=[-1]))
        want = res(rows[None])[0]
        assert (got - want).abs().max() <= 1e-5 * want.abs().max()
    assert (cache.ssm[1] == 0).all() and (cache.conv[1] == 0).all()


def test_block_serves_in_a_graph():
    """Single tokens through a captured serve, replayed token after token with
    new rows and then with other slots, equal the eager calls bit for bit."""
    torch.manual_seed(3)
    d, n = 64, 5
    block = MambaBlock(d_model=d).cuda()
    ain = LoraAdapters(torch.randn(2, 4, d, device="cuda") * 0.1, torch.randn(2, 4 * d, 4, device="cuda") * 0.1)
    eager, cache = block.new_cache(8), block.new_cache(8)
    prompts = RequestBatch([9, 4, 0, 30, 1], sources=[-1] * n, adapters=[0, 1, -1, 1, 0])
    rows = torch.randn(44, d, device="cuda")
    for c in (eager, cache):
        block.serve(rows, c, prompts, ain)
    tokens = RequestBatch([1] * n, adapters=[0, 1, -1, 1, 0])
    x = torch.randn(n, d, device="cuda")
    block.serve(x, block.new_cache(8), tokens, ain)  # the eager call before capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block.serve(x, cache, tokens, ain)
    for k in range(4):
        if k == 2:
            tokens.update(slots=[0, 6, 2, -1, 4], sources=[0, 1, 2, -1, 4], adapters=[1, 0, 0, 0, -1])
        if k == 3:
            tokens.update(slots=[0, 6, 2, 3, 4])
        x.copy_(torch.randn(n, d, device="cuda"))
        want = block.serve(x, eager, tokens, ain)
        graph.replay()
        assert torch.equal(out, want) and torch.equal(cache.ssm, eager.ssm) and torch.equal(cache.conv, eager.conv)


def test_a_refused_serve_leaves_the_cache_as_it_was():
    d = 32
    block = MambaBlock(d_model=d).cuda()
    cache = block.new_cache(2)
    batch, plain = RequestBatch([3, 1], adapters=[0, 1]), RequestBatch([3, 1])
    x = torch.randn(4, d, device="cuda")
    block.serve(x, cache, batch)
    conv, ssm = cache.conv.clone(), cache.ssm.clone()

    def adapters(count, d_in, d_out, dtype=F32):
        return LoraAdapters(torch.ones(count, 4, d_in, device="cuda", dtype=dtype),
                            torch.ones(count, d_out, 4, device="cuda", dtype=dtype))

    good = adapters(2, 2 * d, d)
    for out, bt, error in ((adapters(1, 2 * d, d), batch, ValueError), (adapters(2, d, d), batch, ValueError),
                           (adapters(2, 2 * d, d + 1), batch, ValueError), (good, plain, ValueError),
                           (adapters(2, 2 * d, d, BF16), batch, TypeError), (good.a, batch, TypeError)):
        with pytest.raises(error):
            block.serve(x, cache, bt, out_adapters=out)
    other = block.new_cache(2)
    other.conv = cache.conv
    other.ssm = other.ssm[:1]
    with pytest.raises(ValueError):
        block.serve(x, other, batch)
    narrow = MambaBlock(d_model=d, d_state=8).cuda()
    nc = narrow.new_cache(2)
    with pytest.raises(ValueError, match="d_state"):
        narrow.serve(x, nc, batch)
    assert torch.equal(cache.conv, conv) and torch.equal(cache.ssm, ssm) and not nc.conv.any()
    block.serve(x, cache, batch, out_adapters=good)
    assert not torch.equal(cache.conv, conv)


def test_block_serves_adapters():
    """Adapters on in_proj and out_proj are those projections with W + scale B A."""
    torch.manual_seed(1)
    d = 64
    block = MambaBlock(d_model=d).cuda()
    g = _gen(2)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    ain = LoraAdapters(n(2, 8, d) * d ** -0.5, n(2, 4 * d, 8) * 0.1, [1.0, 2.0])
    aout = LoraAdapters(n(2, 4, 2 * d) * d ** -0.5, n(2, d, 4) * 0.1)
    lengths, picks = [20, 1, 33], [1, -1, 0]
    x = n(sum(lengths), d)
    batch = RequestBatch(lengths, sources=[-1] * 3, adapters=picks)
    y = block.serve(x, block.new_cache(3), batch, ain, aout)
    at = 0
    for l, k in zip(lengths, picks):
        merged = MambaBlock(d_model=d).cuda()
        merged.load_state_dict(block.state_dict())
        with torch.no_grad():
            if k >= 0:
                merged.in_proj.weight += ain.scale[k] * (ain.b[k] @ ain.a[k])
                merged.out_proj.weight += aout.scale[k] * (aout.b[k] @ aout.a[k])
            want = merged.serve(x[at:at + l], merged.new_cache(1), RequestBatch([l], sources=[-1]))
        # the two orders of the same products differ by fp32 roundings of sums of at most 256 terms through
        # a block whose gains are of order one
        assert (y[at:at + l] - want).abs().max() <= 2e-5 * want.abs().max()
        at += l


def test_forward_mode_tangents_are_refused():
    """A dual tensor's tangent is not dropped in silence, and nothing is
    written; with forward mode off, as in inference mode, the call runs."""
    import torch.autograd.forward_ad as fwd

    inp = _scan_inputs(4, 32, 2, seed=5)
    batch = RequestBatch([3, 1], adapters=[0, 1])
    base, x, ads = _lora_inputs(batch, 2, 24, 16, 4, F32)
    w, b, win = torch.randn(32, 4, 1, device="cuda"), torch.randn(32, device="cuda"), torch.randn(2, 3, 32, device="cuda")
    state, window = inp["state"].clone(), win.clone()
    block = MambaBlock(d_model=16).cuda()
    cache = block.new_cache(2)
    with torch.no_grad(), fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for name in ("x", "delta", "A", "B", "C", "D", "z", "state"):
            with pytest.raises(RuntimeError, match="forward-mode"):
                selective_scan_cached_cuda(batch=batch, **dict(inp, **{name: dual(inp[name])}))
        for args in ((dual(inp["x"]), w, b, win), (inp["x"], dual(w), b, win), (inp["x"], w, dual(b), win),
                     (inp["x"], w, b, dual(win))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                conv1d_silu_cached_cuda(*args, batch)
        for args in ((dual(base), x), (base, dual(x))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                lora_add_cuda(*args, ads, batch)
        with pytest.raises(RuntimeError, match="forward-mode"):
            lora_add_cuda(base, x, ads, batch, out=dual(torch.empty_like(base)))
        with pytest.raises(RuntimeError):
            block.serve(dual(torch.randn(4, 16, device="cuda")), cache, batch)
        assert torch.equal(inp["state"], state) and torch.equal(win, window) and not cache.conv.any()
        selective_scan_cached_cuda(batch=batch, **inp)
        with torch.inference_mode():
            lora_add_cuda(base, x, ads, batch)


def test_updates_in_place_are_seen_by_autograd():
    """State, window and `out` count as modified in place: a backward pass that
    has saved one of them refuses to use the new values."""
    inp = _scan_inputs(4, 32, 2, seed=6)
    prompts, tokens = RequestBatch([3, 1], adapters=[0, 1]), RequestBatch([1, 1], slots=[1, 0])
    base, x, ads = _lora_inputs(prompts, 2, 24, 16, 4, F32)
    w, b, win = torch.randn(32, 4, 1, device="cuda"), torch.randn(32, device="cuda"), torch.randn(2, 3, 32, device="cuda")
    two = {k: (v[:2] if k in "x delta B C z".split() else v) for k, v in inp.items()}

    def saved(values, call):
        leaf = values.clone().requires_grad_(True)
        kept = leaf * 2
        loss = (kept * kept).sum()  # saves `kept`
        with torch.no_grad():
            call(kept)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()

    saved(inp["state"], lambda s: selective_scan_cached_cuda(batch=prompts, **dict(inp, state=s)))
    saved(inp["state"], lambda s: selective_scan_cached_cuda(batch=tokens, **dict(two, state=s)))
    saved(win, lambda s: conv1d_silu_cached_cuda(inp["x"], w, b, s, prompts))
    saved(base, lambda s: lora_add_cuda(s, x, ads, prompts, out=s))
    saved(base, lambda s: lora_add_cuda(base, x, ads, prompts, out=s))
    kept = x.clone().requires_grad_(True) * 2  # what is only read stays usable
    loss = (kept * kept).sum()
    with torch.no_grad():
        lora_add_cuda(base, kept, ads, prompts)
    loss.backward()
    with torch.inference_mode():  # inference tensors have no version to count
        state, window = inp["state"].clone(), win.clone()
        selective_scan_cached_cuda(batch=prompts, **dict(inp, state=state))
        conv1d_silu_cached_cuda(inp["x"], w, b, window, prompts)
        lora_add_cuda(base, x, ads, prompts, out=torch.empty_like(base))


def test_inference_mode():
    """First calls inside inference mode, updates outside it and inside, also of
    captured graphs."""
    count, dn = 4, 48
    inp = _scan_inputs(count, dn, 2 * count, seed=14)
    base, xl, ads = _lora_inputs(RequestBatch([1] * count, adapters=[0] * count), 2, 24, 40, 4, F32, seed=3)
    w, b, win = torch.randn(dn, 4, 1, device="cuda"), torch.randn(dn, device="cuda"), torch.randn(2 * count, 3, dn, device="cuda")
    batch = RequestBatch([1] * count, adapters=[0, 1, 0, 1])

    def step(state, window):
        return (conv1d_silu_cached_cuda(inp["x"], w, b, window, batch),
                selective_scan_cached_cuda(batch=batch, **dict(inp, state=state)), lora_add_cuda(base, xl, ads, batch))

    with torch.inference_mode():
        step(inp["state"].clone(), win.clone())
        state, window = inp["state"].clone(), win.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step(state, window)
    for inside, kw in ((False, dict(slots=[4, 5, 6, 7], sources=[0, 1, 2, 3])), (True, dict(slots=[3, 2, 1, 0])),
                       (False, dict(adapters=[1, 1, -1, 0]))):
        with torch.inference_mode(inside):
            batch.update(**kw)
        with torch.inference_mode():
            state.copy_(inp["state"])
            window.copy_(win)
            graph.replay()
            s, v = inp["state"].clone(), win.clone()
            eager = step(s, v)
        for p, q in zip(eager + (s, v), captured + (state, window)):
            assert torch.equal(p, q)
        want = ref.scan(batch=batch, **inp)
        ref.check("y", captured[1], want[0], want[1])
        ref.check("state", state, want[2], want[3])
        want = ref.conv(inp["x"], w, b, win, batch)
        ref.check("conv", captured[0], want[0], want[1])
        want = ref.lora(base, xl, ads, batch)
        ref.check("lora", captured[2], want[0], want[1])


@pytest.mark.parametrize("rank", [8, 24, 64, 100])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("d_in,d_out", [(4096, 512), (4095, 510)])
def test_lora_products_do_not_drift(d_in, d_out, rows, rank):
    """Positive factors, so that what each product of 8 inner indices cuts off
    below its accumulator's last place (2 EPS of the sum so far at most, always
    towards zero) adds up.  A chain of two such products loses at most 4 EPS of
    its own sum in each of the two products, whatever d_in and the rank are;
    roundings to nearest average out (1 EPS for what is left of them)."""
    g = _gen(rank)
    u = lambda *s: 0.5 + torch.rand(s, generator=g, device="cuda")  # noqa: E731
    ads = LoraAdapters(u(1, rank, d_in), u(1, d_out, rank))
    x, zero = u(rows, d_in), torch.zeros(rows, d_out, device="cuda")
    y = lora_add_cuda(zero, x, ads, RequestBatch([rows], adapters=[0])).double()
    exact = (x.double() @ ads.a[0].double().t()) @ ads.b[0].double().t()
    drift = ((y - exact) / exact).mean().item()
    assert abs(drift) <= 9 * ref.EPS, drift / ref.EPS


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rank", [8, 24, 64, 100])
@pytest.mark.parametrize("d_in,d_out", [(384, 520), (130, 257)])
def test_lora_rows_do_not_depend_on_the_rows_beside_them(d_in, d_out, rank, dtype):
    batch = RequestBatch([40, 1, 17, 3], adapters=[0, 0, 1, 1])
    base, x, ads = _lora_inputs(batch, 2, d_in, d_out, rank, dtype, seed=rank)
    y = lora_add_cuda(base, x, ads, batch)
    for row, k in ((0, 0), (39, 0), (40, 0), (57, 1), (60, 1)):
        alone = lora_add_cuda(base[row:row + 1], x[row:row + 1], ads, RequestBatch([1], adapters=[k]))
        assert torch.equal(alone[0], y[row]), row


SPLIT = {"few": [400] * 5 + [1] * 12, "three": [700] * 3 + [40] * 20, "ragged": [1 + i * i * 37 % 900 if i % 3 == 0 else 1 for i in range(40)],
         "long": [1200, 100, 0, 50, 600, 300]}


# the launches of a split scan: overlapped or not, chained by a kernel (more than 8 pieces) or by the pieces, first
# launch with the shared memory of three CTAs an SM or not (of 148 SMs)
@pytest.mark.parametrize("name,dn,dtype,overlapped,chained,claims", [
    ("three", 768, F32, True, False, False),
    ("long", 771, F32, True, True, False),
    ("few", 768, BF16, False, False, False),
    ("long", 768, F32, False, True, False),
    ("ragged", 1536, F32, False, False, True),
    ("ragged", 771, BF16, False, True, True),
])
def test_scan_splits_of_large_calls(name, dn, dtype, overlapped, chained, claims):
    """Every way in which a split scan is launched, against the definition, and
    captured: replayed with other rows and states, and after an update."""
    lengths = SPLIT[name]
    n, groups, sms = len(lengths), (dn + 127) // 128, torch.cuda.get_device_properties(0).multi_processor_count
    batch = RequestBatch(lengths, slots=[2 * i + 1 for i in range(n)], sources=[2 * i if i % 4 else -1 for i in range(n)])
    pieces, first, chains, _, most, uneven = batch._build(("scan", 2 * dn + (dtype == BF16)))[1]
    if sms == 148:
        assert chains > 0 and (pieces * groups <= 3 * sms, most > 8) == (overlapped, chained)
        assert (bool(uneven) and first * groups > 3 * sms) == claims
    inp = _scan_inputs(sum(lengths), dn, 2 * n, dtype, seed=n)
    want = ref.scan_together(batch=batch, **inp)
    run = dict(inp, state=inp["state"].clone())
    y = selective_scan_cached_cuda(batch=batch, **run)
    ref.check("y", y, want[0], want[1])
    ref.check("state", run["state"], want[2], want[3])

    graph, held = torch.cuda.CUDAGraph(), {k: v.clone() for k, v in inp.items()}
    with torch.cuda.graph(graph):
        captured = selective_scan_cached_cuda(batch=batch, **held)
    for k in range(3):
        if k == 2:
            batch.update(slots=[2 * i for i in range(n)], sources=[2 * i + 1 if i % 3 else -1 for i in range(n)])
        new = _scan_inputs(sum(lengths), dn, 2 * n, dtype, seed=n + k)
        for t, v in new.items():
            held[t].copy_(v)
        graph.replay()
        eager = dict(new, state=new["state"].clone())
        assert torch.equal(selective_scan_cached_cuda(batch=batch, **eager), captured), k
        assert torch.equal(eager["state"], held["state"]), k
    want = ref.scan_together(batch=batch, **new)
    ref.check("y after an update", captured, want[0], want[1])
    ref.check("state after an update", held["state"], want[2], want[3])


@pytest.mark.parametrize("c,k,dtype,rows", [(1536, 4, F32, 10000), (1536, 8, BF16, 10000), (771, 5, BF16, 5000), (1536, 1, F32, 9600)])
def test_conv_of_large_calls(c, k, dtype, rows):
    """Pieces of 32 rows, which only large calls have."""
    lengths = [0, 31, 33, 1, 2, 500, 64, rows // 2]
    lengths.append(rows - sum(lengths))
    n = len(lengths)
    assert _native.load().vmscan_cached_conv_rows(rows, c) == 32
    g = _gen(c + k)
    x = torch.randn(rows, c, generator=g, device="cuda").to(dtype)
    w, b = torch.randn(c, k, 1, generator=g, device="cuda"), torch.randn(c, generator=g, device="cuda")
    state = torch.randn(2 * n, k - 1, c, generator=g, device="cuda").to(dtype)
    for batch in (_mixed(lengths), RequestBatch(lengths)):
        want = ref.conv(x, w, b, state, batch)
        new = state.clone()
        ref.check("conv", conv1d_silu_cached_cuda(x, w, b, new, batch), want[0], want[1])
        ref.check("window", new, want[2], torch.zeros_like(want[2]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rank", [16, 24, 64, 100])
@pytest.mark.parametrize("rows,d_in,d_out", [(10000, 96, 520), (10000, 99, 515), (4800, 96, 520), (4800, 99, 515)])
def test_lora_of_large_calls(rows, d_in, d_out, rank, dtype):
    """Tiles enough that a warp goes over several column groups (all nine of a
    tile in the larger call), beside base and in place."""
    lengths = [rows // 2, 0, 77, rows // 4, 1]
    lengths.append(rows - sum(lengths))
    batch = RequestBatch(lengths, adapters=[0, 1, 1, 2, -1, 0])
    base, x, ads = _lora_inputs(batch, 3, d_in, d_out, rank, dtype, seed=rank)
    want = ref.lora(base, x, ads, batch)
    y = lora_add_cuda(base, x, ads, batch)
    ref.check("lora", y, want[0], want[1])
    inside = base.clone()
    lora_add_cuda(inside, x, ads, batch, out=inside)
    assert torch.equal(inside, y)
    wide = torch.zeros(rows, d_out + 8, device="cuda", dtype=dtype)[:, 4:4 + d_out]
    lora_add_cuda(base, x, ads, batch, out=wide)
    assert torch.equal(wide, y)


@pytest.mark.parametrize("lengths,dn", [([1500], 40), ([400] * 5 + [1] * 12, 768)])
def test_growing_states_over_split_prompts(lengths, dn):
    """A > 0: a later piece's factor exp(A sum delta) leaves fp32's range while
    the states do not (nothing has come in yet, or the state is tiny)."""
    n = len(lengths)
    batch = RequestBatch(lengths)
    host, (pieces, _, _, _, most, _) = batch._build(("scan", 2 * dn))
    assert (most > 8) == (n == 1)  # chained by a kernel, by the pieces
    inp = _scan_inputs(batch.tokens, dn, n, gate=False, seed=dn)
    inp["A"] = torch.full((dn, 16), 4.0, device="cuda")
    inp["delta"].fill_(2.0)
    x, state = inp["x"], torch.zeros_like(inp["state"])
    end = lengths[0]
    x[:end - 5] = 0.0
    y = selective_scan_cached_cuda(batch=batch, **dict(inp, state=state))
    last = {k: (v[end - 10:end] if k in ("x", "delta", "B", "C") else v) for k, v in inp.items()}
    alone = torch.zeros_like(state[:1])
    want = selective_scan_cached_cuda(batch=RequestBatch([10]), **dict(last, state=alone))
    assert torch.isfinite(want).all() and torch.equal(y[end - 10:end], want) and torch.equal(state[0], alone[0])
    assert (y[:end - 10] == 0).all()

    rec = host[:8 * pieces].view(-1, 8).tolist()
    t0, t1 = next((r[0], r[1]) for r in rec if r[2] == 0 and r[7] == 2)
    inp["A"].fill_(1.0)
    inp["delta"].zero_()
    inp["delta"][t0:t1] = 100.0 / (t1 - t0)
    x.zero_()
    state = torch.full_like(state, 1e-30)
    selective_scan_cached_cuda(batch=batch, **dict(inp, state=state))
    total = inp["delta"][:end, 0].double().sum()
    want = state.new_tensor(1e-30).double() * torch.exp(total)
    # serving_ref's bound of a split request: its sum of L steps, then the rest of the exponent and its exponentials
    assert ((state[0].double() - want) / want).abs().max() <= (10 + (3 + end) * 100) * ref.EPS

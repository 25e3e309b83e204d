"""64-bit references of the serving operators, each with the bound that the
kernels' arithmetic allows (EPS: half an fp32 step, 2^-24 relative).

Scan.  Per step the kernel forms the decay a = 2^(delta log2(e) A) with one
rounding of delta log2(e), one of that constant, one of the product and ex2's
own error (at most 2^-22 = 4 EPS relative): relative error at most
(5 + 3 |delta A|) EPS; a request that is split sums delta over up to L rows
first, whose error of L EPS relative enters the exponent: (5 + (3 + L) |delta
A|) EPS.  The input delta u B takes two roundings and the new state one.  With
H the state of the absolute values, the error E of the state obeys
    E_t <= a (E_{t-1} + c EPS H_{t-1}) + (2 |b_t| + H_t) EPS
which `scan` runs along.  ex2 (with flush to zero) has no values below TINY =
2^-126: a decay is off by up to TINY in absolute terms there, which adds
TINY (1 + H_{t-1}) to E_t, and the output can lose TINY.  The output adds 16 products and the skip term (at
most 18 roundings of partial sums), and the gate's relative error of at most
(10 + 3 |z|) EPS (ex2, the quotient's 2 steps, the products).

Conv: K + 1 roundings of partial sums, SiLU's slope of at most 1.1 and its own
error as the gate's.  Adapters: d_in + 14 and rank + 14 roundings of partial
sums: 12 cover the products of TF32 parts (a part is rounded to 11 bits, so hi +
lo leaves 2^-22 = 4 EPS of each factor, and the product of the two lo parts
that is not formed is another 2^-22), 2 the scale and the sum over the warps.  A bf16 output is off by
another half step, 2^-8 relative.

All bounds carry a factor 1.05 for their second-order terms.
"""

import torch

EPS = 2.0 ** -24
TINY = 2.0 ** -126
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


def _silu(v):
    return v / (1 + torch.exp(-v))


def _begins(lengths):
    out = [0]
    for l in lengths:
        out.append(out[-1] + l)
    return out


def scan(x, delta, A, B, C, D, state, batch, z=None):
    """(y, bound of y, state, bound of state) in 64 bits on x's device."""
    f = lambda t: t.detach().double()  # noqa: E731
    dtype = x.dtype
    x, delta, A, B, C, D, new = f(x), f(delta), f(A), f(B), f(C), f(D), f(state).clone()
    old = f(state)
    y, tol = torch.zeros_like(x), torch.zeros_like(x)
    state_tol = torch.zeros_like(new)
    at = _begins(batch.lengths.tolist())
    for i, (length, slot, source) in enumerate(zip(batch.lengths.tolist(), batch.slots.tolist(), batch.sources.tolist())):
        if slot < 0:
            continue
        h = old[source].clone() if source >= 0 else torch.zeros_like(old[0])
        H, E = h.abs(), torch.zeros_like(h)
        for t in range(at[i], at[i + 1]):
            arg = delta[t][:, None] * A
            a = torch.exp(arg)
            b = (delta[t] * x[t])[:, None] * B[t]
            E = a * (E + (5 + (3 + length) * arg.abs()) * EPS * H) + TINY * (1 + H)
            h, H = a * h + b, a * H + b.abs()
            E = E + (2 * b.abs() + H) * EPS
            y[t] = h @ C[t]
            tol[t] = E @ C[t].abs() + 18 * EPS * (H @ C[t].abs() + (x[t] * D).abs()) + TINY
        new[slot], state_tol[slot] = h, E
    own = tol > 0  # rows of requests with a slot
    y = torch.where(own, y + x * D, y)
    if z is not None:
        g = _silu(f(z))
        tol = tol * g.abs() + (y * g).abs() * (10 + 3 * f(z).abs()) * EPS
        y = y * g
    return y, 1.05 * tol + y.abs() * HALF_STEP[dtype], new, 1.05 * state_tol


def scan_together(x, delta, A, B, C, D, state, batch, z=None):
    """`scan`, a step of all requests at a time (for many rows)."""
    f = lambda t: t.detach().double()  # noqa: E731
    dtype = x.dtype
    x, delta, A, B, C, D, old = f(x), f(delta), f(A), f(B), f(C), f(D), f(state)
    y, tol, new, state_tol = torch.zeros_like(x), torch.zeros_like(x), old.clone(), torch.zeros_like(old)
    lengths, begins = batch.lengths.tolist(), _begins(batch.lengths.tolist())
    order = sorted((i for i in range(batch.count) if batch.slots[i] >= 0), key=lambda i: -lengths[i])
    source, slot = batch.sources[order].tolist(), batch.slots[order].tolist()
    h = torch.stack([old[s] if s >= 0 else torch.zeros_like(old[0]) for s in source])
    H, E = h.abs(), torch.zeros_like(h)
    long = torch.tensor([float(lengths[i]) for i in order], device=x.device)[:, None, None]
    at = torch.tensor([begins[i] for i in order], device=x.device)
    on = len(order)
    for t in range(max(lengths)):
        while lengths[order[on - 1]] <= t:
            on -= 1
        r = at[:on] + t
        arg = delta[r][:, :, None] * A
        a, b = torch.exp(arg), (delta[r] * x[r])[:, :, None] * B[r][:, None, :]
        e = a * (E[:on] + (5 + (3 + long[:on]) * arg.abs()) * EPS * H[:on]) + TINY * (1 + H[:on])
        h[:on], H[:on] = a * h[:on] + b, a * H[:on] + b.abs()
        E[:on] = e + (2 * b.abs() + H[:on]) * EPS
        c = C[r][:, :, None]
        y[r] = (h[:on] @ c)[:, :, 0] + x[r] * D
        tol[r] = (E[:on] @ c.abs())[:, :, 0] + 18 * EPS * ((H[:on] @ c.abs())[:, :, 0] + (x[r] * D).abs()) + TINY
    if z is not None:
        g = _silu(f(z))
        tol = tol * g.abs() + (y * g).abs() * (10 + 3 * f(z).abs()) * EPS
        y = y * g
    new[slot], state_tol[slot] = h, E
    return y, 1.05 * tol + y.abs() * HALF_STEP[dtype], new, 1.05 * state_tol


def conv(x, weight, bias, state, batch):
    f = lambda t: t.detach().double()  # noqa: E731
    dtype = x.dtype
    x, w, bias, old = f(x), f(weight)[:, :, 0], f(bias), f(state)
    k = w.shape[1]
    new, y, tol = old.clone(), torch.zeros_like(x), torch.zeros_like(x)
    at = _begins(batch.lengths.tolist())
    for i, (length, slot, source) in enumerate(zip(batch.lengths.tolist(), batch.slots.tolist(), batch.sources.tolist())):
        if slot < 0:
            continue
        head = old[source] if source >= 0 else torch.zeros_like(old[0])
        seq = torch.cat((head, x[at[i]:at[i + 1]]))
        pre = bias.expand(length, -1).clone()
        mag = pre.abs()
        for j in range(k):
            pre = pre + w[:, j] * seq[j:j + length]
            mag = mag + (w[:, j] * seq[j:j + length]).abs()
        y[at[i]:at[i + 1]] = _silu(pre)
        tol[at[i]:at[i + 1]] = 1.1 * (k + 1) * EPS * mag + _silu(pre).abs() * (10 + 3 * pre.abs()) * EPS
        new[slot] = seq[length:]
    return y, 1.05 * tol + y.abs() * HALF_STEP[dtype], new


def lora(base, x, adapters, batch):
    f = lambda t: t.detach().double()  # noqa: E731
    y, x, a, b, scale = f(base).clone(), f(x), f(adapters.a), f(adapters.b), f(adapters.scale)
    tol = torch.zeros_like(y)
    at = _begins(batch.lengths.tolist())
    for i, k in enumerate(batch.adapters.tolist()):
        if k < 0:
            continue
        r = slice(at[i], at[i + 1])
        low, mag = x[r] @ a[k].t(), x[r].abs() @ a[k].abs().t()
        part = (mag @ b[k].abs().t()) * scale[k].abs()
        tol[r] = ((adapters.d_in + 14) + (adapters.rank + 14)) * EPS * part + 2 * EPS * y[r].abs()
        y[r] = y[r] + scale[k] * (low @ b[k].t())
        tol[r] = tol[r] + y[r].abs() * (EPS + HALF_STEP[base.dtype])
    return y, 1.05 * tol


def check(name, got, want, tol):
    got = got.detach().double()
    assert got.shape == want.shape, (name, tuple(got.shape), tuple(want.shape))
    assert torch.isfinite(got).all(), f"{name}: non-finite values"
    # tol is zero where a value has to be exact
    bad = (got - want).abs() > tol
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} values are off, the worst "
                           f"{((got - want).abs() / tol.clamp(min=1e-300)).max().item():.3g} times its bound")

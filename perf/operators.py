"""The serving operators as measured calls: the selective scan and the causal
conv1d + SiLU over a cache of request states, and low-rank adapters beside a
shared projection.

A case is one call over a batch of requests packed row after row: `style`
"tokens" (every request brings one new token), "prompts" (ragged prompts, an
empty one among them when there are many) or "mixed" (single tokens and
prompts in one call).  Requests read their state from one slot of the cache
and leave it in another (a request forked off a kept prompt), so a pass can be
repeated; prompts alternate between fresh ones (zero state) and continued ones.

With `own` false, `run` is the operators' plain form in elementary torch
operations and 32 bits; with `own` true it calls the framework.
"""

import math
import random

import torch

own = False

F32, BF16 = "float32", "bfloat16"
N_STATE = 16


def listed():
    return [
        # one new token of one request: pure latency (d_inner 768: a block of d_model 384)
        dict(name="scan token", op="scan", style="tokens", requests=1, tokens=1, channels=768, dtype=F32, gate=True),
        # one token for each of a full serving batch
        dict(name="scan tokens 256", op="scan", style="tokens", requests=256, tokens=256, channels=1536, dtype=F32,
             gate=True),
        # a larger batch, odd sizes, 16-bit activations, no gate
        dict(name="scan tokens odd bf16", op="scan", style="tokens", requests=333, tokens=333, channels=771,
             dtype=BF16, gate=False),
        # the tokens of one 224 x 224 image in patches of 16
        dict(name="scan image", op="scan", style="prompts", requests=1, tokens=196, channels=768, dtype=F32,
             gate=True),
        # a serving step that admits prompts beside running requests
        dict(name="scan mixed", op="scan", style="mixed", requests=24, tokens=9001, channels=768, dtype=F32,
             gate=True),
        # one long document
        dict(name="scan long", op="scan", style="prompts", requests=1, tokens=32768, channels=768, dtype=F32,
             gate=True),
        # a prefill of many prompts, 16-bit activations
        dict(name="scan prompts bf16", op="scan", style="prompts", requests=32, tokens=32768, channels=1536,
             dtype=BF16, gate=True),
        # one new token for each request of a batch
        dict(name="conv tokens", op="conv", style="tokens", requests=64, tokens=64, channels=768, dtype=F32, taps=4),
        # the same prefill as above, in front of the scan
        dict(name="conv prompts", op="conv", style="prompts", requests=32, tokens=32768, channels=1536, dtype=F32,
             taps=4),
        # odd channels: rows that no wide load can take
        dict(name="conv mixed odd bf16", op="conv", style="mixed", requests=40, tokens=3001, channels=771, dtype=BF16,
             taps=5),
        # every request of a decode batch with an adapter of its own choice (in_proj of d_model 384)
        dict(name="lora tokens", op="lora", style="tokens", requests=64, tokens=64, d_in=384, d_out=1536, rank=16,
             adapters=32, dtype=F32),
        # prompts of many requests through the same projection
        dict(name="lora prompts", op="lora", style="prompts", requests=16, tokens=16384, d_in=384, d_out=1536,
             rank=16, adapters=8, dtype=F32),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "conv", "lora"])
    style = rng.choice(["tokens", "prompts", "mixed"])
    dtype = rng.choice([F32, BF16])
    if style == "tokens":
        tokens = requests = _log_int(rng, 1, 512)
    else:
        tokens = _log_int(rng, 2, 32768 if op != "lora" else 16384)
        requests = _log_int(rng, 1, max(1, min(64, tokens // 2)))
    case = dict(op=op, style=style, requests=requests, tokens=tokens, dtype=dtype)
    if op == "lora":
        case.update(d_in=_log_int(rng, 8, 768), d_out=_log_int(rng, 8, 1536), rank=_log_int(rng, 1, 64),
                    adapters=_log_int(rng, 1, 32))
        return case
    channels = _log_int(rng, 8, 1536)
    # half of the widths are what a block has (whole 16-byte rows), half any
    case["channels"] = max(8, channels // 8 * 8) if rng.random() < 0.5 else channels
    if op == "scan":
        case["gate"] = rng.random() < 0.75
    else:
        case["taps"] = rng.randint(1, 8)
    return case


# ---------------------------------------------------------------------------
# what a serving program has in hand
# ---------------------------------------------------------------------------
def _requests(case):
    """(lengths, slots, sources, adapters) of the case's requests: plain numbers
    that depend on the case alone."""
    rng = random.Random("%d %d %s" % (case["requests"], case["tokens"], case["style"]))
    n, total, style = case["requests"], case["tokens"], case["style"]
    if style == "tokens":
        lengths = [1] * n
    else:
        single = n // 2 if style == "mixed" else 0
        single = min(single, max(0, total - 1))
        long = n - single
        w = [rng.expovariate(1.0) + 0.05 for _ in range(long)]
        if long > 4:
            w[rng.randrange(long)] = 0.0  # a request that brings nothing this time
        rest = total - single
        cut, acc = [0], 0.0
        for x in w:
            acc += x
            cut.append(int(round(rest * acc / sum(w))))
        lengths = [b - a for a, b in zip(cut, cut[1:])] + [1] * single
        rng.shuffle(lengths)
    # the cache: slots 0 .. n-1 hold kept states, n .. 2n-1 receive the new ones
    kept, taken = list(range(n)), list(range(n, 2 * n))
    rng.shuffle(kept)
    rng.shuffle(taken)
    fresh = style != "tokens"
    sources = [-1 if fresh and i % 2 == 0 and l > 1 else s for i, (s, l) in enumerate(zip(kept, lengths))]
    count = case.get("adapters", 0)
    adapters = [rng.randrange(-1, count) if rng.random() < 0.1 else rng.randrange(count) for _ in range(n)] if count else None
    return lengths, taken, sources, adapters


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])
    lengths, slots, sources, adapters = _requests(case)
    n, t = case["requests"], case["tokens"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=dev) * scale

    def index(values):
        return torch.tensor(values, dtype=torch.int64, device=dev)

    starts = [0]
    for l in lengths:
        starts.append(starts[-1] + l)
    s = dict(op=case["op"], lengths=lengths, slots=slots, sources=sources, adapters=adapters, longest=max(lengths),
             begin=index(starts[:-1]), end=index(starts[1:]), taken=index(slots), source=index(sources),
             some=index([i for i, l in enumerate(lengths) if l]),
             request=torch.repeat_interleave(torch.arange(n, device=dev), index(lengths), output_size=t))
    if case["op"] == "scan":
        c = case["channels"]
        s["x"] = torch.nn.functional.silu(normal(t, c)).to(dtype)
        s["delta"] = torch.nn.functional.softplus(normal(t, c, scale=0.5) - 3.0).to(dtype)
        steps = torch.arange(1, N_STATE + 1, device=dev, dtype=torch.float32)
        s["A"] = -steps * torch.exp(normal(c, N_STATE, scale=0.1))
        rank = 4 * ((c + 127) // 128)
        dbc = normal(t, rank + 2 * N_STATE).to(dtype)  # the x_proj output: dt | B | C
        s["B"], s["C"] = dbc[:, rank:rank + N_STATE], dbc[:, rank + N_STATE:]
        s["D"] = 1.0 + normal(c, scale=0.1)
        s["z"] = normal(t, c).to(dtype) if case["gate"] else None
        s["state"] = normal(2 * n, c, N_STATE, scale=0.3)
    elif case["op"] == "conv":
        c, k = case["channels"], case["taps"]
        s["x"] = normal(t, c).to(dtype)
        s["weight"] = (torch.rand((c, k, 1), generator=g, device=dev) * 2 - 1) / math.sqrt(k)
        s["bias"] = normal(c, scale=0.1)
        s["state"] = normal(2 * n, k - 1, c).to(dtype)
    else:
        s["x"] = normal(t, case["d_in"]).to(dtype)
        s["base"] = normal(t, case["d_out"]).to(dtype)
        s["a"] = normal(case["adapters"], case["rank"], case["d_in"], scale=case["d_in"] ** -0.5).to(dtype)
        s["b"] = normal(case["adapters"], case["d_out"], case["rank"], scale=case["rank"] ** -0.5).to(dtype)
        s["scale"] = [0.5 + 0.25 * (i % 5) for i in range(case["adapters"])]
        s["factor"] = torch.tensor(s["scale"], device=dev)
        s["adapter"] = index(adapters)
    if own:
        from mlx_vision_mamba_b200 import LoraAdapters, RequestBatch

        s["batch"] = RequestBatch(lengths, slots=slots, sources=sources, adapters=adapters, device=dev)
        if case["op"] == "lora":
            s["lora"] = LoraAdapters(s["a"], s["b"], s["scale"])
    return s


def run(state):
    if own:
        return _own(state)
    return {"scan": _plain_scan, "conv": _plain_conv, "lora": _plain_lora}[state["op"]](state)


def _own(s):
    from mlx_vision_mamba_b200 import conv1d_silu_cached_cuda, lora_add_cuda, selective_scan_cached_cuda

    if s["op"] == "scan":
        y = selective_scan_cached_cuda(s["x"], s["delta"], s["A"], s["B"], s["C"], s["D"], s["state"], s["batch"],
                                       z=s["z"])
        return {"y": y, "state": s["state"]}
    if s["op"] == "conv":
        return {"y": conv1d_silu_cached_cuda(s["x"], s["weight"], s["bias"], s["state"], s["batch"]),
                "state": s["state"]}
    return {"y": lora_add_cuda(s["base"], s["x"], s["lora"], s["batch"])}


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _initial(s):
    kept = s["source"] >= 0
    state = s["state"][s["source"].clamp(min=0)].float()
    return torch.where(kept[:, None, None], state, torch.zeros((), device=state.device))


def _plain_scan(s):
    """The recurrence h = a h + b of every (channel, state) as a doubling scan
    over the packed rows; a request's first row takes its start state into b and
    has a = 0, so nothing crosses from one request into the next."""
    u, delta = s["x"].float(), s["delta"].float()
    a = torch.exp(delta[:, :, None] * s["A"])
    b = (delta * u)[:, :, None] * s["B"].float()[:, None, :]
    init = _initial(s)
    first, last = s["begin"][s["some"]], s["end"][s["some"]] - 1
    b[first] += a[first] * init[s["some"]]
    a[first] = 0.0
    reach = 1
    while reach < s["longest"]:
        b = torch.cat((b[:reach], torch.addcmul(b[reach:], a[reach:], b[:-reach])))
        a = torch.cat((a[:reach], a[reach:] * a[:-reach]))
        reach *= 2
    y = (b * s["C"].float()[:, None, :]).sum(-1) + u * s["D"]
    if s["z"] is not None:
        z = s["z"].float()
        y = y * (z * torch.sigmoid(z))
    init[s["some"]] = b[last]
    s["state"][s["taken"]] = init
    return {"y": y.to(s["x"].dtype), "state": s["state"]}


def _plain_conv(s):
    """Every request's window rows in front of its own rows, then the taps as a
    gather over that array."""
    x, k = s["x"], s["weight"].shape[1]
    n, (t, c) = len(s["lengths"]), x.shape
    ar = lambda m: torch.arange(m, device=x.device)  # noqa: E731
    at = ar(t) + (s["request"] + 1) * (k - 1)  # where row t lies
    front = s["begin"][:, None] + ar(n)[:, None] * (k - 1) + ar(k - 1)
    rows = x.new_empty((t + n * (k - 1), c), dtype=torch.float32)
    rows[at] = x.float()
    rows[front] = _initial(s)
    pre = (rows[at[:, None] + ar(k) - (k - 1)] * s["weight"][:, :, 0].t()).sum(1) + s["bias"]
    behind = s["end"][:, None] + (ar(n)[:, None] + 1) * (k - 1) + ar(k - 1) - (k - 1)
    s["state"][s["taken"]] = rows[behind].to(x.dtype)
    return {"y": (pre * torch.sigmoid(pre)).to(x.dtype), "state": s["state"]}


def _plain_lora(s):
    """All adapters' first factors as one product, each row's own columns kept,
    then all second factors as one product."""
    count, rank, d_in = s["a"].shape
    chosen = s["adapter"][s["request"]]
    keep = (chosen[:, None] == torch.arange(count, device=chosen.device)) * s["factor"]
    low = (s["x"].float() @ s["a"].float().reshape(count * rank, d_in).t()).reshape(-1, count, rank)
    low = (low * keep[:, :, None]).reshape(-1, count * rank)
    up = s["b"].float().permute(0, 2, 1).reshape(count * rank, -1)
    return {"y": (s["base"].float() + low @ up).to(s["base"].dtype)}


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    lengths, slots, sources = s["lengths"], s["slots"], s["sources"]
    starts = [sum(lengths[:i]) for i in range(len(lengths))]
    x = s["x"].double()
    if case["op"] == "lora":
        y = s["base"].double()
        for i, l in enumerate(lengths):
            k, at = s["adapters"][i], slice(starts[i], starts[i] + l)
            if k >= 0:
                y[at] += s["scale"][k] * ((x[at] @ s["a"][k].double().t()) @ s["b"][k].double().t())
        return {"y": y}
    state = s["state"].double()
    if case["op"] == "conv":
        w, y = s["weight"].double(), torch.empty_like(x)
        k = w.shape[1]
        news = []
        for i, l in enumerate(lengths):
            head = state[sources[i]] if sources[i] >= 0 else torch.zeros_like(state[0])
            seq = torch.cat((head, x[starts[i]:starts[i] + l]))
            pre = s["bias"].double().expand(l, -1).clone()
            for j in range(k):
                pre += w[:, j, 0] * seq[j:j + l]
            y[starts[i]:starts[i] + l] = pre / (1 + torch.exp(-pre))
            news.append(seq[l:])
        for i, new in enumerate(news):
            state[slots[i]] = new
        return {"y": y, "state": state}
    # one step at a time over all requests that are still running, longest first
    order = sorted(range(len(lengths)), key=lambda i: -lengths[i])
    delta, A, B, C = s["delta"].double(), s["A"].double(), s["B"].double(), s["C"].double()
    h = torch.stack([state[sources[i]] if sources[i] >= 0 else torch.zeros_like(state[0]) for i in order])
    at = torch.tensor([starts[i] for i in order], device=x.device)
    y = torch.empty_like(x)
    running = len(order)
    for step in range(max(lengths)):
        while lengths[order[running - 1]] <= step:
            running -= 1
        r = at[:running] + step
        d = delta[r]
        h[:running] = torch.exp(d[:, :, None] * A) * h[:running] + (d * x[r])[:, :, None] * B[r][:, None, :]
        y[r] = torch.einsum("rcn,rn->rc", h[:running], C[r])
    y += x * s["D"].double()
    if s["z"] is not None:
        z = s["z"].double()
        y *= z / (1 + torch.exp(-z))
    for k, i in enumerate(order):
        state[slots[i]] = h[k]
    return {"y": y, "state": state}


def work(case):
    e = 4 if case["dtype"] == F32 else 2
    t, n = case["tokens"], case["requests"]
    lengths, _, sources, adapters = _requests(case)
    kept = sum(x >= 0 for x in sources)
    if case["op"] == "scan":
        c = case["channels"]
        moved = e * t * (c * (4 if case["gate"] else 3) + 2 * N_STATE) + 4 * c * (N_STATE + 1)
        # per state and step: the exponent's product, exp, the input's product, two for h, two for y
        return {"bytes": moved + 4 * c * N_STATE * (kept + n), "flops": t * c * (7 * N_STATE + 6)}
    if case["op"] == "conv":
        c, k = case["channels"], case["taps"]
        return {"bytes": 2 * e * t * c + 4 * c * (k + 1) + e * c * (k - 1) * (kept + n), "flops": t * c * (2 * k + 5)}
    d_in, d_out, rank = case["d_in"], case["d_out"], case["rank"]
    rows = sum(l for l, a in zip(lengths, adapters) if a >= 0)
    used = len({a for l, a in zip(lengths, adapters) if a >= 0 and l})
    return {"bytes": e * (rows * d_in + 2 * t * d_out + used * rank * (d_in + d_out)),
            "flops": 2 * rows * rank * (d_in + d_out)}

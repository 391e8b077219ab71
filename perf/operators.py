"""What is timed of the event-stream operators: token lookup with its gradient, and the gated recurrence with its gradient.

A case is one pass of a program that reads an event camera event by event: the events of one or several recordings are
tokens (polarity, y, x), a table holds one row of input currents a token, and leaky state vectors integrate them.

kinds   step    one event (token) for each of `streams` carried states, looked up and integrated
        cell    the same for input rows that the program already has, with gates of its own
        embed   rows of the table for `tokens` events
        embed_grad  gradient of the table (and of the events' weights)
        scan    states after every event of `seqs` recordings
        scan_grad   the same, and the gradients for a given gradient of the states
        train   lookup, scan, and both gradients
decay   "time": a = exp(-dt * rate), dt seconds since the stream's previous event, one rate a channel; "gate": a is an input
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SCALE = 0.125
DAVIS = 2 * 346 * 260          # addresses of a 346 x 260 sensor, two polarities


# ------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one event reaches one running stream: latency is all
        dict(name="step-one", kind="step", streams=1, rows=2 * 80 * 80, dim=200, dtype="float32"),
        # a server with thousands of cameras: one step of every stream, gates computed by the program
        dict(name="step-many", kind="cell", streams=4096, dim=256, dtype="bfloat16"),
        # a burst of events from a small region of interest
        dict(name="embed-burst", kind="embed", tokens=500, rows=2 * 80 * 80, dim=100, dtype="float32", weights=False),
        # a second of a busy recording on a whole sensor, weighted events
        dict(name="embed-recording", kind="embed", tokens=1000003, rows=DAVIS, dim=128, dtype="bfloat16", weights=True),
        # one window of events, odd width, weights learned too
        dict(name="embed-grad-window", kind="embed_grad", tokens=30011, rows=2 * 128 * 128, dim=63, dtype="float32", weights=True),
        # two seconds of a busy recording: the largest gradient
        dict(name="embed-grad-recording", kind="embed_grad", tokens=2000000, rows=DAVIS, dim=256, dtype="bfloat16", weights=False),
        # a few short windows at once
        dict(name="scan-short", kind="scan", tokens=1501, seqs=8, dim=200, dtype="float32", decay="time"),
        # recordings of very different lengths in one call, empty ones among them
        dict(name="scan-recordings", kind="scan", tokens=400009, seqs=37, dim=200, dtype="bfloat16", decay="time"),
        # one long recording with a gate for every event and channel
        dict(name="scan-long", kind="scan", tokens=1048573, seqs=1, dim=128, dtype="bfloat16", decay="gate"),
        # training the time constants on recordings of odd width
        dict(name="scan-grad-recordings", kind="scan_grad", tokens=200003, seqs=16, dim=63, dtype="float32", decay="time"),
        # training on one long recording with gates
        dict(name="scan-grad-long", kind="scan_grad", tokens=524287, seqs=1, dim=256, dtype="bfloat16", decay="gate"),
        # the whole training pass of an event encoder, in 32 bits since its gradients are
        dict(name="train-encoder", kind="train", tokens=262144, seqs=4, rows=2 * 128 * 128, dim=128, dtype="float32", decay="time"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "cell", "embed", "embed_grad", "scan", "scan_grad", "train"])
    dtype = rng.choice(sorted(DTYPES))
    dim = _log(rng, 7, 600)
    roi = _log(rng, 16, 200)
    rows = rng.choice([2 * roi * roi, DAVIS])
    case = dict(kind=kind, dim=dim, dtype="float32" if kind == "train" else dtype)
    if kind in ("step", "cell"):
        case["streams"] = _log(rng, 1, 4096 * 256 // dim)
        if kind == "step":
            case["rows"] = rows
        return case
    if kind in ("embed", "embed_grad", "train"):
        case["rows"] = rows
    case["tokens"] = _log(rng, 1, (64 if kind == "scan_grad" else 16 if kind == "train" else 96) * 10**6 // dim)
    if kind in ("embed", "embed_grad"):
        case["weights"] = rng.random() < 0.5
    else:
        case["seqs"] = min(_log(rng, 1, 64), case["tokens"])
        case["decay"] = rng.choice(["time", "gate"])
    return case


# ------------------------------------------------------------------------------------------------------ the inputs
def _events(case, g, dev):
    """Tokens as a camera sends them: most follow a moving edge, some are noise everywhere, one pixel is hot, a few are
    padding (-1, as a batch of windows has it)."""
    n, rows = case["tokens"], case["rows"]
    u = torch.rand(n, generator=g, device=dev)
    kind = torch.rand(n, generator=g, device=dev)
    when = torch.arange(n, device=dev, dtype=torch.float64) / max(n, 1)
    near = ((0.1 + 0.8 * when + 0.03 * torch.randn(n, generator=g, device=dev)) % 1.0 * rows).long()
    tok = torch.where(kind < 0.7, near, (u.double() * rows).long()).clamp_(0, rows - 1)
    tok = torch.where(kind > 0.99, torch.full_like(tok, rows // 3), tok)
    tok = torch.where((kind > 0.97) & (kind < 0.98), torch.full_like(tok, -1), tok)
    return tok.to(torch.int32)


def _offsets(case, seed):
    """Recordings of very different lengths, some empty; [seqs + 1]."""
    g = torch.Generator().manual_seed(seed)
    n, b = case["tokens"], case["seqs"]
    w = torch.rand(b, generator=g, dtype=torch.float64) ** 3 * (torch.rand(b, generator=g) > 0.1)
    if not float(w.sum()) > 0:
        w[0] = 1.0
    off = torch.cat([torch.zeros(1, dtype=torch.float64), torch.cumsum(w / w.sum(), 0)])
    off = (off * n).round().long()
    off[-1] = n
    return off


def _decay(case, n, g, dev, s):
    d = case["dim"]
    if case.get("decay", "time") == "time":
        # 1 us to some 100 us between events; time constants from 1 ms to 1 s
        s["dt"] = -torch.log(1 - torch.rand(n, generator=g, device=dev)) * 2e-5 + 1e-6
        s["rate"] = torch.exp(torch.rand(d, generator=g, device=dev) * math.log(1e3))
    else:
        s["gate"] = torch.sigmoid(2.0 + 1.5 * torch.randn(n, d, generator=g, device=dev)).to(DTYPES[case["dtype"]])


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    kind, d, t = case["kind"], case["dim"], DTYPES[case["dtype"]]
    rnd = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    s = dict(kind=kind)
    if kind in ("step", "cell"):
        n = case["streams"]
        s["state"], s["out"] = rnd(n, d), torch.empty(n, d, device=dev)
        if kind == "step":
            s["table"] = rnd(case["rows"], d).to(t)
            s["tokens"] = torch.randint(0, case["rows"], (n,), generator=g, device=dev, dtype=torch.int32)
            s["weight"] = 0.5 + torch.rand(n, generator=g, device=dev)
            _decay(dict(case, decay="time"), n, g, dev, s)
        else:
            s["x"] = rnd(n, d).to(t)
            _decay(dict(case, decay="gate"), n, g, dev, s)
        return s
    n = case["tokens"]
    if kind in ("embed", "embed_grad", "train"):
        s["rows"] = case["rows"]
        s["tokens"] = _events(case, g, dev)
        s["weight"] = 0.5 + torch.rand(n, generator=g, device=dev) if case.get("weights") else None
        if kind != "embed_grad" or case["weights"]:
            s["table"] = rnd(case["rows"], d).to(t)
    if kind in ("embed_grad", "scan_grad", "train"):
        s["grad"] = rnd(n, d).to(t)
    if kind in ("scan", "scan_grad"):
        s["x"] = rnd(n, d).to(t)
    if kind in ("scan", "scan_grad", "train"):
        s["off"] = _offsets(case, seed).to(dev)
        s["h0"] = rnd(case["seqs"], d)
        _decay(case, n, g, dev, s)
        if kind != "scan":
            s["grad_last"] = rnd(case["seqs"], d)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _embed(table, tokens, weight):
    live = tokens >= 0
    f = torch.where(live, SCALE if weight is None else SCALE * weight, 0.0)
    return (table[tokens.clamp(min=0).long()].float() * f[:, None]).to(table.dtype)


def _embed_grad(grad, tokens, rows, weight, table):
    live = tokens >= 0
    row = tokens.clamp(min=0).long()
    f = torch.where(live, SCALE if weight is None else SCALE * weight, 0.0)
    gt = torch.zeros(rows, grad.shape[1], dtype=torch.float32, device=grad.device)
    gt.index_add_(0, row, grad.float() * f[:, None])
    if weight is None:
        return gt, None
    return gt, (grad.float() * table[row].float()).sum(1) * torch.where(live, SCALE, 0.0)


class _Where:
    """Of every row: its recording, that one's first and last row; and clocks, in 64 bits since they run far."""

    def __init__(self, off, n, dt):
        self.t = torch.arange(n, device=off.device)
        self.seq = torch.searchsorted(off[1:].contiguous(), self.t, right=True)
        self.first, self.last = off[self.seq], off[self.seq + 1] - 1
        self.clock = None if dt is None else torch.cumsum(dt.double(), 0)


def _over(s, at, k, forward):
    """Decay over k steps: of row t since row t - k (forward), or of row t + k since row t."""
    age = (at.clock[k:] - at.clock[:-k]).float()
    inside = (at.t[k:] - k >= at.first[k:]) if forward else (at.t[:-k] + k <= at.last[:-k])
    return torch.exp(-age[:, None] * s["rate"]) * inside[:, None]


def _doubling(s, at, h, a, forward):
    """h_t += a_t h_{t-1} over whole recordings, the reach doubled in every round. `a`: gates, zero at the edges."""
    n, k = h.shape[0], 1
    while k < n:
        late, early = (slice(k, None), slice(None, -k)) if forward else (slice(None, -k), slice(k, None))
        far = _over(s, at, k, forward) if a is None else a[late]
        nxt = h.clone()
        nxt[late] += far * h[early]
        if a is not None:
            more = a.clone()
            more[late] *= a[early]
            edge = (slice(0, k) if forward else slice(-k, None))
            more[edge] = 0
            a = more
        h, k = nxt, 2 * k
    return h


def _scan(s, x, at):
    off, n = s["off"], x.shape[0]
    a = torch.exp(-s["dt"][:, None] * s["rate"]) if "rate" in s else s["gate"].float()
    first = (at.t == at.first)[:, None]
    h = x.float() + torch.where(first, a * s["h0"][at.seq], 0.0)
    h = _doubling(s, at, h, None if "rate" in s else torch.where(first, 0.0, a), True)
    last = torch.where((off[1:] > off[:-1])[:, None], h[(off[1:] - 1).clamp(0, n - 1)], s["h0"])
    return h, last, a


def _scan_grad(s, h, a, at):
    off, n = s["off"], h.shape[0]
    is_first, is_last = (at.t == at.first)[:, None], (at.t == at.last)[:, None]
    g = s["grad"].float() + torch.where(is_last, s["grad_last"][at.seq], 0.0)
    nxt = None
    if "rate" not in s:
        nxt = torch.where(is_last, 0.0, torch.cat([a[1:], a[:1]]))
    g = _doubling(s, at, g, nxt, False)
    before = torch.where(is_first, s["h0"][at.seq], torch.cat([h[:1], h[:-1]]))
    if "rate" in s:
        da = -(s["dt"][:, None] * a * g * before).sum(0, dtype=torch.float64).float()
    else:
        da = (g * before).to(s["gate"].dtype)
    gl = s["grad_last"]
    g0 = torch.where((off[1:] > off[:-1])[:, None], (a * g)[off[:-1].clamp(0, n - 1)], gl)
    return g, da, g0


def _plain(s):
    kind = s["kind"]
    if kind in ("step", "cell"):
        if kind == "step":
            x = s["table"][s["tokens"].long()].float() * (SCALE * s["weight"])[:, None]
            return torch.exp(-s["dt"][:, None] * s["rate"]) * s["state"] + x
        return s["gate"].float() * s["state"] + s["x"].float()
    if kind == "embed":
        return _embed(s["table"], s["tokens"], s["weight"])
    if kind == "embed_grad":
        return _embed_grad(s["grad"], s["tokens"], s["rows"], s["weight"], s.get("table"))
    x = _embed(s["table"], s["tokens"], s["weight"]) if kind == "train" else s["x"]
    at = _Where(s["off"], x.shape[0], s.get("dt"))
    h, last, a = _scan(s, x, at)
    if kind == "scan":
        return h.to(x.dtype), last
    g, da, g0 = _scan_grad(s, h, a, at)
    if kind == "scan_grad":
        return h.to(x.dtype), last, g.to(x.dtype), da, g0
    return h.to(x.dtype), last, _embed_grad(g.to(x.dtype), s["tokens"], s["rows"], None, None)[0], da, g0


def run(s):
    if not own:
        return _plain(s)
    from lens_amd import engine
    kind = s["kind"]
    if kind == "step":
        return engine.event_step(s["state"], s["table"], s["tokens"], weight=s["weight"], scale=SCALE, dt=s["dt"],
                                 rate=s["rate"], out=s["out"])
    if kind == "cell":
        return engine.gated_step(s["state"], s["x"], gate=s["gate"], out=s["out"])
    if kind == "embed":
        return engine.embed_events(s["table"], s["tokens"], weight=s["weight"], scale=SCALE, check=False)
    if kind == "embed_grad":
        return engine.embed_events_grad(s["grad"], s["tokens"], s["rows"], weight=s["weight"], scale=SCALE, table=s.get("table"))
    decay = dict(gate=s.get("gate"), dt=s.get("dt"), rate=s.get("rate"), seq_off=s["off"], h0=s["h0"])
    if kind == "scan":
        return engine.gated_scan(s["x"], **decay)
    x = s["x"] if kind == "scan_grad" else engine.embed_events(s["table"], s["tokens"], scale=SCALE, check=False)
    h, last, marks = engine.gated_scan(x, marks=True, **decay)
    dx, da, g0 = engine.gated_scan_grad(s["grad"], x, marks, grad_last=s["grad_last"], **decay)
    if kind == "scan_grad":
        return h, last, dx, da, g0
    return h, last, engine.embed_events_grad(dx, s["tokens"], s["rows"], scale=SCALE)[0], da, g0


# ------------------------------------------------------------------------------- bytes and operations of one pass
def work(case):
    kind, d = case["kind"], case["dim"]
    e = 2 if case["dtype"] != "float32" else 4
    if kind in ("step", "cell"):
        n = case["streams"]
        extra = min(n, case["rows"]) * d * e + n * 12 + d * 4 if kind == "step" else 2 * n * d * e
        return dict(bytes=2 * n * d * 4 + extra, flops=4 * n * d)
    n = case["tokens"]
    all_ = n * d * e
    gates = n * 4 + d * 4 if case.get("decay") == "time" else all_
    rows = case.get("rows", 0)
    w = 4 * n if case.get("weights") else 0
    if kind == "embed":
        return dict(bytes=all_ + min(n, rows) * d * e + 4 * n + w, flops=n * d)
    if kind == "embed_grad":
        return dict(bytes=all_ + rows * d * 4 + 4 * n + 2 * w + (min(n, rows) * d * e if w else 0), flops=(4 if w else 2) * n * d)
    ends = 2 * case["seqs"] * d * 4
    if kind == "scan":
        return dict(bytes=2 * all_ + gates + ends, flops=3 * n * d)
    # x and gates once, states out, gradient of the states in, gradients of x and gates out
    both = 4 * all_ + 2 * gates + 2 * ends
    if kind == "scan_grad":
        return dict(bytes=both, flops=9 * n * d)
    # the table's rows and tokens in, states out, their gradient in, the gradient of the table out
    return dict(bytes=2 * all_ + min(n, rows) * d * e + rows * d * 4 + 4 * n + 2 * gates + 2 * ends, flops=12 * n * d)


# ----------------------------------------------------------------------------------------- the definition, in 64 bits
def _walk(a, x):
    """h_t = a_t h_{t-1} + x_t from zero, step by step, in blocks of rows side by side that are joined afterwards."""
    n, d = x.shape
    c = max(1, int(math.sqrt(n)))
    m = -(-n // c)
    pad = m * c - n
    if pad:
        a = torch.cat([a, a.new_ones(pad, d)])
        x = torch.cat([x, x.new_zeros(pad, d)])
    a, x = a.view(m, c, d), x.view(m, c, d)
    h = torch.empty_like(x)
    reach = torch.ones(m, d, dtype=x.dtype, device=x.device)
    v = torch.zeros_like(reach)
    for j in range(c):
        v = a[:, j] * v + x[:, j]
        reach = reach * a[:, j]
    start, carry = torch.zeros_like(v), torch.zeros_like(v[0])
    for i in range(m):
        start[i] = carry
        carry = reach[i] * carry + v[i]
    v = start
    for j in range(c):
        v = a[:, j] * v + x[:, j]
        h[:, j] = v
    return h.view(m * c, d)[:n]


def _exact_scan(s, x, backward):
    off = s["off"].tolist()
    n, d = x.shape
    h0 = s["h0"].double()
    a = torch.exp(-s["dt"].double()[:, None] * s["rate"].double()) if "rate" in s else s["gate"].double()
    h, last = torch.zeros(n, d, dtype=torch.float64, device=x.device), h0.clone()
    g, g0, before = torch.zeros_like(h), None, torch.zeros_like(h)
    if backward:
        g0 = s["grad_last"].double().clone()
    for b, (i, j) in enumerate(zip(off[:-1], off[1:])):
        if i == j:
            continue
        xs = x[i:j].double().clone()
        xs[0] += a[i] * h0[b]
        h[i:j] = _walk(a[i:j], xs)
        last[b] = h[j - 1]
        if backward:
            before[i], before[i + 1:j] = h0[b], h[i:j - 1]
            gs = s["grad"][i:j].double().clone()
            gs[-1] += s["grad_last"][b].double()
            behind = torch.cat([a[i + 1:j], torch.zeros_like(a[:1])])
            g[i:j] = _walk(behind.flip(0), gs.flip(0)).flip(0)
            g0[b] = a[i] * g[i]
    if not backward:
        return h, last
    da = g * before
    if "rate" in s:
        da = -(s["dt"].double()[:, None] * a * da).sum(0)
    return h, last, g, da, g0


def _exact_rows(grad, tokens, rows, weight, table):
    gt = torch.zeros(rows, grad.shape[1], dtype=torch.float64, device=grad.device)
    gw = torch.zeros(grad.shape[0], dtype=torch.float64, device=grad.device)
    for i in range(0, grad.shape[0], 1 << 18):
        tok = tokens[i:i + (1 << 18)].long()
        at = (tok >= 0).nonzero()[:, 0]
        part = grad[i:i + (1 << 18)][at].double()
        if weight is not None:
            gw[i + at] = SCALE * (part * table[tok[at]].double()).sum(1)
            part = part * weight[i + at].double()[:, None]
        gt.index_put_((tok[at],), SCALE * part, accumulate=True)
    return gt, (None if weight is None else gw)


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "step":
        x = SCALE * s["weight"].double()[:, None] * s["table"].double()[s["tokens"].long()]
        return torch.exp(-s["dt"].double()[:, None] * s["rate"].double()) * s["state"].double() + x
    if kind == "cell":
        return s["gate"].double() * s["state"].double() + s["x"].double()
    if kind == "embed_grad":
        return _exact_rows(s["grad"], s["tokens"], s["rows"], s["weight"], s.get("table"))
    if kind in ("embed", "train"):
        tok = s["tokens"].long()
        f = SCALE * (1.0 if s["weight"] is None else s["weight"].double()[:, None])
        x = torch.where(tok[:, None] >= 0, f * s["table"].double()[tok.clamp(min=0)], 0.0)
        if kind == "embed":
            return x
        # from the lookup on without a rounding, as the definition has it
        h, last, g, da, g0 = _exact_scan(s, x, True)
        return h, last, _exact_rows(g, s["tokens"], s["rows"], None, None)[0], da, g0
    return _exact_scan(s, s["x"], kind == "scan_grad")

"""The event-stream operators in 64 bits, row by row (numpy), with bounds of what 32-bit arithmetic may lose.

u = 2^-24 is half a step of float32 relative to the value; half_step(t) that of an output type.

Lookup: scale * w and its product with the element round once each, the output once.
Table gradient: a sum of n terms, each fma rounding once, in any order and grouping: (n + 3) u times the sum of magnitudes.
Scan: with S_t = |a_t| S_{t-1} + |x_t| every |h_t| <= S_t.  A step rounds its product and its sum, and a run of rows that is
joined to another rounds the factor and the sum of its pair once a row: 8 u S_t covers these.  A decay a = exp(z), z = -dt rate:
z is rounded (u |z|, relative in a), so is its product with log2 e (u |z|); the exponential is good to 2 u, the polynomial below
1/2 to 2.5 u of what it is there, 1/2 at most.  A run's z is a sum of at most 128 terms, 8 at a time in pairs (3 roundings) and these
one after the other (15): 18 u more of it, shared out over its rows.  So (8 + 20 |z_t|) u S_t.
Results below the normal numbers are rounded to a multiple of 2^-149, not relative to themselves: up to 2^-150 for each of a
row's four roundings; and an exponential below 2^-126 is zero, which is 2^-126 of what it multiplies.
An error made at a row decays as the state does: E_t = |a_t| E_{t-1} + (8 + 20 |z_t|) u S_t + 4 2^-150 + 2^-126 S_{t-1}.
"""
import numpy as np
import torch

U = 2.0 ** -24
TINY, FLUSHED = 2.0 ** -150, 2.0 ** -126


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half of the smallest number of a type: what a result near zero may be off."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def embed(table, tokens, weight, scale):
    tab, tok = f64(table), tokens.cpu().numpy()
    s = float(np.float32(scale))
    w = np.ones(len(tok)) if weight is None else f64(weight)
    ok = (tok >= 0) & (tok < len(tab))
    out = np.zeros((len(tok), table.shape[1]))
    out[ok] = s * w[ok, None] * tab[tok[ok]]
    return out


def embed_grad(grad, tokens, n_rows, weight, scale, table):
    """(grad_table, its bound, grad_weight, its bound)."""
    g, tok = f64(grad), tokens.cpu().numpy()
    s = float(np.float32(scale))
    w = np.ones(len(tok)) if weight is None else f64(weight)
    gt, mag, n = np.zeros((n_rows, g.shape[1])), np.zeros((n_rows, g.shape[1])), np.zeros((n_rows, 1))
    gw, gwm = np.zeros(len(tok)), np.zeros(len(tok))
    tab = f64(table)
    for i, k in enumerate(tok):
        if 0 <= k < n_rows:
            gt[k] += s * w[i] * g[i]
            mag[k] += np.abs(s * w[i] * g[i])
            n[k] += 1
            if tab is not None:
                gw[i], gwm[i] = s * (g[i] @ tab[k]), abs(s) * (np.abs(g[i]) @ np.abs(tab[k]))
    return gt, (n + 3) * U * mag, gw, (g.shape[1] + 3) * U * gwm


def gates(gate, dt, rate):
    return f64(gate) if gate is not None else np.exp(-f64(dt)[:, None] * f64(rate)[None, :])


def step_loss(a):
    """(8 + 20 |z|) u of every row and channel (gates have no z: that of |a| stands above it)."""
    with np.errstate(divide="ignore"):
        z = np.where(a > 0, np.minimum(np.abs(np.log(np.maximum(a, 1e-300))), 700), 0)
    return (8 + 20 * z) * U


def scan(x, a, off, h0):
    """states [T, D] (zero in rows of no sequence), last [S, D], the states before every row, and the bounds of the states."""
    x = f64(x)
    T, D = x.shape
    off = [0, T] if off is None else [int(v) for v in off]
    S = len(off) - 1
    h0 = np.zeros((S, D)) if h0 is None else f64(h0)
    h, before, E, Eb = np.zeros((T, D)), np.zeros((T, D)), np.zeros((T, D)), np.zeros((T, D))
    last, El = h0.copy(), np.zeros((S, D))
    c = step_loss(a)
    for s in range(S):
        v, m, e = h0[s].copy(), np.abs(h0[s]), np.zeros(D)
        for t in range(off[s], off[s + 1]):
            before[t], Eb[t] = v, e
            v = a[t] * v + x[t]
            e = np.abs(a[t]) * e + 4 * TINY + FLUSHED * m
            m = np.abs(a[t]) * m + np.abs(x[t])
            e = e + c[t] * m
            h[t], E[t] = v, e
        if off[s] < off[s + 1]:
            last[s], El[s] = v, e
    return h, last, before, E, El, Eb


def scan_grad(grad_h, grad_last, x, a, dt, off, h0):
    """grad_x, grad_gate (or grad_rate), grad_h0 and their bounds."""
    T, D = x.shape
    h, last, before, E, El, Eb = scan(x, a, off, h0)
    off = [0, T] if off is None else [int(v) for v in off]
    S = len(off) - 1
    d = np.zeros((T, D)) if grad_h is None else f64(grad_h)
    gl = np.zeros((S, D)) if grad_last is None else f64(grad_last)
    g, ga, Eg, Ea, r_all, Er_all = (np.zeros((T, D)) for _ in range(6))
    g0, E0 = gl.copy(), np.zeros((S, D))
    c = step_loss(a)
    for s in range(S):
        r, m, e = gl[s].copy(), np.abs(gl[s]), np.zeros(D)
        for t in range(off[s + 1] - 1, off[s] - 1, -1):
            g[t] = d[t] + r
            m = m + np.abs(d[t])
            Eg[t] = e + 2 * U * m
            ga[t] = g[t] * before[t]
            Ea[t] = Eg[t] * np.abs(before[t]) + Eb[t] * np.abs(g[t]) + Eg[t] * Eb[t] + U * np.abs(ga[t])
            r = a[t] * g[t]
            e = np.abs(a[t]) * Eg[t] + 4 * TINY + FLUSHED * m
            m = np.abs(a[t]) * m
            e = e + c[t] * m
            r_all[t], Er_all[t] = r, e
        if off[s] < off[s + 1]:
            g0[s], E0[s] = r, e
    if dt is None:
        return g, ga, g0, Eg, Ea, E0
    dt = f64(dt)[:, None]
    terms = -dt * r_all * before
    bound = (dt * (Er_all * np.abs(before) + Eb * np.abs(r_all) + Er_all * Eb)).sum(0) + (T + 4) * U * np.abs(terms).sum(0)
    return g, terms.sum(0), g0, Eg, bound, E0


def check(got, want, bound, name=""):
    """|got - want| <= bound + the rounding of got's type, everywhere."""
    t = got.dtype
    got = f64(got)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    with np.errstate(invalid="ignore"):
        room = bound + half_step(t) * (np.abs(want) + bound) + least(t)
        off = np.abs(got - want) - room
    bad = ~(off <= 0)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.size} off, first at {np.argwhere(bad)[0].tolist()}: got {got[bad][0]!r}, want {want[bad][0]!r}, room {np.broadcast_to(room, bad.shape)[bad][0]!r}"


# ---- the same for many rows in short sequences: torch in 64 bits on x's device, all sequences side by side, one row of each at a time
def _walk_rows(off, backward=False):
    """(sequences, their rows) of every step."""
    start, n = off[:-1], off[1:] - off[:-1]
    for j in range(int(n.max())):
        s = (n > j).nonzero()[:, 0]
        yield s, (start[s] + j if not backward else off[1:][s] - 1 - j)


def _gate_rows(gate, dt, rate, t):
    """a of the rows t, and (8 + 20 |z|) u of them as step_loss has it."""
    a = gate[t].double() if gate is not None else torch.exp(-dt[t].double()[:, None] * rate.double())
    z = torch.where(a > 0, a.clamp(min=1e-300).log().abs().clamp(max=700), 0.0)
    return a, (8 + 20 * z) * U


def scan_side_by_side(x, off, h0, gate=None, dt=None, rate=None):
    """What scan returns, off an int64 tensor."""
    T, D = x.shape
    h, before, E, Eb = (torch.zeros(T, D, dtype=torch.float64, device=x.device) for _ in range(4))
    v = h0.double().clone()
    m, e = v.abs(), torch.zeros_like(v)
    for s, t in _walk_rows(off):
        a, c = _gate_rows(gate, dt, rate, t)
        before[t], Eb[t] = v[s], e[s]
        v[s] = a * v[s] + x[t].double()
        e[s] = a.abs() * e[s] + 4 * TINY + FLUSHED * m[s]
        m[s] = a.abs() * m[s] + x[t].double().abs()
        e[s] += c * m[s]
        h[t], E[t] = v[s], e[s]
    return h, v, before, E, e, Eb


def scan_grad_side_by_side(grad_h, grad_last, x, before, Eb, off, gate=None, dt=None, rate=None, sum_terms=None):
    """What scan_grad returns; before, Eb: of scan_side_by_side.  sum_terms: roundings of a sum over all rows (T + 4)."""
    T, D = x.shape
    g, Eg = (torch.zeros(T, D, dtype=torch.float64, device=x.device) for _ in range(2))
    ga, Ea = (torch.zeros_like(g), torch.zeros_like(g)) if gate is not None else (None, None)
    r = grad_last.double().clone()
    m, e = r.abs(), torch.zeros_like(r)
    total, bound, mag = (torch.zeros(D, dtype=torch.float64, device=x.device) for _ in range(3))
    for s, t in _walk_rows(off, True):
        a, c = _gate_rows(gate, dt, rate, t)
        d = grad_h[t].double()
        gt = d + r[s]
        mm = m[s] + d.abs()
        eg = e[s] + 2 * U * mm
        g[t], Eg[t] = gt, eg
        if gate is not None:
            ga[t] = gt * before[t]
            Ea[t] = eg * before[t].abs() + Eb[t] * gt.abs() + eg * Eb[t] + U * (gt * before[t]).abs()
        rr = a * gt
        ee = a.abs() * eg + 4 * TINY + FLUSHED * mm
        mm = a.abs() * mm
        ee = ee + c * mm
        r[s], m[s], e[s] = rr, mm, ee
        if gate is None:
            w = dt[t].double()[:, None]
            total -= (w * rr * before[t]).sum(0)
            mag += (w * rr * before[t]).abs().sum(0)
            bound += (w.abs() * (ee * before[t].abs() + Eb[t] * rr.abs() + ee * Eb[t])).sum(0)
    if gate is not None:
        return g, ga, r, Eg, Ea, e
    return g, total, r, Eg, bound + (T + 4 if sum_terms is None else sum_terms) * U * mag, e


def check_all(got, want, bound, name=""):
    """check, on the tensors' device."""
    room = bound + half_step(got.dtype) * (want.abs() + bound) + least(got.dtype)
    bad = ~((got.double() - want).abs() <= room)
    if bool(bad.any()):
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off, first at {at}: got {float(got[at])!r}, want {float(want[at])!r}, "
                             f"room {float(room[at])!r}")


# Scans that are read twice, (D, T, dtype): by the rule of event_scan.hip (plan_twice below) a thread walks `run` rows in several batches of 8,
# and the lanes of one run lie in two wavefronts.
MANY_BATCHES = [(200, 81957, torch.bfloat16, 16), (100, 163845, torch.float16, 16), (300, 49163, torch.bfloat16, 16), (3, 524297, torch.float16, 16),
                (200, 327683, torch.bfloat16, 64), (3, 4194319, torch.bfloat16, 128)]


def plan_twice(T, D):
    """lanes and runs of a workgroup, rows of a run, and the scratch bytes of a forward scan, as the library chooses them."""
    def shape(threads):
        cg = -(-D // (4 if D >= 4 else 1))
        ny = -(-cg // 64)
        lanes = -(-cg // ny)
        return ny, lanes, min(threads // lanes, 32)

    def whole(n):
        return -(-n // 256) * 256
    ny, lanes, ts = shape(256)
    run = 128
    while run > 8 and T * ny < 1024 * run * ts:
        run //= 2
    tiles, tiles_one = -(-T // (run * ts)), -(-T // (8 * shape(512)[2]))
    words, level = 0, 0
    while (tiles_one - 1) >> (3 * level) > 0:
        words, level = words + (tiles_one >> (3 * level)) * D, level + 1
    two = whole(tiles * D * 8) + whole(tiles * D * 4) + whole(tiles * ts * 2 * D * 4)
    return lanes, ts, run, max(two, 256 + whole(words * 8))


def ragged_offsets(T, seed):
    """Sequences that end at multiples of 8 rows and anywhere, several within 8 rows, some without a row; rows of no sequence at both ends."""
    rng = np.random.default_rng(seed)
    n = rng.choice([0, 1, 2, 3, 5, 8, 8, 16, 16, 24, 40, 61], size=T // 8)
    off = 11 + np.concatenate([[0], np.cumsum(n)])
    # half of the places are moved to a multiple of 8
    off = np.maximum.accumulate(np.where(rng.random(off.size) < 0.5, off // 8 * 8, off))
    off = off[off <= T - 13]
    return torch.from_numpy(np.ascontiguousarray(off))

"""The event-stream operators (token lookup, gated recurrence, their gradients, single steps) on the GPU against the same in
64 bits, row by row; the bounds are derived in event_stream_ref."""
import itertools

import numpy as np
import pytest
import torch

import event_stream_ref as R

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def E():
    from lens_amd import engine
    return engine


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def decays(kind, T, D, dtype, g):
    """gate / dt / rate of a call: short and long memories, exact ones and zeros among the gates."""
    if kind == "time":
        return dict(dt=torch.rand(T, generator=g, device="cuda") ** 3 * 2, rate=torch.exp(rnd(g, D) * 2 - 2))
    a = torch.sigmoid(rnd(g, T, D) * 2 + 2)
    u = torch.rand(T, D, generator=g, device="cuda")
    a = torch.where(u < 0.05, torch.zeros_like(a), torch.where(u > 0.95, torch.ones_like(a), a))
    a = torch.where((u > 0.5) & (u < 0.55), -a, a)
    return dict(gate=a.to(torch.float32 if kind == "gate32" else dtype))


# ---------------------------------------------------------------------------------------------------------- lookup
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (3, 5, 2), (7, 4, 3), (17, 9, 7), (33, 20, 8), (64, 50, 63), (129, 1000, 100), (500, 300, 200),
                                   (70, 40, 257), (40, 30, 2048), (4099, 179920, 16)])
def test_lookup(dtype, T, V, D):
    g = gen(T + D)
    table, w = rnd(g, V, D, dtype=dtype), rnd(g, T)
    tok = torch.randint(-1, V, (T,), generator=g, device="cuda")
    for tokens, weight in ((tok, w), (tok.int(), None)):
        out = E().embed_events(table, tokens, weight=weight, scale=0.3)
        want = R.embed(table, tokens, weight, 0.3)
        R.check(out, want, 3 * R.U * np.abs(want))
        assert not f64_any(out[tokens == -1])


def f64_any(t):
    return bool((t != 0).any()) or bool(torch.isnan(t).any())


def test_lookup_strides_and_out():
    g = gen(1)
    wide = rnd(g, 40, 70, dtype=torch.bfloat16)
    table = wide[:, 3:66]                                              # rows 70 elements apart, at an odd offset
    tok = torch.randint(0, 40, (55,), generator=g, device="cuda")
    buf = torch.full((57, 80), 7.0, device="cuda", dtype=torch.bfloat16)
    out = E().embed_events(table, tok, out=buf[1:56, 5:68])
    R.check(out, R.embed(table, tok, None, 1.0), 0)
    buf[1:56, 5:68] = 7.0
    assert bool((buf == 7.0).all())                                    # nothing beside it was written


def test_lookup_tokens_that_name_no_row():
    g = gen(2)
    table = rnd(g, 10, 8)
    table[0] = float("nan")                                            # padding must not read row 0
    tok = torch.tensor([3, -1, 9, 10, -2, 2**40], device="cuda")
    w = torch.tensor([1.0, float("inf"), 2.0, 1.0, 1.0, float("nan")], device="cuda")
    with pytest.raises(IndexError, match="event 3: token 10"):
        E().embed_events(table, tok, weight=w)
    out = E().embed_events(table, tok, weight=w, check=False)
    R.check(out, R.embed(table, tok, w, 1.0), 3 * R.U * np.abs(R.embed(table, tok, w, 1.0)))
    assert not f64_any(out[[1, 3, 4, 5]])
    with pytest.raises(IndexError, match="event 1"):
        E().embed_events(table, torch.tensor([-1, -7], device="cuda", dtype=torch.int32))
    assert E().embed_events(table, tok[:0]).shape == (0, 8)
    empty = E().embed_events(table[:0], torch.tensor([-1, -1], device="cuda"))
    assert empty.shape == (2, 8) and not f64_any(empty)


# ---------------------------------------------------------------------------------------------- sort, table gradient
@pytest.mark.parametrize("T,V", [(1, 1), (2, 3), (65536, 300), (65537, 300), (63, 511), (64, 512), (65, 513), (4095, 12800), (4096, 100), (4097, 179920), (20000, 7),
                                 (100003, 262144), (300, 2**31 - 700)])
def test_sort_is_stable(T, V):
    g = gen(T)
    tok = torch.randint(-2, V + 1, (T,), generator=g, device="cuda", dtype=torch.int64)
    for tokens in (tok, tok.to(torch.int32)):
        order = E().sort_events(tokens, V)
        keys, index = order >> 32, order & 0xffffffff
        k = torch.where((tokens >= 0) & (tokens < V), tokens.long(), V)
        want, at = torch.sort(k, stable=True)
        assert torch.equal(keys, want) and torch.equal(index, at)


@pytest.mark.parametrize("T,V", [(1, 5000000), (30000, 5000000), (65536, 100000000), (65537, 100000000), (2000, 2147483000)])
def test_sort_of_large_tables_and_few_tokens(T, V):
    """More rows than a digit has, a list of one token, of two, and one that is sorted the other way."""
    g = gen(T + V)
    wide = torch.randint(0, V, (T,), generator=g, device="cuda")
    one = torch.full((T,), V - 1, device="cuda")
    two = torch.where(torch.rand(T, generator=g, device="cuda") < 0.5, one, one - 1)
    assert torch.equal(E().sort_events(one, 0), torch.arange(T, device="cuda"))
    for tok in (wide, one, two, torch.arange(T, device="cuda").flip(0) % V, two.int()):
        want, at = torch.sort(tok.long(), stable=True)
        assert torch.equal(E().sort_events(tok, V), want << 32 | at)


def skewed(T, V, g, dev="cuda"):
    """A tenth of the events at one row, a stretch of rows without any, padding and tokens outside."""
    tok = torch.randint(0, V, (T,), generator=g, device=dev)
    u = torch.rand(T, generator=g, device=dev)
    tok = torch.where(u < 0.1, torch.full_like(tok, V // 2), tok)
    tok = torch.where((tok > V // 4) & (tok < V // 3), torch.zeros_like(tok), tok)
    tok = torch.where((u > 0.4) & (u < 0.45), torch.full_like(tok, -1), tok)
    return torch.where((u > 0.5) & (u < 0.51), torch.full_like(tok, V + 3), tok)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (1, 700, 4), (2, 3, 2), (9, 4, 3), (17, 9, 7), (60, 5, 8), (64, 64, 63), (500, 30, 9), (1300, 50, 100),
                                   (3000, 200, 33), (2000, 3, 130), (400, 5000, 200), (700, 60, 257), (130, 20, 600), (90, 8, 1100), (70, 12, 2048)])
def test_table_gradient(dtype, T, V, D):
    g = gen(T + V + D)
    grad, table, w = rnd(g, T, D, dtype=dtype), rnd(g, V, D, dtype=dtype), rnd(g, T)
    tok = skewed(T, V, g)
    for weight in (w, None):
        gt, gw = E().embed_events_grad(grad, tok, V, weight=weight, scale=0.3, table=table)
        want, bound, want_w, bound_w = R.embed_grad(grad, tok, V, weight, 0.3, table)
        R.check(gt, want, bound, "table")
        if weight is None:
            assert gw is None
        else:
            R.check(gw, want_w, bound_w, "weight")
        again = E().embed_events_grad(grad, tok, V, weight=weight, scale=0.3, table=table, order=E().sort_events(tok, V))
        assert torch.equal(gt, again[0]) and (gw is None or torch.equal(gw, again[1]))


@pytest.mark.parametrize("D", [16, 128, 300])
def test_table_gradient_of_one_row_and_of_none(D):
    """Every event at one row (joined over many workgroups), at the first, the last; and no event at all."""
    g = gen(D)
    T, V = 40000, 6
    grad = torch.randint(-8, 9, (T, D), generator=g, device="cuda").to(torch.bfloat16)      # sums of integers are exact
    want = grad.double().sum(0)
    for row in (0, 3, V - 1):
        gt, _ = E().embed_events_grad(grad, torch.full((T,), row, device="cuda"), V)
        assert torch.equal(gt[row].double(), want)
        gt[row] = 0
        assert not f64_any(gt)
    gt, _ = E().embed_events_grad(grad, torch.full((T,), -1, device="cuda"), V)
    assert not f64_any(gt)
    gt, _ = E().embed_events_grad(grad[:0], torch.zeros((0,), device="cuda", dtype=torch.int32), 1000)
    assert gt.shape == (1000, D) and not f64_any(gt)


def test_table_gradient_strides_nan_padding_and_one_gradient_for_all():
    g = gen(5)
    T, V, D = 300, 40, 63
    tok = skewed(T, V, g)
    wide = rnd(g, T, 70)
    grad = wide[:, 3:66]
    grad[(tok < 0) | (tok >= V)] = float("nan")                          # rows of padding count for nothing
    table = rnd(g, V, 64)[:, :63]
    w = rnd(g, T)
    gt, gw = E().embed_events_grad(grad, tok, V, weight=w, table=table)
    want, bound, want_w, bound_w = R.embed_grad(grad, tok, V, w, 1.0, table)
    R.check(gt, want, bound)
    R.check(gw, want_w, bound_w)
    one = rnd(g, 1, D).expand(T, D)
    gt, _ = E().embed_events_grad(one, tok, V)
    R.check(gt, *R.embed_grad(one, tok, V, None, 1.0, None)[:2])
    grad[5] = float("inf")
    gt, _ = E().embed_events_grad(grad, torch.arange(T, device="cuda") % V, V)
    assert bool(torch.isinf(gt[5]).any() | torch.isnan(gt[5]).any())


# ------------------------------------------------------------------------------------------------------------- scan
OFFSETS = [None, [0, 1], [0, 0, 5, 5, 5, 16, 17, 33, 33], [2, 7, 30, 31, 64, 64, 190], [0, 0, 0], [5, 5]]


def run_scan(x, d, off, h0, grad_h, grad_last):
    seq = None if off is None else torch.tensor(off, device="cuda")
    h, last, marks = E().gated_scan(x, seq_off=seq, h0=h0, marks=True, **d)
    back = E().gated_scan_grad(grad_h, x, marks, seq_off=seq, h0=h0, grad_last=grad_last, **d)
    a = R.gates(d.get("gate"), d.get("dt"), d.get("rate"))
    want = R.scan(x, a, off, h0)
    R.check(h, want[0], want[3], "h")
    R.check(last, want[1], want[4], "last")
    g, da, g0, Eg, Ea, E0 = R.scan_grad(grad_h, grad_last, x, a, d.get("dt"), off, h0)
    R.check(back[0], g, Eg, "grad_x")
    R.check(back[1], da, Ea, "grad_gate or grad_rate")
    if h0 is None:
        assert back[2] is None
    else:
        R.check(back[2], g0, E0, "grad_h0")
    return (h, last, *back)


@pytest.mark.parametrize("kind", ["time", "gate", "gate32"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 2, 3, 4, 5, 63, 64, 200, 259])
def test_scan_lengths(dtype, kind, D):
    for T in (0, 1, 2, 15, 16, 17, 79, 128, 257, 700):
        g = gen(1000 * D + T)
        x, d = rnd(g, T, D, dtype=dtype), decays(kind, T, D, dtype, g)
        run_scan(x, d, None, rnd(g, 1, D), rnd(g, T, D, dtype=dtype), rnd(g, 1, D))


@pytest.mark.parametrize("kind", ["time", "gate"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off", OFFSETS[1:])
def test_scan_sequences(dtype, kind, off):
    for D, T, given in ((4, 200, True), (63, 200, False), (100, 401, True)):
        g = gen(D + len(off))
        x, d = rnd(g, T, D, dtype=dtype), decays(kind, T, D, dtype, g)
        S = len(off) - 1
        run_scan(x, d, off, rnd(g, S, D) if given else None, rnd(g, T, D, dtype=dtype), rnd(g, S, D) if given else None)


def test_scan_many_sequences_of_every_length():
    g = gen(9)
    n = list(range(0, 40)) + [0, 0, 1, 300, 0, 129, 1, 1, 1, 64, 128, 256, 0]
    off = [0] + list(itertools.accumulate(n))
    T, D, S = off[-1] + 5, 70, len(n)
    x, d = rnd(g, T, D), decays("time", T, D, torch.float32, g)
    run_scan(x, d, off, rnd(g, S, D), rnd(g, T, D), rnd(g, S, D))


@pytest.mark.parametrize("launches", ["1", "3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scan_of_16_bit_rows_both_ways(dtype, launches, monkeypatch):
    """16-bit rows with decays go in one pass or, where there are many, are read twice: one shape through both."""
    monkeypatch.setenv("LENS_AMD_SCAN_LAUNCHES", launches)
    for D in (1, 3, 4, 63, 200, 259):
        for T, off in ((0, None), (1, None), (8, [0, 8]), (79, None), (257, [3, 3, 100, 256, 256]), (700, [0, 1, 1, 300, 428, 428, 700]), (4001, None)):
            g = gen(10 * D + T)
            S = 1 if off is None else len(off) - 1
            x, d = rnd(g, T, D, dtype=dtype), decays("time", T, D, dtype, g)
            run_scan(x, d, off, rnd(g, S, D), rnd(g, T, D, dtype=dtype), rnd(g, S, D))


@pytest.mark.parametrize("kind,launches", [("time", "1"), ("time", "3"), ("gate", "1")])
def test_scan_of_many_sequences_and_few_rows(kind, launches, monkeypatch):
    """Thousands of streams of which few had an event, and not the first or last ones."""
    monkeypatch.setenv("LENS_AMD_SCAN_LAUNCHES", launches)
    g = gen(18)
    for S, T, D in ((5000, 150, 7), (300, 40, 200), (70001, 9, 3)):
        at = torch.sort(torch.randint(S // 9, S - S // 9, (T,), generator=g, device="cuda")).values      # the stream of every row
        off = torch.searchsorted(at, torch.arange(S + 1, device="cuda")).tolist()
        x, d = rnd(g, T, D, dtype=torch.bfloat16), decays(kind, T, D, torch.bfloat16, g)
        run_scan(x, d, off, rnd(g, S, D), rnd(g, T, D, dtype=torch.bfloat16), rnd(g, S, D))
        run_scan(x, d, off, None, None, rnd(g, S, D))


def test_scan_of_no_rows():
    h0, last = rnd(gen(15), 3, 70), rnd(gen(16), 3, 70)
    off = torch.zeros(4, dtype=torch.int64, device="cuda")
    x = torch.empty(0, 70, device="cuda")
    for d in (dict(dt=torch.empty(0, device="cuda"), rate=torch.ones(70, device="cuda")), dict(gate=torch.empty(0, 70, device="cuda"))):
        h, end, marks = E().gated_scan(x, seq_off=off, h0=h0, marks=True, **d)
        gx, ga, g0 = E().gated_scan_grad(None, x, marks, seq_off=off, h0=h0, grad_last=last, **d)
        assert h.shape == gx.shape == (0, 70) and torch.equal(end, h0) and torch.equal(g0, last) and not f64_any(ga)


@pytest.mark.parametrize("kind,dtype,launches", [("time", torch.float32, "1"), ("gate", torch.float32, "1"), ("time", torch.bfloat16, "1"),
                                                 ("time", torch.bfloat16, "3"), ("gate", torch.bfloat16, "1")])
def test_scan_of_many_tiles(kind, dtype, launches, monkeypatch):
    """Groups of groups of tiles; more than 256 sequences, most of them of no row, and a long one."""
    monkeypatch.setenv("LENS_AMD_SCAN_LAUNCHES", launches)
    g = gen(17)
    T, D = 70001, 1
    x, d = rnd(g, T, D, dtype=dtype), decays(kind, T, D, dtype, g)
    if kind == "time":
        d["dt"] *= 1e-4
    run_scan(x, d, None, rnd(g, 1, D), rnd(g, T, D, dtype=dtype), rnd(g, 1, D))
    cuts = sorted(torch.randint(0, 30000, (300,), generator=g, device="cuda").tolist()) + [30000] * 100 + [T - 2]
    run_scan(x, d, cuts, rnd(g, len(cuts) - 1, D), rnd(g, T, D, dtype=dtype), None)


@pytest.mark.parametrize("T,D,dtype,kind", [(t, d, y, k) for t, d in ((2017, 4096), (8401, 1001)) for y in (torch.float32, torch.bfloat16)
                                            for k in ("time", "gate", "gate32")] + [(4101, 4096, torch.bfloat16, "time")])
def test_scan_of_many_elements(dtype, kind, T, D):
    """Enough of them for two batches a thread; more than 2^24, where 16-bit rows with decays are read twice."""
    g = gen(T)
    x, d = rnd(g, T, D, dtype=dtype), decays(kind, T, D, dtype, g)
    if kind == "time":
        d["dt"] *= 1e-2
    off = [0, 700, 700, T - 1]
    run_scan(x, d, off, rnd(g, 3, D), rnd(g, T, D, dtype=dtype), rnd(g, 3, D))


def test_scan_without_gradient_of_states_and_expanded_rows():
    g = gen(10)
    T, D = 300, 96
    x, gate = rnd(g, 1, D).expand(T, D), torch.sigmoid(rnd(g, 1, D) + 2).expand(T, D)
    run_scan(x, dict(gate=gate), [0, 100, 300], None, None, rnd(g, 2, D))
    run_scan(x, dict(gate=gate), None, None, rnd(g, 1, D).expand(T, D), None)
    run_scan(x, dict(gate=gate), None, rnd(g, 1, D), None, None)


def test_scan_strides_and_rows_of_no_sequence():
    g = gen(11)
    T, D = 150, 63
    x = rnd(g, T, 70, dtype=torch.bfloat16)[:, 5:68]
    gate = torch.sigmoid(rnd(g, T, 64))[:, :63].to(torch.bfloat16)
    grad = rnd(g, T, 80, dtype=torch.bfloat16)[:, 9:72]
    off = torch.tensor([3, 60, 60, 120], device="cuda")
    run_scan(x, dict(gate=gate), off.tolist(), None, grad, None)
    buf = torch.full((T, 99), 7.0, device="cuda", dtype=torch.bfloat16)
    h, _ = E().gated_scan(x, gate=gate, seq_off=off, out=buf[:, 17:80])
    fresh, _ = E().gated_scan(x, gate=gate, seq_off=off)
    assert torch.equal(h[3:120], fresh[3:120]) and not f64_any(fresh[:3]) and not f64_any(fresh[120:])
    buf[3:120, 17:80] = 7.0
    assert bool((buf == 7.0).all())                                    # the caller's rows of no sequence, and what lies beside


@pytest.mark.parametrize("kind", ["time", "gate"])
def test_scan_keeps_infinities_in_their_sequence(kind):
    """A sequence full of NaN and infinities (and rows of none) leaves every other one as it is without them."""
    g = gen(12)
    T, D = 700, 64
    off = [0, 100, 101, 400, 401, 650]
    x, d = rnd(g, T, D), decays(kind, T, D, torch.float32, g)
    grad, gl, h0 = rnd(g, T, D), rnd(g, 5, D), rnd(g, 5, D)
    seq = torch.tensor(off, device="cuda")

    def both():
        h, last, marks = E().gated_scan(x, seq_off=seq, h0=h0, marks=True, **d)
        gx, ga, g0 = E().gated_scan_grad(grad, x, marks, seq_off=seq, h0=h0, grad_last=gl, **d)
        return [h, gx, ga if kind == "gate" else gx], [last, g0]
    clean = both()
    for s, bad in ((0, float("inf")), (2, float("nan")), (4, float("-inf")), (None, float("nan"))):
        i, j = (650, T) if s is None else (off[s], off[s + 1])
        kept = [t.clone() for t in (x, grad, gl, h0)]
        x[i:j], grad[i:j] = bad, bad
        if s is not None:
            gl[s], h0[s] = bad, bad
        rows, ends = both()
        for got, want in zip(rows, clean[0]):
            assert torch.equal(got[:i], want[:i]) and torch.equal(got[j:650], want[j:650])
        for got, want in zip(ends, clean[1]):
            others = [k for k in range(5) if k != s]
            assert torch.equal(got[others], want[others])
        if s is not None:
            assert not bool(torch.isfinite(rows[0][i:j]).all())
        for t, k in zip((x, grad, gl, h0), kept):
            t.copy_(k)


def test_scan_remembers_over_a_long_recording():
    """Microseconds between events against time constants of seconds: what 1 - a of a rounded a would lose."""
    g = gen(13)
    T, D = 30000, 8
    d = dict(dt=torch.rand(T, generator=g, device="cuda") * 2e-6, rate=torch.logspace(-2, 4, D, device="cuda"))
    run_scan(torch.rand(T, D, generator=g, device="cuda"), d, None, rnd(g, 1, D), rnd(g, T, D), None)


def test_scan_gradients_against_differences():
    """<grad, direction> against the change of sum(weights * h) + sum(weights * last) in 64 bits: exact for x and h0 (linear),
    a central difference for gates and rates (error of the step squared: third derivative, bounded by the values' own size)."""
    g = gen(14)
    T, D, off = 90, 12, [0, 40, 40, 90]
    x, h0, cw, cl = rnd(g, T, D), rnd(g, 3, D), rnd(g, T, D), rnd(g, 3, D)
    for kind in ("time", "gate"):
        d = decays(kind, T, D, torch.float32, g)
        seq = torch.tensor(off, device="cuda")
        marks = E().gated_scan(x, seq_off=seq, h0=h0, marks=True, **d)[2]
        gx, ga, g0 = E().gated_scan_grad(cw, x, marks, seq_off=seq, h0=h0, grad_last=cl, **d)

        def loss(x_, h_, d_):
            h, last, *_ = R.scan(x_, R.gates(d_.get("gate"), d_.get("dt"), d_.get("rate")), off, h_)
            return (h * R.f64(cw)).sum() + (last * R.f64(cl)).sum()
        vx, vh = rnd(g, T, D).double(), rnd(g, 3, D).double()
        size = float(cw.abs().double().sum())
        assert abs(float((gx.double() * vx).sum()) - (loss(x.double() + vx, h0, d) - loss(x, h0, d))) < 1e-5 * size
        assert abs(float((g0.double() * vh).sum()) - (loss(x, h0.double() + vh, d) - loss(x, h0, d))) < 1e-5 * size
        name = "rate" if kind == "time" else "gate"
        va, e = rnd(g, *d[name].shape).double() * d[name].abs().double(), 1e-4
        up = loss(x, h0, {**d, name: d[name].double() + e * va})
        down = loss(x, h0, {**d, name: d[name].double() - e * va})
        want = (up - down) / (2 * e)
        assert abs(float((ga.double() * va).sum()) - want) < 1e-5 * size * max(1.0, abs(want) / size)


# ------------------------------------------------------------------------------------------------------ single steps
@pytest.mark.parametrize("kind", ["time", "gate", "gate32"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,D", [(1, 1), (1, 200), (5, 3), (33, 63), (100, 64), (3, 4096)])
def test_single_steps(dtype, kind, n, D):
    g = gen(n + D)
    state, x, d = rnd(g, n, D), rnd(g, n, D, dtype=dtype), decays(kind, n, D, dtype, g)
    a = R.gates(d.get("gate"), d.get("dt"), d.get("rate"))
    want = a * R.f64(state) + R.f64(x)
    bound = R.step_loss(a) * (np.abs(a * R.f64(state)) + np.abs(R.f64(x)))
    out = torch.empty_like(state)
    assert E().gated_step(state, x, out=out, **d) is out
    R.check(out, want, bound)
    table, w = rnd(g, 30, D, dtype=dtype), rnd(g, n)
    tok = torch.randint(-1, 30, (n,), generator=g, device="cuda")
    rows = R.embed(table, tok, w, 0.3)
    want = a * R.f64(state) + rows
    got = E().event_step(state, table, tok, weight=w, scale=0.3, out=out, check=True, **d)
    R.check(got, want, R.step_loss(a) * (np.abs(a * R.f64(state)) + np.abs(rows)))
    kept = out.clone()
    assert E().event_step(state, table, tok.int(), weight=w, scale=0.3, **d) is state       # in place: the same bits
    assert torch.equal(state, kept)


def test_steps_follow_the_scan():
    """Event by event through event_step, and all at once through lookup and scan."""
    g = gen(20)
    n, T, D, V = 3, 50, 63, 40
    table, rate = rnd(g, V, D), torch.exp(rnd(g, D))
    tok = torch.randint(-1, V, (n, T), generator=g, device="cuda")
    dt = torch.rand(n, T, generator=g, device="cuda")
    state = torch.zeros(n, D, device="cuda")
    for t in range(T):
        E().event_step(state, table, tok[:, t].contiguous(), scale=0.5, dt=dt[:, t].contiguous(), rate=rate)
    x = E().embed_events(table, tok.reshape(-1), scale=0.5)
    off = torch.arange(n + 1, device="cuda") * T
    a = R.gates(None, dt.reshape(-1), rate)
    _, last = E().gated_scan(x, dt=dt.reshape(-1), rate=rate, seq_off=off)
    want = R.scan(x, a, off.tolist(), None)
    R.check(state, want[1], want[4] + 3 * R.U * np.abs(want[1]))
    R.check(last, want[1], want[4])


def test_step_with_a_token_outside():
    g = gen(21)
    state, table = rnd(g, 4, 8), rnd(g, 5, 8)
    tok = torch.tensor([0, 5, -1, 4], device="cuda")
    d = dict(dt=torch.ones(4, device="cuda"), rate=torch.zeros(8, device="cuda"))
    kept = state.clone()
    with pytest.raises(IndexError, match="event 1: token 5"):
        E().event_step(state, table, tok, check=True, **d)
    assert torch.equal(state[1:3], kept[1:3]) and not torch.equal(state[0], kept[0])


# --------------------------------------------------------------------------------- a training pass, streams and graphs
def encoder_pass(table, tok, w, rate, dt, off, h0, grad):
    """Lookup, scan and all gradients, as a training step of an event encoder runs them."""
    V = table.shape[0]
    x = E().embed_events(table, tok, weight=w, scale=0.5, check=False)
    h, last, marks = E().gated_scan(x, dt=dt, rate=rate, seq_off=off, h0=h0, marks=True)
    gx, gr, g0 = E().gated_scan_grad(grad, x, marks, dt=dt, rate=rate, seq_off=off, h0=h0)
    gt, gw = E().embed_events_grad(gx, tok, V, weight=w, scale=0.5, table=table)
    return h, last, gt, gw, gr, g0


def encoder_inputs(seed, T=600, V=50, D=63):
    g = gen(seed)
    off = torch.tensor([0, 250, 250, T - 7], device="cuda")
    return (rnd(g, V, D), skewed(T, V, g).clamp(max=V - 1), rnd(g, T), torch.exp(rnd(g, D)), torch.rand(T, generator=g, device="cuda"), off,
            rnd(g, 3, D), rnd(g, T, D))


def test_encoder_pass():
    table, tok, w, rate, dt, off, h0, grad = args = encoder_inputs(30)
    h, last, gt, gw, gr, g0 = encoder_pass(*args)
    x = R.embed(table, tok, w, 0.5)
    a = R.gates(None, dt, rate)
    x32 = E().embed_events(table, tok, weight=w, scale=0.5)
    want = R.scan(x32, a, off.tolist(), h0)
    R.check(h, want[0], want[3])
    R.check(last, want[1], want[4])
    g, dr, want0, Eg, Er, E0 = R.scan_grad(grad, None, x32, a, dt, off.tolist(), h0)
    R.check(gr, dr, Er)
    R.check(g0, want0, E0)
    # the table's gradient: 32-bit sums of rows that carry the scan's error
    t64 = torch.from_numpy(g)
    want_t, bound, want_w, bound_w = R.embed_grad(t64, tok, table.shape[0], w, 0.5, table)
    slack = R.embed_grad(torch.from_numpy(Eg + R.U * np.abs(g)), tok, table.shape[0], w.abs(), 0.5, table.abs())
    R.check(gt, want_t, bound + slack[0])
    R.check(gw, want_w, bound_w + slack[2])
    for _ in range(2):
        for got, first in zip(encoder_pass(*args), (h, last, gt, gw, gr, g0)):
            assert torch.equal(got, first)


def test_encoder_pass_on_another_stream():
    args = encoder_inputs(31, T=20000)
    want = encoder_pass(*args)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    other = encoder_inputs(32, T=20000)
    want_other = encoder_pass(*other)
    torch.cuda.synchronize()
    for _ in range(3):                                                   # two passes at once, each with buffers of its own
        with torch.cuda.stream(a):
            got = encoder_pass(*args)
        with torch.cuda.stream(b):
            got_other = encoder_pass(*other)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert all(torch.equal(x, y) for x, y in zip(got_other, want_other))


def test_encoder_pass_in_a_graph():
    args = encoder_inputs(33, T=9000)
    state = torch.zeros(4, 63, device="cuda")
    step = dict(dt=torch.full((4,), 0.1, device="cuda"), rate=args[3])
    tok4 = torch.arange(4, device="cuda")
    encoder_pass(*args)
    E().event_step(state, args[0], tok4, **step)
    state.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = encoder_pass(*args)
        E().event_step(state, args[0], tok4, **step)
    expect = torch.zeros(4, 63, device="cuda")
    for k in range(4):
        fresh = encoder_inputs(40 + k, T=9000)
        for mine, theirs in zip(args, fresh):
            mine.copy_(theirs)                                         # other events, other lengths
        args[5][2] = args[5][3] - 100 * k
        want = encoder_pass(*args)
        E().event_step(expect, args[0], tok4, **step)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))
        assert torch.equal(state, expect)


def test_recording_to_states_and_one_by_one():
    """Events as a sensor records them -> tokens -> lookup -> states; and the same events one at a time, state carried."""
    from lens_amd.events import event_tokens, window_events
    rng = np.random.default_rng(3)
    T, H, W, D = 300, 12, 16, 40
    t = np.cumsum(rng.integers(0, 400, T)).astype(np.float64)
    x, y, p = rng.integers(0, W + 2, T), rng.integers(1, H + 1, T), rng.integers(0, 2, T)
    off, _ = window_events(t, 10.0)
    tok, dt = event_tokens(t, x, y, p, H, W)
    g = gen(50)
    table, rate = rnd(g, 2 * H * W, D), torch.exp(rnd(g, D) * 2 + 4)
    rows = E().embed_events(table, tok, scale=0.25)
    seq = torch.from_numpy(off).cuda()
    h, last = E().gated_scan(rows, dt=dt, rate=rate, seq_off=seq)
    a = R.gates(None, dt, rate)
    want = R.scan(rows, a, off.tolist(), None)
    R.check(h, want[0], want[3])
    R.check(last, want[1], want[4])
    assert (tok == -1).any() and len(off) > 4
    state = torch.zeros(1, D, device="cuda")
    for i in range(off[1]):
        E().event_step(state, table, tok[i:i + 1], scale=0.25, dt=dt[i:i + 1], rate=rate)
        R.check(state[0], want[0][i], want[3][i])           # scale 1/4 is exact: the same x


@pytest.mark.parametrize("dtype,kind,launches", [(torch.bfloat16, "time", "1"), (torch.bfloat16, "time", "3"), (torch.bfloat16, "gate", "1"),
                                                 (torch.float16, "gate32", "1")])
def test_scan_in_a_graph(dtype, kind, launches, monkeypatch):
    """Two graphs of different lengths, replayed in turn with eager calls between them."""
    monkeypatch.setenv("LENS_AMD_SCAN_LAUNCHES", launches)
    D, calls = 100, []
    for T, S in ((5003, 3), (801, 700)):
        g = gen(T)
        x, d, grad, h0, last = rnd(g, T, D, dtype=dtype), decays(kind, T, D, dtype, g), rnd(g, T, D, dtype=dtype), rnd(g, S, D), rnd(g, S, D)
        off = torch.sort(torch.randint(0, T, (S + 1,), generator=g, device="cuda")).values

        def run(x=x, d=d, grad=grad, h0=h0, last=last, off=off):
            h, end, marks = E().gated_scan(x, seq_off=off, h0=h0, marks=True, **d)
            return (h, end, *E().gated_scan_grad(grad, x, marks, seq_off=off, h0=h0, grad_last=last, **d))
        run()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            out = run()
        calls.append((run, graph, out, x, grad, off, g))
    for _ in range(4):
        for run, graph, out, x, grad, off, g in calls:
            x.normal_(generator=g)
            grad.normal_(generator=g)
            off.copy_(torch.sort(torch.randint(0, x.shape[0], off.shape, generator=g, device="cuda")).values)
            want = run()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_offsets_past_32_bits():
    """Operands of more than 2^32 bytes and 2^31 elements; what lies at their ends against the same in 64 bits."""
    g = gen(60)
    T, D, tail = 8400011, 256, 700
    x = torch.empty(T, D, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    off = torch.tensor([0, 5, T - tail, T - 3], device="cuda")
    h0, rate = rnd(g, 3, D), torch.exp(rnd(g, D) + 4)
    for d in (dict(dt=torch.rand(T, generator=g, device="cuda") * 1e-2, rate=rate), dict(gate=torch.sigmoid(x))):
        h, last, marks = E().gated_scan(x, seq_off=off, h0=h0, marks=True, **d)
        grad = E().gated_scan_grad(x, x, marks, seq_off=off, h0=h0, **d)
        s = slice(T - tail, T)
        a = R.gates(d["gate"][s], None, None) if "gate" in d else R.gates(None, d["dt"][s], rate)
        want = R.scan(x[s], a, [0, tail - 3], h0[2:])
        R.check(h[s], want[0], want[3])
        R.check(last[2:], want[1], want[4])
        gx, ga, g0, Eg, Ea, E0 = R.scan_grad(x[s], None, x[s], a, d["dt"][s] if "dt" in d else None, [0, tail - 3], h0[2:])
        R.check(grad[0][s], gx, Eg)
        R.check(grad[2][2:], g0, E0)
        if "gate" in d:
            R.check(grad[1][s], ga, Ea)
        del h, marks, grad, d
    at = torch.arange(T - 1, -1, -1, device="cuda")
    rows = E().embed_events(x, at, check=False)                              # a long table, a long output
    assert all(torch.equal(rows[i:i + 1000], x[T - 1000 - i:T - i].flip(0)) for i in (0, T // 2, T - 1000))
    del rows
    n = 65536
    gt, _ = E().embed_events_grad(x, at % n, n)                              # long rows in; events from the last to the first
    exact, mag = torch.zeros(n, D, dtype=torch.float64, device="cuda"), torch.zeros(n, D, dtype=torch.float64, device="cuda")
    for part in x.flip(0).split(n):
        exact[:len(part)] += part.double()
        mag[:len(part)] += part.double().abs()
    R.check(gt, exact.cpu().numpy(), ((T // n + 4) * R.U * mag).cpu().numpy())
    V = T // 2 + 1                                                           # a long gradient of the table
    few = torch.tensor([V - 1, 0, V - 1], device="cuda")
    gt, _ = E().embed_events_grad(x[:3], few, V)
    assert torch.equal(gt[V - 1], x[0].float() + x[2].float()) and torch.equal(gt[0], x[1].float()) and not f64_any(gt[1:V - 1])


# ---------------------------------------------------------------------------------- scans of many rows that are read twice
def guarded(*shape):
    """A float32 buffer of this shape between rows of sevens, and a check that these are still there."""
    buf = torch.full((shape[0] + 4, *shape[1:]), 7.0, device="cuda")
    return buf[2:-2], lambda: bool((buf[:2] == 7.0).all()) and bool((buf[-2:] == 7.0).all())


def scan_both_ways_guarded(x, d, off, h0, grad, grad_last):
    """Forward and backward through the C entry points, `last` and `grad_h0` between guard rows."""
    from lens_amd import _lib
    (T, D), S, dev = x.shape, off.numel() - 1, x.get_device()
    L, size = _lib.lib(), E()._TYPES[x.dtype]
    h, gx, gr = torch.empty_like(x), torch.empty_like(x), torch.empty(D, device="cuda")
    marks = torch.empty(-(-T // L.lens_scan_mark_rows(D)), D, device="cuda")
    last, last_ok = guarded(S, D)
    g0, g0_ok = guarded(S, D)
    need = L.lens_gated_scan_scratch_bytes(T, D, 0)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    E()._call("lens_gated_scan", dev, x.data_ptr(), size, D, None, 0, 0, d["dt"].data_ptr(), d["rate"].data_ptr(), off.data_ptr(), S,
              h0.data_ptr(), T, D, h.data_ptr(), D, 1, last.data_ptr(), marks.data_ptr(), scratch.data_ptr(), need)
    need = L.lens_gated_scan_scratch_bytes(T, D, 1)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    E()._call("lens_gated_scan_grad", dev, grad.data_ptr(), D, grad_last.data_ptr(), x.data_ptr(), size, D, None, 0, 0, d["dt"].data_ptr(),
              d["rate"].data_ptr(), off.data_ptr(), S, h0.data_ptr(), marks.data_ptr(), T, D, gx.data_ptr(), D, None, D, gr.data_ptr(),
              g0.data_ptr(), scratch.data_ptr(), need)
    assert last_ok() and g0_ok(), "rows in front of or behind the last states, or the gradients of the first, were written"
    return h, last, gx, gr, g0


@pytest.mark.parametrize("D,T,dtype,run", R.MANY_BATCHES)
def test_scan_of_several_batches_a_run(D, T, dtype, run, monkeypatch):
    """Runs of several batches whose lanes lie in two wavefronts, sequences that end where batches do and within them, rows of no
    sequence at both ends: every output, and the same bits again."""
    monkeypatch.setenv("LENS_AMD_SCAN_LAUNCHES", "3")
    g = gen(D + T)
    off = R.ragged_offsets(T, D).cuda()
    S = off.numel() - 1
    x, grad, h0, gl = rnd(g, T, D, dtype=dtype), rnd(g, T, D, dtype=dtype), rnd(g, S, D), rnd(g, S, D)
    d = decays("time", T, D, dtype, g)
    first = scan_both_ways_guarded(x, d, off, h0, grad, gl)
    h, last, before, Eh, El, Eb = R.scan_side_by_side(x, off, h0, **d)
    R.check_all(first[0], h, Eh, "h")
    R.check_all(first[1], last, El, "last")
    del h, Eh
    gx, gr, g0, Eg, Er, E0 = R.scan_grad_side_by_side(grad, gl, x, before, Eb, off, **d)
    R.check_all(first[2], gx, Eg, "grad_x")
    R.check_all(first[3], gr, Er, "grad_rate")
    R.check_all(first[4], g0, E0, "grad_h0")
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(scan_both_ways_guarded(x, d, off, h0, grad, gl), first))


@pytest.mark.parametrize("launches", ["1", "3"])
@pytest.mark.parametrize("T,D", [(700, 64), (81957, 200)])
def test_scan_of_16_bit_rows_keeps_infinities_in_their_sequence(T, D, launches, monkeypatch):
    monkeypatch.setenv("LENS_AMD_SCAN_LAUNCHES", launches)
    g = gen(70)
    off = [0, 100, 101, 400, 401, T - 50]
    x, d = rnd(g, T, D, dtype=torch.bfloat16), decays("time", T, D, torch.bfloat16, g)
    grad, gl, h0 = rnd(g, T, D, dtype=torch.bfloat16), rnd(g, 5, D), rnd(g, 5, D)
    seq = torch.tensor(off, device="cuda")

    def both():
        h, last, marks = E().gated_scan(x, seq_off=seq, h0=h0, marks=True, **d)
        gx, _, g0 = E().gated_scan_grad(grad, x, marks, seq_off=seq, h0=h0, grad_last=gl, **d)
        return [h, gx], [last, g0]
    clean = both()
    for s, bad in ((0, float("inf")), (2, float("nan")), (4, float("-inf")), (None, float("nan"))):
        i, j = (T - 50, T) if s is None else (off[s], off[s + 1])
        kept = [t.clone() for t in (x, grad, gl, h0)]
        x[i:j], grad[i:j] = bad, bad
        if s is not None:
            gl[s], h0[s] = bad, bad
        rows, ends = both()
        for got, want in zip(rows, clean[0]):
            assert torch.equal(got[:i], want[:i]) and torch.equal(got[j:T - 50], want[j:T - 50])
        for got, want in zip(ends, clean[1]):
            others = [k for k in range(5) if k != s]
            assert torch.equal(got[others], want[others])
        if s is not None:
            assert not bool(torch.isfinite(rows[0][i:j]).all())
        for t, k in zip((x, grad, gl, h0), kept):
            t.copy_(k)


# ------------------------------------------------------------------------- orders that are not those of the tokens
def cut_tokens(keys, V, place):
    """Tokens among the first `place` places of the merged list, as a wavefront of the table gradient searches for them."""
    lo, hi = 0, min(place, len(keys))
    while lo < hi:
        step = (hi - lo + 63) // 64
        at = lo + (np.arange(64) + 1) * step - 1
        before = (at < hi) & (at + keys[np.minimum(at, hi - 1)] < place)
        lo += int(before.sum()) * step
        hi = min(lo + step - 1, hi)
    return lo


@pytest.mark.parametrize("D,lanes", [(4, 8), (63, 16), (256, 64)])
def test_table_gradient_of_an_order_that_is_not_sorted(D, lanes):
    """Wrong sums, but every access inside the buffers and every loop ended; the next call with its own order is right."""
    from lens_amd import _lib
    g = gen(D)
    T, V = 30000, 5000
    L, per = _lib.lib(), 256 // lanes * 8                                # places a workgroup at this size, 64 a group at most
    tok = torch.randint(0, V, (T,), generator=g, device="cuda")
    good = E().sort_events(tok, V)
    anything = torch.randint(-2**63, 2**63 - 1, (T,), generator=g, device="cuda")
    orders = [good.flip(0), good[torch.randperm(T, generator=g, device="cuda")], anything, anything.sort().values,
              torch.full_like(good, 2**63 - 1), torch.where(torch.arange(T, device="cuda") % 2 == 0, V << 32 | 7, good)]
    grad, table, w = rnd(g, T, D), rnd(g, V, D), rnd(g, T)
    most = 0
    for order in orders:
        keys = (order >> 32).clamp(0, V).cpu().numpy()
        cuts = [cut_tokens(keys, V, p) for p in range(0, T + V + 1, per)]
        most = max(most, int(np.diff(cuts).max()))
        gt, gt_ok = guarded(V, D)
        gw, gw_ok = guarded(T)
        need = L.lens_embed_events_grad_scratch_bytes(0, T, V, D)
        scratch = torch.full((need + 4096,), 7, dtype=torch.uint8, device="cuda")
        E()._call("lens_embed_events_grad", 0, grad.data_ptr(), 0, D, order.data_ptr(), w.data_ptr(), 0.5, T, V, D, table.data_ptr(), D,
                  gt.data_ptr(), gw.data_ptr(), scratch.data_ptr(), need)
        assert gt_ok() and gw_ok() and bool((scratch[need:] == 7).all())
    assert most > per and (lanes == 8 or most > 8 * per)                # more tokens than places, or than the most that a cut may have
    gt, gw = E().embed_events_grad(grad, tok, V, weight=w, scale=0.5, table=table, order=good)
    want, bound, want_w, bound_w = R.embed_grad(grad, tok, V, w, 0.5, table)
    R.check(gt, want, bound, "table")
    R.check(gw, want_w, bound_w, "weight")


# -------------------------------------------------------------------------------- gradients of tables with few events
def grad_into(out, grad, tok, V, w, table):
    """The table's gradient through the C entry point, into a buffer of the caller."""
    from lens_amd import _lib
    (T, D), L, size, dev = grad.shape, _lib.lib(), E()._TYPES[grad.dtype], grad.get_device()
    order, gw = E().sort_events(tok, V), torch.empty(T, device="cuda")
    need = L.lens_embed_events_grad_scratch_bytes(size, T, V, D)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    E()._call("lens_embed_events_grad", dev, grad.data_ptr(), size, D, order.data_ptr(), w.data_ptr(), 0.5, T, V, D, table.data_ptr(), D,
              out.data_ptr(), gw.data_ptr(), scratch.data_ptr(), need)
    return gw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 3, 4, 7, 8, 63, 64, 200, 293, 600])
def test_table_gradient_of_few_events(dtype, D):
    """Every row is written, those between the events too, and nothing around them: rows next to each other, the first and the last,
    events that stand close in one part of the table and far apart in another, rows that are not aligned to vectors."""
    for V, tokens in ((1, [0]), (2, [1]), (700, [-1, -1]), (5000, [0]), (5000, [4999]), (5000, [2500, 2499, 2501, -1, 2500]), (5001, [0, 1, 2, 4998, 5000]),
                      (20011, list(range(3000, 3600)) + [3100] * 300 + list(range(5000, 20011, 777))),
                      (20011, list(range(0, 20011, 19))), (20011, list(range(5, 20011, 3)) + [11] * 2000)):
        g = gen(V + D + len(tokens))
        tok = torch.tensor(tokens, device="cuda")[torch.randperm(len(tokens), generator=g, device="cuda")]
        grad, table, w = rnd(g, len(tokens), D, dtype=dtype), rnd(g, V, D, dtype=dtype), rnd(g, len(tokens))
        want, bound, want_w, bound_w = R.embed_grad(grad, tok, V, w, 0.5, table)
        first = None
        for shift in (0, 1, 2, 3):
            buf = torch.full((V * D + 64,), float("nan"), device="cuda")
            out = buf[32 + shift:32 + shift + V * D].view(V, D)
            gw = grad_into(out, grad, tok, V, w, table)
            R.check(out, want, bound, f"table {V} {shift}")
            R.check(gw, want_w, bound_w, "weight")
            assert bool(torch.isnan(buf[:32 + shift]).all()) and bool(torch.isnan(buf[32 + shift + V * D:]).all())
            first = out if first is None else first
            assert torch.equal(out, first)
        none = torch.ones(V, dtype=torch.bool, device="cuda")
        none[tok[tok >= 0]] = False
        assert not f64_any(first[none])


def check_rows(out, grad, tok, w, table=None):
    """Rows with events against sums in 64 bits, all others zero."""
    V = out.shape[0]
    rows, at = torch.unique(tok[tok >= 0], return_inverse=True)
    terms = 0.5 * w[tok >= 0].double()[:, None] * grad[tok >= 0].double()
    want, mag = (torch.zeros(len(rows), out.shape[1], device="cuda", dtype=torch.float64).index_add_(0, at, v) for v in (terms, terms.abs()))
    R.check_all(out[rows], want, (len(tok) + 3) * R.U * mag, "rows with events")
    bounds = [-1, *rows.tolist(), V]
    for a, b in zip(bounds[:-1], bounds[1:]):
        for part in out[a + 1:b].split(1 << 17) if b > a + 1 else ():
            assert int(torch.count_nonzero(part)) == 0, (a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,D", [(170003, 300), (200011, 293), (100003, 601), (30011, 2047), (170003, 296)])
def test_gradient_of_a_large_table_with_few_events(dtype, V, D):
    """Tables beyond 192 MB, with few enough events that all zeros are written first, and with a few more."""
    for tokens in ([0], [V - 1, 7, V - 1, -1, 8], [-1], list(range(1000, 1400)) + [1200] * 100, list(range(0, V, 23)), list(range(3, V, 6))):
        g = gen(V + len(tokens))
        tok = torch.tensor(tokens, device="cuda")[torch.randperm(len(tokens), generator=g, device="cuda")]
        grad, table, w = rnd(g, len(tokens), D, dtype=dtype), rnd(g, V, D, dtype=dtype), rnd(g, len(tokens))
        for shift in (0, 3):
            buf = torch.full((V * D + 64,), float("nan"), device="cuda")
            out = buf[32 + shift:32 + shift + V * D].view(V, D)
            grad_into(out, grad, tok, V, w, table)
            assert bool(torch.isnan(buf[:32 + shift]).all()) and bool(torch.isnan(buf[32 + shift + V * D:]).all())
            if len(tokens) < 600:
                check_rows(out, grad, tok, w)
            else:
                order = torch.argsort(tok)                                 # every row has one event
                want = 0.5 * w[order].double()[:, None] * grad[order].double()
                R.check_all(out[tok[order]], want, 4 * R.U * want.abs(), "rows with events")
                out[tok[order]] = 0
                assert not f64_any(out)


def test_gradient_of_a_table_of_more_threads_than_a_launch_has():
    """69 GB: more 16-byte zeros than one launch writes."""
    V, D = 8389000, 2048
    g = gen(80)
    tok = torch.tensor([V - 1, 0, 5000000, 0, -1], device="cuda")
    grad, w = rnd(g, 5, D, dtype=torch.bfloat16), rnd(g, 5)
    out = torch.empty(V, D, device="cuda")
    for part in out.split(1 << 20):
        part.fill_(float("nan"))
    order = E().sort_events(tok, V)
    from lens_amd import _lib
    need = _lib.lib().lens_embed_events_grad_scratch_bytes(1, 5, V, D)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    E()._call("lens_embed_events_grad", 0, grad.data_ptr(), 1, D, order.data_ptr(), w.data_ptr(), 0.5, 5, V, D, None, 0, out.data_ptr(), None,
              scratch.data_ptr(), need)
    check_rows(out, grad, tok, w)



@pytest.mark.parametrize("T", [32769, 33793, 65536, 65537, 131072, 131073, 262143, 262144, 262145, 524289])
@pytest.mark.parametrize("V", [1, 300, 511, 512, 179920, 40000000])
def test_sort_at_the_borders_of_blocks(T, V):
    """Blocks of 1024, 2048 and 4096 tokens, 64 of them and one more, with digits of one bit to nine."""
    g = gen(T + V)
    wide = torch.randint(0, V, (T,), generator=g, device="cuda")
    u = torch.rand(T, generator=g, device="cuda")
    hot = torch.where(u < 0.5, torch.full_like(wide, V // 2), wide)
    outside = torch.where(u < 0.3, torch.full_like(wide, -1), wide)
    for tok in (wide.int(), hot, outside, torch.full_like(wide, V - 1), torch.arange(T, device="cuda").flip(0) % V):
        want, at = torch.sort(torch.where(tok >= 0, tok.long(), V), stable=True)
        assert torch.equal(E().sort_events(tok, V), want << 32 | at)


# ------------------------------------------------------------------------------------------ gradient of the rates, long sums
@pytest.mark.parametrize("dtype,launches,run", [(torch.float32, "1", 16), (torch.bfloat16, "1", 16), (torch.bfloat16, "3", 128)])
@pytest.mark.parametrize("dt", [1.9e-6, 7.3e-6])
def test_rate_gradient_of_a_long_recording(dtype, launches, run, dt, monkeypatch):
    """Rates and inputs of zero keep the state and its gradient as they are, so grad_rate is -h0 grad_last sum(dt) and all that may be off
    is the sum: u for a term's product, u for each of the run's additions in 32 bits, u for the result (64 bits lose nothing here)."""
    monkeypatch.setenv("LENS_AMD_SCAN_LAUNCHES", launches)
    T, D = 16 * 1024 * 1024, 4
    x = torch.zeros(1, D, device="cuda", dtype=dtype).expand(T, D)
    h0, gl = torch.tensor([[1.0, -1.0, 2.0, 0.5]], device="cuda"), torch.tensor([[1.0, 4.0, 0.25, -1.0]], device="cuda")
    d = dict(dt=torch.full((T,), dt, device="cuda"), rate=torch.zeros(D, device="cuda"))
    h, last, marks = E().gated_scan(x, h0=h0, marks=True, **d)
    gx, gr, g0 = E().gated_scan_grad(None, x, marks, h0=h0, grad_last=gl, **d)
    assert torch.equal(last, h0) and torch.equal(g0, gl) and bool((h == h0.to(dtype)).all()) and bool((gx == gl.to(dtype)).all())
    want = -(h0.double() * gl.double())[0] * d["dt"].double().sum()
    assert bool(((gr.double() - want).abs() <= (run + 3) * R.U * want.abs()).all()), ((gr.double() - want) / want / R.U).tolist()


# ------------------------------------------------------------------------------------------ sort, around the longest list of one launch
@pytest.mark.parametrize("T,V", [(32767, 300), (32768, 300), (32769, 300), (32768, 179920), (32769, 179920), (32768, 2147483000), (32769, 2147483000),
                                 (20000, 2147482000)])
def test_sort_at_the_border_of_one_launch(T, V):
    """Lists that fill every round of the kernel for short lists, and the first that takes the one for long lists: tokens anywhere, all
    at one row (several chunks in one workgroup), at two, the other way round, and many in a stretch that one workgroup sorts in
    several digits."""
    g = gen(T + V)
    wide = torch.randint(0, V, (T,), generator=g, device="cuda")
    one = torch.full((T,), V - 1, device="cuda")
    two = torch.where(torch.rand(T, generator=g, device="cuda") < 0.5, one, one - 1)
    close = torch.randint(0, min(V, 8000000), (T,), generator=g, device="cuda")
    outside = torch.where(torch.rand(T, generator=g, device="cuda") < 0.3, torch.full_like(wide, -1), wide)
    for tok in (wide, one, two, close, outside, torch.arange(T, device="cuda").flip(0) % V, two.int(), wide.int()):
        key = torch.where(tok >= 0, tok.long(), V)
        want, at = torch.sort(key, stable=True)
        assert torch.equal(E().sort_events(tok, V), want << 32 | at)


# ------------------------------------------------------------------------------------- gradients of few events, streams and graphs
def few_events(seed):
    """Gradients of 500 events on a table beyond 192 MB, of 40 000 events sorted by small blocks, and of few events among stretches."""
    g = gen(seed)
    sets = []
    for T, V, D, dtype in ((500, 170003, 300, torch.float32), (40000, 5003, 63, torch.bfloat16), (300, 20011, 100, torch.bfloat16)):
        sets.append((rnd(g, T, D, dtype=dtype), skewed(T, V, g).clamp(max=V - 1), V, rnd(g, T), rnd(g, V, D, dtype=dtype)))
    return sets


def few_gradients(sets):
    return [t for grad, tok, V, w, table in sets for t in E().embed_events_grad(grad, tok, V, weight=w, table=table)]


def test_gradients_of_few_events_in_graphs_and_on_streams():
    args = few_events(90)
    few_gradients(args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = few_gradients(args)
    for k in range(4):
        for mine, theirs in zip(args, few_events(91 + k)):
            for i in (0, 1, 3, 4):
                mine[i].copy_(theirs[i])                                   # other events, other tokens
        want = few_gradients(args)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    other = few_events(99)
    wants = few_gradients(args), few_gradients(other)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(a):
            got = few_gradients(args)
        with torch.cuda.stream(b):
            got_other = few_gradients(other)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got + got_other, wants[0] + wants[1]))

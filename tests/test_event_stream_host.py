"""The event-stream operators without a GPU: argument checks of the C entry points (a negative status, nothing enqueued) and of
their Python callers, sizes of scratch memory, and the 64-bit reference's gradients against differences."""
import ctypes

import numpy as np
import pytest
import torch

import event_stream_ref as R


@pytest.fixture(scope="module")
def L():
    from lens_amd import _lib
    _lib.build()
    return _lib.lib()


BUF = ctypes.create_string_buffer(4096 + 64)
P = (ctypes.addressof(BUF) + 63) // 64 * 64
NULL, SIZE, UNSUPPORTED, ALIGN, SCRATCH = -1, -2, -3, -4, -5


def test_lookup_refusals(L):
    ok = dict(table=P, type=0, n_rows=4, ld=8, tokens=P, size=4, weight=None, scale=1.0, T=2, D=8, out=P, ldo=8, bad=None, stream=None)

    def call(**kw):
        return L.lens_embed_events(*{**ok, **kw}.values())
    assert call(T=0) == 0
    assert call(table=None) == NULL and call(tokens=None) == NULL and call(out=None) == NULL
    assert call(type=3) == UNSUPPORTED and call(type=-1) == UNSUPPORTED
    for bad in (dict(T=-1), dict(D=0), dict(D=2049), dict(n_rows=-1), dict(n_rows=2**31), dict(T=2**31), dict(size=2), dict(ld=7), dict(ldo=7)):
        assert call(**bad) == SIZE, bad
    for bad in (dict(table=P + 2), dict(out=P + 1), dict(tokens=P + 2), dict(tokens=P + 4, size=8), dict(weight=P + 2), dict(bad=P + 4)):
        assert call(**bad) == ALIGN, bad


def test_sort_and_table_gradient_refusals(L):
    need = L.lens_sort_tokens_scratch_bytes(100, 50)
    ok = dict(tokens=P, size=4, T=100, n_rows=50, order=P, scratch=P, bytes=need, stream=None)

    def sort(**kw):
        return L.lens_sort_tokens(*{**ok, **kw}.values())
    assert sort(T=0) == 0
    assert sort(tokens=None) == NULL and sort(order=None) == NULL and sort(order=P + 4) == ALIGN and sort(scratch=None) == NULL
    assert sort(size=3) == SIZE and sort(T=-1) == SIZE and sort(n_rows=2**31) == SIZE
    assert sort(scratch=P + 8) == ALIGN and sort(bytes=need - 1) == SCRATCH
    assert L.lens_sort_tokens_scratch_bytes(-1, 5) == 0 and need >= 100 * 8
    need = L.lens_embed_events_grad_scratch_bytes(1, 100, 50, 64)
    ok_g = dict(grad=P, type=1, ld=64, order=P, weight=None, scale=1.0, T=100, n_rows=50, D=64, table=None, ldt=0, gt=P,
                gw=None, scratch=P, bytes=need, stream=None)

    def grad(**kw):
        return L.lens_embed_events_grad(*{**ok_g, **kw}.values())
    assert grad(T=0, n_rows=0) == 0
    for bad in (dict(grad=None), dict(order=None), dict(gt=None), dict(scratch=None), dict(gw=P)):
        assert grad(**bad) == NULL, bad
    for bad in (dict(ld=63), dict(D=0), dict(D=2049), dict(gw=P, table=P, ldt=63), dict(T=-1)):
        assert grad(**bad) == SIZE, bad
    assert grad(type=7) == UNSUPPORTED and grad(grad=P + 1) == ALIGN and grad(gt=P + 2) == ALIGN and grad(bytes=need - 1) == SCRATCH
    assert L.lens_embed_events_grad_scratch_bytes(9, 1, 1, 1) == 0


def scan_args(L, **kw):
    need = L.lens_gated_scan_scratch_bytes(100, 64, 0)
    ok = dict(x=P, type=1, ldx=64, gate=None, gtype=0, ldg=0, dt=P, rate=P, off=None, n_seq=1, h0=None, T=100, D=64, h=P, ldh=64, fill=1,
              last=P, marks=None, scratch=P, bytes=need, stream=None)
    return list({**ok, **kw}.values())


def test_scan_refusals(L):
    def call(**kw):
        return L.lens_gated_scan(*scan_args(L, **kw))
    for bad in (dict(x=None), dict(dt=None), dict(rate=None), dict(h=None), dict(last=None), dict(scratch=None), dict(n_seq=2)):
        assert call(**bad) == NULL, bad
    for bad in (dict(T=-1), dict(T=2**31), dict(D=0), dict(D=4097), dict(n_seq=0), dict(ldx=63), dict(ldh=63), dict(ldh=0)):
        assert call(**bad) == SIZE, bad
    gate = dict(gate=P, dt=None, rate=None, ldg=64)
    assert call(**gate, gtype=2) == UNSUPPORTED                              # gates of another 16-bit type
    assert call(**{**gate, "ldg": 63}, gtype=1) == SIZE
    assert call(gate=P, ldg=64, gtype=1) == UNSUPPORTED                      # gates and decays
    assert call(type=3) == UNSUPPORTED and call(**gate, gtype=5) == UNSUPPORTED
    for bad in (dict(x=P + 1), dict(h=P + 1), dict(dt=P + 2), dict(off=P + 4), dict(last=P + 1), dict(marks=P + 2), dict(scratch=P + 4)):
        assert call(**bad) == ALIGN, bad
    assert call(bytes=L.lens_gated_scan_scratch_bytes(100, 64, 0) - 1) == SCRATCH
    assert L.lens_gated_scan_scratch_bytes(-1, 4, 0) == 0 and L.lens_scan_mark_rows(0) == 0 and L.lens_scan_mark_rows(4097) == 0
    assert all(L.lens_scan_mark_rows(D) >= 8 for D in range(1, 4097))


def test_scan_gradient_refusals(L):
    need = L.lens_gated_scan_scratch_bytes(100, 64, 1)
    ok = dict(grad=P, ldd=64, grad_last=None, x=P, type=1, ldx=64, gate=None, gtype=0, ldg=0, dt=P, rate=P, off=None, n_seq=1, h0=None,
              marks=P, T=100, D=64, gx=P, ldgx=64, gg=None, ldgg=0, gr=P, g0=None, scratch=P, bytes=need, stream=None)

    def call(**kw):
        return L.lens_gated_scan_grad(*{**ok, **kw}.values())
    for bad in (dict(marks=None), dict(gx=None), dict(gr=None), dict(scratch=None), dict(x=None), dict(gate=P, ldg=64, gtype=1, dt=None, rate=None)):
        assert call(**bad) == NULL, bad
    for bad in (dict(ldd=63), dict(ldgx=63), dict(gate=P, ldg=64, gtype=1, dt=None, rate=None, gg=P, ldgg=63)):
        assert call(**bad) == SIZE, bad
    assert call(grad=P + 1) == ALIGN and call(gx=P + 1) == ALIGN and call(g0=P + 2) == ALIGN and call(bytes=need - 1) == SCRATCH


def test_step_refusals(L):
    ok = dict(state=P, lds=8, x=P, type=0, ldx=8, tokens=None, size=0, n_rows=0, weight=None, scale=1.0, gate=None, gtype=0, ldg=0, dt=P,
              rate=P, n=2, D=8, out=P, ldo=8, bad=None, stream=None)

    def call(**kw):
        return L.lens_gated_step(*{**ok, **kw}.values())
    assert call(n=0) == 0
    for bad in (dict(state=None), dict(x=None), dict(out=None), dict(dt=None), dict(rate=None)):
        assert call(**bad) == NULL, bad
    for bad in (dict(n=-1), dict(D=0), dict(D=4097), dict(lds=7), dict(ldo=0), dict(ldx=7), dict(tokens=P, size=2), dict(tokens=P, size=4, n_rows=3, ldx=0)):
        assert call(**bad) == SIZE, bad
    assert call(gate=P, ldg=8) == UNSUPPORTED and call(type=4) == UNSUPPORTED
    assert call(state=P + 2) == ALIGN and call(tokens=P + 4, size=8, n_rows=3) == ALIGN and call(bad=P + 4) == ALIGN


def test_python_callers_refuse_host_tensors_and_wrong_shapes():
    from lens_amd import engine as E
    from lens_amd._lib import LensAmdError
    f, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: E.embed_events(f, i), lambda: E.sort_events(i, 4), lambda: E.embed_events_grad(f, i, 4),
                 lambda: E.gated_scan(f, gate=f), lambda: E.gated_scan_grad(f, f, f, gate=f), lambda: E.gated_step(f, f, gate=f),
                 lambda: E.event_step(f, f, i, gate=f)):
        with pytest.raises(LensAmdError, match="device"):
            call()
    for off in ([0], [0, 5], [3, 2, 4], [-1, 4]):
        with pytest.raises(ValueError, match="seq_off"):
            E._sequences(off, 4, -1)
    assert E._sequences([0, 2, 4], 4, -1)[1] == 2 and E._sequences(None, 4, -1) == (None, 1)
    dev = -1
    with pytest.raises(AssertionError, match="overlap"):
        E._rows(f[:1].expand(4, 8), "out", 4, 8, torch.float32, dev)
    with pytest.raises(AssertionError, match="contiguous"):
        E._rows(torch.zeros(8, 4).t(), "x", 4, 8, torch.float32, dev)
    assert E._rows(f[:1].expand(4, 8), "x", 4, 8, torch.float32, dev, spread=True) == 0
    with pytest.raises(AssertionError, match="either"):
        E._decay(f, i, None, 4, 8, torch.float32, dev)
    with pytest.raises(AssertionError, match="gate must be"):
        E._decay(f.half(), None, None, 4, 8, torch.bfloat16, dev)


def test_reference_gradients_are_the_differences():
    """The 64-bit formulas that the GPU tests compare with, against central differences of the 64-bit forward."""
    rng = np.random.default_rng(1)
    T, D, off = 20, 3, [0, 7, 7, 18]
    x, a = torch.from_numpy(rng.standard_normal((T, D))), rng.uniform(-1, 1, (T, D))
    h0, cw, cl = (torch.from_numpy(rng.standard_normal(s)) for s in ((3, D), (T, D), (3, D)))

    def loss(x, a, h0):
        h, last, *_ = R.scan(x, a, off, h0)
        return float((h[:18] * cw.numpy()[:18]).sum() + (last * cl.numpy()).sum())
    g, ga, g0, *_ = R.scan_grad(cw, cl, x, a, None, off, h0)
    e = 1e-6
    for got, which in ((g, 0), (ga, 1), (g0, 2)):
        for at in np.ndindex(*got.shape):
            args = [x.clone(), a.copy(), h0.clone()]
            args[which][at] += e
            up = loss(*args)
            args[which][at] -= 2 * e
            assert abs((up - loss(*args)) / (2 * e) - got[at]) < 1e-7 * (1 + abs(got[at]))


def test_event_tokens_of_a_recording():
    from lens_amd.events import event_tokens
    t, x, y, p = [10.0, 12.0, 12.0, 2012.0, 5000.0], [1, 4, 5, 4, 0], [1, 3, 1, 3, 2], [0, 1, 1, -1, 1]
    tok, dt = event_tokens(t, x, y, p, height=3, width=4, device="cpu")
    assert tok.dtype == torch.int32 and tok.tolist() == [0, 23, -1, 11, -1]
    assert dt.dtype == torch.float32 and dt.tolist() == [np.float32(v) for v in (0, 2e-6, 0, 2e-3, 2.988e-3)]
    tok, dt = event_tokens(t, x, y, p, 3, 6, t_unit_s=1.0, device="cpu", one_based=False)
    assert tok.tolist() == [7, -1, 29, -1, 30] and dt.tolist() == [0, 2, 0, 2000, 2988]
    assert [v.numel() for v in event_tokens([], [], [], [], 3, 4, device="cpu")] == [0, 0]
    for bad in ((t[::-1], x, y, p, 3, 4), (t, x[:4], y, p, 3, 4), (t, x, y, p, 0, 4), (t, x, y, p, 2 ** 15, 2 ** 15)):
        with pytest.raises(ValueError):
            event_tokens(*bad, device="cpu")


@pytest.mark.parametrize("kind", ["time", "gate"])
def test_reference_side_by_side_is_the_reference_row_by_row(kind):
    g = torch.Generator().manual_seed(3)
    T, D = 257, 5
    off = R.ragged_offsets(T, 4)
    S = off.numel() - 1
    x, gh = torch.randn(T, D, generator=g), torch.randn(T, D, generator=g)
    h0, gl = torch.randn(S, D, generator=g), torch.randn(S, D, generator=g)
    d = dict(dt=torch.rand(T, generator=g), rate=torch.rand(D, generator=g)) if kind == "time" else dict(gate=torch.rand(T, D, generator=g) * 2 - 1)
    a = R.gates(d.get("gate"), d.get("dt"), d.get("rate"))
    rows, ends = R.scan(x, a, off.tolist(), h0), R.scan_grad(gh, gl, x, a, d.get("dt"), off.tolist(), h0)
    mine = R.scan_side_by_side(x, off, h0, **d)
    back = R.scan_grad_side_by_side(gh, gl, x, mine[2], mine[5], off, **d)
    for got, want in zip((*mine, *back), (*rows, *ends)):
        np.testing.assert_allclose(got.numpy(), want, rtol=1e-12, atol=1e-300)


def test_shapes_of_many_batches_have_them(L):
    """The scans that the GPU tests read twice: several batches of 8 rows a run, lanes of one run in two wavefronts, and offsets at
    multiples of 8 inside of runs whose neighbouring batches have starts or ends too.  The scratch memory that the library asks for
    tells its plan."""
    for D, T, _, rows in R.MANY_BATCHES:
        lanes, ts, run, scratch = R.plan_twice(T, D)
        assert scratch == L.lens_gated_scan_scratch_bytes(T, D, 0), (D, T)
        assert run == rows > 8 and any(k * lanes // 64 != ((k + 1) * lanes - 1) // 64 for k in range(ts)), (D, T)
        off = R.ragged_offsets(T, D)
        inside = off[(off % 8 == 0) & (off % run != 0)]
        assert inside.numel() > 500 and int(off[0]) > 0 and int(off[-1]) < T and bool((off[1:] == off[:-1]).any())


def test_python_callers_refuse_what_autograd_would_lose():
    """Inputs that require a gradient are refused where autograd records (the check comes before that of the device), and only there."""
    from lens_amd import engine as E
    from lens_amd._lib import LensAmdError
    f, i, v = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    p, r = torch.zeros(4, 8, requires_grad=True), torch.zeros(8)
    q, u = torch.zeros(8, requires_grad=True), torch.zeros(4, requires_grad=True)
    calls = [lambda: E.embed_events(p, i), lambda: E.embed_events(f, i, weight=u), lambda: E.embed_events(f, i, out=p * 1),
             lambda: E.embed_events_grad(p, i, 4), lambda: E.embed_events_grad(f, i, 4, weight=u, table=f), lambda: E.embed_events_grad(f, i, 4, weight=v, table=p),
             lambda: E.gated_scan(p, gate=f), lambda: E.gated_scan(f, gate=p), lambda: E.gated_scan(f, dt=v, rate=q), lambda: E.gated_scan(f, dt=u, rate=r),
             lambda: E.gated_scan(f, gate=f, h0=q[None]), lambda: E.gated_scan_grad(p, f, f, gate=f), lambda: E.gated_scan_grad(f, f, f, gate=p),
             lambda: E.gated_scan_grad(f, f, f, dt=v, rate=q), lambda: E.gated_scan_grad(f, f, f, gate=f, grad_last=q[None]),
             lambda: E.gated_step(p, f, gate=f), lambda: E.gated_step(f, p, gate=f), lambda: E.event_step(f, p, i, gate=f),
             lambda: E.event_step(f, f, i, weight=u, dt=v, rate=r), lambda: E.event_step(f, f, i, dt=v, rate=q, check=True)]
    for call in calls:
        with pytest.raises(LensAmdError, match="autograd"):
            call()
        with torch.no_grad(), pytest.raises(LensAmdError, match="device"):
            call()

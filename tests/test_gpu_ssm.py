"""Selective scan and causal convolution on the GPU against the 64-bit forms of tests/ssm_reference.py (tolerances there)."""
import itertools

import numpy as np
import pytest
import torch

import ssm_reference as R
from supernnova_amd import _lib as L
from supernnova_amd import ssm

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


class Batch:
    """Inputs in one of the layouts, with NaN in every row that belongs to no step, and each sequence's rows as numpy."""

    def __init__(self, lens, D, dt, layout, seed, pad=3, strided=False):
        self.g = torch.Generator().manual_seed(seed)
        self.lens, self.D, self.dt, self.layout, self.strided = list(lens), D, dt, layout, strided
        self.T, self.B = max(max(lens), 1) + (pad if layout != "rows" else 0), len(lens)
        self.kw = {}
        if layout == "rows":
            off = np.concatenate([[0], np.cumsum(lens)])
            self.off, self.rows = off, int(off[-1]) + pad
            self.kw = dict(offsets=torch.tensor(off, dtype=torch.int64, device="cuda"), max_len=max(max(lens), 1))
        else:
            self.kw = dict(lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"), time_major=layout == "time")

    def par(self, *shape, scale=1.0):
        return (torch.randn(shape, generator=self.g) * scale).cuda()

    def seqs(self, *tail, scale=1.0):
        """A tensor of the batch, NaN outside the sequences."""
        lead = {"rows": lambda: (self.rows,), "time": lambda: (self.T, self.B), "batch": lambda: (self.B, self.T)}[self.layout]()
        wide = tail[:-1] + (tail[-1] + (5 if self.strided else 0),)
        v = (torch.randn(lead + wide, generator=self.g) * scale).to(DT[self.dt])
        for b, n in enumerate(self.lens):
            if self.layout == "time":
                v[n:, b] = float("nan")
            elif self.layout == "batch":
                v[b, n:] = float("nan")
        if self.layout == "rows":
            v[self.off[-1]:] = float("nan")
        v = v.cuda()
        return v[..., 2:2 + tail[-1]] if self.strided else v

    def of(self, t, b):
        """Sequence b's rows of a tensor of the batch."""
        n = self.lens[b]
        a = _np(t)
        return a[:n, b] if self.layout == "time" else a[b, :n] if self.layout == "batch" else a[self.off[b]:self.off[b + 1]]

    def assert_clear(self, t, what):
        """Rows that belong to no step are zero."""
        a = _np(t)
        if self.layout == "rows":
            assert (a[self.off[-1]:] == 0).all(), what
        else:
            for b, n in enumerate(self.lens):
                assert ((a[n:, b] if self.layout == "time" else a[b, n:]) == 0).all(), (what, b)


def _grads_sum(parts):
    return {k: sum(p[k] for p in parts) for k in parts[0]}


CONV = [(dt, lay, W, D, silu) for (dt, lay), (W, D, silu) in itertools.product(
    [("f32", "time"), ("bf16", "batch"), ("f16", "rows"), ("bf16", "time")],
    [(2, 1, True), (3, 7, True), (4, 64, True), (4, 72, False)])]


@pytest.mark.parametrize("dt,layout,W,D,silu", CONV)
@pytest.mark.parametrize("lens,state,strided", [((1, 0, 2, 3, 40), True, False), ((5,), False, True), ((300, 17), True, True)])
def test_conv(dt, layout, W, D, silu, lens, state, strided):
    bt = Batch(lens, D, dt, layout, seed=W * 100 + D, strided=strided)
    x, dy = bt.seqs(D), bt.seqs(D)
    w, bias = bt.par(D, W, scale=0.5), bt.par(D) if D != 7 else None
    s0 = bt.par(bt.B, W - 1, D).to(DT[dt]) if state else None
    ds = bt.par(bt.B, W - 1, D).to(DT[dt]) if state else None
    kw = dict(activation="silu" if silu else None, initial_state=s0, **bt.kw)
    y, end = ssm.causal_conv_forward(x, w, bias, want_final_state=True, **kw)
    g = ssm.causal_conv_backward(x, w, bias, dy, dfinal_state=ds, **kw)
    k, parts, mags = W + 16, [], []
    for b in range(bt.B):
        a = (bt.of(x, b), _np(w), _np(bias), silu, None if s0 is None else _np(s0[b]), bt.of(dy, b), None if ds is None else _np(ds[b]))
        r, m = R.conv(*a), R.conv(*a, mag=True)
        R.close(bt.of(y, b), r["y"], m["y"], k, dt, "y")
        R.close(_np(end[b]), r["end"], m["end"], 0, dt, "end")
        R.close(bt.of(g.dx, b), r["dx"], m["dx"], 2 * k, dt, "dx")
        if state:
            R.close(_np(g.dinitial_state[b]), r["ds0"], m["ds0"], 2 * k, dt, "ds0")
        parts.append({"dw": r["dw"], "db": r["db"]})
        mags.append({"dw": m["dw"], "db": m["db"]})
    r, m, n = _grads_sum(parts), _grads_sum(mags), 2 * k + sum(lens)
    R.close(_np(g.dweight), r["dw"], m["dw"], n, "f32", "dw")
    assert (g.dbias is None) == (bias is None)
    if bias is not None:
        R.close(_np(g.dbias), r["db"], m["db"], n, "f32", "db")
    bt.assert_clear(y, "y")
    bt.assert_clear(g.dx, "dx")


def _scan_inputs(bt, N, G, gate, state, skip=True, dbias=True):
    D = bt.D
    tail = (G, N) if G > 1 or bt.layout == "rows" else (N,)
    i = dict(x=bt.seqs(D), delta=bt.seqs(D, scale=0.7), A=-torch.empty(D, N).uniform_(0.1, 2.0, generator=bt.g).cuda(), B=bt.seqs(*tail), C=bt.seqs(*tail),
             D=bt.par(D) if skip else None, z=bt.seqs(D) if gate else None, delta_bias=bt.par(D, scale=0.5) if dbias else None)
    h0 = bt.par(bt.B, D, N) if state else None
    return i, h0


def _check_scan(bt, i, h0, G, sp, dy, dend, y, end, g):
    D, N, dt = bt.D, i["A"].shape[1], bt.dt
    wide = lambda a: np.repeat(a.reshape(a.shape[0], G, N), D // G, axis=1)          # noqa: E731
    parts, mags = [], []
    for b in range(bt.B):
        T = bt.lens[b]
        a = dict(x=bt.of(i["x"], b), delta=bt.of(i["delta"], b), A=_np(i["A"]), B=wide(bt.of(i["B"], b)), C=wide(bt.of(i["C"], b)),
                 skip=_np(i["D"]), z=None if i["z"] is None else bt.of(i["z"], b), dbias=_np(i["delta_bias"]), sp=sp,
                 h0=None if h0 is None else _np(h0[b]))
        if dy is not None:
            a.update(dy=bt.of(dy, b), dend=None if dend is None else _np(dend[b]))
        r, m = R.scan(**a), R.scan(**a, mag=True)
        k = 16 * T + 32 + N
        R.close(bt.of(y, b), r["y"], m["y"], k, dt, "y")
        if end is not None:
            R.close(_np(end[b]), r["end"], m["end"], k, "f32", "end")
        if dy is None:
            continue
        k *= 2
        R.close(bt.of(g.dx, b), r["dx"], m["dx"], k, dt, "dx")
        R.close(bt.of(g.ddelta, b), r["ddelta"], m["ddelta"], k, dt, "ddelta")
        if i["z"] is not None:
            R.close(bt.of(g.dz, b), r["dz"], m["dz"], k, dt, "dz")
        grp = lambda v: v.reshape(T, G, D // G, N).sum(2)                            # noqa: E731
        R.close(bt.of(g.dB, b).reshape(T, G, N), grp(r["dB"]), grp(m["dB"]), k + D, dt, "dB")
        R.close(bt.of(g.dC, b).reshape(T, G, N), grp(r["dC"]), grp(m["dC"]), k + D, dt, "dC")
        if h0 is not None:
            R.close(_np(g.dinitial_state[b]), r["dh0"], m["dh0"], k, "f32", "dh0")
        keep = ("dA", "dskip", "ddbias")
        parts.append({n: r[n] for n in keep})
        mags.append({n: m[n] for n in keep})
    if dy is not None:
        r, m, k = _grads_sum(parts), _grads_sum(mags), 2 * (16 * max(bt.lens) + 32 + N) + sum(bt.lens)
        R.close(_np(g.dA), r["dA"], m["dA"], k, "f32", "dA")
        for got, name, have in ((g.dD, "dskip", i["D"]), (g.ddelta_bias, "ddbias", i["delta_bias"])):
            assert (got is None) == (have is None)
            if have is not None:
                R.close(_np(got), r[name], m[name], k, "f32", name)
        for n in ("dx", "ddelta", "dB", "dC") + (("dz",) if i["z"] is not None else ()):
            bt.assert_clear(getattr(g, n), n)
    bt.assert_clear(y, "y")


SCAN = [  # dt, layout, D, N, G, lens, gate, state, strided
    ("f32", "time", 1, 1, 1, (1,), False, False, False),
    ("f32", "time", 7, 3, 1, (0, 1, 2, 5), True, True, False),
    ("bf16", "batch", 64, 16, 1, (15, 16, 17, 0, 33), True, True, True),
    ("f16", "rows", 66, 16, 2, (9, 0, 40, 1), True, False, True),
    ("f32", "rows", 130, 8, 1, (31, 8), False, True, False),
    ("f32", "batch", 65, 17, 1, (20, 7), True, True, False),
    ("bf16", "time", 36, 32, 3, (12, 3, 0), False, True, False),
    ("f32", "batch", 48, 33, 4, (11, 4), True, False, True),
    ("f16", "time", 20, 64, 1, (9, 10), True, True, False),
    ("f32", "time", 64, 4, 1, (50, 3), True, True, False),
    ("f32", "batch", 80, 16, 1, (300, 190, 64, 1), True, True, False),      # the time axis is split
    ("bf16", "rows", 16, 16, 1, (0, 515, 128, 0), True, True, False),
    ("f32", "time", 200, 24, 2, (260, 257), False, True, True),
]

# enough workgroups for the sequences to be taken longest first
_MANY = tuple(int(v) for v in np.random.default_rng(0).integers(0, 14, 200))
SCAN += [("f32", "time", 130, 16, 1, _MANY, True, True, False), ("bf16", "rows", 150, 4, 1, _MANY, False, True, False)]


@pytest.mark.parametrize("dt,layout,D,N,G,lens,gate,state,strided", SCAN)
def test_scan(dt, layout, D, N, G, lens, gate, state, strided):
    bt = Batch(lens, D, dt, layout, seed=D + N, strided=strided)
    i, h0 = _scan_inputs(bt, N, G, gate, state, skip=D != 65, dbias=D != 48)
    sp = D != 64 or N != 4
    if not sp:
        i["delta"] = i["delta"].abs()                  # without softplus the steps are the inputs themselves
        i["delta_bias"] = i["delta_bias"].abs()
    dy = bt.seqs(D)
    dend = bt.par(bt.B, D, N) if state else None
    kw = dict(delta_softplus=sp, initial_state=h0, **bt.kw)
    y0, end0 = ssm.selective_scan_forward(**i, want_final_state=state, **kw)
    y, end, tape = ssm.selective_scan_train(**i, want_final_state=state, **kw)
    g = ssm.selective_scan_backward(**i, dy=dy, tape=tape, dfinal_state=dend, **kw)
    assert torch.equal(y0, y) and (end is None or torch.equal(end0, end))
    _check_scan(bt, i, h0, G, sp, dy, dend, y, end, g)


def test_scan_of_one_group_as_three_dimensions():
    bt = Batch((4, 6), 8, "f32", "batch", 1)
    i, _ = _scan_inputs(bt, 5, 1, False, False)
    four = dict(i, B=i["B"][:, :, None], C=i["C"][:, :, None])
    y, _, tape = ssm.selective_scan_train(**i, **bt.kw)
    dy = bt.seqs(8)
    g3 = ssm.selective_scan_backward(**i, dy=dy, tape=tape, **bt.kw)
    g4 = ssm.selective_scan_backward(**four, dy=dy, tape=tape, **bt.kw)
    assert g3.dB.shape == i["B"].shape and torch.equal(g3.dB, g4.dB[:, :, 0]) and torch.equal(ssm.selective_scan_forward(**four, **bt.kw)[0], y)


@pytest.mark.parametrize("dt,D,N,G,W", [("f32", 7, 3, 1, 2), ("bf16", 64, 16, 1, 4), ("f16", 24, 33, 2, 3), ("bf16", 40, 8, 1, 4)])
def test_steps_follow_a_prompt(dt, D, N, G, W):
    """A prompt of six steps, then five single steps, is the sequence of eleven: the states and outputs of the whole."""
    bt = Batch((11, 11, 11), D, dt, "batch", 5, pad=0)
    i, _ = _scan_inputs(bt, N, G, True, False)
    w, bias = bt.par(D, W), bt.par(D)
    yc, cend = ssm.causal_conv_forward(i["x"], w, bias, want_final_state=True, time_major=False)
    ys, send = ssm.selective_scan_forward(**i, want_final_state=True, time_major=False)
    per = ("x", "delta", "B", "C", "z")
    part = lambda a, b: {k: v[:, a:b] if k in per else v for k, v in i.items()}                  # noqa: E731
    c6, cstate = ssm.causal_conv_forward(i["x"][:, :6], w, bias, want_final_state=True, time_major=False)
    s6, sstate = ssm.selective_scan_forward(**part(0, 6), want_final_state=True, time_major=False)
    assert torch.equal(c6, yc[:, :6]) and torch.equal(s6, ys[:, :6])
    for t in range(6, 11):
        one = {k: v[:, t] if k in per else v for k, v in i.items()}
        keep = (cstate.clone(), sstate.clone(), torch.empty_like(cstate), torch.empty_like(sstate))
        y2 = ssm.causal_conv_step(one["x"], keep[0], w, bias, new_state=keep[2])
        z2 = ssm.selective_scan_step(state=keep[1], new_state=keep[3], **one)
        assert torch.equal(keep[0], cstate) and torch.equal(keep[1], sstate)                      # left as they were
        y1 = ssm.causal_conv_step(one["x"], cstate, w, bias)
        z1 = ssm.selective_scan_step(state=sstate, **one)
        assert torch.equal(y1, y2) and torch.equal(z1, z2) and torch.equal(cstate, keep[2]) and torch.equal(sstate, keep[3])
        assert torch.equal(y1, yc[:, t])
        # the step adds the states' products in another order: N roundings of the sum, one step of the type at most
        err = (z1.float() - ys[:, t].float()).abs()
        assert bool((err <= 2 * R.HALF[dt] * ys[:, t].float().abs() + 1e-4 * (dt == "f32") + 1e-2 * (dt != "f32")).all())
    assert torch.equal(cstate, cend)
    assert bool(((sstate - send).abs() <= 11 * 16 * R.EPS32 * (1 + send.abs()) * 10).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_scan_step_against_reference(dt):
    for D, N, G, sp in ((5, 1, 1, True), (64, 16, 1, True), (30, 20, 3, False)):
        bt = Batch((1, 1, 1, 1), D, dt, "batch", D, pad=0)
        i, h0 = _scan_inputs(bt, N, G, D == 64, True)
        st = h0.clone()
        y = ssm.selective_scan_step(state=st, delta_softplus=sp, **{k: v[:, 0] if k in ("x", "delta", "B", "C", "z") and v is not None else v for k, v in i.items()})
        _check_scan(bt, i, h0, G, sp, None, None, y[:, None], st, None)


def test_scan_is_deterministic_and_split_agrees_with_whole():
    bt = Batch((700, 650), 96, "f32", "batch", 3)
    i, h0 = _scan_inputs(bt, 16, 1, True, True)
    dy, kw = bt.seqs(96), dict(initial_state=h0, **bt.kw)
    runs = []
    for _ in range(2):
        y, end, tape = ssm.selective_scan_train(**i, want_final_state=True, **kw)
        runs.append([y, end, *[t for t in ssm.selective_scan_backward(**i, dy=dy, tape=tape, **kw) if t is not None]])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_extreme_inputs():
    """Steps of zero and of thousands, infinite and NaN inputs: what the formulas give, and only in their own sequence."""
    bt = Batch((6, 6, 6), 8, "f32", "batch", 9, pad=0)
    i, _ = _scan_inputs(bt, 4, 1, False, False, dbias=False)
    i["delta"][0, 2] = -200.0                     # a step of zero: the state stays
    i["delta"][0, 4] = 5000.0                     # a decay of zero: the state is forgotten
    clean = {k: v.clone() if v is not None else None for k, v in i.items()}
    i["x"][1, 3, 2] = float("nan")
    i["x"][2, 1, 5] = float("inf")
    y, _ = ssm.selective_scan_forward(**i, time_major=False)
    yc, _ = ssm.selective_scan_forward(**clean, time_major=False)
    assert torch.isfinite(yc).all()
    a = _np(clean["x"][0]), _np(clean["delta"][0]), _np(i["A"])
    wide = lambda t: np.repeat(_np(t)[:, None], 8, axis=1)                                        # noqa: E731
    args = (*a, wide(clean["B"][0]), wide(clean["C"][0]), _np(i["D"]))
    # s A is as large as 10^4 in one step: its rounding is 10^4 half steps of an exponential that is zero
    R.close(_np(y[0]), R.scan(*args)["y"], R.scan(*args, mag=True)["y"], 200, "f32")
    assert torch.equal(y[0], yc[0])
    assert torch.isnan(y[1, 3:, 2]).all() and torch.equal(y[1, :3], yc[1, :3])
    ok = [c for c in range(8) if c != 2]
    assert torch.equal(y[1][:, ok], yc[1][:, ok])
    assert not torch.isfinite(y[2, 1, 5]) and torch.equal(y[2, :1], yc[2, :1])


def test_wrong_lengths_and_offsets_stay_inside_the_tensors():
    x, w = torch.randn(4, 3, 8, device="cuda"), torch.randn(8, 4, device="cuda")
    bad = torch.tensor([-5, 100, 2], dtype=torch.int32, device="cuda")
    good = torch.tensor([0, 4, 2], dtype=torch.int32, device="cuda")
    assert torch.equal(ssm.causal_conv_forward(x, w, lengths=bad)[0], ssm.causal_conv_forward(x, w, lengths=good)[0])
    r = torch.randn(10, 8, device="cuda")
    off = torch.tensor([0, 4, 999], dtype=torch.int64, device="cuda")
    fix = torch.tensor([0, 4, 10], dtype=torch.int64, device="cuda")
    d, A, bc = torch.randn_like(r), -torch.rand(8, 4, device="cuda"), torch.randn(10, 4, device="cuda")
    assert torch.equal(ssm.selective_scan_forward(r, d, A, bc, bc, offsets=off)[0], ssm.selective_scan_forward(r, d, A, bc, bc, offsets=fix)[0])
    # rows in front of the first sequence and past max_len are zero
    late = torch.tensor([2, 10], dtype=torch.int64, device="cuda")
    y, _ = ssm.selective_scan_forward(r, d, A, bc, bc, offsets=late, max_len=5)
    assert (y[:2] == 0).all() and (y[7:] == 0).all() and torch.equal(y[2:7], ssm.selective_scan_forward(r[2:7], d[2:7], A, bc[2:7], bc[2:7],
                                                                                                       offsets=late.new_tensor([0, 5]))[0])
    yc, _ = ssm.causal_conv_forward(r, w, offsets=late, max_len=5)
    assert (yc[:2] == 0).all() and (yc[7:] == 0).all() and (yc[2:7] != 0).any()


def _captured(fn):
    """fn's outputs as a graph leaves them, and its replay."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return out, graph


def test_captured_training_step_and_two_graphs():
    """Forward and explicit backward in graphs, replayed with eager work in between; two graphs keep their own workspaces."""
    def make(seed, T):
        bt = Batch((T, T // 2), 96, "bf16", "batch", seed)
        i, h0 = _scan_inputs(bt, 16, 1, True, True)
        dy, w, bias = bt.seqs(96), bt.par(96, 4), bt.par(96)

        def fn():
            xc, cend = ssm.causal_conv_forward(i["x"], w, bias, want_final_state=True, **bt.kw)
            j = dict(i, x=xc)
            y, end, tape = ssm.selective_scan_train(**j, initial_state=h0, want_final_state=True, **bt.kw)
            g = ssm.selective_scan_backward(**j, dy=dy, tape=tape, initial_state=h0, **bt.kw)
            c = ssm.causal_conv_backward(i["x"], w, bias, g.dx, **bt.kw)
            return [y, end, cend, *[t for t in g if t is not None], c.dx, c.dweight, c.dbias]
        return i, fn
    (i1, f1), (i2, f2) = make(1, 200), make(2, 90)
    o1, g1 = _captured(f1)
    o2, g2 = _captured(f2)
    for n in range(3):
        i1["x"].nan_to_num_().mul_(1.01)
        i2["x"].nan_to_num_().mul_(0.99)
        g1.replay()
        g2.replay()
        e1 = f1()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(o1, e1)), n
        assert all(torch.equal(a, b) for a, b in zip(o2, f2())), n


def test_autograd_is_refused_inside_a_capture():
    x = torch.randn(3, 2, 4, device="cuda", requires_grad=True)
    w = torch.randn(4, 3, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y0 = torch.zeros(4, device="cuda")
        with pytest.raises(L.SnnError, match="captured"):
            ssm.causal_conv(x, w)
        with torch.no_grad():
            y = ssm.causal_conv(x, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ssm.causal_conv_forward(x.detach(), w)[0]) and (y0 == 0).all()


def test_side_stream():
    bt = Batch((130, 40), 64, "f32", "batch", 4)
    i, h0 = _scan_inputs(bt, 16, 1, True, True)
    want = ssm.selective_scan_forward(**i, initial_state=h0, **bt.kw)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ssm.selective_scan_forward(**i, initial_state=h0, **bt.kw)[0] for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(want, g) for g in got)


def test_layer_with_autograd_against_torch():
    """Convolution, scan, clipping and Adam as one training step of a layer, on every gradient against torch in float64."""
    from supernnova_amd import optim
    g = torch.Generator().manual_seed(0)
    T, B, D, N, F = 21, 5, 24, 6, 10
    rnd = lambda *s: torch.randn(s, generator=g)                                                  # noqa: E731
    par = dict(win=rnd(2 * D, F) / F ** .5, wc=rnd(D, 4) / 2, bc=rnd(D) / 4, wx=rnd(D + 2 * N, D) / D ** .5, A=-torch.rand(D, N, generator=g) - 0.1,
               Dk=rnd(D), dtb=rnd(D) / 4, wout=rnd(3, D) / D ** .5)
    x, lens, tgt = rnd(T, B, F), torch.tensor([21, 9, 1, 14, 3]), torch.tensor([0, 2, 1, 1, 0])
    keep = (torch.arange(T)[:, None] < lens)[..., None]

    def layer(p, x, keep, conv, scan):
        xz = x @ p["win"].t()
        u = conv(xz[..., :D], p["wc"], p["bc"])
        dbc = u @ p["wx"].t()
        y = scan(u, dbc[..., :D], p["A"], dbc[..., D:D + N], dbc[..., D + N:], p["Dk"], xz[..., D:], p["dtb"])
        pooled = (y * keep).sum(0) / keep.sum(0)
        return torch.nn.functional.cross_entropy(pooled @ p["wout"].t(), tgt.to(x.device))

    def conv64(x, w, b):
        xx = torch.cat([torch.zeros(3, B, D, dtype=x.dtype), x * keep])
        p = b + sum(w[:, k] * xx[k:k + T] for k in range(4))
        return p * torch.sigmoid(p) * keep

    def scan64(x, delta, A, Bm, Cm, Dk, z, dtb):
        h, ys = torch.zeros(B, D, N, dtype=x.dtype), []
        for t in range(T):
            s = torch.nn.functional.softplus(delta[t] + dtb)
            h = torch.exp(s[..., None] * A) * h + (s * x[t])[..., None] * Bm[t][:, None]
            ys.append(((h * Cm[t][:, None]).sum(-1) + Dk * x[t]) * z[t] * torch.sigmoid(z[t]))
        return torch.stack(ys)
    p64 = {k: v.double().requires_grad_() for k, v in par.items()}
    l64 = layer(p64, x.double(), keep.double(), conv64, scan64)
    l64.backward()
    ln = lens.int().cuda()
    p = {k: v.cuda().requires_grad_() for k, v in par.items()}
    loss = layer(p, x.cuda(), keep.float().cuda(), lambda *a: ssm.causal_conv(*a, lengths=ln), lambda *a: ssm.selective_scan(*a, lengths=ln))
    loss.backward()
    # fp32 over T = 21 steps: (32 T + 64) roundings of the magnitudes, which a random layer of this size holds below 10 x the values
    tol = 10 * (32 * T + 64) * R.EPS32
    assert abs(float(loss.detach()) - float(l64.detach())) <= tol * abs(float(l64.detach()))
    for k in par:
        ref = p64[k].grad
        assert float((p[k].grad.double().cpu() - ref).abs().max()) <= tol * float(ref.abs().max()), k
    norm = optim.clip_grad_norm_(p.values(), 0.05)
    ref = torch.sqrt(sum((v.grad ** 2).sum() for v in p64.values()))
    assert abs(float(norm) - float(ref)) <= tol * float(ref)
    clipped = torch.sqrt(sum((v.grad.double() ** 2).sum() for v in p.values()))
    assert abs(float(clipped) - 0.05) <= 0.05 * (2e-5 / float(ref) + 1e-6)
    before = p["A"].detach().clone()
    torch.optim.Adam(p.values(), lr=1e-2).step()
    assert not torch.equal(before, p["A"])


def test_gradients_through_states_and_broadcast_inputs():
    """Two calls joined by the state differentiate like one; an input expanded over the batch sums its gradients."""
    g = torch.Generator().manual_seed(3)
    T, B, D, N = 12, 3, 8, 5
    rnd = lambda *s: torch.randn(s, generator=g).cuda()                                           # noqa: E731
    leaves = dict(x=rnd(T, B, D), delta=rnd(T, B, D), A=-torch.rand(D, N, generator=g).cuda() - 0.1, B=rnd(T, 1, N), C=rnd(T, B, N))
    w, ct = rnd(T, B, D), rnd(B, D, N)

    def run(cut):
        p = {k: v.clone().requires_grad_() for k, v in leaves.items()}
        q = dict(p, B=p["B"].expand(T, B, N))
        if cut:
            sl = lambda a, b: [q[k][a:b] if k != "A" else q[k] for k in ("x", "delta", "A", "B", "C")]      # noqa: E731
            y1, s1 = ssm.selective_scan(*sl(0, 5), return_final_state=True)
            y2, s2 = ssm.selective_scan(*sl(5, T), initial_state=s1, return_final_state=True)
            y, s = torch.cat([y1, y2]), s2
        else:
            y, s = ssm.selective_scan(*q.values(), return_final_state=True)
        ((y * w).sum() + (s * ct).sum()).backward()
        return {k: v.grad for k, v in p.items()}
    a, b = run(False), run(True)
    for k in leaves:
        # the same sums in another order: (32 T + 64) roundings of the magnitudes, here below 10 times the largest value
        assert float((a[k] - b[k]).abs().max()) <= 10 * (32 * T + 64) * R.EPS32 * float(a[k].abs().max()), k


def test_rows_beyond_31_bits_of_elements():
    """Offsets of more than 2^31 elements, inside one strided view and over a long batch."""
    D, far = 64, (1 << 31) + 64
    buf = torch.zeros(far + 4 * D, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buf, (2, 3, D), (far, D, 1))
    x.copy_(torch.randn(2, 3, D))
    w, A = torch.randn(D, 4, device="cuda"), -torch.rand(D, 4, device="cuda")
    bc = torch.randn(2, 3, 4, device="cuda").bfloat16()
    near = x.contiguous()
    assert torch.equal(ssm.causal_conv_forward(x, w, time_major=False)[0], ssm.causal_conv_forward(near, w, time_major=False)[0])
    assert torch.equal(ssm.selective_scan_forward(x, x, A, bc, bc, time_major=False)[0],
                       ssm.selective_scan_forward(near, near, A, bc, bc, time_major=False)[0])
    del buf, x, near
    T, D = 16400, 2048
    long = torch.zeros(T, 65, D, dtype=torch.bfloat16, device="cuda")
    long[-3:, -1].normal_()
    w = torch.randn(D, 2, device="cuda")
    y, _ = ssm.causal_conv_forward(long, w)
    assert torch.equal(y[-3:, -1:], ssm.causal_conv_forward(long[-4:, -1:].contiguous(), w)[0][1:])


@pytest.mark.parametrize("change,match", [
    (dict(delta=lambda i: i["delta"][:, :, :4]), "delta"), (dict(delta=lambda i: i["delta"].double()), "delta"),
    (dict(A=lambda i: i["A"].bfloat16()), "A must be"), (dict(A=lambda i: i["A"][:4]), "A must be"),
    (dict(B=lambda i: i["B"][..., :3]), "alike"), (dict(D=lambda i: i["D"].cpu()), "D must"),
    (dict(z=lambda i: i["x"].transpose(0, 2).contiguous().transpose(0, 2)), "unit stride"),
    (dict(lengths=lambda i: torch.ones(2, dtype=torch.int64, device="cuda")), "lengths"),
    (dict(lengths=lambda i: torch.ones(3, dtype=torch.int32, device="cuda")), "lengths"),
    (dict(offsets=lambda i: torch.zeros(3, dtype=torch.int64, device="cuda")), "rows"),
    (dict(max_len=lambda i: 3), "offsets"), (dict(initial_state=lambda i: torch.zeros(2, 8, 5, device="cuda")), "initial_state"),
    (dict(x=lambda i: i["x"].double()), "float32, bfloat16 or float16"), (dict(x=lambda i: i["x"][:0]), "at least one"),
    (dict(B=lambda i: torch.zeros(6, 2, 3, 4, device="cuda"), C=lambda i: torch.zeros(6, 2, 3, 4, device="cuda")), "groups"),
    (dict(A=lambda i: torch.zeros(8, 65, device="cuda")), "1..64")])
def test_refusals(change, match):
    g = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=g).cuda()                                           # noqa: E731
    i = dict(x=rnd(6, 2, 8), delta=rnd(6, 2, 8), A=-rnd(8, 4).abs(), B=rnd(6, 2, 4), C=rnd(6, 2, 4), D=rnd(8))
    ssm.selective_scan_forward(**i)
    with pytest.raises(L.SnnError, match=match):
        ssm.selective_scan_forward(**dict(i, **{k: f(i) for k, f in change.items()}))


def test_conv_and_step_refusals():
    x, w = torch.zeros(4, 2, 8, device="cuda"), torch.zeros(8, 4, device="cuda")
    for kw, match in ((dict(weight=torch.zeros(8, 5, device="cuda")), "weight"), (dict(weight=w.half()), "weight"), (dict(activation="relu"), "activation"),
                      (dict(initial_state=torch.zeros(2, 4, 8, device="cuda")), "initial_state"), (dict(bias=torch.zeros(7, device="cuda")), "bias")):
        with pytest.raises(L.SnnError, match=match):
            ssm.causal_conv_forward(x, **dict(dict(weight=w), **kw))
    with pytest.raises(L.SnnError, match="state"):
        ssm.causal_conv_step(x[0], None, w)
    with pytest.raises(L.SnnError, match="new_state"):
        ssm.causal_conv_step(x[0], torch.zeros(2, 3, 8, device="cuda"), w, new_state=torch.zeros(2, 3, 8, device="cuda").half())
    pool = torch.zeros(3, 3, 8, device="cuda")
    with pytest.raises(L.SnnError, match="overlap"):
        ssm.causal_conv_step(x[0], pool[:2], w, new_state=pool[1:])
    with pytest.raises(L.SnnError, match="channels"):
        ssm.causal_conv_step(x, torch.zeros(2, 3, 8, device="cuda"), w)
    y, _, tape = ssm.selective_scan_train(x, x, -torch.ones(8, 4, device="cuda"), x[..., :4], x[..., :4])
    with pytest.raises(L.SnnError, match="too small"):
        ssm.selective_scan_backward(x, x, -torch.ones(8, 4, device="cuda"), x[..., :4], x[..., :4], y, tape[:8])


def test_one_state_pool_shifted_by_whole_states_is_allowed():
    """Disjoint slices of one pool as state and new_state."""
    pool, x, w = torch.randn(4, 3, 8, device="cuda"), torch.randn(2, 8, device="cuda"), torch.randn(8, 4, device="cuda")
    want = pool[:2].clone()
    y = ssm.causal_conv_step(x, want, w)
    assert torch.equal(ssm.causal_conv_step(x, pool[:2], w, new_state=pool[2:]), y) and torch.equal(pool[2:], want)


def test_channels_first_and_odd_strides_through_autograd():
    """The gradient of a sum has no strides of its own, a transposed result's gradient arrives transposed."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn(2, 9, 6, generator=g).cuda().requires_grad_()
    w = torch.randn(6, 3, generator=g).cuda().requires_grad_()
    ssm.causal_conv(x, w, time_major=False).sum().backward()
    a = x.grad.clone(), w.grad.clone()
    x.grad = w.grad = None
    (ssm.causal_conv(x, w, time_major=False).transpose(1, 2) * torch.ones(2, 6, 9, device="cuda")).sum().backward()
    assert torch.equal(a[0], x.grad) and torch.equal(a[1], w.grad)


def test_long_sequences_and_many_of_them():
    """A sequence of 20000 steps (chunks of the time axis), and 70000 of two (more than a grid's other dimensions hold),
    against the same rows one by one."""
    g = torch.Generator().manual_seed(2)
    rnd = lambda *s: torch.randn(s, generator=g).cuda()                                           # noqa: E731
    A = -torch.rand(8, 4, generator=g).cuda()
    x, d, B, C = rnd(1, 20000, 8), rnd(1, 20000, 8), rnd(1, 20000, 4), rnd(1, 20000, 4)
    y, end, tape = ssm.selective_scan_train(x, d, A, B, C, want_final_state=True, time_major=False)
    state, ys = None, []
    for t in range(0, 20000, 5000):
        p, state = ssm.selective_scan_forward(x[:, t:t + 5000], d[:, t:t + 5000], A, B[:, t:t + 5000], C[:, t:t + 5000], initial_state=state,
                                              want_final_state=True, time_major=False)
        ys.append(p)
    # decays of at least exp(-s A) forget: what differs is the last few hundred steps' rounding
    assert float((torch.cat(ys, 1) - y).abs().max()) <= 1000 * R.EPS32 * float(y.abs().max())
    assert float((state - end).abs().max()) <= 1000 * R.EPS32 * float(end.abs().max())
    gr = ssm.selective_scan_backward(x, d, A, B, C, torch.ones_like(y), tape, time_major=False)
    assert all(torch.isfinite(t).all() for t in gr if t is not None)
    many = [rnd(2, 70000, 8), rnd(2, 70000, 8), A, rnd(2, 70000, 4), rnd(2, 70000, 4)]
    y, _, tape = ssm.selective_scan_train(*many)
    gr = ssm.selective_scan_backward(*many, torch.ones_like(y), tape)
    part = [t[:, 69990:] if t is not A else A for t in many]
    y1, _, tape1 = ssm.selective_scan_train(*part)
    g1 = ssm.selective_scan_backward(*part, torch.ones_like(y1), tape1)
    assert torch.equal(y[:, 69990:], y1) and torch.equal(gr.dx[:, 69990:], g1.dx) and torch.equal(gr.dB[:, 69990:], g1.dB)
    assert torch.equal(ssm.causal_conv_forward(many[0], rnd(8, 4))[0].isfinite().all(), torch.tensor(True, device="cuda"))


def test_growing_states_that_are_still_zero_stay_zero():
    """Decays above one whose product over a chunk of the time axis overflows, before the first input and behind the last
    gradient that is not zero: 0 times that product is 0, as step by step."""
    g = torch.Generator().manual_seed(4)
    T, D, N = 400, 8, 4
    x, B, C = torch.randn(1, T, D, generator=g), torch.randn(1, T, N, generator=g), torch.randn(1, T, N, generator=g)
    delta = torch.full((1, T, D), 2.0)
    delta[:, 350:] = -1.0
    x[:, :350] = 0
    dy = torch.randn(1, T, D, generator=g)
    dy[:, 20:] = 0
    A = torch.ones(D, N)
    x, delta, A, B, C, dy = (t.cuda() for t in (x, delta, A, B, C, dy))
    y, end, tape = ssm.selective_scan_train(x, delta, A, B, C, delta_softplus=False, want_final_state=True, time_major=False)
    gr = ssm.selective_scan_backward(x, delta, A, B, C, dy, tape, delta_softplus=False, time_major=False)
    wide = lambda t: np.repeat(_np(t[0])[:, None], D, axis=1)                                     # noqa: E731
    args, kw = (_np(x[0]), _np(delta[0]), _np(A), wide(B), wide(C)), dict(sp=False, dy=_np(dy[0]))
    ref, mag = R.scan(*args, **kw), R.scan(*args, mag=True, **kw)
    R.close(_np(y[0]), ref["y"], mag["y"], 16 * T + 32)
    R.close(_np(end[0]), ref["end"], mag["end"], 16 * T + 32)
    R.close(_np(gr.dx[0]), ref["dx"], mag["dx"], 32 * T + 64)
    R.close(_np(gr.dA), ref["dA"], mag["dA"], 33 * T + 64)

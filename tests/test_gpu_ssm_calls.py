"""The sequence operators and clipping as calls beside autograd, and over batches whose shape the other files leave out; values
against 64-bit forms (tolerances: tests/ssm_reference.py)."""
import numpy as np
import pytest
import torch

import ssm_reference as R
from supernnova_amd import engine as E
from supernnova_amd import ssm

pytestmark = pytest.mark.gpu


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def test_a_state_moved_on_in_place_is_not_differentiated_through():
    """The backward pass of the prompt would read the state of the token behind it."""
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=g).cuda()                                           # noqa: E731
    x, w, s, h = rnd(5, 2, 8).requires_grad_(), rnd(8, 3), rnd(2, 2, 8), rnd(2, 8, 4)
    A, bc = -rnd(8, 4).abs(), rnd(5, 2, 4)
    y, z = ssm.causal_conv(x, w, initial_state=s), ssm.selective_scan(x, x, A, bc, bc, initial_state=h)
    with torch.no_grad():
        ssm.causal_conv_step(x[0], s, w)
        ssm.selective_scan_step(x[0], h, x[0], A, bc[0], bc[0])
    for out in (y, z):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


def test_clipping_tells_autograd_what_it_wrote():
    ts = [torch.ones(5, device="cuda"), torch.ones(3, device="cuda").bfloat16()]
    out = [torch.empty_like(t) for t in ts]
    was = [t._version for t in ts + out]
    E.grad_norm(ts)
    assert [t._version for t in ts + out] == was
    E.clip_grads(ts, 1.0, out=out)
    assert [t._version for t in ts] == was[:2] and all(t._version > v for t, v in zip(out, was[2:]))
    E.clip_grads(ts, 1.0)
    assert all(t._version > v for t, v in zip(ts, was))
    flat = torch.ones(5, device="cuda")
    E.clip_coefficient(flat, 1.0)
    assert flat._version == 0


def test_small_states_that_grow_over_a_chunk():
    """A chunk of the time axis whose decays multiply to more than fp32 holds, over a state, and an adjoint, small enough that the
    product is finite: 1e-30 e^96."""
    g = torch.Generator().manual_seed(7)
    T, D, N = 400, 8, 4
    rnd = lambda *s: torch.randn(s, generator=g)                                                  # noqa: E731
    x, B, C, dy, h0 = rnd(1, T, D), rnd(1, T, N), rnd(1, T, N), rnd(1, T, D), rnd(1, D, N)
    x[:, :128] *= 1e-30
    x[:, 128:] = 0
    dy[:, :192] = 0
    dy[:, 192:] *= 1e-30
    h0 *= 1e-30
    delta = torch.full((1, T, D), -0.1)
    delta[:, :64] = 0.01
    delta[:, 128:192] = 1.5                          # 64 steps: e^96
    A = torch.ones(D, N)
    x, delta, A, B, C, dy, h0 = (t.cuda() for t in (x, delta, A, B, C, dy, h0))
    kw = dict(delta_softplus=False, initial_state=h0, time_major=False)
    y, end, tape = ssm.selective_scan_train(x, delta, A, B, C, want_final_state=True, **kw)
    gr = ssm.selective_scan_backward(x, delta, A, B, C, dy, tape, **kw)
    wide = lambda t: np.repeat(_np(t[0])[:, None], D, axis=1)                                     # noqa: E731
    args, rkw = (_np(x[0]), _np(delta[0]), _np(A), wide(B), wide(C)), dict(sp=False, h0=_np(h0[0]), dy=_np(dy[0]))
    ref, mag = R.scan(*args, **rkw), R.scan(*args, mag=True, **rkw)
    assert np.abs(ref["y"]).max() > 1e9
    k = 16 * T + 32
    R.close(_np(y[0]), ref["y"], mag["y"], k, what="y")
    R.close(_np(end[0]), ref["end"], mag["end"], k, what="end")
    for name, got in (("dx", gr.dx[0]), ("ddelta", gr.ddelta[0]), ("dh0", gr.dinitial_state[0])):
        R.close(_np(got), ref[name], mag[name], 2 * k, what=name)
    R.close(_np(gr.dA), ref["dA"], mag["dA"], 2 * k + T, what="dA")
    for name, got in (("dB", gr.dB[0]), ("dC", gr.dC[0])):
        R.close(_np(got), ref[name].sum(1), mag[name].sum(1), 2 * k + D, what=name)


@pytest.mark.parametrize("low", [-float("inf"), -3.4e38])
@pytest.mark.parametrize("T", [5, 301])
def test_decays_of_the_lowest_value(low, T):
    """exp(s A) is 0 for every step s > 0 and 1 for a step of zero of a finite A, and the steps that fill up the last segment leave
    the state as it is.  In 64 bits -1e30 says the same."""
    g = torch.Generator().manual_seed(T)
    D, N = 6, 4
    rnd = lambda *s: torch.randn(s, generator=g).cuda()                                           # noqa: E731
    x, delta, B, C, dy = rnd(1, T, D), rnd(1, T, D), rnd(1, T, N), rnd(1, T, N), rnd(1, T, D)
    A = -torch.rand(D, N, generator=g).cuda() - 0.1
    finite = A.clone()
    finite[1], finite[:, 2] = -1e30, -1e30
    A[1], A[:, 2] = low, low
    if low > -float("inf"):
        delta[:, 3] = -200.0                         # softplus: 0
    kw = dict(time_major=False)
    y, end, tape = ssm.selective_scan_train(x, delta, A, B, C, want_final_state=True, **kw)
    wide = lambda t: np.repeat(_np(t[0])[:, None], D, axis=1)                                     # noqa: E731
    args, rkw = (_np(x[0]), _np(delta[0]), _np(finite), wide(B), wide(C)), dict(dy=_np(dy[0]))
    # softplus(-200) = 1e-87 in 64 bits, and 1e-87 x 1e30 is still nothing
    ref, mag = R.scan(*args, **rkw), R.scan(*args, mag=True, **rkw)
    k = 16 * T + 32
    R.close(_np(y[0]), ref["y"], mag["y"], k, what="y")
    R.close(_np(end[0]), ref["end"], mag["end"], k, what="end")
    if low > -float("inf"):                          # the slope of exp(s A) at -inf is 0 x inf
        gr = ssm.selective_scan_backward(x, delta, A, B, C, dy, tape, **kw)
        for name, got in (("dx", gr.dx[0]), ("ddelta", gr.ddelta[0])):
            R.close(_np(got), ref[name], mag[name], 2 * k, what=name)
        R.close(_np(gr.dA), ref["dA"], mag["dA"], 2 * k + T, what="dA")
    state, want = rnd(1, D, N), None
    s0 = state.clone()
    y1 = ssm.selective_scan_step(x[:, 3], state, delta[:, 3], A, B[:, 3], C[:, 3])
    one = R.scan(*(a[3:4] if i != 2 else a for i, a in enumerate(args)), h0=_np(s0[0]))
    m1 = R.scan(*(a[3:4] if i != 2 else a for i, a in enumerate(args)), h0=_np(s0[0]), mag=True)
    R.close(_np(y1), one["y"], m1["y"], 48, what="step y")
    R.close(_np(state[0]), one["end"], m1["end"], 48, what="step end")


def _many(B, D, dt, g):
    lens = torch.randint(0, 4, (B,), generator=g)
    lens[B // 2] = 300
    off = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).cuda()
    return lens, off, torch.randn(int(off[-1]) + 7, D, generator=g).to(dt).cuda()


@pytest.mark.parametrize("B,D,dt", [(1 << 20, 1, torch.float32), (5000, 64, torch.bfloat16), (300, 20, torch.float16)])
def test_conv_of_many_sequences_without_max_len(B, D, dt):
    """The bound that max_len defaults to, the number of rows, is as good as the true one: the same bits."""
    g = torch.Generator().manual_seed(B)
    lens, off, x = _many(B, D, dt, g)
    x[off[-1]:] = float("nan")
    dy = torch.randn(x.shape, generator=g).to(dt).cuda()
    w, bias = torch.randn(D, 4, generator=g).cuda(), torch.randn(D, generator=g).cuda()
    s0, ds = torch.randn(B, 3, D, generator=g).to(dt).cuda(), torch.randn(B, 3, D, generator=g).to(dt).cuda()
    outs = []
    for max_len in (None, 300):
        y, end = ssm.causal_conv_forward(x, w, bias, offsets=off, max_len=max_len, initial_state=s0, want_final_state=True)
        gr = ssm.causal_conv_backward(x, w, bias, dy, dfinal_state=ds, offsets=off, max_len=max_len, initial_state=s0)
        outs.append([y, end, *gr])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert (outs[0][0][off[-1]:] == 0).all() and (outs[0][2][off[-1]:] == 0).all()


@pytest.mark.parametrize("dt,D,W", [("f32", 24, 4), ("bf16", 64, 3), ("f16", 7, 2)])
@pytest.mark.parametrize("max_len", [None, 150])
def test_conv_of_rows_that_are_mostly_one_sequence(dt, D, W, max_len):
    """One long sequence among short and empty ones, rows before the first and behind the last, and rows past max_len: values and
    gradients of every sequence, zeros in every row that belongs to no step."""
    g = torch.Generator().manual_seed(D)
    T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dt]
    lens, front, back = [0, 2, 200, 1, 0, 3, 0], 5, 40
    off = np.cumsum([front] + lens)
    R_ = int(off[-1]) + back
    x, dy = (torch.randn(R_, D, generator=g).to(T) for _ in range(2))
    dead = np.ones(R_, bool)
    for b, n in enumerate(lens):
        dead[off[b]:off[b] + min(n, max_len or n)] = False
    x[dead], dy[dead] = float("nan"), float("nan")
    x, dy, w, bias = x.cuda(), dy.cuda(), torch.randn(D, W, generator=g).cuda(), torch.randn(D, generator=g).cuda()
    s0, ds = (torch.randn(len(lens), W - 1, D, generator=g).to(T).cuda() for _ in range(2))
    kw = dict(offsets=torch.tensor(off).cuda(), max_len=max_len, initial_state=s0)
    y, end = ssm.causal_conv_forward(x, w, bias, want_final_state=True, **kw)
    gr = ssm.causal_conv_backward(x, w, bias, dy, dfinal_state=ds, **kw)
    assert (_np(y)[dead] == 0).all() and (_np(gr.dx)[dead] == 0).all()
    k, parts, mags = W + 16, [], []
    for b, n in enumerate(lens):
        at = slice(off[b], off[b] + min(n, max_len or n))
        a = (_np(x)[at], _np(w), _np(bias), True, _np(s0[b]), _np(dy)[at], _np(ds[b]))
        r, m = R.conv(*a), R.conv(*a, mag=True)
        R.close(_np(y)[at], r["y"], m["y"], k, dt, "y")
        R.close(_np(end[b]), r["end"], m["end"], 0, dt, "end")
        R.close(_np(gr.dx)[at], r["dx"], m["dx"], 2 * k, dt, "dx")
        R.close(_np(gr.dinitial_state[b]), r["ds0"], m["ds0"], 2 * k, dt, "ds0")
        parts.append(r)
        mags.append(m)
    for name, got in (("dw", gr.dweight), ("db", gr.dbias)):       # a chunk's at most 16 steps in fp32, chunks of a slot, then fp64
        R.close(_np(got), sum(p[name] for p in parts), sum(p[name] for p in mags), 2 * k + 16 + 32, "f32", name)

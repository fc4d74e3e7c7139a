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

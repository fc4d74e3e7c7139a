"""Selective scan, causal convolution, clipping without a GPU: the written-out gradients the GPU tests compare with, against
differences; argument checks of the host layer and of the C ABI (which launch nothing)."""
import ctypes

import numpy as np
import pytest
import torch

import ssm_reference as R
from supernnova_amd import _lib as L
from supernnova_amd import engine as E
from supernnova_amd import optim, ssm


def _differences(f, args, names, grads, dy, dend, rng):
    """Central differences of sum(dy y) + sum(dend end) along a random direction of every argument."""
    val = lambda a: sum(float((d * o).sum()) for d, o in zip((dy, dend), f(a)) if d is not None)      # noqa: E731
    for n in names:
        v = rng.standard_normal(args[n].shape)
        eps = 1e-5
        hi, lo = dict(args), dict(args)
        hi[n], lo[n] = args[n] + eps * v, args[n] - eps * v
        num = (val(hi) - val(lo)) / (2 * eps)
        ana = float((grads[n] * v).sum())
        # the difference is off by eps^2 / 6 of the third derivative (1e-6 covers 1e4 of it) and by the roundings of the two
        # values, each at most some 64 times 2^-53 of the terms' magnitudes M, divided by 2 eps: without softplus steps may be
        # negative, states then grow like exp(|s A|) per step, and M is not O(1)
        M = sum(float(np.abs(d * o).sum()) for d, o in zip((dy, dend), f(args)) if d is not None)
        assert abs(num - ana) <= 1e-6 * max(1.0, abs(ana)) + 64 * 2.0 ** -53 * M / eps, (n, num, ana, M)


@pytest.mark.parametrize("W,silu,T", [(2, True, 1), (3, False, 5), (4, True, 9), (4, True, 2)])
def test_conv_reference_gradients_against_differences(W, silu, T):
    g = np.random.default_rng(W * 10 + T)
    D = 3
    a = {"x": g.standard_normal((T, D)), "w": g.standard_normal((D, W)), "b": g.standard_normal(D), "s0": g.standard_normal((W - 1, D))}
    dy, ds = g.standard_normal((T, D)), g.standard_normal((W - 1, D))
    o = R.conv(a["x"], a["w"], a["b"], silu, a["s0"], dy, ds)

    def f(q):
        r = R.conv(q["x"], q["w"], q["b"], silu, q["s0"])
        return r["y"], r["end"]
    _differences(f, a, list(a), {"x": o["dx"], "w": o["dw"], "b": o["db"], "s0": o["ds0"]}, dy, ds, g)


@pytest.mark.parametrize("gate,sp,T", [(True, True, 6), (False, True, 1), (True, False, 4)])
def test_scan_reference_gradients_against_differences(gate, sp, T):
    g = np.random.default_rng(T)
    D, N = 3, 4
    a = {"x": g.standard_normal((T, D)), "delta": g.standard_normal((T, D)), "A": -g.uniform(0.3, 2, (D, N)), "B": g.standard_normal((T, D, N)),
         "C": g.standard_normal((T, D, N)), "skip": g.standard_normal(D), "dbias": g.standard_normal(D), "h0": g.standard_normal((D, N))}
    if gate:
        a["z"] = g.standard_normal((T, D))
    dy, de = g.standard_normal((T, D)), g.standard_normal((D, N))
    o = R.scan(**a, sp=sp, dy=dy, dend=de)
    names = {"x": "dx", "delta": "ddelta", "A": "dA", "B": "dB", "C": "dC", "skip": "dskip", "dbias": "ddbias", "h0": "dh0", "z": "dz"}

    def f(q):
        r = R.scan(**q, sp=sp)
        return r["y"], r["end"]
    _differences(f, a, list(a), {k: o[names[k]] for k in a}, dy, de, g)


def test_host_layer_refuses_cpu_tensors():
    x, w = torch.zeros(3, 2, 4), torch.zeros(4, 3)
    with pytest.raises(L.SnnError, match="HIP device"):
        ssm.causal_conv_forward(x, w)
    with pytest.raises(L.SnnError, match="HIP device"):
        ssm.causal_conv_step(x[0], torch.zeros(2, 2, 4), w)
    bc = torch.zeros(3, 2, 5)
    with pytest.raises(L.SnnError, match="HIP device"):
        ssm.selective_scan(x, x, torch.zeros(4, 5), bc, bc)
    with pytest.raises(L.SnnError, match="HIP device"):
        E.clip_grads([x], 1.0)
    with pytest.raises(L.SnnError, match="no gradients"):
        E.grad_norm([])
    with pytest.raises(L.SnnError, match="norm_type"):
        E.grad_norm([x], 3)


def test_clip_of_no_gradients_is_zero():
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(optim.clip_grad_norm_([p], 1.0)) == 0.0


def test_dense_blocks():
    t = torch.zeros(4, 6)
    assert E._dense(t) and E._dense(t.t()) and E._dense(t[1:]) and E._dense(torch.zeros(3, 1, 2).transpose(0, 2))
    assert not E._dense(t[:, :3]) and not E._dense(torch.zeros(3, 1).expand(3, 4))


def _err():
    return L.load().snn_last_error().decode()


def test_c_abi_conv_refusals():
    lib = L.load()
    a = L.SnnConvArgs()
    assert lib.snn_conv_forward(None, None) == -1
    assert lib.snn_conv_forward(ctypes.byref(a), None) == -1 and "positive" in _err()
    a.seq = L.SnnSeq(2, 3, 0, None, None)
    a.channels, a.width = 4, 5
    assert lib.snn_conv_forward(ctypes.byref(a), None) == -2
    a.width = 4
    assert lib.snn_conv_forward(ctypes.byref(a), None) == -1 and "null" in _err()
    assert lib.snn_conv_step(ctypes.byref(a), None) == -1
    assert lib.snn_conv_workspace_bytes(ctypes.byref(a)) > 0
    a.dtype = 7
    assert lib.snn_conv_backward(ctypes.byref(a), None) == -2
    a.dtype, a.seq = 0, L.SnnSeq(2, 3, 0, 16, 16)
    assert lib.snn_conv_forward(ctypes.byref(a), None) == -1 and "exclude" in _err()


def test_c_abi_scan_refusals():
    lib = L.load()
    a = L.SnnScanArgs()
    assert lib.snn_scan_forward(None, None) == -1
    assert lib.snn_scan_forward(ctypes.byref(a), None) == -1
    a.seq = L.SnnSeq(2, 300, 0, None, None)
    a.channels, a.groups, a.states = 6, 4, 16
    assert lib.snn_scan_forward(ctypes.byref(a), None) == -1          # 4 does not divide 6
    a.groups, a.states = 2, 65
    assert lib.snn_scan_step(ctypes.byref(a), None) == -2
    a.states = 16
    assert lib.snn_scan_forward(ctypes.byref(a), None) == -1 and "null" in _err()
    assert lib.snn_scan_backward(ctypes.byref(a), None) == -1 and "null" in _err()
    v = L.SnnView(4096, 12, 6)                                        # never touched: the workspace check comes first
    for k in ("x", "delta", "B", "C", "y", "dy", "dx", "ddelta", "dB", "dC"):
        setattr(a, k, v)
    a.A, a.dA, a.tape, a.ws = 4096, 4096, 4096, 4096
    assert lib.snn_scan_workspace_bytes(ctypes.byref(a), 0) > 0       # 2 sequences x 2 blocks: the time axis is split
    assert lib.snn_scan_forward(ctypes.byref(a), None) == -3
    a.tape_floats = lib.snn_scan_tape_floats(ctypes.byref(a))
    assert a.tape_floats > 0
    assert lib.snn_scan_backward(ctypes.byref(a), None) == -3
    a.tape = 4100
    assert lib.snn_scan_backward(ctypes.byref(a), None) == -1 and "misaligned" in _err()


def test_c_abi_clip_refusals():
    lib = L.load()
    one = (ctypes.c_int64 * 1)(5)
    assert lib.snn_clip_scratch_doubles(1, one) == 1
    assert lib.snn_clip_scratch_doubles(1, (ctypes.c_int64 * 1)(-1)) == -1
    assert lib.snn_clip_scratch_doubles(1, (ctypes.c_int64 * 1)(1 << 50)) == -2
    p, dt = (ctypes.c_void_p * 1)(4096), (ctypes.c_int32 * 1)(0)
    assert lib.snn_clip_grads(1, p, None, one, dt, 2, 1.0, 1.0, None, 4096, 1, None) == -1
    assert lib.snn_clip_grads(1, p, None, one, dt, 3, 1.0, 1.0, 4096, 4096, 1, None) == -1
    assert lib.snn_clip_grads(1, p, None, one, dt, 2, 1.0, 1.0, 4096, 4096, 0, None) == -3
    assert lib.snn_clip_grads(1, p, None, one, (ctypes.c_int32 * 1)(9), 2, 1.0, 1.0, 4096, 4096, 1, None) == -1
    assert lib.snn_clip_grads(1, p, (ctypes.c_void_p * 1)(None), one, dt, 2, 1.0, 1.0, 4096, 4096, 1, None) == -1
    assert lib.snn_adam_step_clipped(1, 1, 1, 1, 1, 1, 0, 0, 0, 0, 0, 1, None, None) == -1
    assert lib.snn_sgd_step_clipped(1, 1, 1, 1, 1, 0, 0, 0, 1, None, None) == -1


def test_autograd_is_refused_while_capturing(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    x = torch.zeros(3, 2, 4, requires_grad=True)
    with pytest.raises(L.SnnError, match="captured"):
        ssm.causal_conv(x, torch.zeros(4, 3))
    with pytest.raises(L.SnnError, match="captured"):
        ssm.selective_scan(x, x, torch.zeros(4, 5), torch.zeros(3, 2, 5), torch.zeros(3, 2, 5))


def test_c_abi_refuses_sizes_beyond_the_grids():
    lib = L.load()
    for n, t, d in ((1 << 24, 4, 8), (1, (1 << 30) + 1, 8), (1, 4, (1 << 19) + 1)):
        a = L.SnnConvArgs(seq=L.SnnSeq(n, t, 0, None, None), channels=d, width=4)
        assert lib.snn_conv_forward(ctypes.byref(a), None) == -2 and "at most" in _err()
        assert lib.snn_conv_workspace_bytes(ctypes.byref(a)) == -2
        b = L.SnnScanArgs(seq=L.SnnSeq(n, t, 0, None, None), channels=d, groups=1, states=16)
        assert lib.snn_scan_forward(ctypes.byref(b), None) == -2 and "at most" in _err()
        assert lib.snn_scan_tape_floats(ctypes.byref(b)) == -2
    v = L.SnnView(4096, 0, 3)                  # one step of more sequences x channels than a grid of single channels holds
    a = L.SnnConvArgs(seq=L.SnnSeq((1 << 24) - 1, 1, 0, None, None), channels=257, width=2, x=v, y=v, weight=4096, state_in=4096, state_out=4096)
    assert lib.snn_conv_step(ctypes.byref(a), None) == -2 and "workgroups" in _err()


def test_c_abi_clip_refuses_overlaps():
    """Addresses only: nothing is launched."""
    lib = L.load()

    def clip(src, dst, numel, dtype):
        n = len(src)
        arr = lambda t, v: (t * n)(*v)                                                            # noqa: E731
        return lib.snn_clip_grads(n, arr(ctypes.c_void_p, src), arr(ctypes.c_void_p, dst), arr(ctypes.c_int64, numel), arr(ctypes.c_int32, dtype),
                                  2, 1.0, 1.0, 4096, 4096, 64, None)
    a, b = 1 << 20, 2 << 20
    assert clip([a, a + 16], [a, a + 16], [5, 5], [0, 0]) == -1 and "twice" in _err()           # 20 bytes at a
    assert clip([a, a + 8], [a, a + 8], [5, 5], [1, 1]) == -1 and "twice" in _err()             # 10 bytes at a
    assert clip([a, b], [b, a], [5, 5], [0, 0]) == -1 and "another gradient" in _err()
    assert clip([a, b], [a, a + 40], [20, 5], [0, 0]) == -1 and "twice" in _err()               # inside a longer one
    assert clip([a], [a + 4], [5], [0]) == -1 and "in part" in _err()
    assert clip([a, b], [b + 64, b + 20 - 4], [5, 5], [0, 0]) == -1 and "in part" in _err()

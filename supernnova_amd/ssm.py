"""Selective state space scan and the short causal convolution in front of it: host layer over snn_scan_* and snn_conv_*
(include/snn_hip.h), beside engine.py's LSTM / GRU / RNN stack.  No counterpart in the reference.

    convolution   y_t = silu(bias + sum_w weight[:, w] x_{t - W + 1 + w})                        per channel, W = 2 .. 4
    scan          s_t = softplus(delta_t + delta_bias)
                  h_t = exp(s_t A) h_{t-1} + s_t x_t B_t ;  y_t = (C_t . h_t + D x_t) silu(z_t)  per channel, N = 1 .. 64 states

Three layouts, as the rest of the package takes its batches; D channels are always the last, unit-stride dimension, the others
may be strided (a slice of a wider projection needs no copy):
    (T, B, D)  time_major=True (default), padded, `lengths` int32 (B,) on the device or None
    (B, T, D)  time_major=False, padded, `lengths` likewise
    (R, D)     ragged rows, `offsets` int64 (B + 1,) on the device: sequence b holds rows offsets[b] .. offsets[b + 1];
               `max_len`: a bound on the lengths known to the host (default: the number of rows; a good one saves workspace)
Rows that belong to no step (behind a sequence's end, outside every sequence, past max_len) are never read, and zero in every
output.  A sequence of length 0 hands its initial state on.  Lengths and offsets stay on the device (no synchronisation);
values out of range are cut to the tensors.

x, delta, z, B, C and what has their shape are float32, bfloat16 or float16, one type per call; parameters, their gradients and
scan states are float32, sums and states are held in float32, and results are rounded once.  B and C are (.., N) or, with
groups of channels that share them, (.., G, N).  States: convolution (B, W - 1, D), the last inputs; scan (B, D, N).

Two levels, as engine.py / modules.py: `*_forward`, `*_train`, `*_backward`, `*_step` launch kernels on the current stream and can
be captured into a graph; `causal_conv` and `selective_scan` are their differentiable forms.  The latter refuse to record or run
a backward pass while a stream is being captured (autograd would accumulate on the streams of whatever graph the leaves were
in before): capture the explicit pair.  The step functions write the state in place unless given `new_state`.
"""
import ctypes
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import engine as E

_NONE = L.SnnView(None, 0, 0)


class ConvGrads(NamedTuple):
    dx: torch.Tensor
    dweight: torch.Tensor
    dbias: Optional[torch.Tensor]
    dinitial_state: Optional[torch.Tensor]


class ScanGrads(NamedTuple):
    dx: torch.Tensor
    ddelta: torch.Tensor
    dA: torch.Tensor
    dB: torch.Tensor
    dC: torch.Tensor
    dD: Optional[torch.Tensor]
    dz: Optional[torch.Tensor]
    ddelta_bias: Optional[torch.Tensor]
    dinitial_state: Optional[torch.Tensor]


def _fail(msg):
    raise L.SnnError(msg)


def _param(t, name, shape, device):
    """A contiguous float32 parameter or state -> its address (None stays None)."""
    if t is None:
        return None
    E._require_cuda(t, name)
    if t.shape != shape or t.device != device:
        _fail(f"{name} must be {tuple(shape)} on {device}, got {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


class _Batch:
    """The layout of one call: sequences, steps, and the strides of a tensor's step and sequence dimensions."""

    def __init__(self, x, lengths, offsets, max_len, time_major):
        if not x.is_cuda:
            _fail("x must live on a HIP device: supernnova_amd runs only on the GPU (no CPU fallback)")
        if x.dtype not in E._DTYPES:
            _fail(f"x must be float32, bfloat16 or float16, got {x.dtype}")
        self.dtype, self.device, self.D = x.dtype, x.device, x.size(-1) if x.dim() else 0
        if offsets is not None:
            if x.dim() != 2:
                _fail(f"ragged rows must be (rows, channels), got {tuple(x.shape)}")
            if lengths is not None:
                _fail("lengths and offsets exclude each other")
            self._index(offsets, "offsets", torch.int64, None)
            self.B, rows = offsets.numel() - 1, x.size(0)
            self.T = rows if max_len is None else min(int(max_len), rows)
            self.t_dim, self.n_dim, lead = 0, None, 1
        else:
            if x.dim() != 3:
                _fail(f"x must be 3-D (or 2-D rows with offsets), got {tuple(x.shape)}")
            if max_len is not None:
                _fail("max_len goes with offsets")
            self.t_dim, self.n_dim = (0, 1) if time_major else (1, 0)
            self.T, self.B, rows, lead = x.size(self.t_dim), x.size(self.n_dim), 0, 2
            if lengths is not None:
                self._index(lengths, "lengths", torch.int32, self.B)
        self.lead = x.shape[:lead]
        if self.T < 1 or self.B < 1 or self.D < 1:
            _fail(f"need at least one sequence, one step and one channel, got x {tuple(x.shape)}, {self.B} sequences, {self.T} steps")
        if max(self.T, self.B, self.D) >= 1 << 31:
            _fail("sizes must fit 31 bits")
        self.seq = L.SnnSeq(self.B, self.T, rows, None if lengths is None else lengths.data_ptr(),
                            None if offsets is None else offsets.data_ptr())

    def _index(self, t, name, dtype, n):
        if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous() or t.device != self.device or t.numel() < 1 or (n is not None and t.numel() != n):
            _fail(f"{name} must be a contiguous {dtype} vector{'' if n is None else f' of {n}'} on {self.device}")

    def view(self, t, name, shape=None):
        """A tensor of the batch (default: of x's shape) as snn_view."""
        if t.dtype != self.dtype or t.device != self.device or t.shape != (self.lead + (self.D,) if shape is None else shape):
            _fail(f"{name} must be {self.dtype} {tuple(self.lead + (self.D,) if shape is None else shape)} on {self.device}, "
                  f"got {t.dtype} {tuple(t.shape)} on {t.device}")
        if t.stride(-1) != 1 and t.size(-1) != 1:
            _fail(f"{name}: the last dimension must have unit stride")
        return L.SnnView(t.data_ptr(), t.stride(self.t_dim), 0 if self.n_dim is None else t.stride(self.n_dim))

    def out(self, t):
        return L.SnnView(t.data_ptr(), t.stride(self.t_dim), 0 if self.n_dim is None else t.stride(self.n_dim))

    def empty(self, *tail):
        return torch.empty(self.lead + (tail or (self.D,)), dtype=self.dtype, device=self.device)


class _Step(_Batch):
    """One step of B sequences: x (B, D)."""

    def __init__(self, x):
        if not x.is_cuda:
            _fail("x must live on a HIP device: supernnova_amd runs only on the GPU (no CPU fallback)")
        if x.dtype not in E._DTYPES or x.dim() != 2 or x.numel() < 1:
            _fail(f"x must be a non-empty (sequences, channels) tensor of float32, bfloat16 or float16, got {x.dtype} {tuple(x.shape)}")
        self.dtype, self.device = x.dtype, x.device
        self.B, self.D = x.shape
        self.T, self.t_dim, self.n_dim, self.lead = 1, 0, 0, x.shape[:1]
        self.seq = L.SnnSeq(self.B, 1, 0, None, None)


def _unit(t):
    """Gradients arrive with whatever strides autograd chose (an expanded sum has none): rows of unit stride."""
    return t if t.stride(-1) == 1 else t.contiguous()


# ------------------------------------------------------------------------------------------------- convolution
def _conv_args(bt, x, weight, bias, activation, state, state_name="initial_state"):
    if activation not in ("silu", None):
        _fail(f"activation must be 'silu' or None, got {activation!r}")
    if weight.dim() != 2 or not 2 <= weight.size(1) <= 4:
        _fail(f"weight must be (channels, 2..4), got {tuple(weight.shape)}")
    W = weight.size(1)
    a = L.SnnConvArgs(seq=bt.seq, dtype=E._DTYPES[bt.dtype], channels=bt.D, width=W, silu=activation == "silu")
    a.x = bt.view(x, "x")
    a.weight = _param(weight, "weight", (bt.D, W), bt.device)
    a.bias = _param(bias, "bias", (bt.D,), bt.device)
    a.state_in = _conv_state(bt, state, state_name, W)
    return a, W


def _conv_state(bt, t, name, W):
    if t is None:
        return None
    if t.dtype != bt.dtype or t.shape != (bt.B, W - 1, bt.D) or t.device != bt.device or not t.is_contiguous():
        _fail(f"{name} must be contiguous {bt.dtype} {(bt.B, W - 1, bt.D)} on {bt.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _launch(fn, what, a, device):
    with E._on_device(device):
        L.check(fn(ctypes.byref(a), E._stream()), what)


def causal_conv_forward(x, weight, bias=None, *, activation="silu", lengths=None, offsets=None, max_len=None,
                        initial_state=None, want_final_state=False, time_major=True):
    """Depthwise causal convolution of a batch of sequences: weight (D, W) with weight[:, -1] on the current step, bias (D,) or
    None, activation "silu" or None.  Returns (y like x, final state (B, W - 1, D) or None); the final state is what
    causal_conv_step and a later call's initial_state go on from."""
    bt = _Batch(x, lengths, offsets, max_len, time_major)
    a, W = _conv_args(bt, x, weight, bias, activation, initial_state)
    y = bt.empty()
    a.y = bt.out(y)
    end = None
    if want_final_state:
        end = torch.empty((bt.B, W - 1, bt.D), dtype=bt.dtype, device=bt.device)
        a.state_out = end.data_ptr()
    _launch(L.load().snn_conv_forward, "snn_conv_forward", a, bt.device)
    return y, end


def causal_conv_backward(x, weight, bias, dy, *, dfinal_state=None, activation="silu", lengths=None, offsets=None, max_len=None,
                         initial_state=None, time_major=True):
    """Gradients of causal_conv_forward's result from dy = dloss/dy and, if the final state was used, dfinal_state.  Sums over
    sequences and steps are taken in an order that depends on the sizes alone."""
    bt = _Batch(x, lengths, offsets, max_len, time_major)
    a, W = _conv_args(bt, x, weight, bias, activation, initial_state)
    dy = _unit(dy)
    a.dy = bt.view(dy, "dy")
    a.dstate_out = _conv_state(bt, dfinal_state, "dfinal_state", W)
    dx = bt.empty()
    a.dx = bt.out(dx)
    dpar = torch.empty(bt.D * (W + 1), dtype=torch.float32, device=bt.device)
    a.dweight = dpar.data_ptr()
    if bias is not None:
        a.dbias = a.dweight + 4 * bt.D * W
    dstate = None
    if initial_state is not None:
        dstate = torch.empty_like(initial_state)
        a.dstate_in = dstate.data_ptr()
    lib = L.load()
    ws = torch.empty(L.check(lib.snn_conv_workspace_bytes(ctypes.byref(a)), "snn_conv_workspace_bytes"), dtype=torch.uint8, device=bt.device)
    a.ws, a.ws_bytes = ws.data_ptr(), ws.numel()
    _launch(lib.snn_conv_backward, "snn_conv_backward", a, bt.device)
    return ConvGrads(dx, dpar[:bt.D * W].view(bt.D, W), dpar[bt.D * W:] if bias is not None else None, dstate)


def causal_conv_step(x, state, weight, bias=None, *, activation="silu", new_state=None):
    """The convolution's output for one new input x (B, D) of every sequence; `state` (B, W - 1, D) holds the inputs before
    it and is moved on in place, or left as it is and its successor written to `new_state`."""
    bt = _Step(x)
    if state is None:
        _fail("causal_conv_step needs the state")
    a, W = _conv_args(bt, x, weight, bias, activation, state, "state")
    a.state_out = a.state_in if new_state is None else _conv_state(bt, new_state, "new_state", W)
    y = bt.empty()
    a.y = bt.out(y)
    _launch(L.load().snn_conv_step, "snn_conv_step", a, bt.device)
    return y


# ------------------------------------------------------------------------------------------------- scan
def _scan_args(bt, x, delta, A, B, C, D, z, delta_bias, delta_softplus, state, state_name="initial_state"):
    if A.dim() != 2 or not 1 <= A.size(1) <= 64:
        _fail(f"A must be (channels, 1..64), got {tuple(A.shape)}")
    N, lead = A.size(1), len(bt.lead)
    if B.dim() not in (lead + 1, lead + 2) or B.shape != C.shape:
        _fail(f"B and C must be alike, (.., states) or (.., groups, states), got {tuple(B.shape)} and {tuple(C.shape)}")
    G = B.size(-2) if B.dim() == lead + 2 else 1
    if G < 1 or bt.D % G:
        _fail(f"{bt.D} channels cannot be dealt to {G} groups")
    shape = bt.lead + ((G, N) if B.dim() == lead + 2 else (N,))
    a = L.SnnScanArgs(seq=bt.seq, dtype=E._DTYPES[bt.dtype], channels=bt.D, states=N, groups=G, softplus=bool(delta_softplus))
    a.x, a.delta = bt.view(x, "x"), bt.view(delta, "delta")
    a.z = _NONE if z is None else bt.view(z, "z")
    a.B, a.C = bt.view(B, "B", shape), bt.view(C, "C", shape)
    if G > 1:
        a.B_stride_g, a.C_stride_g = B.stride(-2), C.stride(-2)
    a.A = _param(A, "A", (bt.D, N), bt.device)
    a.skip = _param(D, "D", (bt.D,), bt.device)
    a.delta_bias = _param(delta_bias, "delta_bias", (bt.D,), bt.device)
    a.state_in = _param(state, state_name, (bt.B, bt.D, N), bt.device)
    return a, G, N


def _scan_forward(x, delta, A, B, C, D, z, delta_bias, delta_softplus, lengths, offsets, max_len, initial_state, want_final_state,
                  time_major, want_tape):
    bt = _Batch(x, lengths, offsets, max_len, time_major)
    a, _, N = _scan_args(bt, x, delta, A, B, C, D, z, delta_bias, delta_softplus, initial_state)
    y = bt.empty()
    a.y = bt.out(y)
    end = tape = None
    if want_final_state:
        end = torch.empty((bt.B, bt.D, N), dtype=torch.float32, device=bt.device)
        a.state_out = end.data_ptr()
    lib = L.load()
    if want_tape:
        tape = torch.empty(L.check(lib.snn_scan_tape_floats(ctypes.byref(a)), "snn_scan_tape_floats"), dtype=torch.float32, device=bt.device)
        a.tape, a.tape_floats = tape.data_ptr(), tape.numel()
    need = L.check(lib.snn_scan_workspace_bytes(ctypes.byref(a), 0), "snn_scan_workspace_bytes")
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=bt.device)
        a.ws, a.ws_bytes = ws.data_ptr(), need
    _launch(lib.snn_scan_forward, "snn_scan_forward", a, bt.device)
    return y, end, tape


def selective_scan_forward(x, delta, A, B, C, D=None, z=None, delta_bias=None, *, delta_softplus=True, lengths=None, offsets=None,
                           max_len=None, initial_state=None, want_final_state=False, time_major=True):
    """The scan over a batch of sequences (module docstring).  A (D, N); B, C (.., [G,] N); D, delta_bias (D,) or None; z like x
    or None.  Returns (y like x, final state (B, D, N) or None)."""
    return _scan_forward(x, delta, A, B, C, D, z, delta_bias, delta_softplus, lengths, offsets, max_len, initial_state,
                         want_final_state, time_major, False)[:2]


def selective_scan_train(x, delta, A, B, C, D=None, z=None, delta_bias=None, *, delta_softplus=True, lengths=None, offsets=None,
                         max_len=None, initial_state=None, want_final_state=False, time_major=True):
    """selective_scan_forward that also returns the tape selective_scan_backward starts from: (y, final state or None, tape).
    The tape holds a state every 16 / 8 / 4 steps for up to 8 / 16 / 64 states."""
    return _scan_forward(x, delta, A, B, C, D, z, delta_bias, delta_softplus, lengths, offsets, max_len, initial_state,
                         want_final_state, time_major, True)


def selective_scan_backward(x, delta, A, B, C, dy, tape, D=None, z=None, delta_bias=None, *, dfinal_state=None, delta_softplus=True,
                            lengths=None, offsets=None, max_len=None, initial_state=None, time_major=True):
    """Gradients from dy = dloss/dy and, if the final state was used, dfinal_state, with the tape of selective_scan_train over the
    same inputs.  Every sum is taken in an order that depends on the sizes alone."""
    bt = _Batch(x, lengths, offsets, max_len, time_major)
    a, G, N = _scan_args(bt, x, delta, A, B, C, D, z, delta_bias, delta_softplus, initial_state)
    dev, Dm = bt.device, bt.D
    dy = _unit(dy)
    a.dy = bt.view(dy, "dy")
    a.dstate_out = _param(dfinal_state, "dfinal_state", (bt.B, Dm, N), dev)
    E._require_cuda(tape, "tape")
    a.tape, a.tape_floats = tape.data_ptr(), tape.numel()
    dx, ddelta = bt.empty(), bt.empty()
    a.dx, a.ddelta = bt.out(dx), bt.out(ddelta)
    dz = None
    if z is not None:
        dz = bt.empty()
        a.dz = bt.out(dz)
    dB, dC = bt.empty(*B.shape[len(bt.lead):]), bt.empty(*C.shape[len(bt.lead):])
    a.dB, a.dC = bt.out(dB), bt.out(dC)
    dpar = torch.empty(Dm * (N + 2), dtype=torch.float32, device=dev)
    a.dA = dpar.data_ptr()
    if D is not None:
        a.dskip = a.dA + 4 * Dm * N
    if delta_bias is not None:
        a.ddelta_bias = a.dA + 4 * Dm * (N + 1)
    dstate = None
    if initial_state is not None:
        dstate = torch.empty_like(initial_state)
        a.dstate_in = dstate.data_ptr()
    lib = L.load()
    ws = torch.empty(L.check(lib.snn_scan_workspace_bytes(ctypes.byref(a), 1), "snn_scan_workspace_bytes"), dtype=torch.uint8, device=dev)
    a.ws, a.ws_bytes = ws.data_ptr(), ws.numel()
    _launch(lib.snn_scan_backward, "snn_scan_backward", a, dev)
    return ScanGrads(dx, ddelta, dpar[:Dm * N].view(Dm, N), dB, dC, dpar[Dm * N:Dm * (N + 1)] if D is not None else None, dz,
                     dpar[Dm * (N + 1):] if delta_bias is not None else None, dstate)


def selective_scan_step(x, state, delta, A, B, C, D=None, z=None, delta_bias=None, *, delta_softplus=True, new_state=None):
    """One step of every sequence: x, delta, z (B, D), B, C (B, [G,] N); `state` (B, D, N) float32 is moved on in place, or left as
    it is and its successor written to `new_state`.  Returns y (B, D)."""
    bt = _Step(x)
    if state is None:
        _fail("selective_scan_step needs the state")
    a, _, N = _scan_args(bt, x, delta, A, B, C, D, z, delta_bias, delta_softplus, state, "state")
    a.state_out = a.state_in if new_state is None else _param(new_state, "new_state", (bt.B, bt.D, N), bt.device)
    y = bt.empty()
    a.y = bt.out(y)
    _launch(L.load().snn_scan_step, "snn_scan_step", a, bt.device)
    return y


# ------------------------------------------------------------------------------------------------- differentiable forms
def _not_captured():
    if torch.cuda.is_current_stream_capturing():
        _fail("a backward pass through autograd cannot be captured into a graph here: capture the *_train / *_forward and *_backward "
              "calls of supernnova_amd.ssm")


class _ConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial_state, opt, want_final_state):
        _not_captured()
        y, end = causal_conv_forward(x, weight, bias, initial_state=initial_state, want_final_state=want_final_state, **opt)
        ctx.save_for_backward(x, weight, bias, initial_state, opt.get("lengths"), opt.get("offsets"))
        ctx.opt = {k: v for k, v in opt.items() if k not in ("lengths", "offsets")}
        ctx.set_materialize_grads(False)
        return y, end

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dend):
        _not_captured()
        x, weight, bias, state, lengths, offsets = ctx.saved_tensors
        dy = torch.zeros_like(x) if dy is None else dy
        g = causal_conv_backward(x, weight, bias, dy, dfinal_state=None if dend is None else dend.contiguous(), initial_state=state,
                                 lengths=lengths, offsets=offsets, **ctx.opt)
        return g.dx, g.dweight, g.dbias, g.dinitial_state, None, None


class _ScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, A, B, C, D, z, delta_bias, initial_state, opt, want_final_state):
        _not_captured()
        y, end, tape = selective_scan_train(x, delta, A, B, C, D, z, delta_bias, initial_state=initial_state,
                                            want_final_state=want_final_state, **opt)
        ctx.save_for_backward(x, delta, A, B, C, D, z, delta_bias, initial_state, tape, opt.get("lengths"), opt.get("offsets"))
        ctx.opt = {k: v for k, v in opt.items() if k not in ("lengths", "offsets")}
        ctx.set_materialize_grads(False)
        return y, end

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dend):
        _not_captured()
        x, delta, A, B, C, D, z, delta_bias, state, tape, lengths, offsets = ctx.saved_tensors
        dy = torch.zeros_like(x) if dy is None else dy
        g = selective_scan_backward(x, delta, A, B, C, dy, tape, D, z, delta_bias, dfinal_state=None if dend is None else dend.contiguous(),
                                    initial_state=state, lengths=lengths, offsets=offsets, **ctx.opt)
        return g.dx, g.ddelta, g.dA, g.dB, g.dC, g.dD, g.dz, g.ddelta_bias, g.dinitial_state, None, None


def _needs_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def causal_conv(x, weight, bias=None, *, activation="silu", lengths=None, offsets=None, max_len=None, initial_state=None,
                return_final_state=False, time_major=True):
    """Differentiable causal_conv_forward: y, or (y, final state) with return_final_state."""
    opt = dict(activation=activation, lengths=lengths, offsets=offsets, max_len=max_len, time_major=time_major)
    if _needs_grad(x, weight, bias, initial_state):
        y, end = _ConvFn.apply(x, weight, bias, initial_state, opt, return_final_state)
    else:
        y, end = causal_conv_forward(x, weight, bias, initial_state=initial_state, want_final_state=return_final_state, **opt)
    return (y, end) if return_final_state else y


def selective_scan(x, delta, A, B, C, D=None, z=None, delta_bias=None, *, delta_softplus=True, lengths=None, offsets=None, max_len=None,
                   initial_state=None, return_final_state=False, time_major=True):
    """Differentiable selective_scan_forward: y, or (y, final state) with return_final_state."""
    opt = dict(delta_softplus=delta_softplus, lengths=lengths, offsets=offsets, max_len=max_len, time_major=time_major)
    if _needs_grad(x, delta, A, B, C, D, z, delta_bias, initial_state):
        y, end = _ScanFn.apply(x, delta, A, B, C, D, z, delta_bias, initial_state, opt, return_final_state)
    else:
        y, end = selective_scan_forward(x, delta, A, B, C, D, z, delta_bias, initial_state=initial_state,
                                        want_final_state=return_final_state, **opt)
    return (y, end) if return_final_state else y

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
               `max_len`: a bound on the lengths known to the host (default: the number of rows; the scan cuts the time axis by it
               as if all sequences were that long: a loose one, or one long sequence among many short ones, costs time)
Rows that belong to no step (behind a sequence's end, outside every sequence, past max_len) are never read, and zero in every
output.  A sequence of length 0 hands its initial state on.  Lengths and offsets stay on the device (no synchronisation);
values out of range are cut to the tensors.  Offsets must not decrease: the results of a batch whose offsets do are not defined.

x, delta, z, B, C and what has their shape are float32, bfloat16 or float16, one type per call; parameters, their gradients and
scan states are float32, sums and states are held in float32, and results are rounded once.  B and C are (.., N) or, with
groups of channels that share them, (.., G, N).  States: convolution (B, W - 1, D), the last inputs; scan (B, D, N).

Two levels, as engine.py / modules.py: `*_forward`, `*_train`, `*_backward`, `*_step` launch kernels on the current stream and can
be captured into a graph; `causal_conv` and `selective_scan` are their differentiable forms.  The latter refuse to record or run
a backward pass while a stream is being captured (autograd would accumulate on the streams of whatever graph the leaves were
in before): capture the explicit pair.  Results of the explicit calls carry no history, whatever their arguments require.  The
step functions write the state in place unless given `new_state`, and refuse to write one that requires grad.  Forward-mode
differentiation and torch.jit.trace, which would lose tangents and launches without a word, are refused.
"""
import ctypes
import functools
import struct
from typing import NamedTuple, Optional

import torch
import torch.autograd.forward_ad as _ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import engine as E

# snn_conv_args / snn_scan_args, packed field by field: a tenth of the time ctypes takes to fill its structures, which at one
# token a call is as long as the kernel runs
_CONV = struct.Struct("@iiqPP4i" + 4 * "Pqq" + "9Pq")
_SCAN = struct.Struct("@iiqPP6i" + 6 * "Pqq" + "2q6Pq" + 6 * "Pqq" + "6Pq")
assert _CONV.size == ctypes.sizeof(L.SnnConvArgs) and _SCAN.size == ctypes.sizeof(L.SnnScanArgs)
_NO_VIEW = (0, 0, 0)


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


def _on_gpu(x):
    if not x.is_cuda:
        _fail("x must live on a HIP device: supernnova_amd runs only on the GPU (no CPU fallback)")


def _traced():
    """torch.jit.trace hands out sizes as tensors; it would record the allocation of the results and nothing that fills them."""
    _fail("supernnova_amd.ssm cannot be traced: the launches are not torch operations")


class _Batch:
    """The layout of one call: sequences, steps, and the strides of a tensor's step and sequence dimensions."""

    def __init__(self, x, lengths, offsets, max_len, time_major):
        _on_gpu(x)
        if x.dtype not in E._DTYPES:
            _fail(f"x must be float32, bfloat16 or float16, got {x.dtype}")
        shape = x.shape
        if len(shape) and type(shape[0]) is not int:
            _traced()
        self.x, self.dtype, self.device, self.index, self.shape = x, x.dtype, x.device, x.get_device(), shape
        lengths_p = offsets_p = rows = 0
        if offsets is not None:
            if len(shape) != 2:
                _fail(f"ragged rows must be (rows, channels), got {tuple(shape)}")
            if lengths is not None:
                _fail("lengths and offsets exclude each other")
            offsets_p = self._vector(offsets, "offsets", torch.int64, None)
            self.B, rows = offsets.numel() - 1, shape[0]
            self.T = rows if max_len is None else min(int(max_len), rows)
            self.t_dim, self.n_dim, self.lead = 0, None, shape[:1]
        else:
            if len(shape) != 3:
                _fail(f"x must be 3-D (or 2-D rows with offsets), got {tuple(shape)}")
            if max_len is not None:
                _fail("max_len goes with offsets")
            self.t_dim, self.n_dim = (0, 1) if time_major else (1, 0)
            self.T, self.B, self.lead = shape[self.t_dim], shape[self.n_dim], shape[:2]
            if lengths is not None:
                lengths_p = self._vector(lengths, "lengths", torch.int32, self.B)
        self.D = shape[-1]
        if self.T < 1 or self.B < 1 or self.D < 1:
            _fail(f"need at least one sequence, one step and one channel, got x {tuple(shape)}, {self.B} sequences, {self.T} steps")
        if max(self.T, self.B, self.D) >= 1 << 31:
            _fail("sizes must fit 31 bits")
        self.seq = (self.B, self.T, rows, lengths_p, offsets_p)

    def _vector(self, t, name, dtype, n):
        if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous() or t.get_device() != self.index or t.numel() < 1 or (n is not None and t.numel() != n):
            _fail(f"{name} must be a contiguous {dtype} vector{'' if n is None else f' of {n}'} on {self.device}")
        return t.data_ptr()

    def view(self, t, name, shape=None):
        """A tensor of the batch (default: of x's shape) as snn_view."""
        if t.dtype != self.dtype or t.get_device() != self.index or t.shape != (self.shape if shape is None else shape):
            _fail(f"{name} must be {self.dtype} {tuple(self.shape if shape is None else shape)} on {self.device}, "
                  f"got {t.dtype} {tuple(t.shape)} on {t.device}")
        st = t.stride()
        if st[-1] != 1 and t.size(-1) != 1:
            _fail(f"{name}: the last dimension must have unit stride")
        return t.data_ptr(), st[self.t_dim], 0 if self.n_dim is None else st[self.n_dim]

    def empty(self, shape=None):
        """A contiguous result of x's (or the given) shape, and its snn_view."""
        t = self.x.new_empty(*(self.shape if shape is None else shape))       # two thirds of the time torch.empty takes
        st = t.stride()
        return t, (t.data_ptr(), st[self.t_dim], 0 if self.n_dim is None else st[self.n_dim])

    def param(self, t, name, shape, dtype=torch.float32):
        """A contiguous parameter or state -> its address (None: 0)."""
        if t is None:
            return 0
        if t.dtype != dtype or t.get_device() != self.index or t.shape != shape or not t.is_contiguous():
            _fail(f"{name} must be contiguous {dtype} {shape} on {self.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
        return t.data_ptr()

    def launch(self, fn, what, args):
        if self.index == torch.cuda.current_device():
            L.check(fn(args, torch._C._cuda_getCurrentRawStream(self.index)), what)
        else:
            with torch.cuda.device(self.index):
                L.check(fn(args, torch._C._cuda_getCurrentRawStream(self.index)), what)


class _Step(_Batch):
    """One step of B sequences: x (B, D)."""

    def __init__(self, x):
        _on_gpu(x)
        shape = x.shape
        if len(shape) and type(shape[0]) is not int:
            _traced()
        if x.dtype not in E._DTYPES or len(shape) != 2 or x.numel() < 1:
            _fail(f"x must be a non-empty (sequences, channels) tensor of float32, bfloat16 or float16, got {x.dtype} {tuple(shape)}")
        self.x, self.dtype, self.device, self.index, self.shape = x, x.dtype, x.device, x.get_device(), shape
        self.B, self.D = self.shape
        self.T, self.t_dim, self.n_dim, self.lead = 1, 0, 0, self.shape[:1]
        self.seq = (self.B, 1, 0, 0, 0)


# Tells autograd that tensors written through their addresses have other values now: a backward pass that saved one raises instead of
# reading them.
_increment_version = torch._C._increment_version


def _apart(state, old, new):
    """The state and what a step writes, at these addresses: the two may be one buffer, but must not overlap in part (other
    sequences would read what is written)."""
    gap = abs(new - old)
    if 0 < gap < state.numel() * state.element_size():
        _fail("state and new_state overlap")


def _written_requires_grad():
    """Written through its address, a tensor would keep the history of the values before."""
    if torch.is_grad_enabled():
        _fail("the state to be written requires grad: the step functions have no gradient (call them under torch.no_grad(), or detach the state)")


def _unit(t):
    """Gradients arrive with whatever strides autograd chose (an expanded sum has none): rows of unit stride."""
    return t if t.stride(-1) == 1 else t.contiguous()


# ------------------------------------------------------------------------------------------------- convolution
def _conv_head(bt, weight, bias, activation):
    if activation not in ("silu", None):
        _fail(f"activation must be 'silu' or None, got {activation!r}")
    if weight.dim() != 2 or not 2 <= weight.size(1) <= 4:
        _fail(f"weight must be (channels, 2..4), got {tuple(weight.shape)}")
    W = weight.size(1)
    return W, (*bt.seq, E._DTYPES[bt.dtype], bt.D, W, activation == "silu"), \
        (bt.param(weight, "weight", (bt.D, W)), bt.param(bias, "bias", (bt.D,)))


def causal_conv_forward(x, weight, bias=None, *, activation="silu", lengths=None, offsets=None, max_len=None,
                        initial_state=None, want_final_state=False, time_major=True):
    """Depthwise causal convolution of a batch of sequences: weight (D, W) with weight[:, -1] on the current step, bias (D,) or
    None, activation "silu" or None.  Returns (y like x, final state (B, W - 1, D) or None); the final state is what
    causal_conv_step and a later call's initial_state go on from."""
    if _ad._current_level >= 0:
        E._no_tangents(x, weight, bias, initial_state)
    bt = _Batch(x, lengths, offsets, max_len, time_major)
    W, head, par = _conv_head(bt, weight, bias, activation)
    vx, state = bt.view(x, "x"), bt.param(initial_state, "initial_state", (bt.B, W - 1, bt.D), bt.dtype)
    y, vy = bt.empty()
    end = x.new_empty(bt.B, W - 1, bt.D) if want_final_state else None
    bt.launch(L.load().snn_conv_forward, "snn_conv_forward",
              _CONV.pack(*head, *vx, *vy, *_NO_VIEW, *_NO_VIEW, *par, state, 0 if end is None else end.data_ptr(), 0, 0, 0, 0, 0, 0))
    return y, end


def causal_conv_backward(x, weight, bias, dy, *, dfinal_state=None, activation="silu", lengths=None, offsets=None, max_len=None,
                         initial_state=None, time_major=True):
    """Gradients of causal_conv_forward's result from dy = dloss/dy and, if the final state was used, dfinal_state.  Sums over
    sequences and steps are taken in an order that depends on the sizes, the layout and the alignment alone."""
    if _ad._current_level >= 0:
        E._no_tangents(x, weight, bias, dy, dfinal_state, initial_state)
    bt = _Batch(x, lengths, offsets, max_len, time_major)
    W, head, par = _conv_head(bt, weight, bias, activation)
    dy, shape = _unit(dy), (bt.B, W - 1, bt.D)
    vx, vdy, state = bt.view(x, "x"), bt.view(dy, "dy"), bt.param(initial_state, "initial_state", shape, bt.dtype)
    dend = bt.param(dfinal_state, "dfinal_state", shape, bt.dtype)
    dx, vdx = bt.empty()
    dweight, dbias = weight.new_empty(bt.D, W), weight.new_empty(bt.D) if bias is not None else None
    dstate = torch.empty_like(initial_state) if initial_state is not None else None
    args = (*head, *vx, *_NO_VIEW, *vdy, *vdx, *par, state, 0, dend, 0 if dstate is None else dstate.data_ptr(), dweight.data_ptr(),
            0 if dbias is None else dbias.data_ptr())
    lib = L.load()
    need = L.check(lib.snn_conv_workspace_bytes(_CONV.pack(*args, 0, 0)), "snn_conv_workspace_bytes")
    ws = weight.new_empty(need // 4)
    bt.launch(lib.snn_conv_backward, "snn_conv_backward", _CONV.pack(*args, ws.data_ptr(), need))
    return ConvGrads(dx, dweight, dbias, dstate)


def causal_conv_step(x, state, weight, bias=None, *, activation="silu", new_state=None):
    """The convolution's output for one new input x (B, D) of every sequence; `state` (B, W - 1, D) holds the inputs before
    it and is moved on in place, or left as it is and its successor written to `new_state`.  No gradient."""
    if _ad._current_level >= 0:
        E._no_tangents(x, state, weight, bias, new_state)
    bt = _Step(x)
    if state is None:
        _fail("causal_conv_step needs the state")
    W, head, par = _conv_head(bt, weight, bias, activation)
    shape = (bt.B, W - 1, bt.D)
    vx, old = bt.view(x, "x"), bt.param(state, "state", shape, bt.dtype)
    if new_state is None:
        new_state, new = state, old
    else:
        new = bt.param(new_state, "new_state", shape, bt.dtype)
        _apart(state, old, new)
    if new_state.requires_grad:
        _written_requires_grad()
    y, vy = bt.empty()
    bt.launch(L.load().snn_conv_step, "snn_conv_step", _CONV.pack(*head, *vx, *vy, *_NO_VIEW, *_NO_VIEW, *par, old, new, 0, 0, 0, 0, 0, 0))
    _increment_version((new_state,))
    return y


# ------------------------------------------------------------------------------------------------- scan
@functools.lru_cache(maxsize=256)
def _scan_sizes(dtype, D, N, G, B, T, rows, lengths, offsets):
    """(tape floats, forward workspace bytes, backward workspace bytes): they depend on the sizes, and on whether there are lengths
    or offsets (the addresses are not looked at)."""
    a = L.SnnScanArgs(seq=L.SnnSeq(B, T, rows, 8 if lengths else None, 8 if offsets else None), dtype=dtype, channels=D, states=N, groups=G)
    lib, p = L.load(), ctypes.byref(a)
    return (L.check(lib.snn_scan_tape_floats(p), "snn_scan_tape_floats"), L.check(lib.snn_scan_workspace_bytes(p, 0), "snn_scan_workspace_bytes"),
            L.check(lib.snn_scan_workspace_bytes(p, 1), "snn_scan_workspace_bytes"))


def _scan_head(bt, x, delta, A, B, C, D, z, delta_bias, delta_softplus, y):
    """The fields up to delta_bias (y: its view), and G, N, the shape of B and C, and the sizes."""
    if A.dim() != 2 or not 1 <= A.size(1) <= 64:
        _fail(f"A must be (channels, 1..64), got {tuple(A.shape)}")
    N, lead, dims = A.size(1), len(bt.lead), B.dim()
    if dims not in (lead + 1, lead + 2) or B.shape != C.shape:
        _fail(f"B and C must be alike, (.., states) or (.., groups, states), got {tuple(B.shape)} and {tuple(C.shape)}")
    G = B.size(-2) if dims == lead + 2 else 1
    if G < 1 or bt.D % G:
        _fail(f"{bt.D} channels cannot be dealt to {G} groups")
    shape = bt.lead + ((G, N) if dims == lead + 2 else (N,))
    dt = E._DTYPES[bt.dtype]
    head = (*bt.seq, dt, bt.D, N, G, bool(delta_softplus), 0, *bt.view(x, "x"), *bt.view(delta, "delta"),
            *(_NO_VIEW if z is None else bt.view(z, "z")), *bt.view(B, "B", shape), *bt.view(C, "C", shape), *y,
            B.stride(-2) if G > 1 else 0, C.stride(-2) if G > 1 else 0,
            bt.param(A, "A", (bt.D, N)), bt.param(D, "D", (bt.D,)), bt.param(delta_bias, "delta_bias", (bt.D,)))
    return head, G, N, shape


_NO_GRADS = (*(6 * _NO_VIEW), 0, 0, 0, 0, 0)


def _scan_forward(x, delta, A, B, C, D, z, delta_bias, delta_softplus, lengths, offsets, max_len, initial_state, want_final_state,
                  time_major, want_tape):
    if _ad._current_level >= 0:
        E._no_tangents(x, delta, A, B, C, D, z, delta_bias, initial_state)
    bt = _Batch(x, lengths, offsets, max_len, time_major)
    y, vy = bt.empty()
    head, G, N, _ = _scan_head(bt, x, delta, A, B, C, D, z, delta_bias, delta_softplus, vy)
    state = bt.param(initial_state, "initial_state", (bt.B, bt.D, N))
    n_tape, need, _ = _scan_sizes(head[5], bt.D, N, G, bt.B, bt.T, bt.seq[2], lengths is not None, offsets is not None)
    end = A.new_empty(bt.B, bt.D, N) if want_final_state else None
    tape = A.new_empty(n_tape) if want_tape else None
    ws = A.new_empty(need // 4) if need else None
    bt.launch(L.load().snn_scan_forward, "snn_scan_forward",
              _SCAN.pack(*head, state, 0 if end is None else end.data_ptr(), 0 if tape is None else tape.data_ptr(), n_tape if want_tape else 0,
                         *_NO_GRADS, 0 if ws is None else ws.data_ptr(), need))
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
    The tape holds a state every 16 steps for up to 8 states, every 8 steps for more."""
    return _scan_forward(x, delta, A, B, C, D, z, delta_bias, delta_softplus, lengths, offsets, max_len, initial_state,
                         want_final_state, time_major, True)


def selective_scan_backward(x, delta, A, B, C, dy, tape, D=None, z=None, delta_bias=None, *, dfinal_state=None, delta_softplus=True,
                            lengths=None, offsets=None, max_len=None, initial_state=None, time_major=True):
    """Gradients from dy = dloss/dy and, if the final state was used, dfinal_state, with the tape of selective_scan_train over the
    same inputs.  Every sum is taken in an order that depends on the sizes, the layout and the sequences' lengths alone."""
    if _ad._current_level >= 0:
        E._no_tangents(x, delta, A, B, C, dy, tape, D, z, delta_bias, dfinal_state, initial_state)
    bt = _Batch(x, lengths, offsets, max_len, time_major)
    head, G, N, shape = _scan_head(bt, x, delta, A, B, C, D, z, delta_bias, delta_softplus, _NO_VIEW)
    dy, Dm, sizes = _unit(dy), bt.D, (bt.B, bt.D, N)
    vdy, state, dend = bt.view(dy, "dy"), bt.param(initial_state, "initial_state", sizes), bt.param(dfinal_state, "dfinal_state", sizes)
    n_tape, _, need = _scan_sizes(head[5], Dm, N, G, bt.B, bt.T, bt.seq[2], lengths is not None, offsets is not None)
    if tape is None or tape.numel() < n_tape:
        _fail(f"the tape is too small: {0 if tape is None else tape.numel()} floats, {n_tape} needed (of selective_scan_train over the same inputs)")
    tape_p = bt.param(tape, "tape", tape.shape)
    (dx, vdx), (ddelta, vdd), (dB, vdB), (dC, vdC) = bt.empty(), bt.empty(), bt.empty(shape), bt.empty(shape)
    dz, vdz = bt.empty() if z is not None else (None, _NO_VIEW)
    dA, dD = A.new_empty(Dm, N), A.new_empty(Dm) if D is not None else None
    dbias = A.new_empty(Dm) if delta_bias is not None else None
    dstate = torch.empty_like(initial_state) if initial_state is not None else None
    ws = A.new_empty(need // 4)
    bt.launch(L.load().snn_scan_backward, "snn_scan_backward",
              _SCAN.pack(*head, state, 0, tape_p, n_tape, *vdy, *vdx, *vdd, *vdz, *vdB, *vdC, dend, dA.data_ptr(), 0 if dD is None else dD.data_ptr(),
                         0 if dbias is None else dbias.data_ptr(), 0 if dstate is None else dstate.data_ptr(), ws.data_ptr(), need))
    return ScanGrads(dx, ddelta, dA, dB, dC, dD, dz, dbias, dstate)


def selective_scan_step(x, state, delta, A, B, C, D=None, z=None, delta_bias=None, *, delta_softplus=True, new_state=None):
    """One step of every sequence: x, delta, z (B, D), B, C (B, [G,] N); `state` (B, D, N) float32 is moved on in place, or left as
    it is and its successor written to `new_state`.  Returns y (B, D).  No gradient."""
    if _ad._current_level >= 0:
        E._no_tangents(x, state, delta, A, B, C, D, z, delta_bias, new_state)
    bt = _Step(x)
    if state is None:
        _fail("selective_scan_step needs the state")
    y, vy = bt.empty()
    head, _, N, _ = _scan_head(bt, x, delta, A, B, C, D, z, delta_bias, delta_softplus, vy)
    old = bt.param(state, "state", (bt.B, bt.D, N))
    if new_state is None:
        new_state, new = state, old
    else:
        new = bt.param(new_state, "new_state", (bt.B, bt.D, N))
        _apart(state, old, new)
    if new_state.requires_grad:
        _written_requires_grad()
    bt.launch(L.load().snn_scan_step, "snn_scan_step", _SCAN.pack(*head, old, new, 0, 0, *_NO_GRADS, 0, 0))
    _increment_version((new_state,))
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

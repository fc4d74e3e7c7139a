"""The sequence operators and clipping as calls beside autograd, and over batches whose shape the other files leave out; values
against 64-bit forms (tolerances: tests/ssm_reference.py)."""
import numpy as np
import pytest
import torch

import ssm_reference as R
from supernnova_amd import engine as E
from supernnova_amd import ssm
from test_gpu_ssm import Batch, _check_scan, _scan_inputs

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


def _scan64(i, h0, dy, dend, live, mag=False):
    """ssm_reference.scan over a whole (T, B, D) batch in torch float64, one group, softplus; `live` (T, B, 1)."""
    f = torch.abs if mag else (lambda v: v)
    x, z, B, C, dy = (torch.where(live, i[k].double() if k else dy.double(), 0.0) for k in ("x", "z", "B", "C", None))
    v = i["delta"].double() + i["delta_bias"].double()
    s, sig = torch.where(live, torch.nn.functional.softplus(v), 0.0), torch.sigmoid(v)
    A, skip = i["A"].double(), f(i["D"].double())
    T = x.shape[0]
    e = torch.sigmoid(z)
    gate = f(z * e)
    hs, ys, a = [f(h0.double())], [], [torch.exp(s[t, :, :, None] * A) for t in range(T)]
    for t in range(T):
        hs.append(a[t] * hs[-1] + (s[t] * f(x[t]))[..., None] * f(B[t])[:, None])
        ys.append((hs[-1] * f(C[t])[:, None]).sum(-1) + skip * f(x[t]))
    y = torch.stack(ys)
    g = f(dy) * gate
    out = dict(y=y * gate, end=hs[T], dz=f(dy) * y * (f(e * (1 + z * (1 - e))) + (1.0 if mag else 0.0)))
    w, r = f(dend.double()), {k: [] for k in ("dx", "ddelta", "dB", "dC")}
    dA = torch.zeros_like(A)
    for t in range(T - 1, -1, -1):
        q = torch.where(live[t][..., None], f(C[t])[:, None] * g[t][..., None], 0.0) + w
        qb, w = (q * f(B[t])[:, None]).sum(-1), a[t] * q
        wh = w * hs[t]
        dA += (wh * s[t][..., None]).sum(0)
        r["ddelta"].append(torch.where(live[t], (f(x[t]) * qb + (wh * f(A)).sum(-1)) * sig[t], 0.0))
        r["dx"].append(skip * g[t] + s[t] * qb)
        r["dB"].append((q * (s[t] * f(x[t]))[..., None]).sum(1))
        r["dC"].append((hs[t + 1] * g[t][..., None]).sum(1))
    out.update({k: torch.stack(u[::-1]) for k, u in r.items()}, dA=dA, dinitial_state=w, dD=(g * f(x)).sum((0, 1)))
    out["ddelta_bias"] = out["ddelta"].sum((0, 1))
    return out


@pytest.mark.parametrize("B,D,N,layout", [(3000, 64, 16, "time"), (5000, 70, 16, "batch"), (4500, 40, 5, "rows"), (2600, 20, 40, "time")])
def test_scan_gradients_of_more_chunks_than_workgroups(B, D, N, layout):
    """A workgroup takes several sequences (with up to 4096 of them longest first) and adds their parameter gradients up.  All
    inputs are positive, so that one sequence too few or too many is 1 / B of a sum, four times the tolerance."""
    T = 6
    g = torch.Generator().manual_seed(B)
    rnd = lambda *s: torch.randn(s, generator=g).abs().cuda()                                     # noqa: E731
    lens = torch.randint(0, T + 1, (B,), generator=g).cuda()
    i = dict(x=rnd(T, B, D), delta=rnd(T, B, D) * 0.7, A=-rnd(D, N) - 0.1, B=rnd(T, B, N), C=rnd(T, B, N), D=rnd(D), z=rnd(T, B, D), delta_bias=rnd(D) * 0.5)
    dy, h0, dend = rnd(T, B, D), rnd(B, D, N), rnd(B, D, N)
    live = (torch.arange(T, device="cuda")[:, None] < lens)[..., None]
    per = ("x", "delta", "B", "C", "z")
    if layout == "rows":
        lay = lambda t: t.transpose(0, 1)[live[..., 0].t()].contiguous()                          # noqa: E731
        kw = dict(offsets=torch.cat([lens.new_zeros(1), lens.cumsum(0)]), max_len=T)
    else:
        lay = (lambda t: t) if layout == "time" else (lambda t: t.transpose(0, 1).contiguous())
        kw = dict(lengths=lens.int(), time_major=layout == "time")
    j, kw = {k: lay(v) if k in per else v for k, v in i.items()}, dict(kw, initial_state=h0)
    y, end, tape = ssm.selective_scan_train(**j, want_final_state=True, **kw)
    gr = ssm.selective_scan_backward(**j, dy=lay(dy), tape=tape, dfinal_state=dend, **kw)
    ref, mag = _scan64(i, h0, dy, dend, live), _scan64(i, h0, dy, dend, live, mag=True)
    k = 16 * T + 32 + N
    joins = -(-B // (2048 // -(-D // (256 // (4 if N <= 16 else 16)))))           # sequences a workgroup adds up in fp32
    tight = 2 * k + T + joins
    assert 4 * tight * R.EPS32 < 1 / B
    for name, got in [("y", y), ("end", end), *zip(gr._fields, gr)]:
        rows = name in ("y", "dx", "ddelta", "dz", "dB", "dC")
        r, m = (lay(torch.where(live, v[name], 0.0)) if rows else v[name] for v in (ref, mag))
        n = {"y": k, "end": k, "dA": tight, "dD": tight, "ddelta_bias": tight, "dB": 2 * k + D, "dC": 2 * k + D}.get(name, 2 * k)
        R.close(_np(got), _np(r), _np(m), n, "f32", name)


@pytest.mark.parametrize("B,T,D,dt,layout", [(1200, 300, 128, "f32", "time"), (70000, 10, 32, "f32", "batch"), (9000, 40, 64, "bf16", "rows")])
def test_conv_gradients_of_more_chunks_than_slots(B, T, D, dt, layout):
    """Chunks of more than 16 steps, several of which a thread adds up.  All inputs are positive: one chunk too few or too many is
    more than the tolerance."""
    W, g = 4, torch.Generator().manual_seed(B)
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}[dt]
    rnd = lambda *s: torch.randn(s, generator=g).abs().cuda()                                     # noqa: E731
    lens = torch.randint(0, T + 1, (B,), generator=g).cuda()
    x, dy, s0, ds = (rnd(*s).to(dtype) for s in ((T, B, D), (T, B, D), (B, W - 1, D), (B, W - 1, D)))
    w, bias = rnd(D, W) / 2, rnd(D)
    live = (torch.arange(T, device="cuda")[:, None] < lens)[..., None]
    if layout == "rows":
        lay = lambda t: t.transpose(0, 1)[live[..., 0].t()].contiguous()                          # noqa: E731
        kw = dict(offsets=torch.cat([lens.new_zeros(1), lens.cumsum(0)]), max_len=T)
    else:
        lay = (lambda t: t) if layout == "time" else (lambda t: t.transpose(0, 1).contiguous())
        kw = dict(lengths=lens.int(), time_major=layout == "time")
    gr = ssm.causal_conv_backward(lay(x), w, bias, lay(dy), dfinal_state=ds, initial_state=s0, **kw)
    xx = torch.cat([s0.double().transpose(0, 1), torch.where(live, x.double(), 0.0)])
    p = bias.double() + sum(w[:, k].double() * xx[k:k + T] for k in range(W))
    sg = torch.sigmoid(p)
    dp = torch.where(live, dy.double() * sg * (1 + p * (1 - sg)), 0.0)
    mag = torch.where(live, dy.double() * (sg * (1 + p * (1 - sg)).abs() + p), 0.0)
    dw = [torch.stack([(v * xx[k:k + T]).sum((0, 1)) for k in range(W)], 1) for v in (dp, mag)]
    dxx = [torch.zeros_like(xx), torch.zeros_like(xx)]
    for d, v in zip(dxx, (dp, mag)):
        for k in range(W):
            d[k:k + T] += w[:, k].double() * v
        d.scatter_add_(0, (lens[None] + torch.arange(W - 1, device="cuda")[:, None])[..., None].expand(W - 1, B, D), ds.double().transpose(0, 1))
    k = W + 16
    tight = 2 * k + 128 + 8                          # a chunk's steps and the joins of a thread in fp32, then fp64
    R.close(_np(gr.dweight), _np(dw[0]), _np(dw[1]), tight, "f32", "dweight")
    R.close(_np(gr.dbias), _np(dp.sum((0, 1))), _np(mag.sum((0, 1))), tight, "f32", "dbias")
    R.close(_np(gr.dinitial_state), *(_np(d[:W - 1].transpose(0, 1)) for d in dxx), 2 * k, dt, "dinitial_state")
    R.close(_np(gr.dx), *(_np(lay(torch.where(live, d[W - 1:], 0.0))) for d in dxx), 2 * k, dt, "dx")


def test_scan_split_over_time_agrees_with_the_whole():
    """Two sequences of 700 steps, whose time axis is split, and the same among 256, which fill the chip and are not."""
    T, D, N, many = 700, 96, 16, 128
    g = torch.Generator().manual_seed(11)
    rnd = lambda *s: torch.randn(s, generator=g)                                                  # noqa: E731
    i = dict(x=rnd(2, T, D), delta=rnd(2, T, D) * 0.7, B=rnd(2, T, N), C=rnd(2, T, N), z=rnd(2, T, D), A=-torch.rand(D, N, generator=g) * 2 - 0.1,
             D=rnd(D), delta_bias=rnd(D) * 0.5)
    dy, h0, dend, lens = rnd(2, T, D), rnd(2, D, N), rnd(2, D, N), torch.tensor([700, 650], dtype=torch.int32)
    runs = []
    for n in (1, many):
        rep = lambda t: t.repeat(n, *[1] * (t.dim() - 1)).cuda()                                  # noqa: E731
        j = {k: rep(v) if k not in ("A", "D", "delta_bias") else v.cuda() for k, v in i.items()}
        kw = dict(initial_state=rep(h0), lengths=rep(lens), time_major=False)
        y, end, tape = ssm.selective_scan_train(**j, want_final_state=True, **kw)
        gr = ssm.selective_scan_backward(**j, dy=rep(dy), tape=tape, dfinal_state=rep(dend), **kw)
        runs.append(dict(y=y[:2], end=end[:2], dx=gr.dx[:2], ddelta=gr.ddelta[:2], dz=gr.dz[:2], dB=gr.dB[:2], dC=gr.dC[:2], dh0=gr.dinitial_state[:2],
                         dA=gr.dA / n, dskip=gr.dD / n, ddbias=gr.ddelta_bias / n))
    assert not torch.equal(runs[0]["y"], runs[1]["y"])                    # two ways of computing it
    mags = []
    for b in range(2):
        n = int(lens[b])
        wide = lambda t: np.repeat(t[b, :n].double().numpy()[:, None], D, axis=1)                 # noqa: E731
        a = dict(x=_np(i["x"][b, :n]), delta=_np(i["delta"][b, :n]), A=_np(i["A"]), B=wide(i["B"]), C=wide(i["C"]), skip=_np(i["D"]),
                 z=_np(i["z"][b, :n]), dbias=_np(i["delta_bias"]), h0=_np(h0[b]), dy=_np(dy[b, :n]), dend=_np(dend[b]))
        m = R.scan(**a, mag=True)
        m["dB"], m["dC"] = m["dB"].sum(1), m["dC"].sum(1)
        k = 16 * n + 32 + N                          # each of the two is off by as much: twice
        for name in ("y", "end", "dx", "ddelta", "dz", "dB", "dC", "dh0"):
            u, v = (_np(r[name][b]) for r in runs)
            if name not in ("end", "dh0"):
                u, v = u[:n], v[:n]
            R.close(u, v, m[name], 2 * k if name in ("y", "end") else 2 * (2 * k + D), what=name)
        mags.append(m)
    for name in ("dA", "dskip", "ddbias"):
        R.close(_np(runs[0][name]), _np(runs[1][name]), mags[0][name] + mags[1][name], 2 * (2 * (16 * T + 32 + N) + T + many), what=name)


@pytest.mark.parametrize("N,layout,lens", [(40, "batch", (300, 190)), (64, "rows", (0, 260, 140)), (33, "time", (515,))])
def test_scan_of_many_states_split_over_time(N, layout, lens):
    bt = Batch(lens, 20, "f32", layout, seed=N)
    i, h0 = _scan_inputs(bt, N, 2, True, True)
    dy, dend, kw = bt.seqs(20), bt.par(bt.B, 20, N), dict(initial_state=h0, **bt.kw)
    y, end, tape = ssm.selective_scan_train(**i, want_final_state=True, **kw)
    gr = ssm.selective_scan_backward(**i, dy=dy, tape=tape, dfinal_state=dend, **kw)
    _check_scan(bt, i, h0, 2, True, dy, dend, y, end, gr)


def _layer(p, kw):
    u = ssm.causal_conv(p["x"], p["w"], p["b"], **kw)
    return ssm.selective_scan(u, p["delta"], p["A"], p["B"], p["C"], p["D"], p["z"], p["dtb"], **kw)


def _layer_inputs(seed, R_, D=24, N=6):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g).cuda()                                           # noqa: E731
    return dict(x=rnd(R_, D), delta=rnd(R_, D), z=rnd(R_, D), B=rnd(R_, N), C=rnd(R_, N), w=rnd(D, 4) / 2, b=rnd(D), A=-torch.rand(D, N, generator=g).cuda() - 0.1,
                D=rnd(D), dtb=rnd(D) / 2), rnd(R_, D)


def test_differentiable_forms_of_rows():
    """Rows with offsets and no max_len through autograd: the explicit calls' bits, twice over one graph, on a side stream, and
    padded to (T, B, D) the same values."""
    lens = [5, 0, 70, 1, 130]
    off = torch.tensor(np.cumsum([0] + lens)).cuda()
    i, dy = _layer_inputs(5, sum(lens))
    kw = dict(offsets=off)
    u, _ = ssm.causal_conv_forward(i["x"], i["w"], i["b"], **kw)
    args = dict(x=u, delta=i["delta"], A=i["A"], B=i["B"], C=i["C"], D=i["D"], z=i["z"], delta_bias=i["dtb"])
    y, _, tape = ssm.selective_scan_train(**args, **kw)
    gs = ssm.selective_scan_backward(**args, dy=dy, tape=tape, **kw)
    gc = ssm.causal_conv_backward(i["x"], i["w"], i["b"], gs.dx, **kw)
    want = dict(x=gc.dx, w=gc.dweight, b=gc.dbias, delta=gs.ddelta, A=gs.dA, B=gs.dB, C=gs.dC, D=gs.dD, z=gs.dz, dtb=gs.ddelta_bias)
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        p = {k: v.clone().requires_grad_() for k, v in i.items()}
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            out = _layer(p, kw)
        torch.cuda.current_stream().wait_stream(stream)
        first = torch.autograd.grad(out, list(p.values()), dy, retain_graph=True)
        again = torch.autograd.grad(out, list(p.values()), dy)
        torch.cuda.synchronize()
        assert torch.equal(out, y)
        for k, a, b in zip(p, first, again):
            assert torch.equal(a, want[k]) and torch.equal(b, want[k]), k
    T, B = max(lens), len(lens)
    at = torch.cat([torch.arange(n) * B + b for b, n in enumerate(lens)]).cuda()
    per = ("x", "delta", "z", "B", "C")
    p = {k: v.new_zeros(T * B, v.shape[1]).index_copy(0, at, v).view(T, B, -1) if k in per else v for k, v in i.items()}
    p = {k: v.clone().requires_grad_() for k, v in p.items()}
    out = _layer(p, dict(lengths=torch.tensor(lens, dtype=torch.int32).cuda()))
    grads = torch.autograd.grad(out, list(p.values()), dy.new_zeros(T * B, dy.shape[1]).index_copy(0, at, dy).view(T, B, -1))
    # the same sums cut elsewhere: (32 T + 64) roundings of magnitudes that a random layer of this size holds below 10 times the values
    tol = 10 * (32 * T + 64) * R.EPS32
    for k, v in zip(p, grads):
        v = v.reshape(T * B, -1)[at] if k in per else v
        assert float((v - want[k]).abs().max()) <= tol * float(want[k].abs().max()), k


def test_two_threads_at_once():
    """Two threads, each with its own stream and sizes: the bits of one after the other."""
    import threading
    cases = []
    for seed, lens in ((1, [300, 20, 44]), (2, [9] * 600)):
        i, dy = _layer_inputs(seed, sum(lens))
        cases.append((i, dy, dict(offsets=torch.tensor(np.cumsum([0] + lens)).cuda(), max_len=max(lens))))

    def run(i, dy, kw):
        p = {k: v.clone().requires_grad_() for k, v in i.items()}
        out = _layer(p, kw)
        grads = list(torch.autograd.grad(out, list(p.values()), dy))
        norm = E.clip_grads(grads, 0.5)
        return [out.detach(), norm, *grads]
    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    got, streams = [[], []], [torch.cuda.Stream(), torch.cuda.Stream()]

    def work(n):
        with torch.cuda.stream(streams[n]):
            for _ in range(5):
                got[n].append(run(*cases[n]))
        streams[n].synchronize()
    threads = [threading.Thread(target=work, args=(n,)) for n in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for n in (0, 1):
        assert len(got[n]) == 5
        for outs in got[n]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[n]))

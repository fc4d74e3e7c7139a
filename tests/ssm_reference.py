"""Plain 64-bit forms of the short causal convolution and the selective scan, with their gradients written out, on numpy
arrays of one sequence; and the size of what is added up on the way (`mag=True`), which the tests' tolerances are made of.

Tolerances.  An output computed in fp32 and rounded once to type t is off by at most
    half_step(t) |value| + k 2^-24 M,
M = the value with every term replaced by its magnitude, k = the number of roundings on the longest path.  Convolution: W
products and sums, silu (exp, reciprocal, three products, each at most 2 roundings): k = W + 16.  Scan: a step adds at most 16
(softplus 8, s A 2, exp 2, s x B 2, multiply-add 2) to a state's relative error, so k = 16 T + 32 for y and the states; an
adjoint adds the same again: 32 T + 64 for gradients.  A sum of n values in fp32 adds n."""
import numpy as np

EPS32 = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 1e-37, "bf16": 1e-37, "f16": 2.0 ** -25}     # half the smallest subnormal step of fp16; flushed fp32 ones


def sigmoid(v):
    return 1.0 / (1.0 + np.exp(-v))


def softplus(v):
    return np.logaddexp(0.0, v)


def conv(x, w, bias, silu, s0, dy=None, ds=None, mag=False):
    """x (T, D), w (D, W), s0 (W - 1, D) or None -> dict of y, end and, with dy, dx, dw, db, ds0."""
    T, D = x.shape
    W = w.shape[1]
    s0 = np.zeros((W - 1, D)) if s0 is None else s0
    b = np.zeros(D) if bias is None else bias
    xx = np.concatenate([s0, x])
    taps = np.stack([xx[k:k + T] for k in range(W)])          # (W, T, D)
    p = b + np.einsum("dw,wtd->td", w, taps)
    f = np.abs if mag else (lambda v: v)
    P = f(b) + np.einsum("dw,wtd->td", f(w), f(taps))
    s = sigmoid(p)
    out = {"y": P * s if silu and mag else p * s if silu else P, "end": f(xx[T:])}
    if silu and mag:
        out["y"] = P * (s + np.abs(p) * s * (1 - s))          # an error of p passes through silu'
    if dy is not None:
        g = s * (1 + (P if mag else p) * (1 - s)) if silu else np.ones_like(p)
        if mag and silu:
            g = g + P                                         # |silu''| <= 1/2: an error of p in the slope
        dp = f(dy) * g
        dxx = np.zeros_like(xx)
        for k in range(W):
            dxx[k:k + T] += f(w[:, k]) * dp
        if ds is not None:
            dxx[T:] += f(ds)
        out.update(dx=dxx[W - 1:], ds0=dxx[:W - 1], dw=np.einsum("td,wtd->dw", dp, f(taps)), db=dp.sum(0))
    return out


def scan(x, delta, A, B, C, skip=None, z=None, dbias=None, sp=True, h0=None, dy=None, dend=None, mag=False):
    """x, delta, z (T, D), A (D, N), B, C (T, D, N) (every channel with its group's row), h0 (D, N) -> dict."""
    T, D = x.shape
    N = A.shape[1]
    f = np.abs if mag else (lambda v: v)
    v = delta + (0.0 if dbias is None else dbias)
    s, sig = (softplus(v), sigmoid(v)) if sp else (v, np.ones_like(v))
    a = np.exp(s[:, :, None] * A)
    h = np.zeros((T + 1, D, N))
    if h0 is not None:
        h[0] = f(h0)
    u = f(s) * f(x)
    for t in range(T):
        h[t + 1] = a[t] * h[t] + u[t][:, None] * f(B[t])
    skip_ = np.zeros(D) if skip is None else f(skip)
    y = (h[1:] * f(C)).sum(-1) + skip_ * f(x)
    zs = None if z is None else z * sigmoid(z)
    out = {"y": y if z is None else y * f(zs), "end": h[T]}
    if dy is None:
        return out
    g = f(dy) if z is None else f(dy) * f(zs)
    if z is not None:
        e = sigmoid(z)
        out["dz"] = f(dy) * y * (f(e * (1 + z * (1 - e))) + (1.0 if mag else 0.0))
    w = np.zeros((D, N)) if dend is None else f(dend).copy()
    q = np.zeros((T, D, N))
    for t in range(T - 1, -1, -1):
        q[t] = f(C[t]) * g[t][:, None] + w
        w = a[t] * q[t]
    qb = (q * f(B)).sum(-1)
    wh = q * a * h[:-1]
    dd = (f(x) * qb + (wh * f(A)).sum(-1)) * sig
    out.update(dx=skip_ * g + f(s) * qb, ddelta=dd, ddbias=dd.sum(0), dA=(wh * f(s)[:, :, None]).sum(0), dskip=(g * f(x)).sum(0),
               dB=q * u[:, :, None], dC=g[:, :, None] * h[1:], dh0=w)
    return out


def close(got, ref, mag, k, dt="f32", what=""):
    """|got - ref| <= half a step of the type + k roundings of the magnitudes (module docstring)."""
    got = np.asarray(got, np.float64)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    tol = HALF[dt] * (np.abs(ref) + k * EPS32 * mag) + k * EPS32 * mag + TINY[dt]
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:3], ref[bad][:3], tol[bad][:3])

"""Global gradient norm and clipping on the GPU against 64-bit sums.  The norm is an fp64 sum rounded to fp32 (one rounding,
2^-24); the coefficient max_norm / (norm + 1e-6) is two more fp32 roundings, a product one, and a 16-bit gradient is rounded
once from fp32: half a step of its type + 4 x 2^-24."""
import math

import numpy as np
import pytest
import torch

import ssm_reference as R
from supernnova_amd import _lib as L
from supernnova_amd import engine as E
from supernnova_amd import optim

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _norm64(ts, p):
    m = [t.double().abs().reshape(-1) for t in ts if t.numel()]
    if not m:
        return 0.0
    v = torch.cat(m)
    return float(v.max()) if p == math.inf else float((v ** p).sum() ** (1 / p))


def _make(shapes, dts, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(DT[d]).cuda() for s, d in zip(shapes, dts)]


CASES = [([(1,)], ["f32"]), ([(3,), (0,), (129, 65), (7, 1, 5)], ["f32", "bf16", "f16", "bf16"]), ([(40000, 3), (32768,), (32769,)], ["f32", "bf16", "f16"]),
         ([(17, k + 1) for k in range(200)], ["f32", "bf16"] * 100), ([(1030, 33000)], ["bf16"])]


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("shapes,dts", CASES)
@pytest.mark.parametrize("place", ["in place", "out", "shifted"])
def test_clip(shapes, dts, p, place):
    ts = _make(shapes, dts, len(shapes))
    want = _norm64(ts, p)
    orig = [t.clone() for t in ts]
    out = None
    if place == "out":
        out = [torch.full_like(t, 9.0) for t in ts]
    elif place == "shifted":                     # views at every odd offset of one buffer
        flat = {d: torch.zeros(2 + sum(t.numel() + 1 for t in ts), dtype=DT[d], device="cuda") for d in set(dts)}
        out, at = [], 1
        for t, d in zip(ts, dts):
            out.append(flat[d][at:at + t.numel()].view(t.shape))
            at += t.numel() + 1
    max_norm = 0.25 * want
    norm = E.clip_grads(ts, max_norm, p, out=out)
    assert norm.shape == () and norm.dtype == torch.float32 and abs(float(norm) - want) <= 2 * R.EPS32 * want
    assert abs(float(E.grad_norm(orig, p)) - want) <= 2 * R.EPS32 * want
    c = min(1.0, max_norm / (want + 1e-6))
    for t, o, d in zip(ts if out is None else out, orig, dts):
        ref = o.double().cpu().numpy() * c
        R.close(t.double().cpu().numpy(), ref, np.abs(ref), 4, d)
    if out is not None:
        assert all(torch.equal(a, b) for a, b in zip(ts, orig))


def test_no_clipping_leaves_gradients_as_they_are():
    ts = _make([(50, 7), (9,)], ["f32", "bf16"], 1)
    keep = [t.clone() for t in ts]
    E.clip_grads(ts, 1e6)
    assert all(torch.equal(a, b) for a, b in zip(ts, keep))
    z = [torch.zeros(5, device="cuda")]
    assert float(E.clip_grads(z, 1.0)) == 0 and (z[0] == 0).all()
    assert float(E.grad_norm([torch.zeros(0, device="cuda")])) == 0


def test_large_and_not_finite_gradients():
    big = [torch.full((4000,), 1e30, device="cuda")]
    assert abs(float(E.grad_norm(big)) - 1e30 * math.sqrt(4000)) <= 1e30 * 64 * 1e-6
    for bad, c in ((float("inf"), 0.0), (float("nan"), float("nan"))):
        for p in (1.0, 2.0, math.inf):
            ts = _make([(1000,), (3,)], ["f32", "bf16"], 2)
            ts[0][7] = bad
            ref = [torch.nn.Parameter(t.clone()) for t in ts]
            for r, t in zip(ref, ts):
                r.grad = t.clone()
            norm = E.clip_grads(ts, 1.0, p)
            assert not math.isfinite(float(norm))
            want = torch.nn.utils.clip_grad_norm_(ref, 1.0, p)
            assert math.isnan(float(want)) == math.isnan(float(norm))
            assert all(torch.equal(torch.isnan(t), torch.isnan(r.grad)) for t, r in zip(ts, ref))
            assert c != 0.0 or (ts[1] == 0).all()


def test_dense_orders_and_refusals():
    t = torch.randn(6, 5, device="cuda")
    a = t.clone().t()
    n = E.clip_grads([a], 0.5)
    assert abs(float(n) - _norm64([t], 2)) <= 2 * R.EPS32 * float(n) and torch.allclose(a, t.t() * (0.5 / (float(n) + 1e-6)), rtol=1e-6)
    with pytest.raises(L.SnnError, match="dense"):
        E.grad_norm([t[:, :3]])
    with pytest.raises(L.SnnError, match="dense"):
        E.grad_norm([t.cpu(), t][::-1])
    with pytest.raises(L.SnnError, match="type"):
        E.grad_norm([t.double()])
    with pytest.raises(L.SnnError, match="out"):
        E.clip_grads([t], 1.0, out=[t.half()])
    with pytest.raises(L.SnnError, match="out"):
        E.clip_grads([t], 1.0, out=[torch.empty(5, 6, device="cuda").t()])
    with pytest.raises(L.SnnError, match="out"):
        E.clip_grads([t], 1.0, out=[torch.empty(29, device="cuda")])
    flat = torch.empty(30, device="cuda")
    E.clip_grads([t], 1.0, out=[flat])
    assert abs(float(flat.double().norm()) - 1.0) <= 2e-6 and torch.equal(flat.sign(), t.sign().reshape(-1))
    with pytest.raises(L.SnnError, match="out has"):
        E.clip_grads([t], 1.0, out=[])
    with pytest.raises(L.SnnError, match="twice"):
        E.clip_grads([t, t], 1.0)
    u = t.clone()
    with pytest.raises(L.SnnError, match="another gradient"):
        E.clip_grads([t, u], 1.0, out=[u, t])
    with pytest.raises(L.SnnError, match="twice"):
        E.clip_grads([t, u], 1.0, out=[t, t])
    with pytest.raises(L.SnnError, match="norm_type"):
        E.clip_grads([t], 1.0, norm_type="inf")


def test_clip_grad_norm_like_torch():
    ps = [torch.nn.Parameter(t) for t in _make([(40, 3), (7,), (2, 2)], ["f32"] * 3, 5)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q, t in zip(ps[:2], qs, _make([(40, 3), (7,)], ["f32"] * 2, 6)):
        p.grad, q.grad = t, t.clone()
    a, b = optim.clip_grad_norm_(ps, 0.7), torch.nn.utils.clip_grad_norm_(qs, 0.7)
    # torch's norm is an fp32 sum of 127 squares: 127 roundings at most; ours one
    assert abs(float(a) - float(b)) <= 130 * R.EPS32 * float(b)
    for p, q in zip(ps[:2], qs):
        assert bool(((p.grad - q.grad).abs() <= 140 * R.EPS32 * q.grad.abs()).all())
    assert ps[2].grad is None
    ps[0].grad[0, 0] = float("nan")
    keep = ps[1].grad.clone()
    with pytest.raises(L.SnnError, match="finite"):
        optim.clip_grad_norm_(ps, 0.7, error_if_nonfinite=True)
    assert torch.equal(ps[1].grad, keep)


def test_captured_clip():
    ts = _make([(300, 50), (77,)], ["f32", "bf16"], 8)
    out = [torch.empty_like(t) for t in ts]
    E.clip_grads(ts, 1.0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = E.clip_grads(ts, 1.0, out=out)
    for n in range(3):
        for t in ts:
            t.mul_(1.5)
        graph.replay()
        want = [torch.empty_like(t) for t in ts]
        wn = E.clip_grads(ts, 1.0, out=want)
        torch.cuda.synchronize()
        assert torch.equal(norm, wn) and all(torch.equal(a, b) for a, b in zip(out, want)), n


@pytest.mark.parametrize("kind", ["adam", "sgd"])
def test_fused_optimizers_clip(kind):
    """A clipped step is the plain step on gradients scaled by hand, an unclipped one the plain step.  The two updates are
    compiled apart and may fuse other products: a handful of roundings of the step (lr = 0.1, |step| <= 0.1 / 0.001) and of
    the parameters, which are below 32 here."""
    g = torch.Generator().manual_seed(4)
    n = 1000

    class Model:
        def __init__(self):
            self.flat = torch.linspace(-1, 1, n, device="cuda")
            self.ps = [torch.nn.Parameter(self.flat[:600].view(20, 30)), torch.nn.Parameter(self.flat[600:])]

        def parameters(self):
            return iter(self.ps)

        def _flat_params(self):
            return self.ps

        def flat_parameters(self):
            return self.flat
    make = (lambda m, **k: optim.FusedAdam(m, lr=0.1, weight_decay=0.01, **k)) if kind == "adam" else \
        (lambda m, **k: optim.FusedSGD(m, lr=0.1, momentum=0.9, weight_decay=0.01, **k))
    a, b, c, d = Model(), Model(), Model(), Model()
    oa, ob, oc, od = make(a, max_grad_norm=0.5), make(b), make(c, max_grad_norm=1e9), make(d)
    for _ in range(3):
        grad = torch.randn(n, generator=g).cuda()
        oa.step_flat(grad.clone())
        norm = float(grad.double().norm())
        assert abs(float(oa.last_grad_norm) - norm) <= 2 * R.EPS32 * norm
        coef = torch.tensor(0.5, device="cuda") / (oa.last_grad_norm + 1e-6)
        ob.step_flat(grad * coef)
        oc.step_flat(grad.clone())
        od.step_flat(grad.clone())
        for u, v in ((a.flat, b.flat), (c.flat, d.flat)):
            assert float((u - v).abs().max()) <= 3 * 16 * 32 * R.EPS32
    assert oa.state_dict()["param_groups"][0]["max_grad_norm"] == 0.5


def test_settings_clip_the_training_step():
    """train_step_fused of a model whose settings name max_grad_norm: one step equals the unclipped optimizer fed scaled gradients."""
    from types import SimpleNamespace
    from supernnova_amd.utils import training_utils as tu
    st = SimpleNamespace(layer_type="lstm", hidden_dim=32, num_layers=2, bidirectional=True, nb_classes=2, dropout=0.0, use_cuda=True,
                         rnn_output_option="mean", learning_rate=1e-2, weight_decay=0.0, model="vanilla", no_dump=True, max_grad_norm=0.01)
    torch.manual_seed(0)
    x = torch.randn(9, 6, 24, device="cuda")
    y = torch.randint(0, 2, (6,), device="cuda")
    packed = torch.nn.utils.rnn.pack_padded_sequence(x, [9, 8, 7, 5, 3, 3])
    rnn = tu.get_model(st, 24).cuda()
    twin = tu.get_model(st, 24).cuda()
    twin.load_state_dict(rnn.state_dict())
    opt = tu.get_optimizer(st, rnn)
    st.max_grad_norm = None
    plain = tu.get_optimizer(st, twin)
    tu.train_step_fused(st, rnn, packed, y, opt, 6, 1)
    seen = {}
    step = plain.step_flat
    plain.step_flat = lambda g, mean=True: (seen.update(g=g.clone()), step(g * (torch.tensor(0.01, device="cuda") / (E.grad_norm([g]) + 1e-6)), mean=mean))
    tu.train_step_fused(st, twin, packed, y, plain, 6, 1)
    assert abs(float(opt.last_grad_norm) - float(seen["g"].double().norm())) <= 2 * R.EPS32 * float(opt.last_grad_norm)
    # Adam's first step is lr g / (|g| + 1e-8): with gradients scaled to a norm of 0.01 over 19 000 parameters a rounding of g
    # moves it by lr 1e-8 |g| 2^-24 / (|g| + 1e-8)^2 <= lr / 4 2^-24 each; 16 of them, and 4 of a parameter below 1
    assert float(opt.last_grad_norm) > 0.01
    assert float((rnn.flat_parameters() - twin.flat_parameters()).abs().max()) <= (16 * 1e-2 / 4 + 4) * R.EPS32


def test_overlapping_slices_are_refused():
    flat = torch.randn(100, device="cuda")
    before = flat.clone()
    with pytest.raises(L.SnnError, match="overlap"):
        E.clip_grads([flat[:60], flat[50:]], 0.5)
    with pytest.raises(L.SnnError, match="overlap"):
        E.clip_grads([flat[:50]], 0.5, out=[flat[1:51]])
    assert torch.equal(flat, before)
    E.clip_grads([flat[50:], flat[:50]], 0.5)                   # neighbours, in any order
    assert abs(float(flat.double().norm()) - 0.5) <= 2e-6
    assert float(E.grad_norm([flat, flat])) > float(E.grad_norm([flat]))            # reading twice is no write

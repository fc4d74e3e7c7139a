"""What the host layer of the sequence operators and of clipping refuses or tells autograd, without a GPU: the launches are
replaced, so that only Python runs."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from supernnova_amd import _lib as L
from supernnova_amd import engine as E
from supernnova_amd import ssm


@pytest.fixture
def host_only(monkeypatch):
    """CPU tensors pass for device tensors, nothing is launched."""
    monkeypatch.setattr(ssm, "_on_gpu", lambda x: None)
    monkeypatch.setattr(ssm._Batch, "launch", lambda self, fn, what, args: None)


def _inputs(lead=(3, 2), D=4, N=5):
    return dict(x=torch.randn(*lead, D), delta=torch.randn(*lead, D), A=-torch.rand(D, N), B=torch.randn(*lead, N), C=torch.randn(*lead, N),
                D=torch.randn(D), z=torch.randn(*lead, D), delta_bias=torch.randn(D))


def _calls():
    """(name, tensors by name, call) of every entry point."""
    w, b = torch.randn(4, 3), torch.randn(4)
    x, s0 = torch.randn(3, 2, 4), torch.randn(2, 2, 4)
    h0, i, one = torch.randn(2, 4, 5), _inputs(), _inputs((2,))
    tape = torch.zeros(1 << 14)
    return [
        ("conv", dict(x=x, weight=w, bias=b, initial_state=s0), ssm.causal_conv),
        ("conv forward", dict(x=x, weight=w, bias=b, initial_state=s0), ssm.causal_conv_forward),
        ("conv backward", dict(x=x, weight=w, bias=b, dy=torch.randn(3, 2, 4), initial_state=s0, dfinal_state=torch.randn(2, 2, 4)),
         ssm.causal_conv_backward),
        ("conv step", dict(x=x[0].clone(), state=s0, weight=w, bias=b), ssm.causal_conv_step),
        ("scan", dict(i, initial_state=h0), ssm.selective_scan),
        ("scan forward", dict(i, initial_state=h0), ssm.selective_scan_forward),
        ("scan train", dict(i, initial_state=h0), ssm.selective_scan_train),
        ("scan backward", dict(i, initial_state=h0, dy=torch.randn(3, 2, 4), tape=tape, dfinal_state=torch.randn(2, 4, 5)), ssm.selective_scan_backward),
        ("scan step", dict(one, state=h0), ssm.selective_scan_step)]


def test_tangents_are_refused(host_only):
    """A tensor of forward-mode differentiation does not require grad, and its tangent would be lost without a word."""
    for name, args, call in _calls():
        for k in args:
            with fw.dual_level():
                call(**args)                                             # a level by itself is no reason to refuse
                dual = dict(args, **{k: fw.make_dual(args[k], torch.ones_like(args[k]))})
                with pytest.raises(L.SnnError, match="forward-mode"):
                    call(**dual)
                    pytest.fail(f"{name}: {k}")
    with fw.dual_level():
        g = fw.make_dual(torch.ones(3), torch.ones(3))
        with pytest.raises(L.SnnError, match="forward-mode"):
            E.grad_norm([g])
        with pytest.raises(L.SnnError, match="forward-mode"):
            E.clip_grads([torch.ones(3), g], 1.0)


@pytest.mark.filterwarnings("ignore")
def test_tracing_is_refused(host_only):
    """torch.jit.trace sees only the allocation of the results: the traced function would return memory nobody wrote."""
    for name, args, call in _calls():
        keys = list(args)
        with pytest.raises(L.SnnError, match="traced"):
            torch.jit.trace(lambda *a: call(**dict(zip(keys, a))), tuple(args.values()), check_trace=False)
            pytest.fail(name)
    with pytest.raises(L.SnnError, match="traced"):
        torch.jit.trace(lambda g: E.grad_norm([g]), (torch.ones(3),), check_trace=False)


def test_steps_tell_autograd_what_they_wrote(host_only):
    """A state that a differentiable call has saved and a step then moves on in place: the backward pass must not use it."""
    w = torch.randn(4, 3)
    for inference in (False, True):
        with torch.inference_mode(inference):
            x, s, h, one = torch.randn(2, 4), torch.randn(2, 2, 4), torch.randn(2, 4, 5), _inputs((2,))
            ssm.causal_conv_step(x, s, w, new_state=torch.empty_like(s))
            ssm.selective_scan_step(**one, state=h, new_state=torch.empty_like(h))
            ssm.causal_conv_step(x, s, w)
            ssm.selective_scan_step(**one, state=h)
    x, s, h, one = torch.randn(2, 4), torch.randn(2, 2, 4), torch.randn(2, 4, 5), _inputs((2,))
    s2, h2 = torch.empty_like(s), torch.empty_like(h)
    was = [t._version for t in (s, h, s2, h2)]
    ssm.causal_conv_step(x, s, w, new_state=s2)
    ssm.selective_scan_step(**one, state=h, new_state=h2)
    assert [t._version for t in (s, h)] == was[:2] and s2._version > was[2] and h2._version > was[3]
    y = (torch.ones(4, requires_grad=True) * s).sum()
    ssm.causal_conv_step(x, s, w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    y = (torch.ones(5, requires_grad=True) * h).sum()
    ssm.selective_scan_step(**one, state=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_steps_refuse_to_write_a_state_with_a_gradient(host_only):
    """The written state would keep the history of the one before it."""
    w, x, one = torch.randn(4, 3), torch.randn(2, 4), _inputs((2,))
    for of in (lambda t: t.requires_grad_(), lambda t: t.requires_grad_() * 2):          # a leaf, and a result
        s, h = of(torch.randn(2, 2, 4)), of(torch.randn(2, 4, 5))
        s0, h0 = torch.randn(2, 2, 4), torch.randn(2, 4, 5)
        for call in (lambda: ssm.causal_conv_step(x, s, w), lambda: ssm.causal_conv_step(x, s0, w, new_state=s),
                     lambda: ssm.selective_scan_step(**one, state=h), lambda: ssm.selective_scan_step(**one, state=h0, new_state=h)):
            with pytest.raises(L.SnnError, match="requires grad"):
                call()
            with torch.no_grad():
                call()
        ssm.causal_conv_step(x, s, w, new_state=s0)                      # reading one is no matter
        ssm.selective_scan_step(**one, state=h, new_state=h0)

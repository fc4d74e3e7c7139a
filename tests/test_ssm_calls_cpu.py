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

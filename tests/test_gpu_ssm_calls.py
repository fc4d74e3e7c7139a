"""The sequence operators and clipping as calls beside autograd, and over batches whose shape the other files leave out; values
against 64-bit forms (tolerances: tests/ssm_reference.py)."""
import pytest
import torch

from supernnova_amd import engine as E
from supernnova_amd import ssm

pytestmark = pytest.mark.gpu


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

"""GPU: the feed-forward operators where a plain call does not go -- under forward-mode differentiation and a trace, with values
that are not finite, at the ends of their sizes, in memory orders that are not the dense one.  Values against the formulas in 64
bits (ff_reference: derived bounds), or against another call that has to give the same bits."""
import pytest
import torch

from closerlook3d_amd import feed_forward as ff
from tests import ff_reference as ref
from tests.test_feed_forward_gpu import TYPES, features, ffn_check, ffn_inputs, gen, norm_check, rows, vector

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------- what a call without a gradient is seen by
def _calls():
    """Every operator as a function of its features, on tensors that require no gradient."""
    g = gen(1)
    x = features(g, 2, 24, 40, torch.float32)
    w, v = vector(g, 32, 24, dtype=torch.float32), vector(g, 24, dtype=torch.float32)
    d = vector(g, 24, 32, dtype=torch.float32)
    rng = torch.tensor([3, 0], device="cuda")
    return x, {
        "gated_feed_forward": lambda t: ff.gated_feed_forward(t, w, w, d),
        "point_norm": lambda t: ff.point_norm(t, v, kind='layer'),
        "norm_gate_residual": lambda t: ff.norm_gate_residual(t, x, gate=v),
        "norm_gate_residual_next": lambda t: ff.norm_gate_residual(x, t, v, p=0.2, rng=rng, next_kind='rms')[1],
        "dropout": lambda t: ff.dropout(t, 0.4, rng),
    }


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["gated_feed_forward", "point_norm", "norm_gate_residual", "norm_gate_residual_next", "dropout"])
def test_a_tangent_is_refused_and_not_lost(name, grad):
    """No operator has a forward-mode derivative: a dual tensor is refused, whether or not anything requires a gradient.  Tensors
    without a tangent are computed as ever inside such a level."""
    import torch.autograd.forward_ad as fwd
    x, calls = _calls()
    want = calls[name](x)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        assert torch.equal(calls[name](x), want)
        with pytest.raises(NotImplementedError, match="jvp"):
            calls[name](fwd.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("name", ["gated_feed_forward", "point_norm", "norm_gate_residual", "norm_gate_residual_next", "dropout",
                                  "to_point_major", "take"])
def test_a_trace_is_refused(name):
    """A trace would hold a call's allocations and nothing of what the launches put there: its results would be memory as it was."""
    x, calls = _calls()
    rng = ff.CounterRng(5, "cuda")
    calls["to_point_major"] = lambda t: ff.to_point_major(t.contiguous())
    calls["take"] = lambda t: t * rng.take(8)[0]
    for grad in (False, True):
        with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(calls[name], (x.clone().requires_grad_(grad),), check_trace=False)
    assert rng.state.tolist() == [5, 0]

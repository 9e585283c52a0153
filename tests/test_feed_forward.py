"""CPU: what the feed-forward operators refuse, before any launch; the generator's published vectors; the references of the GPU
tests against autograd and differences."""
import ctypes

import numpy as np
import pytest
import torch

from tests import ff_reference as ref
from closerlook3d_amd import _lib
from closerlook3d_amd import feed_forward as ff


# ------------------------------------------------------------------------------------------------------------ refusals
def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 8), torch.zeros(16, 8)
    for call in (lambda: ff.gated_feed_forward(x, w, w, torch.zeros(8, 16)), lambda: ff.point_norm(x),
                 lambda: ff.norm_gate_residual(x, x), lambda: ff.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64)),
                 lambda: ff.to_point_major(x[None]), lambda: ff.CounterRng(0, 'cpu')):
        with pytest.raises(RuntimeError, match="CPU not supported"):
            call()


class _Fake(torch.Tensor):
    """A CPU tensor that calls itself a CUDA one: the checks of Python arguments, without a GPU (nothing is launched)."""

    @property
    def is_cuda(self):
        return True


def fake(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(_Fake)


@pytest.mark.parametrize("call, error, text", [
    (lambda: ff.gated_feed_forward([1.0], None, None), TypeError, "x is a tensor"),
    (lambda: ff.gated_feed_forward(fake(4, 8, dtype=torch.float64), fake(16, 8), fake(16, 8)), TypeError, "float32, bfloat16 or float16"),
    (lambda: ff.gated_feed_forward(fake(8), fake(16, 8), fake(16, 8)), ValueError, r"\(B, C, N\)"),
    (lambda: ff.gated_feed_forward(fake(4, 8), None, fake(16, 8)), TypeError, "w_gate is missing"),
    (lambda: ff.gated_feed_forward(fake(4, 8), fake(16, 7), fake(16, 8)), ValueError, "w_gate has the shape"),
    (lambda: ff.gated_feed_forward(fake(4, 8), fake(16, 8), fake(15, 8)), ValueError, "w_up has the shape"),
    (lambda: ff.gated_feed_forward(fake(4, 8), fake(16, 8), fake(16, 8), fake(16, 8)), ValueError, "w_down has the shape"),
    (lambda: ff.gated_feed_forward(fake(4, 8, dtype=torch.bfloat16), fake(16, 8), fake(16, 8)), TypeError, "w_gate is torch.float32"),
    (lambda: ff.gated_feed_forward(fake(4, 8), fake(16, 8), fake(16, 8), activation='tanh'), ValueError, "activation"),
    (lambda: ff.gated_feed_forward(fake(4, 8), fake(16, 8), fake(16, 8), precision='fp8'), ValueError, "precision"),
    (lambda: ff.gated_feed_forward(fake(4, 0), fake(16, 0), fake(16, 0)), ValueError, "no channels"),
    (lambda: ff.point_norm(fake(4, 8), kind='batch'), ValueError, "a norm is one of"),
    (lambda: ff.point_norm(fake(4, 8), kind='none'), ValueError, "a norm is one of"),
    (lambda: ff.point_norm(fake(4, 8), eps=-1.0), ValueError, "eps"),
    (lambda: ff.point_norm(fake(4, 8), eps=float('nan')), ValueError, "eps"),
    (lambda: ff.point_norm(fake(4, 4097)), ValueError, "channels"),
    (lambda: ff.point_norm(fake(4, 8), fake(7)), ValueError, "weight has the shape"),
    (lambda: ff.point_norm(fake(4, 8), fake(8, dtype=torch.float16)), TypeError, "weight is torch.float16"),
    (lambda: ff.norm_gate_residual(fake(4, 8), fake(4, 9)), ValueError, "one shape"),
    (lambda: ff.norm_gate_residual(fake(4, 8), fake(4, 8, dtype=torch.float16)), ValueError, "one shape, type"),
    (lambda: ff.norm_gate_residual(fake(2, 8, 3), fake(2, 8, 3), gate=fake(3, 8)), ValueError, "gate has the shape"),
    (lambda: ff.norm_gate_residual(fake(4, 8), fake(4, 8), next_weight=fake(8)), ValueError, "not asked for"),
    (lambda: ff.norm_gate_residual(fake(4, 8), fake(4, 8), p=1.5), ValueError, "probability"),
    (lambda: ff.norm_gate_residual(fake(4, 8), fake(4, 8), p=0.5), TypeError, "rng"),
    (lambda: ff.norm_gate_residual(fake(4, 8), fake(4, 8), next_kind='none'), ValueError, "a norm is one of"),
    (lambda: ff.dropout(fake(4), -0.1, None), ValueError, "probability"),
    (lambda: ff.dropout(fake(4), float('nan'), None), ValueError, "probability"),
    (lambda: ff.dropout(fake(4), 0.5, torch.zeros(2)), TypeError, "int64"),
    (lambda: ff.dropout(fake(4), 0.5, torch.zeros(4, dtype=torch.int64)[::2]), TypeError, "dense"),
    (lambda: ff.dropout(fake(4, dtype=torch.int32), 0.5, None), TypeError, "float32, bfloat16 or float16"),
    (lambda: ff.CounterRng(2 ** 64, 'cpu'), ValueError, "64 bits"),
    (lambda: ff.CounterDropout(2.0), ValueError, "probability"),
    (lambda: ff.GatedFeedForward(8, 16, activation='tanh'), ValueError, "activation"),
    (lambda: ff.FeedForwardBlock(8, 16, pre_norm='none'), ValueError, "norms are"),
])
def test_python_arguments_are_checked(call, error, text):
    with pytest.raises(error, match=text):
        call()


def _block(**kw):
    base = dict(B=2, N=3, C=8, dtype=0, kind=1, next_kind=0, residual_scale=1.0, eps=1e-6, next_eps=1e-6)
    return _lib.NormResidual(**{**base, **kw})


def test_c_entries_return_codes_and_say_why():
    """No pointer is followed before the checks have passed (the addresses here are not addresses)."""
    lib = _lib.lib()

    def refused(rc, code, text):
        assert rc == code and text in lib.cl3d_last_error_string().decode(), (rc, lib.cl3d_last_error_string())

    a = 1 << 20  # a 16-byte aligned number
    ffn = lambda *args: lib.cl3d_gated_ffn_fwd(*args)  # noqa: E731
    refused(ffn(a, a, a, a, 3, 0, 1, 8, 4, 16, 0, 0, a, None, a, 0, None), -1, "element type")
    refused(ffn(a, a, a, a, 1, 2, 1, 8, 4, 16, 0, 0, a, None, a, 0, None), -1, "memory order")
    refused(ffn(a, a, a, a, 1, 0, 1, 8, 4, 16, 3, 0, a, None, a, 0, None), -1, "activation")
    refused(ffn(a, a, a, a, 1, 0, 1, 8, 4, 16, 0, 2, a, None, a, 0, None), -1, "precision")
    refused(ffn(a, a, a, a, 1, 0, 1, 0, 4, 16, 0, 0, a, None, a, 0, None), -1, "bad sizes")
    refused(ffn(a, a, a, a, 1, 0, 1, 1 << 21, 4, 16, 0, 0, a, None, a, 0, None), -4, "sizes outside")
    refused(ffn(None, a, a, a, 1, 0, 1, 8, 4, 16, 0, 0, a, None, a, 0, None), -1, "null pointer")
    refused(ffn(a + 2, a, a, a, 1, 0, 1, 8, 4, 16, 0, 0, a, None, a, 0, None), -1, "16 bytes")
    refused(ffn(a, a, a, a, 1, 0, 1, 8, 4, 16, 0, 0, a, None, a, 8, None), -3, "bytes of scratch")
    assert ffn(None, None, None, None, 1, 0, 0, 8, 4, 16, 0, 0, None, None, None, 0, None) == 0  # no clouds: nothing to do
    refused(ffn(a, a, a, a, 1, 0, 1, 8, 4, 16, 0, 0, a, a, a, 0, None), -1, "no hidden activations")  # few points
    refused(ffn(a, a, a, None, 1, 0, 1, 8, 400, 16, 0, 0, a, a, a, 0, None), -1, "no hidden activations")  # no last product
    bwd = lambda *args: lib.cl3d_gated_ffn_bwd(*args)  # noqa: E731
    refused(bwd(a, a, a, None, a, None, 1, 0, 1, 8, 4, 16, 0, 0, a, a, a, a, a, 0, None), -1, "not there")
    refused(bwd(a, a, a, a, a, None, 1, 0, 0, 8, 4, 16, 0, 0, a, a, a, a, a, 0, None), -1, "no points")
    refused(bwd(a, a, a, a, a, None, 1, 0, 1, 8, 4, 16, 0, 0, a, a, a, a, a, 0, None), -3, "bytes of scratch")
    assert bwd(a, a, a, a, a, None, 1, 0, 1, 8, 4, 16, 0, 0, None, None, None, None, None, 0, None) == 0  # nothing wanted

    norm = lambda p: lib.cl3d_norm_residual_fwd(ctypes.byref(p), None)  # noqa: E731
    assert lib.cl3d_norm_residual_fwd(None, None) == -1
    refused(norm(_block(dtype=5, x=a, y=a, out=a)), -1, "element type")
    refused(norm(_block(C=0, x=a, y=a, out=a)), -1, "bad sizes")
    refused(norm(_block(kind=3, x=a, y=a, out=a)), -1, "unknown norm")
    refused(norm(_block(x=a)), -1, "neither a block")
    refused(norm(_block(x=a, next_kind=1, gate=a, next=a)), -1, "not there")
    refused(norm(_block(C=4097, x=a, y=a, out=a)), -4, "channels")
    refused(norm(_block(p=0.5, x=a, y=a, out=a)), -1, "generator state")
    refused(norm(_block(p=-0.5, rng=a, x=a, y=a, out=a)), -1, "probability")
    refused(norm(_block(x=a, y=a)), -1, "null pointer")
    refused(norm(_block(B=70000, gate_cloud=1, gate=a, x=a, y=a, out=a)), -4, "65535 clouds")
    refused(norm(_block(x=a, y=a, out=a, stats=a + 8)), -1, "16 bytes")
    nb = lambda p: lib.cl3d_norm_residual_bwd(ctypes.byref(p), None)  # noqa: E731
    refused(nb(_block(x=a, y=a, stats=a)), -1, "null pointer")
    refused(nb(_block(x=a, y=a, stats=a, dnext=a)), -1, "was not formed")
    refused(nb(_block(x=a, next_kind=1, stats=a, dout=a)), -1, "was not formed")
    refused(nb(_block(x=a, y=a, weight=a, stats=a, dout=a, dweight=a)), -3, "bytes of scratch")

    refused(lib.cl3d_dropout(a, 4, 8, 0.5, a, a, None), -1, "element type")
    refused(lib.cl3d_dropout(a, 0, -1, 0.5, a, a, None), -1, "bad size")
    refused(lib.cl3d_dropout(a, 0, 8, 1.5, a, a, None), -1, "probability")
    refused(lib.cl3d_dropout(a, 0, 8, 0.5, None, a, None), -1, "generator state")
    refused(lib.cl3d_dropout(None, 0, 8, 0.5, a, a, None), -1, "null pointer")
    assert lib.cl3d_dropout(None, 0, 0, 0.5, a, None, None) == 0
    refused(lib.cl3d_rng_take(a, 4, a, None), -1, "into the state itself")
    refused(lib.cl3d_rng_take(a, -1, a + 16, None), -1, "bad size")
    refused(lib.cl3d_transpose16(None, 1, 2, 2, a, None), -1, "null pointer")
    refused(lib.cl3d_transpose16(a, 70000, 2, 2, a, None), -4, "65535 clouds")


def test_norm_argument_block_matches_the_header(tmp_path):
    """cl3d_norm_residual against its ctypes mirror, as the C compiler lays the header's struct out."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [n for n, _ in _lib.NormResidual._fields_]
    src = tmp_path / "offsets.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "cl3d.h"\nint main(void) {\n'
                   + '  printf("%zu\\n", sizeof(cl3d_norm_residual));\n'
                   + "".join(f'  printf("%zu\\n", offsetof(cl3d_norm_residual, {n}));\n' for n in names) + "  return 0;\n}\n")
    exe = tmp_path / "offsets"
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), "-o", str(exe), str(src)])
    got = [int(v) for v in subprocess.check_output([str(exe)], text=True).split()]
    assert got == [ctypes.sizeof(_lib.NormResidual)] + [getattr(_lib.NormResidual, n).offset for n in names]


# ----------------------------------------------------------------------------------------------------- the references
def test_generator_against_its_published_vectors():
    """Philox 4x32-10 of the all-zero counter and key, and of the all-one key's low half of the paper's scheme."""
    assert [hex(int(v)) for v in ref.words(0, 0, 4)] == ['0x6627e8d5', '0xe169c58d', '0xbc57ac4c', '0x9b00dbd8']


def _double(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape))


@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("down", [True, False])
def test_feed_forward_reference_is_the_gradient_of_its_formula(kind, down):
    rng = np.random.default_rng(0)
    x, wg, wu, wd = _double(rng, 7, 5), _double(rng, 6, 5), _double(rng, 6, 5), _double(rng, 5, 6)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu}[kind]
    y = act(x @ wg.t()) * (x @ wu.t())
    y = y @ wd.t() if down else y
    dy = _double(rng, *y.shape)
    grads = torch.autograd.grad(y, leaves[:4 if down else 3], dy)
    got = ref.ffn(*[t.detach() for t in (x, wg, wu)], wd.detach() if down else None, kind, dy)
    for name, want in zip(("dx", "dwg", "dwu", "dwd"), grads):
        assert torch.allclose(got[name][0], want, rtol=1e-12, atol=1e-12), name
    assert torch.allclose(got["y"][0], y)


@pytest.mark.parametrize("kind, next_kind", [("rms", "rms"), ("layer", None), ("none", "layer"), ("layer", "layer")])
@pytest.mark.parametrize("clouds", [0, 3])
def test_norm_reference_is_the_gradient_of_its_formula(kind, next_kind, clouds):
    rng = np.random.default_rng(1)
    R, C, p = 6, 5, 0.25
    x, y, w, b, w2, b2 = (_double(rng, *s).requires_grad_(True) for s in ((R, C), (R, C), (C,), (C,), (C,), (C,)))
    gate = _double(rng, *((clouds, C) if clouds else (C,))).requires_grad_(True)
    mask = ref.keep(3, 9, p, (R, C))

    def normed(v, k):
        if k == 'none':
            return v
        if k == 'layer':
            return torch.nn.functional.layer_norm(v, (C,), eps=1e-6)
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6)

    n = (normed(y, kind) * w + b) * mask / (1 - p)
    o = 0.7 * x + (gate.repeat_interleave(2, 0) if clouds else gate) * n
    dout, dnext = _double(rng, R, C), _double(rng, R, C)
    outs, given = [o], [dout]
    if next_kind:
        outs.append(normed(o, next_kind) * w2 + b2)
        given.append(dnext)
    leaves = {"dx": x, "dy": y, "dweight": w, "dbias": b, "dgate": gate}
    if next_kind:
        leaves.update(dnext_weight=w2, dnext_bias=b2)
    grads = torch.autograd.grad(outs, list(leaves.values()), given)
    got = ref.norm(x.detach(), y.detach(), w.detach(), b.detach(), gate.detach(), 0.7, kind, 1e-6, mask, p, next_kind, w2.detach(),
                   b2.detach(), dout, dnext if next_kind else None, clouds=clouds or 1)
    for name, want in zip(leaves, grads):
        assert torch.allclose(got[name][0], want, rtol=1e-11, atol=1e-11), name
    assert torch.allclose(got["out"][0], o)


def test_gradients_of_the_references_against_differences():
    """A central difference of the 64-bit formulas along a random direction, both at h and h / 2: they agree with the gradient to
    the difference's own third-order error."""
    rng = np.random.default_rng(2)
    x, wg, wu, wd, dy = _double(rng, 7, 5), _double(rng, 6, 5), _double(rng, 6, 5), _double(rng, 5, 6), _double(rng, 7, 5)
    args, names = [x, wg, wu, wd], ["dx", "dwg", "dwu", "dwd"]
    grads = ref.ffn(*args, "silu", dy)
    for i, name in enumerate(names):
        v = _double(rng, *args[i].shape)

        def loss(h):
            moved = [a + h * v if k == i else a for k, a in enumerate(args)]
            return float((ref.ffn(*moved, "silu")["y"][0] * dy).sum())

        d1, d2 = ((loss(h) - loss(-h)) / (2 * h) for h in (1e-3, 5e-4))
        want = float((grads[name][0] * v).sum())
        # the error of d2 is a third of d1 - d2 (fourth order aside); 1e-9 for the cancellation
        assert abs(d2 - want) <= abs(d1 - d2) * 0.5 + 1e-9 * max(1.0, abs(want)), (name, d1, d2, want)


def test_a_module_keeps_its_generator_of_each_device(monkeypatch):
    """Going back to a device goes on with its numbers."""
    made = []

    class Rng:
        def __init__(self, seed, device):
            made.append((seed, device))

        def take(self, n):
            return made, n

    monkeypatch.setattr(ff, "CounterRng", Rng)
    draws = ff._Draws(5)
    here, there = torch.empty(3), torch.empty(4, device="meta")
    for x in (here, there, here, there):
        assert draws.take(x)[1] == x.numel()
    assert made == [(5, here.device), (5, there.device)]

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
    from torch.fx.experimental.proxy_tensor import make_fx
    x, calls = _calls()
    rng = ff.CounterRng(5, "cuda")
    calls["to_point_major"] = lambda t: ff.to_point_major(t.contiguous())
    calls["take"] = lambda t: t * rng.take(8)[0]
    for grad in (False, True):
        with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(calls[name], (x.clone().requires_grad_(grad),), check_trace=False)
        with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="traced"):
            make_fx(calls[name])(x.clone().requires_grad_(grad))
    assert rng.state.tolist() == [5, 0]


# --------------------------------------------------------------------------------------------------------- f32 at f32 accuracy
def test_an_f32_product_is_as_good_as_one():
    """One product of two f32 values, in h = relu(a b) * 1 (the other terms of every sum are zero), against 64 bits.

    The kernel forms six of the nine products of two values of three planes.  What it leaves out is at most 2^-24 of |a b|: a plane
    holds 8 bits and is rounded to nearest, so the second is at most 2^-8 of the value and the third 2^-17, and the products left
    out are second by third (twice) and third by third.  Six additions in f32, the largest last: at most a step (2^-23) of the
    result for the last one, whichever way it rounds, and of its 2^-7 th part for the five before.  The sum is below 1.6 x 2^-23."""
    g = gen(4)
    R, H = 96, 512
    a, b = torch.randn((R,), device="cuda", generator=g).abs() + 0.25, torch.randn((H,), device="cuda", generator=g).abs() + 0.25
    worst = torch.tensor([0x3f80ffff, 0x3f81ffff, 0x3fffffff, 0x3f807fff, 0x3f808000, 0x3fff8000, 0x3f800001], dtype=torch.int32, device="cuda")
    a[:7] = b[:7] = worst.view(torch.float32)
    x = torch.stack([a, torch.ones_like(a)], 1)
    w_gate, w_up = torch.stack([b, torch.zeros_like(b)], 1), torch.stack([torch.zeros_like(b), torch.ones_like(b)], 1)
    h = ff.gated_feed_forward(x, w_gate, w_up, activation='relu').double()
    want = a.double()[:, None] * b.double()[None]
    off = ((h - want) / want).abs() * 2.0 ** 23
    assert float(off.max()) <= 1.6, float(off.max())


def test_f32_values_at_the_ends_of_their_range():
    """The largest finite values (a leading plane that rounded up would be an infinity) and the smallest normal ones, each through a
    product by one: the value itself."""
    ends = ["0x1.fffffep127", "0x1.ff0002p127", "0x1.fep127", "0x1p-126", "0x1.8p-126", "0x1.00fffep0", "0x1.fffffep-100"]
    v = torch.tensor([float.fromhex(s) for s in ends], device="cuda")
    n = len(ends)
    x = torch.zeros((80, n + 1), device="cuda")
    x[:n, :n] = torch.diag(v)
    x[:, n] = 1.0  # for the second projection
    w_gate, w_up = torch.zeros((n, n + 1), device="cuda"), torch.zeros((n, n + 1), device="cuda")
    w_gate[:, :n] = torch.eye(n, device="cuda")
    w_up[:, n] = 1.0
    h = ff.gated_feed_forward(x, w_gate, w_up, activation='relu')
    assert torch.equal(h[:n], torch.diag(v)) and not h[n:].any()


# -------------------------------------------------------------------------------------------- what is not finite, without a norm
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("order", ["point", "channel"])
@pytest.mark.parametrize("size", [(1, 40, 70), (2, 33, 21), (1, 1024, 19), (3, 8, 5)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_around_what_is_not_finite(size, order, kind):
    """kind 'none': the gradient of y does not depend on y, whatever y is; a dropped element adds nothing to a parameter's gradient;
    an infinity that stays makes its column's gradient an infinity of the right sign, also in the last point (where idle lanes
    work on the same point)."""
    B, C, N = size
    dtype, g = TYPES[kind], gen(5)
    rng = torch.tensor([11, 7], device="cuda")
    x, y = features(g, B, C, N, dtype, order), features(g, B, C, N, dtype, order)
    bad = y.clone(memory_format=torch.preserve_format)
    places = [(B - 1, 3, N - 1, float('inf')), (B - 1, 5, N - 1, float('-inf')), (0, 6, 1, float('inf')), (0, 7, 2, float('nan'))]
    for b, c, n, value in places:
        bad[b, c, n] = value
        y[b, c, n] = 0.0
    w, gate = vector(g, C, dtype=dtype, mean=2.0), vector(g, C, dtype=dtype, mean=2.0)
    given = features(g, B, C, N, dtype, order)
    mask = ref.keep(11, 7, 0.5, (B * N, C)).reshape(B, N, C)
    for p in (0.0, 0.5):
        def grads(y):
            leaves = [t.detach().requires_grad_(True) for t in (x, y, w, gate)]
            o = ff.norm_gate_residual(leaves[0], leaves[1], leaves[2], gate=leaves[3], kind='none', p=p, rng=rng)
            return torch.autograd.grad(o, leaves, given)
        want, got = grads(y), grads(bad)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        sums = {}
        for b, c, n, value in places:
            if p == 0 or bool(mask[b, n, c]):
                sums[c] = value
        other = [c for c in range(C) if c not in sums]
        for k, coefficient in ((2, gate), (3, w)):
            assert torch.equal(got[k][other], want[k][other]), (p, k)
            for c, value in sums.items():
                b, n = next((b, n) for b, cc, n, _ in places if cc == c)
                sign = float(given[b, c, n]) * float(coefficient[c])
                assert float(got[k][c].float()) == sign * value or value != value and bool(got[k][c].isnan()), (p, k, c)


# -------------------------------------------------------------------------------------------------------------------- dropout
def test_a_generator_that_moved_on_is_noticed():
    """A draw from the generator's own state tensor: take() changes it, and the backward pass says so."""
    rng = ff.CounterRng(9, "cuda")
    x = torch.randn((40,), device="cuda", requires_grad=True)
    y = ff.dropout(x, 0.5, rng.state)
    kept = rng.take(8)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [x], torch.ones_like(y))
    y = ff.dropout(x, 0.5, kept)
    rng.take(8)  # (a draw of its own is not touched by the next)
    (d,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    assert torch.equal(d != 0, y != 0)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("size", [(1, 1, 1), (1, 8, 1), (3, 5, 2), (2, 24, 3), (2, 33, 4), (1, 72, 65), (3, 144, 77), (2, 201, 130), (1, 2304, 9),
                                  (70, 3, 31), (1, 2, 5001)], ids=lambda s: "x".join(map(str, s)))
def test_dropout_of_point_major_features(size, kind):
    """The elements are numbered by the dimensions and the result lies as x does: the values of the dense call, in x's order; the
    gradient, for one in either order, too."""
    B, C, N = size
    dtype, g = TYPES[kind], gen(6)
    rng = torch.tensor([2 ** 40 + 3, 2 ** 32 - 2], device="cuda")
    x, d = features(g, B, C, N, dtype), features(g, B, C, N, dtype)
    leaf = x.detach().requires_grad_(True)
    dense = x.contiguous().requires_grad_(True)
    for p in (0.3, 1.0):
        y, want = ff.dropout(leaf, p, rng), ff.dropout(dense, p, rng)
        assert torch.equal(y, want) and y.stride() == torch.empty_like(x).stride()
        (dw,) = torch.autograd.grad(want, [dense], d.contiguous())
        for given in (d, d.contiguous()):
            (dx,) = torch.autograd.grad(y, [leaf], given, retain_graph=True)
            assert torch.equal(dx, dw)
    off = torch.zeros((x.numel() + 1,), dtype=dtype, device="cuda")[1:].view(B, N, C).transpose(1, 2).copy_(x)  # (off 16 bytes)
    assert torch.equal(ff.dropout(off, 0.3, rng), ff.dropout(dense.detach(), 0.3, rng))
    bad = torch.full_like(x, float('nan'))
    assert torch.equal(ff.dropout(bad, 0.3, rng).isnan(), ref.keep(2 ** 40 + 3, 2 ** 32 - 2, 0.3, (B, C, N)).cuda())


def test_dropout_in_a_chain_keeps_its_order():
    """Point-major features through the operators of a block and dropout: no result of the chain changes its order."""
    g = gen(7)
    rng = torch.tensor([1, 0], device="cuda")
    x, ws = ffn_inputs(g, 2, 40, 30, 64, torch.bfloat16)
    y = ff.dropout(ff.gated_feed_forward(ff.point_norm(x), *ws), 0.2, rng)
    out = ff.dropout(ff.norm_gate_residual(x, y), 0.2, rng)
    for t in (y, out):
        assert ff._point_major(t) and not t.is_contiguous()


# ----------------------------------------------------------------------------------------------------------- the widest stages
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("size", [(1, 4608, 5), (2, 4104, 3), (1, 5120, 2), (3, 6144, 1), (1, 4608, 1030)], ids=lambda s: "x".join(map(str, s)))
def test_norms_of_the_widest_stages(size, kind):
    """A backbone of width 288 ends in 4608 channels: above 4096, multiples of 8 up to 6144."""
    norm_check(size, kind, "layer", "rms", "cloud", 0.25, "point", kind)
    if size[2] < 100:
        norm_check(size, kind, "none", "layer", "channel", 0.0, "channel", "f32", bias=False)
        norm_check(size, kind, "rms", None, "none", 0.5, "point", kind, bias=False)


def test_parameters_of_a_wide_norm_need_not_be_aligned():
    g = gen(8)
    x = vector(g, 6, 4608, dtype=torch.bfloat16)
    w = vector(g, 4609, dtype=torch.bfloat16)
    assert torch.equal(ff.point_norm(x, w[1:]), ff.point_norm(x, w[1:].clone()))


def test_feed_forward_block_of_the_widest_stage():
    g = gen(9)
    block = ff.FeedForwardBlock(4608, 64, post_norm='layer', dropout=0.1, seed=3).cuda()
    x = features(g, 1, 4608, 9, torch.float32, "channel").requires_grad_(True)
    y = block(x)
    grads = torch.autograd.grad(y, [x] + list(block.parameters()), torch.ones_like(y))
    with torch.no_grad():
        h = ff.point_norm(x, block.pre_weight, None, 'rms', block.eps)
        want = ff.norm_gate_residual(x, block.feed_forward(h), block.post_weight, block.post_bias, block.gate, 1.0, 'layer', block.eps, 0.1,
                                     torch.tensor([3, 0], device="cuda"))
    # (the same kernels on the other memory order: the same bits)
    assert torch.equal(y, want) and all(bool(t.isfinite().all()) and t.shape == s.shape for t, s in zip(grads, [x] + list(block.parameters())))


# ------------------------------------------------------------------------------------------------------------- clouds of millions
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_memory_orders_of_a_cloud_of_millions(kind):
    """2 200 000 points x 72 channels: there, back, and a feed-forward in either order."""
    B, C, N = 1, 72, 2200000
    x = vector(gen(10), B, C, N, dtype=TYPES[kind])
    y = ff.to_point_major(x)
    assert ff._point_major(y) and torch.equal(y, x)
    assert torch.equal(ff.to_channel_major(y), x)
    ws = [vector(gen(11), 8, C, dtype=TYPES[kind], std=0.1), vector(gen(12), 8, C, dtype=TYPES[kind], std=0.1), vector(gen(13), C, 8, dtype=TYPES[kind])]
    assert torch.equal(ff.gated_feed_forward(x, *ws), ff.gated_feed_forward(y, *ws))


# ------------------------------------------------------------------------------------------------------------------ long sums
# up to 64 points, one, two and more turns of the direct kernel's loop over k (1024 elements of 16 bits, half as many of 32, half of
# either above 32 points), whole vectors and ragged; above, sums and tiles past every listed training width
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("size", [(1, 1160, 1, 2320), (16, 2304, 1, 4608), (1, 513, 17, 1025), (33, 1031, 1, 2057), (64, 545, 1, 1100), (4, 2056, 16, 1032),
                                  (2, 520, 31, 264)], ids=lambda s: "x".join(map(str, s)))
def test_few_points_of_many_channels(size, kind):
    B, C, N, H = size
    dtype, g = TYPES[kind], gen(14)
    order = "channel" if N > 1 and C % 2 else "point"
    x, ws = ffn_inputs(g, B, C, N, H, dtype, order)
    ffn_check(x, ws, ["silu", "gelu", "relu"][(C + N) % 3], dtype, features(g, B, C, N, dtype, order), order, tag=(size, kind))


@pytest.mark.parametrize("kind, precision, size", [("bf16", "f32", (130, 2304, 1, 4608)), ("f16", "f32", (1, 1153, 200, 2305)), ("f32", "f32", (2, 1153, 100, 2305)),
                                                   ("f32", "bf16", (1, 2304, 256, 1160)), ("bf16", "f32", (2, 577, 513, 1152)),
                                                   ("f32", "f32", (1, 576, 1030, 1152))], ids=str)
def test_wide_products_and_their_gradients(kind, precision, size):
    B, C, N, H = size
    dtype, g = TYPES[kind], gen(15)
    order = "channel" if N > 1 and C % 2 else "point"
    x, ws = ffn_inputs(g, B, C, N, H, dtype, order)
    ffn_check(x, ws, "gelu" if C % 2 else "silu", dtype, features(g, B, C, N, dtype, order), order, precision, tag=(size, kind))


def test_wide_projections_alone():
    for kind, size in (("bf16", (16, 2304, 1, 4608)), ("f32", (33, 1031, 1, 2057)), ("f16", (130, 1153, 1, 2305))):
        B, C, N, H = size
        g = gen(16)
        x, ws = ffn_inputs(g, B, C, N, H, TYPES[kind], down=False)
        ffn_check(x, ws, "gelu", TYPES[kind], features(g, B, H, N, TYPES[kind]), "point", tag=(kind, size))


# --------------------------------------------------------------------------------------------------------------- as they are used
@pytest.mark.parametrize("precision", ["f32", "bf16"])
def test_a_whole_model_with_feed_forward_blocks_is_captured(precision):
    """A classifier whose bottlenecks end in feed-forward blocks and whose head drops by the counter: a training step, captured with
    its backward pass, gives in every replay what the eager step gives from the same numbers."""
    import closerlook3d_amd
    from closerlook3d_amd import compat
    torch.manual_seed(0)
    cfg = compat.default_config()
    cfg.width, cfg.nsamples, cfg.npoints, cfg.radius, cfg.sampleDl = 24, [8] * 5, [128, 64, 32, 16], 0.2, 0.08
    cfg.cl3d_feed_forward, cfg.cl3d_feed_forward_dropout, cfg.cl3d_counter_dropout, cfg.cl3d_precision = 2.0, 0.2, True, precision
    model = compat.build_model(cfg, 'classification').cuda().train()
    draws = [m._draws for m in model.modules() if hasattr(m, "_draws")]
    assert len(draws) > 8
    g = gen(17)
    xyz = torch.rand((4, 512, 3), device="cuda", generator=g)
    mask = torch.ones((4, 512), dtype=torch.int32, device="cuda")
    features = torch.randn((4, 3, 512), device="cuda", generator=g)
    probe = torch.randn((4, cfg.num_classes), device="cuda", generator=g)
    params = list(model.parameters())
    buffers = [b for b in model.buffers()]
    start = [b.clone() for b in buffers]

    def step():
        for b, s in zip(buffers, start):
            b.copy_(s)
        out = model(xyz, mask, features)
        return [out] + list(torch.autograd.grad(out, params, probe))

    def at(n):
        for d in draws:
            d.rng.state[1] = n

    side = closerlook3d_amd.step_stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
        wants = []
        for n in (0, 500, 1000):
            at(n)
            wants.append([t.detach().clone() for t in step()])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert not torch.equal(wants[0][0], wants[1][0])
    graph = torch.cuda.CUDAGraph()
    with closerlook3d_amd.whole_step_capture(), torch.cuda.graph(graph, stream=side):
        static = step()
    for turn in range(2):
        for n, want in zip((0, 500, 1000), wants):
            at(n)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for k, (a, b) in enumerate(zip(static, want)):
                assert bool(a.isfinite().all()) and torch.equal(a, b), (turn, n, k)


@pytest.mark.parametrize("reentrant", [True, False])
def test_a_draw_made_again_in_a_backward_pass_is_refused(reentrant):
    """Activation checkpointing runs a module a second time, which would draw another mask than the forward pass had; numbers drawn
    outside give the gradients of the mask that was."""
    from torch.utils.checkpoint import checkpoint
    g = gen(18)
    x = features(g, 2, 24, 30, torch.float32).detach().requires_grad_(True)
    block = ff.FeedForwardBlock(24, 48, dropout=0.5, seed=1).cuda()
    drop = ff.CounterDropout(0.5, seed=2)
    for module in (block, drop):
        y = checkpoint(module, x, use_reentrant=reentrant)
        with pytest.raises(RuntimeError, match="draws its own numbers"):
            torch.autograd.backward(y, torch.ones_like(y))
        assert torch.autograd.grad(module(x).sum(), [x])[0].shape == x.shape
    rng = torch.tensor([4, 0], device="cuda")
    x.grad = None
    y = checkpoint(lambda t: ff.dropout(ff.point_norm(t), 0.5, rng), x, use_reentrant=reentrant)
    y.sum().backward()
    (want,) = torch.autograd.grad(ff.dropout(ff.point_norm(x), 0.5, rng).sum(), [x])
    assert torch.equal(x.grad, want)
    block.eval()
    checkpoint(block, x, use_reentrant=reentrant).sum().backward()


@pytest.mark.parametrize("name", ["gated_feed_forward", "point_norm", "norm_gate_residual", "norm_gate_residual_next"])
def test_a_derivative_of_a_gradient_is_refused_and_not_zero(name):
    """A penalty on the gradients of a constant sum beside another term: without the refusal the penalty's part would silently be
    nothing."""
    x, calls = _calls()
    scale = torch.full((24,), 2.0, device="cuda", requires_grad=True)
    if name == "norm_gate_residual":
        calls[name] = lambda t: ff.norm_gate_residual(t, t, gate=scale, kind='none')  # (its gradient is the gate's, not x's)
    x = x.requires_grad_(True)
    (g,) = torch.autograd.grad(calls[name](x).sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        ((g * g).sum() + (x * x).sum() + (scale * scale).sum()).backward()
    (plain,) = torch.autograd.grad(calls[name](x).sum(), [x])
    assert torch.equal(g, plain) and not plain.requires_grad


def test_second_derivatives_that_are_zero_are_zero():
    """Dropout, a memory order and a sum without parameters are linear: their gradient does not depend on x."""
    x, calls = _calls()
    x = x.contiguous().requires_grad_(True)
    rng = torch.tensor([3, 0], device="cuda")
    for call in (calls["dropout"], ff.to_point_major, lambda t: ff.norm_gate_residual(t, t, kind='none', p=0.3, rng=rng)):
        (g,) = torch.autograd.grad(call(x).sum(), [x], create_graph=True)
        (d,) = torch.autograd.grad((g * x).sum(), [x])
        assert torch.equal(d, g)

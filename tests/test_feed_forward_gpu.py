"""GPU: the feed-forward operators against their formulas in 64 bits (ff_reference: values and derived bounds)."""
import copy

import pytest
import torch

from closerlook3d_amd import feed_forward as ff
from tests import ff_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", [(1, 8, 8), (3, 16, 264), (2, 72, 520), (2, 144, 70), (1, 201, 65), (2, 2, 300), (70, 64, 1000)],
                         ids=lambda s: "x".join(map(str, s)))
def test_memory_orders_there_and_back(size, kind):
    x = torch.randn(size, device="cuda", generator=gen(1)).to(TYPES[kind])
    y = ff.to_point_major(x)
    assert ff._point_major(y) and torch.equal(y, x)
    z = ff.to_channel_major(y)
    assert z.is_contiguous() and torch.equal(z, x)
    off = torch.zeros((x.numel() + 1,), dtype=x.dtype, device="cuda")[1:].view(size).copy_(x)  # (starts off 16 bytes)
    assert torch.equal(ff.to_point_major(off), x)


def features(g, B, C, N, dtype, order="point", scale=1.0):
    rows = (torch.randn((B, N, C), device="cuda", generator=g) * scale).to(dtype)
    return rows.transpose(1, 2) if order == "point" else rows.transpose(1, 2).contiguous()


def rows(t):
    """Point-major rows of features, in 64 bits."""
    return (t if t.dim() == 2 else t.transpose(1, 2).reshape(-1, t.shape[1])).detach().double()


def vector(g, *shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, device="cuda", generator=g) * std + mean).to(dtype)


def ffn_inputs(g, B, C, N, H, dtype, order="point", down=True):
    x = features(g, B, C, N, dtype, order)
    ws = [vector(g, H, C, dtype=dtype, std=C ** -0.5), vector(g, H, C, dtype=dtype, std=C ** -0.5),
          vector(g, C, H, dtype=dtype, std=H ** -0.5) if down else None]
    return x, ws


def ffn_check(x, ws, act, dtype, dy, order, precision="f32", tag=""):
    leaves = [t.requires_grad_(True) for t in [x] + ws if t is not None]
    y = ff.gated_feed_forward(*([x] + ws), activation=act, precision=precision)
    grads = torch.autograd.grad(y, leaves, dy)
    want = ref.ffn(rows(x), *[None if w is None else w.detach().double() for w in ws], act, rows(dy), dtype,
                   torch.bfloat16 if precision == "bf16" else dtype)
    assert y.dtype == dtype and (y.dim() == 2 or ff._order(y)[1] == ff._order(x)[1])
    ref.check(rows(y), want["y"], (tag, "y"))
    ref.check(rows(grads[0]), want["dx"], (tag, "dx"))
    for name, g in zip(("dwg", "dwu", "dwd"), grads[1:]):
        assert g.dtype == dtype
        ref.check(g, want[name], (tag, name))
    return y, grads


# one point, a wave's rows and its neighbours, tiles' ends; channels that no vector, wave or tile divides
SIZES = [(1, 8, 1, 8), (1, 1, 1, 1), (3, 24, 5, 33), (1, 37, 15, 64), (1, 64, 16, 130), (2, 144, 9, 71), (1, 72, 33, 96), (16, 36, 4, 128),
         (1, 201, 129, 95), (2, 144, 150, 576), (1, 130, 515, 257), (1, 8, 2049, 40), (5, 288, 64, 192)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_feed_forward_matches_its_formula(size, kind):
    B, C, N, H = size
    dtype, g = TYPES[kind], gen(1)
    order = "point" if (B + C) % 2 else "channel"
    x, ws = ffn_inputs(g, B, C, N, H, dtype, order)
    ffn_check(x, ws, ["silu", "gelu", "relu"][(C + N) % 3], dtype, features(g, B, C, N, dtype, order), order, tag=(size, kind))


# many narrow points: the forward pass in one kernel, at the widths and point counts where it changes its shape
@pytest.mark.parametrize("size", [(1, 24, 32768, 40), (1, 33, 32775, 47), (2, 144, 16385, 96), (1, 160, 33000, 33), (1, 72, 65537, 64),
                                  (1, 200, 32769, 100), (1, 224, 65540, 70), (1, 217, 65536, 31), (1, 225, 32768, 32)],
                         ids=lambda s: "x".join(map(str, s)))
def test_feed_forward_of_many_narrow_points(size):
    B, C, N, H = size
    for kind, precision in (("bf16", "f32"), ("f16", "f32"), ("f32", "bf16")):
        dtype, g = TYPES[kind], gen(16)
        order = "channel" if C % 3 == 0 and kind != "f16" else "point"
        x, ws = ffn_inputs(g, B, C, N, H, dtype, order)
        ffn_check(x, ws, "gelu" if C % 2 else "silu", dtype, features(g, B, C, N, dtype, order), order, precision, tag=(size, kind))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_projections_without_the_last_product(kind, act):
    dtype = TYPES[kind]
    for B, C, N, H, order in ((1, 40, 77, 24, "point"), (3, 21, 34, 50, "channel"), (7, 64, 1, 128, "point")):
        g = gen(2)
        x, ws = ffn_inputs(g, B, C, N, H, dtype, order, down=False)
        ffn_check(x, ws, act, dtype, features(g, B, H, N, dtype, order), order, tag=(kind, act, B))


@pytest.mark.parametrize("size", [(2, 144, 70, 200), (1, 33, 40, 47), (9, 64, 1, 64)], ids=str)
def test_f32_tensors_at_bf16_precision(size):
    B, C, N, H = size
    g = gen(3)
    x, ws = ffn_inputs(g, B, C, N, H, torch.float32, "channel")
    ffn_check(x, ws, "silu", torch.float32, features(g, B, C, N, torch.float32, "channel"), "channel", "bf16")


def test_rows_strides_and_orders_give_the_same_bits():
    """(R, C) rows, features in both orders, a strided view, a slice that starts off 16 bytes, an expanded gradient, a gradient in
    the other order: one result."""
    g = gen(4)
    B, C, N, H = 3, 40, 50, 88
    for dtype in (torch.bfloat16, torch.float32):
        x, ws = ffn_inputs(g, B, C, N, H, dtype)
        dy = features(g, B, C, N, dtype)

        def both(x, dy):
            x = x.detach().requires_grad_(True)
            y = ff.gated_feed_forward(x, *ws)
            return [y, *torch.autograd.grad(y, [x] + [w for w in ws], dy)]

        for w in ws:
            w.requires_grad_(True)
        want = both(x, dy)
        as_rows = lambda t: t.transpose(1, 2).reshape(-1, C)  # noqa: E731
        wide = torch.zeros((B, N, C + 24), dtype=dtype, device="cuda")
        wide[..., 16:16 + C] = x.transpose(1, 2)
        off = torch.zeros((B * N * C + 1,), dtype=dtype, device="cuda")
        off[1:] = x.transpose(1, 2).reshape(-1)
        for xx, dd in ((x.contiguous(), dy.contiguous()), (x, dy.contiguous()), (x.contiguous(), dy),
                       (wide[..., 16:16 + C].transpose(1, 2), dy), (off[1:].view(B, N, C).transpose(1, 2), dy)):
            for a, b in zip(both(xx, dd), want):
                assert torch.equal(a, b)
        got = both(as_rows(x), as_rows(dy))
        for a, b in zip(got, [as_rows(t) if t.dim() == 3 else t for t in want]):
            assert torch.equal(a, b)
        one = torch.ones((1, C, 1), dtype=dtype, device="cuda").expand(B, C, N)
        for a, b in zip(both(x, one), both(x, one.contiguous())):
            assert torch.equal(a, b)
        # weights that are views: transposed storage, a slice of one matrix
        packed = torch.cat([ws[0], ws[1]], 0).detach()
        y = ff.gated_feed_forward(x, packed[:H], packed[H:], ws[2].detach().t().contiguous().t())
        assert torch.equal(y, want[0])


def test_only_the_wanted_gradients_are_formed():
    g = gen(5)
    x, ws = ffn_inputs(g, 2, 48, 60, 72, torch.bfloat16)
    dy = features(g, 2, 48, 60, torch.bfloat16)
    tensors = [x] + ws
    for t in tensors:
        t.requires_grad_(True)
    full = torch.autograd.grad(ff.gated_feed_forward(*tensors), tensors, dy)
    for k in range(4):
        for i, t in enumerate(tensors):
            t.requires_grad_(i == k)
        (got,) = torch.autograd.grad(ff.gated_feed_forward(*tensors), [tensors[k]], dy)
        assert torch.equal(got, full[k]), k
    for t in tensors:
        t.requires_grad_(True)
    with torch.no_grad():
        assert not ff.gated_feed_forward(*tensors).requires_grad


def test_one_tensor_in_several_places():
    """The same matrix as both projections: its gradient is the sum of the two."""
    g = gen(6)
    x, (w, _, wd) = ffn_inputs(g, 1, 32, 40, 64, torch.float32)
    dy = features(g, 1, 32, 40, torch.float32)
    w.requires_grad_(True)
    (got,) = torch.autograd.grad(ff.gated_feed_forward(x, w, w, wd), [w], dy)
    want = ref.ffn(rows(x), w.detach().double(), w.detach().double(), wd.double(), "silu", rows(dy))
    ref.check(got, (want["dwg"][0] + want["dwu"][0], want["dwg"][1] + want["dwu"][1] + 2 * ref.U32 * want["dwg"][0].abs()), "dw")


@pytest.mark.parametrize("shape", [(0, 8, 5), (3, 8, 0), (0, 8)], ids=str)
def test_no_points(shape):
    for dtype in (torch.float32, torch.float16):
        x = torch.zeros(shape, dtype=dtype, device="cuda", requires_grad=True)
        ws = [torch.ones(s, dtype=dtype, device="cuda", requires_grad=True) for s in ((16, 8), (16, 8), (8, 16))]
        y = ff.gated_feed_forward(x, *ws)
        for t, v in zip([x] + ws, torch.autograd.grad(y, [x] + ws, torch.zeros_like(y))):
            assert v.shape == t.shape and not v.any()
        w = torch.ones((8,), dtype=dtype, device="cuda", requires_grad=True)
        o, h = ff.norm_gate_residual(x, x, w, gate=w, next_kind='rms', next_weight=w)
        assert o.shape == x.shape and h.shape == x.shape
        for t, v in zip([x, w], torch.autograd.grad([o, h], [x, w], [torch.zeros_like(o)] * 2)):
            assert v.shape == t.shape and not v.any()
        rng = torch.tensor([1, 2], device="cuda")
        assert ff.dropout(x, 0.5, rng).shape == x.shape


@pytest.mark.parametrize("kind", list(TYPES))
def test_what_is_not_finite_stays_in_its_point(kind):
    """A NaN or an infinity reaches its own point only, and of the weights' gradients what the formula says; the infinity of an f32
    value stays one (its split is not inf - inf)."""
    dtype, g = TYPES[kind], gen(7)
    for R, C, H in ((40, 24, 40), (300, 21, 35), (32800, 40, 45)):
        x, ws = ffn_inputs(g, 1, C, R, H, dtype)
        x = x.transpose(1, 2)[0].contiguous()
        clean = ff.gated_feed_forward(x, *ws)
        bad = x.clone()
        bad[3, 2], bad[17, 0], bad[18, 1] = float('nan'), float('inf'), float('-inf')
        got = ff.gated_feed_forward(bad, *ws, activation='relu')
        clean = ff.gated_feed_forward(x, *ws, activation='relu')
        others = [r for r in range(R) if r not in (3, 17, 18)]
        assert torch.equal(got[others], clean[others])
        assert bool(got[3].isnan().all())
        # relu(+-inf) is inf or 0, times an infinity of either sign: the projections alone follow the formula in kind
        h = ff.gated_feed_forward(bad[17:19], ws[0], ws[1], activation='relu').double()
        gg, uu = bad[17:19].double() @ ws[0].double().t(), bad[17:19].double() @ ws[1].double().t()
        want = torch.relu(gg) * uu
        assert torch.equal(h.isnan(), want.isnan()) and torch.equal(h.isinf(), want.isinf())
        assert torch.equal(h[h.isinf()], want[want.isinf()])


def test_feed_forward_is_the_same_bit_for_bit():
    g = gen(8)
    x, ws = ffn_inputs(g, 4, 72, 700, 288, torch.bfloat16)
    dy = features(g, 4, 72, 700, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in [x] + ws]
    first = None
    for _ in range(5):
        y = ff.gated_feed_forward(*leaves)
        got = [y] + list(torch.autograd.grad(y, leaves, dy))
        first = first or got
        for a, b in zip(got, first):
            assert torch.equal(a, b)


def test_feed_forward_gradients_against_differences():
    """f32: a central difference of the operator's own outputs.  The difference quotient is off by what the same quotient of the
    64-bit formula is off (third order in the step), and by the outputs' bounds over twice the step."""
    g = gen(9)
    x, ws = ffn_inputs(g, 2, 20, 30, 28, torch.float32)
    dy = features(g, 2, 20, 30, torch.float32)
    leaves = [t.requires_grad_(True) for t in [x] + ws]
    grads = torch.autograd.grad(ff.gated_feed_forward(*leaves), leaves, dy)
    step = 2.0 ** -6
    for k, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, device="cuda", generator=g)
        sides, exact, noise = [], [], 0.0
        for h in (step, -step):
            moved = [(t.detach() + h * v if i == k else t.detach()) for i, t in enumerate(leaves)]
            sides.append(float((ff.gated_feed_forward(*moved).double() * dy.double()).sum()))
            y, e = ref.ffn(rows(moved[0]), *[w.double() for w in moved[1:]], "silu")["y"]
            exact.append(float((y * rows(dy)).sum()))
            noise += float((e * rows(dy).abs()).sum())
        have, formula = (sides[0] - sides[1]) / (2 * step), (exact[0] - exact[1]) / (2 * step)
        along = float((grads[k].double() * v.double()).sum())
        assert abs(have - formula) <= noise / (2 * step), (k, have, formula)
        # the 64-bit quotient is off by its third-order term: a quarter of it is left at half the step
        half = []
        for h in (step / 2, -step / 2):
            moved = [(t.detach().double() + h * v.double() if i == k else t.detach().double()) for i, t in enumerate(leaves)]
            half.append(float((ref.ffn(rows(moved[0]), *moved[1:], "silu")["y"][0] * rows(dy)).sum()))
        third = abs(formula - (half[0] - half[1]) / step)
        assert abs(along - formula) <= 2 * third + 1e-4 * abs(formula) + noise, (k, along, formula, third)


# --------------------------------------------------------------------------------------------------------------- norms
def norm_check(size, kind, norm, next_norm, gate, p, order, types, seed=11, offset=0, scale=0.9, bias=True):
    B, C, N = size
    dtype, pt, g = TYPES[kind], TYPES[types], gen(seed)
    x, y = features(g, B, C, N, dtype, order), features(g, B, C, N, dtype, order, 3.0) + 1.0
    vec = lambda m: vector(g, C, dtype=pt, std=0.3, mean=m).requires_grad_(True)  # noqa: E731
    w, b = (vec(1.0), vec(0.0) if bias else None) if norm != 'none' else (None, None)
    gt = {"none": None, "channel": vec(0.5), "cloud": vector(g, B, C, dtype=pt, std=0.3, mean=0.5).requires_grad_(True)}[gate]
    w2, b2 = (vec(1.0), vec(0.0) if bias else None) if next_norm else (None, None)
    rng = torch.tensor([seed * 1000003, offset], device="cuda") if p else None
    x.requires_grad_(True)
    y = y.detach().requires_grad_(True)
    outs = ff.norm_gate_residual(x, y, w, b, gt, scale, norm, 1e-5, p, rng, next_kind=next_norm, next_weight=w2, next_bias=b2)
    outs = outs if next_norm else (outs,)
    given = [features(g, B, C, N, dtype, order) for _ in outs]
    leaves = {"dx": x, "dy": y, "dweight": w, "dbias": b, "dgate": gt, "dnext_weight": w2, "dnext_bias": b2}
    leaves = {k: v for k, v in leaves.items() if v is not None}
    grads = torch.autograd.grad(outs, list(leaves.values()), given)
    wide = lambda t: None if t is None else t.detach().double()  # noqa: E731
    mask = ref.keep(seed * 1000003, offset, p, (B * N, C)).cuda() if p else None
    want = ref.norm(rows(x), rows(y), wide(w), wide(b), wide(gt), scale, norm, 1e-5, mask, p, next_norm, wide(w2), wide(b2),
                    rows(given[0]), rows(given[1]) if next_norm else None, dtype=dtype, clouds=B)
    for name, t in zip(("out", "next"), outs):
        assert t.dtype == dtype and t.shape == x.shape and ff._order(t)[1] == ff._order(x)[1]
        ref.check(rows(t), want[name], (name, size))
    for (name, leaf), t in zip(leaves.items(), grads):
        assert t.dtype == leaf.dtype and t.shape == leaf.shape
        value, bound = want[name]
        if leaf.dtype != dtype:  # a parameter of its own type: its own rounding
            bound = bound - ref.rounding(value, dtype) + ref.rounding(value, leaf.dtype)
        ref.check(rows(t) if t.dim() == 3 else t, (value, bound), (name, size))


NORM_SIZES = [(1, 8, 1), (1, 1, 1), (2, 3, 2), (3, 24, 5), (1, 72, 130), (2, 144, 77), (1, 201, 65), (1, 288, 129), (4, 512, 9),
              (1, 513, 12), (1, 1152, 33), (2, 2304, 3), (1, 2303, 5), (1, 2056, 6), (1, 4096, 4), (1, 4095, 2), (16, 40, 1)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("size", NORM_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_norms_around_a_block_match_their_formula(size, kind):
    B, C, N = size
    k = (B * 7 + C + N) % 4
    norm_check(size, kind, ["rms", "layer", "rms", "none"][k], ["rms", "layer", None, "layer"][k], ["channel", "cloud", "none", "cloud"][k],
               [0.0, 0.25, 0.5, 0.1][k], "point" if (C + N) % 2 else "channel", kind if k % 2 else "f32", offset=C * 1000)


@pytest.mark.parametrize("norm", ["none", "rms", "layer"])
@pytest.mark.parametrize("next_norm", [None, "rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "channel", "cloud"])
def test_every_form_of_the_exit(norm, next_norm, gate):
    norm_check((3, 56, 31), "bf16", norm, next_norm, gate, 0.3, "point", "bf16", bias=norm == "layer")
    norm_check((3, 57, 31), "f32", norm, next_norm, gate, 0.0, "channel", "f32", bias=False)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("size", [(1, 4, 2), (5, 8, 64), (3, 72, 65), (2, 128, 63), (1, 132, 130), (2, 144, 77), (2, 256, 200), (70000, 4, 3),
                                  (2, 260, 70), (2, 126, 70), (70, 288, 300), (9, 512, 40), (3, 772, 33), (2, 1024, 17), (1, 1028, 20), (300, 36, 70),
                                  (300, 200, 70)], ids=lambda s: "x".join(map(str, s)))
def test_channel_major_features_match_their_formula(size, kind):
    """Up to 256 channels, a multiple of four: read as they lie; others by transposed copies."""
    k = (size[1] // 4 + len(kind)) % 3
    norm_check(size, kind, ["rms", "layer", "none"][k], [None, "rms", "layer"][k], ["channel", "none", "channel"][k], [0.0, 0.3, 0.1][k], "channel",
               kind, offset=2 ** 32 - 5, bias=k != 0)
    if size[0] <= 300:
        norm_check(size, kind, "layer", "rms", "cloud", 0.3, "channel", "f32", bias=k == 0)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_entry_norm_matches_its_formula(kind, norm):
    dtype = TYPES[kind]
    for B, C, N, order in ((1, 8, 1, "point"), (2, 36, 50, "channel"), (1, 145, 33, "point"), (3, 1152, 4, "point"), (1, 1, 6, "point")):
        g = gen(12)
        x = (features(g, B, C, N, dtype, order, 2.0) + 0.5).detach().requires_grad_(True)
        w, b = (vector(g, C, dtype=dtype, std=0.3, mean=m).requires_grad_(True) for m in (1.0, 0.0))
        dn = features(g, B, C, N, dtype, order)
        y = ff.point_norm(x, w, b, norm, 1e-5)
        grads = torch.autograd.grad(y, [x, w, b], dn)
        want = ref.norm(rows(x), next_kind=norm, eps=1e-5, next_weight=w.detach().double(), next_bias=b.detach().double(), dnext=rows(dn), dtype=dtype)
        ref.check(rows(y), want["next"], "next")
        ref.check(rows(grads[0]), want["dx"], "dx")
        ref.check(grads[1], want["dnext_weight"], "dnext_weight")
        ref.check(grads[2], want["dnext_bias"], "dnext_bias")


def test_norm_of_a_far_mean_and_of_equal_channels():
    """layer: the variance is taken about the mean (1000 +- 1 loses no more than the subtraction does); equal channels give the bias."""
    g = gen(13)
    x = torch.randn((64, 96), device="cuda", generator=g) + 1000.0
    ref.check(ff.point_norm(x, kind='layer'), ref.norm(x.double(), next_kind='layer')["next"], "far")
    same = torch.full((5, 40), 3.0, device="cuda")
    b = torch.randn((40,), device="cuda", generator=g)
    assert torch.equal(ff.point_norm(same, None, b, 'layer'), b.expand(5, 40))
    assert torch.equal(ff.point_norm(torch.zeros((5, 40), device="cuda"), None, b), b.expand(5, 40))


def test_norm_outputs_used_alone():
    """Either result without the other: its gradient is zero."""
    g = gen(14)
    x, y = (features(g, 2, 48, 20, torch.float32).detach().requires_grad_(True) for _ in range(2))
    w2 = torch.ones((48,), device="cuda", requires_grad=True)
    d = features(g, 2, 48, 20, torch.float32)
    zero = torch.zeros_like(d)

    def grads(which):
        o = ff.norm_gate_residual(x, y, next_kind='rms', next_weight=w2)
        return torch.autograd.grad(o[which], [x, y, w2], d, allow_unused=True)

    both = torch.autograd.grad(ff.norm_gate_residual(x, y, next_kind='rms', next_weight=w2), [x, y, w2], [zero, d])
    for a, b in zip(grads(1), both):
        assert torch.equal(a, b)
    both = torch.autograd.grad(ff.norm_gate_residual(x, y, next_kind='rms', next_weight=w2), [x, y, w2], [d, zero])
    got = grads(0)
    assert torch.equal(got[0], both[0]) and torch.equal(got[1], both[1])


def test_mixed_parameter_types_and_what_is_not_finite():
    g = gen(15)
    x, y = (features(g, 1, 32, 40, torch.bfloat16) for _ in range(2))
    w, gate = vector(g, 32, dtype=torch.bfloat16), vector(g, 32, dtype=torch.float32)
    o = ff.norm_gate_residual(x, y, w, gate=gate)
    ref.check(rows(o), ref.norm(rows(x), rows(y), w.double(), None, gate.double(), dtype=torch.bfloat16)["out"], "mixed")
    # a NaN in one point stays there; under a mask that drops all of the block only x is left, whatever y is
    bad = y.clone()
    bad[0, 3, 7] = float('nan')
    got = ff.norm_gate_residual(x, bad, w, gate=gate)
    keep = [n for n in range(40) if n != 7]
    assert torch.equal(got[..., keep], o[..., keep]) and bool(got[..., 7].isnan().all())
    rng = torch.tensor([1, 0], device="cuda")
    assert torch.equal(ff.norm_gate_residual(x, bad, w, gate=gate, p=1.0, rng=rng), x)


# ------------------------------------------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 17, 255, 1025, 100003])
def test_dropout_follows_its_words(kind, n):
    dtype, g = TYPES[kind], gen(21)
    seed, offset = -(2 ** 62) - 12345, 2 ** 33 + 5
    rng = torch.tensor([seed, offset], device="cuda")
    x = vector(g, n, dtype=dtype).requires_grad_(True)
    d = vector(g, n, dtype=dtype)
    for p in (0.1, 0.5, 0.999):
        mask = ref.keep(seed % 2 ** 64, offset, p, (n,)).cuda()
        scale = torch.tensor(1.0 / (1.0 - p), dtype=torch.float32, device="cuda")
        y = ff.dropout(x, p, rng)
        (dx,) = torch.autograd.grad(y, [x], d)
        # one f32 product and one rounding: the same bits
        assert torch.equal(y, torch.where(mask, x.detach().float() * scale, 0.0).to(dtype))
        assert torch.equal(dx, torch.where(mask, d.float() * scale, 0.0).to(dtype))
    assert ff.dropout(x, 0.0, None) is x
    assert not ff.dropout(x, 1.0, rng).any()


def test_dropout_of_views_and_of_what_is_not_finite():
    g = gen(22)
    rng = torch.tensor([7, 0], device="cuda")
    x = torch.randn((6, 50), device="cuda", generator=g)
    want = ff.dropout(x, 0.4, rng)
    wide = torch.zeros((301,), device="cuda")
    wide[1:] = x.reshape(-1)
    assert torch.equal(ff.dropout(wide[1:].view(6, 50), 0.4, rng), want)               # starts off 16 bytes
    assert torch.equal(ff.dropout(x.t().contiguous().t(), 0.4, rng), want)             # counted by dimensions, not by memory
    assert torch.equal(ff.dropout(x.view(2, 3, 50), 0.4, rng), want.view(2, 3, 50))
    bad = torch.full_like(x, float('nan'))
    got = ff.dropout(bad, 0.4, rng)
    assert torch.equal(got == 0, want == 0) and bool(got[want != 0].isnan().all())
    # the counter's carry into its high half, and its wrap
    for offset in (2 ** 32 - 3, -5):
        rng = torch.tensor([7, offset], device="cuda")
        assert torch.equal(ff.dropout(x, 0.4, rng) != 0, ref.keep(7, offset % 2 ** 64, 0.4, (6, 50)).cuda())


def test_fused_dropout_is_the_same_draw():
    """norm_gate_residual's mask on (R, C) rows is dropout()'s, for rows of whole vectors and others."""
    g = gen(23)
    for C in (32, 33):
        y = torch.randn((70, C), device="cuda", generator=g) + 3.0
        rng = torch.tensor([5, 11], device="cuda")
        o = ff.norm_gate_residual(torch.zeros_like(y), y, kind='none', p=0.3, rng=rng)
        assert torch.equal(o != 0, ff.dropout(y, 0.3, rng) != 0)


def test_draws_do_not_overlap_and_streams_may_draw_at_once():
    rng = ff.CounterRng(99, "cuda")
    a, b = rng.take(10), rng.take(1)
    c = rng.take(0)
    assert a.tolist() == [99, 0] and b.tolist() == [99, 3] and c.tolist() == [99, 4] and rng.state.tolist() == [99, 4]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            got.append(rng.take(8))
    torch.cuda.synchronize()
    assert sorted(int(t[1]) for t in got) == list(range(4, 84, 2))


def test_a_draw_changed_before_the_backward_pass_is_noticed():
    x = torch.randn((40,), device="cuda", requires_grad=True)
    rng = torch.tensor([1, 0], device="cuda")
    y = ff.dropout(x, 0.5, rng)
    rng[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [x], torch.ones_like(y))


# ------------------------------------------------------------------------------------- offsets past 32 bits, streams, graphs
def test_rows_past_32_bits():
    """Tensors of more than 2^32 bytes and 2^31 elements: the last rows are right."""
    R, C, H = (1 << 20) + 70, 16, 2056
    g = gen(31)
    x = vector(g, R, C, dtype=torch.bfloat16)
    ws = [vector(g, H, C, dtype=torch.bfloat16, std=0.25), vector(g, H, C, dtype=torch.bfloat16, std=0.25)]
    h = ff.gated_feed_forward(x, *ws)  # R x H = 2^31 elements
    assert h.numel() > 2 ** 31
    ref.check(h[-100:].double(), ref.ffn(x[-100:].double(), *[w.double() for w in ws], None, "silu", dtype=torch.bfloat16)["y"], "h")
    o, nxt = ff.norm_gate_residual(h, h, next_kind='layer')
    want = ref.norm(h[-100:].double(), h[-100:].double(), next_kind='layer', dtype=torch.bfloat16)
    ref.check(o[-100:].double(), want["out"], "out")
    ref.check(nxt[-100:].double(), want["next"], "next")
    del o, nxt
    rng = torch.tensor([3, 0], device="cuda")
    d = ff.dropout(h, 0.5, rng)
    first = (R - 100) * H
    mask = ref.words(3, first // 4, 100 * H) >= 2 ** 31
    assert first % 4 == 0
    assert torch.equal(d[-100:], torch.where(torch.from_numpy(mask).cuda().view(100, H), h[-100:].float() * 2.0, 0.0).bfloat16())


def _block_step(block, x, dy):
    leaves = [x] + list(block.parameters())
    y = block(x)
    return [y] + list(torch.autograd.grad(y, leaves, dy))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_captured_step_repeats_the_eager_one(kind):
    """Forward and backward of a whole block in one graph, replayed between eager work: each replay the eager result.  With dropout
    every replay is the next draw."""
    dtype, g = TYPES[kind], gen(32)
    for p in (0.0, 0.3):
        block = ff.FeedForwardBlock(48, 96, post_norm='layer', pre_norm='layer', dropout=p, seed=5).cuda().to(dtype)
        x = features(g, 2, 48, 200, dtype, "channel").requires_grad_(True)
        dy = features(g, 2, 48, 200, dtype, "channel")
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(2):
                _block_step(block, x, dy)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            static = _block_step(block, x, dy)
        for turn in range(4):
            with torch.no_grad():
                x.copy_(features(g, 2, 48, 200, dtype, "channel"))
            if p:
                block._draws.rng.state[1] = 1000 * turn
            want = [t.detach().clone() for t in _block_step(block, x, dy)]
            torch.cuda.synchronize()
            if p:
                block._draws.rng.state[1] = 1000 * turn
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(static, want):
                assert torch.equal(a, b), (p, turn)
        if p:
            graph.replay()
            torch.cuda.synchronize()
            assert not torch.equal(static[0], want[0])


def test_two_graphs_and_a_side_stream_do_not_share_scratch():
    g = gen(33)
    block = ff.GatedFeedForward(64, 160).cuda().bfloat16()
    xs = [features(g, 1, 64, 900, torch.bfloat16).requires_grad_(True) for _ in range(2)]
    dy = features(g, 1, 64, 900, torch.bfloat16)
    want = [[t.detach().clone() for t in _block_step(block, x, dy)] for x in xs]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [[t.detach() for t in _block_step(block, x, dy)] for x in xs]
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(got[0] + got[1], want[0] + want[1]):
        assert torch.equal(a, b)
    graphs, static = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            static.append(_block_step(block, x, dy))
        graphs.append(graph)
    for _ in range(3):
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for a, b in zip(static[0] + static[1], want[0] + want[1]):
            assert torch.equal(a, b)


_ALIVE = r"""
import torch
from closerlook3d_amd import feed_forward as ff
w = torch.ones((64, 16), device="cuda", requires_grad=True)
d = torch.ones((16, 64), device="cuda", requires_grad=True)
n = torch.ones((16,), device="cuda", requires_grad=True)
x = torch.randn((40, 16), device="cuda", requires_grad=True)
rng = torch.tensor([1, 0], device="cuda")
calls = {"ffn": (lambda: ff.gated_feed_forward(x, w, w, d), [w, d]), "norm": (lambda: ff.point_norm(x, n), [n]),
         "dropout": (lambda: ff.dropout(x, 0.5, rng), [x])}
st = torch.cuda.Stream()
for name, (call, leaves) in calls.items():
    alive = call()
    torch.cuda.synchronize()
    for keep in (True, False):
        if not keep:
            del alive
        g = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.graph(g, stream=st):
                y = call()
                got = torch.autograd.grad(y, leaves, y.detach())
            print(name, keep, "captured", flush=True)
        except RuntimeError as e:
            print(name, keep, "eager graph of the same leaves" in str(e), flush=True)
        y = got = None
import os
os._exit(0)
"""


def test_a_captured_backward_names_a_living_eager_graph():
    """In a process of its own: what it refuses would end it."""
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", _ALIVE], capture_output=True, text=True, timeout=100,
                       cwd=__file__.rsplit("/", 2)[0])
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split("\n")[:6] == [f"{n} {k}" for n in ("ffn", "norm", "dropout") for k in ("True True", "False captured")], r.stdout


# ------------------------------------------------------------------------------------------------------ as they are used
def _composed(block, x, mask, order):
    """FeedForwardBlock from the 64-bit formulas, with autograd."""
    P = {k: v.detach().double().requires_grad_(True) for k, v in block.named_parameters()}
    r = rows(x).requires_grad_(True)

    def normed(v, kind, w, b):
        if kind == 'none':
            return v
        if kind == 'layer':
            v = v - v.mean(1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(1, keepdim=True) + block.eps)
        return v * w + (0 if b is None else b)

    h = normed(r, block.pre_norm, P["pre_weight"], P.get("pre_bias"))
    a = h @ P["feed_forward.w_gate"].t()
    y = (torch.nn.functional.silu(a) * (h @ P["feed_forward.w_up"].t())) @ P["feed_forward.w_down"].t()
    y = normed(y, block.post_norm, P.get("post_weight"), P.get("post_bias"))
    if mask is not None:
        y = y * mask / (1 - block.p)
    return r, P, block.residual_scale * r + P["gate"] * y


@pytest.mark.parametrize("order", ["point", "channel"])
@pytest.mark.parametrize("post", ["none", "rms", "layer"])
def test_feed_forward_block_is_its_formula(order, post):
    g = gen(41)
    B, C, N = 2, 60, 75
    block = ff.FeedForwardBlock(C, 130, pre_norm='layer', post_norm=post, gate_init=0.5, residual_scale=0.8, dropout=0.25, seed=77).cuda()
    x = features(g, B, C, N, torch.float32, order).requires_grad_(True)
    dy = features(g, B, C, N, torch.float32, order)
    got = _block_step(block, x, dy)
    assert ff._order(got[0])[1] == ff._order(x)[1]
    mask = ref.keep(77, 0, 0.25, (B * N, C)).cuda()
    r, P, y = _composed(block, x, mask, order)
    want = torch.autograd.grad(y, [r] + list(P.values()), rows(dy))
    # chained f32 operators: sums of at most max(H, B N) + 8 terms, a handful in a row, against the largest element
    for name, a, b in zip(["y", "x"] + list(P), got, [y.detach()] + list(want)):
        a = rows(a) if a.dim() == 3 else a.double()
        assert float((a - b).abs().max()) <= 8 * (B * N + 8) * ref.U32 * float(b.abs().max()), name
    block.eval()
    r, P, y = _composed(block, x, None, order)
    assert float((rows(block(x)) - y.detach()).abs().max()) <= 8 * (138) * ref.U32 * float(y.abs().max())
    # a run of them: entry and exit of neighbouring blocks in one pass give what two calls give
    h2 = ff.norm_gate_residual(x, block.feed_forward(x), gate=block.gate, kind='none', next_kind='rms')
    assert torch.equal(h2[0], ff.norm_gate_residual(x, block.feed_forward(x), gate=block.gate, kind='none'))
    again = ff.point_norm(h2[0])
    assert float((h2[1] - again).abs().max()) <= 8 * (C + 8) * ref.U32 * float(again.abs().max())


def test_classifier_with_counter_dropout_and_backbone_with_feed_forward():
    """The places that use them: config.cl3d_feed_forward appends a block to every bottleneck, config.cl3d_counter_dropout
    replaces the classifier's dropout; without them the modules and their state dicts are what they were."""
    from closerlook3d_amd.backbones import Bottleneck, ClassifierResNet
    from tests.helpers import default_config
    torch.manual_seed(0)
    cfg = default_config('pospool', {'pospool__reduction': 'avg'})
    plain = Bottleneck(24, 36, 2, 0.3, 8, cfg)
    cfg.cl3d_feed_forward = 2.0
    cfg.cl3d_feed_forward_dropout = 0.1
    torch.manual_seed(0)
    block = Bottleneck(24, 36, 2, 0.3, 8, cfg).cuda().train()
    extra = {k for k in block.state_dict() if k not in plain.state_dict()}
    assert extra and all(k.startswith("feed_forward.") for k in extra)
    assert block.feed_forward.feed_forward.w_gate.shape == (72, 36)
    block.load_state_dict(plain.state_dict(), strict=False)
    plain.cuda().train()
    g = gen(51)
    xyz = torch.rand((2, 128, 3), device="cuda", generator=g)
    mask = torch.ones((2, 128), dtype=torch.int32, device="cuda")
    f = torch.randn((2, 24, 128), device="cuda", generator=g)
    f1, f2 = f.clone().requires_grad_(True), f.clone().requires_grad_(True)
    _, _, want = plain(xyz, mask, f1)
    state = copy.deepcopy(block.feed_forward)
    _, _, got = block(xyz, mask, f2)
    inner = state(want)
    assert got.shape == want.shape and got.is_contiguous()
    assert (got - want).abs().max() > 0
    state._draws = ff._Draws(block.feed_forward._draws.seed)
    inner = state(want)
    assert torch.equal(inner, got)
    (d1,) = torch.autograd.grad(inner, [f1], torch.ones_like(inner))
    (d2,) = torch.autograd.grad(got, [f2], torch.ones_like(got))
    assert torch.equal(d1, d2)

    cfg = default_config('pospool')
    head, counted = ClassifierResNet(7, 8), None
    cfg.cl3d_counter_dropout = True
    counted = ClassifierResNet(7, 8, config=cfg)
    assert list(head.state_dict()) == list(counted.state_dict())
    counted.load_state_dict(head.state_dict())
    points = {"res5_mask": torch.ones((4, 10), device="cuda"), "res5_features": torch.randn((4, 128, 10), device="cuda", generator=g)}
    head.cuda().eval(), counted.cuda().eval()
    assert torch.equal(head(points), counted(points))
    counted.train()
    a, b = counted(points), counted(points)
    assert not torch.equal(a, b)
    a.sum().backward()
    assert all(p.grad is not None for p in counted.parameters())

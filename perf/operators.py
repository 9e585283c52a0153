"""What the feed-forward operators of closerlook3d_amd.feed_forward are measured on: a gated feed-forward over point
features, the norms either side of a block with its gate, dropout and residual, and dropout from a counter.

Every case is one pass as a program makes it: a forward call, or a forward call and the gradients of its inputs.  With `own`
false the operators are computed from elementary torch operations in 32 bits, rounded once at the end; with `own` true by the
package.  Sizes follow the residual backbone of this repository: widths 144 .. 2304 (res1 .. res5), clouds of 4096 points and
scenes of 10 000 .. 81 920, pooled vectors in front of a classifier.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one pooled shape vector through a narrow feed-forward: the latency of a single call
        dict(name="ffn_one_vector", op="ffn", B=1, N=1, C=288, H=768, type="f16", act="silu", train=False, order="point"),
        # a batch of 16 pooled res5 vectors at the classifier's entry: the weights are read once, little else
        dict(name="ffn_pooled_batch", op="ffn", B=16, N=1, C=2304, H=4608, type="bf16", act="silu", train=False, order="point"),
        # inference on 16 clouds of 4096 points at the width of the first stage
        dict(name="ffn_clouds", op="ffn", B=16, N=4096, C=144, H=576, type="bf16", act="silu", train=False, order="point"),
        # a training step of the third stage: 16 clouds x 1024 points
        dict(name="ffn_train_stage", op="ffn", B=16, N=1024, C=288, H=1152, type="bf16", act="silu", train=True, order="point"),
        # the framework's own type and memory order: f32, channel-major features, four clouds
        dict(name="ffn_train_f32", op="ffn", B=4, N=4096, C=144, H=576, type="f32", act="gelu", train=True, order="channel"),
        # a ragged scene and widths that no tile divides
        dict(name="ffn_train_odd", op="ffn", B=1, N=9973, C=201, H=533, type="f16", act="gelu", train=True, order="point"),
        # entry norm of a deep stage: few points, wide rows
        dict(name="norm_entry_deep", op="norm", B=16, N=16, C=2304, type="f32", kind="layer", train=False, order="point",
             exit=False, next=False, gate="none", p=0.0),
        # exit of one block and entry of the next, inference, 16 clouds
        dict(name="norm_join_clouds", op="norm", B=16, N=4096, C=144, type="bf16", kind="rms", train=False, order="point",
             exit=True, next=True, gate="channel", p=0.0),
        # the same as a training step on a whole scene, with dropout: the largest pass
        dict(name="norm_join_train", op="norm", B=1, N=81920, C=288, type="bf16", kind="rms", train=True, order="point",
             exit=True, next=True, gate="channel", p=0.1),
        # block exit in the framework's own order and type, a gate for each cloud
        dict(name="norm_exit_train_f32", op="norm", B=4, N=10000, C=72, type="f32", kind="layer", train=True, order="channel",
             exit=True, next=False, gate="cloud", p=0.2),
        # the classifier's hidden vectors, with the gradient
        dict(name="dropout_classifier", op="dropout", B=16, N=1, C=1152, type="f32", train=True, p=0.5),
        # features of 16 clouds, with the gradient
        dict(name="dropout_clouds", op="dropout", B=16, N=4096, C=144, type="bf16", train=True, p=0.1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "norm", "norm", "dropout"])
    kind = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.5
    order = rng.choice(["point", "point", "channel"])
    if op == "ffn":
        C, H = _log_int(rng, 16, 2304), _log_int(rng, 32, 4608)
        if rng.random() < 0.5:
            C, H = -(-C // 8) * 8, -(-H // 8) * 8
        most = 16384 * 1152 * 288 // (C * H)
        rows = _log_int(rng, 1, max(1, min(65536, most if kind != "f32" else most // 4)))
        B = rng.choice([1, 1, 2, 4, 16])
        return dict(op=op, B=B, N=max(1, rows // B), C=C, H=H, type=kind, act=rng.choice(["silu", "gelu"]), train=train, order=order)
    rows = _log_int(rng, 1, 81920)
    C = _log_int(rng, 8, max(8, min(2304, 81920 * 288 // rows)))
    B = rng.choice([1, 1, 2, 4, 16])
    N = max(1, rows // B)
    C = min(C, 81920 * 288 // (B * N))
    p = rng.choice([0.0, 0.1, 0.5])
    if op == "dropout":
        return dict(op=op, B=B, N=N, C=C, type=kind, train=train, p=p or 0.3)
    leaves = rng.random() < 0.7
    follows = leaves and rng.random() < 0.6
    return dict(op=op, B=B, N=N, C=C, type=kind, kind=rng.choice(["rms", "layer"]), train=train, order=order, exit=leaves, next=follows,
                gate=rng.choice(["none", "channel", "cloud"]) if leaves else "none", p=p if leaves else 0.0)


# ------------------------------------------------------------------------------------------------------------- inputs
def _features(g, case, scale=1.0):
    """(B, C, N) features in the case's memory order; point-major memory is a transposed view of dense (B, N, C) rows."""
    B, N, C, t = case["B"], case["N"], case["C"], _TYPES[case["type"]]
    rows = torch.randn((B, N, C), device="cuda", generator=g) * scale
    if case.get("order", "channel") == "point":
        return rows.to(t).transpose(1, 2)
    return rows.transpose(1, 2).contiguous().to(t)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, C = _TYPES[case["type"]], case["C"]
    s = {"case": case, "x": _features(g, case)}
    leaves = ["x"]

    def vector(mean, std, *shape):
        return (torch.randn(shape, device="cuda", generator=g) * std + mean).to(t)

    if case["op"] == "ffn":
        H = case["H"]
        s["w_gate"], s["w_up"] = vector(0.0, C ** -0.5, H, C), vector(0.0, C ** -0.5, H, C)
        s["w_down"] = vector(0.0, H ** -0.5, C, H)
        s["dout"] = _features(g, case)
        leaves += ["w_gate", "w_up", "w_down"]
    elif case["op"] == "norm":
        if case["exit"]:
            s["y"] = _features(g, case, 2.0)
            s["weight"], s["bias"] = vector(1.0, 0.2, C), vector(0.0, 0.2, C) if case["kind"] == "layer" else None
            s["gate"] = {"none": None, "channel": vector(0.3, 0.1, C), "cloud": vector(0.3, 0.1, case["B"], C)}[case["gate"]]
            s["dout"] = _features(g, case)
            leaves += ["y", "weight", "bias", "gate"]
        if case["next"] or not case["exit"]:
            s["next_weight"], s["next_bias"] = vector(1.0, 0.2, C), vector(0.0, 0.2, C) if case["kind"] == "layer" else None
            s["dnext"] = _features(g, case)
            leaves += ["next_weight", "next_bias"]
    else:
        s["dout"] = _features(g, case)
    if case.get("p"):
        s["rng"] = torch.tensor([seed * 7919 + 12345, (seed % 97) << 20], dtype=torch.int64, device="cuda")  # (seed, offset)
    s["leaves"] = [k for k in leaves if s.get(k) is not None]
    if case["train"]:
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _random_words(rng, count):
    """`count` 32-bit words of the counter-based generator (Philox 4x32, ten rounds; Salmon et al., 2011) as int64: word i is
    number i % 4 of the block with counter offset + i / 4 under the key `seed`.  A product of two 32-bit numbers is formed
    from 16-bit halves, so that it stays inside a signed 64-bit number."""
    low = 0xFFFFFFFF
    at = rng[1] + torch.arange((count + 3) // 4, device=rng.device)
    c = [at & low, (at >> 32) & low, torch.zeros_like(at), torch.zeros_like(at)]
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low

    def product(a, m):
        p0, p1 = (a & 0xFFFF) * m, (a >> 16) * m
        t = p0 + ((p1 & 0xFFFF) << 16)
        return (p1 >> 16) + (t >> 32), t & low

    for _ in range(10):  # the generator's rounds
        h0, l0 = product(c[0], 0xD2511F53)
        h1, l1 = product(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack(c, 1).reshape(-1)[:count]


def _kept(rng, p, shape):
    """1 / (1 - p) where the element stays and 0 where it is dropped, in 32 bits."""
    stays = _random_words(rng, math.prod(shape)) >= int(p * 4294967296.0)
    return (stays.float() * (1.0 / (1.0 - p))).reshape(shape)


def _plain_norm(v, kind, weight, bias):
    """Over the channels of (B, N, C) rows."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * weight
    return v if bias is None else v + bias


def _plain(s):
    """The case's outputs and, of a training pass, the gradients of its leaves: everything in 32 bits."""
    case, t = s["case"], _TYPES[s["case"]["type"]]
    v = {k: s[k].detach().float() for k in s["leaves"]}
    if case["train"]:
        v = {k: a.requires_grad_(True) for k, a in v.items()}
    rows = v["x"].transpose(1, 2)
    outs, given = [], []
    if case["op"] == "ffn":
        a = rows @ v["w_gate"].t()
        a = a * torch.sigmoid(a) if case["act"] == "silu" else 0.5 * a * (1.0 + torch.erf(a * 0.5 ** 0.5))
        outs.append(((a * (rows @ v["w_up"].t())) @ v["w_down"].t()).transpose(1, 2))
        given.append(s["dout"])
    elif case["op"] == "norm":
        if case["exit"]:
            b = _plain_norm(v["y"].transpose(1, 2), case["kind"], v["weight"], v.get("bias"))
            if case["p"]:
                b = b * _kept(s["rng"], case["p"], b.shape)
            if "gate" in v:
                b = b * (v["gate"] if v["gate"].dim() == 1 else v["gate"][:, None, :])
            rows = 0.9 * rows + b
            outs.append(rows.transpose(1, 2))
            given.append(s["dout"])
        if "next_weight" in v:
            outs.append(_plain_norm(rows, case["kind"], v["next_weight"], v.get("next_bias")).transpose(1, 2))
            given.append(s["dnext"])
    else:
        outs.append(v["x"] * _kept(s["rng"], case["p"], v["x"].shape))
        given.append(s["dout"])
    grads = []
    if case["train"]:
        grads = torch.autograd.grad(outs, [v[k] for k in s["leaves"]], [d.float() for d in given])
    return [o.detach().to(t) for o in outs], [g.to(t) for g in grads]


# --------------------------------------------------------------------------------------------------- the package's calls
def _own(s):
    from closerlook3d_amd import feed_forward as ff
    case, x = s["case"], s["x"]
    if case["op"] == "ffn":
        outs = [ff.gated_feed_forward(x, s["w_gate"], s["w_up"], s["w_down"], activation=case["act"])]
        given = [s["dout"]]
    elif case["op"] == "norm" and not case["exit"]:
        outs = [ff.point_norm(x, s["next_weight"], s["next_bias"], kind=case["kind"], eps=1e-6)]
        given = [s["dnext"]]
    elif case["op"] == "norm":
        follows = dict(next_kind=case["kind"], next_weight=s["next_weight"], next_bias=s["next_bias"]) if case["next"] else {}
        outs = ff.norm_gate_residual(x, s["y"], s["weight"], s["bias"], gate=s["gate"], residual_scale=0.9, kind=case["kind"],
                                     eps=1e-6, p=case["p"], rng=s.get("rng"), **follows)
        outs, given = (list(outs), [s["dout"], s["dnext"]]) if case["next"] else ([outs], [s["dout"]])
    else:
        outs, given = [ff.dropout(x, case["p"], s["rng"])], [s["dout"]]
    grads = torch.autograd.grad(outs, [s[k] for k in s["leaves"]], given) if case["train"] else []
    return [o.detach() for o in outs], list(grads)


def run(state):
    outs, grads = _own(state) if own else _plain(state)
    return {"outputs": outs, "gradients": grads}


# ------------------------------------------------------------------------------------------------------------- in 64 bits
def _words_64(seed, offset, count):
    """The generator's words by numpy's unsigned 64-bit products."""
    at = (np.arange((count + 3) // 4, dtype=np.uint64) + np.uint64(offset))
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    a, b = at & low, at >> shift
    c, d = np.zeros_like(a), np.zeros_like(a)
    for r in range(10):
        k = (seed + r * 0x9E3779B9) & 0xFFFFFFFF, ((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF
        u, w = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (w >> shift) ^ b ^ np.uint64(k[0]), w & low, (u >> shift) ^ d ^ np.uint64(k[1]), u & low
    return np.stack([a, b, c, d], 1).reshape(-1)[:count]


def _mask_64(s, p, shape):
    seed, offset = (int(a) for a in s["rng"])
    stays = torch.from_numpy(_words_64(seed, offset, math.prod(shape)) >= np.uint64(int(p * 2 ** 32))).cuda()
    return stays.double().reshape(shape) / (1.0 - p)


def _norm_64(v, kind):
    """The normalised rows and the reciprocal deviations that they were multiplied with."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    inv = 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6)
    return v * inv, inv


def _norm_grad_64(dhat, hat, inv, kind):
    d = dhat - hat * (dhat * hat).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - dhat.mean(-1, keepdim=True)
    return d * inv


def exact(case, seed):
    s = prepare(case, seed)
    C = case["C"]
    v = {k: (a.detach().double() if torch.is_tensor(a) and a.is_floating_point() else a) for k, a in s.items()}
    as_rows = lambda a: a.transpose(1, 2).reshape(-1, C)  # noqa: E731
    back = lambda a: a.reshape(case["B"], case["N"], C).transpose(1, 2)  # noqa: E731
    if case["op"] == "dropout":
        m = _mask_64(s, case["p"], v["x"].shape)
        return {"outputs": [v["x"] * m], "gradients": [v["dout"] * m] if case["train"] else []}
    x = as_rows(v["x"])
    if case["op"] == "ffn":
        g, u = x @ v["w_gate"].t(), x @ v["w_up"].t()
        if case["act"] == "silu":
            sig = 1.0 / (1.0 + torch.exp(-g))
            a, slope = g * sig, sig * (1.0 + g * (1.0 - sig))
        else:
            cdf = 0.5 * (1.0 + torch.erf(g / math.sqrt(2.0)))
            a, slope = g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
        outs = [back((a * u) @ v["w_down"].t())]
        if not case["train"]:
            return {"outputs": outs, "gradients": []}
        dy = as_rows(v["dout"])
        dh = dy @ v["w_down"]
        dg, du = dh * u * slope, dh * a
        return {"outputs": outs, "gradients": [back(dg @ v["w_gate"] + du @ v["w_up"]), dg.t() @ x, du.t() @ x, dy.t() @ (a * u)]}
    outs, kind = [], case["kind"]
    if case["exit"]:
        yhat, yinv = _norm_64(as_rows(v["y"]), kind)
        n = yhat * v["weight"] + (0.0 if v["bias"] is None else v["bias"])
        m = _mask_64(s, case["p"], n.shape) if case["p"] else 1.0
        gate = 1.0 if v["gate"] is None else v["gate"] if v["gate"].dim() == 1 else v["gate"].repeat_interleave(case["N"], 0)
        x = 0.9 * x + gate * (n * m)
        outs.append(back(x))
    if "next_weight" in v:
        hat, inv = _norm_64(x, kind)
        outs.append(back(hat * v["next_weight"] + (0.0 if v["next_bias"] is None else v["next_bias"])))
    if not case["train"]:
        return {"outputs": outs, "gradients": []}
    d = as_rows(v["dout"]) if case["exit"] else torch.zeros_like(x)
    tail = []
    if "next_weight" in v:
        dn = as_rows(v["dnext"])
        d = d + _norm_grad_64(dn * v["next_weight"], hat, inv, kind)
        tail = [(dn * hat).sum(0)] + ([] if v["next_bias"] is None else [dn.sum(0)])
    if not case["exit"]:
        return {"outputs": outs, "gradients": [back(d)] + tail}
    dm = d * gate * m
    grads = [back(0.9 * d), back(_norm_grad_64(dm * v["weight"], yhat, yinv, kind)), (dm * yhat).sum(0)]
    if v["bias"] is not None:
        grads.append(dm.sum(0))
    if v["gate"] is not None:
        dgate = d * n * m
        grads.append(dgate.sum(0) if v["gate"].dim() == 1 else dgate.reshape(case["B"], case["N"], C).sum(1))
    return {"outputs": outs, "gradients": grads + tail}


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["type"]]
    rows, C = case["B"] * case["N"], case["C"]
    points = rows * C
    if case["op"] == "ffn":
        weights = 3 * C * case["H"]
        if not case["train"]:
            return {"bytes": size * (2 * points + weights), "flops": 2 * rows * weights}
        # x and dy in, y and dx out, the weights in and their gradients out; the three products once forward, twice backward
        return {"bytes": size * (4 * points + 2 * weights), "flops": 6 * rows * weights}
    if case["op"] == "dropout":
        return {"bytes": size * points * (4 if case["train"] else 2), "flops": (2 if case["train"] else 1) * points}
    forward = 1 + (1 if case["exit"] else 0) + (1 if case["exit"] and case["next"] else 0) + 1  # x, y in; out and / or next out
    moved = forward
    if case["train"]:  # the gradients of the outputs in, those of x and y out
        moved += (1 if case["exit"] else 0) + (1 if case["next"] or not case["exit"] else 0) + (2 if case["exit"] else 1)
    return {"bytes": size * points * moved, "flops": points * (8 + 8 * case["exit"]) * (3 if case["train"] else 1)}

"""CPU: what the feed-forward operators refuse before any launch, beyond what test_feed_forward.py asks."""
import ctypes

import pytest
import torch

from closerlook3d_amd import _lib
from closerlook3d_amd import feed_forward as ff
from tests.test_feed_forward import fake


def _block(**kw):
    base = dict(B=2, N=3, C=8, dtype=0, kind=1, next_kind=1, residual_scale=1.0, eps=1e-6, next_eps=1e-6)
    return _lib.NormResidual(**{**base, **kw})


@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("name", ["weight", "bias", "gate", "next_weight", "next_bias"])
def test_a_gradient_of_a_parameter_that_is_not_given_is_refused(name, order):
    """It would be a sum of scratch that no kernel has written."""
    lib = _lib.lib()
    a = 1 << 20  # a 16-byte aligned number (no pointer is followed before the checks have passed)
    given = dict(order=order, x=a, y=a, weight=a, bias=a, gate=a, next_weight=a, next_bias=a, stats=a, dout=a, dnext=a, dx=a, dy=a)
    given[name] = None
    rc = lib.cl3d_norm_residual_bwd(ctypes.byref(_block(**given, **{"d" + name: a})), None)
    assert rc == -1 and "a parameter that is not there" in lib.cl3d_last_error_string().decode()


@pytest.mark.parametrize("name", ["weight", "gate", "next_weight"])
def test_a_gradient_of_a_step_that_is_not_taken_is_refused(name):
    """A parameter of an exit, or of an entry, that the call does not have."""
    lib = _lib.lib()
    a = 1 << 20
    given = dict(x=a, stats=a, dnext=a, dx=a, next_weight=a) if name != "next_weight" else dict(x=a, y=a, next_kind=0, stats=a, dout=a, next_weight=a)
    rc = lib.cl3d_norm_residual_bwd(ctypes.byref(_block(**given, **{"d" + name: a})), None)
    assert rc == -1 and "a parameter that is not there" in lib.cl3d_last_error_string().decode()


def test_a_learned_residual_scale_is_refused():
    """The scale is read on the host: a tensor that wants a gradient would get none."""
    scale = torch.nn.Parameter(torch.ones(()))
    for x in (fake(4, 8), fake(2, 8, 3)):
        with pytest.raises(TypeError, match="residual_scale is a number"):
            ff.norm_gate_residual(x, x, residual_scale=scale)


def test_the_point_major_dropout_returns_codes_and_says_why():
    lib = _lib.lib()
    a = 1 << 20
    for args, text in (((a, 4, 2, 8, 3, 0.5, a, a, None), "element type"), ((a, 0, 2, 8, -1, 0.5, a, a, None), "bad size"),
                       ((a, 0, -2, 8, 3, 0.5, a, a, None), "bad size"), ((a, 0, 2, 8, 3, 1.5, a, a, None), "probability"),
                       ((a, 0, 2, 8, 3, 0.5, None, a, None), "generator state"), ((a, 0, 2, 8, 3, 0.0, None, a, None), "null pointer"),
                       ((None, 0, 2, 8, 3, 0.5, a, a, None), "null pointer"), ((a, 0, 2, 8, 3, 0.5, a, None, None), "null pointer")):
        assert lib.cl3d_dropout_point_major(*args) == -1 and text in lib.cl3d_last_error_string().decode(), (args, lib.cl3d_last_error_string())
    for sizes in ((0, 8, 3), (2, 0, 3), (2, 8, 0)):
        assert lib.cl3d_dropout_point_major(None, 0, *sizes, 0.5, a, None, None) == 0


@pytest.mark.parametrize("shape", [(2 ** 31, 1), (2 ** 32 + 5, 1), (2 ** 32 + 5, 1, 1), (1, 1, 2 ** 32 + 5), (1, 2 ** 32 + 1, 2)], ids=str)
def test_sizes_past_31_bits_are_refused(shape):
    """The C entries take 32-bit sizes; a longer axis would arrive with its high half cut off."""
    x = fake(1).expand(shape)
    C = shape[1]
    calls = [lambda: ff.point_norm(x), lambda: ff.norm_gate_residual(x, x)]
    if C == 1:
        calls.append(lambda: ff.gated_feed_forward(x, fake(8, 1), fake(8, 1), fake(1, 8)))
        many = fake(1).expand(2 ** 32 + 3, 1)
        calls.append(lambda: ff.gated_feed_forward(fake(4, 1), many, many))
    if len(shape) == 3:
        calls += [lambda: ff.to_point_major(x), lambda: ff.to_channel_major(x)]
    for call in calls:
        with pytest.raises(ValueError, match="2147483647"):
            call()


def test_dropout_of_point_major_features_past_31_bits_is_refused():
    x = fake(1).expand(2, 2 ** 32 + 4, 2)
    rng = torch.zeros(2, dtype=torch.int64)
    with pytest.MonkeyPatch.context() as patch:
        patch.setattr(ff, "_point_major", lambda t: True)  # (no memory for features that are)
        with pytest.raises(ValueError, match="2147483647"):
            ff.dropout(x, 0.5, rng)


@pytest.mark.parametrize("channels", [0, 4098, 4100, 4612, 6150, 6152])
def test_a_block_of_too_many_channels_is_refused_where_it_is_made(channels):
    with pytest.raises(ValueError, match="channels, or a multiple of 8"):
        ff.FeedForwardBlock(channels, 16)
    if channels:
        with pytest.raises(ValueError, match="channels, or a multiple of 8"):
            ff.point_norm(fake(2, channels))


def test_wide_norms_start_on_16_bytes():
    lib = _lib.lib()
    a = 1 << 20
    names = ("x", "y", "weight", "bias", "gate", "next_weight", "next_bias", "out", "next")
    for name in names:
        given = {n: a for n in names}
        given[name] = a + 4
        rc = lib.cl3d_norm_residual_fwd(ctypes.byref(_block(C=4608, **given)), None)
        assert rc == -4 and "16 bytes" in lib.cl3d_last_error_string().decode(), name
    for C in (4100, 6152):
        rc = lib.cl3d_norm_residual_fwd(ctypes.byref(_block(C=C, **{n: a for n in names})), None)
        assert rc == -4 and "channels" in lib.cl3d_last_error_string().decode()


def test_capture_checks_beside_threads_that_make_graphs(monkeypatch):
    """A captured backward pass looks through the living eager graphs while other threads make and drop theirs."""
    import sys
    import threading
    monkeypatch.setattr(ff, "_raw_stream", lambda index: 1)
    leaf = torch.nn.Parameter(torch.zeros(3))

    class Context:
        pass

    capturing = threading.local()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: getattr(capturing, "yes", False))
    stop, failed = threading.Event(), []
    alive = [Context() for _ in range(400)]
    for ctx in alive:
        ff._track(ctx, leaf)

    def make():
        kept = []
        try:
            while not stop.is_set():
                kept.append(Context())
                ff._track(kept[-1], leaf)
                if len(kept) > 50:
                    kept.clear()
        except Exception as e:  # noqa: BLE001 (what a thread raises is looked at below)
            failed.append(e)

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    threads = [threading.Thread(target=make) for _ in range(3)]
    try:
        for t in threads:
            t.start()
        mine = Context()
        mine.leaves, mine.made_on = [], 1
        capturing.yes = True
        for _ in range(300):
            ff._check_capture(mine, torch.device("cuda", 0))
    finally:
        stop.set()
        for t in threads:
            t.join()
        sys.setswitchinterval(interval)
    assert not failed
    del alive, ctx


def test_a_gate_of_each_cloud_has_a_limit():
    for shape in ((70000, 8), (70000, 8, 3)):
        x = fake(1).expand(shape)
        with pytest.raises(ValueError, match="up to 65535 clouds"):
            ff.norm_gate_residual(x, x, gate=fake(1).expand(70000, 8))


def test_capture_checks_beside_threads_that_drop_graphs(monkeypatch):
    """The same while other threads free graphs one by one: a context that goes in another thread changes nothing under the walk."""
    import sys
    import threading
    monkeypatch.setattr(ff, "_raw_stream", lambda index: 1)
    leaf = torch.nn.Parameter(torch.zeros(3))

    class Context:
        pass

    capturing = threading.local()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: getattr(capturing, "yes", False))
    stop, failed = threading.Event(), []
    alive = [Context() for _ in range(50)]
    for ctx in alive:
        ff._track(ctx, leaf)

    def drop():
        try:
            while not stop.is_set():
                ff._track(Context(), leaf)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    threads = [threading.Thread(target=drop) for _ in range(3)]
    try:
        for t in threads:
            t.start()
        mine = Context()
        mine.leaves, mine.made_on = [], 1
        capturing.yes = True
        for _ in range(4000):
            ff._check_capture(mine, torch.device("cuda", 0))
        assert not failed
    finally:
        stop.set()
        for t in threads:
            t.join()
        sys.setswitchinterval(interval)
    del alive, ctx

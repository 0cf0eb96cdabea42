"""The dense operators' refusals: the C calls check their arguments before they touch a device, the Python
calls refuse what is not on one."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from quickrank_amd import build, _capi
    build.build()
    return _capi.lib()


# (an address that is never followed: every call below is refused first)
P, Q, R = 1 << 30, 1 << 31, 1 << 32
ARG = 3


def message(L):
    return L.qr_last_error(None).decode()


def norm(L, type=0, ptype=0, rows=4, cols=8, x=P, ldx=8, w=None, b=None, eps=1e-5, y=Q, ldy=8):
    return L.qr_layer_norm_async(0, None, type, ptype, rows, cols, x, ldx, w, b, eps, y, ldy, None, None)


@pytest.mark.parametrize("bad", [dict(type=3), dict(type=-1), dict(type=0, ptype=1), dict(type=1, ptype=2), dict(cols=0),
                                 dict(rows=1 << 60), dict(ldx=1 << 60), dict(eps=-1.0),
                                 dict(eps=float("nan")), dict(eps=float("inf")), dict(ldy=7), dict(x=None), dict(y=None)])
def test_norm_refusals(L, bad):
    assert norm(L, **bad) == ARG and message(L).startswith("layer norm")


def test_norm_of_rows_beyond_2_24_columns_is_unsupported(L):
    c = (1 << 24) + 1
    assert norm(L, cols=c, ldx=c, ldy=c, y=R) == 5
    assert norm_back(L, cols=c, lddy=c, ldx=c, lddx=c, n=1 << 50) == 5


def norm_back(L, type=0, ptype=0, rows=4, cols=8, dy=P, lddy=8, x=Q, ldx=8, mean=P, rstd=P, dx=R, lddx=8, dw=P, ws=P, n=1 << 30):
    return L.qr_layer_norm_backward_async(0, None, type, ptype, rows, cols, dy, lddy, x, ldx, None, mean, rstd, dx, lddx, dw, None,
                                          ws, n)


@pytest.mark.parametrize("bad", [dict(type=9), dict(type=2, ptype=1), dict(cols=0), dict(rows=1 << 60), dict(lddx=7), dict(dy=None),
                                 dict(x=None), dict(mean=None), dict(rstd=None), dict(ws=None), dict(n=8)])
def test_norm_backward_refusals(L, bad):
    assert norm_back(L, **bad) == ARG and message(L).startswith("layer norm backward")


def drop(L, type=0, rows=4, cols=8, x=P, ldx=8, r=None, ldr=0, y=Q, ldy=8, p=0.1):
    return L.qr_dropout_async(0, None, type, rows, cols, x, ldx, r, ldr, y, ldy, p, 1, 0, None)


@pytest.mark.parametrize("bad", [dict(type=7), dict(p=-1e-9), dict(p=1.0000001), dict(p=float("nan")), dict(rows=1 << 60),
                                 dict(cols=1 << 60), dict(ldy=7), dict(x=None), dict(y=None), dict(r=P, ldr=1 << 60)])
def test_dropout_refusals(L, bad):
    assert drop(L, **bad) == ARG and message(L).startswith("dropout")


def ffn(L, type=0, act=0, m=4, k=8, n=16, x=P, ldx=8, wg=Q, wu=R, ldw=8, h=R + Q, ldh=16, g=None, u=None, ws=None,
        nbytes=0):
    return L.qr_gated_ffn_async(0, None, type, act, m, k, n, x, ldx, wg, wu, ldw, h, ldh, g, u, ws, nbytes)


@pytest.mark.parametrize("bad", [dict(type=5), dict(act=5), dict(act=-1), dict(k=0), dict(n=0), dict(m=1 << 60), dict(ldh=15),
                                 dict(g=P + Q), dict(u=P + Q), dict(x=None), dict(wg=None), dict(wu=None), dict(h=None), dict(h=P + 64),
                                 dict(h=Q), dict(h=R + 128), dict(g=R + Q + 32, u=R + R), dict(g=R + R, u=R + R + 255),
                                 dict(g=P, u=R + R)])
def test_ffn_refusals(L, bad):
    assert ffn(L, **bad) == ARG and message(L).startswith("gated ffn")


@pytest.mark.parametrize("bad", [dict(x=P + 4), dict(ldx=9), dict(ldw=10), dict(wu=R + 8), dict(x=P + 4, ws=2 * R),
                                 dict(x=P + 4, ws=2 * R, nbytes=256), dict(x=P + 4, ws=R, nbytes=1 << 20)])
def test_ffn_many_rows_off_boundaries_need_the_workspace(L, bad):
    assert ffn(L, m=200, n=4096, ldh=4096, **bad) == ARG and message(L).startswith("gated ffn")


def test_ffn_rows_beyond_4_mb_are_unsupported(L):
    k = (1 << 20) + 1
    assert ffn(L, m=200, n=4096, ldh=4096, k=k, ldx=k, ldw=k, wu=64 * R, h=128 * R, ws=256 * R, nbytes=1 << 50) == 5
    assert ffn_back(L, m=200, k=k, x=2 * Q, wg=8 * R, wu=16 * R, g=32 * R, u=64 * R, dx=128 * R, lddx=k, dwg=256 * R, dwu=512 * R,
                    ws=1024 * R, nbytes=1 << 50) == 5
    assert ffn_back(L, m=200, n=k, dh=16 * R, lddh=k, x=2 * Q, wg=8 * R, wu=20 * R, g=32 * R, u=64 * R, dx=128 * R, dwg=256 * R,
                    dwu=512 * R, ws=1024 * R, nbytes=1 << 50) == 5


def ffn_back(L, type=0, act=0, m=4, k=8, n=16, dh=P, lddh=16, x=Q, wg=R, wu=R + P, g=R + Q, u=2 * R, dx=2 * R + P, lddx=8,
             dwg=2 * R + Q, dwu=3 * R, ws=3 * R + Q, nbytes=1 << 30):
    return L.qr_gated_ffn_backward_async(0, None, type, act, m, k, n, dh, lddh, x, 8, wg, wu, 8, g, u, dx, lddx, dwg, dwu, ws, nbytes)


@pytest.mark.parametrize("bad", [dict(type=5), dict(act=5), dict(k=0), dict(n=0), dict(m=1 << 60), dict(lddx=7), dict(dh=None),
                                 dict(x=None), dict(wg=None), dict(wu=None), dict(g=None), dict(u=None), dict(dwg=None),
                                 dict(dwu=None), dict(ws=None), dict(nbytes=64), dict(dx=Q), dict(dwg=R), dict(ws=2 * R),
                                 dict(ws=3 * R - 64), dict(dwu=2 * R + Q + 64)])
def test_ffn_backward_refusals(L, bad):
    assert ffn_back(L, **bad) == ARG and message(L).startswith("gated ffn backward")


def test_workspace_queries(L):
    n = C.c_size_t(99)
    assert L.qr_layer_norm_backward_workspace(0, 8, C.byref(n)) == 0 and n.value == 0
    assert L.qr_layer_norm_backward_workspace(1000, 136, C.byref(n)) == 0 and n.value >= 2 * 136 * 4
    assert L.qr_layer_norm_backward_workspace(4, 0, C.byref(n)) == ARG
    assert L.qr_gated_ffn_workspace(0, 100, 9, 16, C.byref(n)) == 0 and n.value >= (100 + 32) * 12 * 4
    assert L.qr_gated_ffn_workspace(0, 100, 0, 16, C.byref(n)) == ARG
    assert L.qr_gated_ffn_backward_workspace(1, 100, 8, 16, C.byref(n)) == 0 and n.value >= 2 * 100 * 16 * 2
    assert L.qr_gated_ffn_backward_workspace(1, 0, 8, 16, C.byref(n)) == 0
    assert L.qr_gated_ffn_backward_workspace(4, 1, 8, 16, C.byref(n)) == ARG
    assert L.qr_gated_ffn_backward_workspace(1, 1, 8, 16, None) == ARG
    assert L.qr_layer_norm_backward_workspace(4, 8, None) == ARG


def test_no_rows_is_no_work(L):
    """Nothing is followed or launched: these hold where there is no device, too."""
    assert norm(L, rows=0, x=None, y=None) == 0
    assert drop(L, rows=0, x=None, y=None) == 0 and drop(L, cols=0) == 0
    assert ffn(L, m=0, x=None, h=None) == 0


def test_without_a_device(L):
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    assert norm(L) in (1, ARG) and "device" in message(L)


def test_python_refuses_host_tensors():
    from quickrank_amd import QrError, dense
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    for call in (lambda: dense.layer_norm(x), lambda: dense.dropout(x, 0.1, 1), lambda: dense.gated_ffn(x, w, w),
                 lambda: dense.layer_norm_backward(x, x, None, x[:, 0], x[:, 0]),
                 lambda: dense.gated_ffn_backward(x, x, w, w, x, x), lambda: dense.layer_norm([1.0]), lambda: dense.dropout(x.int(), 0.1, 1)):
        with pytest.raises(QrError) as e:
            call()
        assert e.value.code == ARG


def test_ffn_of_more_rows_or_outputs_than_a_launch_has_threads_for_is_unsupported(L):
    big = 1 << 52
    assert ffn(L, m=(1 << 30) + 1, h=big) == 5 and "2^30 rows" in message(L)
    n = (1 << 28) + 1
    assert ffn(L, m=100, n=n, ldh=n, wg=1 << 50, wu=1 << 51, h=big) == 5 and "2^28 outputs" in message(L)
    assert ffn_back(L, m=(1 << 30) + 1, ws=big, nbytes=1 << 50) == 5 and "2^30 rows" in message(L)


def test_norm_workspace_of_long_rows_stays_small(L):
    n = C.c_size_t()
    for cols in (16385, 100_000, 1 << 24):
        assert L.qr_layer_norm_backward_workspace(1 << 20, cols, C.byref(n)) == 0
        assert 2 * cols * 4 <= n.value <= 2 * max(cols, 1 << 21) * 4


def _laid_out(n, k, sn, sk):
    return torch.zeros(n * max(sn, 1) + k * max(sk, 1)).as_strided((n, k), (sn, sk))


@pytest.mark.parametrize("n,k,gate,up", [
    (50, 1, (64, 1), (1, 1)), (50, 1, (1, 1), (64, 1)), (50, 1, (64, 1), (64 * 2, 64)), (50, 1, (0, 1), (1, 1)),  # one feature
    (1, 8, (8, 1), (1, 2)), (1, 8, (1, 1), (1, 50)), (1, 8, (8, 2), (8, 1)),                                      # one unit
    (5, 8, (8, 1), (9, 1)), (5, 8, (8, 1), (8, 2)), (5, 8, (8, 1), (0, 1)), (5, 8, (1, 5), (1, 5))])
def test_weights_of_two_layouts_are_refused(monkeypatch, n, k, gate, up):
    """Both weights are read by w_gate's row stride and in contiguous rows, also where a matrix has one row or one column."""
    from quickrank_amd import QrError, dense
    monkeypatch.setattr(dense, "_check", lambda t, what, device=None: 0)
    with pytest.raises(QrError) as e:
        dense._weights(torch.zeros(3, k), k, _laid_out(n, k, *gate), _laid_out(n, k, *up), 0)
    assert e.value.code == ARG and "w_" in str(e.value)


@pytest.mark.parametrize("n,k,gate,up,ldw", [
    (50, 1, (64, 1), (64, 1), 64), (50, 1, (64, 7), (64, 1), 64), (50, 1, (0, 1), (0, 1), 0), (1, 8, (8, 1), (99, 1), 8),
    (1, 1, (5, 3), (2, 9), 1), (5, 8, (11, 1), (11, 1), 11), (5, 8, (0, 1), (0, 1), 0)])
def test_weights_of_one_layout(monkeypatch, n, k, gate, up, ldw):
    """Strides of a dimension of one element say nothing about where its element lies."""
    from quickrank_amd import dense
    monkeypatch.setattr(dense, "_check", lambda t, what, device=None: 0)
    assert dense._weights(torch.zeros(3, k), k, _laid_out(n, k, *gate), _laid_out(n, k, *up), 0) == (n, ldw)


def test_forward_mode_tangents_are_refused():
    """A dual tensor requires no gradient; its tangent would be lost without a word."""
    from torch.autograd import forward_ad
    from quickrank_amd import QrError, dense
    x, w = torch.rand(4, 6), torch.rand(6, 6)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: dense.layer_norm(d), lambda: dense.dropout(d, 0.1, 1), lambda: dense.dropout_backward(d, 0.1, 1),
                     lambda: dense.gated_ffn(d, w, w), lambda: dense.layer_norm_backward(x, d, None, x[:, 0], x[:, 0]),
                     lambda: dense.gated_ffn_backward(x, d, w, w, x, x), lambda: dense._check(d, "w_gate")):
            with pytest.raises(QrError) as e:
                call()
            assert e.value.code == ARG and "tangent" in str(e.value)
        with pytest.raises(QrError) as e:
            dense.layer_norm(x)  # one without a tangent
        assert "GPU" in str(e.value)


def test_views_that_are_negated_when_read_are_refused():
    """The imaginary part of a conjugate shares its memory with the number's own: what lies there has the other sign."""
    from quickrank_amd import QrError, dense
    z = torch.complex(torch.rand(5, 1), torch.rand(5, 1))
    x = z.conj().imag
    assert x.is_neg() and x.dtype == torch.float32
    for call in (lambda: dense.layer_norm(x), lambda: dense.dropout(x, 0.1, 1), lambda: dense.gated_ffn(x, x, x)):
        with pytest.raises(QrError) as e:
            call()
        assert e.value.code == ARG and "negated" in str(e.value)
    assert not x.resolve_neg().is_neg()


def test_ffn_of_more_tiles_than_a_launch_has_threads_for_is_unsupported(L):
    """2^24 tiles of 256 threads: rows and outputs within their own limits, in the forward pass and in dx."""
    big, ws = 1 << 56, 1 << 57
    for m, n, type in ((1 << 30, 65, 1), (1 << 30, 128, 0), (1 << 26, 2048, 2), ((1 << 30) - 127, 100, 0)):
        assert ffn(L, type=type, m=m, k=16, n=n, ldx=16, ldw=16, ldh=n, wg=1 << 50, wu=1 << 51, h=big, ws=ws, nbytes=ws) == 5
        assert "tiles" in message(L)
    for m, k, type in ((1 << 30, 128, 1), (1 << 30, 65, 0), (1 << 26, 2048, 2)):
        assert ffn_back(L, type=type, m=m, k=k, dh=big >> 1, x=big >> 2, wg=R + Q, wu=8 * R, g=big >> 3, u=big >> 4, dx=big, lddx=k,
                        dwg=16 * R, dwu=32 * R, ws=ws, nbytes=ws) == 5
        assert "tiles" in message(L)


# matrices of 4 rows of 8 f32: a row is 32 bytes
@pytest.mark.parametrize("bad", [dict(y=P, ldy=9), dict(y=P, ldx=0), dict(y=P + 4, ldx=16, ldy=16), dict(y=P + 28, ldx=16, ldy=16),
                                 dict(y=P + 16, ldx=16, ldy=16), dict(y=P + 64 - 16, ldx=16, ldy=16), dict(y=P + 64 + 4, ldx=16, ldy=16),
                                 dict(y=P + 8), dict(y=P - 8), dict(y=P + 2, ldx=16, ldy=16)])
def test_outputs_that_lie_over_an_input_elsewhere_are_refused(L, bad):
    """Layer norm's and dropout's result may be an input, of one stride, and lie over none otherwise."""
    assert norm(L, **bad) == ARG and "lies over" in message(L)
    assert drop(L, **bad) == ARG and "lies over" in message(L)
    over_residual = {{"x": "r", "ldx": "ldr"}.get(k, k): v for k, v in bad.items()}
    assert drop(L, **{**dict(x=R, r=P, ldr=8), **over_residual}) == ARG and "lies over" in message(L)
    back = {{"y": "dx", "ldy": "lddx", "ldx": "lddy"}.get(k, k): v for k, v in bad.items()}
    assert norm_back(L, **back) == ARG and "lies over" in message(L)
    back = {{"y": "dx", "ldy": "lddx"}.get(k, k): v for k, v in bad.items()}
    assert norm_back(L, **{**back, "dy": R, "x": P}) == ARG and "lies over" in message(L)


@pytest.mark.parametrize("fine", [dict(y=P), dict(y=P, ldx=16, ldy=16), dict(y=P + 32, ldx=16, ldy=16), dict(y=P - 32, ldx=16, ldy=16),
                                  dict(y=P + 36, ldx=17, ldy=17), dict(y=P + 64 * 2 + 32, ldx=16, ldy=16), dict(y=P + 128),
                                  dict(y=P, ldy=9, rows=1)])
def test_outputs_in_place_and_beside_an_input(L, fine):
    """Nothing but the device is missing."""
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    assert norm(L, **fine) in (1, ARG) and "device" in message(L)
    assert drop(L, **fine) in (1, ARG) and "device" in message(L)


def test_ffn_outputs_beside_the_inputs(L):
    """x, h of 4 rows of 8 and 16 in one buffer of rows of 24; dx beside dh: no element is shared.  One element is refused."""
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    W = dict(wg=8 * R, wu=16 * R)
    assert ffn(L, x=P, ldx=24, h=P + 32, ldh=24, **W) in (1, ARG) and "device" in message(L)
    assert ffn(L, x=P, ldx=24, h=P + 28, ldh=24, **W) == ARG and "lies over" in message(L)
    assert ffn(L, x=P, ldx=23, h=P + 32, ldh=23, **W) == ARG and "lies over" in message(L)
    assert ffn_back(L, dh=P, lddh=24, dx=P + 64, lddx=24, x=64 * R) in (1, ARG) and "device" in message(L)
    assert ffn_back(L, dh=P, lddh=24, dx=P + 60, lddx=24, x=64 * R) == ARG and "lies over" in message(L)
    assert ffn_back(L, dh=P, lddh=24, dx=P + 64, lddx=23, x=64 * R) == ARG and "lies over" in message(L)

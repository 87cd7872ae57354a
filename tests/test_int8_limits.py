"""Sizes that do not fit the 32-bit counts of the C entries are refused before they could wrap.  Tensors on the meta device:
shapes and strides without memory."""
import types

import pytest
import torch

from tests.test_int8_refusals import desc, p  # noqa: F401 (p: a fixture)
from tf_depth_estimation_amd import _lib, int8


def meta(shape, strides=None, dtype=torch.float32):
    if strides is None:
        return torch.empty(shape, device="meta", dtype=dtype)
    return torch.empty_strided(shape, strides, device="meta", dtype=dtype)


@pytest.mark.parametrize("shape,strides", [((2 ** 32 + 1, 1), None), ((2 ** 30 + 1, 4), None), ((2 ** 16, 2 ** 15, 3), None),
                                           ((3, 20), (2 ** 32 + 20, 1)), ((3, 20), (2 ** 31, 1)), ((2 ** 30 + 1, 4), (8, 1)),
                                           ((2, 3, 4, 5), (12 * 2 ** 31, 4 * 2 ** 31, 2 ** 31, 1)), ((1, 2 ** 32 + 4), None)])
def test_views_past_the_limits(shape, strides):
    with pytest.raises(ValueError, match="at most 2\\^30 rows"):
        int8._rows(meta(shape, strides), "x")


@pytest.mark.parametrize("shape,strides,want", [((2 ** 30, 4), None, (2 ** 30, 4, 4)),
                                                ((3, 20), (2 ** 31 - 1, 1), (3, 20, 2 ** 31 - 1)),
                                                ((2 ** 15, 2 ** 15, 4), (2 ** 15 * 8, 8, 1), (2 ** 30, 4, 8))])
def test_views_at_the_limits(shape, strides, want):
    assert int8._rows(meta(shape, strides), "x") == want


def conv(kh, kw, cin, K, stride, deconv=False):
    c = object.__new__(int8.Conv8)
    c.kh, c.kw, c.cin, c.K, c.stride, c.deconv = kh, kw, cin, K, stride, deconv
    return c


@pytest.mark.parametrize("c,shape", [(conv(1, 1, 1, 4, 1), (2 ** 32 + 1, 1)), (conv(1, 1, 1, 4, 1), (2 ** 26 + 1, 1)),
                                     (conv(3, 3, 4, 4, 1), (1, 2 ** 32 + 8, 8, 4)), (conv(3, 3, 4, 4, 2), (2 ** 32, 8, 8, 4)),
                                     (conv(3, 3, 4, 4, 2, True), (1, 2 ** 12, 2 ** 13, 4))])
def test_pixels_past_the_limit(c, shape):
    with pytest.raises(ValueError, match="2\\^26"):
        c._make_geometry(torch.Size(shape))


def test_geometry_within_the_limit():
    assert conv(1, 1, 1, 4, 1)._make_geometry(torch.Size((2 ** 26, 1))) == (1, 1, 2 ** 26, (2 ** 26, 4))
    assert conv(3, 3, 4, 8, 2)._make_geometry(torch.Size((2, 7, 9, 4))) == (2, 7, 9, (2, 4, 5, 8))
    assert conv(3, 3, 4, 8, 2, True)._make_geometry(torch.Size((1, 2 ** 12, 2 ** 12, 4)))[3] == (1, 2 ** 13, 2 ** 13, 8)
    assert conv(3, 3, 8, 4, 1)._make_geometry(torch.Size((0, 5, 6, 8)))[3] == (0, 5, 6, 4)


def test_the_calls_refuse(monkeypatch):
    """The public calls reach these checks (tensors taken as if on the current device)."""
    monkeypatch.setattr(int8, "_check", lambda *a, **k: None)
    monkeypatch.setattr(int8._lib, "load", lambda: types.SimpleNamespace())
    many, wide = meta((2 ** 32 + 4, 4)), meta((4, 4), (2 ** 32 + 4, 1))
    beta = types.SimpleNamespace(shape=torch.Size((4,)), is_contiguous=lambda: True, data_ptr=lambda: 0)
    for x in (many, wide):
        with pytest.raises(ValueError, match="2\\^30"):
            int8.quantize_rows(x)
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: 0)
    with pytest.raises(ValueError, match="2\\^30"):
        int8.bn_relu_forward(many, beta)
    with pytest.raises(ValueError, match="2\\^30"):
        int8.Tape8(meta((2 ** 32 + 4, 4), dtype=torch.int8), meta((2 ** 32 + 4, 1)), meta((1, 4)))
    tape = int8.Tape8(meta((4, 4), dtype=torch.int8), meta((4, 1)), meta((1, 4)))
    with pytest.raises(ValueError, match="2\\^30"):
        tape.restore(out=wide)
    with pytest.raises(ValueError, match="2\\^30"):
        int8.bn_relu_backward(tape, beta, wide)


@pytest.mark.parametrize("C", [0, -1, 4097, 2 ** 32 + 4])
def test_channels_past_the_limit(C):
    with pytest.raises(ValueError, match="channels"):
        int8.row_bytes(C)


def test_the_c_entries_refuse_what_wraps(p):  # noqa: F811
    """Sums of a channel offset near 2^31 and products of three sizes near 2^64 are taken without wrapping."""
    lib = _lib.load()
    for co in (2 ** 31 - 4, 2 ** 31 - 1):
        assert lib.tde_q8_rows(2, 4, p, 8, co, p, p, None) == -1
        assert lib.tde_q8_conv2d_bias_act(desc(y_coff=co), p, p, p, p, None, 1, p, None) == -1
        assert lib.tde_q8_deconv2d_bias_act(desc(x_coff=co), p, p, p, p, None, 1, p, None) == -1
        assert lib.tde_q8_conv2d_f32_bias_act(desc(x_coff=co), p, p, p, p, p, None, 1, p, None) == -1
        assert lib.tde_q8_deconv2d_f32_bias_act(desc(y_coff=co), p, p, p, p, p, None, 1, p, None) == -1
    co = 2 ** 31 - 4
    assert lib.tde_tape8_restore(8, 4, p, p, 1, p, 8, co, None) == -1
    assert lib.tde_tape8_bn_fwd(8, 4, 1, p, p, 1e-3, 0.99, 1, None, None, p, p, p, 8, co, p, p, p, 1 << 20, None) == -1
    assert lib.tde_tape8_bn_bwd(8, 4, 1, p, p, p, p, p, 8, co, p, None, 0, None, p, 1 << 20, None) == -1
    for big in (dict(N=1 << 22, H=1 << 21, W=1 << 21), dict(N=1 << 22, OH=1 << 21, OW=1 << 21),
                dict(N=1 << 30, H=1 << 30, W=16)):
        d = desc(**big)
        assert lib.tde_q8_conv2d_bias_act(d, p, p, p, p, None, 1, p, None) == -1, big
        assert lib.tde_q8_deconv2d_bias_act(d, p, p, p, p, None, 1, p, None) == -1, big
        assert lib.tde_q8_one_launch(d, 0) == 0 and lib.tde_q8_one_launch(d, 1) == 0, big


def test_weights_on_another_device(monkeypatch):
    """Conv8 made on one device and called with a tensor of another, current one."""
    monkeypatch.setattr(int8, "_check", lambda *a, **k: None)
    monkeypatch.setattr(int8._lib, "current_device", lambda: 0)
    c = conv(1, 1, 4, 4, 1)
    c.codes = types.SimpleNamespace(get_device=lambda: 1, device="cuda:1")
    with pytest.raises(ValueError, match="weights are on cuda:1"):
        c(meta((5, 4)))

"""What the 8-bit operators refuse, on the host, before any device work."""
import ctypes

import pytest
import torch

from tf_depth_estimation_amd import _lib, int8


def buf(n=4096):
    return ctypes.create_string_buffer(n + 64)


def aligned(b):
    a = ctypes.addressof(b)
    return ctypes.c_void_p((a + 15) // 16 * 16)


@pytest.fixture()
def p():
    b = buf()
    v = aligned(b)
    v.keep = b
    return v


def test_cpu_and_wrong_type_tensors_are_refused():
    with pytest.raises(ValueError, match="on the GPU"):
        int8.quantize_rows(torch.zeros(2, 4))
    with pytest.raises(ValueError, match="float32"):
        int8.quantize_rows(torch.zeros(2, 4, dtype=torch.float16))
    with pytest.raises(ValueError, match="weights"):
        int8.Conv8(torch.zeros(3, 3, 4, 4))
    with pytest.raises(ValueError, match="stride"):
        int8.Conv8(torch.zeros(3, 3, 4, 4), stride=0)
    with pytest.raises(ValueError, match="z must"):
        int8.bn_relu_forward(torch.zeros(2, 4), torch.zeros(4))
    with pytest.raises(ValueError, match="Tape8"):
        int8.bn_relu_backward(None, torch.zeros(4), torch.zeros(2, 4))
    with pytest.raises(ValueError, match="int8"):
        int8.Tape8(torch.zeros(2, 4), torch.zeros(2, 1), torch.zeros(1, 4))


@pytest.mark.parametrize("shape,strides,ok", [((2, 3, 4, 5), (60, 20, 5, 1), True), ((2, 3, 4, 5), (96, 32, 8, 1), True),
                                              ((1, 1, 4, 5), (7, 9, 8, 1), True), ((2, 3, 4, 5), (1, 60, 20, 5), False),
                                              ((2, 3, 4, 5), (60, 24, 5, 1), False), ((3, 5), (0, 1), False),
                                              ((3, 5), (4, 1), False), ((3, 5), (10, 2), False), ((6, 1), (3, 9), True)])
def test_channel_views(shape, strides, ok):
    t = torch.zeros(4096).as_strided(shape, strides)
    if ok:
        rows, C, cs = int8._rows(t, "x")
        assert (rows, C) == (t.numel() // shape[-1], shape[-1]) and cs >= C
    else:
        with pytest.raises(ValueError, match="channel view"):
            int8._rows(t, "x")


def test_row_bytes():
    lib = _lib.load()
    assert [lib.tde_q8_row_bytes(c) for c in (1, 32, 33, 64, 65, 4096)] == [32, 32, 64, 64, 128, 4096]
    assert [lib.tde_q8_row_bytes(c) for c in (0, -1, 4097)] == [0, 0, 0]
    with pytest.raises(ValueError, match="channels"):
        int8.row_bytes(5000)
    assert lib.tde_q8_weights_size(9, 17, 10) == 9 * 16 * 32
    assert lib.tde_q8_weights_size(9, 4097, 10) == 0 and lib.tde_q8_weights_size(0, 4, 4) == 0


def test_rows_arguments(p):
    lib = _lib.load()
    bad = [(0, 4, p, 4, 0, p, p), (2, 0, p, 4, 0, p, p), (2, 5000, p, 5000, 0, p, p), (2, 4, None, 4, 0, p, p),
           (2, 4, p, 4, 1, p, p), (2, 4, p, 8, -1, p, p), (2, 4, p, 4, 0, None, p), (2, 4, p, 4, 0, p, None),
           (2, 4, p, 4, 0, ctypes.c_void_p(p.value + 4), p)]
    for a in bad:
        assert lib.tde_q8_rows(*a, None) == -1, a
    assert lib.tde_q8_weights(9, 4, 4, 2, p, p, p, None) == -1
    assert lib.tde_q8_weights(9, 5000, 4, 0, p, p, p, None) == -1
    assert lib.tde_q8_weights(9, 4, 4, 0, None, p, p, None) == -1


def desc(**kw):
    d = _lib.ConvDesc(N=1, H=8, W=8, C=4, OH=8, OW=8, K=4, KH=3, KW=3, stride=1, pad_top=1, pad_left=1, w_cin=4,
                      x_cstride=4, x_coff=0, y_cstride=4, y_coff=0)
    for k, v in kw.items():
        setattr(d, k, v)
    return ctypes.byref(d)


def test_conv_arguments(p):
    lib = _lib.load()
    for fn, view in ((lib.tde_q8_conv2d_bias_act, "y"), (lib.tde_q8_deconv2d_bias_act, "x")):
        for kw in (dict(N=0), dict(H=0), dict(OW=-1), dict(KH=0), dict(KW=65), dict(stride=0), dict(pad_top=3),
                   dict(pad_left=-1), dict(N=1 << 28), {view + "_coff": 1}, {view + "_coff": -4}, {view + "_cstride": 3},
                   dict(w_cin=5000, K=5000)):
            assert fn(desc(**kw), p, p, p, p, None, 1, p, None) == -1, kw
        assert fn(desc(), p, p, p, p, None, 2, p, None) == -1
        for i in (0, 1, 2, 3, 5):
            args = [p, p, p, p, p, p]
            args[i] = None
            assert fn(desc(), args[0], args[1], args[2], args[3], None, 1, args[5], None) == -1, i
        assert fn(None, p, p, p, p, None, 1, p, None) == -1
    for fn, view, src in ((lib.tde_q8_conv2d_f32_bias_act, "y", "x"), (lib.tde_q8_deconv2d_f32_bias_act, "x", "y")):
        for kw in (dict(N=0), dict(stride=0), dict(pad_top=3), dict(N=1 << 28), {view + "_cstride": 3}, {src + "_coff": 1},
                   {src + "_coff": -4}, {src + "_cstride": 3}, dict(w_cin=5000, K=5000)):
            assert fn(desc(**kw), p, p, p, p, p, None, 1, p, None) == -1, kw
        for i in (0, 1, 2, 3, 4, 6):          # (codes and scales: this geometry takes two launches)
            args = [p, p, p, p, p, None, p]
            args[i] = None
            assert fn(desc(), *args[:6], 1, args[6], None) == -1, i
        assert fn(None, p, p, p, p, p, None, 1, p, None) == -1


def test_one_launch(p):
    lib = _lib.load()
    d = desc(H=1, W=1, OH=1, OW=1, KH=1, KW=1, pad_top=0, pad_left=0, C=64, w_cin=64, K=64, x_cstride=64, y_cstride=64)
    assert lib.tde_q8_one_launch(d, 0) == 1        # ... but not onto the input: then the codes are needed
    assert lib.tde_q8_conv2d_f32_bias_act(d, p, None, None, p, p, None, 1, p, None) == -1
    small = dict(H=4, W=4, OH=4, OW=4, C=64, w_cin=64, K=64, x_cstride=64, y_cstride=64)
    assert [lib.tde_q8_one_launch(desc(**{**small, **kw}), dec) for kw, dec in (
        (dict(), 0), (dict(), 1), (dict(x_cstride=66), 0), (dict(x_coff=2, x_cstride=68), 0), (dict(w_cin=32), 0),
        (dict(N=0), 0), (dict(H=400, W=400, OH=400, OW=400), 0), (dict(H=40, W=40, OH=4, OW=4, stride=10), 0))
            ] == [1, 1, 0, 0, 0, 0, 0, 0]
    assert lib.tde_q8_one_launch(None, 0) == 0


def test_tape_arguments(p):
    lib = _lib.load()
    odd = ctypes.c_void_p(p.value + 4)
    big = 1 << 20
    assert lib.tde_tape8_workspace_size(0, 4) == 0 and lib.tde_tape8_workspace_size(8, 6) == 0
    assert lib.tde_tape8_workspace_size(8, 1028) == 0 and lib.tde_tape8_workspace_size(8, 4) > 0

    def fwd(M=8, C=4, G=1, z=p, beta=p, mm=None, mv=None, sm=p, si=p, y=p, cs=4, co=0, codes=p, scales=p, ws=p, nb=big):
        return lib.tde_tape8_bn_fwd(M, C, G, z, beta, 1e-3, 0.99, 1, mm, mv, sm, si, y, cs, co, codes, scales, ws, nb, None)

    for kw in (dict(M=0), dict(C=3), dict(C=1028, cs=1028), dict(G=0), dict(G=9), dict(G=3), dict(z=None), dict(z=odd),
               dict(beta=None), dict(mm=p), dict(sm=None), dict(si=None), dict(y=None), dict(y=odd), dict(cs=6),
               dict(co=4), dict(co=-4), dict(codes=None), dict(codes=odd), dict(scales=None)):
        assert fwd(**kw) == -1, kw
    # (few rows run as one launch that needs no workspace)
    assert lib.tde_tape8_one_launch(8, 4, 1) == 1 and lib.tde_tape8_one_launch(1 << 20, 4, 2) == 0
    assert lib.tde_tape8_one_launch(8, 4, 3) == 0
    assert fwd(M=1 << 20, nb=16) == -2 and fwd(M=1 << 20, ws=None) == -2 and fwd(M=1 << 20, ws=odd) == -2

    def bwd(M=8, C=4, G=1, codes=p, scales=p, si=p, beta=p, dy=p, cs=4, co=0, dz=p, ws=p, nb=big):
        return lib.tde_tape8_bn_bwd(M, C, G, codes, scales, si, beta, dy, cs, co, dz, None, 0, None, ws, nb, None)

    for kw in (dict(M=0), dict(C=2), dict(G=3), dict(codes=None), dict(scales=None), dict(si=None), dict(si=odd),
               dict(beta=None), dict(beta=odd), dict(dy=None), dict(dy=odd), dict(cs=5), dict(co=8), dict(dz=None),
               dict(dz=odd)):
        assert bwd(**kw) == -1, kw
    assert bwd(M=1 << 20, nb=16) == -2
    assert lib.tde_tape8_restore(8, 4, p, p, 2, p, 4, 0, None) == -1
    assert lib.tde_tape8_restore(8, 4, p, p, 1, p, 4, 4, None) == -1
    good = _lib.TapeRestore(8, 4, p.value, p.value, p.value, 4, 0)
    for n, bad in ((0, good), (17, good), (1, _lib.TapeRestore(8, 6, p.value, p.value, p.value, 8, 0)),
                   (2, _lib.TapeRestore(8, 4, p.value, p.value, odd.value, 4, 0)),
                   (2, _lib.TapeRestore(8, 4, p.value, None, p.value, 4, 0))):
        jobs = (_lib.TapeRestore * 17)(*([good] * 17))
        jobs[max(n - 1, 0)] = bad
        assert lib.tde_tape8_restore_multi(jobs, n, 1, None) == -1, n
    assert lib.tde_tape8_restore_multi(None, 1, 1, None) == -1
    assert lib.tde_tape8_bn_fwd_from_sums(8, 4, 2, 3, p, p, p, 1e-3, 0.99, 1, None, None, p, p, p, 4, 0, p, p, None) == -1
    assert lib.tde_tape8_bn_bwd_sums(8, 4, 1, p, p, p, p, 4, 0, None, None, p, big, None) == -1
    assert lib.tde_tape8_bn_bwd_from_sums(8, 4, 1, 7, p, p, p, p, p, 4, 0, p, p, p, None, 0, None, None) == -1


def test_tape_contexts_nest():
    assert not int8.tape8_active()
    with int8.tape8():
        assert int8.tape8_active()
        with int8.tape8(False):
            assert not int8.tape8_active()
        assert int8.tape8_active()
    assert not int8.tape8_active()

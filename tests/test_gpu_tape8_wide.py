"""The many-row forms of the 8-bit tape on views whose pixels lie 2^29 floats apart: the offset of a lane's row within a step
passes 2^31 (row 4) and 2^32 (row 8).  Given sums always take these forms, few rows too."""
import numpy as np
import pytest
import torch

from tests.test_gpu_int8 import dev, tape_data
from tf_depth_estimation_amd import _lib, int8

pytestmark = pytest.mark.gpu

STEP, M, C = 1 << 29, 9, 20


def wide(extra=0):
    """[M, C] view with pixel stride STEP (17 GB)."""
    buf = torch.empty((M - 1) * STEP + C + extra, device="cuda")
    v = buf.as_strided((M, C), (STEP, 1))
    v.fill_(-3.5)
    return v


def test_forward_from_sums():
    z, beta, _ = tape_data(M, C)
    zd, bd = dev(z), dev(beta)
    sums = torch.stack([zd.double().sum(0), (zd.double() ** 2).sum(0)]).view(1, 2, C).contiguous()
    got = []
    for y, cs in ((wide(), STEP), (torch.empty(M, C, device="cuda"), C)):
        codes = torch.empty(M, C, device="cuda", dtype=torch.int8)
        scales, st = torch.empty(M, 1, device="cuda"), torch.empty(2, C, device="cuda")
        _lib.check(_lib.load().tde_tape8_bn_fwd_from_sums(
            M, C, 1, M, zd.data_ptr(), sums.data_ptr(), bd.data_ptr(), 1e-3, 0.99, 1, None, None, st[0].data_ptr(),
            st[1].data_ptr(), y.data_ptr(), cs, 0, codes.data_ptr(), scales.data_ptr(), _lib.stream_ptr()), "forward")
        got.append((y.clone(), codes, scales, st))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_backward_from_sums():
    z, beta, r = tape_data(M, C)
    _, tape = int8.bn_relu_forward(dev(z), dev(beta))
    bd, dense = dev(beta), dev(r.standard_normal((M, C)).astype(np.float32))
    dyw = wide()
    dyw.copy_(dense)
    codes, scales, invstd = tape.codes.contiguous(), tape.scales.contiguous(), tape.invstd.clone()
    lib = _lib.load()
    nb = lib.tde_tape8_workspace_size(M, C)
    ws = torch.empty(nb, device="cuda", dtype=torch.uint8)
    got = []
    for dy, cs in ((dyw, STEP), (dense, C)):
        sums, copy = torch.empty(1, 2, C, device="cuda", dtype=torch.float64), torch.empty(2, C, device="cuda", dtype=torch.float64)
        dz, db = torch.empty(M, C, device="cuda"), torch.empty(C, device="cuda")
        _lib.check(lib.tde_tape8_bn_bwd_sums(M, C, 1, codes.data_ptr(), scales.data_ptr(), bd.data_ptr(), dy.data_ptr(), cs, 0,
                                             sums.data_ptr(), copy.data_ptr(), ws.data_ptr(), nb, _lib.stream_ptr()), "sums")
        _lib.check(lib.tde_tape8_bn_bwd_from_sums(
            M, C, 1, M, codes.data_ptr(), scales.data_ptr(), invstd.data_ptr(), bd.data_ptr(), dy.data_ptr(), cs, 0,
            sums.data_ptr(), copy.data_ptr(), dz.data_ptr(), db.data_ptr(), 0, None, _lib.stream_ptr()), "backward")
        got.append((sums, copy, dz, db))
    for a, b in zip(*got):
        assert torch.equal(a, b)

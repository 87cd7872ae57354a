"""The 8-bit tape's codes are floor(128 |u| / max|u|) with the block's maximum unrounded (include/tde.h): a division by the
stored fp32 scale gives another code where |u| lies between the two borders."""
import numpy as np
import pytest
import torch

from tests import int8_oracle as O
from tests.test_gpu_int8 import dev, tape_data
from tf_depth_estimation_amd import _lib, int8

pytestmark = pytest.mark.gpu


def encode(u):
    """Codes [M, C] of float64 pre-activations."""
    M, C = u.shape
    q = np.zeros((M, C))
    for c in range(0, C, 64):
        ub = u[:, c:c + 64]
        a = np.abs(ub).max(axis=1, keepdims=True)
        t = np.where(a > 0, np.minimum(np.floor(128 * np.abs(ub) / np.where(a > 0, a, 1)), 127), 0)
        q[:, c:c + 64] = np.where(ub > 0, t, -1 - t)
    return q.astype(np.int8)


# M, C, groups, codes that the rounded scale would change
CASES = [(8200, 4, 1, 1), (40000, 68, 8, 3), (98304, 16, 1, 3), (96, 512, 1, 0), (513, 64, 1, 0)]


@pytest.mark.parametrize("M,C,G,other", CASES)
def test_codes_of_the_forward(M, C, G, other):
    z, beta, _ = tape_data(M, C)
    u = O.bn_forward(z, beta, G)[0]
    codes = encode(u)
    if other:
        assert (O.tape_encode(u)[0] != codes).sum() == other
    _, tape = int8.bn_relu_forward(dev(z), dev(beta), groups=G)
    np.testing.assert_array_equal(tape.codes.cpu().numpy(), codes)


@pytest.mark.parametrize("C,L", [(4, 1), (8, 2), (16, 4), (32, 8), (64, 16), (128, 16)])
def test_codes_between_the_borders(C, L):
    """Given sums of mean 0 and variance 1, u = z + beta up to the last bits of fp64.  Channel 0 of a block holds the
    maximum 1 + d, |d| < 2^-25 or so, which rounds to 1 in fp32, and the others k / 128 (1 + d / 2): with the unrounded
    maximum their codes are k - 1 for d > 0 and k for d < 0, with the rounded one k and k - 1."""
    M = 40
    for d in (0.45 * 2.0 ** -23, -0.45 * 2.0 ** -24):
        z, beta = np.zeros((M, C), np.float32), np.zeros(C, np.float32)
        want = np.zeros((M, C), np.int8)
        r = np.random.default_rng([C, d > 0])
        ks = np.array([127 if c % 64 == 0 else r.integers(2, 127) for c in range(C)])
        for c in range(C):
            if c % 64 == 0:
                z[:, c], beta[c], want[:, c] = 1, d, 127
            else:
                z[:, c], beta[c], want[:, c] = ks[c] / 128, ks[c] / 128 * (d / 2), ks[c] - 1 if d > 0 else ks[c]
        z[1::2, 0::64] = 0.5                  # other rows: another maximum, no borders to check
        u = z.astype(np.float64) + beta
        assert (np.abs(u[0, 0::64]).astype(np.float32) == 1).all()
        np.testing.assert_array_equal(encode(u)[0::2], want[0::2])
        sums = torch.zeros(1, 2, C, dtype=torch.float64)
        sums[0, 1] = M                        # variance 1 with eps 0
        zd, bd, sd = dev(z), dev(beta), sums.cuda()
        y = torch.empty(M, C, device="cuda")
        codes = torch.empty(M, C, device="cuda", dtype=torch.int8)
        scales = torch.empty(M, (C + 63) // 64, device="cuda")
        st = torch.empty(2, C, device="cuda")
        _lib.check(_lib.load().tde_tape8_bn_fwd_from_sums(
            M, C, 1, M, zd.data_ptr(), sd.data_ptr(), bd.data_ptr(), 0.0, 0.99, 1, None, None, st[0].data_ptr(),
            st[1].data_ptr(), y.data_ptr(), C, 0, codes.data_ptr(), scales.data_ptr(), _lib.stream_ptr()), "forward")
        np.testing.assert_array_equal(codes.cpu().numpy(), encode(u))
        assert (scales.cpu().numpy()[0::2] == np.float32(1 / 128)).all()


def test_codes_of_tiny_and_zero_blocks():
    """A block whose maximum is subnormal in fp32, or rounds to scale 0, keeps its signs and its quotients' codes."""
    C = 64
    beta = (np.linspace(-1, 1, C) * 1e-40).astype(np.float32)
    z = np.zeros((8, C), np.float32)
    _, tape = int8.bn_relu_forward(dev(z), dev(beta))
    np.testing.assert_array_equal(tape.codes.cpu().numpy(), encode(np.tile(beta.astype(np.float64), (8, 1))))
    _, tape = int8.bn_relu_forward(dev(z), torch.zeros(C, device="cuda"))
    assert (tape.codes.cpu().numpy() == -1).all() and not tape.scales.cpu().numpy().any()

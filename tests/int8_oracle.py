"""Plain 64-bit implementations of the 8-bit activation operators (NumPy), for tests/test_gpu_int8.py."""
import numpy as np


def quantize(x, axis):
    """codes (float64 holding integers) and float32 scales of x: one scale per index outside `axis`."""
    x = np.asarray(x, dtype=np.float64)
    a = np.abs(x).max(axis=axis, keepdims=True)
    bad = ~np.isfinite(a)
    safe = np.where((a > 0) & ~bad, a, 1.0)
    q = np.where(bad | (a == 0), 0.0, np.rint(np.where(bad, 0.0, x) * 127.0 / safe))
    with np.errstate(invalid="ignore"):
        s = np.where(bad, np.nan, np.where(bad, 0.0, a) / 127.0).astype(np.float32)
    return q, s


def same_pad(n, k, s):
    out = -(-n // s)
    return out, max((out - 1) * s + k - n, 0) // 2


def conv8(x, w, b, s, deconv, relu):
    """(y, sum of the absolute products) of the 8-bit conv of x [N,H,W,C]; w conv [k,k,C,K] / deconv [k,k,K,C]."""
    k = w.shape[0]
    kw = w.shape[1]
    wt = w.transpose(0, 1, 3, 2) if deconv else w
    C, K = wt.shape[2:]
    qx, sx = quantize(x, 3)
    qw, sw = quantize(wt.reshape(-1, K), 0)
    qw, sw = qw.reshape(k, kw, C, K), sw.reshape(K).astype(np.float64)
    sx = sx.astype(np.float64)
    N, H, W = x.shape[:3]
    OH, OW = (H * s, W * s) if deconv else (same_pad(H, k, s)[0], same_pad(W, kw, s)[0])
    pt, pl = (same_pad(OH, k, s)[1], same_pad(OW, kw, s)[1]) if deconv else (same_pad(H, k, s)[1], same_pad(W, kw, s)[1])
    y, mag = np.zeros((N, OH, OW, K)), np.zeros((N, OH, OW, K))
    for ty in range(k):
        for tx in range(kw):
            p = (qx.reshape(-1, C) @ qw[ty, tx]).reshape(N, H, W, K) * sx
            pm = (np.abs(qx).reshape(-1, C) @ np.abs(qw[ty, tx])).reshape(N, H, W, K) * sx
            for o in range(OH):
                num = o + pt - ty if deconv else o * s + ty - pt
                if deconv and num % s:
                    continue
                i = num // s if deconv else num
                if not 0 <= i < H:
                    continue
                for q in range(OW):
                    num = q + pl - tx if deconv else q * s + tx - pl
                    if deconv and num % s:
                        continue
                    j = num // s if deconv else num
                    if 0 <= j < W:
                        y[:, o, q] += p[:, i, j]
                        mag[:, o, q] += pm[:, i, j]
    y, mag = y * sw + b, mag * sw + np.abs(b)
    return (np.where(y < 0, 0, y) if relu else y), mag


def tape_encode(u):
    """codes [M, C] and float32 scales [M, blocks] of float64 pre-activations."""
    M, C = u.shape
    nb = -(-C // 64)
    s = np.zeros((M, nb), np.float32)
    q = np.zeros((M, C))
    for b in range(nb):
        ub = u[:, 64 * b:64 * b + 64]
        with np.errstate(invalid="ignore", over="ignore"):
            a = np.abs(ub).max(axis=1).astype(np.float32)
        bad = ~np.isfinite(a) | np.isnan(ub).any(axis=1)
        sb = np.where(bad, np.nan, a / np.float32(128)).astype(np.float32)
        sd = np.where(bad | (sb == 0), 1.0, sb).astype(np.float64)[:, None]
        with np.errstate(invalid="ignore"):
            t = np.minimum(np.floor(np.abs(ub) / sd), 127)
            t = np.where((bad | (sb == 0))[:, None], 0, t)
            q[:, 64 * b:64 * b + 64] = np.where(ub > 0, t, -1 - t)
        s[:, b] = sb
    return q.astype(np.int8), s


def tape_value(codes, scales):
    C = codes.shape[1]
    return (codes.astype(np.float64) + 0.5) * np.repeat(scales.astype(np.float64), 64, axis=1)[:, :C]


def bn_forward(z, beta, groups, eps=1e-3):
    """u [M, C], mean, invstd, biased variance [groups, C] in float64."""
    M, C = z.shape
    zg = z.astype(np.float64).reshape(groups, M // groups, C)
    mean = zg.mean(axis=1)
    var = ((zg - mean[:, None]) ** 2).mean(axis=1)
    invstd = 1 / np.sqrt(var + np.float32(eps).astype(np.float64))
    u = (zg - mean[:, None]) * invstd[:, None] + beta.astype(np.float64)
    return u.reshape(M, C), mean, invstd, var


def bn_backward(codes, scales, invstd, beta, dy, groups):
    """dz [M, C], dbeta [C] and the bound of a float32 evaluation's error of dz."""
    M, C = codes.shape
    n = M // groups
    uv = tape_value(codes, scales)
    xh = (uv - beta.astype(np.float64)).reshape(groups, n, C)
    g = np.where(codes >= 0, dy.astype(np.float64), 0.0).reshape(groups, n, C)
    is_ = invstd.astype(np.float64)[:, None]
    m0, m1 = g.mean(axis=1, keepdims=True), (g * xh).mean(axis=1, keepdims=True)
    dz = is_ * (g - m0 - xh * m1)
    # float32 steps, each off by at most half a step e = 2^-24 of its result: the value (q + 1/2) s and its difference
    # with beta (exh), the mean of g xhat through exh and its own rounding (em1), the mean of g (m0), then xhat * m1, two
    # subtractions and the product with invstd
    e = 2.0 ** -24
    exh = e * (np.abs(uv).reshape(groups, n, C) + np.abs(xh))
    em1 = (np.abs(g) * exh).mean(axis=1, keepdims=True) + e * np.abs(m1)
    mag = np.abs(g) + np.abs(m0) + np.abs(xh * m1)
    bound = is_ * (np.abs(xh) * em1 + exh * np.abs(m1) + e * np.abs(m0) + 3 * e * mag) + e * np.abs(dz)
    return dz.reshape(M, C), g.sum(axis=(0, 1)), 1.01 * bound.reshape(M, C) + 1e-30

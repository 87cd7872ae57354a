"""Activations held as 8-bit codes with fp32 scales: an integer conv for prediction and an 8-bit tape for training.

The reference computes and keeps everything in fp32 (nets_optflow_depth.py:76-147 has no reduced form); both uses are
opt-in here.

  * `Conv8` -- a conv / transposed conv + bias + ReLU as a product of 8-bit integers with one scale per input pixel
    (token) and one per output channel; a 1x1 conv on [M, C] rows is the plain product of tokens and weights.
    `batch_prediction.Predictor(int8=True)` runs every folded conv layer this way.
  * `bn_relu_forward` / `bn_relu_backward` / `Tape8` -- training BatchNorm + ReLU whose backward needs one byte per
    element (the coded pre-activation: its sign is the ReLU mask, its value both the normalised input and, through
    `Tape8.restore`, the layer's output).  `program.NetRun(tape8=True)`, `train.Trainer.enable_tape8` and `tape8()` use
    it for whole networks.

Like the rest of the package these are calls on the current stream of the current device without a CPU fallback;
none of them records an autograd graph (an input that requires a gradient is refused while gradients are enabled, one with a
forward-mode tangent always).
The formulas stand in include/tde.h, "8-bit activations".
"""
import contextlib
import contextvars
import ctypes
import functools
import weakref

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import ConvDesc
from .program import same_pad

BLOCK = 64            # TDE_TAPE8_BLOCK: channels of a row that share a tape scale
MAX_CHANNELS = 4096   # of a Conv8 input
# what the C entries take: they count rows and strides in 32 bits, where larger numbers would wrap on the way there
MAX_ROWS = 1 << 30
MAX_PIXELS = 1 << 26  # of a Conv8 input or output
MAX_STRIDE = (1 << 31) - 1


def _check(t, name, dtype=torch.float32):
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or not t.is_cuda:
        raise ValueError(f"{name} must be a {str(dtype).split('.')[-1]} tensor on the GPU")
    if t.get_device() != _lib.current_device():
        raise ValueError(f"{name} is on {t.device}, not on the current device (cuda:{_lib.current_device()})")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: 8-bit operators record none (detach it, or use torch.no_grad())")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:      # (-1: outside any level)
        raise ValueError(f"{name} has a forward-mode tangent: 8-bit operators carry none")


def _rows(t, name):
    """(rows, C, pixel stride) of a [..., C] channel view: consecutive pixels a fixed stride apart."""
    shape = t.shape
    if len(shape) < 2:
        raise ValueError(f"{name} must have at least two dimensions, got {tuple(shape)}")
    C = shape[-1]
    if C and t.is_contiguous():
        rows = t.numel() // C
        if rows > MAX_ROWS or C > MAX_STRIDE:
            raise ValueError(f"{name}: {rows} rows of {C}: at most 2^30 rows of 2^31 - 1")
        return rows, C, C
    rows, cs = 1, None
    for n, s in zip(reversed(shape[:-1]), reversed(t.stride()[:-1])):
        if n != 1:
            if cs is None:
                cs = s
            elif s != rows * cs:
                raise ValueError(f"{name} must be a pixel-major channel view (strides {t.stride()})")
        rows *= n
    cs = C if cs is None else cs
    if rows and (C == 0 or (C > 1 and t.stride(-1) != 1) or cs < C):
        raise ValueError(f"{name} must be a pixel-major channel view of at least one channel (strides {t.stride()})")
    if rows > MAX_ROWS or cs > MAX_STRIDE:
        raise ValueError(f"{name}: {rows} rows {cs} apart: at most 2^30 rows and a pixel stride of 2^31 - 1")
    return rows, C, cs


@functools.lru_cache(maxsize=1024)
def _strides(shape):
    st, n = [], 1
    for s in reversed(shape):
        st.append(n)
        n *= max(s, 1)
    return tuple(reversed(st))


def _out(out, shape, device, name="out"):
    if out is None:      # (empty_strided: 1.3 us, torch.empty of a torch.Size 2.1)
        return torch.empty_strided(shape, _strides(shape), dtype=torch.float32, device=device)
    _check(out, name)
    if out.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(out.shape)}")
    return out


# ---------------------------------------------------------------- integer product
@functools.lru_cache(maxsize=None)
def row_bytes(C):
    if not 1 <= C <= MAX_CHANNELS:
        raise ValueError(f"{C} channels: 1 to {MAX_CHANNELS} are supported")
    return _lib.load().tde_q8_row_bytes(C)


class Rows8:
    """Pixels as 8-bit codes with a scale each; `shape` is that of the fp32 tensor [..., C].  One row more than pixels:
    the last is all zero (the pixel outside the image).  `codes` is [rows + 1, row_bytes(C)], `scales` [rows + 1]."""

    def __init__(self, shape, device="cuda"):
        self.C, self.rows = shape[-1], 1
        for n in shape[:-1]:
            self.rows *= n
        self.row_bytes = row_bytes(self.C)
        self._scales_at = (self.rows + 1) * self.row_bytes       # one buffer: scales behind the codes
        self.buffer = torch.empty(self._scales_at + 4 * (self.rows + 1), dtype=torch.int8, device=device)
        self.shape = tuple(shape)

    @property
    def codes(self):
        return self.buffer[:self._scales_at].view(self.rows + 1, self.row_bytes)

    @property
    def scales(self):
        return self.buffer[self._scales_at:].view(torch.float32)

    def pointers(self):
        p = self.buffer.data_ptr()
        return p, p + self._scales_at


def quantize_rows(x, out=None):
    """fp32 [..., C] channel view -> Rows8.  out: a Rows8 of the same rows and channels to write into."""
    _check(x, "x")
    rows, C, cs = _rows(x, "x")
    if out is None:
        out = Rows8(x.shape, x.device)
    elif not isinstance(out, Rows8) or (out.rows, out.C) != (rows, C):
        raise ValueError(f"out must be the Rows8 of {rows} rows of {C} channels")
    else:
        _check(out.buffer, "out", torch.int8)
        out.shape = tuple(x.shape)
    if rows:
        codes, scales = out.pointers()
        _lib.check(_lib.load().tde_q8_rows(rows, C, x.data_ptr(), cs, 0, codes, scales,
                                           _lib.raw_stream(x.get_device())), "quantize_rows")
    return out


class Conv8:
    """One conv layer in 8-bit integers: y = relu?(conv(x, weights) + bias), TF 'SAME' padding.

    weights: conv [KH, KW, Cin, Cout], or with deconv=True conv2d_transpose [KH, KW, Cout, Cin] (the TF checkpoint
    layouts), fp32.  They are quantised once (per output channel) by __init__ / load; later changes of the tensor are not
    seen, as with NetProgram.fold_bn.  load of weights of the same shape writes the buffers in place, so a captured graph of
    calls goes on with the new ones; after a load of another shape (or of a bias where there was none) it must be captured
    again."""

    def __init__(self, weights, bias=None, stride=1, relu=True, deconv=False):
        if not isinstance(stride, int) or not 1 <= stride <= 64:
            raise ValueError(f"stride {stride!r}: an integer from 1 to 64 is expected")
        self.stride, self.relu, self.deconv = stride, bool(relu), bool(deconv)
        self.load(weights, bias)

    def load(self, weights, bias=None):
        _check(weights, "weights")
        if weights.dim() != 4 or 0 in weights.shape:
            raise ValueError(f"weights must be [KH, KW, Cin, Cout] or [KH, KW, Cout, Cin], got {tuple(weights.shape)}")
        kh, kw, a, b = weights.shape
        cin, K = (b, a) if self.deconv else (a, b)
        if max(kh, kw) > 64 or K > 65535:
            raise ValueError(f"weights {tuple(weights.shape)}: at most 64x64 taps and 65535 output channels")
        row_bytes(cin)
        if bias is not None:
            _check(bias, "bias")
            if tuple(bias.shape) != (K,):
                raise ValueError(f"bias must be ({K},), got {tuple(bias.shape)}")
        lib = _lib.load()
        w = weights.contiguous()
        if (kh, kw, cin, K, w.device) != getattr(self, "_loaded", None):
            codes = torch.empty(lib.tde_q8_weights_size(kh * kw, cin, K), dtype=torch.int8, device=w.device)
            scales = torch.empty((K + 15) // 16 * 16, dtype=torch.float32, device=w.device)
            me = weakref.ref(self)      # (a cache that held the layer would keep its weights until a garbage collection)
            self._geometry = functools.lru_cache(maxsize=64)(lambda *a: me()._make_geometry(*a))
            self._desc = functools.lru_cache(maxsize=64)(lambda *a: me()._make_desc(*a))
            self.codes, self.scales, self.bias = codes, scales, None
            self.kh, self.kw, self.cin, self.K = kh, kw, cin, K
            self._loaded = (kh, kw, cin, K, w.device)
        if bias is None:
            self.bias = None
        elif self.bias is None:
            self.bias = bias.detach().clone().contiguous()
        else:
            with torch.inference_mode():      # (a bias cloned in that mode takes no other writes)
                self.bias.copy_(bias)
        _lib.check(lib.tde_q8_weights(kh * kw, cin, K, 1 if self.deconv else 0, w.data_ptr(), self.codes.data_ptr(),
                                      self.scales.data_ptr(), _lib.raw_stream(w.get_device())), "Conv8 weights")
        return self

    def out_size(self, H, W):
        if self.deconv:
            return H * self.stride, W * self.stride
        return same_pad(H, self.kh, self.stride)[0], same_pad(W, self.kw, self.stride)[0]

    def _make_geometry(self, shape):
        """(N, H, W, output shape) of an input shape."""
        if shape[-1] != self.cin:
            raise ValueError(f"x has {shape[-1]} channels, the weights {self.cin}")
        if len(shape) == 2 and (self.kh, self.kw, self.stride) == (1, 1, 1):
            N, H, W, oshape = 1, 1, shape[0], (shape[0], self.K)
        elif len(shape) != 4:
            raise ValueError(f"x must be [N, H, W, C], or [M, C] for a 1x1 stride-1 conv, got {tuple(shape)}")
        else:
            N, H, W = shape[:3]
            oshape = (N,) + self.out_size(H, W) + (self.K,)
        OH, OW = self.out_size(H, W)
        if max(N * H * W, N * OH * OW) > MAX_PIXELS:
            raise ValueError(f"x {tuple(shape)}: at most 2^26 input and output pixels")
        return N, H, W, torch.Size(oshape)

    def _make_desc(self, N, H, W, ics, ocs):
        """The conv descriptor of a batch whose input and output have pixel strides ics and ocs (a transposed conv's is
        that of its virtual forward conv), and whether the call is one launch if the input starts on 16 bytes."""
        OH, OW = self.out_size(H, W)
        d = ConvDesc()
        big, small = ((OH, OW), (H, W)) if self.deconv else ((H, W), (OH, OW))
        d.N, (d.H, d.W), (d.OH, d.OW) = N, big, small
        d.C, d.K = (self.K, self.cin) if self.deconv else (self.cin, self.K)
        d.w_cin = d.C
        d.KH, d.KW, d.stride = self.kh, self.kw, self.stride
        d.pad_top, d.pad_left = same_pad(d.H, self.kh, self.stride)[1], same_pad(d.W, self.kw, self.stride)[1]
        d.x_cstride, d.y_cstride = (ocs, ics) if self.deconv else (ics, ocs)
        return d, bool(_lib.load().tde_q8_one_launch(ctypes.byref(d), self.deconv))

    quantize = staticmethod(quantize_rows)      # the Rows8 of an input, for several layers that read it

    def __call__(self, x, out=None):
        """x: fp32 [N, H, W, Cin] channel view (or its Rows8), or [M, Cin] rows for a 1x1 stride-1 conv.  Returns
        [N, OH, OW, Cout] ([M, Cout]), written into the channel view `out` if given (which may lie on x)."""
        rows8 = isinstance(x, Rows8)
        _check(x.buffer if rows8 else x, "x", torch.int8 if rows8 else torch.float32)
        if self.codes.get_device() != (x.buffer if rows8 else x).get_device():
            raise ValueError(f"the weights are on {self.codes.device}, not on the current device "
                             f"(cuda:{_lib.current_device()})")
        ics = self.cin if rows8 else _rows(x, "x")[2]
        N, H, W, oshape = self._geometry(x.shape)
        y = _out(out, oshape, x.buffer.device if rows8 else x.device)
        rows, _, ocs = _rows(y, "out")
        if rows:
            lib = _lib.load()
            desc, one = self._desc(N, H, W, ics, ocs)
            tail = (self.codes.data_ptr(), self.scales.data_ptr(), None if self.bias is None else self.bias.data_ptr(),
                    self.relu, y.data_ptr(), _lib.raw_stream(y.get_device()))
            if rows8:
                fn = lib.tde_q8_deconv2d_bias_act if self.deconv else lib.tde_q8_conv2d_bias_act
                rc = fn(ctypes.byref(desc), *x.pointers(), *tail)
            else:
                fn = lib.tde_q8_deconv2d_f32_bias_act if self.deconv else lib.tde_q8_conv2d_f32_bias_act
                px, py = x.data_ptr(), y.data_ptr()
                apart = px + 4 * N * H * W * ics <= py or py + 4 * rows * ocs <= px
                if one and px % 16 == 0 and apart:      # (an output on the input: its rows are quantised first)
                    rc = fn(ctypes.byref(desc), px, None, None, *tail)
                else:
                    x8 = Rows8(x.shape, x.device)
                    rc = fn(ctypes.byref(desc), px, *x8.pointers(), *tail)
            _lib.check(rc, "Conv8")
        return y


# ---------------------------------------------------------------- 8-bit tape
class Tape8:
    """What the backward of one BatchNorm + ReLU keeps: codes [..., C] (int8), scales [..., ceil(C / 64)], the inverse
    standard deviations [groups, C] (and the means, when the forward made it)."""

    def __init__(self, codes, scales, invstd, mean=None):
        _check(codes, "codes", torch.int8)
        _check(scales, "scales")
        _check(invstd, "invstd")
        C = codes.shape[-1] if codes.dim() >= 2 else 0
        if C == 0 or C % 4 or C > 1024:
            raise ValueError(f"codes must be [..., C] with C a multiple of 4 up to 1024, got {tuple(codes.shape)}")
        if tuple(scales.shape) != tuple(codes.shape[:-1]) + ((C + BLOCK - 1) // BLOCK,):
            raise ValueError(f"scales {tuple(scales.shape)} do not fit codes {tuple(codes.shape)}")
        if invstd.dim() != 2 or invstd.shape[1] != C:
            raise ValueError(f"invstd must be [groups, {C}], got {tuple(invstd.shape)}")
        if not (codes.is_contiguous() and scales.is_contiguous() and invstd.is_contiguous()):
            raise ValueError("codes, scales and invstd must be contiguous")
        if any(t.data_ptr() % 16 for t in (codes, scales, invstd)):
            raise ValueError("codes, scales and invstd must start on 16 bytes")
        self.shape, self.C, self.rows, self.groups = codes.shape, C, _rows(codes, "codes")[0], invstd.shape[0]
        _check_groups(self.rows, self.groups)
        self._buffer, self._views = codes, (codes, scales, invstd, mean)
        self._ptrs = (codes.data_ptr(), scales.data_ptr(), invstd.data_ptr())

    @classmethod
    def _empty(cls, shape, C, rows, groups, device):
        """The tape of a forward, in one buffer of floats: codes, scales, invstd and mean behind one another, 16 bytes
        aligned."""
        t = cls.__new__(cls)
        t.shape, t.C, t.rows, t.groups = shape, C, rows, groups
        s = (rows * C + 15) // 16 * 4
        i = s + (rows * ((C + BLOCK - 1) // BLOCK) + 3) // 4 * 4
        m = i + groups * C
        t._buffer, t._views, t._at = torch.empty(m + groups * C, dtype=torch.float32, device=device), None, (s, i, m)
        p = t._buffer.data_ptr()
        t._ptrs, t._mean_ptr = (p, p + 4 * s, p + 4 * i), p + 4 * m
        return t

    @property
    def codes(self):
        if self._views is not None:
            return self._views[0]
        return self._buffer.view(torch.int8)[:self.rows * self.C].view(self.shape)

    @property
    def scales(self):
        if self._views is not None:
            return self._views[1]
        nb, s = (self.C + BLOCK - 1) // BLOCK, self._at[0]
        return self._buffer[s:s + self.rows * nb].view(self.shape[:-1] + (nb,))

    @property
    def invstd(self):
        if self._views is not None:
            return self._views[2]
        return self._buffer.as_strided((self.groups, self.C), (self.C, 1), self._at[1])

    @property
    def mean(self):
        if self._views is not None:
            return self._views[3]
        return self._buffer.as_strided((self.groups, self.C), (self.C, 1), self._at[2])

    def restore(self, relu=True, out=None):
        """The tape's values [..., C]: relu=True the layer's output as the consumers' filter gradients read it, relu=False
        the coded pre-activation."""
        _check(self._buffer, "tape", self._buffer.dtype)
        dev = self._buffer.device
        y = _out(out, self.shape, dev)
        rows, _, cs = _rows(y, "out")
        py = _check_view(y, cs, "out")
        if rows:
            codes, scales, _ = self._ptrs
            _lib.check(_lib.load().tde_tape8_restore(rows, self.C, codes, scales, bool(relu), py, cs, 0,
                                                     _lib.raw_stream(dev.index)), "Tape8.restore")
        return y


def _check_groups(rows, groups):
    if not 1 <= groups <= 8 or rows % groups:
        raise ValueError(f"{rows} rows are not {groups} equal groups (1 to 8)")


def _check_view(t, cs, name):
    """The view's pointer."""
    p = t.data_ptr()
    if p % 16 or cs % 4:
        raise ValueError(f"{name}: the channel view must start on 16 bytes with a pixel stride of a multiple of 4")
    return p


def _check_apart(pa, acs, pb, bcs, rows, C, what):
    """Two [rows, C] fp32 views at pa and pb with pixel strides acs and bcs are one and the same, or lie apart: a kernel that
    writes one while its other blocks read the other gives no defined result in between."""
    if pa == pb and acs == bcs:
        return
    if pa < pb + 4 * ((rows - 1) * bcs + C) and pb < pa + 4 * ((rows - 1) * acs + C):
        raise ValueError(f"{what} overlap: they must lie apart, or be the same view")


def _check_beta(C, beta):
    if C == 0 or C % 4 or C > 1024:
        raise ValueError(f"{C} channels: a multiple of 4 up to 1024 is expected")
    _check(beta, "beta")
    if beta.shape != (C,) or not beta.is_contiguous() or beta.data_ptr() % 16:
        raise ValueError(f"beta must be a contiguous ({C},) tensor that starts on 16 bytes")


@functools.lru_cache(maxsize=256)
def _workspace_bytes(rows, C, groups):
    lib = _lib.load()
    return 0 if lib.tde_tape8_one_launch(rows, C, groups) else lib.tde_tape8_workspace_size(rows, C)


def _workspace(rows, C, groups, device):
    """(keeper, pointer, bytes) of the call's workspace."""
    nb = _workspace_bytes(rows, C, groups)
    if nb == 0:
        return None, None, 0
    ws = torch.empty(nb, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), nb


def bn_relu_forward(z, beta, groups=1, eps=1e-3, decay=0.99, moving=None, bessel=True, out=None):
    """Training BatchNorm (scale=False) + ReLU of z [..., C] (contiguous) that keeps an 8-bit tape: returns (y, Tape8).

    The rows are `groups` equal consecutive groups, each normalised over its own rows.  moving: (moving_mean,
    moving_variance), updated in place in group order.  out: a channel view for y (16-byte aligned), z itself or apart from
    it."""
    _check(z, "z")
    shape, dev = z.shape, z.device
    C = shape[-1] if len(shape) >= 2 else 0
    _check_beta(C, beta)
    pz = z.data_ptr()
    if not z.is_contiguous() or pz % 16:
        raise ValueError("z must be a contiguous [..., C] tensor that starts on 16 bytes")
    rows = z.numel() // C
    if not 0 < rows <= MAX_ROWS:
        raise ValueError(f"z: {rows} rows: at most 2^30" if rows else "BatchNorm over no rows has no statistics")
    _check_groups(rows, groups)
    mm = mv = None
    if moving is not None:
        for t in moving:
            _check(t, "moving")
            if t.shape != (C,) or not t.is_contiguous():
                raise ValueError(f"moving statistics must be contiguous ({C},) tensors")
        mm, mv = (t.data_ptr() for t in moving)
    y = _out(out, shape, dev)
    _, _, cs = _rows(y, "out")
    py = _check_view(y, cs, "out")
    if out is not None:
        _check_apart(pz, C, py, cs, rows, C, "z and out")
    tape = Tape8._empty(shape, C, rows, groups, dev)
    codes, scales, invstd = tape._ptrs
    keep, ws, nb = _workspace(rows, C, groups, dev)
    _lib.check(_lib.load().tde_tape8_bn_fwd(rows, C, groups, pz, beta.data_ptr(), eps, decay, bool(bessel), mm,
                                            mv, tape._mean_ptr, invstd, py, cs, 0, codes, scales, ws, nb,
                                            _lib.raw_stream(dev.index)), "bn_relu_forward")
    return y, tape


def bn_relu_backward(tape, beta, dy, dz=None, dbeta=None):
    """(dz, dbeta) of the layer whose forward made `tape`, from the gradient dy [..., C] (channel view) of its output;
    beta as in that forward.  dz: a contiguous tensor to write, dy itself or apart from it; dbeta: a tensor to ADD to (a
    fresh one is written)."""
    if not isinstance(tape, Tape8):
        raise ValueError("tape must be a Tape8")
    _check(dy, "dy")
    _check(tape._buffer, "tape", tape._buffer.dtype)
    shape, dev, C = tape.shape, dy.device, tape.C
    _check_beta(C, beta)
    if dy.shape != shape:
        raise ValueError(f"dy must be {tuple(shape)}, got {tuple(dy.shape)}")
    rows, _, cs = _rows(dy, "dy")
    if rows == 0:
        raise ValueError("BatchNorm over no rows has no gradient")
    pdy = _check_view(dy, cs, "dy")
    given = dz is not None
    dz = _out(dz, shape, dev, "dz")
    pdz = dz.data_ptr()
    if not dz.is_contiguous() or pdz % 16:
        raise ValueError("dz must be contiguous and start on 16 bytes")
    if given:
        _check_apart(pdy, cs, pdz, C, rows, C, "dy and dz")
    acc = dbeta is not None
    dbeta = _out(dbeta, (C,), dev, "dbeta")
    if not dbeta.is_contiguous():
        raise ValueError("dbeta must be contiguous")
    keep, ws, nb = _workspace(rows, C, tape.groups, dev)
    codes, scales, invstd = tape._ptrs
    _lib.check(_lib.load().tde_tape8_bn_bwd(rows, C, tape.groups, codes, scales, invstd, beta.data_ptr(), pdy, cs,
                                            0, pdz, dbeta.data_ptr(), acc, None, ws, nb,
                                            _lib.raw_stream(dev.index)), "bn_relu_backward")
    return dz, dbeta


# ---------------------------------------------------------------- whole networks
# the open tape8() blocks of this thread (of this task), innermost last: (block, on)
_TAPE8 = contextvars.ContextVar("tape8", default=())


@contextlib.contextmanager
def tape8(on=True):
    """`with int8.tape8(): outs = disp_net(images)`: the reference-named network functions called inside keep their
    training tape in 8 bits (program.NetRun(tape8=True)); the backward may run outside.  It holds for the calls of the
    thread (asyncio: the task) that entered it; each block ends with itself, whatever order blocks are left in."""
    block = object()
    _TAPE8.set(_TAPE8.get() + ((block, bool(on)),))
    try:
        yield
    finally:
        _TAPE8.set(tuple(b for b in _TAPE8.get() if b[0] is not block))


def tape8_active():
    blocks = _TAPE8.get()
    return bool(blocks) and blocks[-1][1]

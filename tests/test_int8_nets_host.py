"""Host side of the 8-bit tape of whole networks: which buffers a run shares, what it holds, what it refuses."""
import types

import pytest
import torch

from tf_depth_estimation_amd import _netlib
from tf_depth_estimation_amd.program import ConvBN, Head, NetProgram, NetRun


def program(builder, *a, **kw):
    return NetProgram(builder(*a, **kw), types.SimpleNamespace(prefix="m"))


NETS = [(_netlib.disp_net_spec, (64, 96, 3), {}), (_netlib.depth_net_spec, (64, 96, 6), dict(levels=4)),
        (_netlib.depthflow_net_spec, (64, 96, 6), {})]


@pytest.mark.parametrize("builder,a,kw", NETS)
def test_runs_share_all_but_input_outputs_and_tape(builder, a, kw):
    prog = program(builder, *a, **kw)
    r1, r2 = NetRun(prog, 2, device="cpu", tape8=True), NetRun(prog, 2, device="cpu", tape8=True)
    fp32 = NetRun(prog, 2, device="cpu")
    for r in (r1, r2, fp32):
        r.ensure_grad()
    own = {prog.spec.input.name} | {v.buf.name for v in prog.spec.outputs} | {o.dst.buf.name for o in prog.spec.ops
                                                                               if isinstance(o, Head)}
    out = {v.buf.name for v in prog.spec.outputs}
    for b in prog.spec.bufs:
        assert (r1.act[b.name] is r2.act[b.name]) == (b.name not in own), b.name
        assert (r1.grad[b.name] is r2.grad[b.name]) == (b.name not in out), b.name
        assert r1.act[b.name].shape == fp32.act[b.name].shape
        if b.zero:
            assert not r1.act[b.name].any()
    for i, op in enumerate(prog.spec.ops):
        if isinstance(op, ConvBN):
            assert r1.z[i].data_ptr() == r2.z[i].data_ptr() and tuple(r1.z[i].shape) == op.zshape(2)
            codes, scales = r1.tape[i]
            assert codes.dtype == torch.int8 and tuple(codes.shape) == op.zshape(2)
            assert tuple(scales.shape) == op.zshape(2)[:3] + (-(-op.K // 64),)
            assert codes.data_ptr() != r2.tape[i][0].data_ptr()
    # one byte and a scale per 64 channels instead of z, y and the gradient buffers
    assert r1.held_bytes() < 0.2 * fp32.held_bytes()


def test_a_run_switches_without_moving_what_others_point_at():
    prog = program(_netlib.disp_net_spec, 64, 96, 3)
    r = NetRun(prog, 2, device="cpu")
    r.ensure_grad()
    before = (r.input_tensor().data_ptr(), [r.view_tensor(v).data_ptr() for v in prog.spec.outputs],
              [r.grad_tensor(v).data_ptr() for v in prog.spec.outputs])
    held = r.held_bytes()
    assert r.enable_tape8().enable_tape8() is r and r.tape8
    assert before == (r.input_tensor().data_ptr(), [r.view_tensor(v).data_ptr() for v in prog.spec.outputs],
                      [r.grad_tensor(v).data_ptr() for v in prog.spec.outputs])
    assert r.held_bytes() < 0.2 * held
    other = torch.zeros(2, 64, 96, 1)
    r.bind_output_grads([other])
    assert r.grad[prog.spec.outputs[0].buf.name] is other


def test_refusals():
    prog = program(_netlib.disp_net_spec, 64, 96, 3, bn=False)
    with pytest.raises(ValueError, match="BatchNorm"):
        NetRun(prog, 2, device="cpu", tape8=True)
    prog = program(_netlib.disp_net_spec, 64, 96, 3)
    r = NetRun(prog, 2, device="cpu", tape8=True)
    with pytest.raises(ValueError, match="forward first"):
        prog._backward(r, [None] * 4, False, None, True)
    with pytest.raises(ValueError, match="equal groups"):
        NetRun(prog, 3, device="cpu", groups=2, tape8=True)


def test_trainer_refuses_after_capture():
    from tf_depth_estimation_amd.train import Trainer
    t = Trainer()
    t.graphs = [object()]
    with pytest.raises(ValueError, match="before capture"):
        t.enable_tape8()

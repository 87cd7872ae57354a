"""The pair step with the 8-bit tape against the fp32 step run on the decoded tape, parameter by parameter: a lost, doubled or
stale term of any call or layer shows in its own parameters."""
import pytest
import torch

from tests.test_gpu_int8_nets import config4, fresh_store  # noqa: F401 (fresh_store: an autouse fixture)
from tf_depth_estimation_amd import int8
from tf_depth_estimation_amd.program import ConvBN

pytestmark = pytest.mark.gpu


def decode(r8, run):
    """The tape of r8 where the fp32 executor keeps its own: activations, pre-BN outputs, statistics."""
    prog = r8.prog
    prog._restore_tape8(r8)
    for name, t in r8.act.items():
        run.act[name].copy_(t)
    for i, op in enumerate(prog.spec.ops):
        if isinstance(op, ConvBN):
            K, G = op.K, r8.groups
            u = int8.Tape8(r8.tape[i][0], r8.tape[i][1], r8.stats[i][1].view(G, K)).restore(relu=False)
            mean, invstd = (r8.stats[i][j].double().view(G, 1, K) for j in (0, 1))
            xh = (u.double() - prog.P(f"{op.layer}/BatchNorm/beta").double()).view(G, -1, K)
            run.z[i].copy_((xh / invstd + mean).view(run.z[i].shape))
            run.stats[i].copy_(r8.stats[i])


@pytest.mark.parametrize("twin", [True, False])
@pytest.mark.parametrize("overlap", [False, True])
def test_step_parameter_by_parameter(twin, overlap):
    B, H, W = 2, 64, 96
    tr = config4(B, H, W, twin).enable_tape8()
    tr.enable_deterministic()
    if overlap:
        tr.enable_wgrad_overlap()
        tr.enable_net_overlap()
    tr.phase_compute()
    torch.cuda.synchronize()

    ref = config4(B, H, W, twin)
    ref.enable_deterministic()
    pair = {id(ref.runs[k]): tr.runs[k] for k in ref.runs}
    for prog in (ref.single, ref.pair):
        fwd, bwd = prog.forward, prog.backward

        def forward(run, *a, fwd=fwd, **kw):
            outs = fwd(run, *a, **kw)
            for v in run.prog.spec.outputs:          # the same outputs, so the same gradients of the losses
                run.view_tensor(v).copy_(pair[id(run)].view_tensor(v))
            return outs

        def backward(run, *a, bwd=bwd, **kw):
            decode(pair[id(run)], run)
            return bwd(run, *a, **kw)

        prog.forward, prog.backward = forward, backward
    ref.phase_compute()
    torch.cuda.synchronize()
    # Both backwards evaluate the same formulas on the same numbers in fp32: about 30 layers, each off by some 10 roundings of
    # 2^-24 and a product of 2^-20 of the sum of its terms, which is some 20 times the sum: 1e-3 of a parameter's gradient, and
    # of the whole for those that cancel further.
    worst = 0.0
    for c8, c in zip(tr.chunks, ref.chunks):
        whole = float(c.grad.norm())
        assert whole > 0
        for name in c.offsets:
            g8, g = c8.grad_view(name), c.grad_view(name)
            err, bar = float((g8 - g).norm()), 1e-3 * float(g.norm()) + 1e-5 * whole
            worst = max(worst, err / bar)
            assert err <= bar, (name, err, float(g.norm()), whole)
    print("worst share of the bar", worst)

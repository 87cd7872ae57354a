"""Whole networks on the 8-bit operators: training steps with the 8-bit tape and 8-bit prediction."""
import numpy as np
import pytest
import torch

from tests import int8_oracle as O
from tests.test_gpu_trainers import intrinsics, small_pose, texture
from tf_depth_estimation_amd import _api, _netlib, int8, variables
from tf_depth_estimation_amd.program import ConvBN, NetRun, Resize

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def fresh_store():
    variables.get_store().reset(seed=1)
    _api.clear_programs()
    yield
    variables.get_store().reset(seed=1)
    _api.clear_programs()


def get(builder, H, W, cin, scope="model", **kw):
    with variables.variable_scope(scope):
        return _api.get_program("net", builder, H, W, cin, **kw)


def images(N, H, W, C, seed):
    return torch.randn(N, H, W, C, generator=torch.Generator().manual_seed(seed)).mul_(0.3).cuda()


def out_grads(prog, N, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(N, v.H, v.W, v.C, generator=g).cuda() for v in prog.spec.outputs]


NETS = [(_netlib.disp_net_spec, 3, {}, 1), (_netlib.disp_net_spec, 3, {}, 2), (_netlib.depth_net_spec, 6, dict(levels=4), 2),
        (_netlib.depthflow_net_spec, 6, {}, 1)]


@pytest.mark.parametrize("builder,cin,kw,groups", NETS)
def test_tape8_network(builder, cin, kw, groups):
    """Outputs equal the fp32 tape's; the backward equals the fp32 executor's run on the decoded tape (z, statistics and
    activations replaced by the tape's values): the same formulas on the same numbers."""
    N, H, W = 2, 64, 96
    prog = get(builder, H, W, cin, **kw)
    x, gs = images(N, H, W, cin, 1), out_grads(prog, N, 2)
    r8, r32 = NetRun(prog, N, groups=groups, tape8=True), NetRun(prog, N, groups=groups)
    o32 = [t.clone() for t in prog.forward(r32, x)]
    o8 = [t.clone() for t in prog.forward(r8, x)]
    for a, b in zip(o8, o32):
        assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max())
    prog.chunk.grad.zero_()
    prog.backward(r8, gs)
    g8 = prog.chunk.grad.clone()
    # the decoded tape, put where the fp32 executor keeps its own
    prog._restore_tape8(r8)
    for name, t in r8.act.items():
        r32.act[name].copy_(t)
    for i, op in enumerate(prog.spec.ops):
        if isinstance(op, ConvBN):
            K = op.K
            u = int8.Tape8(r8.tape[i][0], r8.tape[i][1], r8.stats[i][1].view(groups, K)).restore(relu=False)
            mean, invstd = (r8.stats[i][j].double().view(groups, 1, K) for j in (0, 1))
            xh = (u.double() - prog.P(f"{op.layer}/BatchNorm/beta").double()).view(groups, -1, K)
            r32.z[i].copy_((xh / invstd + mean).view(r32.z[i].shape))
            r32.stats[i].copy_(r8.stats[i])
    prog.chunk.grad.zero_()
    prog.backward(r32, gs)
    g32 = prog.chunk.grad
    # the whole-gradient bar of the fp32 step tests (tests/test_gpu_trainers.py)
    assert float((g8 - g32).norm()) <= 1e-3 * float(g32.norm())


def test_tape8_runs_take_turns():
    """Two runs of one program, forward A, forward B, backward A, backward B, against each alone: bit for bit."""
    N, H, W = 2, 64, 96
    prog = get(_netlib.disp_net_spec, H, W, 3)
    xs, gs = [images(N, H, W, 3, s) for s in (3, 4)], [out_grads(prog, N, s) for s in (5, 6)]
    alone = []
    for x, g in zip(xs, gs):
        r = NetRun(prog, N, tape8=True)
        outs = [t.clone() for t in prog.forward(r, x)]
        prog.chunk.grad.zero_()
        dx = prog.backward(r, g, need_input_grad=True)
        alone.append((outs, prog.chunk.grad.clone(), dx.clone()))
    runs = [NetRun(prog, N, tape8=True) for _ in xs]
    outs = [prog.forward(r, x) for r, x in zip(runs, xs)]
    for r, g, o, (ref, gref, dref) in zip(runs, gs, outs, alone):
        for a, b in zip(o, ref):
            assert torch.equal(a, b)
        prog.chunk.grad.zero_()
        dx = prog.backward(r, g, need_input_grad=True)
        assert torch.equal(prog.chunk.grad, gref) and torch.equal(dx, dref)
        prog.chunk.grad.zero_()
        prog.backward(r, g)                  # a second backward of the same forward: the tape is still whole
        assert torch.equal(prog.chunk.grad, gref)


@pytest.mark.parametrize("groups", [1, 2])
def test_tape8_sync_bn(groups):
    """SyncBN over two replicas that hold the same batch (the all-reduce doubles the sums): the statistics, outputs and
    gradients of one replica alone."""
    N, H, W = 2, 64, 96
    prog = get(_netlib.disp_net_spec, H, W, 3)
    x, gs = images(N, H, W, 3, 8), out_grads(prog, N, 9)
    run = NetRun(prog, N, groups=groups, tape8=True)
    ref = [t.clone() for t in prog.forward(run, x)]
    prog.chunk.grad.zero_()
    prog.backward(run, gs)
    gref = prog.chunk.grad.clone()
    calls = []

    def sync(t):
        calls.append(t.numel())
        t.mul_(2)
    prog.bn_sync, prog.bn_world = sync, 2
    try:
        outs = [t.clone() for t in prog.forward(run, x)]
        prog.chunk.grad.zero_()
        prog.backward(run, gs)
    finally:
        prog.bn_sync, prog.bn_world = None, 1
    layers = sum(isinstance(op, ConvBN) for op in prog.spec.ops)
    assert len(calls) == 2 * layers
    for a, b in zip(outs, ref):
        assert torch.equal(a, b)          # sums and rows doubled: the same quotients
    # the few-row layers' backward sums run in another order (fp64); the whole-gradient bar of the step tests
    assert float((prog.chunk.grad - gref).norm()) <= 1e-3 * float(gref.norm())


def test_tape8_through_autograd():
    from tf_depth_estimation_amd import nets_optflow_depth as nd
    x = images(2, 64, 96, 3, 7)
    with variables.variable_scope("model"):
        with int8.tape8():
            outs, _ = nd.disp_net(x, True)
    loss = sum((o * o).mean() for o in outs)
    prog = next(iter(_api._PROGRAMS.values()))
    prog.chunk.grad.zero_()
    loss.backward()
    g = prog.chunk.grad.clone()
    run = NetRun(prog, 2, tape8=True)
    o2 = prog.forward(run, x)
    prog.chunk.grad.zero_()
    prog.backward(run, [2 * o / o.numel() for o in o2])
    assert float(g.norm()) > 0 and float((g - prog.chunk.grad).norm()) <= 1e-3 * float(g.norm())


def config4(B, H, W, twin=True):
    from tf_depth_estimation_amd import train
    variables.get_store().reset(seed=1)
    _api.clear_programs()
    tr = train.DepthThenCamTrainer(B, H, W, twin=twin)
    lab = torch.from_numpy(np.random.default_rng(5).uniform(0.25, 4.0, (B, H, W, 1)).astype(np.float32))
    tr.set_batch(texture(B, H, W, 1), texture(B, H, W, 2), lab, intrinsics(B, H, W), small_pose(B, 3))
    return tr


@pytest.mark.parametrize("twin", [True, False])
def test_tape8_training_step(twin):
    """The config-4 step: losses as with the fp32 tape, gradients as that step's up to the coding, less memory held;
    captured with both overlaps, replayed several times: the eager serial steps' parameters bit for bit (the warp loss
    in its deterministic mode)."""
    B, H, W = 2, 64, 96
    ref = config4(B, H, W, twin)
    ref.enable_deterministic()
    ref.phase_compute()
    losses = ref.loss_parts()
    grads = [c.grad.clone() for c in ref.chunks]
    held = sum(r.held_bytes() for r in ref.runs.values())

    tr = config4(B, H, W, twin).enable_tape8()
    tr.enable_deterministic()
    tr.phase_compute()
    for k, v in losses.items():
        assert abs(tr.loss_parts()[k] - v) <= 1e-4 * abs(v) + 1e-7, k
    for c, g in zip(tr.chunks, grads):
        # coded activations: a step of 1/128 of a block's largest value, uniform, so about 1 % of the gradient; far
        # from a lost or doubled term
        assert float((c.grad - g).norm()) <= 0.3 * float(g.norm())
    assert sum(r.held_bytes() for r in tr.runs.values()) < 0.25 * held

    eager = config4(B, H, W, twin).enable_tape8()
    eager.enable_deterministic()
    eager.enable_wgrad_overlap(serial=True)
    graph = config4(B, H, W, twin).enable_tape8()
    graph.enable_deterministic()
    graph.enable_wgrad_overlap()
    graph.enable_net_overlap()
    graph.capture(warmup=2)
    params = None
    for _ in range(2):
        eager.step_eager()
    for i in range(3):
        eager.step_eager()
        graph.step()
        torch.cuda.synchronize()
    # (both trainers follow the same variables' initial values: separate stores, five steps each)
    for a, b in zip(eager.chunks, graph.chunks):
        assert torch.equal(a.flat, b.flat) and torch.equal(a.bn, b.bn)


@pytest.mark.parametrize("net,kw", [("disp_net", {}), ("depthflow_net", {}), ("depth_net", {}), ("depth_net", dict(cin=11))])
def test_int8_predictor(net, kw):
    """Every layer of the 8-bit Predictor against the definition on the activations it read; the captured graph equals
    the eager calls."""
    from tf_depth_estimation_amd.batch_prediction import Predictor
    H, W, N = 64, 64, 1
    pred = Predictor(net, H, W, batch=N, graph=False, int8=True, **kw)
    st = pred.prog.chunk
    r = np.random.default_rng(11)
    for name, (o, c) in st.bn_offsets.items():
        m, v = st.moving(name)
        m.copy_(torch.from_numpy(r.normal(0, 0.1, c).astype(np.float32)))
        v.copy_(torch.from_numpy(r.uniform(0.5, 1.5, c).astype(np.float32)))
    pred.refresh()
    x = images(N, H, W, pred.x.shape[3], 12)
    outs = [t.clone() for t in pred(x)]
    assert all(bool(torch.isfinite(t).all()) for t in outs)
    for op in pred.prog.spec.ops:
        if not isinstance(op, ConvBN):
            continue
        src = pred.run.view_tensor(op.src)[..., :op.src.creal].cpu().numpy()
        got = pred.run.view_tensor(op.dst).cpu().numpy()
        w, b, _ = pred.prog._folded[op.layer]
        y, mag = O.conv8(src, w.cpu().numpy(), b.cpu().numpy(), op.s, op.deconv, True)
        # rounding of the fp32 sum over taps (tests/test_gpu_int8.py, conv_bound)
        assert (np.abs(got - y) <= (op.k * op.k + 38) * 2.0 ** -24 * mag + 1e-37).all(), op.layer
    graph = Predictor(net, H, W, batch=N, int8=True, **kw)
    for i in range(3):
        for a, c in zip(graph(x), outs):
            assert torch.equal(a, c)
        pred(images(N, H, W, pred.x.shape[3], 20 + i))
        graph(images(N, H, W, pred.x.shape[3], 30 + i))


def test_int8_predictor_refuses_unfolded():
    from tf_depth_estimation_amd.batch_prediction import Predictor
    with pytest.raises(ValueError, match="fold_bn"):
        Predictor("disp_net", 64, 64, fold_bn=False, int8=True)

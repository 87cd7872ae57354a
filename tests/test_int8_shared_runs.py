"""What runs of one program with the 8-bit tape hand out does not lie in the buffers they share."""
import types
import weakref

import pytest
import torch

from tf_depth_estimation_amd import _api, _netlib, int8, variables
from tf_depth_estimation_amd.program import NetProgram, NetRun


@pytest.mark.parametrize("cin", [3, 4, 8])
def test_input_gradients_are_their_own(cin):
    prog = NetProgram(_netlib.disp_net_spec(64, 96, cin), types.SimpleNamespace(prefix="m"))
    runs = [NetRun(prog, 2, device="cpu", tape8=True) for _ in range(2)]
    got = []
    for i, r in enumerate(runs):
        r.ensure_grad()
        r.view_tensor(prog.spec.input_view, True).fill_(i + 1)       # what a backward leaves
        got.append(r.input_grad())
    for i, g in enumerate(got):
        assert tuple(g.shape) == (2, 64, 96, cin) and g.is_contiguous() and bool((g == i + 1).all())


def test_a_switched_run_gives_its_buffers_back_first(monkeypatch):
    """enable_tape8 makes the shared set when the run holds no more of its fp32 buffers than those that stay."""
    prog = NetProgram(_netlib.disp_net_spec(64, 96, 3), types.SimpleNamespace(prefix="m"))
    run = NetRun(prog, 2, device="cpu")
    run.ensure_grad()
    stays = prog.own_buffers()
    outs = {v.buf.name for v in prog.spec.outputs}
    gone = [weakref.ref(t) for n, t in run.act.items() if n not in stays] + [weakref.ref(t) for t in run.z.values()]
    gone += [weakref.ref(t) for n, t in run.grad.items() if n not in outs]
    before = sum(r() is not None for r in gone)
    seen = []
    make = NetProgram.shared_tape8

    def shared(self, *a):
        seen.append(sum(r() is not None for r in gone))
        return make(self, *a)

    monkeypatch.setattr(NetProgram, "shared_tape8", shared)
    run.enable_tape8()
    assert before == len(gone) > 20 and seen[0] == 0


@pytest.fixture()
def fresh_store():
    variables.get_store().reset(seed=1)
    _api.clear_programs()
    yield
    variables.get_store().reset(seed=1)
    _api.clear_programs()


@pytest.mark.gpu
@pytest.mark.parametrize("cin", [3, 4])
def test_input_gradients_through_autograd(cin, fresh_store):
    """Two calls of one network under int8.tape8(): each input's gradient is that of the call alone, one input of both calls
    gets their sum, and a gradient autograd took over keeps its values."""
    from tf_depth_estimation_amd import nets_optflow_depth as nd

    def image(seed):
        return torch.randn(2, 64, 96, cin, generator=torch.Generator().manual_seed(seed)).mul_(0.3).cuda()

    def loss(x):
        with variables.variable_scope("model"), int8.tape8():
            return sum((o * o).mean() for o in nd.disp_net(x, True)[0])

    alone = []
    for s in (1, 2):
        x = image(s).requires_grad_()
        loss(x).backward()
        alone.append(x.grad.clone())
    assert all(bool(torch.isfinite(g).all()) and float(g.abs().max()) > 0 for g in alone)
    xs = [image(s).requires_grad_() for s in (1, 2)]
    (loss(xs[0]) + loss(xs[1])).backward()
    for x, g in zip(xs, alone):
        assert torch.equal(x.grad, g)
    x = image(1).requires_grad_()
    (loss(x) + loss(x)).backward()
    assert torch.equal(x.grad, alone[0] + alone[0])
    kept = xs[0].grad
    loss(image(3).requires_grad_()).backward()
    assert torch.equal(kept, alone[0])


@pytest.mark.gpu
def test_the_first_run_is_made_before_a_capture(fresh_store):
    """The shared buffers are refused under capture; with them there, a run made, stepped forward and back inside a capture
    replays as the eager run between whose steps it is replayed."""
    N, H, W = 2, 64, 96
    with variables.variable_scope("model"):
        prog = _api.get_program("depth_net", _netlib.disp_net_spec, H, W, 3)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(N, H, W, 3, generator=g).mul_(0.3).cuda()
    gs = [torch.randn(N, v.H, v.W, v.C, generator=g).cuda() for v in prog.spec.outputs]
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            NetRun(prog, N, tape8=True)
    eager = NetRun(prog, N, tape8=True)

    def step(run):
        outs = prog.forward(run, x)
        return outs + [prog.backward(run, gs, need_input_grad=True, grad_accumulate=False)]

    step(eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(NetRun(prog, N, tape8=True))
    for i in range(3):
        x.copy_(torch.randn(x.shape, generator=g).mul_(0.3))
        outs = prog.forward(eager, x)
        graph.replay()                                   # the shared buffers are another run's now
        torch.cuda.synchronize()
        replayed, pgrad = [t.clone() for t in captured], prog.chunk.grad.clone()
        dx = prog.backward(eager, gs, need_input_grad=True, grad_accumulate=False)
        for a, b in zip(replayed, outs + [dx]):
            assert torch.equal(a, b), i
        assert torch.equal(pgrad, prog.chunk.grad), i


@pytest.mark.gpu
@pytest.mark.parametrize("cin", [3, 4])
@pytest.mark.parametrize("tape", [False, True])
def test_two_backwards_of_one_call(cin, tape, fresh_store):
    """retain_graph: the second backward adds to the gradient autograd took over from the first."""
    from tf_depth_estimation_amd import nets_optflow_depth as nd
    x = torch.randn(2, 64, 96, cin, generator=torch.Generator().manual_seed(1)).mul_(0.3).cuda().requires_grad_()
    with variables.variable_scope("model"), int8.tape8(tape):
        outs = nd.disp_net(x, True)[0]
    losses = [(outs[0] * outs[0]).mean(), 5 * outs[0].mean()]
    apart = [torch.autograd.grad(v, x, retain_graph=True)[0].clone() for v in losses]
    assert not torch.equal(*apart)
    for v in losses:
        v.backward(retain_graph=True)
    assert torch.equal(x.grad, apart[0] + apart[1])


def test_a_refused_switch_leaves_the_run_whole(monkeypatch):
    """enable_tape8 inside a capture, or of a network without BatchNorm: the fp32 run keeps every buffer."""
    prog = NetProgram(_netlib.disp_net_spec(64, 96, 3), types.SimpleNamespace(prefix="m"))
    run = NetRun(prog, 2, device="cpu")
    run.ensure_grad()
    before = [dict(d) for d in (run.act, run.z, run.grad)]

    def capturing(self, N, device):
        raise ValueError("before the capture")

    monkeypatch.setattr(NetProgram, "check_tape8_capture", capturing, raising=False)
    monkeypatch.setattr(NetProgram, "shared_tape8", capturing)
    with pytest.raises(ValueError, match="before the capture"):
        run.enable_tape8()
    assert not run.tape8
    for was, now in zip(before, (run.act, run.z, run.grad)):
        assert now is not None and all(now[k] is t for k, t in was.items())

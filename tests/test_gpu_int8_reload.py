"""Conv8's weights: loaded under a captured graph, and given back."""
import gc
import weakref

import pytest
import torch

from tf_depth_estimation_amd import int8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,deconv,stride,x", [((3, 3, 40, 24), False, 1, (2, 9, 11, 40)), ((1, 1, 64, 20), False, 1, (7, 64)),
                                                   ((3, 3, 16, 40), True, 2, (2, 5, 6, 40))])
def test_load_reaches_a_captured_graph(shape, deconv, stride, x):
    """Weights and bias of the same shape are loaded in place: a graph captured before replays with them, as the eager call,
    also when memory has been freed and given out again in between."""
    g = torch.Generator().manual_seed(3)

    def new(*s):
        return torch.randn(s, generator=g).cuda()

    K = shape[2] if deconv else shape[3]
    xb = new(*x)
    conv = int8.Conv8(new(*shape), new(K), stride=stride, deconv=deconv, relu=False)
    conv(xb)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = conv(xb)
    for i in range(3):
        w, b = new(*shape), new(K)
        conv.load(w, b)
        filler = [torch.full((n,), 77, dtype=torch.int8, device="cuda") for n in (256, 1024, 4096, 16384) for _ in range(4)]
        want = int8.Conv8(w, b, stride=stride, deconv=deconv, relu=False)(xb)
        assert torch.equal(conv(xb), want)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), i
        del filler
    # another shape, and a bias that comes and goes, still load
    conv.load(w, None)
    assert torch.equal(conv(xb), int8.Conv8(w, None, stride=stride, deconv=deconv, relu=False)(xb))
    conv.load(w, b)
    assert torch.equal(conv(xb), want)
    w2 = torch.cat([w, w], dim=2 if deconv else 3)
    conv.load(w2, torch.cat([b, b]))
    assert torch.equal(conv(xb), torch.cat([want, want], dim=-1))


def test_weights_are_given_back_with_the_layer():
    """Without a garbage collection."""
    gc.collect()
    gc.disable()
    try:
        conv = int8.Conv8(torch.ones(1, 1, 8, 4, device="cuda"))
        conv(torch.ones(5, 8, device="cuda"))
        codes = weakref.ref(conv.codes)
        del conv
        assert codes() is None
    finally:
        gc.enable()


def test_load_in_and_out_of_inference_mode():
    w, x = torch.randn(1, 1, 8, 4, device="cuda"), torch.randn(5, 8, device="cuda")
    with torch.inference_mode():
        conv = int8.Conv8(w, torch.zeros(4, device="cuda"), relu=False)
        y = conv(x)
    conv.load(w, torch.ones(4, device="cuda"))
    assert torch.equal(conv(x), int8.Conv8(w, torch.ones(4, device="cuda"), relu=False)(x))
    with torch.inference_mode():
        conv.load(w, torch.zeros(4, device="cuda"))
        assert torch.equal(conv(x), y)
    other = int8.Conv8(w, torch.ones(4, device="cuda"), relu=False)
    with torch.inference_mode():
        other.load(w, torch.zeros(4, device="cuda"))
    assert torch.equal(other(x), y)

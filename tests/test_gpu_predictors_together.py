"""Predictors of one network side by side: the graph of each reads its own folded weights."""
import pytest
import torch

from tests.test_gpu_int8_nets import fresh_store, images  # noqa: F401 (fresh_store: an autouse fixture)
from tf_depth_estimation_amd.batch_prediction import Predictor

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("other", [dict(int8=True), dict(batch=2), dict(graph=False)])
def test_a_second_predictor_leaves_the_first_its_weights(other):
    H, W = 64, 64
    first = Predictor("disp_net", H, W)
    x = images(1, H, W, 3, 1)
    want = [t.clone() for t in first(x)]
    torch.cuda.synchronize()
    second = Predictor("disp_net", H, W, **other)
    # memory that the first may have lost is given out and filled
    filler = [torch.full((n,), 1e3, device="cuda") for n in (1 << 10, 1 << 14, 1 << 18, 1 << 20, 9 * 512 * 512) for _ in range(12)]
    torch.cuda.synchronize()
    for _ in range(2):
        for a, b in zip(first(x), want):
            assert torch.equal(a, b)
        second(images(other.get("batch", 1), H, W, 3, 2))
    del filler

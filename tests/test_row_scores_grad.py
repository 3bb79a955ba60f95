"""Row scores have no backward forms: a tensor that requires a gradient is refused, not answered with
a result that has lost it."""
import pytest
import torch

from m3_memory_b200 import cabi, row_scores as R


@pytest.fixture(scope="module")
def eng():
    return cabi.Engine()


def calls(eng, t):
    return [lambda: R.pack_rows(eng, t), lambda: R.row_scores(eng, t, t),
            lambda: R.list_scores(eng, t, t, None, None, None, None, None),
            lambda: R.score_probs(eng, t)]


@pytest.mark.parametrize("i", range(4))
def test_tensors_that_require_a_gradient_are_refused(eng, i):
    leaf = torch.zeros(4, 16, dtype=torch.bfloat16, requires_grad=True)
    for t in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="gradient"):
            calls(eng, t)[i]()
    # refused as a CPU tensor only, where no gradient is asked for
    with pytest.raises(ValueError, match="CUDA"):
        calls(eng, leaf.detach())[i]()
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        calls(eng, leaf)[i]()


@pytest.mark.gpu
def test_each_tensor_of_a_call(eng):
    x = torch.randn(8, 64, device="cuda").bfloat16()
    w = x.clone().requires_grad_()
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    pair = torch.tensor([0, 1], device="cuda")
    length = torch.tensor([8], dtype=torch.int32, device="cuda")
    out = torch.zeros(8, 8, device="cuda", requires_grad=True)
    vec = torch.zeros(8, device="cuda", requires_grad=True)
    for call in (lambda: R.row_scores(eng, w, x), lambda: R.row_scores(eng, x, w),
                 lambda: R.row_scores(eng, x, x, out=out),
                 lambda: R.list_scores(eng, w, x, zero, length, pair, zero, vec.detach()),
                 lambda: R.list_scores(eng, x, x, zero, length, pair, zero, vec)):
        with pytest.raises(ValueError, match="gradient"):
            call()
    with torch.no_grad():
        R.row_scores(eng, w, w, out=out)
    want = R.row_scores(eng, x, x)
    assert torch.equal(out.detach(), want)
    eng.sync_errors()

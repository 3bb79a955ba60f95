"""Row scores at the limits of what a call may be given."""
import pytest
import torch

from m3_memory_b200 import cabi
from test_gpu_row_scores import make_rows, scores_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def R(cuda_ok):
    from m3_memory_b200 import row_scores

    return row_scores


@pytest.fixture(scope="module")
def eng(cuda_ok):
    return cabi.Engine()


def T(a, dtype=torch.int64):
    return torch.tensor(a, dtype=dtype, device="cuda")


# ---------------- pairs and outputs that end past their arrays ----------------


@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
@pytest.mark.parametrize("npair", [7, 40, 300])
def test_more_pairs_than_queries_without_pair_row(R, eng, kind, npair):
    """Pair p without pair_row is row p of q: those past the last row are left out and reported,
    and nothing of q (codes, scales) is read there."""
    nq, n, dim = 5, 300, 256
    q, qv = make_rows(R, eng, kind, nq, dim, 1)
    x, xv = make_rows(R, eng, kind, n, dim, 2)
    length = 40
    out = torch.full((npair * length,), 7.0, device="cuda")
    R.list_scores(eng, q, x, T([100]), T([length], torch.int32), T([0, npair]),
                  torch.arange(npair, device="cuda") * length, out)
    with pytest.raises(IndexError):
        eng.sync_errors()
    ref, tol = scores_ref(qv, xv[100:100 + length], 1.0, 0.0, torch.float32, dim)
    got = out.view(npair, length)
    assert ((got[:nq].double() - ref).abs() <= tol).all()
    assert (got[nq:] == 7.0).all()

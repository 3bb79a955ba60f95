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


# ---------------- wide strides ----------------


def spread(p, dim, codes_ld, scales_ld):
    """The same packed rows with other row strides."""
    n = p.codes.shape[0]
    codes = torch.empty(n, codes_ld, dtype=torch.uint8, device="cuda")[:, :p.codes.shape[1]]
    scales = torch.empty(n, scales_ld, dtype=torch.uint8, device="cuda")[:, :p.scales.shape[1]]
    codes.copy_(p.codes)
    scales.copy_(p.scales)
    return type(p)(codes, scales, dim)


@pytest.mark.parametrize("n,dim,scales_ld", [(130, 600, 1 << 24), (1000, 640, 1 << 18),
                                             (300, 520, 132), (257, 17000, 256)])
def test_scales_far_apart(R, eng, n, dim, scales_ld):
    """Scale bytes that are a small part of wider records: only they are touched, and the records'
    size costs nothing (walking all of 130 x 16 MB would outlast the waits' limit)."""
    x = R.pack_rows(eng, torch.randn(n, dim, device="cuda"))
    q = R.pack_rows(eng, torch.randn(20, dim, device="cuda"))
    want = R.row_scores(eng, q, x)
    wide = spread(x, dim, -(-dim // 16) * 16 + 16, scales_ld)
    assert torch.equal(R.row_scores(eng, q, wide), want)
    assert torch.equal(R.row_scores(eng, spread(q, dim, -(-dim // 16) * 16, scales_ld), x), want)
    out = torch.empty(20 * n, device="cuda")
    R.list_scores(eng, q, wide, T([0]), T([n], torch.int32), T([0, 20]),
                  torch.arange(20, device="cuda") * n, out)
    assert torch.equal(out.view(20, n), want)
    eng.sync_errors()


def test_codes_and_scales_in_one_record(R, eng):
    """Records of a row's codes and its scales behind them, the last row's scales at the end."""
    n, dim = 300, 1024
    p = R.pack_rows(eng, torch.randn(n, dim, device="cuda"))
    rec = torch.empty(n, dim + 16, dtype=torch.uint8, device="cuda")
    rec[:, :dim], rec[:, dim:dim + 8] = p.codes, p.scales
    x = R.PackedRows(rec[:, :dim], rec[:, dim:dim + 8], dim)
    for nq in (1, 100):
        q = R.pack_rows(eng, torch.randn(nq, dim, device="cuda"))
        assert torch.equal(R.row_scores(eng, q, x), R.row_scores(eng, q, p))
    eng.sync_errors()

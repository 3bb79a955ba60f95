"""Row scores on a CPU-only box: every refusal fires before any device work (the pointers below are
never read), and the torch form checks its tensors."""
import ctypes as ct

import pytest
import torch

from m3_memory_b200 import cabi

P = 1 << 20  # an aligned address that is not memory
UNSUPPORTED = cabi.M3G_EUNSUPPORTED


def rows(**kw):
    v = dict(data=P, scales=P, n=8, ld=256, ld_scales=4, dim=200, dtype=cabi.E4M3)
    v.update(kw)
    return cabi.Rows(**v)


@pytest.fixture(scope="module")
def eng():
    return cabi.Engine()


BAD_ROWS = [dict(dtype=cabi.F32), dict(dtype=7), dict(n=-1), dict(dim=0), dict(dim=-3),
            dict(ld=199), dict(ld=200), dict(ld=1 << 40), dict(data=None), dict(data=P + 8),
            dict(ld_scales=1), dict(ld_scales=3), dict(ld_scales=0), dict(scales=None),
            dict(scales=P + 2), dict(dtype=cabi.BF16, ld=204)]


@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
@pytest.mark.parametrize("side", ["q", "x"])
def test_rows_refused(eng, bad, side):
    q, x = (rows(**bad), rows()) if side == "q" else (rows(), rows(**bad))
    if bad.get("dtype") == cabi.BF16:
        q, x = (q, rows(dtype=cabi.BF16)) if side == "q" else (rows(dtype=cabi.BF16), x)
    with pytest.raises(ValueError):
        eng.row_scores_device(q, x, 1.0, 0.0, P, cabi.F32, 8)
    with pytest.raises(ValueError):
        eng.list_scores_device(q, x, 1, P, P, P, 1, P, P, 1.0, 0.0, P, cabi.F32, 8)


@pytest.mark.parametrize("big", [dict(n=1 << 31), dict(dim=(1 << 20) + 1, ld=1 << 21,
                                                       ld_scales=1 << 16)])
def test_too_many_rows_or_dims_unsupported(eng, big):
    with pytest.raises(cabi.M3GError) as ei:
        eng.row_scores_device(rows(), rows(**big), 1.0, 0.0, P, cabi.F32, 1 << 31)
    assert ei.value.code == UNSUPPORTED


@pytest.mark.parametrize("case", [
    dict(x=dict(dim=128)), dict(x=dict(dtype=cabi.BF16)), dict(out_dtype=cabi.E4M3),
    dict(ld_out=7), dict(alpha=float("nan")), dict(beta=float("inf")), dict(out=None),
    dict(out=P + 2)], ids=str)
def test_row_scores_refused(eng, case):
    with pytest.raises(ValueError):
        eng.row_scores_device(rows(), rows(**case.get("x", {})), case.get("alpha", 1.0),
                              case.get("beta", 0.0), case.get("out", P),
                              case.get("out_dtype", cabi.F32), case.get("ld_out", 8))


def test_null_rows_and_null_engine(eng):
    L = cabi.lib()
    assert L.m3g_row_scores_device(eng.h, None, ct.byref(rows()), 1.0, 0.0, P, 0, 8,
                                   None) == cabi.M3G_EINVAL
    assert L.m3g_row_scores_device(None, ct.byref(rows()), ct.byref(rows()), 1.0, 0.0, P, 0, 8,
                                   None) == cabi.M3G_EINVAL
    assert L.m3g_pack_rows_device(eng.h, P, 0, 8, 200, 200, None, None) == cabi.M3G_EINVAL
    assert L.m3g_score_probs_work(eng.h, 1, 1, 0, 0, 0, None) == cabi.M3G_EINVAL


@pytest.mark.parametrize("case", [
    dict(ngroup=-1), dict(npair=-1), dict(out_n=-1), dict(list_off=None), dict(list_len=None),
    dict(pair_off=None), dict(out_off=None), dict(list_off=P + 4), dict(list_len=P + 2),
    dict(pair_row=P + 2), dict(out_off=P + 4), dict(out=None)], ids=str)
def test_list_scores_refused(eng, case):
    v = dict(ngroup=2, list_off=P, list_len=P, pair_off=P, npair=3, pair_row=P, out_off=P, out=P,
             out_n=64)
    v.update(case)
    with pytest.raises(ValueError):
        eng.list_scores_device(rows(), rows(), v["ngroup"], v["list_off"], v["list_len"],
                               v["pair_off"], v["npair"], v["pair_row"], v["out_off"], 1.0, 0.0,
                               v["out"], cabi.F32, v["out_n"])


def test_list_scores_sizes_unsupported(eng):
    for ngroup, npair in (((1 << 22) + 1, 3), (2, 1 << 31)):
        with pytest.raises(cabi.M3GError) as ei:
            eng.list_scores_device(rows(), rows(), ngroup, P, P, P, npair, P, P, 1.0, 0.0, P,
                                   cabi.F32, 64)
        assert ei.value.code == UNSUPPORTED


@pytest.mark.parametrize("case", [
    dict(dtype=cabi.E4M3), dict(n=7), dict(dim=199), dict(ldx=199), dict(x=None), dict(x=P + 2),
    dict(out=dict(dtype=cabi.BF16)), dict(out=dict(ld=208 - 8)), dict(out=dict(ld_scales=2))],
    ids=str)
def test_pack_rows_refused(eng, case):
    with pytest.raises(ValueError):
        eng.pack_rows_device(case.get("x", P), case.get("dtype", cabi.F32), case.get("n", 8),
                             case.get("dim", 200), case.get("ldx", 200),
                             rows(**case.get("out", {})))


@pytest.mark.parametrize("case", [
    dict(dtype=cabi.E4M3), dict(nq=-1), dict(n=-1), dict(ld=99), dict(scale=0.0),
    dict(scale=float("inf")), dict(scale=float("nan")), dict(k=-1), dict(ngiven=-1),
    dict(scores=None), dict(lse=None), dict(entropy=None), dict(given=None),
    dict(out_given=None), dict(top=None), dict(top_index=None), dict(scores=P + 2),
    dict(given=P + 4), dict(top_index=P + 4), dict(row_off=P + 4)], ids=str)
def test_score_probs_refused(eng, case):
    v = dict(scores=P, dtype=cabi.F32, nq=4, n=100, ld=100, row_off=None, scale=1.0, given=P,
             ngiven=2, k=3, lse=P, entropy=P, out_given=P, top_index=P, top=P)
    v.update(case)
    with pytest.raises(ValueError):
        eng.score_probs_device(*v.values(), P, 1 << 40)


def test_score_probs_limits(eng):
    with pytest.raises(cabi.M3GError) as ei:
        eng.score_probs_device(P, cabi.F32, 4, 1000, 1000, None, 1.0, None, 0, 129, P, P, None, P,
                               P, P, 1 << 40)
    assert ei.value.code == UNSUPPORTED
    with pytest.raises(cabi.M3GError) as ei:
        eng.score_probs_device(P, cabi.F32, 4, 1 << 31, 1 << 31, None, 1.0, None, 0, 0, P, P, None,
                               None, None, P, 1 << 40)
    assert ei.value.code == UNSUPPORTED


def test_empty_calls_touch_nothing(eng):
    """Calls of no rows, queries or pairs return before any device work."""
    none = rows(n=0, data=None, scales=None)
    eng.pack_rows_device(None, cabi.F32, 0, 200, 200, none)
    eng.row_scores_device(none, rows(), 1.0, 0.0, None, cabi.F32, 8)
    eng.row_scores_device(rows(), none, 1.0, 0.0, None, cabi.F32, 0)
    eng.list_scores_device(rows(), rows(), 0, None, None, None, 0, None, None, 1.0, 0.0, None,
                           cabi.F32, 0)
    eng.score_probs_device(None, cabi.F32, 0, 0, 0, None, 1.0, None, 0, 0, None, None, None, None,
                           None, None, 0)


def test_device_of(eng):
    assert eng.device() == 0
    assert cabi.lib().m3g_device_of(eng.h, None) == cabi.M3G_EINVAL
    assert cabi.lib().m3g_device_of(None, None) == cabi.M3G_EINVAL


def test_storage_stays_fp32_or_bf16(eng):
    """The 8-bit type is one of rows that cross the boundary, not a list storage."""
    with pytest.raises(ValueError):
        eng.create_ivf(1, 4, cabi.IP, False, [[0.0] * 4], storage=cabi.E4M3)


def test_torch_form_refuses_cpu_tensors(eng):
    from m3_memory_b200 import row_scores as R

    x = torch.zeros(4, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        R.pack_rows(eng, x)
    with pytest.raises(ValueError):
        R.row_scores(eng, x, x)
    with pytest.raises(ValueError):
        R.score_probs(eng, torch.zeros(2, 3))


def test_packed_values_on_cpu():
    """PackedRows.values: what codes and scale bytes stand for."""
    from m3_memory_b200.row_scores import PackedRows

    codes = torch.zeros(2, 144, dtype=torch.uint8)
    codes[0, 0], codes[0, 127], codes[0, 128], codes[1, 129] = 0x38, 0x7E, 0x01, 0xB8
    scales = torch.tensor([[127, 130, 0, 0], [1, 120, 0, 0]], dtype=torch.uint8)
    v = PackedRows(codes, scales, 130).values()
    assert v.shape == (2, 130)
    assert v[0, 0] == 1.0 and v[0, 127] == 448.0 and v[0, 128] == 8 * 2.0 ** -9
    assert v[1, 129] == -(2.0 ** -7) and v[1].abs().sum() == 2.0 ** -7

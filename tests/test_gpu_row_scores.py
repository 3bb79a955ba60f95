"""Row scores against plain 64-bit forms: packing, scores of every row, scores of probed lists,
scores as probabilities, and a retrieval that uses them together."""
import math

import numpy as np
import pytest
import torch

from m3_memory_b200 import cabi

pytestmark = pytest.mark.gpu
U32, U16 = 2.0 ** -24, 2.0 ** -8  # half a step of fp32 and of bf16, relative


@pytest.fixture(scope="module")
def R(cuda_ok):
    from m3_memory_b200 import row_scores

    return row_scores


@pytest.fixture(scope="module")
def eng(cuda_ok):
    return cabi.Engine()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, device="cuda", generator=gen(seed)) * scale


# ---------------- packing ----------------


def pack_ref(x):
    """Codes (as values) and scale bytes of fp64 numpy rows, straight from the definition."""
    n, dim = x.shape
    nblk = -(-dim // 128)
    vals, sb = np.empty((n, dim)), np.empty((n, nblk), np.int64)
    grid = np.array([(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:-1] +
                    [m * 2.0 ** -9 for m in range(8)])
    grid = np.unique(grid)  # the non-negative e4m3 values
    assert grid[-1] == 448.0 and len(grid) == 127
    for b in range(nblk):
        v = x[:, b * 128:(b + 1) * 128]
        a = np.where(np.isfinite(v), np.abs(v), 0.0).max(1)
        e = np.full(n, -126)
        for i in range(n):
            while a[i] > 448.0 * 2.0 ** float(e[i]):
                e[i] += 1
        sb[:, b] = e + 127
        y = v * 2.0 ** -e[:, None].astype(np.float64)
        ay = np.minimum(np.abs(y), 448.0)
        hi = np.searchsorted(grid, np.nan_to_num(ay)).clip(0, 126)
        lo = np.maximum(hi - 1, 0)
        dl, dh = ay - grid[lo], grid[hi] - ay
        even_lo = lo % 2 == 0  # the grid's index parity is the code's last bit
        pick = np.where((dl < dh) | ((dl == dh) & even_lo), grid[lo], grid[hi])
        vals[:, b * 128:(b + 1) * 128] = np.where(np.isnan(y), np.nan, np.copysign(pick, y))
    return vals, sb


def special_rows(dim):
    x = np.zeros((12, dim), np.float32)
    r = np.random.default_rng(3)
    x[1] = r.standard_normal(dim)
    x[2] = np.float32(1e-45) * np.arange(dim)
    x[3] = 3.4e38 * r.uniform(-1, 1, dim)
    x[4] = r.standard_normal(dim)
    x[4, ::5] = np.inf
    x[4, 1::5] = -np.inf
    x[4, 2::5] = np.nan
    x[5] = np.nan
    x[6] = -np.inf
    x[7] = np.tile([17.0, 19.0, 1.0625, 1.1875, 448.0, -464.0, 2.0 ** -10, 3 * 2.0 ** -10],
                   -(-dim // 8))[:dim]  # ties, the largest code, the smallest ones
    x[8] = 448.0
    x[9] = np.nextafter(np.float32(448.0), np.float32(1e9))
    x[10] = 2.0 ** -126 * r.uniform(0, 2, dim)
    x[11] = -0.0
    return x


@pytest.mark.parametrize("dim", [1, 7, 100, 127, 128, 129, 250, 768, 1024, 1030])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pack_rows_exact(R, eng, dim, dtype):
    x = torch.from_numpy(np.concatenate([special_rows(dim),
                                         np.random.default_rng(dim).standard_normal((37, dim))
                                         .astype(np.float32)])).cuda().to(dtype)
    p = R.pack_rows(eng, x)
    vals, sb = pack_ref(x.double().cpu().numpy())
    got = p.codes[:, :dim].view(torch.float8_e4m3fn).double().cpu().numpy()
    nblk = -(-dim // 128)
    assert np.array_equal(p.scales[:, :nblk].cpu().numpy(), sb)
    assert np.array_equal(got, vals, equal_nan=True)
    assert np.array_equal(np.signbit(got), np.signbit(vals) | (np.isnan(got) & np.signbit(got)))


@pytest.mark.parametrize("n,dim,pad,shift", [(1, 1, 0, 0), (5, 130, 3, 0), (64, 256, 4, 1),
                                             (3, 1000, 8, 2), (1000, 64, 1, 3),
                                             (20011, 96, 0, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pack_rows_strides_and_bounds(R, eng, n, dim, pad, shift, dtype):
    """Rows with a gap, from any element on, into rows with a gap: only what the rows hold is
    written."""
    store = randn(n * (dim + pad) + shift, seed=n).to(dtype)
    x = torch.as_strided(store, (n, dim), (dim + pad, 1), shift)
    nblk = -(-dim // 128)
    codes = torch.full((n + 2, -(-dim // 16) * 16 + 32), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((n + 2, -(-nblk // 4) * 4 + 4), 0x5A, dtype=torch.uint8, device="cuda")
    R.pack_rows(eng, x, out=R.PackedRows(codes[1:-1], scales[1:-1], dim))
    vals, sb = pack_ref(x.double().cpu().numpy())
    got = codes[1:-1, :dim].contiguous().view(torch.float8_e4m3fn).double().cpu().numpy()
    assert np.array_equal(got, vals)
    assert np.array_equal(scales[1:-1, :nblk].cpu().numpy(), sb)
    assert (codes[0] == 0xA5).all() and (codes[-1] == 0xA5).all() and (codes[:, dim:] == 0xA5).all()
    assert (scales[0] == 0x5A).all() and (scales[-1] == 0x5A).all()
    assert (scales[:, nblk:] == 0x5A).all()


# ---------------- scores ----------------


def make_rows(R, eng, kind, n, dim, seed, gap=0, scale=1.0):
    """(rows, their values in fp64); gap: 16-byte units between rows."""
    x = randn(max(n, 1), dim, seed=seed, scale=scale)[:n]
    # blocks of very different sizes, so that every scale byte matters
    x = x * torch.pow(2.0, (torch.arange(dim, device="cuda") // 128 * 5 % 7 - 3).float())
    if kind == "bf16":
        st = torch.full((n, -(-dim // 8) * 8 + 8 * gap), float("nan"), device="cuda",
                        dtype=torch.bfloat16)
        st[:, :dim] = x
        r = st[:, :dim]
        return r, r.double()
    nblk = -(-dim // 128)
    codes = torch.full((n, -(-dim // 16) * 16 + 16 * gap), 0x7F, dtype=torch.uint8, device="cuda")
    scales = torch.full((n, -(-nblk // 4) * 4 + 4 * gap), 0xFF, dtype=torch.uint8, device="cuda")
    p = R.PackedRows(codes, scales, dim)
    R.pack_rows(eng, x, out=p)
    v = codes[:, :dim].contiguous().view(torch.float8_e4m3fn).double()
    s = torch.pow(2.0, scales[:, :nblk].double() - 127.0)
    return p, v * s.repeat_interleave(128, 1)[:, :dim]


def scores_ref(q, x, alpha, beta, out_dtype, dim):
    """fp64 scores and how far a result may be off: the products of 8-bit or bf16 values are exact
    in fp32; each of the dim additions may lose one step (2^-23, truncation included) of the sum
    of the terms' sizes; scale and shift round once each (2^-24); the type's own rounding."""
    s = alpha * (q @ x.t()) + beta
    terms = abs(alpha) * (q.abs() @ x.abs().t())
    tol = (dim + 2) * 2 * U32 * 1.01 * terms + 2 * U32 * (s.abs() + abs(beta))
    if out_dtype == torch.bfloat16:
        tol = tol * (1 + U16) + U16 * s.abs()
    return s, tol


SHAPES = [(1, 1, 1), (1, 2, 128), (1, 300, 128), (1, 5000, 1024), (2, 127, 16), (3, 129, 100),
          (8, 1000, 256), (16, 128, 513), (17, 1000, 1024), (33, 257, 130), (64, 640, 768),
          (65, 333, 384), (129, 200, 90), (240, 256, 128), (241, 384, 256), (250, 513, 768),
          (300, 700, 136), (700, 1300, 640), (1000, 129, 1100), (31, 40000, 64), (520, 60000, 64), (60, 200000, 32)]


@pytest.mark.parametrize("nq,n,dim", SHAPES)
@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
def test_row_scores(R, eng, nq, n, dim, kind):
    q, qv = make_rows(R, eng, kind, nq, dim, 1, gap=nq % 3)
    x, xv = make_rows(R, eng, kind, n, dim, 2, gap=n % 2)
    for out_dtype, alpha, beta in ((torch.float32, 1.0, 0.0), (torch.bfloat16, -1.0, 1.0)):
        got = R.row_scores(eng, q, x, alpha=alpha, beta=beta, out_dtype=out_dtype)
        ref, tol = scores_ref(qv, xv, alpha, beta, out_dtype, dim)
        bad = (got.double() - ref).abs() > tol
        assert got.dtype == out_dtype and not bad.any(), (out_dtype, int(bad.sum()))
    eng.sync_errors()


@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_row_scores_into_strided_output(R, eng, kind, out_dtype, off):
    """An output with a gap between rows and any first element: nothing else is written."""
    nq, n, dim = 70, 301, 200
    q, qv = make_rows(R, eng, kind, nq, dim, 5)
    x, xv = make_rows(R, eng, kind, n, dim, 6)
    store = torch.full((nq + 2, n + 9), 7.0, device="cuda", dtype=out_dtype)
    out = store[1:-1, off:off + n]
    R.row_scores(eng, q, x, out=out)
    ref, tol = scores_ref(qv, xv, 1.0, 0.0, out_dtype, dim)
    assert ((out.double() - ref).abs() <= tol).all()
    rest = store.clone()
    rest[1:-1, off:off + n] = 7.0
    assert (rest == 7.0).all()


@pytest.mark.parametrize("dim", [96, 512, 513, 1024, 1536, 1537, 2048, 4000])
@pytest.mark.parametrize("nq", [1, 40, 300])
def test_fp32_scores_of_bf16_rows_are_not_low(R, eng, dim, nq):
    """Sums of like terms (a query and rows near one another): the tensor core cuts sums at every
    16 dims, by half a step of fp32 each on average; sums of a quarter (from 1537 dims on, or with
    up to 64 queries), half (from 513) or all of the dims keep what is lost below dim / 16 / parts
    half steps of 2^-23, and fp32 rounding of the parts' sum below two more."""
    base = randn(1, dim, seed=dim)
    x = (base + 0.3 * randn(2000, dim, seed=1)).bfloat16()
    q = (base + 0.3 * randn(nq, dim, seed=2)).bfloat16()
    st = lambda v: torch.nn.functional.pad(v, (0, -dim % 8))[:, :dim]  # noqa: E731
    got = R.row_scores(eng, st(q), st(x)).double()
    want = q.double() @ x.double().t()
    parts = 4 if nq <= 64 or dim > 1536 else 2 if dim > 512 else 1
    low = ((want - got) / want).mean().item()
    assert abs(low) <= (dim / 16 / parts / 2 + 2) * 2 * U32, low


def test_row_scores_nan_rows(R, eng):
    """A NaN in one row reaches that row's scores alone, whatever the neighbours in its tile are;
    rows past the last one are not read into anything."""
    dim = 256
    for kind in ("e4m3", "bf16"):
        v = randn(200, dim, seed=9)
        v[7, 3] = math.nan
        w = randn(30, dim, seed=10)
        w[11, 200] = math.nan
        if kind == "e4m3":
            x, q = R.pack_rows(eng, v), R.pack_rows(eng, w)
            x = R.PackedRows(x.codes[:150], x.scales[:150], dim)
        else:
            x, q = v.bfloat16()[:150], w.bfloat16()
        s = R.row_scores(eng, q, x)
        nan = torch.zeros(30, 150, dtype=torch.bool, device="cuda")
        nan[11] = True
        nan[:, 7] = True
        assert torch.equal(s.isnan(), nan), kind


def test_row_scores_extreme_scales(R, eng):
    """Scale bytes at both ends: exact powers of two come through, products past fp32's range
    become infinite and those below it vanish."""
    dim = 256
    codes = torch.full((4, dim), 0x38, dtype=torch.uint8, device="cuda")  # ones
    scales = torch.tensor([[127, 127], [190, 127], [1, 1], [254, 254]], dtype=torch.uint8,
                          device="cuda").repeat(1, 2)
    p = R.PackedRows(codes, scales, dim)
    s = R.row_scores(eng, p, p).double().cpu()
    one = 128.0
    assert s[0, 0] == 2 * one and s[0, 1] == one * (2.0 ** 63 + 1) and s[1, 0] == s[0, 1]
    assert s[0, 2] == 2 * one * 2.0 ** -126 and s[2, 2] == 0.0 and s[3, 3] == math.inf
    assert s[1, 1] == math.inf  # 128 * 2^126 = 2^133 is past fp32's largest, below 2^128


# ---------------- scores of probed lists ----------------


def make_lists(rng, nlist, mean, n, npair_of, nq, skip=0.0, overlap=False):
    length = rng.integers(0, 2 * mean + 1, nlist)
    length[rng.random(nlist) < 0.2] = 0
    if overlap:
        off = rng.integers(0, max(1, n - 2 * mean), nlist)
    else:
        off = np.cumsum(length + rng.integers(0, 5, nlist)) - length
        assert off[-1] + length[-1] <= n
    count = np.array([npair_of(rng, g) for g in range(nlist)])
    pair_off = np.concatenate([[0], np.cumsum(count)])
    group = np.repeat(np.arange(nlist), count)
    row = rng.integers(0, nq, len(group))
    row[rng.random(len(group)) < skip] = -1
    size = length[group]
    gap = rng.integers(0, 3, len(group))
    order = rng.permutation(len(group))
    start = np.empty(len(group), np.int64)
    start[order] = np.cumsum((size + gap)[order]) - size[order]
    out_n = int((size + gap).sum()) + 5
    return off, length, pair_off, group, row, start, out_n


def lists_check(R, eng, kind, out_dtype, nq, n, dim, lay, gather=True, alpha=1.0, beta=0.0):
    off, length, pair_off, group, row, start, out_n = lay
    q, qv = make_rows(R, eng, kind, nq, dim, 21, gap=1)
    x, xv = make_rows(R, eng, kind, n, dim, 22)
    t = lambda a, d: torch.from_numpy(np.ascontiguousarray(a)).to(d).cuda()  # noqa: E731
    out = torch.full((out_n,), 7.0, device="cuda", dtype=out_dtype)
    R.list_scores(eng, q, x, t(off, torch.int64), t(length, torch.int32),
                  t(pair_off, torch.int64), t(start, torch.int64), out,
                  pair_row=t(row, torch.int32) if gather else None, alpha=alpha, beta=beta)
    eng.sync_errors()
    ref = torch.full((out_n,), 7.0, device="cuda", dtype=torch.float64)
    tol = torch.zeros(out_n, device="cuda", dtype=torch.float64)
    for p in range(len(group)):
        g, r = group[p], row[p] if gather else p
        if r < 0 or length[g] == 0:
            continue
        s, e = scores_ref(qv[r:r + 1], xv[off[g]:off[g] + length[g]], alpha, beta, out_dtype, dim)
        ref[start[p]:start[p] + length[g]] = s[0]
        tol[start[p]:start[p] + length[g]] = e[0]
    bad = ~((out.double() - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:5].tolist())


LISTS = [  # nlist, mean rows, queries, dim, pairs per list
    (1, 5, 1, 16, lambda r, g: 1), (5, 3, 4, 128, lambda r, g: int(r.integers(0, 3))),
    (16, 100, 9, 256, lambda r, g: int(r.integers(0, 6))),
    (40, 130, 50, 1024, lambda r, g: int(r.integers(0, 20))),
    (12, 200, 300, 200, lambda r, g: int(r.choice([0, 1, 15, 16, 17, 63, 64, 65, 240, 241, 300]))),
    (700, 20, 64, 64, lambda r, g: int(r.random() < 0.5)),
    (300, 64, 100, 130, lambda r, g: int(r.integers(0, 4))),
    (3, 3000, 20, 96, lambda r, g: 5), (2500, 3, 64, 128, lambda r, g: int(r.integers(0, 3))),
    (9, 150, 40, 48, lambda r, g: int(r.choice([0, 33, 40, 48, 64, 90]))),
    (8, 150, 200, 640, lambda r, g: int(r.choice([0, 100, 111, 112, 113, 200]))),
    (9, 150, 40, 1030, lambda r, g: int(r.choice([0, 33, 40, 48, 64, 90]))),
    (8, 150, 200, 1600, lambda r, g: int(r.choice([0, 64, 65, 100, 129, 200])))]


@pytest.mark.parametrize("i", range(len(LISTS)))
@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
def test_list_scores(R, eng, i, kind):
    nlist, mean, nq, dim, per = LISTS[i]
    rng = np.random.default_rng(100 + i)
    n = nlist * (2 * mean + 5) + 3
    lay = make_lists(rng, nlist, mean, n, per, nq, skip=0.1 if i % 2 else 0.0)
    lists_check(R, eng, kind, torch.bfloat16 if i % 2 else torch.float32, nq, n, dim, lay,
                alpha=-1.0 if i % 3 else 1.0, beta=float(i % 3))


@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
def test_list_scores_without_gather_and_with_shared_rows(R, eng, kind):
    rng = np.random.default_rng(5)
    lay = make_lists(rng, 30, 90, 1000, lambda r, g: int(r.integers(0, 9)), 1, overlap=True)
    npair = len(lay[3])
    lists_check(R, eng, kind, torch.float32, npair, 1000, 160, lay, gather=False)


def test_list_scores_bad_items_left_out(R, eng):
    """Lists and pairs out of range are left out and reported; the others are right."""
    dim, nq, n = 64, 6, 400
    q, qv = make_rows(R, eng, "bf16", nq, dim, 1)
    x, xv = make_rows(R, eng, "bf16", n, dim, 2)
    T = lambda a, d=torch.int64: torch.tensor(a, dtype=d, device="cuda")  # noqa: E731
    list_off = T([0, 390, -1, 100, 200, 300])
    list_len = T([100, 20, 10, 100, -5, 50], torch.int32)
    pair_off = T([0, 2, 3, 4, 7, 8, 9])
    row = T([0, 99, 1, 2, 3, 4, -2, 5, 5], torch.int32)
    out_off = T([0, 100, 200, 220, 300, 1000, 400, 500, 600])
    out = torch.full((700,), 7.0, device="cuda")
    R.list_scores(eng, q, x, list_off, list_len, pair_off, out_off, out, pair_row=row)
    with pytest.raises(IndexError):
        eng.sync_errors()
    eng.sync_errors()  # reported once
    want = torch.full((700,), 7.0, device="cuda", dtype=torch.float64)
    for p, a, m, o in ((0, 0, 100, 0), (3, 100, 100, 300), (5, 300, 50, 600)):
        want[o:o + m] = (qv[p:p + 1] @ xv[a:a + m].t())[0]
    assert torch.allclose(out.double(), want, rtol=1e-4, atol=1e-4)
    # pair offsets that fall, or end past the pairs
    for po in ([0, 2, 1, 4, 7, 8, 9], [0, 2, 3, 4, 7, 8, 10], [-1, 2, 3, 4, 7, 8, 9]):
        R.list_scores(eng, q, x, T([0] * 6), T([10] * 6, torch.int32), T(po),
                      T([10 * i for i in range(9)]), out, pair_row=T([0] * 9, torch.int32))
        with pytest.raises(IndexError):
            eng.sync_errors()


# ---------------- probabilities ----------------


def probs_ref(rows, scale, k, given):
    """fp64 results of a list of rows, with how far fp32 results may be off.  Each exp is within
    2^-21 of its value (its own error and the rounding of its argument, which is at most 2^-22 of
    an argument d, so 2^-22 |d| more); a sum of m terms loses at most (m / 256 + 40) half steps;
    logarithms and the final sums lose 4 half steps of their results."""
    out = []
    for i, s in enumerate(rows):
        l = np.asarray(s, np.float64) * scale
        held = l > -np.inf
        none = np.full(k, -np.inf)
        if not held.any():
            g = None if given is None else np.full(given.shape[1], -np.inf)
            out.append((-np.inf, 0.0, g, none, np.full(k, -1), 0.0, 0.0, 0.0))
            continue
        m = l[held].max()
        d = np.where(held, l - m, 0.0)
        p = np.where(held, np.exp(d), 0.0)
        z, t = p.sum(), (p * d).sum()
        lse, ent = m + np.log(z), np.log(z) - t / z
        adds = (len(l) / 256 + 40) * U32
        rel = adds + 2.0 ** -21 + 2.0 ** -22 * (p * abs(d)).sum() / z
        e_lse = rel + 4 * U32 * (abs(lse) + abs(m) + abs(np.log(z)))
        e_ent = rel * (1 + abs(t) / z) + 8 * U32 * (abs(np.log(z)) + abs(t) / z) + \
            (adds + 2.0 ** -20) * abs(t) / z + 2.0 ** -22 * (p * d * d).sum() / z
        logp = np.where(held, l - lse, -np.inf)
        logp[logp < -3.4028236e38] = -np.inf  # past fp32's range
        g = None
        if given is not None:
            g = np.array([logp[a] if 0 <= a < len(l) else -np.inf for a in given[i]])
        order = np.argsort(np.where(held, -np.sign(scale) * np.asarray(s, np.float64), np.inf),
                           kind="stable")
        order = order[held[order]][:k]
        idx = np.full(k, -1)
        idx[:len(order)] = order
        top = none.copy()
        top[:len(order)] = logp[order]
        out.append((lse, ent, g, top, idx, e_lse, e_ent, m))
    return out


def close(got, want, tol):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    same = (got == want) | (np.abs(np.where(np.isfinite(got), got, 0) -
                                   np.where(np.isfinite(want), want, 0)) <= tol)
    return bool((same & (np.isfinite(got) == np.isfinite(want))).all())


def probs_check(R, eng, scores, rows, scale, k, given=None, row_off=None):
    got = R.score_probs(eng, scores, scale=scale, k=k, given=given, row_off=row_off)
    ref = probs_ref(rows, scale, k, None if given is None else given.cpu().numpy())
    lse, ent = got.logsumexp.cpu().numpy(), got.entropy.cpu().numpy()
    for i, (l, h, g, top, idx, el, eh, m) in enumerate(ref):
        assert close(lse[i], l, el), (i, lse[i], l, el)
        assert close(ent[i], h, eh), (i, ent[i], h, eh)
        if k:
            assert np.array_equal(got.top_index[i].cpu().numpy(), idx), i
            t = got.top[i].cpu().numpy()
            assert close(t, top, el + 4 * U32 * (np.abs(np.nan_to_num(top, neginf=0)) + abs(m))), i
        if given is not None:
            assert close(got.given[i].cpu().numpy(), g,
                         el + 4 * U32 * (np.abs(np.nan_to_num(g, neginf=0)) + abs(m))), i
    assert (got.top is None) == (k == 0) and (got.given is None) == (given is None)


def some_scores(nq, n, dtype, seed, ties=False):
    s = randn(nq, n, seed=seed, scale=0.1)
    if ties:
        s = (s * 20).round() / 20
    s[torch.rand(nq, n, device="cuda", generator=gen(seed + 1)) < 0.05] = -math.inf
    s[torch.rand(nq, n, device="cuda", generator=gen(seed + 2)) < 0.02] = math.nan
    if nq > 3:
        s[1] = math.nan
        s[2] = -math.inf
        s[3, 1:] = -math.inf
    return s.to(dtype)


@pytest.mark.parametrize("nq,n,k", [(1, 1, 1), (1, 1, 0), (5, 2, 4), (4, 31, 32), (7, 33, 1),
                                    (3, 1000, 10), (2, 4096, 33), (6, 5001, 100), (4, 257, 128),
                                    (1, 300001, 10), (2, 100003, 128), (300, 777, 5),
                                    (1, 50001, 1), (3, 40000, 3), (2, 70001, 33), (1, 30000, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [30.0, -1.0])
def test_score_probs(R, eng, nq, n, k, dtype, scale):
    s = some_scores(nq, n, dtype, nq + n, ties=n % 2 == 1) * math.copysign(1.0, scale)
    given = torch.randint(-2, n + 2, (nq, 3), device="cuda", generator=gen(4))
    probs_check(R, eng, s, list(s.float().cpu().numpy()), scale, k, given)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off,ld", [(0, 505), (1, 503), (3, 512), (7, 611)])
def test_score_probs_strided(R, eng, dtype, off, ld):
    """Rows of any stride from any element on; what is between them does not count."""
    store = torch.full((9 * ld + 64,), 50.0, device="cuda", dtype=dtype)
    s = torch.as_strided(store, (9, 500), (ld, 1), off)
    s.copy_(some_scores(9, 500, dtype, 8))
    probs_check(R, eng, s, list(s.float().cpu().numpy()), 10.0, 7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [0, 4, 100])
def test_score_probs_ragged(R, eng, dtype, k):
    rng = np.random.default_rng(k)
    size = np.concatenate([[0, 1, 2, 0, 31, 32, 33, 5000, 20011, 0],
                           rng.integers(0, 900, 90), [0]])
    off = np.concatenate([[0], np.cumsum(size)]) + 3  # the first entries belong to no row
    flat = some_scores(1, int(off[-1]) + 11, dtype, 3, ties=True)[0]
    f = flat.float().cpu().numpy()
    rows = [f[a:b] for a, b in zip(off, off[1:])]
    given = torch.from_numpy(rng.integers(-1, 50, (len(size), 2))).cuda()
    probs_check(R, eng, flat, rows, 25.0, k, given, torch.from_numpy(off).cuda())


def test_score_probs_scratch_on_any_8_byte_boundary(R, eng):
    """Split rows of every odd and even k, the scratch 8 bytes off a 16-byte boundary, and nothing
    written past its end."""
    nq, n = 3, 40001
    s = some_scores(nq, n, torch.float32, 1)
    rows = list(s.cpu().numpy())
    for k in (0, 1, 2, 3, 7, 127):
        need = eng.score_probs_work(nq, n, False, cabi.F32, k)
        assert need > 0
        work = torch.full((need + 64,), 0x5A, dtype=torch.uint8, device="cuda")
        lse, ent = torch.empty(nq, device="cuda"), torch.empty(nq, device="cuda")
        top = torch.empty(nq, max(k, 1), device="cuda")
        idx = torch.empty(nq, max(k, 1), dtype=torch.int64, device="cuda")
        eng.score_probs_device(s.data_ptr(), cabi.F32, nq, n, n, None, 2.0, None, 0, k,
                               lse.data_ptr(), ent.data_ptr(), None, idx.data_ptr(),
                               top.data_ptr(), work.data_ptr() + 8, need)
        assert (work[:8] == 0x5A).all() and (work[8 + need:] == 0x5A).all()
        for i, r in enumerate(probs_ref(rows, 2.0, k, None)):
            assert close(lse[i].item(), r[0], r[5]) and close(ent[i].item(), r[1], r[6])
            assert not k or np.array_equal(idx[i].cpu().numpy(), r[4])


def test_score_probs_many_equal_scores(R, eng):
    """Rows of one value, and of values that only differ beyond k: the lowest places are taken."""
    for dtype in (torch.float32, torch.bfloat16):
        s = torch.full((3, 70001), 0.25, device="cuda", dtype=dtype)
        s[1, 50000:] = 0.5
        s[2, ::2] = -0.0
        s[2, 1::2] = 0.0
        probs_check(R, eng, s, list(s.float().cpu().numpy()), 3.0, 128)
    # the best entries all in one part of a long row, and spread one to a part
    s = randn(1, 600000, seed=5, scale=0.1)
    s[0, 300000:300200] += 2.0
    probs_check(R, eng, s, list(s.cpu().numpy()), 4.0, 30)
    s[0, ::3001] += 3.0
    for k in (1, 10, 100, 128):
        probs_check(R, eng, s, list(s.cpu().numpy()), 4.0, k)
    long = torch.arange(700000, device="cuda", dtype=torch.float32)[None] / 700000
    probs_check(R, eng, long, list(long.cpu().numpy()), 4.0, 20)
    up = torch.arange(60000, device="cuda", dtype=torch.float32)[None] / 60000
    probs_check(R, eng, up, list(up.cpu().numpy()), 4.0, 128)  # every entry enters the best k
    probs_check(R, eng, -up, list(-up.cpu().numpy()), 4.0, 128)


def test_score_probs_extremes(R, eng):
    """Scores of the type's largest sizes, an infinite logit, and scales at both ends."""
    big = torch.tensor([[3e38, -3e38, 3e38, 1.0], [-3.4028235e38] * 4, [1e-40, 2e-40, 0, -1e-40]],
                       device="cuda")
    probs_check(R, eng, big, list(big.cpu().numpy()), 1.0, 4)
    probs_check(R, eng, big[2:], list(big[2:].cpu().numpy()), 1e38, 4)
    probs_check(R, eng, big, list(big.cpu().numpy()), 1e-38, 4)
    inf = torch.tensor([[1.0, math.inf, 0.0]], device="cuda")
    got = R.score_probs(eng, inf, scale=2.0, k=1)
    assert got.logsumexp.item() == math.inf and math.isnan(got.entropy.item())
    assert got.top_index.item() == 1


def test_score_probs_bad_rows_reported(R, eng):
    """Row offsets that fall, or leave the scores: those rows count as empty, the others are right."""
    s = some_scores(1, 1000, torch.float32, 2)[0]
    f = s.cpu().numpy()
    off = [0, 100, 90, 300, 2000, 400, 500, -5, 10]
    good = [(a, b) if 0 <= a <= b <= 1000 else (0, 0) for a, b in zip(off, off[1:])]
    t = torch.tensor(off, device="cuda")
    got = R.score_probs(eng, s, scale=3.0, k=4, row_off=t)
    with pytest.raises(IndexError):
        eng.sync_errors()
    eng.sync_errors()
    for i, (a, b) in enumerate(good):
        r = probs_ref([f[a:b]], 3.0, 4, None)[0]
        assert close(got.logsumexp[i].item(), r[0], r[5])
        assert np.array_equal(got.top_index[i].cpu().numpy(), r[4])


def test_score_probs_no_rows_or_entries(R, eng):
    got = R.score_probs(eng, torch.empty(0, 5, device="cuda"), k=2)
    assert got.top.shape == (0, 2)
    got = R.score_probs(eng, torch.empty(3, 0, device="cuda"), k=2,
                        given=torch.zeros(3, 1, dtype=torch.int64, device="cuda"))
    assert (got.logsumexp == -math.inf).all() and (got.entropy == 0).all()
    assert (got.top_index == -1).all() and (got.top == -math.inf).all()
    assert (got.given == -math.inf).all()


# ---------------- streams, graphs, use together ----------------


def retrieval(R, eng, q, x, lay, k):
    """Pack the queries, score their probed lists, and the distribution over what was scored."""
    packed = R.pack_rows(eng, q)
    out = torch.full((lay["total"],), math.nan, device="cuda")
    R.list_scores(eng, packed, x, lay["list_off"], lay["list_len"], lay["pair_off"],
                  lay["out_off"], out, pair_row=lay["pair_row"])
    return out, R.score_probs(eng, out, scale=30.0, k=k, row_off=lay["row_off"])


def probe_layout(probes, list_len):
    """Pairs grouped by list, each query's scores one after another in probe order."""
    nq, P = probes.shape
    flat = probes.reshape(-1).long()
    order = flat.sort(stable=True).indices
    size = list_len[flat].long()
    start = size.cumsum(0) - size
    z = torch.zeros(1, dtype=torch.int64, device="cuda")
    return dict(list_off=list_len.long().cumsum(0) - list_len, list_len=list_len.int(),
                pair_off=torch.cat([z, torch.bincount(flat, minlength=len(list_len)).cumsum(0)]),
                pair_row=(order // P).int(), out_off=start[order].contiguous(),
                row_off=torch.cat([z, size.view(nq, P).sum(1).cumsum(0)]), start=start.view(nq, P),
                size=size.view(nq, P), total=int(size.sum()))


def test_retrieval_with_probabilities_matches_search(R, eng):
    """An engine's index and the row scores together: the entries the distribution ranks first
    are the ones a search over the packed values returns."""
    n, dim, nlist, nq, P, k = 6000, 192, 24, 33, 5, 10
    x = randn(n, dim, seed=1)
    x = x / x.norm(dim=1, keepdim=True)
    packed = R.pack_rows(eng, x)
    values = packed.values()
    assign = torch.randint(0, nlist, (n,), device="cuda", generator=gen(2)).int()
    order = assign.long().sort(stable=True).indices
    C = torch.stack([values[assign == c].mean(0) for c in range(nlist)])
    e = cabi.Engine()
    e.create_ivf(1, dim, cabi.IP, False, C.cpu().numpy())
    ids = torch.arange(n, device="cuda", dtype=torch.int64) * 3 + 1
    e.load_lists_device(1, assign.data_ptr(), ids.data_ptr(), values.data_ptr(), n)
    q = R.pack_rows(eng, randn(nq, dim, seed=3)).values()  # already 8-bit values: packing keeps them
    probes = torch.empty(nq, P, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    e.select_probes_device(1, q.data_ptr(), nq, P, probes.data_ptr())
    lay = probe_layout(probes, torch.bincount(assign.long(), minlength=nlist))
    by_list = R.PackedRows(packed.codes[order], packed.scales[order], dim)
    scores, got = retrieval(R, e, q, by_list, lay, k)
    e.sync_errors()
    want, want_sc, cnt = e.search(1, q.cpu().numpy(), k, P)
    assert (cnt == k).all()
    # a place in a query's row of scores -> the row of the list it falls in -> its id
    ends = (lay["start"] - lay["start"][:, :1] + lay["size"])
    slot = torch.searchsorted(ends, got.top_index, right=True)
    at = got.top_index - (ends - lay["size"]).gather(1, slot)
    row = lay["list_off"][probes.long().gather(1, slot)] + at
    got_ids = ids[order][row].cpu().numpy()
    top_scores = torch.gather(torch.nn.utils.rnn.pad_sequence(
        [scores[a:b] for a, b in zip(lay["row_off"].tolist(), lay["row_off"].tolist()[1:])],
        batch_first=True), 1, got.top_index).cpu().numpy()
    # both are fp32 sums of the same dim products, at most dim steps of the terms' sizes apart
    assert np.allclose(-want_sc, top_scores, rtol=0, atol=dim * 2.0 ** -22 * 20)
    differ = got_ids != want
    assert np.abs(-want_sc - top_scores)[differ].max(initial=0) <= dim * 2.0 ** -22 * 20
    assert differ.mean() < 0.02
    p = got.top.exp().sum(1)
    # (an entropy below 2^-24, one entry having nearly all of the probability, may come out as 0)
    assert ((p > 0) & (p <= 1 + 1e-4)).all() and (got.entropy >= 0).all()
    assert (got.entropy > 0).float().mean() > 0.5


def test_streams_and_concurrent_calls(R, eng):
    """Calls on several streams at once, each ordered with its own stream's work."""
    x, xv = make_rows(R, eng, "e4m3", 3000, 256, 1)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for rep in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                q = randn(40 + i, 256, seed=10 * rep + i)
                s = R.row_scores(eng, R.pack_rows(eng, q), x)
                outs.append((q, s, R.score_probs(eng, s, scale=0.1, k=3)))
    torch.cuda.synchronize()
    eng.sync_errors()
    for q, s, p in outs:
        again = R.row_scores(eng, R.pack_rows(eng, q), x)
        want = R.score_probs(eng, again, scale=0.1, k=3)
        assert torch.equal(s, again) and torch.equal(p.top_index, want.top_index)
        assert torch.equal(p.logsumexp, want.logsumexp) and torch.equal(p.entropy, want.entropy)


def test_host_thread_calls_at_once(R, eng):
    """The calls hold no state of the engine: host threads may make them at the same time."""
    import threading

    x, _ = make_rows(R, eng, "bf16", 2000, 128, 1)
    q, _ = make_rows(R, eng, "bf16", 50, 128, 2)
    want = R.row_scores(eng, q, x)
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = R.row_scores(eng, q, x)
            torch.cuda.current_stream().synchronize()

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert all(torch.equal(g, want) for g in got)


def test_two_graphs_of_one_retrieval(R, eng):
    """The run captured twice, replayed at once on two streams with new inputs."""
    nlist, dim, nq, P = 12, 256, 20, 4
    list_len = torch.randint(0, 300, (nlist,), device="cuda", generator=gen(1))
    n = int(list_len.sum())
    x, _ = make_rows(R, eng, "e4m3", n, dim, 2)
    probes = torch.stack([torch.randperm(nlist, device="cuda", generator=gen(i))[:P]
                          for i in range(nq)])
    lay = probe_layout(probes, list_len)
    qs = [torch.zeros(nq, dim, device="cuda") for _ in range(2)]
    retrieval(R, eng, qs[0], x, lay, 5)  # first call outside a capture
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(retrieval(R, eng, qs[i], x, lay, 5))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(3):
        new = [randn(nq, dim, seed=50 + 2 * rep + i) for i in range(2)]
        for i in range(2):
            qs[i].copy_(new[i])
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            s, p = retrieval(R, eng, new[i], x, lay, 5)
            assert torch.equal(s, outs[i][0])
            assert torch.equal(p.top_index, outs[i][1].top_index)
            assert torch.equal(p.entropy, outs[i][1].entropy)
    eng.sync_errors()
    del graphs


def test_graph_of_split_rows(R, eng):
    """Rows split over blocks (two kernels) captured and replayed with new scores, eager calls of
    the same shape between."""
    s = some_scores(3, 60001, torch.float32, 1)
    R.score_probs(eng, s, scale=4.0, k=6)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = R.score_probs(eng, s, scale=4.0, k=6)
    for rep in range(4):
        new = some_scores(3, 60001, torch.float32, 10 + rep)
        s.copy_(new)
        g.replay()
        want = R.score_probs(eng, new, scale=4.0, k=6)
        torch.cuda.synchronize()
        assert torch.equal(got.logsumexp, want.logsumexp)
        assert torch.equal(got.top_index, want.top_index) and torch.equal(got.top, want.top)
    del g


def test_null_stream_waits_and_reports(R, eng):
    """Without a stream a call waits, and reports what its kernels found."""
    x, xv = make_rows(R, eng, "bf16", 100, 64, 1)
    out = torch.zeros(100, 100, device="cuda")
    r = cabi.Rows(x.data_ptr(), None, 100, x.stride(0), 0, 64, cabi.BF16)
    eng.row_scores_device(r, r, 1.0, 0.0, out.data_ptr(), cabi.F32, 100)
    ref, tol = scores_ref(xv, xv, 1.0, 0.0, torch.float32, 64)
    assert ((out.double() - ref).abs() <= tol).all()
    one = torch.zeros(2, dtype=torch.int64, device="cuda")
    one[1] = 1
    length = torch.tensor([200], dtype=torch.int32, device="cuda")
    with pytest.raises(IndexError):
        eng.list_scores_device(r, r, 1, one.data_ptr(), length.data_ptr(), one.data_ptr(), 1,
                               None, one.data_ptr(), 1.0, 0.0, out.data_ptr(), cabi.F32, 10000)
    assert ((out.double() - ref).abs() <= tol).all()
    eng.sync_errors()


def test_results_do_not_change_from_call_to_call(R, eng):
    q, _ = make_rows(R, eng, "e4m3", 100, 512, 1)
    x, _ = make_rows(R, eng, "e4m3", 20000, 512, 2)
    s = R.row_scores(eng, q, x)
    p = R.score_probs(eng, s, scale=0.3, k=20)
    for _ in range(5):
        s2 = R.row_scores(eng, q, x)
        p2 = R.score_probs(eng, s2, scale=0.3, k=20)
        assert torch.equal(s, s2) and torch.equal(p.top_index, p2.top_index)
        assert torch.equal(p.logsumexp, p2.logsumexp) and torch.equal(p.entropy, p2.entropy)
        assert torch.equal(p.top, p2.top)


def test_outputs_are_written_whole(R, eng):
    """Every score is written, whatever was there."""
    for kind in ("e4m3", "bf16"):
        for nq, n, dim in ((1, 1000, 128), (70, 700, 300)):
            q, _ = make_rows(R, eng, kind, nq, dim, 1)
            x, _ = make_rows(R, eng, kind, n, dim, 2)
            out = torch.full((nq, n), math.nan, device="cuda")
            R.row_scores(eng, q, x, out=out)
            assert not out.isnan().any()

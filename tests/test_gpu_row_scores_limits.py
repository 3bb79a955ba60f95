"""Row scores at the limits of what a call may be given."""
import threading
import time

import numpy as np
import pytest
import torch

from m3_memory_b200 import cabi
from test_gpu_row_scores import close, make_rows, probs_check, scores_ref

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24  # half a step of fp32, relative


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


@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
@pytest.mark.parametrize("gather", [True, False])
def test_pair_that_ends_past_the_output_is_left_out_whole(R, eng, kind, gather):
    """A list of several tiles, written for one pair to the last elements, for others past them by
    one or by more than a tile: none of their scores is written, before the end either."""
    nq, n, dim, length = 4, 900, 192, 700
    q, qv = make_rows(R, eng, kind, nq, dim, 1)
    x, xv = make_rows(R, eng, kind, n, dim, 2)
    out_n = 3 * length
    out = torch.full((out_n,), 7.0, device="cuda")
    start = [out_n - length, out_n - length + 1, length, out_n - 200]
    R.list_scores(eng, q, x, T([150]), T([length], torch.int32), T([0, nq]), T(start), out,
                  pair_row=T([0, 1, 2, 3], torch.int32) if gather else None)
    with pytest.raises(IndexError):
        eng.sync_errors()
    ref, tol = scores_ref(qv, xv[150:150 + length], 1.0, 0.0, torch.float32, dim)
    assert (out[:length] == 7.0).all()
    assert ((out[length:2 * length].double() - ref[2]).abs() <= tol[2]).all()
    assert ((out[2 * length:].double() - ref[0]).abs() <= tol[0]).all()
    # alone: nothing at all
    out.fill_(7.0)
    R.list_scores(eng, q, x, T([150]), T([length], torch.int32), T([0, 1]), T(start[3:]), out)
    with pytest.raises(IndexError):
        eng.sync_errors()
    assert (out == 7.0).all()


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


# ---------------- large logits ----------------


def near_equal(nq, n, size, dtype, seed):
    """Scores within a few steps of their type below `size` (whose products with a scale fp32
    rounds by many units), a few far below, some left out."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    step = size * torch.finfo(dtype).eps
    s = size - step * torch.randint(0, 6, (nq, n), device="cuda", generator=g)
    s[torch.rand(nq, n, device="cuda", generator=g) < 0.3] *= -0.5
    s[torch.rand(nq, n, device="cuda", generator=g) < 0.05] = float("nan")
    s[torch.rand(nq, n, device="cuda", generator=g) < 0.05] = -float("inf")
    return s.to(dtype)


@pytest.mark.parametrize("nq,n,k", [(3, 1, 1), (2, 7, 3), (5, 1000, 10), (4, 5003, 100),
                                    (2, 100003, 10), (300, 777, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size,scale", [(3e8, 50.3), (-3e8, 50.3), (1e6, 1.7), (2.5e4, 50.3),
                                        (1e9, 7.7), (1e30, 1.1), (4e7, 1e20), (1.2e10, -0.3)])
def test_large_logits(R, eng, nq, n, k, dtype, size, scale):
    """Logits far past 2^20, where fp32 rounds the largest one by more than e^x bears."""
    s = near_equal(nq, n, size, dtype, nq + n) * (1.0 if scale > 0 else -1.0)
    # the formula's scale is the fp32 value; a product of it with a score is exact in 64 bits
    given = torch.randint(-1, n + 1, (nq, 2), device="cuda")
    rows, scale = list(s.float().cpu().numpy()), float(np.float32(scale))
    probs_check(R, eng, s, rows, scale, k, given)
    # log p again, without the largest logit's size in the tolerance: l - m is exact to 2^-22 of
    # itself, log z to the relative error of z (see probs_ref), the difference to half a step
    got = R.score_probs(eng, s, scale=scale, k=k, given=given)
    for i, r in enumerate(rows):
        l = np.asarray(r, np.float64) * scale
        held = l > -np.inf
        if not held.any():
            continue
        d = np.where(held, l - l[held].max(), -np.inf)
        p = np.exp(d)
        z, x = p.sum(), -(p * np.where(held, d, 0.0)).sum()
        e_z = (n / 256 + 40) * U32 + 2.0 ** -21 + 2.0 ** -22 * x / z
        pairs = [(got.given[i].cpu().numpy(),
                  [d[j] if 0 <= j < n else -np.inf for j in given[i].tolist()])]
        if k:
            at = got.top_index[i].cpu().numpy()
            pairs.append((got.top[i].cpu().numpy()[at >= 0], d[at[at >= 0]]))
        for have, want in pairs:
            want = np.asarray(want)
            dist = np.abs(np.nan_to_num(want, neginf=0.0))
            logp = want - np.log(z)
            tol = e_z + 4 * U32 * dist + 4 * U32 * (dist + abs(np.log(z)))
            assert close(have, logp, tol), (i, have, logp, tol)


def test_large_logits_ragged(R, eng):
    size = [0, 1, 40, 9000, 3, 20011]
    off = T(size).cumsum(0)
    off = torch.cat([T([0]), off])
    s = near_equal(1, sum(size), 3e8, torch.float32, 5)[0]
    f = s.cpu().numpy()
    rows = [f[a:b] for a, b in zip(off.tolist(), off.tolist()[1:])]
    probs_check(R, eng, s, rows, float(np.float32(50.3)), 12, row_off=off)


@pytest.mark.parametrize("mask", [-1e9, -3e4, -1e30, torch.finfo(torch.float32).min,
                                  torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [50.3, 0.7])
def test_rows_masked_by_a_large_value(R, eng, mask, dtype, scale):
    """Entries masked by a large finite value instead of -inf: runs of them at the start, at the
    end, whole parts of a long row, and rows of nothing else."""
    g = torch.Generator(device="cuda").manual_seed(3)
    scale = float(np.float32(scale))
    for nq, n, k in ((6, 9000, 10), (4, 60001, 100)):
        s = torch.randn(nq, n, device="cuda", generator=g)
        s[0, :n // 2] = mask
        s[1, n // 3:] = mask
        s[2] = mask
        s[3, torch.rand(n, device="cuda", generator=g) < 0.9] = mask
        s = s.to(dtype)
        rows = s.float().cpu().numpy()
        # l is an fp32 value: a product below fp32's range is -inf, and such entries are left out
        rows[rows.astype(np.float64) * scale < -3.4028235677973366e38] = -np.inf
        probs_check(R, eng, s, list(rows), scale, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_masked_rows_that_are_not_split(R, eng, dtype):
    """So many rows that a warp takes each whole: masked runs of long rows, and rows of large
    logits, sum up as well as other rows (a lane adds n / 512 blocks of at most 16 sums, and the
    lanes' are joined in 5 steps)."""
    nq, n, scale = 1800, 60001, float(np.float32(50.3))
    g = torch.Generator(device="cuda").manual_seed(8)
    s = torch.randn(nq, n, device="cuda", generator=g) * 0.004
    s[0, :20000] = -1e9
    s[1, 40000:] = -1e9
    s[2, ::2] = -1e30
    s[3] = 3e8
    s = s.to(dtype)
    got = R.score_probs(eng, s, scale=scale, k=2)
    for i in range(5):
        l = s[i].double() * scale
        d = l - l.max()
        p = d.exp()
        z, t = p.sum().item(), (p * d).sum().item()
        adds = (n / 512 + 16 + 5) * U32
        rel = adds + 2.0 ** -21 + 2.0 ** -22 * abs(t) / z  # (see probs_ref)
        lse, ent = l.max().item() + np.log(z), np.log(z) - t / z
        assert abs(got.logsumexp[i].item() - lse) <= rel + 4 * U32 * (abs(lse) + 12.0), i
        assert abs(got.entropy[i].item() - ent) <= rel * (1 + 2 * abs(t) / z) + 8 * U32 * 12.0, i
        assert abs(got.top[i, 0].item() + np.log(z)) <= rel + 4 * U32 * 12.0, i


# ---------------- several callers ----------------


def busy_stream(seconds=0.5):
    """A stream with a wait of the GPU's own on it, and an event behind that."""
    st, done = torch.cuda.Stream(), torch.cuda.Event()
    with torch.cuda.stream(st):
        torch.cuda._sleep(int(seconds * 1.9e9))
        done.record()
    return st, done


def test_calls_do_not_wait_for_another_threads_sync_errors(R, eng):
    """While one thread waits for the device in sync_errors, calls of others are enqueued."""
    q, _ = make_rows(R, eng, "bf16", 20, 128, 1)
    x, _ = make_rows(R, eng, "bf16", 500, 128, 2)
    want = R.row_scores(eng, q, x)
    p = R.score_probs(eng, want, k=3)
    torch.cuda.synchronize()
    _, done = busy_stream()
    waiting = threading.Thread(target=eng.sync_errors)
    waiting.start()
    time.sleep(0.1)  # it is inside
    with torch.cuda.stream(torch.cuda.Stream()):
        s = R.row_scores(eng, q, x)
        again = R.score_probs(eng, s, k=3)
    still_busy = not done.query()
    waiting.join()
    assert still_busy
    assert torch.equal(s, want) and torch.equal(again.top_index, p.top_index)


def test_first_cuda_call_of_a_host_thread(R, eng):
    """A thread that has not used CUDA before makes the calls (by their addresses: torch would set
    the thread up)."""
    x, xv = make_rows(R, eng, "bf16", 100, 64, 1)
    out = torch.zeros(100, 100, device="cuda")
    R.row_scores(eng, x, x)  # its kernel is set up
    off, length, pairs = T([0]), T([100], torch.int32), T([0, 1])
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    stream, r = st.cuda_stream, cabi.Rows(x.data_ptr(), None, 100, x.stride(0), 0, 64, cabi.BF16)
    raised = []

    def run(call):
        def work():
            try:
                call()
            except Exception as e:  # noqa: BLE001
                raised.append(e)
        t = threading.Thread(target=work)
        t.start()
        t.join()
        torch.cuda.synchronize()
        assert not raised, raised

    run(lambda: eng.row_scores_device(r, r, 1.0, 0.0, out.data_ptr(), cabi.F32, 100, stream))
    ref, tol = scores_ref(xv, xv, 1.0, 0.0, torch.float32, 64)
    assert ((out.double() - ref).abs() <= tol).all()
    R.list_scores(eng, x, x, off, length, pairs, off, out.view(-1))
    out.zero_()
    torch.cuda.synchronize()
    run(lambda: eng.list_scores_device(r, r, 1, off.data_ptr(), length.data_ptr(),
                                       pairs.data_ptr(), 1, None, off.data_ptr(), 1.0, 0.0,
                                       out.data_ptr(), cabi.F32, 10000, stream))
    assert ((out[0].double() - ref[0]).abs() <= tol[0]).all()


def plain_call(eng, x, out):
    """row_scores of bf16 rows without a stream: the call waits."""
    r = cabi.Rows(x.data_ptr(), None, x.shape[0], x.stride(0), 0, x.shape[1], cabi.BF16)
    eng.row_scores_device(r, r, 1.0, 0.0, out.data_ptr(), cabi.F32, out.stride(0))


def bad_lists(R, eng, x, out):
    """An enqueued call with a list past the rows."""
    R.list_scores(eng, x, x, T([0]), T([x.shape[0] + 1], torch.int32), T([0, 1]), T([0]), out)


def test_waiting_call_waits_for_its_stream_alone(R, eng):
    x, xv = make_rows(R, eng, "bf16", 100, 64, 1)
    out = torch.zeros(100, 100, device="cuda")
    plain_call(eng, x, out)
    still_busy = 0
    for _ in range(6):  # (streams that share a hardware queue do wait for one another)
        _, done = busy_stream(0.1)
        plain_call(eng, x, out)
        still_busy += not done.query()
        torch.cuda.synchronize()
    assert still_busy > 0
    ref, tol = scores_ref(xv, xv, 1.0, 0.0, torch.float32, 64)
    assert ((out.double() - ref).abs() <= tol).all()


def test_waiting_call_reports_its_own_errors_alone(R, eng):
    x, _ = make_rows(R, eng, "bf16", 100, 64, 1)
    out = torch.zeros(100, 100, device="cuda")
    bad_lists(R, eng, x, out.view(-1))
    torch.cuda.synchronize()
    plain_call(eng, x, out)  # nothing wrong with this one
    with pytest.raises(IndexError):
        eng.sync_errors()
    # and what a waiting call raised is not reported again
    r = cabi.Rows(x.data_ptr(), None, 100, x.stride(0), 0, 64, cabi.BF16)
    off, length, pairs = T([0]), T([101], torch.int32), T([0, 1])
    torch.cuda.synchronize()
    for _ in range(2):
        with pytest.raises(IndexError):
            eng.list_scores_device(r, r, 1, off.data_ptr(), length.data_ptr(), pairs.data_ptr(), 1,
                                   None, off.data_ptr(), 1.0, 0.0, out.data_ptr(), cabi.F32, 10000)
        plain_call(eng, x, out)
    eng.sync_errors()


def test_waiting_calls_of_several_threads(R, eng):
    """Each raises for itself: the bad ones always, the good ones never."""
    x, _ = make_rows(R, eng, "bf16", 100, 64, 1)
    outs = [torch.zeros(100, 100, device="cuda") for _ in range(4)]
    r = cabi.Rows(x.data_ptr(), None, 100, x.stride(0), 0, 64, cabi.BF16)
    off, length, pairs = T([0]), T([101], torch.int32), T([0, 1])
    torch.cuda.synchronize()
    raised = [0] * 4

    def work(i):
        for _ in range(50):
            try:
                if i % 2:
                    eng.list_scores_device(r, r, 1, off.data_ptr(), length.data_ptr(),
                                           pairs.data_ptr(), 1, None, off.data_ptr(), 1.0, 0.0,
                                           outs[i].data_ptr(), cabi.F32, 10000)
                else:
                    plain_call(eng, x, outs[i])
            except IndexError:
                raised[i] += 1

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert raised == [0, 50, 0, 50]
    eng.sync_errors()


def test_no_error_of_concurrent_calls_is_lost(R, eng):
    """Bad calls, one after another, while another thread takes errors all the time: after each has
    ended, an error is reported once more (two calls between two reports share one)."""
    x, _ = make_rows(R, eng, "bf16", 100, 64, 1)
    out = torch.zeros(10000, device="cuda")
    bad_lists(R, eng, x, out)
    with pytest.raises(IndexError):
        eng.sync_errors()
    reports, stop = [0], [False]

    def take():
        while not stop[0]:
            try:
                eng.sync_errors()
            except IndexError:
                reports[0] += 1

    t = threading.Thread(target=take)
    t.start()
    try:
        for i in range(300):
            before = reports[0]
            bad_lists(R, eng, x, out)
            deadline = time.time() + 10
            while reports[0] == before and time.time() < deadline:
                time.sleep(1e-5)
            assert reports[0] > before, i
    finally:
        stop[0] = True
        t.join()
    eng.sync_errors()


# ---------------- first calls within a capture ----------------


@pytest.mark.parametrize("warm_up", ["none", "pack", "empty"])
@pytest.mark.parametrize("what", ["scores", "lists", "probs"])
def test_first_call_of_an_engine_is_captured(R, what, warm_up):
    """A new engine's first call, or its first after packing or an empty call, is made in a
    capture: the graph holds it and reports through the engine."""
    e = cabi.Engine()
    n, dim, nq = 300, 128, 9
    x, xv = make_rows(R, cabi.Engine(), "e4m3", n, dim, 1)
    q, qv = make_rows(R, cabi.Engine(), "e4m3", nq, dim, 2)
    if warm_up == "pack":
        R.pack_rows(e, torch.randn(5, dim, device="cuda"))
    elif warm_up == "empty":
        R.row_scores(e, R.PackedRows(q.codes[:0], q.scales[:0], dim), x)
    out = torch.zeros(nq, n, device="cuda")
    off, length, pairs = T([0]), T([n], torch.int32), T([0, nq])
    at = torch.arange(nq, device="cuda") * n
    s = torch.randn(3, 60001, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        if what == "scores":
            R.row_scores(e, q, x, out=out)
        elif what == "lists":
            R.list_scores(e, q, x, off, length, pairs, at, out.view(-1))
        else:
            got = R.score_probs(e, s, k=5)
    g.replay()
    torch.cuda.synchronize()
    if what == "probs":
        assert torch.equal(got.top_index, R.score_probs(e, s, k=5).top_index)
    else:
        ref, tol = scores_ref(qv, xv, 1.0, 0.0, torch.float32, dim)
        assert ((out.double() - ref).abs() <= tol).all()
    e.sync_errors()
    if what == "lists":
        length.fill_(n + 1)
        g.replay()
        with pytest.raises(IndexError):
            e.sync_errors()
    del g


# ---------------- sizes ----------------


@pytest.mark.parametrize("dim", [1, 2, 3, 7, 8, 9, 15, 17, 31, 33, 63, 65, 20001])
@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
def test_rows_of_few_and_of_many_dims(R, eng, kind, dim):
    q, qv = make_rows(R, eng, kind, 70, dim, 1, gap=1)
    x, xv = make_rows(R, eng, kind, 200, dim, 2, gap=1)
    ref, tol = scores_ref(qv, xv, 1.0, 0.0, torch.float32, dim)
    assert ((R.row_scores(eng, q, x).double() - ref).abs() <= tol).all()
    for gather in (True, False):
        out = torch.full((70, 200), 7.0, device="cuda")
        R.list_scores(eng, q, x, T([0]), T([200], torch.int32), T([0, 70]),
                      torch.arange(70, device="cuda") * 200, out.view(-1),
                      pair_row=torch.arange(70, device="cuda").int() if gather else None)
        assert ((out.double() - ref).abs() <= tol).all()
    eng.sync_errors()


@pytest.mark.parametrize("nlist", [300001, 1 << 22])
def test_many_lists(R, eng, nlist):
    """Most lists empty or not probed; the last one and every 1009th are."""
    dim, n, nq = 64, 5000, 12
    q, qv = make_rows(R, eng, "e4m3", nq, dim, 1)
    x, xv = make_rows(R, eng, "e4m3", n, dim, 2)
    g = torch.arange(nlist, device="cuda")
    probed = (g % 1009 == 0) | (g == nlist - 1)
    length = (g * 7 % 5).int()
    off = g * 31 % (n - 5)
    pair_off = torch.cat([T([0]), probed.long().cumsum(0)])
    group = probed.nonzero()[:, 0]
    npair = len(group)
    row = torch.arange(npair, device="cuda") % nq
    size = length[group].long()
    start = size.cumsum(0) - size
    out = torch.full((int(size.sum()),), 7.0, device="cuda")
    R.list_scores(eng, q, x, off, length, pair_off, start, out, pair_row=row.int())
    eng.sync_errors()
    pair = torch.repeat_interleave(torch.arange(npair, device="cuda"), size)
    j = torch.arange(len(pair), device="cuda") - start[pair]
    a, b = qv[row[pair]], xv[off[group[pair]] + j]
    tol = (dim + 2) * 2 * U32 * 1.01 * (a.abs() * b.abs()).sum(1)  # (see scores_ref)
    assert ((out.double() - (a * b).sum(1)).abs() <= tol + 2 * U32 * (a * b).sum(1).abs()).all()


FAR = (1 << 32) + 24  # elements: past what 32 bits hold, a multiple of 8


def test_outputs_and_scores_past_32_bits(R, eng):
    """Rows of scores more than 2^32 elements apart, written and read there."""
    nq, n, dim = 2, 700, 96
    q, qv = make_rows(R, eng, "bf16", nq, dim, 1)
    x, xv = make_rows(R, eng, "bf16", n, dim, 2)
    store = torch.empty(FAR + n, dtype=torch.bfloat16, device="cuda")
    out = store.as_strided((nq, n), (FAR, 1))
    R.row_scores(eng, q, x, out=out)
    ref, tol = scores_ref(qv, xv, 1.0, 0.0, torch.bfloat16, dim)
    assert ((out.double() - ref).abs() <= tol).all()
    got = R.score_probs(eng, out, scale=0.01, k=5)
    near = R.score_probs(eng, out.contiguous(), scale=0.01, k=5)
    assert all(torch.equal(a, b) for a, b in zip((got.logsumexp, got.entropy, got.top_index),
                                                 (near.logsumexp, near.entropy, near.top_index)))
    # as lists: a pair's scores that start past 2^32, and a ragged row there
    store.view(-1)[FAR:] = 7.0
    R.list_scores(eng, q, x, T([0]), T([n], torch.int32), T([0, 1]), T([FAR]), store,
                  pair_row=T([1], torch.int32))
    assert ((store[FAR:].double() - ref[1]).abs() <= tol[1]).all()
    far = R.score_probs(eng, store, scale=0.01, k=5, row_off=T([FAR, FAR + n]))
    assert torch.equal(far.top_index[0], near.top_index[1])
    eng.sync_errors()


@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
def test_rows_past_32_bits(R, eng, kind):
    """Rows (and their scales) more than 2^32 bytes from the first, packed, scored and gathered."""
    dim, n, nq = 128, 3, 20
    ld = 1 << 31
    v = torch.randn(n, dim, device="cuda")
    if kind == "e4m3":
        src = torch.empty((n - 1) * ld + dim, dtype=torch.bfloat16, device="cuda").as_strided(
            (n, dim), (ld, 1))
        src.copy_(v)
        codes = torch.empty((n - 1) * ld * 2 + dim, dtype=torch.uint8,
                            device="cuda").as_strided((n, dim), (2 * ld, 1))
        scales = torch.empty((n - 1) * ld * 2 + 4, dtype=torch.uint8,
                             device="cuda").as_strided((n, 4), (2 * ld, 1))
        x = R.pack_rows(eng, src, out=R.PackedRows(codes, scales, dim))
        near = R.pack_rows(eng, v.bfloat16())
        assert torch.equal(codes, near.codes) and torch.equal(scales[:, 0], near.scales[:, 0])
        q, _ = make_rows(R, eng, kind, nq, dim, 3)
    else:
        near = v.bfloat16()
        x = torch.empty((n - 1) * ld + dim, dtype=torch.bfloat16, device="cuda").as_strided(
            (n, dim), (ld, 1))
        x.copy_(near)
        q, _ = make_rows(R, eng, kind, nq, dim, 3)
    assert torch.equal(R.row_scores(eng, q, x), R.row_scores(eng, q, near))
    assert torch.equal(R.row_scores(eng, x, q), R.row_scores(eng, near, q))
    row = torch.arange(2 * n, device="cuda").int() % n
    outs = []
    for a in (x, near):
        out = torch.empty(2 * n * nq, device="cuda")
        R.list_scores(eng, a, q, T([0]), T([nq], torch.int32), T([0, 2 * n]),
                      torch.arange(2 * n, device="cuda") * nq, out, pair_row=row)
        outs.append(out)
    assert torch.equal(*outs)
    eng.sync_errors()


@pytest.mark.parametrize("dim,pairs", [(96, 300), (513, 40), (640, 300), (1536, 64), (1537, 300),
                                       (2048, 10), (2048, 300)])
@pytest.mark.parametrize("gather", [True, False])
def test_fp32_list_scores_of_bf16_rows_are_not_low(R, eng, dim, pairs, gather):
    """Sums of like terms in lists, as for every row: what the tensor core cuts off, half a step of
    fp32 on average every 16 dims of each of the sums (four for up to 64 pairs a list or from 1537
    dims on, two from 513 on, else one), and fp32 rounding of their sum."""
    base = torch.randn(1, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(dim))
    pad = -dim % 8

    def rows(n):
        v = (base + 0.3 * torch.randn(n, dim, device="cuda")).bfloat16()
        return torch.nn.functional.pad(v, (0, pad))[:, :dim]

    x, q = rows(700), rows(pairs)
    out = torch.empty(pairs, 700, device="cuda")
    R.list_scores(eng, q, x, T([0]), T([700], torch.int32), T([0, pairs]),
                  torch.arange(pairs, device="cuda") * 700, out.view(-1),
                  pair_row=torch.arange(pairs, device="cuda").int() if gather else None)
    want = q.double() @ x.double().t()
    parts = 4 if pairs <= 64 or dim > 1536 else 2 if dim > 512 else 1
    low = ((want - out.double()) / want).mean().item()
    assert abs(low) <= (dim / 16 / parts / 2 + 2) * 2 * U32, low

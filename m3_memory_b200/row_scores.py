"""Scores of queries against rows, on torch tensors of the engine's GPU.

``search`` answers with the best k entries; these calls give the scores themselves and what follows
from them: rows packed to 8 bits (``pack_rows``), the scores of every row (``row_scores``) or of the
rows of each query's probed lists (``list_scores``), and a row of scores as a distribution
(``score_probs``: how sure a retrieval is, and which entries it might have been).  No counterpart in
the reference, whose searches return k scores (AgentMemory/M3/src/m3_index.cpp:444-475).

Every call is enqueued on the current torch stream and returns at once; ``Engine.sync_errors()``
reports what a kernel found wrong (see include/m3gpu.h, which states the formulas).  Rows are bf16
tensors ``[n, dim]`` or ``PackedRows``; a tensor's rows must start on 16-byte boundaries.  There are
no backward forms: a tensor that requires a gradient is refused (detach it, or call under
``torch.no_grad()``).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import cabi

BLOCK = 128  # dims that share one scale

_F32, _BF16, _U8, _I32, _I64 = (torch.float32, torch.bfloat16, torch.uint8, torch.int32,
                                torch.int64)
_DTYPES = {_F32: cabi.F32, _BF16: cabi.BF16}
_LEGACY_STREAM = 1  # cudaStreamLegacy: torch's default stream, named so that the call does not wait
try:
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:  # a torch without CUDA, or without this short cut
    def _raw_stream(dev):
        return torch.cuda.current_stream(dev).cuda_stream


class PackedRows(NamedTuple):
    """8-bit rows: ``codes`` uint8 ``[n, >= dim]`` (e4m3 bit patterns, row stride a multiple of 16)
    and ``scales`` uint8 ``[n, >= ceil(dim / 128)]`` (row stride a multiple of 4): dim i of a row
    stands for ``codes[i] * 2**(scales[i // 128] - 127)``."""

    codes: torch.Tensor
    scales: torch.Tensor
    dim: int

    def values(self) -> torch.Tensor:
        """The rows as fp32 ``[n, dim]``."""
        v = self.codes[:, :self.dim].view(torch.float8_e4m3fn).float()
        s = torch.pow(2.0, self.scales.double() - 127.0).float()
        return v * s.repeat_interleave(BLOCK, dim=1)[:, :self.dim]


class ScoreProbs(NamedTuple):
    """``score_probs``'s answer; ``given``, ``top`` and ``top_index`` are None where not asked for."""

    logsumexp: torch.Tensor
    entropy: torch.Tensor
    given: Optional[torch.Tensor]
    top: Optional[torch.Tensor]
    top_index: Optional[torch.Tensor]


# The calls below are made per batch, small ones too, so their checks cost little: plain
# comparisons, messages built only where one fails.


def _stream(dev):
    return _raw_stream(dev) or _LEGACY_STREAM


def _matrix_of(n, d, dtype, device):
    """A new contiguous matrix (the cheapest way to one)."""
    return torch.empty_strided((n, d), (d or 1, 1), dtype=dtype, device=device)


def _vector_of(n, dtype, device):
    return torch.empty_strided((n,), (1,), dtype=dtype, device=device)


def _bad(what, msg):
    raise ValueError(f"{what} {msg}")


def _no_grad(t, what):
    if t.requires_grad and torch.is_grad_enabled():
        _bad(what, "requires a gradient, which these calls do not give")


def _device_of(engine, t, what):
    if not isinstance(t, torch.Tensor):
        _bad(what, "must be a CUDA tensor")
    _no_grad(t, what)
    if not t.is_cuda:
        _bad(what, "must be a CUDA tensor")
    dev = t.get_device()
    if dev != engine.device():
        _bad(what, f"is on {t.device}, the engine on cuda:{engine.device()}")
    return dev


def _vector(t, dtype, n, dev, what):
    """The address of a contiguous vector of n values on the device."""
    if t.dtype != dtype or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
        _bad(what, f"must be a contiguous {dtype} vector of {n}")
    if t.get_device() != dev:
        _bad(what, f"is on {t.device}, not on cuda:{dev}")
    return t.data_ptr()


def _matrix(t, dev, what):
    """(n, d, row stride) of a matrix with contiguous rows; a single row has stride d."""
    if t.dim() != 2:
        _bad(what, "must be 2D")
    if t.get_device() != dev:
        _bad(what, f"is on {t.device}, not on cuda:{dev}")
    n, d = t.shape
    ld, one = t.stride()
    if one != 1 and d > 1:
        _bad(what, "must have contiguous rows")
    if n <= 1:
        ld = d
    elif ld < d:
        _bad(what, "must not overlap itself")
    return n, d, ld


def _rows(r, dev, what):
    """The m3g_rows of PackedRows or of a bf16 matrix."""
    if isinstance(r, PackedRows):
        codes, scales, dim = r
        if codes.dtype != _U8 or scales.dtype != _U8:
            _bad(what, "must hold uint8 codes and scales")
        n, d, ld = _matrix(codes, dev, what)
        ns, ds, lds = _matrix(scales, dev, what)
        nblk = (dim + BLOCK - 1) // BLOCK
        if ns != n or dim <= 0 or d < dim or ds < nblk:
            _bad(what, f"codes and scales do not hold {n} rows of {dim} dims")
        if n <= 1:  # no stride to go by
            ld, lds = (dim + 15) // 16 * 16, (nblk + 3) // 4 * 4
        return cabi.Rows(codes.data_ptr(), scales.data_ptr(), n, ld, lds, dim, cabi.E4M3)
    if not isinstance(r, torch.Tensor) or r.dtype != _BF16:
        _bad(what, "must be PackedRows or a bf16 tensor")
    _no_grad(r, what)
    n, dim, ld = _matrix(r, dev, what)
    if n <= 1:
        ld = (dim + 7) // 8 * 8
    return cabi.Rows(r.data_ptr(), None, n, ld, 0, dim, cabi.BF16)


def _dtype(t, what):
    d = _DTYPES.get(t)
    if d is None:
        _bad(what, "must be float32 or bfloat16")
    return d


def _device(engine, rows, what):
    return _device_of(engine, rows.codes if isinstance(rows, PackedRows) else rows, what)


def pack_rows(engine, x, out=None) -> PackedRows:
    """Packs fp32 or bf16 rows ``x [n, dim]`` to 8 bits (m3g_pack_rows_device): e4m3 codes with one
    power-of-two scale per 128 dims.  ``out``: PackedRows to write instead of new ones."""
    dev = _device_of(engine, x, "x")
    dtype = _dtype(x.dtype, "x")
    n, dim, ldx = _matrix(x, dev, "x")
    if out is None:
        if dim == 0:
            _bad("x", "has no dims")
        nblk = (dim + BLOCK - 1) // BLOCK
        out = PackedRows(_matrix_of(n, (dim + 15) // 16 * 16, _U8, x.device),
                         _matrix_of(n, (nblk + 3) // 4 * 4, _U8, x.device), dim)
    elif out.dim != dim or out.codes.shape[0] != n:
        _bad("out", f"does not hold {n} rows of {dim} dims")
    engine.pack_rows_device(x.data_ptr(), dtype, n, dim, ldx, _rows(out, dev, "out"),
                            _stream(dev))
    return out


def row_scores(engine, q, x, alpha=1.0, beta=0.0, out_dtype=torch.float32, out=None):
    """``alpha * q @ x.T + beta`` for every row of q and x (m3g_row_scores_device), ``[len(q),
    len(x)]`` in float32 or bfloat16.  ``out``: a matrix to write instead of a new one."""
    dev = _device(engine, x, "x")
    a, b = _rows(q, dev, "q"), _rows(x, dev, "x")
    if out is None:
        _dtype(out_dtype, "out_dtype")
        t = x.codes if isinstance(x, PackedRows) else x
        out = _matrix_of(a.n, b.n, out_dtype, t.device)
        ld = b.n
    else:
        _no_grad(out, "out")
        n, d, ld = _matrix(out, dev, "out")
        if n != a.n or d != b.n:
            _bad("out", f"must be [{a.n}, {b.n}]")
    engine.row_scores_device(a, b, alpha, beta, out.data_ptr(), _dtype(out.dtype, "out"), ld,
                             _stream(dev))
    return out


def list_scores(engine, q, x, list_off, list_len, pair_off, out_off, out, pair_row=None,
                alpha=1.0, beta=0.0):
    """The scores of every row of each query's probed lists (m3g_list_scores_device), written to
    the vector ``out`` (float32 or bfloat16) and returned.

    List g is rows ``list_off[g] .. list_off[g] + list_len[g]`` of x (int64, int32); the pairs
    ``pair_off[g] .. pair_off[g + 1]`` (int64, one entry more) probe it; pair p is row
    ``pair_row[p]`` of q (int32; row p without it, -1 for none) and writes ``list_len[g]`` scores
    from ``out[out_off[p]]`` (int64) on."""
    dev = _device(engine, x, "x")
    a, b = _rows(q, dev, "q"), _rows(x, dev, "x")
    ngroup, npair, n = list_off.numel(), out_off.numel(), out.numel()
    _no_grad(out, "out")
    engine.list_scores_device(
        a, b, ngroup, _vector(list_off, _I64, ngroup, dev, "list_off"),
        _vector(list_len, _I32, ngroup, dev, "list_len"),
        _vector(pair_off, _I64, ngroup + 1, dev, "pair_off"), npair,
        None if pair_row is None else _vector(pair_row, _I32, npair, dev, "pair_row"),
        _vector(out_off, _I64, npair, dev, "out_off"), alpha, beta,
        _vector(out, out.dtype, n, dev, "out"), _dtype(out.dtype, "out"), n, _stream(dev))
    return out


def score_probs(engine, scores, scale=1.0, k=0, given=None, row_off=None) -> ScoreProbs:
    """Each row of scores as a distribution, p = softmax(scale * scores) (m3g_score_probs_device):
    its log-sum-exp and entropy, the log probability of the ``given`` entries (int64 ``[nq, m]``,
    places in the row; -1 for none) and the k most probable entries.  Entries that are NaN, or
    -inf after scaling, are left out.  ``scores``: float32 or bfloat16 ``[nq, n]``, or a vector
    whose row i is ``scores[row_off[i]:row_off[i + 1]]`` (``row_off`` int64)."""
    dev = _device_of(engine, scores, "scores")
    dtype = _dtype(scores.dtype, "scores")
    off = None
    if row_off is None:
        nq, n, ld = _matrix(scores, dev, "scores")
    else:
        n, ld = scores.numel(), 0
        nq = row_off.numel() - 1
        if nq < 0:
            _bad("row_off", "holds one entry more than there are rows")
        _vector(scores, scores.dtype, n, dev, "scores")
        off = _vector(row_off, _I64, nq + 1, dev, "row_off")
    on, ngiven, given_at = scores.device, 0, None
    out_given = top = top_index = work = None
    if given is not None:
        if given.dtype != _I64 or not given.is_contiguous():
            _bad("given", "must be contiguous int64")
        g, ngiven, _ = _matrix(given, dev, "given")
        if g != nq:
            _bad("given", f"must have {nq} rows")
        out_given = _matrix_of(nq, ngiven, _F32, on)
        given_at = given.data_ptr() if ngiven else None
    lse, entropy = _vector_of(nq, _F32, on), _vector_of(nq, _F32, on)
    if k > 0:
        top, top_index = _matrix_of(nq, k, _F32, on), _matrix_of(nq, k, _I64, on)
    nbytes = engine.score_probs_work(nq, n, off is not None, dtype, k)
    if nbytes:
        work = _vector_of(nbytes, _U8, on)
    engine.score_probs_device(
        scores.data_ptr(), dtype, nq, n, ld, off, scale, given_at, ngiven, k, lse.data_ptr(),
        entropy.data_ptr(), out_given.data_ptr() if ngiven else None,
        top_index.data_ptr() if k > 0 else None, top.data_ptr() if k > 0 else None,
        work.data_ptr() if nbytes else None, nbytes, _stream(dev))
    return ScoreProbs(lse, entropy, out_given, top, top_index)

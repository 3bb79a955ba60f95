"""Scores of queries against rows, on torch tensors of the engine's GPU.

``search`` answers with the best k entries; these calls give the scores themselves and what follows
from them: rows packed to 8 bits (``pack_rows``), the scores of every row (``row_scores``) or of the
rows of each query's probed lists (``list_scores``), and a row of scores as a distribution
(``score_probs``: how sure a retrieval is, and which entries it might have been).  No counterpart in
the reference, whose searches return k scores (AgentMemory/M3/src/m3_index.cpp:444-475).

Every call is enqueued on the current torch stream and returns at once; ``Engine.sync_errors()``
reports what a kernel found wrong (see include/m3gpu.h, which states the formulas).  Rows are bf16
tensors ``[n, dim]`` or ``PackedRows``; a tensor's rows must start on 16-byte boundaries.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import cabi

BLOCK = 128  # dims that share one scale

_LEGACY_STREAM = 1  # cudaStreamLegacy: torch's default stream, named so that the call does not wait
_DTYPES = {torch.float32: cabi.F32, torch.bfloat16: cabi.BF16}


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


def _stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream or _LEGACY_STREAM


def _need(ok, msg):
    if not ok:
        raise ValueError(msg)


def _on(t, dev, what):
    _need(t.device == dev, f"{what} is on {t.device}, not on {dev}")


def _vector(t, dtype, n, dev, what):
    _need(t.dtype == dtype and t.dim() == 1 and t.is_contiguous() and (n is None or len(t) == n),
          f"{what} must be a contiguous {dtype} vector" + ("" if n is None else f" of {n}"))
    _on(t, dev, what)


def _matrix_ld(t, what):
    """The row stride of a matrix with contiguous rows."""
    _need(t.dim() == 2, f"{what} must be 2D")
    n, d = t.shape
    _need(d <= 1 or t.stride(1) == 1, f"{what} must have contiguous rows")
    ld = t.stride(0) if n > 1 else max(d, t.stride(0))
    _need(n <= 1 or ld >= d, f"{what} must not overlap itself")
    return ld


def _rows(r, dev, what):
    if isinstance(r, PackedRows):
        c, s = r.codes, r.scales
        _need(c.dtype == torch.uint8 and s.dtype == torch.uint8, f"{what}: packed rows are uint8")
        _on(c, dev, what)
        _on(s, dev, what)
        ld, lds = _matrix_ld(c, what), _matrix_ld(s, what)
        n, nblk = c.shape[0], -(-r.dim // BLOCK)
        _need(s.shape[0] == n and c.shape[1] >= r.dim > 0 and s.shape[1] >= nblk,
              f"{what}: codes and scales do not hold {n} rows of {r.dim} dims")
        if n == 1:  # a single row has no stride to go by
            ld, lds = -(-max(ld, r.dim) // 16) * 16, -(-max(lds, nblk) // 4) * 4
        return cabi.Rows(c.data_ptr(), s.data_ptr(), n, ld, lds, r.dim, cabi.E4M3)
    _need(isinstance(r, torch.Tensor) and r.dtype == torch.bfloat16,
          f"{what} must be PackedRows or a bf16 tensor")
    _on(r, dev, what)
    ld = _matrix_ld(r, what)
    n, dim = r.shape
    if n == 1:
        ld = -(-max(ld, dim) // 8) * 8
    return cabi.Rows(r.data_ptr(), None, n, ld, 0, dim, cabi.BF16)


def _out_dtype(dtype):
    _need(dtype in _DTYPES, "scores are float32 or bfloat16")
    return _DTYPES[dtype]


def _device(rows):
    t = rows.codes if isinstance(rows, PackedRows) else rows
    _need(isinstance(t, torch.Tensor) and t.is_cuda, "rows must be on a CUDA device")
    return t.device


def pack_rows(engine, x, out=None) -> PackedRows:
    """Packs fp32 or bf16 rows ``x [n, dim]`` to 8 bits (m3g_pack_rows_device): e4m3 codes with one
    power-of-two scale per 128 dims.  ``out``: PackedRows to write instead of new ones."""
    _need(isinstance(x, torch.Tensor) and x.is_cuda, "x must be a CUDA tensor")
    _need(x.dtype in _DTYPES, "x must be float32 or bfloat16")
    ldx = _matrix_ld(x, "x")
    n, dim = x.shape
    dev = x.device
    if out is None:
        _need(dim > 0, "x has no dims")
        nblk = -(-dim // BLOCK)
        out = PackedRows(torch.empty((n, -(-dim // 16) * 16), dtype=torch.uint8, device=dev),
                         torch.empty((n, -(-nblk // 4) * 4), dtype=torch.uint8, device=dev), dim)
    _need(out.dim == dim and len(out.codes) == n, f"out does not hold {n} rows of {dim} dims")
    engine.pack_rows_device(x.data_ptr(), _DTYPES[x.dtype], n, dim, max(ldx, dim),
                            _rows(out, dev, "out"), _stream(dev))
    return out


def row_scores(engine, q, x, alpha=1.0, beta=0.0, out_dtype=torch.float32, out=None):
    """``alpha * q @ x.T + beta`` for every row of q and x (m3g_row_scores_device), ``[len(q),
    len(x)]`` in float32 or bfloat16.  ``out``: a matrix to write instead of a new one."""
    dev = _device(x)
    a, b = _rows(q, dev, "q"), _rows(x, dev, "x")
    if out is None:
        out = torch.empty((a.n, b.n), dtype=out_dtype, device=dev)
        ld = b.n
    else:
        _need(tuple(out.shape) == (a.n, b.n), f"out must be [{a.n}, {b.n}]")
        _on(out, dev, "out")
        ld = max(_matrix_ld(out, "out"), b.n)
    engine.row_scores_device(a, b, alpha, beta, out.data_ptr(), _out_dtype(out.dtype), ld,
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
    dev = _device(x)
    a, b = _rows(q, dev, "q"), _rows(x, dev, "x")
    ngroup, npair = len(list_off), len(out_off)
    _vector(list_off, torch.int64, ngroup, dev, "list_off")
    _vector(list_len, torch.int32, ngroup, dev, "list_len")
    _vector(pair_off, torch.int64, ngroup + 1, dev, "pair_off")
    _vector(out_off, torch.int64, npair, dev, "out_off")
    if pair_row is not None:
        _vector(pair_row, torch.int32, npair, dev, "pair_row")
    _vector(out, out.dtype, None, dev, "out")
    engine.list_scores_device(a, b, ngroup, list_off.data_ptr(), list_len.data_ptr(),
                              pair_off.data_ptr(), npair,
                              None if pair_row is None else pair_row.data_ptr(),
                              out_off.data_ptr(), alpha, beta, out.data_ptr(),
                              _out_dtype(out.dtype), len(out), _stream(dev))
    return out


def score_probs(engine, scores, scale=1.0, k=0, given=None, row_off=None) -> ScoreProbs:
    """Each row of scores as a distribution, p = softmax(scale * scores) (m3g_score_probs_device):
    its log-sum-exp and entropy, the log probability of the ``given`` entries (int64 ``[nq, m]``,
    places in the row; -1 for none) and the k most probable entries.  Entries that are NaN, or
    -inf after scaling, are left out.  ``scores``: float32 or bfloat16 ``[nq, n]``, or a vector
    whose row i is ``scores[row_off[i]:row_off[i + 1]]`` (``row_off`` int64)."""
    _need(isinstance(scores, torch.Tensor) and scores.is_cuda, "scores must be a CUDA tensor")
    _need(scores.dtype in _DTYPES, "scores must be float32 or bfloat16")
    dev = scores.device
    if row_off is None:
        ld = max(_matrix_ld(scores, "scores"), scores.shape[1])
        nq, n = scores.shape
    else:
        _vector(scores, scores.dtype, None, dev, "scores")
        _need(len(row_off) >= 1, "row_off holds one entry more than there are rows")
        _vector(row_off, torch.int64, None, dev, "row_off")
        nq, n, ld = len(row_off) - 1, len(scores), 0
    ngiven = 0
    if given is not None:
        _need(given.dtype == torch.int64 and given.dim() == 2 and given.shape[0] == nq and
              given.is_contiguous(), f"given must be contiguous int64 [{nq}, m]")
        _on(given, dev, "given")
        ngiven = given.shape[1]
    lse = torch.empty(nq, device=dev)
    entropy = torch.empty(nq, device=dev)
    out_given = None if given is None else torch.empty((nq, ngiven), device=dev)
    top = torch.empty((nq, k), device=dev) if k > 0 else None
    top_index = torch.empty((nq, k), dtype=torch.int64, device=dev) if k > 0 else None
    nbytes = engine.score_probs_work(nq, n, row_off is not None, k)
    work = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    engine.score_probs_device(
        scores.data_ptr(), _DTYPES[scores.dtype], nq, n, ld,
        None if row_off is None else row_off.data_ptr(), scale,
        given.data_ptr() if ngiven else None, ngiven, k, lse.data_ptr(), entropy.data_ptr(),
        out_given.data_ptr() if ngiven else None, top_index.data_ptr() if k > 0 else None,
        top.data_ptr() if k > 0 else None, work.data_ptr() if nbytes else None, nbytes,
        _stream(dev))
    return ScoreProbs(lse, entropy, out_given, top, top_index)

"""Measured cases of the row-score operators: packing rows to 8 bits, scores of every row, scores of
the rows of probed lists, and scores as probabilities.

``run`` computes each operator in plain torch operations (``own`` false) or through
``m3_memory_b200.row_scores`` (``own`` true).  Vectors are unit-norm embeddings in a few clusters, as
the index holds them; 8-bit rows are e4m3 codes with one power-of-two scale per 128 dims.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128  # dims that share one scale


# ---------------------------------------------------------------------------------------------
# cases


def listed():
    return [
        # one embedding, packed before it is scored: a call's latency
        {"name": "pack_1x1024_f32", "op": "pack", "n": 1, "dim": 1024, "dtype": "f32"},
        # a batch of queries that arrives as bf16
        {"name": "pack_4096x768_bf16", "op": "pack", "n": 4096, "dim": 768, "dtype": "bf16"},
        # a whole memory of fp32 vectors, packed once
        {"name": "pack_1000000x1024_f32", "op": "pack", "n": 1000000, "dim": 1024, "dtype": "f32"},
        # one query against a whole memory: the rows are read once, nothing is shared
        {"name": "scores_1x1000000x1024_e4m3", "op": "scores", "nq": 1, "n": 1000000, "dim": 1024,
         "rows": "e4m3", "out": "f32"},
        # a batch of queries against a memory of odd size
        {"name": "scores_1024x100003x1024_e4m3", "op": "scores", "nq": 1024, "n": 100003,
         "dim": 1024, "rows": "e4m3", "out": "f32"},
        # a large batch against the centroids of a large index, rows kept as bf16
        {"name": "scores_4096x16384x768_bf16", "op": "scores", "nq": 4096, "n": 16384, "dim": 768,
         "rows": "bf16", "out": "bf16"},
        # one query's probed lists: a call's latency
        {"name": "lists_1x8of256_1024_e4m3", "op": "lists", "nq": 1, "nprobe": 8, "nlist": 256,
         "mean": 390, "dim": 1024, "rows": "e4m3", "out": "f32"},
        # a batch of 1024 queries over a memory of a million rows in 4096 lists
        {"name": "lists_1024x32of4096_1024_e4m3", "op": "lists", "nq": 1024, "nprobe": 32,
         "nlist": 4096, "mean": 244, "dim": 1024, "rows": "e4m3", "out": "f32"},
        # a large batch over bf16 rows
        {"name": "lists_4096x16of4096_768_bf16", "op": "lists", "nq": 4096, "nprobe": 16,
         "nlist": 4096, "mean": 244, "dim": 768, "rows": "bf16", "out": "bf16"},
        # one query's distribution over a whole memory
        {"name": "probs_1x1000003_f32", "op": "probs", "nq": 1, "n": 1000003, "dtype": "f32",
         "k": 10, "given": 4, "scale": 50.0, "ragged": False},
        # a batch's distributions
        {"name": "probs_1024x100003_f32", "op": "probs", "nq": 1024, "n": 100003, "dtype": "f32",
         "k": 10, "given": 4, "scale": 50.0, "ragged": False},
        # a large batch's distributions over the rows of its probed lists, bf16 scores
        {"name": "probs_4096xragged3904_bf16", "op": "probs", "nq": 4096, "n": 3904,
         "dtype": "bf16", "k": 100, "given": 1, "scale": 20.0, "ragged": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pack", "scores", "lists", "probs"])
    if op == "pack":
        dim = _log_int(rng, 64, 2048)
        n = _log_int(rng, 1, 1000000)
        return {"op": op, "n": max(1, min(n, 1000000 * 1024 // dim)), "dim": dim,
                "dtype": rng.choice(["f32", "bf16"])}
    if op == "scores":
        dim = _log_int(rng, 96, 2048)
        nq = _log_int(rng, 1, 4096)
        n = _log_int(rng, 256, 1000000)
        n = max(1, min(n, 100003 * 1024 // nq, 1024 * 100003 * 1024 // (nq * dim),
                       1000000 * 1024 // dim))
        return {"op": op, "nq": nq, "n": n, "dim": dim, "rows": rng.choice(["e4m3", "bf16"]),
                "out": rng.choice(["f32", "bf16"])}
    if op == "lists":
        dim = _log_int(rng, 96, 1024)
        nlist = _log_int(rng, 16, 4096)
        nprobe = min(_log_int(rng, 1, 64), max(1, nlist // 4))
        nq = max(1, min(_log_int(rng, 1, 4096), 65536 // nprobe, 24 * nlist // nprobe))
        mean = max(4, min(_log_int(rng, 24, 1000), 1000000 // nlist))
        return {"op": op, "nq": nq, "nprobe": nprobe, "nlist": nlist, "mean": mean, "dim": dim,
                "rows": rng.choice(["e4m3", "bf16"]), "out": rng.choice(["f32", "bf16"])}
    nq = _log_int(rng, 1, 4096)
    n = max(16, min(_log_int(rng, 64, 1000003), 1024 * 100003 // nq))
    return {"op": op, "nq": nq, "n": n, "dtype": rng.choice(["f32", "bf16"]),
            "k": rng.choice([0, 1, 5, 10, 32, 100]), "given": rng.choice([0, 1, 4]),
            "scale": rng.choice([1.0, 20.0, 50.0, -20.0]), "ragged": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------
# inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _vectors(n, dim, g, dtype=torch.float32):
    """Unit-norm rows around a few means, the rows of bf16 tensors padded to 16 bytes."""
    x = torch.randn(n, dim, device="cuda", generator=g)
    means = torch.randn(64, dim, device="cuda", generator=g)
    which = torch.randint(0, 64, (n,), device="cuda", generator=g)
    for i in range(0, n, 131072):
        x[i:i + 131072].mul_(0.7).add_(means[which[i:i + 131072]])
        x[i:i + 131072] /= x[i:i + 131072].norm(dim=1, keepdim=True)
    if dtype == torch.float32:
        return x
    out = torch.zeros(n, -(-dim // 8) * 8, device="cuda", dtype=dtype)
    out[:, :dim] = x
    return out[:, :dim]


def _rows(n, dim, kind, g):
    """Rows as a user's program keeps them: bf16, or 8-bit codes with their scale bytes."""
    if kind == "bf16":
        return {"kind": kind, "dim": dim, "data": _vectors(n, dim, g, torch.bfloat16)}
    codes = torch.zeros(n, -(-dim // 16) * 16, device="cuda", dtype=torch.uint8)
    nblk = -(-dim // BLOCK)
    scales = torch.full((n, -(-nblk // 4) * 4), 127, device="cuda", dtype=torch.uint8)
    x = _vectors(n, dim, g)
    for i in range(0, n, 131072):
        c, s = _pack(x[i:i + 131072])
        codes[i:i + 131072, :dim] = c.view(torch.uint8)
        scales[i:i + 131072, :nblk] = s
    return {"kind": kind, "dim": dim, "data": codes, "scales": scales}


def _layout(case):
    """The index of a `lists` case: the lengths of its lists (up to twice the mean, some empty) and
    how often each is probed."""
    rng = np.random.default_rng(case["nlist"] * 7919 + case["mean"])
    length = np.minimum(rng.gamma(4.0, case["mean"] / 4.0, case["nlist"]), 2 * case["mean"])
    length = np.maximum(np.round(length), 0).astype(np.int64)
    length[rng.random(case["nlist"]) < 0.01] = 0
    length[0] = max(length[0], 1)
    weight = (1.0 + rng.permutation(case["nlist"])) ** -0.4
    return length, weight / weight.sum()


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    state = {"case": case}
    if op == "pack":
        dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        state["x"] = _vectors(case["n"], case["dim"], g, dtype)
    elif op == "scores":
        state["q"] = _rows(case["nq"], case["dim"], case["rows"], g)
        state["x"] = _rows(case["n"], case["dim"], case["rows"], g)
    elif op == "lists":
        length, weight = _layout(case)
        nq, nprobe = case["nq"], case["nprobe"]
        state["q"] = _rows(nq, case["dim"], case["rows"], g)
        state["x"] = _rows(int(length.sum()), case["dim"], case["rows"], g)
        list_len = torch.from_numpy(length).cuda()
        # which lists are probed goes by the case alone: every seed's scores have one shape
        fixed = _gen(case["nlist"] * 31 + nq)
        noise = torch.rand(nq, case["nlist"], device="cuda", generator=fixed)
        noise = noise.log_().neg_().log_().neg_()
        probes = (noise + torch.from_numpy(weight).cuda().log().float()).topk(nprobe, dim=1).indices
        del noise
        flat = probes.reshape(-1)
        size = list_len[flat]
        start = size.cumsum(0) - size  # the pair's place in its query's row of scores
        order = flat.sort(stable=True).indices
        count = torch.bincount(flat, minlength=case["nlist"])
        zero = torch.zeros(1, device="cuda", dtype=torch.int64)
        state["pair_off"] = torch.cat([zero, count.cumsum(0)])
        state["pair_row"] = (order // nprobe).to(torch.int32)
        state["list_off"] = list_len.cumsum(0) - list_len
        state["list_len"] = list_len.to(torch.int32)
        state["out_off"] = start[order].contiguous()
        state["total"] = int(size.sum())
        state["most_pairs"], state["most_rows"] = int(count.max()), int(length.max())
    else:
        nq, n = case["nq"], case["n"]
        dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        if case["ragged"]:
            size = torch.randint(max(1, n // 2), n + n // 2, (nq,), device="cuda", generator=g)
            size[torch.rand(nq, device="cuda", generator=g) < 0.02] = 0  # no list held a row
            state["row_off"] = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64),
                                          size.cumsum(0)])
            shape = (int(size.sum()),)
            state["most"] = max(1, int(size.max()))
        else:
            shape = (nq, n)
        # inner products of unit vectors: most near zero, a few near one
        s = torch.randn(shape, device="cuda", generator=g).mul_(0.06)
        s += torch.rand(shape, device="cuda", generator=g).pow_(24.0).mul_(0.8)
        dead = torch.rand(shape, device="cuda", generator=g) < 0.01  # removed rows
        s.masked_fill_(dead, -math.inf if case["scale"] > 0 else math.inf)
        if not case["ragged"] and nq > 2:
            s[nq // 2] = math.nan  # a query without a vector
        state["scores"] = s.to(dtype)
        if case["given"]:
            at = torch.randint(0, max(1, n // 2), (nq, case["given"]), device="cuda", generator=g)
            at[torch.rand(at.shape, device="cuda", generator=g) < 0.05] = -1  # none given
            state["given"] = at
    return state


# ---------------------------------------------------------------------------------------------
# the plain forms


def _power(e):
    """2^e as fp32, by its bits; -126 <= e <= 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _pack(x):
    """e4m3 codes and scale bytes of rows: a block's scale is the least power of two 2^e with
    |x| <= 448 * 2^e for its finite values, e >= -126, kept as e + 127."""
    n, dim = x.shape
    nblk = -(-dim // BLOCK)
    v = torch.nn.functional.pad(x.float(), (0, nblk * BLOCK - dim)).view(n, nblk, BLOCK)
    a = v.abs()
    top = torch.where(a < math.inf, a, 0.0).amax(2)
    frac, e = torch.frexp(top)  # top = frac * 2^e, frac in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(frac > 0.875, e - 8, e - 9)
    e = torch.where(top > 0, e, -126).clamp(min=-126)
    y = (v * _power(-e).unsqueeze(2)).clamp(-448.0, 448.0)
    codes = y.to(torch.float8_e4m3fn).view(n, nblk * BLOCK)[:, :dim]
    return codes, (e + 127).to(torch.uint8)


def _values(rows):
    """What rows stand for, as fp32."""
    if rows["kind"] == "bf16":
        return rows["data"].float()
    dim = rows["dim"]
    v = rows["data"][:, :dim].view(torch.float8_e4m3fn).float()
    scale = _power(rows["scales"].to(torch.int32) - 127)
    return v * scale.repeat_interleave(BLOCK, dim=1)[:, :dim]


def _kind(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _plain_lists(s):
    """Products of each list's queries and rows, padded to the largest list and the most queries,
    written to each pair's place."""
    q, x = _values(s["q"]), _values(s["x"])
    ngroup, npair = s["list_off"].numel(), s["pair_row"].numel()
    dev = q.device
    row = torch.arange(s["most_rows"], device=dev)
    slot = torch.arange(s["most_pairs"], device=dev)
    rows = (s["list_off"][:, None] + row).clamp(max=x.shape[0] - 1)
    pairs = (s["pair_off"][:-1, None] + slot).clamp(max=npair - 1)
    padded = torch.bmm(q[s["pair_row"].long()[pairs]], x[rows].transpose(1, 2))
    group = torch.repeat_interleave(torch.arange(ngroup, device=dev), s["pair_off"].diff(),
                                    output_size=npair)
    size = s["list_len"].long()[group]
    pair = torch.repeat_interleave(torch.arange(npair, device=dev), size, output_size=s["total"])
    j = torch.arange(s["total"], device=dev) - (size.cumsum(0) - size)[pair]
    value = padded[group[pair], pair - s["pair_off"][group[pair]], j]
    out = torch.empty(s["total"], device=dev, dtype=_kind(s["case"]["out"]))
    out[s["out_off"][pair] + j] = value.to(out.dtype)
    return out


def _plain_probs(s):
    case = s["case"]
    scores, scale, k = s["scores"].float(), case["scale"], case["k"]
    if case["ragged"]:
        at = s["row_off"][:-1, None] + torch.arange(s["most"], device=scores.device)
        there = at < s["row_off"][1:, None]
        scores = torch.where(there, scores[at.clamp(max=scores.numel() - 1)], math.nan)
    logit = scores * scale
    held = logit > -math.inf  # false for NaN
    logit = torch.where(held, logit, -math.inf)
    top = logit.amax(1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp(logit - top)
    total = p.sum(1)
    lse = top[:, 0] + total.log()
    spread = (p * torch.where(held, logit - top, 0.0)).sum(1)
    entropy = torch.where(total > 0, total.log() - spread / total, 0.0)
    out = {"logsumexp": lse, "entropy": entropy}
    if case["given"]:
        at = s["given"]
        inside = (at >= 0) & (at < scores.shape[1])
        there = logit.gather(1, torch.where(inside, at, 0))
        inside &= there > -math.inf
        out["given"] = torch.where(inside, there - lse[:, None], -math.inf)
    if k:
        # whole-number keys, so that equal scores are taken by the lowest index
        bits = ((scores if scale > 0 else -scores) + 0.0).view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
        place = torch.arange(scores.shape[1], device=scores.device)
        key = torch.where(held, key + (0x7FFFFFFF - place), torch.iinfo(torch.int64).min)
        if key.shape[1] < k:
            key = torch.nn.functional.pad(key, (0, k - key.shape[1]),
                                          value=torch.iinfo(torch.int64).min)
        best = key.topk(k, dim=1).values
        there = best > torch.iinfo(torch.int64).min
        index = torch.where(there, 0x7FFFFFFF - (best & 0x7FFFFFFF), -1)
        value = logit.gather(1, index.clamp(min=0))
        out["top_index"] = index
        out["top"] = torch.where(there, value - lse[:, None], -math.inf)
    return out


# ---------------------------------------------------------------------------------------------
# the framework's operators

_engines = {}


def _engine():
    """The program's engine, made once."""
    if "engine" not in _engines:
        from m3_memory_b200 import cabi

        _engines["engine"] = cabi.Engine()
    return _engines["engine"]


def _own_rows(rows):
    if rows["kind"] == "bf16":
        return rows["data"]
    from m3_memory_b200 import row_scores

    return row_scores.PackedRows(rows["data"], rows["scales"], rows["dim"])


def _own_run(s):
    from m3_memory_b200 import row_scores

    case, eng = s["case"], _engine()
    if case["op"] == "pack":
        packed = row_scores.pack_rows(eng, s["x"])
        return {"codes": packed.codes[:, :case["dim"]].view(torch.float8_e4m3fn),
                "scales": packed.scales[:, :-(-case["dim"] // BLOCK)]}
    if case["op"] == "scores":
        return row_scores.row_scores(eng, _own_rows(s["q"]), _own_rows(s["x"]),
                                     out_dtype=_kind(case["out"]))
    if case["op"] == "lists":
        out = torch.empty(s["total"], device="cuda", dtype=_kind(case["out"]))
        return row_scores.list_scores(eng, _own_rows(s["q"]), _own_rows(s["x"]), s["list_off"],
                                      s["list_len"], s["pair_off"], s["out_off"], out,
                                      pair_row=s["pair_row"])
    got = row_scores.score_probs(eng, s["scores"], scale=case["scale"], k=case["k"],
                                 given=s.get("given"), row_off=s.get("row_off"))
    out = {"logsumexp": got.logsumexp, "entropy": got.entropy}
    if case["given"]:
        out["given"] = got.given
    if case["k"]:
        out["top_index"], out["top"] = got.top_index, got.top
    return out


def run(state):
    if own:
        return _own_run(state)
    case = state["case"]
    if case["op"] == "pack":
        codes, scales = _pack(state["x"])
        return {"codes": codes, "scales": scales}
    if case["op"] == "scores":
        return torch.mm(_values(state["q"]), _values(state["x"]).t()).to(_kind(case["out"]))
    if case["op"] == "lists":
        return _plain_lists(state)
    return _plain_probs(state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits


def work(case):
    size = {"f32": 4, "bf16": 2, "e4m3": 1}
    op = case["op"]
    if op == "pack":
        nblk = -(-case["dim"] // BLOCK)
        return {"bytes": case["n"] * (case["dim"] * (size[case["dtype"]] + 1) + nblk),
                "flops": 3 * case["n"] * case["dim"]}
    if op in ("scores", "lists"):
        row = case["dim"] * size[case["rows"]]
        if case["rows"] == "e4m3":
            row += -(-case["dim"] // BLOCK)
    if op == "scores":
        pairs = case["nq"] * case["n"]
        return {"bytes": (case["nq"] + case["n"]) * row + pairs * size[case["out"]],
                "flops": 2 * pairs * case["dim"]}
    if op == "lists":
        length, weight = _layout(case)
        share = np.minimum(1.0, case["nprobe"] * weight)  # of the queries that probe each list
        share *= case["nprobe"] / share.sum()
        read = float(((1 - (1 - np.minimum(share, 1.0)) ** case["nq"]) * length).sum())
        pairs = float((case["nq"] * share * length).sum())
        offsets = case["nlist"] * 20 + case["nq"] * case["nprobe"] * 12
        return {"bytes": int((read + case["nq"]) * row + pairs * size[case["out"]] + offsets),
                "flops": int(2 * pairs * case["dim"])}
    entries = case["nq"] * case["n"]
    out = case["nq"] * (8 + 12 * case["given"] + 12 * case["k"] + (8 if case["ragged"] else 0))
    return {"bytes": entries * size[case["dtype"]] + out, "flops": 6 * entries}


def _exact_power(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_rows(rows):
    if rows["kind"] == "bf16":
        return rows["data"].double()
    n, dim = rows["data"].shape[0], rows["dim"]
    table = np.array([(-1.0) ** (c >> 7) * (math.nan if (c & 127) == 127 else (c & 7) * 2.0 ** -9
                      if not (c >> 3) & 15 else (8 + (c & 7)) * 2.0 ** (((c >> 3) & 15) - 10))
                      for c in range(256)])
    v = torch.from_numpy(table).cuda()[rows["data"].int()][:, :dim]
    for b in range(-(-dim // BLOCK)):
        scale = _exact_power(rows["scales"][:, b].long() - 127)
        v[:, b * BLOCK:(b + 1) * BLOCK] *= scale.view(n, 1)
    return v


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "pack":
        x = s["x"].double()
        out = torch.empty_like(x)
        scales = []
        for b in range(0, case["dim"], BLOCK):
            v = x[:, b:b + BLOCK]
            top = v.abs().amax(1).clamp(min=2.0 ** -140)
            e = torch.ceil(torch.log2(top / 448.0))
            e = torch.where(top > 448.0 * _exact_power(e), e + 1, e)  # where log2 was rounded
            e = torch.where(top <= 448.0 * _exact_power(e - 1), e - 1, e).clamp(min=-126.0)
            scales.append(e + 127.0)
            y = v * _exact_power(-e).view(-1, 1)
            # three bits after the leading one, and none below 2^-9
            step = y.abs().clamp(min=2.0 ** -6).view(torch.int64) >> 52
            step = _exact_power(step - 1026)
            out[:, b:b + BLOCK] = torch.round(y / step) * step
        return {"codes": out, "scales": torch.stack(scales, 1)}
    if op == "scores":
        q, x = _exact_rows(s["q"]), _exact_rows(s["x"])
        return torch.cat([q @ x[i:i + 65536].t() for i in range(0, x.shape[0], 65536)], 1)
    if op == "lists":
        q, x = _exact_rows(s["q"]), _exact_rows(s["x"])
        out = torch.full((s["total"],), math.nan, device="cuda", dtype=torch.float64)
        pair_off, list_off = s["pair_off"].tolist(), s["list_off"].tolist()
        for g, n in enumerate(s["list_len"].tolist()):
            a, b = pair_off[g], pair_off[g + 1]
            if a < b and n:
                value = q[s["pair_row"][a:b].long()] @ x[list_off[g]:list_off[g] + n].t()
                out[s["out_off"][a:b, None] + torch.arange(n, device="cuda")] = value
        return out
    nq, k, got = case["nq"], case["k"], {"logsumexp": [], "entropy": []}
    many = max(1, 30000000 // max(1, case["n"]))
    for i in range(0, nq, many):
        if case["ragged"]:
            off = s["row_off"][i:i + many + 1].tolist()
            part = torch.nn.utils.rnn.pad_sequence(
                [s["scores"][a:b].double() for a, b in zip(off, off[1:])], batch_first=True,
                padding_value=math.nan)
        else:
            part = s["scores"][i:i + many].double()
        logit = (part * case["scale"]).nan_to_num(nan=-math.inf, neginf=-math.inf)
        if not logit.shape[1]:
            logit = torch.full((logit.shape[0], 1), -math.inf, device="cuda", dtype=torch.float64)
        lse = torch.logsumexp(logit, 1)
        logp = torch.where(logit > -math.inf, logit - lse[:, None], -math.inf)
        got["logsumexp"].append(lse)
        got["entropy"].append(torch.where(logp > -math.inf, -logp.exp() * logp, 0.0).sum(1))
        if case["given"]:
            at = s["given"][i:i + many]
            inside = (at >= 0) & (at < logp.shape[1])
            there = logp.gather(1, torch.where(inside, at, 0))
            got.setdefault("given", []).append(torch.where(inside, there, -math.inf))
        if k:
            best = logp.topk(min(k, logp.shape[1]), dim=1).values
            best = torch.nn.functional.pad(best, (0, k - best.shape[1]), value=-math.inf)
            got.setdefault("top", []).append(best)
    out = {name: torch.cat(v) for name, v in got.items()}
    if k:
        out["top_index"] = None
    return out

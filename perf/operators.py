"""Rows kept at four bits (e2m1 values, one power-of-two scale per 32 elements): written, read back, and multiplied
with queries.  Each operator here in elementary torch operations, and as the calls of ``rag_amd.QuantizedIndex``.

A store is given in its natural layout: ``codes`` uint8 [n, 16 * ceil(dim / 32)], element 2j in the low and 2j + 1 in
the high four bits of byte j; ``scales`` uint8 [n, ceil(dim / 32)], byte b meaning 2^(b - 127) and 255 NaN."""
import math

import numpy as np
import torch

if not torch.cuda.is_available():
    DEVICE = "cpu"
else:
    DEVICE = "cuda"

own = False

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def _groups_of(dim):
    return (dim + 31) // 32


def _row_bytes(dim):
    return _groups_of(dim) * 17


def listed():
    return [
        # one new chunk's embedding replaces an old one: latency
        {"name": "write_one_768_bf16", "op": "write", "n": 1, "table": 100_000, "dim": 768, "type": "bf16", "scatter": True},
        # ingest of a whole collection as the encoder hands it over
        {"name": "write_block_100k_384_fp32", "op": "write", "n": 100_000, "table": 100_000, "dim": 384, "type": "fp32", "scatter": False},
        # a batch of updates at scattered positions, some of them named twice, some padding (position -1)
        {"name": "write_scatter_40k_1024_fp16", "op": "write", "n": 40_000, "table": 65_536, "dim": 1024, "type": "fp16", "scatter": True},
        # the 200 candidates of a search fetched for diversification, unfilled slots among them
        {"name": "read_200_768_fp32", "op": "read", "n": 200, "table": 1_000_000, "dim": 768, "type": "fp32"},
        # a large share of a store read back in any order, for a half-precision consumer
        {"name": "read_131071_1024_bf16", "op": "read", "n": 131_071, "table": 262_144, "dim": 1024, "type": "bf16"},
        # one query over a small collection: latency
        {"name": "scores_1x100k_384_fp32", "op": "scores", "nq": 1, "n": 100_000, "dim": 384, "type": "fp32"},
        # odd sizes: neither the rows nor the dimension fill a tile
        {"name": "scores_3x33333_100_fp32", "op": "scores", "nq": 3, "n": 33_333, "dim": 100, "type": "fp32"},
        # one query over a store far larger than any cache
        {"name": "scores_1x4M_768_fp32", "op": "scores", "nq": 1, "n": 4_000_000, "dim": 768, "type": "fp32"},
        # a serving batch over a large store
        {"name": "scores_16x1M_1024_bf16", "op": "scores", "nq": 16, "n": 1_000_000, "dim": 1024, "type": "bf16"},
        # a large batch: bound by arithmetic and by the scores it writes
        {"name": "scores_256x200k_768_fp32", "op": "scores", "nq": 256, "n": 200_000, "dim": 768, "type": "fp32"},
        # three formulations of a question against each of 100 documents of uneven length
        {"name": "grouped_100docs_3q_384_fp32", "op": "grouped", "groups": 100, "rows": 700, "queries": 3, "shared": True, "sizes": 11, "dim": 384, "type": "fp32"},
        # a batch sorted by inverted list: uneven lists, uneven numbers of queries, some lists without any
        {"name": "grouped_512lists_1024_bf16", "op": "grouped", "groups": 512, "rows": 400, "queries": 8, "shared": False, "sizes": 12, "dim": 1024, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "scores", "scores", "grouped"])
    dim = _log(rng, 32, 2048) if rng.random() < 0.5 else 32 * _log(rng, 1, 64)
    kind = rng.choice(["fp32", "bf16", "fp16"])
    room = 150_000_000
    if op == "write":
        n = _log(rng, 1, max(2, min(200_000, room // (2 * dim))))
        scatter = rng.random() < 0.6
        return {"op": op, "n": n, "table": n + _log(rng, 1, n + 1) if scatter else n, "dim": dim, "type": kind, "scatter": scatter}
    if op == "read":
        n = _log(rng, 1, max(2, min(200_000, room // dim)))
        return {"op": op, "n": n, "table": max(16, _log(rng, max(1, n // 2), 2 * n)), "dim": dim, "type": kind}
    if op == "scores":
        nq = _log(rng, 1, 300)
        most = min(2_000_000, 3_000_000_000 // dim, 60_000_000 // nq, 40_000_000_000 // (dim * nq))
        return {"op": op, "nq": nq, "n": _log(rng, 1, max(2, most)), "dim": dim, "type": kind}
    shared = rng.random() < 0.5
    groups = _log(rng, 1, 400)
    queries = rng.randint(1, 4) if shared else _log(rng, 1, 24)
    rows = _log(rng, 1, max(2, min(1500, 150_000 // groups, 100_000_000 // (groups * dim))))
    return {"op": op, "groups": groups, "rows": rows, "queries": queries, "shared": shared, "sizes": rng.randrange(1 << 30), "dim": dim, "type": kind}


# ---------------------------------------------------------------------- inputs
def _vectors(gen, n, dim, dtype=torch.float32):
    """Embedding-like rows of about unit length: uneven spread over the dimensions."""
    x = torch.randn((n, dim), generator=gen, device=DEVICE, dtype=torch.float32)
    spread = torch.exp(0.4 * torch.randn((dim,), generator=gen, device=DEVICE, dtype=torch.float32))
    return (x * (spread / math.sqrt(dim))).to(dtype)


def _store(gen, n, dim):
    """A store of quantised embeddings, made a part at a time."""
    codes = torch.empty((n, 16 * _groups_of(dim)), dtype=torch.uint8, device=DEVICE)
    scales = torch.empty((n, _groups_of(dim)), dtype=torch.uint8, device=DEVICE)
    part = max(1, 200_000_000 // dim)
    for at in range(0, n, part):
        c, s = _quantise(_vectors(gen, min(part, n - at), dim))
        codes[at:at + part], scales[at:at + part] = c, s
    return codes, scales


def _group_sizes(case):
    """Uneven group sizes, [groups, 4]: queries [begin, end) and rows [begin, end) of every group."""
    r = np.random.RandomState(case["sizes"])
    g = case["groups"]
    rows = r.randint(0, 2 * case["rows"] + 1, g)
    if case["shared"]:
        q_begin, q_end = np.zeros(g, np.int64), np.full(g, case["queries"], np.int64)
    else:
        counts = r.randint(0, 2 * case["queries"] + 1, g)
        counts[r.rand(g) < 0.1] = 0
        q_end = np.cumsum(counts).astype(np.int64)
        q_begin = q_end - counts
    row_end = np.cumsum(rows).astype(np.int64)
    if int(rows.sum()) == 0:
        row_end[-1] = 1
    row_begin = np.concatenate([[0], row_end[:-1]]).astype(np.int64)
    return np.stack([q_begin, q_end, row_begin, row_end], 1)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    op, dim, dtype = case["op"], case["dim"], TYPES[case["type"]]
    state = {"case": case}
    if op == "grouped":
        groups = _group_sizes(case)
        n = int(groups[:, 3].max())
        state["groups"] = groups
        state["q"] = _vectors(gen, max(1, int(groups[:, 1].max())), dim, dtype)
    elif op == "scores":
        n = case["n"]
        state["q"] = _vectors(gen, case["nq"], dim, dtype)
    else:
        n = case["table"]
    codes, scales = _store(gen, n, dim)
    if op == "write":
        state["x"] = _vectors(gen, case["n"], dim, dtype)
        if case["scatter"]:
            rows = torch.randint(0, n, (case["n"],), generator=gen, device=DEVICE)
            pad = torch.rand((case["n"],), generator=gen, device=DEVICE) < (0.05 if case["n"] > 16 else 0.0)
            state["rows"] = torch.where(pad, torch.full_like(rows, -1), rows)
        else:
            state["rows"] = torch.arange(n, device=DEVICE)
        state["back"] = torch.arange(n, device=DEVICE) if case["n"] > 16 else state["rows"]
    if op == "read":
        rows = torch.randint(0, n, (case["n"],), generator=gen, device=DEVICE)
        pad = torch.rand((case["n"],), generator=gen, device=DEVICE) < 0.02
        state["rows"] = torch.where(pad, torch.full_like(rows, -1), rows)
    if own:
        from rag_amd import QuantizedIndex
        state["index"] = QuantizedIndex.from_packed(codes, scales, dim, metric="ip")
        if op == "grouped" and case["shared"]:
            state["plan"] = state["index"].plan_groups(state["groups"], state["q"].shape[0], dtype)   # the documents stay the same from question to question
    else:
        state["codes"], state["scales"] = codes, scales
    return state


# ----------------------------------------------------------------- plain forms
def _power(e):
    """2^e in 32 bits, exactly, for whole e from -126 to 127 (128: infinity)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x):
    """x [n, dim] -> (codes, scales): the formulas, in 32 bits (every step of them is exact there)."""
    n, dim = x.shape
    g = _groups_of(dim)
    x = torch.nn.functional.pad(x.float(), (0, 32 * g - dim)).view(n, g, 32)
    most = x.abs().amax(2)
    mantissa, exponent = torch.frexp(most)
    scale = torch.where(most > 0, exponent - 3 + (mantissa > 0.875), torch.full_like(exponent, -126)).clamp(-126, 125)
    bad = ~torch.isfinite(most)
    half = torch.div(scale, 2, rounding_mode="floor")                # 2^-scale as two factors that are normal numbers
    v = x.abs() * _power(-half)[:, :, None] * _power(half - scale)[:, :, None]
    code = ((v > 0.25).byte() + (v >= 0.75).byte() + (v > 1.25).byte() + (v >= 1.75).byte() + (v > 2.5).byte()
            + (v >= 3.5).byte() + (v > 5.0).byte() + 8 * torch.signbit(x).byte()).view(n, 32 * g)
    return code[:, 0::2] | (code[:, 1::2] << 4), torch.where(bad, torch.full_like(scale, 128), scale).add(127).to(torch.uint8)


def _values(codes, scales, dim):
    """The 32-bit values that codes and scales stand for, [n, dim]."""
    n = codes.shape[0]
    table = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    pairs = torch.stack([table.repeat(16), table.repeat_interleave(16)], 1)
    v = pairs[codes.int()].view(n, scales.shape[1], 32)
    factor = torch.where(scales == 0, 2.0 ** -127, _power(scales.int() - 127))
    factor = torch.where(scales == 255, math.nan, factor)
    return (v * factor[:, :, None]).view(n, -1)[:, :dim]


def _read(codes, scales, dim, rows, dtype):
    inside = (rows >= 0) & (rows < codes.shape[0])
    at = torch.where(inside, rows, torch.zeros_like(rows))
    return torch.where(inside[:, None], _values(codes[at], scales[at], dim), torch.zeros((), device=codes.device)).to(dtype)


def _pairs(groups):
    """For every score of every group, in order: which query and which row."""
    g = torch.from_numpy(groups).to(DEVICE)
    nq, rows = g[:, 1] - g[:, 0], g[:, 3] - g[:, 2]
    many = nq * rows
    which = torch.repeat_interleave(torch.arange(len(groups), device=DEVICE), many)
    at = torch.arange(which.numel(), device=DEVICE) - (torch.cumsum(many, 0) - many)[which]
    return g[which, 0] + at // rows[which], g[which, 2] + at % rows[which]


def run(state):
    case = state["case"]
    op, dim, dtype = case["op"], case["dim"], TYPES[case["type"]]
    if own:
        index = state["index"]
        if op == "write":
            index.write(state["rows"] if case["scatter"] else 0, state["x"])
            return index.reconstruct(state["back"], dtype=dtype)
        if op == "read":
            return index.reconstruct(state["rows"], dtype=dtype)
        if op == "scores":
            return index.scores(state["q"])
        return index.scores_grouped(state["q"], state["plan"] if case["shared"] else state["groups"])
    codes, scales = state["codes"], state["scales"]
    if op == "write":
        rows, count = state["rows"], state["rows"].numel()
        new_codes, new_scales = _quantise(state["x"])
        last = torch.full((codes.shape[0],), -1, dtype=torch.int64, device=DEVICE)      # of the rows meant for one position the last
        inside = torch.nonzero((rows >= 0) & (rows < codes.shape[0])).view(-1)
        last.scatter_reduce_(0, rows[inside], torch.arange(count, device=DEVICE)[inside], "amax")
        at = last[rows[inside]]
        codes[rows[inside]], scales[rows[inside]] = new_codes[at], new_scales[at]
        return _read(codes, scales, dim, state["back"], dtype)
    if op == "read":
        return _read(codes, scales, dim, state["rows"], dtype)
    s = torch.matmul(state["q"].float(), _values(codes, scales, dim).t())
    if op == "scores":
        return s
    qi, ri = _pairs(state["groups"])
    return s[qi, ri]


# ----------------------------------------------------------------------- work
def work(case):
    op, dim, size = case["op"], case["dim"], SIZE[case["type"]]
    if op == "write":
        back = case["table"] if case["n"] > 16 else case["n"]
        return {"bytes": case["n"] * (dim * size + _row_bytes(dim) + 8) + back * (dim * size + _row_bytes(dim) + 8), "flops": 0}
    if op == "read":
        return {"bytes": case["n"] * (_row_bytes(dim) + dim * size + 8), "flops": 0}
    if op == "scores":
        nq, n = case["nq"], case["n"]
        return {"bytes": n * _row_bytes(dim) + nq * dim * size + 4 * nq * n, "flops": 2 * nq * n * dim}
    groups = _group_sizes(case)
    queries, rows = groups[:, 1] - groups[:, 0], groups[:, 3] - groups[:, 2]
    scores, used = int((queries * rows).sum()), int(rows[queries > 0].sum())
    return {"bytes": used * _row_bytes(dim) + int(groups[:, 1].max()) * dim * size + 4 * scores, "flops": 2 * scores * dim}


# -------------------------------------------------------- the definitions, in 64 bits
def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_rows(x):
    """What rows of x read back as: the nearest grid value, found by trying all of them."""
    n, dim = x.shape
    g = _groups_of(dim)
    full = torch.zeros((n, g * 32), dtype=torch.float64, device=x.device)
    full[:, :dim] = x.double()
    full = full.view(n * g, 32)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    odd = torch.arange(8, device=x.device) % 2
    out = torch.empty_like(full)
    for at in range(0, n * g, 500_000):
        part = full[at:at + 500_000]
        a = part.abs().max(1).values
        f = (a.view(torch.int64) >> 52) - 1023                       # the exponent bits: floor(log2(a))
        unit = _power64((f - 2 + ((a / _power64(f)) > 1.75).long()).clamp(-126, 125))
        far = ((part.abs() / unit[:, None])[:, :, None] - grid).abs()
        nearest = far.min(2).values
        # of the nearest ones (two at a tie) the even code
        pick = torch.where(far == nearest[:, :, None], odd, 2).argmin(2)
        out[at:at + 500_000] = torch.copysign(grid[pick], part) * unit[:, None]
    return out.view(n, g * 32)[:, :dim]


def _exact_values(codes, scales, dim):
    n = codes.shape[0]
    c = torch.empty((n, codes.shape[1] * 2), dtype=torch.uint8, device=codes.device)
    c[:, 0::2] = codes % 16
    c[:, 1::2] = torch.div(codes, 16, rounding_mode="floor")
    e, m = ((c % 8) // 2).double(), (c % 2).double()
    v = torch.where(e == 0, m / 2, (1 + m / 2) * _power64(e - 1)) * torch.where(c >= 8, -1.0, 1.0)
    return (v.view(n, -1, 32) * _power64(scales.long() - 127)[:, :, None]).reshape(n, -1)[:, :dim]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    op, dim = case["op"], case["dim"]
    codes, scales = state["codes"], state["scales"]
    if op == "read" or op == "write":
        if op == "write":
            table = _exact_values(codes, scales, dim)
            new = _exact_rows(state["x"])
            where = {int(r): i for i, r in enumerate(state["rows"].tolist()) if 0 <= r < codes.shape[0]}
            if where:
                table[torch.tensor(list(where.keys()), device=DEVICE)] = new[torch.tensor(list(where.values()), device=DEVICE)]
            rows = state["back"]
        else:
            rows = state["rows"]
            table = _exact_values(codes, scales, dim)
        out = table[rows.clamp(min=0)]
        out[rows < 0] = 0
        return out
    q = state["q"].double()
    part = max(1, 400_000_000 // dim)
    if op == "scores":
        return torch.cat([q @ _exact_values(codes[at:at + part], scales[at:at + part], dim).T for at in range(0, codes.shape[0], part)], 1)
    parts = [(q[a:b] @ _exact_values(codes[c:d], scales[c:d], dim).T).reshape(-1) for a, b, c, d in state["groups"].tolist()]
    return torch.cat(parts)

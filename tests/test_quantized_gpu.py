"""rag_amd.QuantizedIndex: rows kept at four bits, against oracle/mx4.py (float64)."""
import numpy as np
import pytest

from oracle import mx4

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]


def _t(name):
    import torch
    return getattr(torch, name)


def _rows(rng, n, dim, dtype="float32", scale=1.0):
    """CUDA rows of the type, and the same values in float64."""
    import torch
    x = rng.standard_normal((n, dim)) * np.exp(0.5 * rng.standard_normal(dim)) * scale
    t = torch.from_numpy(x.astype(np.float32)).to(_t(dtype))
    return t.cuda(), t.double().numpy()


def _index(rng, n, dim, metric="ip"):
    import torch
    from rag_amd import QuantizedIndex
    codes, scales = mx4.quantise(rng.standard_normal((n, dim)).astype(np.float32) * np.exp2(rng.integers(-3, 4, (n, 1))))
    index = QuantizedIndex.from_packed(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), dim, metric=metric)
    return index, mx4.values(codes, scales, dim)


def _same_packed(index, want):
    codes, scales = index.packed()
    assert np.array_equal(scales.cpu().numpy(), want[1])
    assert np.array_equal(codes.cpu().numpy(), want[0])


# ------------------------------------------------------------------------------------------------ writing, reading
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim", [(1, 1), (3, 31), (5, 32), (7, 33), (64, 100), (65, 128), (1, 384), (130, 385), (257, 768), (33, 1000),
                                   (40, 1024), (9, 2047), (3, 8192)])
def test_rows_are_quantised_as_they_are_added(n, dim, dtype):
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(n * 10007 + dim)
    x, x64 = _rows(rng, n, dim, dtype)
    index = QuantizedIndex(dim, metric="ip")
    index.add(x[: n // 2])
    index.add(x[n // 2:])
    assert len(index) == n
    _same_packed(index, mx4.quantise(x64))


def test_special_values_are_quantised_as_documented():
    """Zero groups, ties, values past the largest code, the ends of the fp32 range, NaN and infinities."""
    import torch
    from rag_amd import QuantizedIndex
    rows = []
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], np.float32)
    for s in (-126, -125, -60, -1, 0, 7, 100, 124):
        rows.append(np.concatenate([ties * np.float32(2.0) ** s, -ties * np.float32(2.0) ** s, np.zeros(16, np.float32)]))
        rows.append(np.nextafter(rows[-1], np.float32(np.inf)).astype(np.float32))
        rows.append(np.nextafter(rows[-2], np.float32(-np.inf)).astype(np.float32))
    for a in (7.0, np.nextafter(np.float32(7.0), np.float32(8.0)), 8.0, 3.4e38, np.float32(np.finfo(np.float32).max), 1e-38, 1.2e-38, 1e-45,
              -0.0, 3.0e-39):
        r = np.zeros(32, np.float32)
        r[::3] = a
        r[1::3] = -np.float32(a) / 3
        rows.append(r)
    for bad in (np.nan, np.inf, -np.inf):
        r = np.ones(32, np.float32)
        r[17] = bad
        rows.append(r)
    x = np.stack(rows)
    x = np.concatenate([x, x[::-1], np.ones((len(x), 3), np.float32)], 1)          # a bad group leaves its neighbours alone
    index = QuantizedIndex(x.shape[1], metric="ip")
    index.add(torch.from_numpy(x).cuda())
    want = mx4.quantise(x)
    _same_packed(index, want)
    got = index.reconstruct(np.arange(len(x)))
    assert np.array_equal(got.astype(np.float64), mx4.values(*want, x.shape[1]), equal_nan=True)


@pytest.mark.parametrize("dim", [100, 768])
def test_rows_that_lie_apart_and_unaligned_ones(dim):
    import torch
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(dim)
    big = torch.from_numpy(rng.standard_normal((50, dim + 9)).astype(np.float32)).cuda()
    for view in (big[:, :dim], big[:, 3:3 + dim], big[::2, 1:1 + dim], big[:, :dim].half()[:, :], big.bfloat16()[:, 5:5 + dim],
                 big[:, :dim].t().contiguous().t(), big[:1, 4:4 + dim].expand(6, dim)):
        index = QuantizedIndex(dim, metric="ip")
        index.add(view)
        _same_packed(index, mx4.quantise(view.cpu().double().numpy()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [33, 768])
def test_cosine_rows_are_normalised_first(dim, dtype):
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(dim)
    x, x64 = _rows(rng, 200, dim, dtype, scale=30.0)
    x[7] = 0
    x64[7] = 0
    index = QuantizedIndex(dim)
    index.add(x)
    # a factor on a rounding border could differ in its last bit: at most one of the 200 rows may
    codes, scales = index.packed()
    want = mx4.quantise(mx4.normalise(x64.astype(np.float32)))
    differ = (codes.cpu().numpy() != want[0]).any(1) | (scales.cpu().numpy() != want[1]).any(1)
    assert differ.sum() <= 1 and not differ[7]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,count,dim", [(1, 1, 40), (50, 1, 384), (40, 100, 100), (3000, 2000, 768), (300, 5000, 96), (20, 64, 8192)])
def test_scattered_write_keeps_the_last_of_a_position_and_leaves_the_rest(n, count, dim, dtype):
    import torch
    rng = np.random.default_rng(n + count)
    index, _ = _index(rng, n, dim)
    codes, scales = (t.cpu().numpy().copy() for t in index.packed())
    for again in range(2):
        x, x64 = _rows(rng, count, dim, dtype)
        at = rng.integers(-3, n + 3, count)
        if count > 1:
            at[1] = -2 ** 62
            at[0] = at[-1] = n - 1
        index.write(torch.from_numpy(at).cuda() if again else at, x)
        new = mx4.quantise(x64)
        for i, r in enumerate(at):
            if 0 <= r < n:
                codes[r], scales[r] = new[0][i], new[1][i]
        _same_packed(index, (codes, scales))
    x, x64 = _rows(rng, n, dim, dtype)                    # consecutive positions behind scattered ones
    index.write(0, x)
    _same_packed(index, mx4.quantise(x64))
    if n > 2:
        index.write(1, x[:1])
        new = mx4.quantise(np.concatenate([x64[:1], x64[:1], x64[2:]]))
        _same_packed(index, new)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim", [(1, 1), (77, 33), (50, 100), (300, 768), (10, 1001), (5, 8192)])
def test_rows_read_back(n, dim, dtype):
    import torch
    rng = np.random.default_rng(dim)
    index, v = _index(rng, n, dim)
    at = rng.integers(-2, n + 2, 3 * n + 5)
    got = index.reconstruct(torch.from_numpy(at).cuda(), dtype=_t(dtype))
    assert got.dtype == _t(dtype) and got.shape == (at.size, dim)
    want = np.where(((at >= 0) & (at < n))[:, None], v[np.clip(at, 0, n - 1)], 0.0)
    assert torch.equal(got.cpu(), torch.from_numpy(want).to(_t(dtype)))
    inside = at[(at >= 0) & (at < n)]
    assert np.array_equal(index.reconstruct(inside), v[inside].astype(np.float32))


@pytest.mark.parametrize("dim", [1, 7, 8, 9, 16, 17])
def test_many_short_rows(dim):
    """Rows of one or two units of eight elements, many to a workgroup."""
    import torch
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(dim)
    n = 70_000
    x, x64 = _rows(rng, n, dim)
    index = QuantizedIndex(dim, metric="ip")
    index.add(x)
    want = mx4.quantise(x64)
    _same_packed(index, want)
    v = mx4.values(*want, dim)
    at = rng.permutation(n)
    for name in TYPES:
        got = index.reconstruct(torch.from_numpy(at).cuda(), dtype=_t(name))
        assert torch.equal(got.cpu(), torch.from_numpy(v[at]).to(_t(name)))


@pytest.mark.parametrize("count", [2, 3, 255, 256, 257, 300])
def test_repeated_positions_in_short_and_long_writes(count):
    """Up to 256 positions a workgroup finds repeated ones itself, beyond that they are claimed first: one rule."""
    import torch
    rng = np.random.default_rng(count)
    index, _ = _index(rng, 40, 384)
    codes, scales = (t.cpu().numpy().copy() for t in index.packed())
    at = rng.integers(-1, 41, count)
    x, x64 = _rows(rng, count, 384)
    index.write(torch.from_numpy(at).cuda(), x)
    new = mx4.quantise(x64)
    for i, r in enumerate(at):
        if 0 <= r < 40:
            codes[r], scales[r] = new[0][i], new[1][i]
    _same_packed(index, (codes, scales))


def test_every_code_under_every_scale_reads_back():
    """All 16 codes with all 256 scale bytes, in the three types (fp16 overflows and underflows with one rounding)."""
    import torch
    from rag_amd import QuantizedIndex
    codes = np.tile(np.arange(16, dtype=np.uint8) * 17, (256, 1))
    codes[:, ::2] = (np.arange(8, dtype=np.uint8) * 2) | ((np.arange(8, dtype=np.uint8) * 2 + 1) << 4)
    scales = np.arange(256, dtype=np.uint8)[:, None]
    index = QuantizedIndex.from_packed(codes, scales, 32)
    v = mx4.values(codes, scales, 32)
    for name in TYPES:
        got = index.reconstruct(torch.arange(256, device="cuda"), dtype=_t(name)).cpu()
        want = torch.from_numpy(v).to(torch.float32).to(_t(name)) if name == "bfloat16" else torch.from_numpy(v).to(_t(name))
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want)), name
    again = index.packed()
    assert np.array_equal(again[0].cpu().numpy(), codes) and np.array_equal(again[1].cpu().numpy(), scales)


# ------------------------------------------------------------------------------------------------ products
def _check_scores(got, q64, v, dtype, inv=None):
    digits = 5 if dtype == "float32" else 4
    want, bound = mx4.scores(q64, v), mx4.score_bound(q64, v, digits)
    if inv is not None:        # the factor 1 / |q| is rounded to fp32, and its product with the score once more
        want, bound = want * inv[:, None], bound * inv[:, None] + np.abs(want * inv[:, None]) * 2.0 ** -23
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape
    bad = np.abs(got - want) > bound + np.abs(want) * 2.0 ** -24 + 1e-37
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - want).max()), np.argwhere(bad)[:4].tolist())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,n,dim", [
    (1, 1, 1), (1, 17, 33), (2, 16, 128), (3, 15, 100), (4, 100, 129), (5, 1000, 384), (6, 333, 640), (7, 513, 768), (8, 64, 896),
    (9, 777, 1024), (12, 65, 1100), (13, 1500, 384), (16, 70, 1536), (17, 129, 2048), (24, 500, 768), (25, 1027, 256), (31, 40, 8192),
    (33, 2000, 384), (64, 300, 1000), (70, 900, 768), (100, 64, 4096), (129, 333, 130), (300, 1111, 200), (1, 5000, 8192), (2, 20000, 64),
    (1, 70001, 96), (3, 3, 5000)])
def test_scores(nq, n, dim, dtype):
    rng = np.random.default_rng(nq * 31 + n + dim)
    index, v = _index(rng, n, dim)
    q, q64 = _rows(rng, nq, dim, dtype)
    got = index.scores(q).cpu().numpy()
    _check_scores(got, q64, v, dtype)
    # a score does not depend on what it is computed together with
    i = int(rng.integers(nq))
    assert np.array_equal(index.scores(q[i]).cpu().numpy()[0], got[i])
    b = int(rng.integers(n))
    e = int(rng.integers(b, n + 1))
    assert np.array_equal(index.scores(q, b, e).cpu().numpy(), got[:, b:e])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [31, 100, 257, 384, 500, 640, 768, 900, 1000, 1024, 1100, 1536, 2048, 4096, 8192])
def test_many_queries_against_many_rows(dim, dtype):
    """Rows enough for the kernels that take 8, 16 and 32 queries at a time, for every number of blocks: the scores are those that
    the kernels for few queries give the same rows, bit for bit."""
    import torch
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(dim)
    small, v = _index(rng, 256, dim)
    codes, scales = small.packed()
    at = torch.from_numpy(rng.integers(0, 256, 40_001)).cuda()
    index = QuantizedIndex.from_packed(codes[at], scales[at], dim)
    for nq, first in ((7, 0), (16, 0), (37, 0), (37, 1)):               # first 1: rows that start between the elements of a wide load
        wide, wide64 = _rows(rng, nq, dim + first, dtype)
        q, q64 = wide[:, first:], wide64[:, first:]
        part = torch.cat([small.scores(q[i:i + 1]) for i in range(nq)])
        _check_scores(part.cpu().numpy(), q64, v, dtype)
        assert torch.equal(index.scores(q), part[:, at]), (nq, first)


def test_the_average_error_of_a_score_is_that_of_fp32():
    """Root mean square: independent roundings of half a step at most, spread evenly (2^-24 / sqrt(3)) over 8 partial sums per
    block and 4 digit sums, of the sum of |products|; a plain fp32 product is allowed the same."""
    rng = np.random.default_rng(4)
    index, v = _index(rng, 4000, 768)
    for dtype in TYPES:
        q, q64 = _rows(rng, 20, 768, dtype)
        err = index.scores(q).cpu().numpy() - mx4.scores(q64, v)
        size = np.abs(q64) @ np.abs(v).T
        assert np.sqrt((err ** 2).mean()) <= 2.0 ** -24 / np.sqrt(3) * np.sqrt(8 * 6 + 4) * np.sqrt((size ** 2).mean()), dtype


@pytest.mark.parametrize("dtype", TYPES)
def test_cosine_scores(dtype):
    rng = np.random.default_rng(9)
    index, v = _index(rng, 600, 384, metric="cosine")
    for nq in (1, 4, 30):
        q, q64 = _rows(rng, nq, 384, dtype, scale=5.0)
        _check_scores(index.scores(q).cpu().numpy(), q64, v, dtype, inv=1 / np.sqrt((q64 ** 2).sum(1)))
    zero = index.scores(np.zeros((2, 384), np.float32))
    assert np.array_equal(zero, np.zeros((2, 600), np.float32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,n,dim", [(1, 3_500_003, 100), (3, 3_400_017, 128), (4, 1_900_001, 200), (8, 1_300_031, 384), (5, 800_050, 700),
                                      (16, 1_300_033, 350), (30, 700_063, 768), (2, 600_035, 1000), (9, 500_001, 1024), (1, 300_033, 2048),
                                      (7, 262_171, 2500), (20, 500_007, 1024), (3, 262_145, 4200)])
def test_scores_of_stores_beyond_the_caches(nq, n, dim, dtype):
    """Stores over 256 MiB take kernels of their own; their scores are those of any part of the store, which a smaller one holds."""
    rng = np.random.default_rng(nq + n + dim)
    small, v = _index(rng, 4099, dim)
    import torch
    from rag_amd import QuantizedIndex
    codes, scales = small.packed()
    at = torch.from_numpy(rng.integers(0, 4099, n)).cuda()
    index = QuantizedIndex.from_packed(codes[at], scales[at], dim)
    assert n * (index._code_bytes + index._scale_bytes) > 256 << 20
    q, q64 = _rows(rng, nq, dim, dtype)
    part = small.scores(q)
    _check_scores(part.cpu().numpy(), q64, v, dtype)
    assert torch.equal(index.scores(q), part[:, at])
    b = 1017                                                 # a range that begins inside a block of sixteen rows and ends inside one
    assert torch.equal(index.scores(q, b, n - 3), part[:, at[b:n - 3]])


def test_a_result_whose_rows_lie_far_apart():
    """Scores of several queries more than 2^31 bytes apart: through the C entry point with a long out_stride."""
    import ctypes as C
    import torch
    from rag_amd import _lib
    rng = np.random.default_rng(31)
    for dim, nq in ((96, 9), (300, 20)):
        index, _ = _index(rng, 3000, dim)
        for dtype in TYPES:
            q, _ = _rows(rng, nq, dim, dtype)
            want = index.scores(q)
            stride = 700_000_000
            out = torch.empty((nq - 1) * stride + 3000, dtype=torch.float32, device="cuda")
            _lib.check(_lib.lib.rag_mx4_scores_device(C.byref(index._st), 0, 3000, nq, q.data_ptr(), TYPES.index(dtype), dim, 0, out.data_ptr(),
                                                      stride, torch.cuda.current_stream().cuda_stream))
            for i in range(nq):
                assert torch.equal(out[i * stride: i * stride + 3000], want[i]), (dtype, i)
            del out


def test_queries_that_lie_apart_and_host_queries():
    import torch
    rng = np.random.default_rng(2)
    index, v = _index(rng, 300, 100)
    big = torch.from_numpy(rng.standard_normal((40, 120)).astype(np.float32)).cuda()
    for view, dtype in ((big[:, 1:101], "float32"), (big[::3, :100], "float32"), (big.half()[:, 7:107], "float16"),
                        (big.bfloat16()[5:6, :100], "bfloat16"), (big[:, :100].t().contiguous().t(), "float32"),
                        (big[:1, 2:102].expand(5, 100), "float32")):
        _check_scores(index.scores(view).cpu().numpy(), view.cpu().double().numpy(), v, dtype)
    q = rng.standard_normal((3, 100))
    got = index.scores(q)
    assert isinstance(got, np.ndarray) and got.dtype == np.float32
    assert np.array_equal(got, index.scores(torch.from_numpy(q.astype(np.float32)).cuda()).cpu().numpy())


def test_far_apart_magnitudes_inside_a_query():
    """Groups of very different size, elements far below their group's largest one, and queries near the ends of fp32."""
    import torch
    rng = np.random.default_rng(3)
    index, v = _index(rng, 200, 256)
    q = rng.standard_normal((6, 256)) * np.exp2(rng.integers(-30, 30, (6, 256)))
    q[1] = rng.standard_normal(256) * np.repeat(np.exp2(rng.integers(-40, 40, 8)), 32)
    q[2] = 0
    q[2, 255] = 1e-30
    q[3] = rng.standard_normal(256) * 1e30
    q[4] = rng.standard_normal(256) * 1e-28
    q[5, :128] = 0
    q = q.astype(np.float32)
    _check_scores(index.scores(torch.from_numpy(q).cuda()).cpu().numpy(), q.astype(np.float64), v, "float32")


def test_nan_and_infinities_stay_with_their_query_and_row():
    import torch
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(5)
    x = rng.standard_normal((100, 200)).astype(np.float32)
    x[13, 5] = np.nan
    x[40, 199] = np.inf
    index = QuantizedIndex(200, metric="ip")
    index.add(torch.from_numpy(x).cuda())
    for nq in (3, 9, 40):
        q = rng.standard_normal((nq, 200)).astype(np.float32)
        clean = index.scores(torch.from_numpy(q).cuda()).cpu().numpy()
        assert np.isnan(clean[:, [13, 40]]).all() and np.isfinite(np.delete(clean, [13, 40], 1)).all()
        for bad in (np.nan, np.inf, -np.inf):
            p = q.copy()
            p[1, 77] = bad
            got = index.scores(torch.from_numpy(p).cuda()).cpu().numpy()
            assert np.isnan(got[1]).all()
            assert np.array_equal(np.delete(got, 1, 0), np.delete(clean, 1, 0), equal_nan=True)
    D, I = index.search(torch.from_numpy(q).cuda(), 100)
    assert (I[:, :98] >= 0).all() and (I[:, 98:] == -1).all() and not ((I == 13) | (I == 40)).any()


def test_offsets_past_32_bits():
    """A store whose codes pass 4 GiB: its last rows are written, read and scored."""
    import torch
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(6)
    n, dim = 1_100_000, 8192
    index = QuantizedIndex(dim, metric="ip", capacity=n)
    index.add(torch.zeros((1, dim), device="cuda").expand(1, dim))
    index._n = n                                             # the rows between are zeros as allocated
    index._renew()
    x, x64 = _rows(rng, 70, dim, "bfloat16")
    index.write(n - 70, x)
    v = mx4.values(*mx4.quantise(x64), dim)
    assert np.array_equal(index.reconstruct(np.arange(n - 70, n)), v.astype(np.float32))
    q, q64 = _rows(rng, 2, dim, "bfloat16")
    got = index.scores(q, n - 100, n).cpu().numpy()
    assert (got[:, :30] == 0).all()
    _check_scores(got[:, 30:], q64, v, "bfloat16")
    D, I = index.search(q, 3)
    best = np.argsort(-got, axis=1, kind="stable")[:, :3] + n - 100
    assert np.array_equal(I.cpu().numpy(), best)


# ------------------------------------------------------------------------------------------------ groups
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ngroups,most_q,most_r,dim,nq", [(1, 1, 1, 32, 1), (7, 3, 50, 100, 9), (40, 4, 700, 384, 4), (100, 20, 60, 768, 300),
                                                          (13, 90, 300, 128, 200), (300, 2, 9, 1024, 40), (5, 33, 5000, 64, 64), (4, 9, 20, 8192, 9)])
def test_grouped_scores(ngroups, most_q, most_r, dim, nq, dtype):
    rng = np.random.default_rng(ngroups + dim)
    n = 6000 if dim <= 128 else 900
    index, v = _index(rng, n, dim)
    q, q64 = _rows(rng, nq, dim, dtype)
    a, b = rng.integers(0, nq, ngroups), rng.integers(0, n, ngroups)
    groups = np.stack([a, np.minimum(nq, a + rng.integers(0, most_q + 1, ngroups)), b, np.minimum(n, b + rng.integers(0, most_r + 1, ngroups))], 1)
    groups[0] = [0, min(nq, most_q), 0, min(n, most_r)]                # the widest one is there
    plan = index.plan_groups(groups, nq, q.dtype)
    got = index.scores_grouped(q, plan)
    assert got.numel() == plan.total == int(((groups[:, 1] - groups[:, 0]) * (groups[:, 3] - groups[:, 2])).sum())
    full = index.scores(q).cpu().numpy()
    for part, (q0, q1, r0, r1) in zip(plan.split(got), groups):
        assert np.array_equal(part.cpu().numpy(), full[q0:q1, r0:r1])
    assert np.array_equal(index.scores_grouped(q, groups).cpu().numpy(), got.cpu().numpy())
    _check_scores(full, q64, v, dtype)


def test_groups_of_very_many_scores():
    """More than 10^8 scores: pieces for the kernels that reach results any distance apart."""
    import torch
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(41)
    small, _ = _index(rng, 4096, 32)
    codes, scales = small.packed()
    n = 26_000_000
    at = torch.from_numpy(rng.integers(0, 4096, n)).cuda()
    index = QuantizedIndex.from_packed(codes[at], scales[at], 32)
    for dtype in TYPES:
        q, _ = _rows(rng, 11, 32, dtype)
        groups = np.array([[0, 3, 5, n - 7], [2, 11, 17, 3000], [10, 11, 0, n]])
        plan = index.plan_groups(groups, 11, q.dtype)
        assert plan.total > 100_000_000
        part = small.scores(q)
        for got, (q0, q1, r0, r1) in zip(plan.split(index.scores_grouped(q, plan)), groups):
            assert torch.equal(got, part[q0:q1][:, at[r0:r1]])


def test_rows_and_queries_of_extreme_norms():
    """COSINE: norms whose reciprocal, or whose square, fp32 does not hold."""
    import torch
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(42)
    x = rng.standard_normal((6, 64)).astype(np.float32)
    scale = np.array([1e-44, 1e-38, 1e-30, 1.0, 1e30, 1e37], np.float32)[:, None]
    index = QuantizedIndex(64)
    index.add(torch.from_numpy(x * scale).cuda())
    s = index.scores(torch.from_numpy(x * scale).cuda()).cpu().numpy()
    assert np.isfinite(s).all()
    D, I = index.search(torch.from_numpy(x[2:]).cuda(), 1)
    assert I[:, 0].tolist() == [2, 3, 4, 5]
    codes, scales = index.packed()
    unit = x.astype(np.float64) / np.linalg.norm(x.astype(np.float64), axis=1, keepdims=True)
    want = mx4.scores(unit, mx4.values(codes.cpu().numpy(), scales.cpu().numpy(), 64))
    # as in _check_scores, with the queries' norms rounded once more by the fp32 scaling of the inputs here
    assert (np.abs(s - want)[2:, 2:] <= (12 * 16 / 15 + 4) * 2.0 ** -24 * (np.abs(unit) @ np.abs(mx4.values(codes.cpu().numpy(), scales.cpu().numpy(), 64)).T)[2:, 2:]).all()


def test_pieces_that_do_not_fit_are_left_out():
    """Through the C entry point: pieces for other sizes write nothing, the others their scores."""
    import ctypes as C
    import torch
    from rag_amd import _lib
    rng = np.random.default_rng(21)
    index, _ = _index(rng, 200, 64)
    q, _ = _rows(rng, 3, 64)
    want = index.scores(q).cpu().numpy()
    item = np.dtype([("row0", "<i8"), ("at", "<i8"), ("rows", "<i4"), ("ld", "<i4"), ("q0", "<i4"), ("nq", "<i4")])
    good = [(0, 0, 50, 50, 0, 3), (150, 150, 50, 60, 1, 2)]
    bad = [(151, 0, 50, 50, 0, 1), (-1, 0, 5, 5, 0, 1), (0, 0, 0, 5, 0, 1), (0, -1, 5, 5, 0, 1), (0, 0, 5, 4, 0, 1), (0, 0, 5, 5, 1, 3),
           (0, 0, 5, 5, -1, 1), (0, 0, 5, 5, 0, 4), (0, 0, 5, 5, 0, 0), (0, 256, 5, 5, 0, 1), (0, 100, 50, 60, 0, 3), (2 ** 62, 0, 5, 5, 0, 1),
           (0, 2 ** 62, 5, 5, 0, 1)]
    items = torch.from_numpy(np.array(bad[:6] + good + bad[6:], dtype=item).view(np.uint8)).cuda()
    out = torch.full((260,), 7.0, device="cuda")
    _lib.check(_lib.lib.rag_mx4_scores_grouped_device(C.byref(index._st), 3, q.data_ptr(), 0, 64, 0, items.data_ptr(), len(good) + len(bad), 3,
                                                      out.data_ptr(), 260, torch.cuda.current_stream().cuda_stream))
    got = out.cpu().numpy()
    expect = np.full(260, 7.0, np.float32)
    expect[:150] = want[:, :50].reshape(-1)
    expect[150:200], expect[210:260] = want[1, 150:], want[2, 150:]
    assert np.array_equal(got, expect)


def test_many_plans_on_their_way_at_once():
    """More plans than there are blocks to copy them through, behind work that keeps the stream busy, and one too long for a block."""
    import torch
    rng = np.random.default_rng(23)
    index, _ = _index(rng, 9000, 64)
    q, _ = _rows(rng, 6, 64)
    full = index.scores(q)
    busy = torch.randn((4096, 4096), device="cuda")
    for _ in range(40):
        busy = busy @ busy * 1e-2
    results = []
    for i in range(150):
        a = rng.integers(0, 9000, 8)
        groups = np.stack([np.zeros(8, np.int64), rng.integers(1, 7, 8), a, np.minimum(9000, a + rng.integers(0, 400, 8))], 1)
        results.append((groups, index.scores_grouped(q, groups)))
    rows = np.arange(9000)
    long = np.stack([rows % 6, rows % 6 + 1, rows, rows + 1], 1)
    got = index.scores_grouped(q, long)
    for groups, r in results:
        want = torch.cat([full[b:e, c:d].reshape(-1) for b, e, c, d in groups.tolist()])
        assert torch.equal(r, want)
    at = torch.from_numpy(rows).cuda()
    assert torch.equal(got, full[at % 6, at])


def test_groups_are_planned_outside_of_a_capture():
    import torch
    rng = np.random.default_rng(22)
    index, _ = _index(rng, 64, 64)
    q, _ = _rows(rng, 2, 64)
    graph = torch.cuda.CUDAGraph()
    said = None
    with torch.cuda.graph(graph):
        out = index.scores(q)
        try:
            index.scores_grouped(q, [[0, 2, 0, 64]])
        except ValueError as e:
            said = str(e)
    assert "outside of a graph capture" in said
    graph.replay()
    assert torch.equal(out, index.scores(q))


def test_groups_that_leave_nothing():
    import torch
    rng = np.random.default_rng(8)
    index, _ = _index(rng, 50, 64)
    q, _ = _rows(rng, 4, 64)
    for groups in (np.zeros((0, 4), np.int64), [[0, 0, 0, 50], [4, 4, 3, 9]], [[0, 4, 7, 7]]):
        assert index.scores_grouped(q, groups).numel() == 0
    for bad in ([[0, 5, 0, 1]], [[2, 1, 0, 1]], [[-1, 1, 0, 1]], [[0, 1, 0, 51]], [[0, 1, 9, 8]], [[0, 1, -1, 8]]):
        with pytest.raises(Exception, match="inside"):
            index.scores_grouped(q, bad)
    with pytest.raises(ValueError):
        index.scores_grouped(q, [[0, 1, 2]])
    plan = index.plan_groups([[0, 4, 0, 50]], 4)
    for other in (q[:3], q.half()):
        with pytest.raises(ValueError):
            index.scores_grouped(other, plan)
    index.add(q)
    assert index.scores_grouped(q, plan).numel() == 200                # a longer index still holds the plan's rows
    short, _ = _index(rng, 49, 64)
    with pytest.raises(ValueError):
        short.scores_grouped(q, plan)


# ------------------------------------------------------------------------------------------------ search
def _best(scores, k, allowed=None, min_score=None):
    """The order rule: score descending, ties by position, empty slots behind."""
    nq, n = scores.shape
    D = np.full((nq, k), -np.finfo(np.float32).max, np.float32)
    I = np.full((nq, k), -1, np.int64)
    for i in range(nq):
        ok = ~np.isnan(scores[i])
        if allowed is not None:
            ok &= allowed
        if min_score is not None:
            ok &= scores[i] >= min_score
        rows = np.flatnonzero(ok)
        rows = rows[np.argsort(-scores[i][rows], kind="stable")][:k]
        D[i, :rows.size], I[i, :rows.size] = scores[i][rows], rows
    return D, I


@pytest.mark.parametrize("nq,n,dim,k", [(1, 1, 8, 1), (1, 5, 32, 10), (3, 1000, 100, 10), (2, 32768, 64, 100), (5, 32769, 32, 1024),
                                        (1, 200_001, 96, 10), (40, 70_000, 64, 65), (600, 140_000, 32, 3), (1, 300_000, 32, 1024)])
def test_search_gives_the_best_of_the_scores(nq, n, dim, k):
    import torch
    rng = np.random.default_rng(n)
    index, _ = _index(rng, n, dim)
    # many equal rows: equal scores
    codes, scales = index.packed()
    codes[n // 2:] = codes[: n - n // 2].clone()
    scales[n // 2:] = scales[: n - n // 2].clone()
    from rag_amd import QuantizedIndex
    index = QuantizedIndex.from_packed(codes, scales, dim)
    q, _ = _rows(rng, nq, dim)
    s = index.scores(q).cpu().numpy()
    D, I = index.search(q, k)
    wd, wi = _best(s, k)
    assert np.array_equal(I.cpu().numpy(), wi) and np.array_equal(D.cpu().numpy(), wd)
    mask = (rng.random(n) < 0.3).astype(np.uint8)
    if n > 4:
        index.set_active([0, n - 1, n // 2], False)
    on = np.ones(n, bool)
    if n > 4:
        on[[0, n - 1, n // 2]] = False
    limit = float(np.median(s))
    wd, wi = _best(s, k, on & (mask != 0), limit)
    for m in (mask, index.make_filter(mask), torch.from_numpy(mask).cuda()):
        D, I = index.search(q, k, min_score=limit, row_mask=m)
        assert np.array_equal(I.cpu().numpy(), wi) and np.array_equal(D.cpu().numpy(), wd)
    D, I = index.search(q, k, row_mask=np.zeros(n, np.uint8))
    assert (I == -1).all() and (D == -torch.finfo(torch.float32).max).all()
    wd, wi = _best(s, k, on)
    D, I = index.search(q.cpu().numpy(), k)
    assert np.array_equal(I, wi) and np.array_equal(D, wd)


def test_empty_index_and_empty_batches():
    import torch
    from rag_amd import QuantizedIndex
    index = QuantizedIndex(48)
    q = torch.ones((2, 48), device="cuda")
    D, I = index.search(q, 4)
    assert (I == -1).all() and index.last_path == "empty"
    assert index.scores(q).shape == (2, 0)
    assert index.scores(q[:0]).shape == (0, 0)
    assert torch.equal(index.reconstruct(torch.tensor([0, -1], device="cuda")), torch.zeros((2, 48), device="cuda"))
    index.write(np.array([0, 3]), q)                       # all positions outside
    index.add(q[:0])
    assert len(index) == 0
    index.add(q)
    assert index.search(q[:0], 4)[0].shape == (0, 4)
    index.write(np.zeros(0, np.int64), q[:0])
    assert index.reconstruct(np.zeros(0, np.int64)).shape == (0, 48)
    index.close()
    assert len(index) == 0


# ------------------------------------------------------------------------------------------------ streams, graphs, files
def test_captured_calls_replay_as_they_ran():
    """Write, read, products and search in one graph, replayed with new inputs and eager work between."""
    import torch
    rng = np.random.default_rng(11)
    index, _ = _index(rng, 40_000, 96)
    q, _ = _rows(rng, 5, 96)
    x, _ = _rows(rng, 64, 96)
    at = torch.from_numpy(rng.permutation(40_000)[:64]).cuda()
    plan = index.plan_groups([[0, 5, 10, 900], [2, 3, 39_000, 40_000]], 5)

    def work():
        index.write(at, x)
        D, I = index.search(q, 12)
        return index.reconstruct(at), index.scores(q, 5, 20_005), index.scores_grouped(q, plan), D, I
    work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for again in range(4):
        q.copy_(torch.from_numpy(rng.standard_normal((5, 96)).astype(np.float32)))
        x.copy_(torch.from_numpy(rng.standard_normal((64, 96)).astype(np.float32)))
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        want = work()
        for a, b in zip(got, want):
            assert torch.equal(a, b), again


def test_two_streams_and_two_searches_at_once():
    import torch
    rng = np.random.default_rng(12)
    index, _ = _index(rng, 100_000, 128)
    qs = [_rows(rng, 9, 128)[0] for _ in range(6)]
    want = [index.search(q, 20) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [None] * 6
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 3]):
            got[i] = index.search(q, 20)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_snapshot_round_trip(tmp_path):
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(13)
    index = QuantizedIndex(70)
    index.add(rng.standard_normal((90, 70)))
    index.set_active([3, 4], False)
    path = str(tmp_path / "rows.mx4")
    index.save(path)
    other = QuantizedIndex.load(path)
    assert other.metric == "cosine" and len(other) == 90
    _same_packed(other, tuple(t.cpu().numpy() for t in index.packed()))
    q = rng.standard_normal((2, 70))
    for a, b in zip(index.search(q, 100), other.search(q, 100)):
        assert np.array_equal(a, b)


def test_optimizer_over_four_bit_rows(tmp_path):
    """SearchConfig(quantization_config={"mx4": ...}): upsert, search, filters, soft delete, vectors and backup of a collection."""
    from rag_amd.schemas import IndexType, MetricType, SearchConfig, SearchError
    from rag_amd.search_optimizer import HipSearchOptimizer
    rng = np.random.default_rng(14)
    n, dim = 3000, 96
    x = rng.standard_normal((n, dim)).astype(np.float32)
    config = SearchConfig(dimension=dim, metric=MetricType.COSINE, collection_name="c", quantization_config={"mx4": {}})
    opt = HipSearchOptimizer(config)
    meta = [{"chunk_id": f"c{i}", "document_id": 1, "page": i % 5, "text": str(i)} for i in range(n)]
    opt.upsert(x, meta, list(range(n)))
    opt.upsert(x[:1] * -1, [dict(meta[7])], [7])                     # point 7 is replaced
    codes, scales = opt.index.packed()
    v = mx4.values(codes.cpu().numpy(), scales.cpu().numpy(), dim)
    q = rng.standard_normal((4, dim)).astype(np.float32)
    s = mx4.scores(q / np.linalg.norm(q.astype(np.float64), axis=1, keepdims=True), v)
    s[:, 7] = -np.inf

    def check(lists, allowed=None, limit=10):
        for i, hits in enumerate(lists):
            order = np.argsort(-(s[i] if allowed is None else np.where(allowed, s[i], -np.inf)))[:limit]
            assert [h[0].metadata["text"] for h in hits] == [str(r) if r < n else "7" for r in order]
            assert np.allclose([h[1] for h in hits], s[i][order], rtol=1e-6, atol=1e-7)
    check(opt.batch_search_sync(q, limit=10, min_score=-1.0))
    assert opt.index.last_path == "mx4"
    check([opt.search_sync(q[0].tolist(), limit=3, min_score=-1.0)], limit=3)
    pages = np.array([i % 5 == 2 for i in range(n)] + [True])
    for _ in range(2):                                               # the second time with the filter kept on the device
        check(opt.batch_search_sync(q, limit=10, min_score=-1.0, filters={"page": 2}), pages)
    assert opt.get_vector(5)["vector"] == v[5].astype(np.float32).tolist()
    path = str(tmp_path / "c.bin")
    opt.backup(path)
    again = HipSearchOptimizer.restore(path, config)
    check(again.batch_search_sync(q, limit=10, min_score=-1.0))
    opt.set_points_active(False)
    assert opt.search_sync(q[0].tolist(), limit=3, min_score=-1.0) == []
    for kwargs in ({"metric": MetricType.EUCLIDEAN}, {"index_type": IndexType.IVF}):
        with pytest.raises(SearchError):
            HipSearchOptimizer(SearchConfig(dimension=dim, collection_name="c", quantization_config={"mx4": {}}, **kwargs))


def test_refusals():
    import torch
    from rag_amd import QuantizedIndex, RagHipError
    for dim in (0, 8193, -1):
        with pytest.raises(RagHipError):
            QuantizedIndex(dim)
    for kwargs in ({"metric": "l2"}, {"device": 99}, {"device": -1}):
        with pytest.raises(ValueError):
            QuantizedIndex(32, **kwargs)
    index = QuantizedIndex(32, metric="ip")
    x = torch.ones((4, 32), device="cuda")
    index.add(x)
    for bad in (x[:, :31], x.double(), x.int(), torch.ones((2, 2, 32), device="cuda")):
        for call in (index.add, index.scores, lambda t: index.write(0, t), lambda t: index.search(t, 1)):
            with pytest.raises(ValueError):
                call(bad)
    for call in (lambda: index.write(1, x), lambda: index.write(-1, x[:1]), lambda: index.write(np.array([1, 2]), x),
                 lambda: index.write(torch.zeros(4, device="cuda"), x), lambda: index.reconstruct([4]), lambda: index.reconstruct([-1]),
                 lambda: index.scores(x, 2, 5), lambda: index.scores(x, 3, 2), lambda: index.scores(x, -1, 2),
                 lambda: index.search(x, 0), lambda: index.search(x, 1025), lambda: index.search(x, 2, row_mask=np.ones(3, np.uint8)),
                 lambda: index.set_active([4], False), lambda: index.make_filter(np.ones(5, np.uint8)),
                 lambda: index.reconstruct(torch.zeros(2, dtype=torch.int64, device="cuda"), dtype=torch.float64),
                 lambda: QuantizedIndex.from_packed(np.zeros((2, 16), np.uint8), np.zeros((2, 2), np.uint8), 32),
                 lambda: QuantizedIndex.from_packed(np.zeros((2, 16), np.uint8), np.zeros((3, 1), np.uint8), 32)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RagHipError):
        index.search(x, 1, min_score=float("nan"))
    assert len(index) == 4


# ------------------------------------------------------------------------------------------------ many rows, threads, streams
def test_more_rows_than_one_launch_takes():
    """Rows and positions beyond the workgroups of one launch (2^20 of 64 rows)."""
    import torch
    from rag_amd import QuantizedIndex
    n = 64 * 2 ** 20 + 77
    index = QuantizedIndex(1, metric="ip")
    grid = torch.tensor([0.0, 1.0, 1.5, 2.0, -3.0, 0.75, -1.0, 6.0], dtype=torch.float16, device="cuda")     # each is kept exactly in a group of its own
    x = grid[torch.randint(0, 8, (n, 1), device="cuda")]
    index.add(x)
    rows = torch.arange(n, device="cuda")
    assert torch.equal(index.reconstruct(rows, dtype=torch.float16), x)
    turn = rows.flip(0)
    index.write(turn, x)
    assert torch.equal(index.reconstruct(rows, dtype=torch.float16), x.flip(0))


def test_more_groups_and_queries_than_one_launch_takes():
    import torch
    rng = np.random.default_rng(51)
    index, _ = _index(rng, 700, 1)
    q, _ = _rows(rng, 5, 1)
    full = index.scores(q)
    many = 2 ** 20 + 9                                                  # a piece each
    a, b = rng.integers(0, 5, many), rng.integers(0, 700, many)
    got = index.scores_grouped(q, np.stack([a, a + 1, b, b + 1], 1))
    assert torch.equal(got, full[torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda()])
    at = torch.randint(0, 5, (2 ** 22 + 5,), device="cuda")
    assert torch.equal(index.scores(q[at], 7, 9), full[at][:, 7:9])


def test_an_index_of_too_many_rows_is_refused():
    import torch
    from rag_amd import QuantizedIndex
    index = QuantizedIndex(1, metric="ip")
    x = torch.ones((3, 1), dtype=torch.bfloat16, device="cuda")
    index.add(x)
    with pytest.raises(ValueError):
        index.add(x[:1].expand(2 ** 31 - 2, 1))
    assert len(index) == 3 and index.reconstruct([0, 1, 2]).ravel().tolist() == [1.0, 1.0, 1.0]


def test_what_grows_is_refused_inside_a_capture():
    import torch
    rng = np.random.default_rng(52)
    index, _ = _index(rng, 64, 64)
    q, _ = _rows(rng, 2, 64)
    x, _ = _rows(rng, 30, 64)
    said = []
    graph = torch.cuda.CUDAGraph()
    before = index.packed()
    with torch.cuda.graph(graph):
        out = index.scores(q)
        for call in (lambda: index.add(x), lambda: index.reserve(500), lambda: index.set_active([3], False)):
            try:
                call()
            except ValueError as e:
                said.append(str(e))
    assert len(said) == 3 and all("outside of a graph capture" in s for s in said)
    assert len(index) == 64 and torch.equal(index.packed()[0], before[0]) and torch.equal(index.packed()[1], before[1])
    for _ in range(3):
        graph.replay()
        assert torch.equal(out, index.scores(q))
    index.set_active([3], False)                                        # room for one more, but hidden rows
    index.reserve(128)
    graph = torch.cuda.CUDAGraph()
    refused = False
    with torch.cuda.graph(graph):
        out = index.scores(q)
        try:
            index.add(x)
        except ValueError:
            refused = True
    assert refused and len(index) == 64


def test_an_index_that_grows_on_another_stream():
    """Buffers that are given up while another stream still copies them are not handed out again before it has."""
    import torch
    rng = np.random.default_rng(53)
    index, _ = _index(rng, 60_000, 64)
    more, _ = _rows(rng, 40_000, 64)
    index.set_active(np.arange(0, 60_000, 3), False)
    index.add(more[:1])
    codes, scales = index.packed()
    size = index._codes.numel(), index._scales.numel()
    busy = torch.randn((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(60):
            busy = busy @ busy * 1e-2
        index.add(more)
        index.add(more)
    trash = [torch.full((s,), 255, dtype=torch.uint8, device="cuda") for s in size for _ in range(3)]
    trash += [torch.zeros((60_001,), dtype=torch.uint8, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    got = index.packed()
    assert torch.equal(got[0][:60_001], codes) and torch.equal(got[1][:60_001], scales)
    assert torch.equal(got[0][60_001:100_001], got[0][100_001:]) and len(index) == 140_001
    I = index.search(more[:2], 1000)[1]
    assert not ((I < 60_000) & (I % 3 == 0)).any() and (I >= 0).all()
    del trash


def test_a_plan_that_is_used_on_another_stream():
    import torch
    rng = np.random.default_rng(54)
    index, _ = _index(rng, 5000, 64)
    q, _ = _rows(rng, 4, 64)
    groups = [[0, 4, 0, 5000], [1, 3, 17, 900]]
    want = index.scores_grouped(q, groups)
    busy = torch.randn((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(first):
        for _ in range(40):
            busy = busy @ busy * 1e-2
        plan = index.plan_groups(groups, 4)
    with torch.cuda.stream(second):
        got = index.scores_grouped(q, plan)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    # made on a stream of its own, used on the default one
    with torch.cuda.stream(first):
        plan = index.plan_groups(groups, 4)
    assert torch.equal(index.scores_grouped(q, plan), want)
    plan = index.plan_groups(groups, 4)
    with torch.cuda.stream(second):
        got = index.scores_grouped(q, plan)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_threads_share_an_index():
    """Searches while another thread adds rows: every answer is that of the rows of some moment."""
    import threading
    import torch
    rng = np.random.default_rng(55)
    index, _ = _index(rng, 2000, 64)
    q, _ = _rows(rng, 3, 64)
    more, _ = _rows(rng, 500, 64)
    answers, wrong = [], []
    torch.cuda.synchronize()

    def ask():
        try:
            for _ in range(60):
                answers.append((len(index),) + index.search(q, 10) + (len(index),))
        except Exception as e:                              # told below
            wrong.append(e)

    def grow():
        try:
            for _ in range(60):
                index.add(more)
        except Exception as e:
            wrong.append(e)
    threads = [threading.Thread(target=f) for f in (ask, grow, ask)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and len(index) == 32_000 and len(answers) == 120
    full = index.scores(q)
    for least, D, I, most in answers:
        possible = []
        for n in range(least, most + 1, 500):
            top = torch.sort(full[:, :n], dim=1, descending=True, stable=True)
            possible.append(torch.equal(D, top.values[:, :10]) and torch.equal(I, top.indices[:, :10]))
        assert any(possible)


def test_a_snapshot_whose_soft_deletes_do_not_fit(tmp_path):
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(56)
    index, _ = _index(rng, 40, 64)
    index.set_active([1, 2], False)
    path = str(tmp_path / "rows")
    index.save(path)
    QuantizedIndex.load(path)
    with np.load(path) as f:
        kept = dict(f)
    for active in (kept["active"][:39], kept["active"].astype(np.int64), np.ones((40, 2), np.uint8)):
        with open(path, "wb") as f:
            np.savez(f, **dict(kept, active=active))
        with pytest.raises(ValueError):
            QuantizedIndex.load(path)

"""rag_amd.QuantizedIndex over the whole range of its operands: every bit of a query counts, whatever else its group holds,
and cosine scores hold for vectors of any norm.  Against float64; bounds come from the definition (oracle/mx4.py, product_bound)."""
import numpy as np
import pytest

from oracle import mx4

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]


def _t(name):
    import torch
    return getattr(torch, name)


def _unit_rows(dim, n):
    """An index whose row r holds a one at element r % dim and zeros elsewhere: its scores are the queries' elements."""
    import torch
    from rag_amd import QuantizedIndex
    g = (dim + 31) // 32
    codes = np.zeros((dim, 16 * g), np.uint8)
    i = np.arange(dim)
    codes[i, i // 2] = 2 << (4 * (i % 2))
    at = torch.arange(n, device="cuda") % dim
    return QuantizedIndex.from_packed(torch.from_numpy(codes).cuda()[at], torch.full((n, g), 127, dtype=torch.uint8, device="cuda"), dim), at


def _any_bits(rng, shape, dtype):
    """Finite values of the type with any exponent, subnormal ones and zeros among them, as a CUDA tensor."""
    import torch
    if dtype == "float32":
        bits = rng.integers(0, 2 ** 32, shape, dtype=np.uint32)
        x = torch.from_numpy(bits.view(np.int32)).view(torch.float32)
    else:
        bits = rng.integers(0, 2 ** 16, shape, dtype=np.uint16)
        x = torch.from_numpy(bits.view(np.int16)).view(_t(dtype))
    return torch.where(torch.isfinite(x), x, torch.ones_like(x)).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,n", [(32, 32), (45, 3000), (128, 128), (384, 40_001), (640, 700), (768, 30_000), (900, 2000), (1024, 20_000), (1500, 9000),
                                   (2048, 4096), (4096, 20_000), (5000, 10_001), (8192, 8192)])
def test_scores_of_unit_rows_are_the_queries(dim, n, dtype):
    """One product per score: it is the query's element, to the last bit, beside elements of any size."""
    import torch
    rng = np.random.default_rng(dim)
    index, at = _unit_rows(dim, n)
    for nq in (1, 2, 4, 5, 7, 16, 17, 33, 70):
        q = _any_bits(rng, (nq, dim), dtype)
        if nq > 1:
            q[0] = torch.tensor(1e-2, dtype=q.dtype)
            q[0, ::32] = torch.tensor(60000.0, dtype=q.dtype)
            q[1] = torch.randn(dim, device="cuda").to(q.dtype)
            q[1, 5::32] *= 3000
        got = index.scores(q)
        want = q.float()[:, at]
        assert torch.equal(got, want), (nq, int((got != want).sum()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,nq,n", [(32, 1, 500), (64, 3, 5000), (100, 8, 700), (384, 40, 20_000), (768, 5, 3000), (2048, 20, 2000)])
@pytest.mark.parametrize("outlier", [30.0, 300.0, 3000.0])
def test_outliers_that_meet_zeros(dim, nq, n, dtype, outlier):
    """One large element in every group of a query, where most rows hold a zero: the rest of the group counts in full."""
    import torch
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(dim + int(outlier))
    x = rng.standard_normal((min(n, 700), dim))
    place = rng.integers(0, 32, (dim + 31) // 32) + np.arange(0, dim, 32)
    place = place[place < dim]
    x[:, place] = np.where(rng.random((len(x), 1)) < 0.9, 0.0, x[:, place])
    codes, scales = mx4.quantise(x)
    v = mx4.values(codes, scales, dim)
    at = rng.integers(0, len(x), n)
    index = QuantizedIndex.from_packed(codes[at], scales[at], dim)
    q = rng.standard_normal((nq, dim))
    q[:, place] = outlier * np.where(rng.random((nq, len(place))) < 0.5, -1, 1)
    q = torch.from_numpy(q.astype(np.float32)).to(_t(dtype)).cuda()
    q64 = q.double().cpu().numpy()
    got = index.scores(q).cpu().numpy()
    bound = mx4.product_bound(q64, v)[:, at]
    assert (np.abs(got - mx4.scores(q64, v)[:, at]) <= bound).all()


def _spread(rng, dim, n):
    """A small index, and a long one of its rows in a random order."""
    import torch
    from rag_amd import QuantizedIndex
    codes, scales = mx4.quantise(rng.standard_normal((256, dim)) * np.exp2(rng.integers(-3, 4, (256, 1))))
    small = QuantizedIndex.from_packed(codes, scales, dim)
    codes, scales = small.packed()
    at = torch.from_numpy(rng.integers(0, 256, n)).cuda()
    return small, QuantizedIndex.from_packed(codes[at], scales[at], dim), at, mx4.values(codes.cpu().numpy(), scales.cpu().numpy(), dim)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [31, 100, 257, 640, 768, 900, 1300, 2048, 4096, 8192])
def test_large_batches_have_the_scores_of_single_queries(dim, dtype):
    """Batches and rows enough for the kernels that take the most queries at a time, with rows whole in LDS and in parts."""
    import torch
    rng = np.random.default_rng(dim + 7)
    small, index, at, v = _spread(rng, dim, 30_011)
    for nq, first in ((130, 0), (193, 1)):
        wide = torch.from_numpy((rng.standard_normal((nq, dim + first)) * np.exp2(rng.integers(-9, 9, (nq, dim + first)))).astype(np.float32))
        q = wide.to(_t(dtype)).cuda()[:, first:]
        part = torch.cat([small.scores(q[i:i + 1]) for i in range(nq)])
        q64 = q.double().cpu().numpy()
        assert (np.abs(part.cpu().numpy() - mx4.scores(q64, v)) <= mx4.product_bound(q64, v)).all()
        assert torch.equal(index.scores(q), part[:, at])
        assert torch.equal(index.scores(q, 5, 29_990), part[:, at[5:29_990]])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [96, 768, 1300])
def test_groups_of_many_queries_have_the_same_scores(dim, dtype):
    import torch
    rng = np.random.default_rng(dim + 8)
    small, index, at, _ = _spread(rng, dim, 20_000)
    q = torch.from_numpy(rng.standard_normal((150, dim)).astype(np.float32)).to(_t(dtype)).cuda()
    part = torch.cat([small.scores(q[i:i + 1]) for i in range(150)])
    for most in (7, 16, 33, 90):
        a, b = rng.integers(0, 140, 200), rng.integers(0, 19_000, 200)
        groups = np.stack([a, np.minimum(150, a + rng.integers(0, most + 1, 200)), b, np.minimum(20_000, b + rng.integers(0, 1500, 200))], 1)
        plan = index.plan_groups(groups, 150, q.dtype)
        for got, (q0, q1, r0, r1) in zip(plan.split(index.scores_grouped(q, plan)), groups):
            assert torch.equal(got, part[q0:q1][:, at[r0:r1]])


def test_queries_beyond_the_range_of_their_type_are_nan():
    """An infinity or a NaN makes every score of its query NaN, and of no other; the largest finite numbers are finite."""
    import torch
    rng = np.random.default_rng(3)
    for n in (64, 40_000):
        index, at = _unit_rows(96, n)
        for dtype in TYPES:
            for nq in (3, 40, 130):
                q = _any_bits(rng, (nq, 96), dtype)
                q[2] = torch.finfo(q.dtype).max * torch.from_numpy(rng.choice([-1.0, 1.0], 96)).cuda()
                clean = index.scores(q)
                assert torch.equal(clean, q.float()[:, at])
                for bad in (np.inf, -np.inf, np.nan):
                    p = q.clone()
                    p[1, 70] = bad
                    got = index.scores(p)
                    assert torch.isnan(got[1]).all()
                    got[1] = clean[1]
                    assert torch.equal(got, clean)


def _unit(q64):
    norm = np.linalg.norm(q64, axis=1, keepdims=True)
    return q64 / np.where(norm > 0, norm, 1.0)              # (zero vectors stay zero)


def _cosine_bound(unit64, v):
    """product_bound of the unit queries; the factor that makes them so is rounded once (2^-24), its product with the sum again."""
    return mx4.product_bound(unit64, v) + np.abs(mx4.scores(unit64, v)) * 2.0 ** -23 + 1e-37


NORMS = [1e-43, 1e-40, 1e-38, 1e-36, 1e-33, 1e-28, 1e-20, 1.0, 1e5, 1e20, 1e30, 1e37, 1.2e38]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,n", [(33, 700), (768, 40_000), (1100, 30_000), (8192, 500)])
def test_cosine_scores_of_queries_of_any_norm(dim, n, dtype):
    """Few and many queries, whose elements are of the type's smallest to its largest size."""
    import torch
    rng = np.random.default_rng(dim + 20)
    codes, scales = mx4.quantise(rng.standard_normal((256, dim)) / np.sqrt(dim))
    v = mx4.values(codes, scales, dim)
    at = rng.integers(0, 256, n)
    from rag_amd import QuantizedIndex
    index = QuantizedIndex.from_packed(codes[at], scales[at], dim, metric="cosine")
    info = torch.finfo(_t(dtype))
    for nq in (len(NORMS), 7 * len(NORMS)):
        q = rng.uniform(-1, 1, (nq, dim)) * np.tile(NORMS, nq // len(NORMS))[:, None]
        if dtype == "float16":
            q = q / np.abs(q).max(1, keepdims=True) * np.exp2(rng.uniform(-23, 15.9, (nq, 1)))
        q = torch.from_numpy(q.clip(-info.max, info.max).astype(np.float32)).to(_t(dtype)).cuda()
        q64 = q.double().cpu().numpy()
        unit = _unit(q64)
        got = index.scores(q).cpu().numpy()
        assert (np.abs(got - mx4.scores(unit, v)[:, at]) <= _cosine_bound(unit, v)[:, at]).all()
        one = index.scores(q[:1]).cpu().numpy()
        assert np.array_equal(one[0], got[0])
    D, I = index.search(q[:len(NORMS)], 3)
    assert np.array_equal(D.cpu().numpy(), np.sort(got[:len(NORMS)], 1)[:, ::-1][:, :3])


@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_cosine_scores(dtype):
    """Pieces that begin behind the first query, of queries of very different norms."""
    import torch
    rng = np.random.default_rng(21)
    small, index, at, v = _spread(rng, 384, 20_000)
    index = type(index).from_packed(*index.packed(), 384, metric="cosine")
    q = torch.from_numpy((rng.standard_normal((150, 384)) * np.exp2(rng.integers(-12, 12, (150, 1)))).astype(np.float32)).to(_t(dtype)).cuda()
    q64 = q.double().cpu().numpy()
    unit = _unit(q64)
    want, bound = mx4.scores(unit, v), _cosine_bound(unit, v)
    at = at.cpu().numpy()
    for most in (1, 5, 40):
        a, b = rng.integers(0, 140, 150), rng.integers(0, 19_000, 150)
        groups = np.stack([a, np.minimum(150, a + rng.integers(0, most + 1, 150)), b, np.minimum(20_000, b + rng.integers(0, 1500, 150))], 1)
        plan = index.plan_groups(groups, 150, q.dtype)
        for got, (q0, q1, r0, r1) in zip(plan.split(index.scores_grouped(q, plan)), groups):
            i = np.ix_(np.arange(q0, q1), at[r0:r1])
            assert (np.abs(got.cpu().numpy() - want[i]) <= bound[i]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [40, 768])
def test_cosine_rows_of_any_norm_are_stored_as_unit_rows(dim, dtype):
    """Appended, and written to named positions; a zero row stays zero."""
    import torch
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(dim + 30)
    info = torch.finfo(_t(dtype))
    x = rng.uniform(-1, 1, (len(NORMS) * 5, dim)) * np.repeat(NORMS, 5)[:, None]
    if dtype == "float16":
        x = x / np.abs(x).max(1, keepdims=True) * np.exp2(rng.uniform(-23, 15.9, (len(x), 1)))
    x[11] = 0
    x = torch.from_numpy(x.clip(-info.max, info.max).astype(np.float32)).to(_t(dtype))
    want = mx4.quantise(mx4.normalise(x.float().numpy()))
    index = QuantizedIndex(dim)
    index.add(x.cuda())
    for again in range(2):
        codes, scales = index.packed()
        # a factor on a rounding border could differ in its last bit: at most one of the rows may
        differ = (codes.cpu().numpy() != want[0]).any(1) | (scales.cpu().numpy() != want[1]).any(1)
        assert differ.sum() <= 1 and not differ[11]
        norm = np.linalg.norm(index.reconstruct(np.arange(len(x))), axis=1)
        there = (x.float() != 0).any(1).numpy()
        # a value is off by at most a third of itself or a quarter of its group's unit u, whose largest element is 3.5 u at least: the
        # error's norm is at most sqrt(1 / 9 + 32 / 16 / 3.5^2) = 0.53 of the row's
        assert (np.abs(norm[there] - 1) <= 0.53).all() and (norm[~there] == 0).all()
        index.write(torch.arange(len(x), device="cuda").flip(0), x.cuda().flip(0))


@pytest.mark.parametrize("dim", [1, 32, 33, 100, 128, 200, 520, 768])
def test_written_rows_are_those_that_were_packed_byte_for_byte(dim):
    """The store's own buffers: zeros behind a row's elements and groups however it came there."""
    import torch
    from rag_amd import QuantizedIndex
    rng = np.random.default_rng(dim)
    x = rng.standard_normal((50, dim)).astype(np.float32)
    packed = QuantizedIndex.from_packed(*mx4.quantise(x), dim)
    added = QuantizedIndex(dim, metric="ip", capacity=50)
    added.add(torch.from_numpy(x).cuda())
    for again in range(2):
        assert torch.equal(added._codes, packed._codes) and torch.equal(added._scales, packed._scales)
        added.write(np.arange(50), x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,n", [(96, 50), (768, 1003), (768, 40_013), (1300, 30_001), (8192, 300)])
def test_what_lies_around_the_scores_is_left_as_it_was(dim, n, dtype):
    """Through the C entry point: rows of results that lie apart, before and behind them other data."""
    import ctypes as C
    import torch
    from rag_amd import _lib
    rng = np.random.default_rng(n)
    _, index, _, _ = _spread(rng, dim, n)
    for nq in (1, 5, 9, 40, 131):
        q = torch.from_numpy(rng.standard_normal((nq, dim)).astype(np.float32)).to(_t(dtype)).cuda()
        for begin, end in ((0, n), (7, n - 3)):
            want = index.scores(q, begin, end)
            room = torch.full((nq + 2, end - begin + 37), 7.0, device="cuda")
            _lib.check(_lib.lib.rag_mx4_scores_device(C.byref(index._st), begin, end, nq, q.data_ptr(), TYPES.index(dtype), dim, 0, room[1:].data_ptr(),
                                                      room.shape[1], torch.cuda.current_stream().cuda_stream))
            assert torch.equal(room[1:-1, :end - begin], want)
            room[1:-1, :end - begin] = 7.0
            assert (room == 7.0).all()


@pytest.mark.parametrize("dtype,nq", [("float32", 16), ("float32", 20), ("float16", 20), ("bfloat16", 34), ("bfloat16", 20)])
def test_large_batches_whose_results_lie_far_apart(dtype, nq):
    """More than 2^31 bytes from query to query, for the kernels that take the most queries."""
    import ctypes as C
    import torch
    from rag_amd import _lib
    rng = np.random.default_rng(41)
    n, stride = 70_000, 600_000_000
    _, index, _, _ = _spread(rng, 96, n)
    q = torch.from_numpy(rng.standard_normal((nq, 96)).astype(np.float32)).to(_t(dtype)).cuda()
    want = index.scores(q)
    out = torch.empty((nq - 1) * stride + n, dtype=torch.float32, device="cuda")
    _lib.check(_lib.lib.rag_mx4_scores_device(C.byref(index._st), 0, n, nq, q.data_ptr(), TYPES.index(dtype), 96, 0, out.data_ptr(), stride,
                                              torch.cuda.current_stream().cuda_stream))
    for i in range(nq):
        assert torch.equal(out[i * stride: i * stride + n], want[i]), i


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [33, 520, 640, 1200, 5200, 5300, 8000])
def test_rows_with_values_beyond_the_range(dim, dtype):
    """Packed rows whose scale takes a value out of fp32: their scores are not finite, in single queries and batches alike; those of the
    rows around them are."""
    import torch
    from rag_amd import QuantizedIndex
    g = (dim + 31) // 32
    n = 3 * g
    codes, scales = np.full((n, 16 * g), 0x22, np.uint8), np.full((n, g), 100, np.uint8)      # ones, times 2^-27
    row = np.arange(n)
    codes.reshape(n, g, 16)[row, row // 3] = np.array([0x66, 0xEE, 0x22])[row % 3][:, None]
    scales[row, row // 3] = np.array([254, 254, 100])[row % 3]                                  # 4 times 2^127, its negative, or ones again
    index = QuantizedIndex.from_packed(codes, scales, dim)
    big = QuantizedIndex.from_packed(np.tile(codes, (1 + 40_000 // n, 1)), np.tile(scales, (1 + 40_000 // n, 1)), dim)
    for nq in (1, 5, 20, 130):
        q = torch.rand((nq, dim), device="cuda").add_(0.5).to(_t(dtype))
        got = torch.cat([index.scores(q[i:i + 1]) for i in range(nq)])
        assert torch.equal(torch.isfinite(got), torch.from_numpy(row % 3 == 2).cuda().expand(nq, n)), nq
        if dtype == "bfloat16":
            assert (got[:, 0::3] == np.inf).all() and (got[:, 1::3] == -np.inf).all()
        for other in (index.scores(q), big.scores(q)):
            want = got.repeat(1, other.shape[1] // n)
            assert torch.equal(torch.isnan(other), torch.isnan(want)) and torch.equal(torch.nan_to_num(other), torch.nan_to_num(want)), nq

"""The four-bit entry points without a GPU: layout, the cutting of ragged groups, and refused arguments."""
import ctypes as C

import numpy as np
import pytest

from rag_amd import _lib

lib = _lib.lib
ITEM = np.dtype([("row0", "<i8"), ("at", "<i8"), ("rows", "<i4"), ("ld", "<i4"), ("q0", "<i4"), ("nq", "<i4")])


def test_layout_and_scale_places():
    a, b = C.c_int64(), C.c_int64()
    for dim, codes, scales in ((1, 64, 16), (128, 64, 16), (129, 128, 16), (384, 192, 16), (768, 384, 32), (1024, 512, 32), (8192, 4096, 256)):
        assert lib.rag_mx4_layout(dim, C.byref(a), C.byref(b)) == 0 and (a.value, b.value) == (codes, scales)
    for dim in (0, -3, 8193):
        assert lib.rag_mx4_layout(dim, C.byref(a), C.byref(b)) == _lib.RAG_ERR_INVALID
    assert lib.rag_mx4_layout(8, None, C.byref(b)) == _lib.RAG_ERR_INVALID
    from rag_amd.quantized import _scale_places
    for groups in (1, 5, 16, 24, 33, 256):
        at = _scale_places(groups)
        assert len(set(at.tolist())) == groups and at.max() < (((groups + 3) // 4) + 3) // 4 * 16
        assert [(g // 16) * 16 + (g % 4) * 4 + (g // 4) % 4 for g in range(groups)] == at.tolist()


def _plan(groups, nq, n, dim=384, kind=0, room=100_000):
    g = np.ascontiguousarray(groups, np.int64).reshape(-1, 4)
    items = np.zeros(room, ITEM)
    begin = np.zeros(len(g), np.int64)
    count, total, widest = C.c_int64(-1), C.c_int64(-1), C.c_int32(-1)
    rc = lib.rag_mx4_plan_groups(dim, kind, nq, n, len(g), g.ctypes.data, room, items.ctypes.data, C.byref(count), begin.ctypes.data,
                                 C.byref(total), C.byref(widest))
    return rc, items, count.value, begin, total.value, widest.value


@pytest.mark.parametrize("seed", range(12))
def test_pieces_cover_every_score_of_every_group_once(seed):
    rng = np.random.default_rng(seed)
    dim, kind = int(rng.choice([32, 100, 384, 768, 2048, 8192])), int(rng.integers(0, 3))
    ng, nq, n = int(rng.integers(1, 40)), int(rng.integers(1, 200)), int(rng.integers(1, 5000))
    a, b = rng.integers(0, nq + 1, ng), rng.integers(0, n + 1, ng)
    groups = np.stack([a, np.minimum(nq, a + rng.integers(0, rng.integers(1, 60), ng)), b, np.minimum(n, b + rng.integers(0, 3000, ng))], 1)
    rc, items, count, begin, total, widest = _plan(groups, nq, n, dim, kind)
    assert rc == 0 and 0 <= count <= 100_000
    sizes = (groups[:, 1] - groups[:, 0]) * (groups[:, 3] - groups[:, 2])
    assert total == sizes.sum() and np.array_equal(begin, np.cumsum(sizes) - sizes)
    assert widest == max([int(n) for n in items[:count]["nq"]], default=0)
    want_q, want_r = np.full(total, -1), np.full(total, -1)
    for (q0, q1, r0, r1), o in zip(groups, begin):
        want_q[o:o + (q1 - q0) * (r1 - r0)] = np.repeat(np.arange(q0, q1), r1 - r0)
        want_r[o:o + (q1 - q0) * (r1 - r0)] = np.tile(np.arange(r0, r1), q1 - q0)
    got_q, got_r = np.full(total, -1), np.full(total, -1)
    for it in items[:count]:
        assert it["rows"] > 0 and 0 < it["nq"] <= 32
        for i in range(it["nq"]):
            at = it["at"] + i * it["ld"] + np.arange(it["rows"])
            assert (got_q[at] == -1).all()
            got_q[at], got_r[at] = it["q0"] + i, it["row0"] + np.arange(it["rows"])
    assert np.array_equal(got_q, want_q) and np.array_equal(got_r, want_r)
    # too little room: the number is told and nothing is written behind the room
    if count > 1:
        small = _plan(groups, nq, n, dim, kind, room=count - 1)
        assert small[0] == 0 and small[2] == count


def test_groups_outside_are_refused():
    for bad in ([0, 5, 0, 1], [2, 1, 0, 1], [-1, 1, 0, 1], [0, 1, 0, 51], [0, 1, 9, 8], [0, 1, -1, 8], [0, 2 ** 40, 0, 1]):
        rc, *_ = _plan([[0, 1, 0, 1], bad], 4, 50)
        assert rc == _lib.RAG_ERR_INVALID and "group 1" in _lib.last_error()
    assert _plan([[0, 1, 0, 1]], 4, 50, kind=3)[0] == _lib.RAG_ERR_INVALID
    assert _plan([[0, 1, 0, 1]], 4, 50, dim=0)[0] == _lib.RAG_ERR_INVALID
    assert _plan([[0, 1, 0, 1]], -1, 50)[0] == _lib.RAG_ERR_INVALID
    assert _plan(np.zeros((0, 4)), 4, 50)[:1] + _plan(np.zeros((0, 4)), 4, 50)[2:3] == (0, 0)


def test_arguments_are_refused_before_a_device_is_touched():
    """Every call here ends in a check on the host: the addresses are never followed."""
    p = 1 << 20                                                 # stands for device memory
    st = _lib.Mx4Store(p, p, 100, 384, 0)
    ref = C.byref(st)
    bad = _lib.RAG_ERR_INVALID

    def store(**kw):
        s = _lib.Mx4Store(p, p, 100, 384, 0)
        for k, v in kw.items():
            setattr(s, k, v)
        return C.byref(s)
    for s in (None, store(codes=None), store(scales=None), store(codes=p + 8), store(scales=p + 4), store(n=-1), store(n=2 ** 31), store(dim=0),
              store(dim=8193)):
        assert lib.rag_mx4_scores_device(s, 0, 10, 1, p, 0, 384, 0, p, 10, None) == bad
        assert lib.rag_mx4_read_device(s, p, 1, p, 0, None) == bad
        assert lib.rag_mx4_write_device(s, 0, None, None, 1, p, 0, 384, 0, None) == bad
        assert lib.rag_mx4_scores_grouped_device(s, 1, p, 0, 384, 0, p, 1, 1, p, 100, None) == bad
        assert lib.rag_mx4_search_device(s, 1, p, 0, 384, 0, 10, 0.0, None, None, p, p, p, 1 << 40, None) == bad
    for args in ((-1, 10, 1, p, 0, 384, 0, p, 10), (5, 4, 1, p, 0, 384, 0, p, 10), (0, 101, 1, p, 0, 384, 0, p, 101), (0, 10, -1, p, 0, 384, 0, p, 10),
                 (0, 10, 1, None, 0, 384, 0, p, 10), (0, 10, 1, p, 3, 384, 0, p, 10), (0, 10, 1, p, 0, 383, 0, p, 10), (0, 10, 1, p, 0, 384, 0, None, 10),
                 (0, 10, 1, p, 0, 384, 0, p, 9), (0, 10, 1, p + 2, 0, 384, 0, p, 10), (0, 10, 1, p + 1, 1, 384, 0, p, 10)):
        assert lib.rag_mx4_scores_device(ref, *args, None) == bad, args
    for args in ((-1, None, None, 1, p, 0, 384), (100, None, None, 1, p, 0, 384), (0, None, None, 101, p, 0, 384), (0, None, None, -1, p, 0, 384),
                 (0, None, None, 1, None, 0, 384), (0, None, None, 1, p, 0, 383), (0, None, None, 1, p, 7, 384), (0, p, None, 1, p, 0, 384),
                 (0, None, None, 1, p + 2, 0, 384), (2 ** 62, None, None, 2 ** 30, p, 0, 384)):
        assert lib.rag_mx4_write_device(ref, *args, 0, None) == bad, args
    for args in ((None, 1, p, 0), (p, 1, None, 0), (p, -1, p, 0), (p, 1, p, 5), (p, 1, p + 1, 1)):
        assert lib.rag_mx4_read_device(ref, *args, None) == bad, args
    for args in ((1, p, 0, 384, 0, p, -1, 1, p), (1, p, 0, 384, 0, None, 1, 1, p), (1, p, 0, 384, 0, p, 1, 1, None), (1, p, 0, 384, 0, p + 8, 1, 1, p),
                 (1, p, 0, 384, 0, p, 1, 0, p), (1, p, 0, 384, 0, p, 1, 2, p), (0, p, 0, 384, 0, p, 1, 1, p)):
        assert lib.rag_mx4_scores_grouped_device(ref, *args, 100, None) == bad, args
    for args in ((1, p, 0, 384, 0, 0, 0.0, None, None, p, p), (1, p, 0, 384, 0, 1025, 0.0, None, None, p, p),
                 (1, p, 0, 384, 0, 10, float("nan"), None, None, p, p), (1, p, 0, 384, 0, 10, 0.0, None, None, None, p)):
        assert lib.rag_mx4_search_device(ref, *args, p, 1 << 40, None) == bad, args
    for args in ((p, -1, p), (p, 1, None), (None, 1, p), (p, 1, p + 8)):
        assert lib.rag_mx4_upload_groups(*args, 0, None) == bad, args
    # nothing to do is no error
    assert lib.rag_mx4_upload_groups(None, 0, None, 0, None) == 0
    assert lib.rag_mx4_scores_device(ref, 5, 5, 1, p, 0, 384, 0, None, 0, None) == 0
    assert lib.rag_mx4_scores_device(ref, 0, 100, 0, None, 0, 0, 0, None, 100, None) == 0
    assert lib.rag_mx4_write_device(ref, 100, None, None, 0, None, 0, 384, 0, None) == 0
    assert lib.rag_mx4_read_device(ref, None, 0, None, 0, None) == 0
    assert lib.rag_mx4_scores_grouped_device(ref, 1, p, 0, 384, 0, None, 0, 0, None, 0, None) == 0
    assert lib.rag_mx4_search_workspace(100, 1, 0) == -1 and lib.rag_mx4_search_workspace(-1, 1, 1) == -1
    assert lib.rag_mx4_search_workspace(100, 1, 10) > 0


def test_unaligned_buffers_are_refused():
    p = 1 << 20
    ref = C.byref(_lib.Mx4Store(p, p, 100, 384, 0))
    bad = _lib.RAG_ERR_INVALID
    assert lib.rag_mx4_scores_device(ref, 0, 10, 1, p, 0, 384, 0, p + 2, 10, None) == bad
    assert lib.rag_mx4_scores_grouped_device(ref, 1, p, 0, 384, 0, p, 1, 1, p + 2, 100, None) == bad
    assert lib.rag_mx4_write_device(ref, 0, p + 4, p, 1, p, 0, 384, 0, None) == bad
    assert lib.rag_mx4_write_device(ref, 0, p, p + 2, 1, p, 0, 384, 0, None) == bad
    assert lib.rag_mx4_read_device(ref, p + 4, 1, p, 0, None) == bad
    assert lib.rag_mx4_search_device(ref, 1, p, 0, 384, 0, 10, 0.0, None, None, p + 2, p, p, 1 << 40, None) == bad
    assert lib.rag_mx4_search_device(ref, 1, p, 0, 384, 0, 10, 0.0, None, None, p, p + 4, p, 1 << 40, None) == bad


def test_more_pieces_than_a_plan_can_hold():
    rc, *_ = _plan([[0, 2 ** 30, 0, 2 ** 29]], 2 ** 30, 2 ** 29)
    assert rc == _lib.RAG_ERR_INVALID and "pieces" in _lib.last_error()
    # many pieces, no room: the number comes without a walk over them
    rc, items, count, _, total, widest = _plan([[0, 2 ** 10, 0, 2 ** 29]], 2 ** 10, 2 ** 29, kind=1, room=4)
    assert rc == 0 and count == 2 ** 7 * 2 ** 16 and total == 2 ** 39 and widest == 8 and not items["rows"].any()


def test_the_oracle_rounds_to_the_nearest_value():
    from oracle import mx4
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 70))
    codes, scales = mx4.quantise(x)
    v = mx4.values(codes, scales, 70)
    p = np.zeros((50, 96))
    p[:, :70] = x
    unit = np.repeat(np.exp2(scales.astype(float) - 127), 32, axis=1)[:, :70]
    grid = np.concatenate([mx4.TABLE, -mx4.TABLE])
    nearest = np.abs(x[:, :, None] / unit[:, :, None] - grid).min(2)
    assert np.allclose(np.abs(v - x) / unit, nearest, atol=1e-12)
    most = np.abs(p.reshape(50, 3, 32)).max(2) / np.exp2(scales.astype(float) - 127)
    assert (most <= 7.0).all() and (most > 3.5).all()


def test_quantised_index_needs_a_gpu():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    from rag_amd import QuantizedIndex, RagHipError
    with pytest.raises(RagHipError):
        QuantizedIndex(16)


def test_only_a_mapping_with_the_key_asks_for_four_bit_rows():
    """Any other quantization_config that is given keeps its meaning (a compressed copy that is searched first)."""
    from types import SimpleNamespace
    from rag_amd.schemas import SearchConfig
    from rag_amd.search_optimizer import _four_bit
    for given, want in (({"mx4": {}}, True), ({"mx4": None}, True), ({"scalar": {"type": "int8"}}, False), ({}, False), (None, False), (True, False),
                        (SimpleNamespace(scalar=1), False), ("mx4", False), (object(), False)):
        assert _four_bit(SearchConfig(dimension=8, quantization_config=given)) is want, given

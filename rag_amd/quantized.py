"""Vector index whose rows are kept at four bits: what the reference's ``quantization_config`` asks its server for
(vector_db/search_optimizer.py:51,130), without the originals beside it.

``QuantizedIndex`` has the method names of ``DeviceIndex`` (add, search, reconstruct, set_active, make_filter, save / load)
and two products of its own, ``scores`` and ``scores_grouped``.  A row takes 0.53 bytes per element -- four-bit values (e2m1)
with one power-of-two scale per 32 elements -- and every answer is exact for the rows as they are stored.  The buffers are
torch tensors; every device call runs on torch's current stream of the index's device, allocates through torch only, and may be
captured into a CUDA graph.  Calls that write the index and calls that use it are ordered by the caller's streams; host threads
may share an index.  A graph works on the buffers and the number of rows of its capture: what grows or hides rows for the first time
(``reserve``, ``add``, ``set_active``) is done before, and a graph from before a growth is captured anew.
"""
from __future__ import annotations

import ctypes as C
import threading
from typing import Optional, Tuple

import numpy as np
import torch

from . import _lib
from ._lib import check, lib
from .index import FLT_MAX, MAX_K, DeviceFilter, _device_mask_ptr, _is_torch_cuda, _ptr

MAX_ROWS = 2 ** 31 - 1


_TYPES = {torch.float32: _lib.MX4_F32, torch.bfloat16: _lib.MX4_BF16, torch.float16: _lib.MX4_F16}


def _type_of(dtype) -> int:
    kind = _TYPES.get(dtype)
    if kind is None:
        raise ValueError(f"expected float32, bfloat16 or float16, got {dtype}")
    return kind


def _capturing(device: int) -> bool:
    if torch.cuda.current_device() == device:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _outside_capture(device: int, what: str) -> None:
    if _capturing(device):
        raise ValueError(f"{what} outside of a graph capture")


class _Kept:
    """Device tensors that calls on several streams may use: a stream other than the one they were made on is made
    known to torch's allocator, so that their memory is not handed out again before that stream is done with them."""

    def __init__(self, device: int):
        self.device = device
        self._homes = []                                    # (tensor, the stream it was made on)

    def hold(self, *tensors) -> None:
        """From here on these; the ones that are new were made on the current stream."""
        raw = torch._C._cuda_getCurrentRawStream(self.device)
        known = {id(t): home for t, home in self._homes}
        self._homes = [(t, known.get(id(t), raw)) for t in tensors if t is not None]

    def stream(self) -> int:
        """The current stream, as the C ABI takes it, about to use the tensors."""
        raw = torch._C._cuda_getCurrentRawStream(self.device)
        for t, home in self._homes:
            if raw != home:
                t.record_stream(torch.cuda.current_stream(self.device))
        return raw


class GroupPlan:
    """Ragged groups of queries and rows, checked and cut into pieces for the device (``rag_mx4_plan_groups``).
    ``total``: scores of all groups; ``out_begin[g]``: where those of group g start; ``shapes[g]``: (queries, rows).
    Made outside of a graph capture; a graph that uses a plan needs it for as long as it is replayed."""

    def __init__(self, groups, nq: int, n: int, dim: int, dtype, device: int):
        g = np.ascontiguousarray(groups, dtype=np.int64)
        if g.size == 0:
            g = g.reshape(0, 4)
        if g.ndim != 2 or g.shape[1] != 4:
            raise ValueError("groups must be [n, 4]: query begin, query end, row begin, row end")
        _outside_capture(int(device), "groups are planned (pass a GroupPlan)")
        self.nq, self.n, self.dim, self.type, self.device = int(nq), int(n), int(dim), _type_of(dtype), int(device)
        self._groups = g = g.copy() if g is groups else g
        self.out_begin = np.empty(g.shape[0], dtype=np.int64)
        count, total, widest = C.c_int64(0), C.c_int64(0), C.c_int32(0)
        room = 2 * g.shape[0] + 64
        while True:
            staging = np.empty((room, _lib.MX4_ITEM_BYTES), dtype=np.uint8)
            check(lib.rag_mx4_plan_groups(self.dim, self.type, self.nq, self.n, g.shape[0], g.ctypes.data, room, staging.ctypes.data,
                                          C.byref(count), self.out_begin.ctypes.data, C.byref(total), C.byref(widest)))
            if count.value <= room:
                break
            room = count.value
        self.total, self.widest, self.n_items = total.value, widest.value, count.value
        self._kept = _Kept(self.device)
        self.items = torch.empty((self.n_items, _lib.MX4_ITEM_BYTES), dtype=torch.uint8, device=torch.device("cuda", self.device))
        self._kept.hold(self.items)
        self._made_on = self._kept.stream()
        self._behind = {self._made_on}                      # streams that come behind the upload
        if self.n_items:
            check(lib.rag_mx4_upload_groups(staging.ctypes.data, self.n_items, self.items.data_ptr(), self.device, self._made_on))

    def _use(self) -> None:
        """The current stream is about to read the pieces: behind their upload (a capture begins behind it by itself)."""
        raw = self._kept.stream()
        if raw not in self._behind and not _capturing(self.device):
            made_on = torch.cuda.ExternalStream(self._made_on, self.device) if self._made_on else torch.cuda.default_stream(self.device)
            torch.cuda.current_stream(self.device).wait_stream(made_on)
            self._behind.add(raw)

    @property
    def shapes(self):
        g = self._groups
        return np.stack([g[:, 1] - g[:, 0], g[:, 3] - g[:, 2]], 1)

    def split(self, scores):
        """The flat result of ``scores_grouped`` as one [queries, rows] view per group."""
        return [scores[b:b + q * r].view(q, r) for b, (q, r) in zip(self.out_begin.tolist(), self.shapes.tolist())]


class QuantizedIndex:
    """metric: 'ip' | 'cosine' (rows are divided by their norm when written, queries when scored)."""

    kind = "mx4"

    def __init__(self, dim: int, metric: str = "cosine", device: int = 0, capacity: int = 0):
        if metric not in ("ip", "dot", "cosine"):
            raise ValueError(f"unknown metric {metric!r}")
        self.dim, self.metric, self.device = int(dim), metric, int(device)
        code_bytes, scale_bytes = C.c_int64(0), C.c_int64(0)
        check(lib.rag_mx4_layout(self.dim, C.byref(code_bytes), C.byref(scale_bytes)))
        self._code_bytes, self._scale_bytes = int(code_bytes.value), int(scale_bytes.value)
        n = C.c_int(0)
        check(lib.rag_device_count(C.byref(n)))
        if not 0 <= self.device < n.value:
            raise ValueError(f"no device {self.device}")
        self._lock = threading.RLock()                      # the host side of a call: buffers and number of rows belong together
        self._kept = _Kept(self.device)
        self._dev = torch.device("cuda", self.device)
        self._normalize = 1 if metric == "cosine" else 0
        self._n = 0
        self._codes = self._scales = self._owner = self._active = None
        self.last_path = "none"
        self._renew()
        self.reserve(int(capacity))

    # ------------------------------------------------------------------ lifetime
    def close(self) -> None:
        with self._lock:
            self._n = 0
            self._codes = self._scales = self._owner = self._active = None
            self._renew()

    def __len__(self) -> int:
        return self._n

    @property
    def ntotal(self) -> int:
        return self._n

    def _renew(self) -> None:
        """After a change of the buffers or of the number of rows: what the C ABI is told about them."""
        self._st = _lib.Mx4Store()
        if self._codes is not None:
            self._st.codes, self._st.scales = self._codes.data_ptr(), self._scales.data_ptr()
        self._st.n, self._st.dim, self._st.device = self._n, self.dim, self.device
        self._st_ref = C.byref(self._st)
        self._kept.hold(self._codes, self._scales, self._owner, self._active)

    def reserve(self, nrows: int) -> None:
        """Room for ``nrows`` rows, so that adds up to there move nothing."""
        with self._lock:
            if nrows <= (0 if self._codes is None else self._codes.shape[0]):
                return
            _outside_capture(self.device, "an index grows")
            nrows = (nrows + 15) // 16 * 16                  # sixteen rows lie together
            dev = self._dev
            codes = torch.zeros((nrows, self._code_bytes), dtype=torch.uint8, device=dev)
            scales = torch.zeros((nrows, self._scale_bytes), dtype=torch.uint8, device=dev)
            owner = torch.zeros((nrows,), dtype=torch.int32, device=dev)
            if self._n:
                self._kept.stream()
                used = (self._n + 15) // 16 * 16
                codes[:used] = self._codes[:used]
                scales[:self._n] = self._scales[:self._n]
            self._codes, self._scales, self._owner = codes, scales, owner
            self._renew()

    # -------------------------------------------------------------------- ingest
    def _rows_in(self, x, what="rows"):
        """x as a device matrix [n, dim] whose rows may lie apart (inner stride 1): (x, n, elements from row to row, type)."""
        if isinstance(x, torch.Tensor) and x.is_cuda:
            if x.get_device() != self.device:
                raise ValueError("tensor is on another device than the index")
        else:
            x = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(self._dev)
        kind = _TYPES.get(x.dtype)
        if kind is None:
            raise ValueError(f"expected float32, bfloat16 or float16, got {x.dtype}")
        shape = x.shape
        if len(shape) == 1:
            x = x[None, :]
            shape = x.shape
        if len(shape) != 2 or shape[1] != self.dim:
            raise ValueError(f"expected {what} [n, {self.dim}], got {tuple(shape)}")
        if x.is_contiguous():
            return x, shape[0], self.dim, kind
        if x.stride(1) == 1 and x.stride(0) >= self.dim:
            return x, shape[0], x.stride(0), kind
        return x.contiguous(), shape[0], self.dim, kind

    def add(self, x) -> None:
        """Append rows (numpy, or a CUDA tensor in float32, bfloat16 or float16), quantised as they are written."""
        x, count, ld, kind = self._rows_in(x)
        if count == 0:
            return
        with self._lock:
            first = self._n
            if first + count > MAX_ROWS:
                raise ValueError(f"an index holds at most {MAX_ROWS} rows")
            have = 0 if self._codes is None else self._codes.shape[0]
            if first + count > have:
                self.reserve(min(max(first + count, have + have // 2), MAX_ROWS))
            if self._active is not None:
                _outside_capture(self.device, "rows are added to an index with hidden ones")
                self._kept.stream()
                self._active = torch.cat([self._active, torch.ones((count,), dtype=torch.uint8, device=self._dev)])
            self._n = first + count
            self._renew()
            self._write(first, None, count, x, ld, kind)

    def write(self, rows, x) -> None:
        """Replace rows.  ``rows``: the first of consecutive positions (int), or one position per row of ``x`` (numpy, or
        a CUDA int64 tensor); a position outside the index is skipped, of several rows for one position the last is kept."""
        x, count, ld, kind = self._rows_in(x)
        first, at = 0, None
        if isinstance(rows, (int, np.integer)):
            first = int(rows)
        else:
            at = self._positions(rows)
            if at.numel() != count:
                raise ValueError("one position per row")
        with self._lock:
            if at is None and not 0 <= first <= self._n - count:
                raise ValueError("the rows do not lie inside the index")
            self._write(first, at, count, x, ld, kind)

    def _positions(self, rows):
        if isinstance(rows, torch.Tensor) and rows.is_cuda:
            if rows.dtype != torch.int64 or rows.get_device() != self.device:
                raise ValueError("positions must be an int64 tensor on the index's device")
            return rows if rows.dim() == 1 and rows.is_contiguous() else rows.reshape(-1).contiguous()
        return torch.from_numpy(np.ascontiguousarray(rows, dtype=np.int64).reshape(-1)).to(self._dev)

    def _write(self, first, at, count, x, ld, kind):
        if count == 0 or self._n == 0:
            return
        check(lib.rag_mx4_write_device(self._st_ref, first, None if at is None else at.data_ptr(),
                                       None if at is None else self._owner.data_ptr(), count, x.data_ptr(), kind, ld,
                                       self._normalize, self._kept.stream()))

    @classmethod
    def from_packed(cls, codes, scales, dim: int, metric: str = "ip", device: Optional[int] = None) -> "QuantizedIndex":
        """An index over rows that are quantised already (a checkpoint in the MX layout).  ``codes`` uint8
        [n, 16 * ceil(dim / 32)]: element 2j in the low, 2j + 1 in the high half of byte j; ``scales`` uint8 [n, ceil(dim / 32)].
        Both are copied; elements behind ``dim`` are set to zero."""
        groups = (int(dim) + 31) // 32
        codes = codes if isinstance(codes, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(codes, dtype=np.uint8))
        scales = scales if isinstance(scales, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(scales, dtype=np.uint8))
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2 or scales.dim() != 2 \
                or codes.shape[0] != scales.shape[0] or codes.shape[1] != 16 * groups or scales.shape[1] != groups:
            raise ValueError(f"expected uint8 codes [n, {16 * groups}] and scales [n, {groups}]")
        if device is None:
            device = codes.device.index if codes.is_cuda else 0
        n = codes.shape[0]
        self = cls(dim, metric=metric, device=device, capacity=n)
        if n:
            dev = self._dev
            rows = torch.zeros((self._codes.shape[0], self._code_bytes), dtype=torch.uint8, device=dev)
            rows[:n, :16 * groups] = codes.to(dev)
            if self.dim % 32:
                rows[:, (self.dim + 1) // 2:] = 0
                if self.dim % 2:
                    rows[:, self.dim // 2] &= 15
            self._codes.view(-1, self._code_bytes // 64, 16, 64).copy_(rows.view(-1, 16, self._code_bytes // 64, 64).transpose(1, 2))
            self._scales[:n, torch.from_numpy(_scale_places(groups)).to(dev)] = scales.to(dev)
            self._n = n
            self._renew()
        return self

    def packed(self) -> Tuple[object, object]:
        """(codes, scales) of all rows as ``from_packed`` takes them, copied."""
        groups = (self.dim + 31) // 32
        with self._lock:
            if self._n == 0:
                dev = self._dev
                return (torch.empty((0, 16 * groups), dtype=torch.uint8, device=dev), torch.empty((0, groups), dtype=torch.uint8, device=dev))
            self._kept.stream()
            places = torch.from_numpy(_scale_places(groups)).to(self._codes.device)
            used = (self._n + 15) // 16 * 16
            rows = self._codes[:used].view(-1, self._code_bytes // 64, 16, 64).transpose(1, 2).reshape(used, self._code_bytes)
            return rows[:self._n, :16 * groups].contiguous(), self._scales[:self._n][:, places]

    def set_active(self, rows, active: bool) -> None:
        """Hide rows from every search, or show them again (vector_db/qdrant_client.py:826-883)."""
        rows = np.ascontiguousarray(rows, dtype=np.int64).reshape(-1)
        _outside_capture(self.device, "rows are hidden and shown")
        with self._lock:
            if rows.size and (rows.min() < 0 or rows.max() >= self._n):
                raise ValueError("row position out of range")
            if rows.size == 0:
                return
            if self._active is None:
                if active:
                    return
                self._active = torch.ones((self._n,), dtype=torch.uint8, device=self._dev)
                self._renew()
            self._kept.stream()
            self._active[torch.from_numpy(rows).to(self._active.device)] = 1 if active else 0

    def make_filter(self, mask) -> DeviceFilter:
        f = DeviceFilter(mask, self.device)
        if f.n != self._n:
            f.close()
            raise ValueError("row_mask must have one byte per row")
        return f

    # --------------------------------------------------------------------- reads
    def reconstruct(self, rows, dtype=None):
        """The values that rows stand for.  Numpy positions: numpy float32, every position inside the index.  CUDA int64
        positions: a CUDA tensor of ``dtype`` (default float32); a position outside the index -- an unfilled slot of a search -- gives zeros."""
        on_device = isinstance(rows, torch.Tensor) and rows.is_cuda
        if not on_device:
            rows = np.ascontiguousarray(rows, dtype=np.int64).reshape(-1)
            if rows.size and (rows.min() < 0 or rows.max() >= self._n):
                raise ValueError("row position out of range")
        at = self._positions(rows)
        if dtype is None or not on_device:
            dtype = torch.float32
        kind, count = _type_of(dtype), at.numel()
        out = torch.empty((count, self.dim), dtype=dtype, device=self._dev)
        if count:
            with self._lock:
                check(lib.rag_mx4_read_device(self._st_ref, at.data_ptr(), count, out.data_ptr(), kind, self._kept.stream()))
        return out if on_device else out.cpu().numpy()

    # ------------------------------------------------------------------ products
    def scores(self, q, begin: int = 0, end: Optional[int] = None):
        """Every query against the rows [begin, end): float32 [nq, end - begin], a CUDA tensor for CUDA queries and numpy
        for numpy ones."""
        on_device = isinstance(q, torch.Tensor) and q.is_cuda
        q, nq, ld, kind = self._rows_in(q, "queries")
        begin = int(begin)
        with self._lock:
            end = self._n if end is None else int(end)
            if not 0 <= begin <= end <= self._n:
                raise ValueError("rows [begin, end) do not lie inside the index")
            out = torch.empty((nq, end - begin), dtype=torch.float32, device=self._dev)
            if nq and end > begin:
                check(lib.rag_mx4_scores_device(self._st_ref, begin, end, nq, q.data_ptr(), kind, ld,
                                                self._normalize, out.data_ptr(), end - begin, self._kept.stream()))
        return out if on_device else out.cpu().numpy()

    def plan_groups(self, groups, nq: int, dtype=None) -> GroupPlan:
        """Groups for ``scores_grouped`` that are used more than once: [n, 4] of (query begin, query end, row begin, row end),
        for ``nq`` queries of ``dtype`` (default: float32).  Good as long as the index does not shrink."""
        return GroupPlan(groups, nq, self._n, self.dim, torch.float32 if dtype is None else dtype, self.device)

    def scores_grouped(self, q, groups):
        """Ragged groups in one launch: the scores of each group, [its queries][its rows], one behind the other in a
        flat float32 CUDA tensor.  ``groups``: a ``GroupPlan`` (whose ``split`` gives the views), or what ``plan_groups`` takes."""
        q, nq, ld, kind = self._rows_in(q, "queries")
        plan = groups if isinstance(groups, GroupPlan) else self.plan_groups(groups, nq, q.dtype)
        with self._lock:
            if plan.device != self.device or plan.nq != nq or plan.type != kind or plan.n > self._n or plan.dim != self.dim:
                raise ValueError("the plan was made for other queries, another device or a longer index")
            out = torch.empty((plan.total,), dtype=torch.float32, device=self._dev)
            if plan.n_items:
                plan._use()
                check(lib.rag_mx4_scores_grouped_device(self._st_ref, nq, q.data_ptr(), plan.type, ld, self._normalize,
                                                        plan.items.data_ptr(), plan.n_items, plan.widest, out.data_ptr(), plan.total,
                                                        self._kept.stream()))
            return out

    # -------------------------------------------------------------------- search
    def search(self, q, k: int, min_score: Optional[float] = None, nprobe: int = 1, row_mask=None) -> Tuple[object, object]:
        """``DeviceIndex.search`` over the stored rows: (D [nq, k] float32, I [nq, k] int64 row positions), best first, equal
        scores by position, empty slots (-FLT_MAX, -1).  ``nprobe`` is accepted and unused."""
        k = int(k)
        if not 1 <= k <= MAX_K:
            raise ValueError(f"k must be in [1, {MAX_K}]")
        on_device = _is_torch_cuda(q)
        dev = self._dev
        q, nq, ld, kind = self._rows_in(q, "queries")
        D = torch.empty((nq, k), dtype=torch.float32, device=dev)
        I = torch.empty((nq, k), dtype=torch.int64, device=dev)
        with self._lock:
            if isinstance(row_mask, DeviceFilter) or _is_torch_cuda(row_mask):
                m_ptr, keep = _device_mask_ptr(row_mask, self)
                if _is_torch_cuda(row_mask) and row_mask.get_device() != self.device:
                    raise ValueError("tensor is on another device than the index")
            elif row_mask is not None:
                m = np.ascontiguousarray(row_mask, dtype=np.uint8).reshape(-1)
                if m.size != self._n:
                    raise ValueError("row_mask must have one byte per row")
                keep = torch.from_numpy(m).to(dev)
                m_ptr = keep.data_ptr()
            else:
                m_ptr = keep = None
            if nq:
                need = int(lib.rag_mx4_search_workspace(self._n, nq, k))
                ws = torch.empty((need,), dtype=torch.uint8, device=dev)
                check(lib.rag_mx4_search_device(self._st_ref, nq, q.data_ptr(), kind, ld, self._normalize, k,
                                                -FLT_MAX if min_score is None else float(min_score), m_ptr,
                                                None if self._active is None else self._active.data_ptr(), D.data_ptr(), I.data_ptr(),
                                                ws.data_ptr(), need, self._kept.stream()))
            self.last_path = "mx4" if self._n else "empty"
        return (D, I) if on_device else (D.cpu().numpy(), I.cpu().numpy())

    # --------------------------------------------------------------- persistence
    def save(self, path: str) -> None:
        """Rows as stored (the natural layout of ``packed``), soft deletes and metric, in one file."""
        with self._lock:
            codes, scales = self.packed()
            active = np.zeros(0, np.uint8) if self._active is None else self._active.cpu().numpy()
        with open(path, "wb") as f:
            np.savez(f, codes=codes.cpu().numpy(), scales=scales.cpu().numpy(), active=active, dim=np.int64(self.dim),
                     cosine=np.int64(self._normalize))

    @classmethod
    def load(cls, path: str, device: int = 0) -> "QuantizedIndex":
        with np.load(path, allow_pickle=False) as f:
            self = cls.from_packed(f["codes"], f["scales"], int(f["dim"]), metric="cosine" if int(f["cosine"]) else "ip", device=device)
            active = f["active"]
            if active.size:
                if active.dtype != np.uint8 or active.shape != (len(self),):
                    raise ValueError("the file's soft deletes are not one byte per row")
                self._active = torch.from_numpy(active).to(self._dev)
                self._renew()
        return self


def _scale_places(groups: int) -> np.ndarray:
    """Where the scale of every group lies inside a row's scale bytes (rag_hip.h, rag_mx4_layout)."""
    g = np.arange(groups, dtype=np.int64)
    return (g // 16) * 16 + (g % 4) * 4 + (g // 4) % 4

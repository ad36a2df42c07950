"""Autograd wrappers over the gfx950 HIP kernels (libasme_mi.so).

Each Function here replaces a chain of stock PyTorch ops of the reference (cited per Function) with
one or two hand-written kernels; the Linear projections run on the package's own weight-stationary GEMM
(csrc/wsgemm.hip) and split-T weight-gradient GEMM (csrc/gemm.hip), no library GEMM.

Dropout: every call with p > 0 draws a fresh 64-bit seed from torch's default CPU generator; the
kernels derive the mask from (seed, element index) with Philox, so the backward regenerates it.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call, ptr, stream

ctypes_i64, ctypes_vp = ctypes.c_int64, ctypes.c_void_p
_N_PARTIALS = 1024  # blocks (and partial rows) used by the grid-stride backward reductions
_EMB_PARTIALS = 2048  # the embedding backward's (2x the waves in flight: 124 -> 102 us at the bench shape)
# lazy table Adam: stage the step's unique rows (asme_lazy_adam_stage) so every reader gathers them in slot order
# (True), or catch them up in place in the table and gather by id (False; the A/B switch)
STAGE_ROWS = True


def new_seed(p: float) -> int:
    if p <= 0.0:
        return 0
    return int(torch.randint(0, 2 ** 62, (1,), dtype=torch.int64).item())


def as_u8(mask: torch.Tensor) -> torch.Tensor:
    """a 0/1 mask as contiguous uint8 bytes: a bool mask is reinterpreted in place (same bytes, no copy kernel)"""
    if mask.dtype == torch.bool:
        return mask.contiguous().view(torch.uint8)
    return mask.to(torch.uint8).contiguous()


def _f32(t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.float32:
        raise TypeError(f"expected float32 tensor, got {t.dtype}")
    return t.contiguous()


def _i64(t: torch.Tensor) -> torch.Tensor:
    return t.to(torch.int64).contiguous()


_DTYPES = {torch.float32: 0, torch.bfloat16: 1}  # the `dtype` argument of the C ABI


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype not in _DTYPES:
        raise TypeError(f"expected a float32 or bfloat16 tensor, got {t.dtype}")
    return _DTYPES[t.dtype]


def _alike(like: torch.Tensor, dtype: Optional[torch.dtype] = None, **tensors):
    """every given tensor on `like`'s device and (where `dtype` is given) of that dtype; like is on a ROCm device"""
    ptr(like)
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device != like.device:
            raise ValueError(f"{name} is on {t.device}, expected {like.device}")
        if dtype is not None and t.dtype != dtype:
            raise TypeError(f"{name} is {t.dtype}, expected {dtype}")


def _call_on(t: torch.Tensor, name: str, *args):
    """call(name, *args, stream) on t's device, whichever is current, and its current stream"""
    dev = t.get_device()
    if dev == torch._C._cuda_getDevice():
        call(name, *args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            call(name, *args, torch._C._cuda_getCurrentRawStream(dev))


def _ws_bytes(name: str, *sizes, device) -> Tuple[Optional[torch.Tensor], int]:
    """a workspace of the size a *_workspace query names"""
    n = int(getattr(_lib.load(), name)(*sizes))
    return (torch.empty(n, device=device, dtype=torch.uint8), n) if n else (None, 0)


def _reduce_partials(part: torch.Tensor, width: int) -> torch.Tensor:
    out = torch.empty(width, device=part.device, dtype=torch.float32)
    call("asme_reduce_rows", ptr(part), part.shape[0], width, ptr(out), 0, stream())
    return out


# ------------------------------------------------------------------------------------ table gradients
class TableGrad:
    """How the item-table gradient leaves the backward pass.

    dense  -> a dense (V, d) gradient tensor returned to autograd (nn.Embedding semantics)
    sparse -> contributions are scatter-added into a compact (U, d) buffer of the step's unique rows
              (`SparseTablePlan`); the table parameter gets no .grad and FusedAdam applies the exact
              dense update from the compact rows (rows without gradient still decay)."""

    def __init__(self):
        self.plan: Optional["SparseTablePlan"] = None
        self.lazy: Optional["LazyTableState"] = None
        # the plan of the last optimizer step, kept like a .grad that was not zeroed: another step without a
        # new backward applies the same rows again (torch.optim semantics); dropped by zero_grad / next plan
        self.applied: Optional["SparseTablePlan"] = None

    def drop_applied(self):
        if self.applied is not None:
            self.applied.release()
            self.applied = None


REST_STEP = -1  # last_step of a row at rest (csrc/adam_math.h kRestStep)


class LazyTableState:
    """Exact lazy dense Adam for the item table (asme_lazy_adam_*): rows are caught up to the current
    step only when read (before a forward that gathers them, or in flush()).  Bit-identical to updating
    every row every step (same per-element fp32 operations, same per-step constants)."""

    def __init__(self, param: torch.Tensor, exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor):
        self.param, self.exp_avg, self.exp_avg_sq = param, exp_avg, exp_avg_sq
        self.last_step = torch.zeros(param.shape[0], dtype=torch.int32, device=param.device)
        self.hist = torch.zeros(1024, 8, dtype=torch.float32, device=param.device)
        self.step = 0
        self.rest = False  # some rows may be at rest (last_step == REST_STEP)
        self._current_at = None  # the step every row is known to be current at (a full catch-up), else None

    def start(self, step: int, fresh: bool, wd: float, rest_rows: bool = True):
        """every row is current up to `step`; `fresh` (moments just created, all +0) without weight decay: every row
        starts AT REST (last_step = REST_STEP, csrc/adam_math.h kRestStep) -- its zero-gradient dense update is the
        identity bit for bit, so no kernel replays, reads or writes it until its first gradient (rest_rows=False:
        every row starts current, the A/B form; FusedAdam(rest_rows=...))"""
        self.step = step
        self.rest = bool(rest_rows and fresh and wd == 0.0)
        self.last_step.fill_(REST_STEP if self.rest else step)
        self._current_at = step

    def record(self, step: int, lr, b1, b2, eps, wd):
        if wd != 0.0 and self.rest:  # rows at rest are current up to the previous step; from now on they decay
            self.last_step.masked_fill_(self.last_step < 0, self.step)
            self.rest = False
        cap = self.hist.shape[0]
        while step >= cap:  # a resumed run can start at any step
            cap *= 2
        if cap != self.hist.shape[0]:
            grown = torch.zeros(cap, 8, dtype=torch.float32, device=self.hist.device)
            grown[: self.hist.shape[0]] = self.hist
            self.hist = grown
        call("asme_lazy_adam_record_step", ptr(self.hist), cap, step, lr, b1, b2, eps, wd, stream())
        self.step = step

    def catch_up(self, rows: Optional[torch.Tensor] = None, count: Optional[torch.Tensor] = None, cap: int = 0):
        if self.step == 0:
            return
        V, D = self.param.shape
        if rows is None:
            if self._current_at == self.step:
                return  # every row is current already (a second flush, an evaluation after one): nothing to replay
            self._current_at = self.step
            cap = V
        note_param_write()  # (writes table rows behind torch's version counter: cached catalogue planes are stale)
        call("asme_lazy_adam_catch_up", ptr(rows), ptr(count), cap, ptr(self.last_step), ptr(self.param),
             ptr(self.exp_avg), ptr(self.exp_avg_sq), D, ptr(self.hist), self.hist.shape[0], self.step, stream())

    def stage_ok(self) -> bool:
        D = self.param.shape[1]
        return STAGE_ROWS and bool(_lib.load().asme_lazy_adam_stage_supported(D)) and all(
            t.data_ptr() % 16 == 0 for t in (self.param, self.exp_avg, self.exp_avg_sq))

    def stage(self, rows: torch.Tensor, count: torch.Tensor, cap: int) -> torch.Tensor:
        """(3, cap, d): param / exp_avg / exp_avg_sq of rows[s] brought up to the current step, in slot order;
        the table itself is not written (asme_lazy_adam_stage)"""
        D = self.param.shape[1]
        out = torch.empty(3, max(cap, 1), D, device=self.param.device, dtype=torch.float32)
        call("asme_lazy_adam_stage", ptr(rows), ptr(count), cap, ptr(self.last_step), ptr(self.param),
             ptr(self.exp_avg), ptr(self.exp_avg_sq), D, ptr(self.hist), self.hist.shape[0], self.step, ptr(out[0]),
             ptr(out[1]), ptr(out[2]), stream())
        return out

    def apply(self, plan: "SparseTablePlan", step: int, fused: bool = True):
        """the step's Adam update of the plan's rows; `fused`: reduce the table gradient and apply the staged step in
        one pass (asme_table_grad_reduce_apply) when nothing else needs the gradient rows (FusedAdam(fused_apply=...))"""
        D = self.param.shape[1]
        if plan.staged is not None:
            if fused and plan.reduce_apply(self, step):
                plan.staged = None
                return
            st = plan.staged
            call("asme_lazy_adam_apply_staged", ptr(plan.unique), ptr(plan.count), plan.capacity, ptr(plan.grad_rows),
                 ptr(st[0]), ptr(st[1]), ptr(st[2]), ptr(self.last_step), ptr(self.param), ptr(self.exp_avg),
                 ptr(self.exp_avg_sq), D, ptr(self.hist), self.hist.shape[0], step, stream())
            plan.staged = None  # the staged values are one step old now (a re-apply catches up from the table)
            return
        call("asme_lazy_adam_apply", ptr(plan.unique), ptr(plan.count), plan.capacity, ptr(plan.grad_rows),
             ptr(self.last_step), ptr(self.param), ptr(self.exp_avg), ptr(self.exp_avg_sq), D, ptr(self.hist),
             self.hist.shape[0], step, stream())

    def flush(self):
        """bring every row up to date (before evaluation, checkpointing or any other reader)."""
        self.catch_up(None)


_MAP_FREE = {}  # slot map data_ptr -> the event after which its entries are all -1 again (TableIdsAhead waits on it)


def _note_map_free(slot_map: torch.Tensor):
    ev = torch.cuda.Event()
    ev.record(torch.cuda.current_stream(slot_map.device))
    _MAP_FREE[slot_map.data_ptr()] = ev


def new_slot_map(rows: int, device) -> torch.Tensor:
    """a (rows,) int32 dedup slot map, -1 at rest; its fill is recorded as the point from which another stream's
    dedup (TableIdsAhead) may use it"""
    m = torch.full((rows,), -1, dtype=torch.int32, device=device)
    if m.is_cuda:
        _note_map_free(m)
    return m


class TableIdsAhead:
    """The id-only half of a step's SparseTablePlan -- the dedup of its table ids (asme_dedup_ids_segments) and the
    occurrence CSR of the table gradient (asme_occurrence_csr) -- enqueued on the CURRENT stream (a producer's side
    stream) a step ahead.  Neither depends on the table's values, only on the ids, so they run beside the previous
    step's kernels instead of in front of the next step's; the table-dependent half (staging the rows through the
    lazy Adam) stays with SparseTablePlan on the training stream.  `slot_map` must not be the map of a plan that
    is still live (the module alternates two); the dedup waits for the event of that map's last release
    (_note_map_free), so it never sees a previous plan's entries."""

    def __init__(self, vocab: int, dim: int, id_sets: Sequence[torch.Tensor], slot_map: torch.Tensor):
        cur = torch.cuda.current_stream(slot_map.device)
        ev = _MAP_FREE.get(slot_map.data_ptr())
        if ev is not None:
            cur.wait_event(ev)
        self.id_sets = list(id_sets)
        self.keys = [(x.data_ptr(), tuple(x.shape)) for x in id_sets]
        self.plan = SparseTablePlan(None, id_sets, slot_map, vocab=vocab, dim=dim)
        self.plan._csr = self.plan._occurrence_csr() if self.plan.capacity > 0 else None
        self.ready = torch.cuda.Event()
        self.ready.record(cur)

    def matches(self, id_sets: Sequence[torch.Tensor]) -> bool:
        return [(x.data_ptr(), tuple(x.shape)) for x in id_sets] == self.keys

    def tensors(self):
        p = self.plan
        out = [p.unique, p.count, p._flat_inverse] + list(self.id_sets)
        if p._csr is not None:
            out += [t for t in p._csr[:4]]
        return out

    def adopt(self):
        """make the current stream wait for the work of the ahead stream and keep its tensors alive for this stream
        (the caching allocator returns them to the side stream's pool only after this stream's reads)"""
        cur = torch.cuda.current_stream(self.plan.unique.device)
        cur.wait_event(self.ready)
        for t in self.tensors():
            t.record_stream(cur)

    def discard(self):
        """an ahead plan that no step will take: its slot map entries reset (on the current stream, after it)"""
        self.adopt()
        self.plan.release()


class SparseTablePlan:
    """Per-step dedup of every id that touches the table: slot map, unique rows, compact grad."""

    def __init__(self, table: Optional[torch.Tensor], id_sets: Sequence[torch.Tensor], slot_map: torch.Tensor,
                 vocab: Optional[int] = None, dim: int = 0, ahead: Optional[TableIdsAhead] = None):
        """ahead: the dedup and occurrence CSR of exactly these id tensors, computed a step ahead on another stream
        (TableIdsAhead, over `slot_map`): taken over instead of running them here"""
        dev = slot_map.device
        tg = getattr(table, "_asme_table_grad", None) if table is not None else None
        if tg is not None:
            tg.drop_applied()  # the previous step's plan still marks the shared slot map
        self.vocab, self.dim = table.shape if table is not None else (vocab, dim)
        self.slot_map = slot_map
        self._csr = None
        if ahead is not None:
            if ahead.plan.slot_map is not slot_map or not ahead.matches(id_sets):
                raise ValueError("SparseTablePlan: the ahead dedup is of other ids or another slot map")
            ahead.adopt()
            n = ahead.plan.capacity
            self.unique, inverse, self.count = ahead.plan.unique, ahead.plan._flat_inverse, ahead.plan.count
            self._csr = ahead.plan._csr
        else:
            # the id sets are read in place as segments of one occurrence list (no concatenated copy)
            segs = [_i64(x).reshape(-1) for x in id_sets]
            segs = [x if x.is_contiguous() else x.contiguous() for x in segs]
            if len(segs) > 4:
                segs = [torch.cat(segs)]
            n = sum(x.numel() for x in segs)
            self.unique = torch.empty(n, device=dev, dtype=torch.int64)
            inverse = torch.empty(n, device=dev, dtype=torch.int64)
            # (asme_dedup_ids always writes the count)
            self.count = torch.empty(1, device=dev, dtype=torch.int32) if n > 0 else torch.zeros(1, device=dev,
                                                                                              dtype=torch.int32)
            if n > 0:
                ws_bytes = int(_lib.load().asme_dedup_workspace_bytes(n))
                ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
                k = len(segs)
                call("asme_dedup_ids_segments", k, (ctypes_vp * k)(*[x.data_ptr() for x in segs]),
                     (ctypes_i64 * k)(*[x.numel() for x in segs]), self.vocab, ptr(slot_map), ptr(ws), ws_bytes,
                     ptr(self.unique), ptr(inverse), ptr(self.count), stream())
        self.capacity = n
        self._slots_mapped = False
        self.grad_scale = 1.0  # factor on every reduced gradient row (the sharded owner: 1/W, DDP averaging)
        self._grad_rows = None
        self._inverse = {}
        self._flat_inverse = inverse
        self._offset = {}
        self._contrib = []  # (flat offset, n, rows (n, d), scale (n,) or None) -- see add_rows / add_scaled
        off = 0
        for x in id_sets:
            k = x.numel()
            key = (x.data_ptr(), tuple(x.shape))
            self._inverse[key] = inverse[off:off + k].view(x.shape)
            self._offset[key] = off
            off += k
        self.consumed = False
        # (3, capacity, d) param / moments of unique[s] brought up to date, or None: the step's readers take
        # `rows` + `gather_ids(ids)` instead of the table (see LazyTableState.stage)
        self.staged: Optional[torch.Tensor] = None
        if tg is not None and tg.lazy is not None:
            # rows gathered by this step's forward must carry every earlier (zero-gradient) update
            if tg.lazy.stage_ok():
                self.staged = tg.lazy.stage(self.unique, self.count, self.capacity)
            else:
                tg.lazy.catch_up(self.unique, self.count, self.capacity)

    def gather_source(self, table: torch.Tensor, ids: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """(rows, row ids) a reader of `ids` gathers from: the staged rows by slot when this step staged them,
        else the table itself by id"""
        if self.staged is not None and self.has(ids):
            if self._distinct:  # slot s holds ids[s]: the staged rows are the gathered rows themselves
                return self.staged[0], None
            return self.staged[0], self.inverse_of(ids)
        return table, ids

    _distinct = False
    _csr = None  # (order, slot, seg_off, parts, part_bytes) once built (ahead, or by the first reduction)

    def has(self, ids: torch.Tensor) -> bool:
        return (ids.data_ptr(), tuple(ids.shape)) in (self._offset if self._distinct else self._inverse)

    @classmethod
    def identity(cls, n_rows: int, id_sets: Sequence[torch.Tensor], dim: int) -> "SparseTablePlan":
        """plan over ids that already are row indices of a compact (n_rows, dim) table in which every row
        occurs (the sharded step's table of fetched rows): no dedup, slot s == row s, so grad_rows[:n_rows]
        is the table's gradient in row order, from the same ordered (deterministic) reduction"""
        self = cls.__new__(cls)
        flat = torch.cat([_i64(x).reshape(-1) for x in id_sets])
        n = flat.numel()
        if n_rows > n:
            raise ValueError("identity plan: every row must occur at least once")
        dev = flat.device
        self.vocab, self.dim = n_rows, dim
        self.slot_map = None
        self.unique = torch.arange(n_rows, device=dev, dtype=torch.int64)
        self.count = torch.full((1,), n_rows, device=dev, dtype=torch.int32)
        self.capacity = n
        self._slots_mapped = True  # (no map: slot s == row s)
        self.grad_scale = 1.0
        self._grad_rows = None
        self._inverse, self._offset, self._contrib = {}, {}, []
        self._flat_inverse = flat
        self.staged = None
        off = 0
        for x in id_sets:
            key = (x.data_ptr(), tuple(x.shape))
            self._inverse[key] = x
            self._offset[key] = off
            off += x.numel()
        self.consumed = False
        return self

    @classmethod
    def distinct(cls, table: torch.Tensor, ids: torch.Tensor,
                 slot_map: Optional[torch.Tensor] = None) -> "SparseTablePlan":
        """plan over ids known to be distinct (the row-shard owner's requests at one rank): no dedup, slot s ==
        ids[s]; the rows are staged like any plan's, and a single unscaled gradient contribution (one row per
        slot) is applied as it is -- no occurrence CSR, no reduction.  `slot_map` ((|V|,) int32, -1 at rest): the
        row -> slot table row_slot_map() fills on demand (the non-lazy row Adam reads it); without one that call
        raises"""
        self = cls.__new__(cls)
        ids = _i64(ids).reshape(-1)
        n = ids.numel()
        dev = ids.device
        self.vocab, self.dim = table.shape
        self.slot_map = slot_map
        self.unique = ids
        self.count = torch.tensor([n], dtype=torch.int32).to(dev, non_blocking=True)
        self.capacity = n
        self._slots_mapped = False  # the map is written only when row_slot_map() asks for it
        self._distinct = True
        self.grad_scale = 1.0
        self._grad_rows = None
        key = (ids.data_ptr(), tuple(ids.shape))
        self._flat_inverse = None
        self._inverse, self._offset, self._contrib = {}, {key: 0}, []
        self.consumed = False
        self.staged = None
        tg = getattr(table, "_asme_table_grad", None)
        if tg is not None:
            tg.drop_applied()
            if tg.lazy is not None:
                if tg.lazy.stage_ok():
                    self.staged = tg.lazy.stage(self.unique, self.count, self.capacity)
                else:
                    tg.lazy.catch_up(self.unique, self.count, self.capacity)
        return self

    @classmethod
    def for_ids(cls, vocab: int, id_sets: Sequence[torch.Tensor], slot_map: torch.Tensor) -> "SparseTablePlan":
        """dedup only (no table attached): unique ids in first-occurrence order + inverse per id set"""
        return cls(None, id_sets, slot_map, vocab=vocab, dim=0)

    def adopt_contributions(self, other: "SparseTablePlan"):
        """take over the gradient contributions of `other`, a plan over the same slots (the one-rank sharded step:
        the requester's compact identity plan, whose row s is this distinct plan's slot s): its occurrence -> slot
        map and registered rows, reduced (and applied) by this plan"""
        if not self._distinct or other.capacity == 0 or other._grad_rows is not None:
            raise RuntimeError("adopt_contributions: a distinct plan taking an unreduced plan over its slots")
        self._flat_inverse = other._flat_inverse
        self._csr = None  # (over the adopted occurrences)
        self.capacity = other.capacity  # occurrences (>= slots): the CSR's length; count stays the slot count
        self._contrib = other._contrib
        other._contrib = []
        self._adopted = True
        other.release()

    _adopted = False

    def add_rows(self, ids: torch.Tensor, rows: torch.Tensor):
        """register the gradient rows (one per occurrence of the registered id set `ids`) of this step;
        summed per unique row, in occurrence order, when grad_rows is first read"""
        self._add(ids, _f32(rows).reshape(ids.numel(), self.dim), None)

    def add_scaled(self, ids: torch.Tensor, scale: torch.Tensor, rows: torch.Tensor):
        """register scale[t] * rows[t] per occurrence t of `ids` (the sampled head: g_pos/g_neg * h)"""
        self._add(ids, _f32(rows).reshape(ids.numel(), self.dim), _f32(scale).reshape(ids.numel()))

    def _add(self, ids, rows, scale):
        key = (ids.data_ptr(), tuple(ids.shape))
        if key not in self._offset:
            raise KeyError("ids were not registered with the sparse table plan of this step")
        if self._grad_rows is not None:
            raise RuntimeError("table gradient already materialised for this step")
        self._contrib.append((self._offset[key], ids.numel(), rows, scale))

    def _occurrence_csr(self):
        if self._csr is not None:
            return self._csr
        n = self.capacity
        dev = self.unique.device
        lib = _lib.load()
        ws_bytes = int(lib.asme_occurrence_csr_workspace(n))
        ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
        order = torch.empty(n, device=dev, dtype=torch.int32)
        slot = torch.empty(n, device=dev, dtype=torch.int32)
        seg_off = torch.empty(n + 1, device=dev, dtype=torch.int32)
        if self._flat_inverse is None:  # a distinct plan: occurrence s is slot s
            self._flat_inverse = torch.arange(n, device=dev, dtype=torch.int64)
        call("asme_occurrence_csr", ptr(self._flat_inverse), n, n, ptr(ws), ws_bytes, ptr(order), ptr(slot),
             ptr(seg_off), stream())
        part_bytes = int(lib.asme_table_grad_workspace(n, self.dim))
        parts = torch.empty(max(part_bytes, 4) // 4, device=dev, dtype=torch.float32)
        self._csr = (order, slot, seg_off, parts, part_bytes)
        return self._csr

    @staticmethod
    def _contrib_arrays(part):
        k = len(part)
        return (k, (ctypes_i64 * k)(*[c[0] for c in part]), (ctypes_i64 * k)(*[c[1] for c in part]),
                (ctypes_vp * k)(*[c[2].data_ptr() for c in part]),
                (ctypes_vp * k)(*[(c[3].data_ptr() if c[3] is not None else None) for c in part]))

    def reduce_apply(self, lazy: "LazyTableState", step: int) -> bool:
        """the table gradient reduced and applied as the lazy Adam's real-gradient step in one pass from the staged
        rows (asme_table_grad_reduce_apply); False (nothing done) where the gradient rows are needed as such"""
        if self.staged is None or self._grad_rows is not None or not 1 <= len(self._contrib) <= 4 \
                or self.capacity == 0 or (self._distinct and not self._adopted):
            return False
        order, slot, seg_off, parts, part_bytes = self._occurrence_csr()
        k, offs, ns, rows, scales = self._contrib_arrays(sorted(self._contrib, key=lambda c: c[0]))
        st = self.staged
        n, d = self.capacity, self.dim
        call("asme_table_grad_reduce_apply", ptr(order), ptr(slot), ptr(seg_off), ptr(self.count), n, n, d, k, offs,
             ns, rows, scales, self.grad_scale, ptr(parts), part_bytes, ptr(self.unique), ptr(st[0]), ptr(st[1]),
             ptr(st[2]), ptr(lazy.last_step), ptr(lazy.param), ptr(lazy.exp_avg), ptr(lazy.exp_avg_sq),
             ptr(lazy.hist), lazy.hist.shape[0], step, stream())
        # (the contributions stay registered: a re-step without a new backward reduces them again via grad_rows)
        return True

    def _reduce_contributions(self) -> torch.Tensor:
        """deterministic table gradient: occurrences grouped by row (counting sort), sums in a fixed order
        (asme_occurrence_csr + asme_table_grad_reduce); no float atomics, no zero fill"""
        dev = self.unique.device
        n, d = self.capacity, self.dim
        if n == 0:
            return torch.zeros(0, d, device=dev, dtype=torch.float32)
        order, slot, seg_off, parts, part_bytes = self._occurrence_csr()
        out = torch.empty(n, d, device=dev, dtype=torch.float32)
        contrib = sorted(self._contrib, key=lambda c: c[0])
        for i in range(0, len(contrib), 4):
            k, offs, ns, rows, scales = self._contrib_arrays(contrib[i:i + 4])
            dest = out if i == 0 else torch.empty_like(out)  # more than 4 contributions: add the rest
            call("asme_table_grad_reduce", ptr(order), ptr(slot), ptr(seg_off), ptr(self.count), n, n, d, k, offs,
                 ns, rows, scales, self.grad_scale, ptr(parts), part_bytes, ptr(dest), stream())
            if i:
                out += dest
        self._contrib = []
        return out

    @property
    def grad_rows(self) -> torch.Tensor:
        """compact (capacity, d) gradient rows, slot s <-> unique[s]: the ordered sums of the registered
        contributions (add_rows / add_scaled), or a zeroed buffer for callers that scatter-add into it"""
        if self._grad_rows is None:
            if self._distinct and len(self._contrib) == 1 and self._contrib[0][3] is None \
                    and self._contrib[0][1] == self.capacity:
                rows = self._contrib[0][2]  # one row per slot, in slot order: the gradient as it is
                self._grad_rows = rows if self.grad_scale == 1.0 else rows * self.grad_scale
                self._contrib = []
            elif self._contrib:
                self._grad_rows = self._reduce_contributions()
            else:
                self._grad_rows = torch.zeros(self.capacity, self.dim, device=self.unique.device,
                                              dtype=torch.float32)
        return self._grad_rows

    def has_gradient(self) -> bool:
        """a backward registered gradient rows with this plan"""
        return bool(self._contrib) or self._grad_rows is not None

    def n_unique(self) -> int:
        """number of distinct ids (device -> host sync)"""
        return int(self.count.item())

    def row_slot_map(self) -> torch.Tensor:
        """the slot map as a row -> slot table (row r's gradient is grad_rows[map[r]], -1: none), rewritten from the
        dedup's first-occurrence entries once (asme_dedup_map_slots)"""
        if self.slot_map is None:
            raise RuntimeError("this plan has no row -> slot map (a distinct plan built without slot_map)")
        if not self._slots_mapped:
            call("asme_dedup_map_slots", ptr(self.unique), ptr(self.count), self.capacity, ptr(self.slot_map),
                 stream())
            self._slots_mapped = True
        return self.slot_map

    def inverse_of(self, ids: torch.Tensor) -> torch.Tensor:
        key = (ids.data_ptr(), tuple(ids.shape))
        if self._distinct and key in self._offset:
            if key not in self._inverse:
                self._inverse[key] = torch.arange(ids.numel(), device=ids.device, dtype=torch.int64).view(ids.shape)
            return self._inverse[key]
        if key not in self._inverse:
            raise KeyError("ids were not registered with the sparse table plan of this step")
        return self._inverse[key]

    def release(self):
        # (a distinct plan's map holds entries only once row_slot_map() wrote them)
        if self.slot_map is not None and (self._slots_mapped or not self._distinct):
            call("asme_dedup_reset", ptr(self.unique), ptr(self.count), self.capacity, ptr(self.slot_map), stream())
            if self.slot_map.data_ptr() in _MAP_FREE:  # a map another stream's dedup may use next (TableIdsAhead)
                _note_map_free(self.slot_map)
        self.consumed = True


# ------------------------------------------------------------------------------------ embedding
@dataclass
class EmbeddingSpec:
    """TransformerEmbedding (+ PreFusion) configuration for one forward call."""
    seq_len: int
    ln1_eps: float = 1e-5
    p1: float = 0.0
    ln2_eps: float = 1e-5
    p2: float = 0.0
    table_grad: Optional[TableGrad] = None


def embedding_keep_chunks(keep: torch.Tensor, D: int) -> torch.Tensor:
    """the embedding forward's stored keep bytes (T, D/4) in chunk order (byte c: elements 4c..4c+3; bit i: drop1 of
    element 4c+i, bit 4+i: drop2).  The kernels store a lane's chunks adjacently when the row layout covers the row
    exactly (csrc/embedding.hip emb_keep_store: D = 128 on 16 lanes x 2 chunks, D = 512 on 64 x 2)"""
    T = keep.shape[0]
    lanes = {128: 16, 512: 64}.get(D)
    if lanes is None:
        return keep
    return keep.reshape(T, lanes, 2).transpose(1, 2).reshape(T, D // 4)


class _EmbeddingFn(torch.autograd.Function):
    """transformer_layers.py:55-80 (+ kebert4rec/components.py:54-63):
    drop2(LN2(drop1(LN1(E[ids] + P[pos])) + extra))"""

    @staticmethod
    def forward(ctx, ids, table, pos, ln1_w, ln1_b, extra, ln2_w, ln2_b, spec: EmbeddingSpec):
        ids = _i64(ids)
        T = ids.numel()
        D = table.shape[1]
        # rows staged in slot order by this step's lazy Adam (SparseTablePlan.gather_source), else the table
        plan = spec.table_grad.plan if spec.table_grad is not None else None
        src, src_ids = plan.gather_source(table, ids) if plan is not None else (table, ids)
        V = src.shape[0]
        out = torch.empty(T, D, device=table.device, dtype=torch.float32)
        stats = torch.empty(T, 4, device=table.device, dtype=torch.float32)
        s1, s2 = new_seed(spec.p1), new_seed(spec.p2)
        extra_c = None if extra is None else _f32(extra).reshape(T, D)
        keep = None
        if (spec.p1 > 0 or spec.p2 > 0) and D % 4 == 0:  # dropout decisions, one byte per 4 elements
            keep = torch.empty(T, D // 4, device=table.device, dtype=torch.uint8)
        call("asme_embedding_fwd", ptr(src_ids), T, spec.seq_len, ptr(src), V, D, ptr(pos), ptr(ln1_w), ptr(ln1_b),
             spec.ln1_eps, spec.p1, s1, ptr(extra_c), ptr(ln2_w), ptr(ln2_b), spec.ln2_eps, spec.p2, s2, ptr(out),
             ptr(stats), ptr(keep), None, stream())
        ctx.save_for_backward(ids, src_ids, src, pos, ln1_w, ln1_b, extra_c, ln2_w, stats, keep)
        ctx.table_shape = tuple(table.shape)
        ctx.spec, ctx.seeds = spec, (s1, s2)
        ctx.has = (pos is not None, ln1_w is not None, extra is not None, ln2_w is not None)
        return out.view(*ids.shape, D)

    @staticmethod
    def backward(ctx, dout):
        ids, src_ids, src, pos, ln1_w, ln1_b, extra, ln2_w, stats, keep = ctx.saved_tensors
        spec = ctx.spec
        s1, s2 = ctx.seeds
        T = ids.numel()
        V, D = ctx.table_shape
        dev = src.device
        dout = _f32(dout).reshape(T, D)
        d_rows = torch.empty(T, D, device=dev, dtype=torch.float32)
        d_extra = torch.empty(T, D, device=dev, dtype=torch.float32) if ctx.has[2] else None
        has_ln = ctx.has[1] or ctx.has[3]
        part = torch.empty(_EMB_PARTIALS, 4 * D, device=dev, dtype=torch.float32) if has_ln else None
        call("asme_embedding_bwd", ptr(src_ids), T, spec.seq_len, ptr(src), src.shape[0], D, ptr(pos), ptr(ln1_w),
             ptr(ln1_b),
             spec.p1, s1, ptr(extra), ptr(ln2_w), spec.p2, s2, ptr(keep), ptr(dout), ptr(stats), ptr(d_rows),
             ptr(d_extra), ptr(part), _EMB_PARTIALS, stream())
        g_table = None
        if ctx.needs_input_grad[1]:
            plan = spec.table_grad.plan if spec.table_grad is not None else None
            if plan is not None:
                plan.add_rows(ids, d_rows)
            else:
                g_table = dense_table_grad(ids, d_rows, V, D)
        g_pos = None
        if ctx.has[0] and ctx.needs_input_grad[2]:
            L = spec.seq_len
            B = T // L
            # rows [0, L) are written (accumulate = 0); only rows past the sequence length need zeros
            g_pos = torch.empty_like(pos) if pos.shape[0] == L else torch.zeros_like(pos)
            nch = max(1, min(32, B))
            ws = torch.empty(nch, L, D, device=dev, dtype=torch.float32)
            call("asme_position_grad", ptr(d_rows), B, L, D, ptr(ws), nch, ptr(g_pos), 0, stream())
        g = [None] * 4
        if has_ln:
            red = _reduce_partials(part, 4 * D)
            g = [red[0:D], red[D:2 * D], red[2 * D:3 * D], red[3 * D:4 * D]]
        g_extra = d_extra.view(*ids.shape, D) if d_extra is not None else None
        return (None, g_table, g_pos, g[0] if ctx.has[1] else None, g[1] if ctx.has[1] else None, g_extra,
                g[2] if ctx.has[3] else None, g[3] if ctx.has[3] else None, None)


class _EmbeddingLnFn(torch.autograd.Function):
    """_EmbeddingFn + the first transformer block's input LayerNorm on its output in the same kernel
    (asme_embedding_ln_fwd / _bwd): returns (x, LN3(x)); x is the block's residual stream, LN3(x) the attention
    input (transformer_layers.py:251-258), so the separate LayerNorm pass over x and its backward disappear."""

    @staticmethod
    def forward(ctx, ids, table, pos, ln1_w, ln1_b, extra, ln2_w, ln2_b, ln3_w, ln3_b, spec: EmbeddingSpec,
                ln3_eps: float):
        ids = _i64(ids)
        T = ids.numel()
        D = table.shape[1]
        plan = spec.table_grad.plan if spec.table_grad is not None else None
        src, src_ids = plan.gather_source(table, ids) if plan is not None else (table, ids)
        V = src.shape[0]
        dev = table.device
        out = torch.empty(T, D, device=dev, dtype=torch.float32)
        ln = torch.empty(T, D, device=dev, dtype=torch.float32)
        stats = torch.empty(T, 4, device=dev, dtype=torch.float32)
        stats3 = torch.empty(T, 2, device=dev, dtype=torch.float32)
        s1, s2 = new_seed(spec.p1), new_seed(spec.p2)
        extra_c = None if extra is None else _f32(extra).reshape(T, D)
        keep = None
        if spec.p1 > 0 or spec.p2 > 0:
            keep = torch.empty(T, D // 4, device=dev, dtype=torch.uint8)
        call("asme_embedding_ln_fwd", ptr(src_ids), T, spec.seq_len, ptr(src), V, D, ptr(pos), ptr(ln1_w), ptr(ln1_b),
             spec.ln1_eps, spec.p1, s1, ptr(extra_c), ptr(ln2_w), ptr(ln2_b), spec.ln2_eps, spec.p2, s2, ptr(ln3_w),
             ptr(ln3_b), ln3_eps, ptr(out), ptr(stats), ptr(ln), ptr(stats3), ptr(keep), None, stream())
        ctx.save_for_backward(ids, src_ids, src, pos, ln1_w, ln1_b, extra_c, ln2_w, ln2_b, ln3_w, stats, stats3, keep)
        ctx.table_shape = tuple(table.shape)
        ctx.spec, ctx.seeds = spec, (s1, s2)
        ctx.has = (pos is not None, ln1_w is not None, extra is not None, ln2_w is not None)
        shape = (*ids.shape, D)
        return out.view(shape), ln.view(shape)

    @staticmethod
    def backward(ctx, dout, dln):
        ids, src_ids, src, pos, ln1_w, ln1_b, extra, ln2_w, ln2_b, ln3_w, stats, stats3, keep = ctx.saved_tensors
        spec = ctx.spec
        s1, s2 = ctx.seeds
        T = ids.numel()
        V, D = ctx.table_shape
        dev = src.device
        dout = _f32(dout).reshape(T, D) if dout is not None else torch.zeros(T, D, device=dev)
        dln = _f32(dln).reshape(T, D) if dln is not None else torch.zeros(T, D, device=dev)
        d_rows = torch.empty(T, D, device=dev, dtype=torch.float32)
        d_extra = torch.empty(T, D, device=dev, dtype=torch.float32) if ctx.has[2] else None
        part = torch.empty(_EMB_PARTIALS, 6 * D, device=dev, dtype=torch.float32)
        call("asme_embedding_ln_bwd", ptr(src_ids), T, spec.seq_len, ptr(src), src.shape[0], D, ptr(pos), ptr(ln1_w),
             ptr(ln1_b), spec.p1, s1, ptr(extra), ptr(ln2_w), ptr(ln2_b), spec.p2, s2, ptr(ln3_w), ptr(stats3),
             ptr(keep), ptr(dout), ptr(dln), ptr(stats), ptr(d_rows), ptr(d_extra), ptr(part), _EMB_PARTIALS, stream())
        g_table = None
        if ctx.needs_input_grad[1]:
            plan = spec.table_grad.plan if spec.table_grad is not None else None
            if plan is not None:
                plan.add_rows(ids, d_rows)
            else:
                g_table = dense_table_grad(ids, d_rows, V, D)
        g_pos = None
        if ctx.has[0] and ctx.needs_input_grad[2]:
            L = spec.seq_len
            B = T // L
            g_pos = torch.empty_like(pos) if pos.shape[0] == L else torch.zeros_like(pos)
            nch = max(1, min(32, B))
            ws = torch.empty(nch, L, D, device=dev, dtype=torch.float32)
            call("asme_position_grad", ptr(d_rows), B, L, D, ptr(ws), nch, ptr(g_pos), 0, stream())
        red = _reduce_partials(part, 6 * D)
        g = [red[i * D:(i + 1) * D] for i in range(6)]
        g_extra = d_extra.view(*ids.shape, D) if d_extra is not None else None
        return (None, g_table, g_pos, g[0] if ctx.has[1] else None, g[1] if ctx.has[1] else None, g_extra,
                g[2] if ctx.has[3] else None, g[3] if ctx.has[3] else None, g[4], g[5], None, None)



def embedding(ids, table, pos=None, ln1=None, extra=None, ln2=None, spec: EmbeddingSpec = None, ln3=None):
    """The fused embedding; `ln3` (an nn.LayerNorm): also return ln3(x) from the same kernel -> (x, ln3(x))."""
    ln1_w, ln1_b = (None, None) if ln1 is None else ln1
    ln2_w, ln2_b = (None, None) if ln2 is None else ln2
    if ln3 is not None:
        D = table.shape[1]
        # the fused next LayerNorm (ln3) when the hidden size allows the 4-wide kernels (whether ln3 is handed in at
        # all is the model's fuse_embedding_norm property)
        if D % 4 == 0 and (ln2_w is None or ln2_b is not None):
            return _EmbeddingLnFn.apply(ids, table, pos, ln1_w, ln1_b, extra, ln2_w, ln2_b, ln3.weight, ln3.bias,
                                        spec, float(ln3.eps))
        x = _EmbeddingFn.apply(ids, table, pos, ln1_w, ln1_b, extra, ln2_w, ln2_b, spec)
        return layer_norm_pass(x, ln3)
    return _EmbeddingFn.apply(ids, table, pos, ln1_w, ln1_b, extra, ln2_w, ln2_b, spec)


class _GatherSumFn(torch.autograd.Function):
    """kebert4rec/components.py:15-24 content_embedding (k=1) / layers.py:15-27 LinearUpscaler
    (multi-hot -> Linear == sum of weight columns of the non-pad ids, + bias)."""

    @staticmethod
    def forward(ctx, ids, table, bias, skip_zero: bool, multi_hot: bool):
        ids = _i64(ids)
        shape = ids.shape
        if multi_hot:  # (N, S, K) multi-hot ids
            n, k = ids.numel() // shape[-1], shape[-1]
            out_shape = shape[:-1]
        else:
            n, k = ids.numel(), 1
            out_shape = shape
        V, D = table.shape
        out = torch.empty(n, D, device=table.device, dtype=torch.float32)
        call("asme_gather_sum_fwd", ptr(ids), n, k, int(skip_zero), ptr(table), V, D, ptr(bias), ptr(out), 0,
             stream())
        ctx.save_for_backward(ids)
        ctx.meta = (n, k, skip_zero, V, D, bias is not None)
        return out.view(*out_shape, D)

    @staticmethod
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        n, k, skip_zero, V, D, has_bias = ctx.meta
        dout = _f32(dout).reshape(n, D)
        # (fp32 atomics, like torch's embedding backward: the ordered-sum path of dense_table_grad measured slower here,
        # 89 -> ~130 us per KeBERT4Rec step, for a 64-row attribute table -- its ~18 launches outweigh the contention)
        g_table = torch.zeros(V, D, device=dout.device, dtype=torch.float32)
        call("asme_gather_sum_bwd", ptr(dout), ptr(ids), n, k, int(skip_zero), ptr(g_table), V, D, stream())
        g_bias = None
        if has_bias:
            g_bias = _reduce_rows(dout)
        return None, g_table, g_bias, None, None


_DENSE_SLOT_MAPS = {}


def dense_table_grad(ids: torch.Tensor, rows: torch.Tensor, V: int, D: int) -> torch.Tensor:
    """nn.Embedding's dense (V, D) gradient (embedding_dense_backward) without float atomics: the occurrences are
    deduplicated and summed per row in occurrence order (the sparse plan's ordered reduction), then written to their
    rows (asme_scatter_rows).  Deterministic, and a hot id (the cloze MASK token: ~18 % of a BERT4Rec batch) no
    longer serialises tens of thousands of atomics on one row (0.78 ms per C3 step)."""
    dev = rows.device
    key = (dev, V)
    slot_map = _DENSE_SLOT_MAPS.get(key)
    if slot_map is None:  # -1 at rest; every plan resets the entries it used
        slot_map = _DENSE_SLOT_MAPS[key] = torch.full((V,), -1, dtype=torch.int32, device=dev)
    plan = SparseTablePlan(None, [ids], slot_map, vocab=V, dim=D)
    plan.add_rows(ids, rows)
    g = torch.zeros(V, D, device=dev, dtype=torch.float32)
    call("asme_scatter_rows", ptr(plan.grad_rows), ptr(plan.unique), ptr(plan.count), plan.capacity, D, ptr(g), V,
         stream())
    plan.release()
    return g


def scatter_add_rows(rows: torch.Tensor, ids: torch.Tensor, dest: torch.Tensor, scale: float = 1.0):
    """dest[ids[r]] += scale * rows[r]  (fp32 atomics)"""
    rows, ids = _f32(rows), _i64(ids)
    call("asme_scatter_add_rows", ptr(rows), ptr(ids), ids.numel(), rows.shape[1], ptr(dest), dest.shape[0], scale,
         stream())


def _reduce_rows(x: torch.Tensor) -> torch.Tensor:
    x = _f32(x)
    out = torch.empty(x.shape[-1], device=x.device, dtype=torch.float32)
    call("asme_reduce_rows", ptr(x), x.numel() // x.shape[-1], x.shape[-1], ptr(out), 0, stream())
    return out


def gather_rows(ids: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """table[ids] (no autograd; zero rows for ids outside the table) on asme_gather_rows"""
    ids = _i64(ids).reshape(-1)
    V, D = table.shape
    out = torch.empty(ids.numel(), D, device=table.device, dtype=torch.float32)
    if ids.numel():
        call("asme_gather_rows", ptr(ids), ids.numel(), ptr(_f32(table)), V, D, ptr(out), stream())
    return out


def padding_mask(seq: torch.Tensor, pad: int) -> torch.Tensor:
    """seq != pad as a bool tensor of seq's shape (asme_padding_mask)"""
    seq = seq.contiguous()
    if seq.data_ptr() % 16:  # a view at an odd offset: the kernel reads 16-B pairs
        return seq.ne(pad)
    out = torch.empty(seq.shape, device=seq.device, dtype=torch.bool)
    call("asme_padding_mask", ptr(seq), seq.numel(), int(pad), ptr(out), stream())
    return out


def row_inverse(rows: torch.Tensor, n: int) -> torch.Tensor:
    """inverse[t] = k where rows[k] = t, else -1 (int64, n entries) -- the map select_rows' backward reads"""
    inv = torch.full((n,), -1, dtype=torch.int64, device=rows.device)
    inv[rows] = torch.arange(rows.numel(), device=rows.device)
    return inv


class _SelectRowsFn(torch.autograd.Function):
    """x2[rows] for distinct row indices (the masked / predicted positions of a flattened (B*L, d) representation)
    on asme_gather_rows.  The backward is the same kernel reading the inverse map: row t of the dense (T, d) input
    gradient is the gradient of the selected row that came from t, and a zero row (id -1, outside the table)
    everywhere else -- one launch instead of a zero fill plus an index_add."""

    @staticmethod
    def forward(ctx, x2, rows, inverse):
        ctx.save_for_backward(rows, inverse)
        ctx.n = x2.shape[0]
        return gather_rows(rows, x2)

    @staticmethod
    def backward(ctx, g):
        rows, inverse = ctx.saved_tensors
        if rows.numel() == 0:
            return g.new_zeros(ctx.n, g.shape[-1]), None, None
        if inverse is None:
            inverse = row_inverse(rows, ctx.n)
        return gather_rows(inverse, g.contiguous()), None, None


def select_rows(x2: torch.Tensor, rows: torch.Tensor, inverse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x2[rows] (x2: (T, d), rows: distinct indices) with the backward above; `inverse` (row_inverse(rows, T)) may be
    built ahead, e.g. on the producer's side stream, else the backward builds it"""
    if x2.shape[-1] > 512:  # wider than asme_gather_rows takes
        return x2.index_select(0, rows)
    return _SelectRowsFn.apply(x2.contiguous(), _i64(rows).reshape(-1), inverse)


def bucket_by_owner(unique: torch.Tensor, world: int, count: Optional[torch.Tensor] = None,
                    split: Optional[torch.Tensor] = None):
    """stable grouping of unique ids by owner (id % world): (order, send_local, counts (int64, world), pos) with
    unique[order[j]] the j-th id sent, send_local[j] its owner-local row, pos[order[j]] = j.  count (int32 (1,) on
    the device, optional): only unique[:count] take part, the outputs past it are unspecified (no host sync).
    split (int32 (1,) on the device, optional): two classes -- unique[:split] by owner, then the rest by owner;
    counts then has 2 * world entries, class-major (asme_bucket_by_owner_split)"""
    u = _i64(unique).reshape(-1)
    n = u.numel()
    dev = u.device
    nbk = 2 * world if split is not None else world
    ws = torch.empty(max(8, int(_lib.load().asme_bucket_by_owner_workspace(n, nbk))), device=dev, dtype=torch.uint8)
    order = torch.empty(n, device=dev, dtype=torch.int64)
    send_local = torch.empty(n, device=dev, dtype=torch.int32)
    counts = torch.empty(nbk, device=dev, dtype=torch.int64)
    pos = torch.empty(n, device=dev, dtype=torch.int64)
    if split is None:
        call("asme_bucket_by_owner", ptr(u), n, ptr(count), world, ptr(ws), ws.numel(), ptr(order), ptr(send_local),
             ptr(counts), ptr(pos), stream())
    else:
        sp = split.to(torch.int32).reshape(1)
        call("asme_bucket_by_owner_split", ptr(u), n, ptr(count), world, ptr(sp), ptr(ws), ws.numel(), ptr(order),
             ptr(send_local), ptr(counts), ptr(pos), stream())
    return order, send_local, counts, pos


def gather_sum(ids, table, bias=None, skip_zero=False, multi_hot=None):
    """sum over the last id dimension of table rows (+ bias): multi_hot (default: skip_zero) = (..., K) ids summed
    per position (LinearUpscaler: the pad category 0 skipped; UBERT4Rec's user upscaler counts it), else one row
    per id (nn.Embedding)"""
    return _GatherSumFn.apply(ids, table, bias, skip_zero, skip_zero if multi_hot is None else multi_hot)


# ------------------------------------------------------------------------------------ linear
_WS_SUPPORTED = {}


def _ws_ok(M: int, K: int, N: int) -> bool:
    """(M, K, N) runs on the weight-stationary MFMA GEMM (csrc/wsgemm.hip)"""
    key = (M, K, N)
    if key not in _WS_SUPPORTED:
        _WS_SUPPORTED[key] = bool(_lib.load().asme_ws_linear_supported(M, K, N))
    return _WS_SUPPORTED[key]


def _ws(x2, w, N: int, trans: int, bias=None, epi: int = 0, pre_out=None, pre_in=None, p: float = 0.0,
        seed: int = 0):
    """Y = x2 . w^T (+ bias) (trans = 0, w: N x K) or x2 . w (trans = 1, w: K x N) with epilogue epi"""
    M, K = x2.shape
    y = torch.empty(M, N, device=x2.device, dtype=torch.float32)
    call("asme_ws_linear", ptr(x2), M, K, ptr(w), N, trans, ptr(bias), epi, ptr(pre_out), ptr(pre_in), p, seed,
         ptr(y), stream())
    return y


def _weight_grad(dy2, x2, has_bias: bool):
    """dW = dY^T X, db = sum_t dY on the split-token MFMA kernel (asme_linear_weight_grad)"""
    dy2, x2 = _f32(dy2), _f32(x2)
    T, N = dy2.shape
    K = x2.shape[1]
    if N % 4 or K % 4:  # shapes the kernel does not tile: library GEMM
        return dy2.t() @ x2, (dy2.sum(0) if has_bias else None)
    nbytes = int(_lib.load().asme_linear_weight_grad_workspace(T, N, K))
    ws = torch.empty(max(4, nbytes // 4), device=dy2.device, dtype=torch.float32)
    dw = torch.empty(N, K, device=dy2.device, dtype=torch.float32)
    db = torch.empty(N, device=dy2.device, dtype=torch.float32) if has_bias else None
    call("asme_linear_weight_grad", ptr(dy2), N, ptr(x2), K, T, N, K, ptr(ws), nbytes, ptr(dw), ptr(db), 0, stream())
    return dw, db


def _tile4_ok(*ts) -> bool:
    """shapes the general fp32-MFMA Linear kernels (csrc/linear.hip) take: contiguous, every row a multiple
    of 4 floats, 16-B aligned"""
    return all(t.is_contiguous() and t.shape[-1] % 4 == 0 and t.data_ptr() % 16 == 0 for t in ts)


def _linear_fwd(x2, w, b):
    """x2 . w^T + b: the weight-stationary bf16x6 GEMM where it tiles (K in {128..512}), otherwise the
    general fp32-MFMA kernel (asme_linear_fwd); a library GEMM only for rows that are not a multiple of 4
    floats (no kernel here tiles them)"""
    M, K = x2.shape
    N = w.shape[0]
    w = _f32(w)
    b = _f32(b) if b is not None else None
    if _ws_ok(M, K, N):
        return _ws(x2, w, N, 0, bias=b)
    if _tile4_ok(x2, w) and N % 4 == 0:
        y = torch.empty(M, N, device=x2.device, dtype=torch.float32)
        call("asme_linear_fwd", ptr(x2), K, M, K, ptr(w), ptr(b), N, ptr(y), N, stream())
        return y
    return torch.nn.functional.linear(x2, w, b)


def _linear_dx(dy2, w):
    """dy2 . w (the input gradient of a Linear with weight w: N x K), same kernel choice as _linear_fwd"""
    M, N = dy2.shape
    K = w.shape[1]
    w = _f32(w)
    if _ws_ok(M, N, K):
        return _ws(dy2, w, K, 1)
    if _tile4_ok(dy2, w) and N % 4 == 0:
        dx = torch.empty(M, K, device=dy2.device, dtype=torch.float32)
        call("asme_linear_dx", ptr(dy2), N, M, N, ptr(w), K, ptr(dx), K, 0, stream())
        return dx
    return dy2 @ w


class _LinearFn(torch.autograd.Function):
    """nn.Linear on the weight-stationary MFMA GEMM (forward and input gradient; library GEMM for shapes it
    does not take) with the weight/bias gradient on the split-token MFMA kernel (asme_linear_weight_grad)."""

    @staticmethod
    def forward(ctx, x, w, b):
        N, K = w.shape
        x2 = _f32(x).reshape(-1, K)
        ctx.save_for_backward(x2, w)
        ctx.has_bias = b is not None
        ctx.xshape = x.shape
        return _linear_fwd(x2, w, b).view(*x.shape[:-1], N)

    @staticmethod
    def backward(ctx, dy):
        x2, w = ctx.saved_tensors
        N, K = w.shape
        dy2 = _f32(dy).reshape(-1, N)
        dx = _linear_dx(dy2, w).view(ctx.xshape) if ctx.needs_input_grad[0] else None
        dw = db = None
        if ctx.needs_input_grad[1] or (ctx.has_bias and ctx.needs_input_grad[2]):
            dw, db = _weight_grad(dy2, x2, ctx.has_bias)
        return dx, dw, db


def linear(x, w, b=None):
    return _LinearFn.apply(x, w, b)


def adjacent_rows(parts: Sequence[torch.Tensor]) -> Optional[torch.Tensor]:
    """the tensors' rows as ONE tensor when they are consecutive row blocks of one buffer (a view, no copy), else None"""
    t0 = parts[0]
    if not all(t.is_contiguous() and t.dtype == t0.dtype and t.device == t0.device and t.shape[1:] == t0.shape[1:]
               for t in parts):
        return None
    if any(t.untyped_storage().data_ptr() != t0.untyped_storage().data_ptr() for t in parts):
        return None
    row = t0[0].numel() if t0.dim() > 1 else 1
    off = t0.storage_offset()
    for t in parts:
        if t.storage_offset() != off:
            return None
        off += t.shape[0] * row
    rows = sum(t.shape[0] for t in parts)
    return t0.detach().as_strided((rows,) + tuple(t0.shape[1:]), t0.stride())


def fuse_rows_(params: Sequence[torch.nn.Parameter]) -> None:
    """re-home parameters onto consecutive row blocks of one new buffer (values unchanged), so adjacent_rows finds
    them; optimizer state is keyed by the parameter objects and is unaffected"""
    with torch.no_grad():
        buf = torch.cat([p.detach() for p in params], 0)
        r = 0
        for p in params:
            p.data = buf[r:r + p.shape[0]]
            r += p.shape[0]


class _RowPartsLinearFn(torch.autograd.Function):
    """_LinearFn for a weight / bias given as k row blocks that lie consecutively in one buffer (W, B views of it):
    the GEMMs read the buffer in place (no per-forward concatenation) and each block's gradient is a row block of
    the one fused weight / bias gradient."""

    @staticmethod
    def forward(ctx, x, W, B, *parts):
        N, K = W.shape
        x2 = _f32(x).reshape(-1, K)
        ctx.save_for_backward(x2, W)
        ctx.xshape = x.shape
        ctx.rows = [t.shape[0] for t in parts[:len(parts) // 2]]
        return _linear_fwd(x2, W, B).view(*x.shape[:-1], N)

    @staticmethod
    def backward(ctx, dy):
        x2, W = ctx.saved_tensors
        N, K = W.shape
        dy2 = _f32(dy).reshape(-1, N)
        dx = _linear_dx(dy2, W).view(ctx.xshape) if ctx.needs_input_grad[0] else None
        dw, db = _weight_grad(dy2, x2, True)
        gw, gb, r = [], [], 0
        for n in ctx.rows:
            gw.append(dw[r:r + n])
            gb.append(db[r:r + n])
            r += n
        return (dx, None, None, *gw, *gb)


def linear_row_parts(x, weights: Sequence[torch.Tensor], biases: Sequence[torch.Tensor]):
    """linear(x, cat(weights), cat(biases)) without the concatenation when the blocks are adjacent in memory"""
    W, B = adjacent_rows(weights), adjacent_rows(biases)
    if W is None or B is None:
        return linear(x, torch.cat(list(weights), 0), torch.cat(list(biases), 0))
    return _RowPartsLinearFn.apply(x, W, B, *weights, *biases)


class _FFNFn(torch.autograd.Function):
    """PositionwiseFeedForward W2(dropout(GELU_erf(W1 x + b1))) + b2 (transformer_layers.py:212-220) with the
    activation fused into the GEMMs: forward GEMM1 writes dropout(GELU(pre)) and the activation factor
    A = keep * GELU'(pre); the backward input-gradient GEMM of W2 multiplies by A in its epilogue.  Same dropout
    decisions as gelu_dropout (salt 5, element index over the (T, d_ff) activation)."""

    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, p: float):
        F, D = w1.shape
        x2 = _f32(x).reshape(-1, D)
        M = x2.shape[0]
        seed = new_seed(p)
        fac = torch.empty(M, F, device=x.device, dtype=torch.float32)
        g = _ws(x2, w1, F, 0, bias=b1, epi=1, pre_out=fac, p=p, seed=seed)
        y = _linear_fwd(g, w2, b2)
        ctx.save_for_backward(x2, fac, g, w1, w2)
        ctx.meta = (p, seed, b1 is not None, b2 is not None, x.shape)
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2, fac, g, w1, w2 = ctx.saved_tensors
        p, seed, hb1, hb2, xshape = ctx.meta
        F, D = w1.shape
        dy2 = _f32(dy).reshape(-1, D)
        d_pre = _ws(dy2, w2, F, 1, epi=2, pre_in=fac, p=p, seed=seed)
        dw2, db2 = _weight_grad(dy2, g, hb2)
        dx = _linear_dx(d_pre, w1).view(xshape) if ctx.needs_input_grad[0] else None
        dw1, db1 = _weight_grad(d_pre, x2, hb1)
        return dx, dw1, db1, dw2, db2, None


def ffn(x, w1, b1, w2, b2, p: float = 0.0):
    """W2(dropout(GELU(W1 x + b1))) + b2; fused on the weight-stationary GEMM when the shapes allow"""
    F, D = w1.shape
    M = x.numel() // D
    if (_ws_ok(M, D, F) and _ws_ok(M, F, D) and w1.is_contiguous() and w2.is_contiguous()
            and b1 is not None and b1.is_contiguous()):
        return _FFNFn.apply(x, w1, b1, w2, b2, p)
    return linear(gelu_dropout(linear(x, w1, b1), p), w2, b2)


class _DropoutFn(torch.autograd.Function):
    """nn.Dropout in training mode on asme_dropout; the backward replays the decisions from the seed"""

    @staticmethod
    def forward(ctx, x, p: float):
        xc = _f32(x)
        seed = new_seed(p)
        y = torch.empty_like(xc)
        call("asme_dropout", ptr(xc), xc.numel(), p, seed, ptr(y), stream())
        ctx.meta = (p, seed)
        return y

    @staticmethod
    def backward(ctx, dy):
        p, seed = ctx.meta
        g = _f32(dy)
        dx = torch.empty_like(g)
        call("asme_dropout", ptr(g), g.numel(), p, seed, ptr(dx), stream())
        return dx, None


def dropout(x, p: float):
    return _DropoutFn.apply(x, p) if p > 0.0 else x


class _DropoutRowsFn(torch.autograd.Function):
    """nn.Dropout2d in training mode on (N, C, L): whole rows of L values dropped together (asme_dropout_rows)"""

    @staticmethod
    def forward(ctx, x, p: float):
        xc = _f32(x)
        seed = new_seed(p)
        y = torch.empty_like(xc)
        call("asme_dropout_rows", ptr(xc), xc.numel(), xc.shape[-1], p, seed, ptr(y), stream())
        ctx.meta = (p, seed)
        return y

    @staticmethod
    def backward(ctx, dy):
        p, seed = ctx.meta
        g = _f32(dy)
        dx = torch.empty_like(g)
        call("asme_dropout_rows", ptr(g), g.numel(), g.shape[-1], p, seed, ptr(dx), stream())
        return dx, None


def dropout_rows(x, p: float):
    """Dropout2d semantics for a 3-D (N, C, L) input (torch 1.11 and 2.10 alike): one draw per (n, c) row"""
    return _DropoutRowsFn.apply(x, p) if p > 0.0 else x


# ------------------------------------------------------------------------------------ NARM encoders
def _pad_hidden(t: torch.Tensor, H: int, hp: int, cols: bool = False) -> torch.Tensor:
    """(3H, K) / (3H,) gate-stacked GRU parameter -> (3hp, K') with each gate block zero-padded to hp rows
    (and, cols=True, the K = H columns to hp); differentiable, a no-op when H == hp"""
    if hp == H:
        return t
    g = t.reshape(3, H, -1)
    g = torch.nn.functional.pad(g, (0, hp - H if cols else 0, 0, hp - H))
    return g.reshape(3 * hp, -1) if t.dim() == 2 else g.reshape(3 * hp)


class _GRULayerFn(torch.autograd.Function):
    """One nn.GRU layer (batch_first, h_0 = 0) on the hand kernels (core/models/narm/components.py:32-56): the input
    half x W_ih^T + b_ih for all steps as one Linear GEMM, the recurrence on asme_gru_fwd; backward through time on
    asme_gru_bwd, then dX, dW_ih, db_ih, dW_hh, db_hh as Linear / weight-gradient GEMMs over all steps.  Parameters
    arrive padded to hp hidden units (zero rows / columns), x (B, L, K) with K the padded width of the layer below."""

    @staticmethod
    def forward(ctx, x, w_ih, b_ih, w_hh, b_hh):
        B, L, K = x.shape
        hp = w_hh.shape[1]
        x2 = _f32(x).reshape(B * L, K)
        w_hh = _f32(w_hh)
        gx = _linear_fwd(x2, _f32(w_ih), _f32(b_ih))
        hout = torch.empty(B, L, hp, device=x.device, dtype=torch.float32)
        gates = torch.empty(B, L, 4, hp, device=x.device, dtype=torch.float32)
        call("asme_gru_fwd", ptr(gx), ptr(w_hh), ptr(_f32(b_hh)), None, B, L, hp, ptr(hout), ptr(gates), stream())
        ctx.save_for_backward(x2, w_ih, w_hh, hout, gates)
        ctx.shape = (B, L, K)
        return hout

    @staticmethod
    def backward(ctx, dh):
        x2, w_ih, w_hh, hout, gates = ctx.saved_tensors
        B, L, K = ctx.shape
        hp = w_hh.shape[1]
        dgx = torch.empty(B * L, 3 * hp, device=dh.device, dtype=torch.float32)
        dgh = torch.empty_like(dgx)
        call("asme_gru_bwd", ptr(_f32(dh)), None, ptr(w_hh), None, ptr(hout), ptr(gates), B, L, hp, ptr(dgx),
             ptr(dgh), None, stream())
        dx = _linear_dx(dgx, _f32(w_ih)).view(B, L, K) if ctx.needs_input_grad[0] else None
        dw_ih, db_ih = _weight_grad(dgx, x2, True)
        hprev = torch.cat([hout.new_zeros(B, 1, hp), hout[:, :-1]], dim=1).reshape(B * L, hp)
        dw_hh, db_hh = _weight_grad(dgh, hprev, True)
        return dx, dw_ih, db_ih, dw_hh, db_hh


def gru(x: torch.Tensor, module: torch.nn.GRU) -> torch.Tensor:
    """outputs h_i (B, L, H) of the last layer of a batch_first, unidirectional nn.GRU run from h_0 = 0 over the
    padded batch (causal: identical to the packed run at every valid position)"""
    if not module.batch_first or module.bidirectional or module.proj_size or (module.dropout and module.training
                                                                              and module.num_layers > 1):
        raise NotImplementedError("asme gru: batch_first, unidirectional, no projection, no inter-layer dropout")
    H = module.hidden_size
    hp = -(-H // 16) * 16
    if hp > 128:
        # wider than the register-resident W_hh of csrc/narm.hip (the reference configs use 128 and 30): the
        # library GRU on the same device (MIOpen), as before the kernel existed; a CPU tensor still raises
        if not x.is_cuda:
            raise _lib.ASMEKernelError("asme gru: tensors must be on the ROCm device")
        return module(x)[0]
    h = x
    for k in range(module.num_layers):
        w_ih = getattr(module, f"weight_ih_l{k}")
        w_hh = getattr(module, f"weight_hh_l{k}")
        b_ih = getattr(module, f"bias_ih_l{k}") if module.bias else w_ih.new_zeros(3 * H)
        b_hh = getattr(module, f"bias_hh_l{k}") if module.bias else w_hh.new_zeros(3 * H)
        h = _GRULayerFn.apply(h, _pad_hidden(w_ih, H, hp, cols=k > 0), _pad_hidden(b_ih, H, hp),
                              _pad_hidden(w_hh, H, hp, cols=True), _pad_hidden(b_hh, H, hp))
    return h if hp == H else h[..., :H].contiguous()


class _NarmAttendFn(torch.autograd.Function):
    """LocalEncoderLayer's v . sigmoid(A1 c_g + A2 h_i) attention and masked weighted sum (core/models/narm/
    layers.py:32-66) after the two projections, on asme_narm_attend_fwd / _bwd"""

    @staticmethod
    def forward(ctx, p1, p2, v, hs, mask):
        N, S, H = hs.shape
        p1, p2, v, hs = _f32(p1), _f32(p2), _f32(v), _f32(hs)
        m = as_u8(mask)
        out = torch.empty(N, H, device=hs.device, dtype=torch.float32)
        alpha = torch.empty(N, S, device=hs.device, dtype=torch.float32)
        call("asme_narm_attend_fwd", ptr(p1), ptr(p2), ptr(v), ptr(hs), ptr(m), N, S, H, ptr(out), ptr(alpha),
             stream())
        ctx.save_for_backward(p1, p2, v, hs, m, alpha)
        return out

    @staticmethod
    def backward(ctx, dc):
        p1, p2, v, hs, m, alpha = ctx.saved_tensors
        N, S, H = hs.shape
        dp1 = torch.empty_like(p1)
        dp2 = torch.empty_like(p2)
        dhs = torch.empty_like(hs)
        dv_part = torch.empty(N, H, device=hs.device, dtype=torch.float32)
        call("asme_narm_attend_bwd", ptr(_f32(dc)), ptr(p1), ptr(p2), ptr(v), ptr(hs), ptr(m), ptr(alpha), N, S, H,
             ptr(dp1), ptr(dp2), ptr(dhs), ptr(dv_part), stream())
        return dp1, dp2, _reduce_rows(dv_part), dhs, None


def narm_attend(p1, p2, v, hs, mask):
    return _NarmAttendFn.apply(p1, p2, v, hs, mask)


# ------------------------------------------------------------------------------------ layer norm
class _LayerNormFn(torch.autograd.Function):
    """nn.LayerNorm over the last dim (fp32, biased variance)."""

    @staticmethod
    def forward(ctx, x, w, b, eps: float):
        shape = x.shape
        D = shape[-1]
        x2 = _f32(x).reshape(-1, D)
        n = x2.shape[0]
        y = torch.empty_like(x2)
        stats = torch.empty(n, 2, device=x.device, dtype=torch.float32)
        call("asme_layernorm_fwd", ptr(x2), n, D, ptr(w), ptr(b), eps, ptr(y), ptr(stats), stream())
        ctx.save_for_backward(x2, w, stats)
        return y.view(shape)

    @staticmethod
    def backward(ctx, dy):
        x2, w, stats = ctx.saved_tensors
        n, D = x2.shape
        dy2 = _f32(dy).reshape(n, D)
        dx = torch.empty_like(x2)
        part = torch.empty(_N_PARTIALS, 2 * D, device=x2.device, dtype=torch.float32)
        call("asme_layernorm_bwd", ptr(x2), n, D, ptr(w), ptr(stats), ptr(dy2), ptr(dx), 0, ptr(part), _N_PARTIALS,
             stream())
        red = _reduce_partials(part, 2 * D)
        return dx.view(dy.shape), red[:D], red[D:], None


def layer_norm(x, norm: torch.nn.LayerNorm):
    return _LayerNormFn.apply(x, norm.weight, norm.bias, norm.eps)


class _LayerNormPassFn(torch.autograd.Function):
    """(x, LN(x)) for a tensor that feeds both a LayerNorm and a residual (the first pre-LN block's input,
    transformer_layers.py:120-130): the backward sums the two gradients of x inside the LN backward pass."""

    @staticmethod
    def forward(ctx, x, w, b, eps: float):
        shape = x.shape
        D = shape[-1]
        x2 = _f32(x).reshape(-1, D)
        n = x2.shape[0]
        y = torch.empty_like(x2)
        stats = torch.empty(n, 2, device=x.device, dtype=torch.float32)
        call("asme_layernorm_fwd", ptr(x2), n, D, ptr(w), ptr(b), eps, ptr(y), ptr(stats), stream())
        ctx.save_for_backward(x2, w, stats)
        return x.view_as(x), y.view(shape)

    @staticmethod
    def backward(ctx, d_x, dy):
        x2, w, stats = ctx.saved_tensors
        n, D = x2.shape
        if dy is None:
            return d_x, None, None, None
        dy2 = _f32(dy).reshape(n, D)
        dadd = None if d_x is None else _f32(d_x).reshape(n, D)
        dx = torch.empty_like(x2)
        part = torch.empty(_N_PARTIALS, 2 * D, device=x2.device, dtype=torch.float32)
        call("asme_layernorm_bwd_add", ptr(x2), n, D, ptr(w), ptr(stats), ptr(dy2), ptr(dadd), ptr(dx), ptr(part),
             _N_PARTIALS, stream())
        red = _reduce_partials(part, 2 * D)
        return dx.view(dy.shape), red[:D], red[D:], None


def layer_norm_pass(x, norm: torch.nn.LayerNorm):
    """(x, norm(x)); use the returned x wherever x is used again so its gradients meet in one pass"""
    return _LayerNormPassFn.apply(x, norm.weight, norm.bias, norm.eps)


class _ResidualLNFn(torch.autograd.Function):
    """SublayerConnection epilogue + block dropout + next pre-LN (transformer_layers.py:120-130, 251-258):
    s = drop_b(res + drop_a(y));  ln = LN(s)"""

    @staticmethod
    def forward(ctx, res, y, w, b, eps: float, p_a: float, p_b: float):
        shape = res.shape
        D = shape[-1]
        r2 = _f32(res).reshape(-1, D)
        y2 = _f32(y).reshape(-1, D)
        n = r2.shape[0]
        s = torch.empty_like(r2)
        has_ln = w is not None
        ln = torch.empty_like(r2) if has_ln else None
        stats = torch.empty(n, 2, device=res.device, dtype=torch.float32) if has_ln else None
        sa, sb = new_seed(p_a), new_seed(p_b)
        call("asme_residual_ln_fwd", ptr(r2), ptr(y2), n, D, p_a, sa, p_b, sb, ptr(w), ptr(b), eps, ptr(s), ptr(ln),
             ptr(stats), stream())
        ctx.save_for_backward(s, w, stats)
        ctx.meta = (p_a, sa, p_b, sb, has_ln, shape)
        if has_ln:
            return s.view(shape), ln.view(shape)
        return s.view(shape), s.new_empty(0)

    @staticmethod
    def backward(ctx, d_s, d_ln):
        s, w, stats = ctx.saved_tensors
        p_a, sa, p_b, sb, has_ln, shape = ctx.meta
        d_res, dy, gw, gb = _residual_ln_backward(s, w, stats, (p_a, sa, p_b, sb, has_ln), d_s, d_ln)
        return d_res.view(shape), dy.view(shape), gw, gb, None, None, None


def _residual_ln_backward(s, w, stats, meta, d_s, d_ln):
    """(d_res, d_y, d_w, d_b) of s = drop_b(res + drop_a(y)), ln = LN(s) (asme_residual_ln_bwd)"""
    p_a, sa, p_b, sb, has_ln = meta
    n, D = s.shape
    ds2 = None if d_s is None else _f32(d_s).reshape(n, D)
    dl2 = None if (d_ln is None or not has_ln) else _f32(d_ln).reshape(n, D)
    d_res = torch.empty_like(s)
    d_y = torch.empty_like(s) if p_a > 0 else None
    part = torch.empty(_N_PARTIALS, 2 * D, device=s.device, dtype=torch.float32) if dl2 is not None else None
    call("asme_residual_ln_bwd", ptr(s), n, D, p_a, sa, p_b, sb, ptr(w), ptr(stats), ptr(ds2), ptr(dl2),
         ptr(d_res), ptr(d_y), ptr(part), _N_PARTIALS, stream())
    gw = gb = None
    if has_ln:
        if part is not None:
            red = _reduce_partials(part, 2 * D)
            gw, gb = red[:D], red[D:]
        else:
            gw, gb = torch.zeros_like(w), torch.zeros_like(w)
    return d_res, (d_y if d_y is not None else d_res), gw, gb


class _LinearResidualLNFn(torch.autograd.Function):
    """_LinearFn followed by _ResidualLNFn as ONE kernel (asme_ws_linear_residual_ln: the residual, dropouts and the
    next pre-LN in the GEMM's epilogue, no Y round trip): s = drop_b(res + drop_a(x W^T + b)), ln = LN(s).  The
    attention output projection and the SublayerConnection around it (transformer_layers.py:120-130, 181-199,
    251-258).  Values and gradients are bit-identical to the two separate ops with the same seeds; the backward is
    theirs (asme_residual_ln_bwd, then the Linear's input and weight gradients)."""

    @staticmethod
    def forward(ctx, x, w, b, res, ln_w, ln_b, eps: float, p_a: float, p_b: float):
        shape = res.shape
        N, K = w.shape
        x2 = _f32(x).reshape(-1, K)
        r2 = _f32(res).reshape(-1, N)
        n = r2.shape[0]
        s = torch.empty_like(r2)
        has_ln = ln_w is not None
        ln = torch.empty_like(r2) if has_ln else None
        stats = torch.empty(n, 2, device=res.device, dtype=torch.float32) if has_ln else None
        sa, sb = new_seed(p_a), new_seed(p_b)  # (drawn in _ResidualLNFn's order)
        call("asme_ws_linear_residual_ln", ptr(x2), n, K, ptr(_f32(w)), N, ptr(_f32(b)) if b is not None else None,
             ptr(r2), p_a, sa, p_b, sb, ptr(ln_w), ptr(ln_b), eps, ptr(s), ptr(ln), ptr(stats), stream())
        ctx.save_for_backward(x2, w, s, ln_w, stats)
        ctx.meta = (p_a, sa, p_b, sb, has_ln)
        ctx.has_bias = b is not None
        ctx.shapes = (x.shape, shape)
        if has_ln:
            return s.view(shape), ln.view(shape)
        return s.view(shape), s.new_empty(0)

    @staticmethod
    def backward(ctx, d_s, d_ln):
        x2, w, s, ln_w, stats = ctx.saved_tensors
        xshape, shape = ctx.shapes
        d_res, d_y, gw, gb = _residual_ln_backward(s, ln_w, stats, ctx.meta, d_s, d_ln)
        N, K = w.shape
        dx = _linear_dx(d_y, w).view(xshape) if ctx.needs_input_grad[0] else None
        dw = db = None
        if ctx.needs_input_grad[1] or (ctx.has_bias and ctx.needs_input_grad[2]):
            dw, db = _weight_grad(d_y, x2, ctx.has_bias)
        return dx, dw, db, d_res.view(shape), gw, gb, None, None, None


def linear_residual_ln_ok(x: torch.Tensor, w: torch.Tensor, res: torch.Tensor) -> bool:
    """the fused output projection + residual + LayerNorm kernel takes this call"""
    N, K = w.shape
    if not (x.is_cuda and x.dtype == torch.float32 and w.dtype == torch.float32 and res.dtype == torch.float32
            and x.shape[-1] == K and res.shape[-1] == N and x.shape[:-1] == res.shape[:-1]):
        return False
    M = res.numel() // N
    key = ("rln", M, K, N)
    if key not in _WS_SUPPORTED:
        _WS_SUPPORTED[key] = bool(_lib.load().asme_ws_linear_residual_ln_supported(M, K, N))
    return _WS_SUPPORTED[key]


def linear_residual_ln(x, w, b, res, norm: Optional[torch.nn.LayerNorm], p_a: float, p_b: float):
    """(s, LN(s) or None) with s = drop_b(res + drop_a(linear(x, w, b))) in one kernel (linear_residual_ln_ok)"""
    if norm is None:
        s, _ = _LinearResidualLNFn.apply(x, w, b, res, None, None, 1e-5, p_a, p_b)
        return s, None
    return _LinearResidualLNFn.apply(x, w, b, res, norm.weight, norm.bias, norm.eps, p_a, p_b)


def residual_ln(res, y, norm: Optional[torch.nn.LayerNorm], p_a: float, p_b: float):
    if norm is None:
        s, _ = _ResidualLNFn.apply(res, y, None, None, 1e-5, p_a, p_b)
        return s, None
    return _ResidualLNFn.apply(res, y, norm.weight, norm.bias, norm.eps, p_a, p_b)


class _GatedResidualNormFn(torch.autograd.Function):
    """s = residual_scale * res + gate * Npost(y);  z = Npre(s)  (csrc/gatednorm.hip)"""

    @staticmethod
    def forward(ctx, res, y, gate, post_w, post_b, pre_w, pre_b, rows_per_gate: int, residual_scale: float, eps: float,
                rms: bool):
        ctx.set_materialize_grads(False)
        ctx.types = tuple(None if w is None else w.dtype for w in (post_w, post_b, pre_w, pre_b))
        res, y, gate = (None if t is None else _aligned(t) for t in (res, y, gate))
        post_w, post_b, pre_w, pre_b = (None if w is None else w.to(torch.float32).contiguous()
                                        for w in (post_w, post_b, pre_w, pre_b))
        D = res.shape[-1]
        n = res.numel() // D
        s = torch.empty_like(res)
        z = torch.empty_like(res) if pre_w is not None else None
        stats = torch.empty(n, 4, device=res.device, dtype=torch.float32)
        _call_on(res, "asme_gated_residual_norm_fwd", ptr(res), ptr(y), ptr(gate), rows_per_gate, ptr(post_w),
                 ptr(post_b), ptr(pre_w), ptr(pre_b), n, D, residual_scale, eps, int(rms), _dtype_code(res), ptr(s),
                 ptr(z), ptr(stats))
        ctx.save_for_backward(res, y, gate, post_w, post_b, pre_w, stats)
        ctx.meta = (rows_per_gate, residual_scale, rms)
        return s, z

    @staticmethod
    @once_differentiable
    def backward(ctx, ds, dz):
        if ds is None and dz is None:
            return (None,) * 11
        res, y, gate, post_w, post_b, pre_w, stats = ctx.saved_tensors
        rows_per_gate, residual_scale, rms = ctx.meta
        D = res.shape[-1]
        n = res.numel() // D
        need = ctx.needs_input_grad
        ds, dz = (None if g is None else _aligned(g) for g in (ds, dz))
        dres = torch.empty_like(res) if need[0] else None
        dy = torch.empty_like(res) if need[1] else None
        dgate = torch.empty_like(gate) if need[2] else None
        dw = torch.empty(4, D, device=res.device, dtype=torch.float32) if any(need[3:7]) else None
        shared = n if gate is None or rows_per_gate == 1 else rows_per_gate
        ws, nb = _ws_bytes("asme_gated_residual_norm_bwd_workspace", n, D, shared, device=res.device)
        _call_on(res, "asme_gated_residual_norm_bwd", ptr(res), ptr(y), ptr(gate), rows_per_gate, ptr(post_w),
                 ptr(post_b), ptr(pre_w), n, D, residual_scale, int(rms), _dtype_code(res), ptr(stats), ptr(ds), ptr(dz),
                 ptr(dres), ptr(dy), ptr(dgate), ptr(dw), ptr(ws), nb)
        w = [dw[i].to(ctx.types[i]) if need[3 + i] else None for i in range(4)]
        return (dres, dy, dgate, w[0], w[1], w[2], w[3], None, None, None, None)


def gated_residual_norm(res: torch.Tensor, y: torch.Tensor, post_w: torch.Tensor,
                        post_b: Optional[torch.Tensor] = None, pre_w: Optional[torch.Tensor] = None,
                        pre_b: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                        residual_scale: float = 1.0, eps: float = 1e-5, rms: bool = False):
    """The end of a block and the start of the next: (s, z) with
        s = residual_scale * res + gate * Npost(y),   z = Npre(s)   (None without pre_w)
    over the last axis (up to 8192 values), N a LayerNorm or (rms=True) a root-mean-square norm with weight and optional
    bias.  gate: None, one value per channel (D,), or of res's rank with the trailing axes before the channels 1 --
    (B, 1, D): a gate per sequence -- or of res's shape; it multiplies as it is (a tanh or sigmoid is the caller's).
    res, y and gate of one dtype, float32 or bfloat16; the norms' weights of any floating type, their sums float32.
    Differentiable once in everything but residual_scale and eps."""
    D = res.shape[-1]
    if res.shape != y.shape or res.dim() < 1:
        raise ValueError(f"res {tuple(res.shape)} and y {tuple(y.shape)} differ")
    if not 1 <= D <= 8192:
        raise ValueError(f"{D} channels: expected 1 to 8192")
    if pre_w is None and pre_b is not None:
        raise ValueError("pre_b without pre_w")
    if not (math.isfinite(residual_scale) and 0.0 <= eps < math.inf):
        raise ValueError(f"residual_scale {residual_scale}, eps {eps}: expected finite numbers, eps >= 0")
    _dtype_code(res)
    _alike(res, res.dtype, y=y, gate=gate)
    weights = dict(post_w=post_w, post_b=post_b, pre_w=pre_w, pre_b=pre_b)
    _alike(res, **weights)
    for name, w in weights.items():
        if w is not None and (w.shape != (D,) or not w.is_floating_point()):
            raise ValueError(f"{name} {tuple(w.shape)} of {w.dtype}: expected {D} floating values")
    n = res.numel() // D
    per = 1
    if gate is not None:
        lead = gate.shape[:-1] if gate.dim() > 1 else (1,) * (res.dim() - 1)
        same = next((i for i, (a, b) in enumerate(zip(lead, res.shape)) if a != b), len(lead))
        if gate.shape[-1:] != (D,) or len(lead) != res.dim() - 1 or any(a != 1 for a in lead[same:]):
            raise ValueError(f"gate {tuple(gate.shape)} for rows {tuple(res.shape)}: expected ({D},), the rows' shape, "
                             "or that with 1 in trailing axes before the channels")
        per = n // max(1, gate.numel() // D)
    if n == 0:
        s = res + y + 0 * sum(t.sum() for t in (gate, *weights.values()) if t is not None)  # (of every input)
        return s, (s * 1 if pre_w is not None else None)
    return _GatedResidualNormFn.apply(res, y, gate, *weights.values(), per, float(residual_scale), float(eps), bool(rms))


class _GeluDropoutFn(torch.autograd.Function):
    """dropout(GELU_erf(x)) (transformer_layers.py:217-220; ffn_modifier.py:24-26 with p = 0)"""

    @staticmethod
    def forward(ctx, x, p: float):
        x = _f32(x)
        y = torch.empty_like(x)
        seed = new_seed(p)
        call("asme_gelu_dropout_fwd", ptr(x), x.numel(), p, seed, ptr(y), stream())
        ctx.save_for_backward(x)
        ctx.meta = (p, seed)
        return y

    @staticmethod
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        p, seed = ctx.meta
        dy = _f32(dy)
        dx = torch.empty_like(x)
        call("asme_gelu_dropout_bwd", ptr(x), ptr(dy), x.numel(), p, seed, ptr(dx), stream())
        return dx, None


def gelu_dropout(x, p: float = 0.0):
    return _GeluDropoutFn.apply(x, p)


# ------------------------------------------------------------------------------------ attention
def _mask_bytes(batch: int, heads: int, seq_len: int) -> int:
    return int(_lib.load().asme_attention_dropout_mask_bytes(batch, heads, seq_len))


def _attn_bwd_ws_bytes(batch: int, heads: int, seq_len: int, head_dim: int) -> int:
    return int(_lib.load().asme_attention_bwd_workspace(batch, heads, seq_len, head_dim))


class _AttentionFn(torch.autograd.Function):
    """Attention.forward (transformer_layers.py:138-155) on a fused (B, L, 3*H*dk) QKV tensor.
    key_valid (B, L) uint8; causal selects SASRec's tril mask (sequence_representation.py:34-48)."""

    @staticmethod
    def forward(ctx, qkv, key_valid, heads: int, causal: bool, p_drop: float, kernels: int):
        B, L, three_d = qkv.shape
        Dm = three_d // 3
        dk = Dm // heads
        qkv = _f32(qkv)
        out = torch.empty(B, L, Dm, device=qkv.device, dtype=torch.float32)
        lse = torch.empty(B * heads, L, 2, device=qkv.device, dtype=torch.float32)  # (max, 1/sum)
        seed = new_seed(p_drop)
        scale = 1.0 / math.sqrt(dk)
        base = qkv.data_ptr()
        mask = torch.empty(_mask_bytes(B, heads, L), device=qkv.device, dtype=torch.uint8) if p_drop > 0 else None
        if kernels == 0:
            call("asme_attention_fwd", base, base + 4 * Dm, base + 8 * Dm, three_d, three_d, three_d, ptr(key_valid),
                 B, heads, L, dk, int(causal), scale, p_drop, seed, ptr(out), Dm, ptr(lse), ptr(mask), stream())
        else:
            call("asme_attention_fwd_kernels", kernels, base, base + 4 * Dm, base + 8 * Dm, three_d, three_d, three_d,
                 ptr(key_valid), B, heads, L, dk, int(causal), scale, p_drop, seed, ptr(out), Dm, ptr(lse), ptr(mask),
                 stream())
        ctx.save_for_backward(qkv, key_valid, out, lse, mask)
        ctx.meta = (heads, causal, p_drop, seed, scale, kernels)
        return out

    @staticmethod
    def backward(ctx, dout):
        qkv, key_valid, out, lse, mask = ctx.saved_tensors
        heads, causal, p_drop, seed, scale, kernels = ctx.meta
        B, L, three_d = qkv.shape
        Dm = three_d // 3
        dk = Dm // heads
        dout = _f32(dout)
        dqkv = torch.empty_like(qkv)
        ws = torch.empty((_attn_bwd_ws_bytes(B, heads, L, dk) + 3) // 4, device=qkv.device, dtype=torch.float32)
        base, gb = qkv.data_ptr(), dqkv.data_ptr()
        args = (base, base + 4 * Dm, base + 8 * Dm, three_d, three_d, three_d, ptr(out), Dm, ptr(dout), Dm, ptr(lse),
                ptr(key_valid), B, heads, L, dk, int(causal), scale, p_drop, seed, ptr(mask), ptr(ws), gb, three_d,
                gb + 4 * Dm, three_d, gb + 8 * Dm, three_d, stream())
        if kernels == 0:
            call("asme_attention_bwd", *args)
        else:
            call("asme_attention_bwd_kernels", kernels, *args)
        return dqkv, None, None, None, None, None


def attention(qkv, key_valid, heads: int, causal: bool, p_drop: float = 0.0, kernels: int = 0):
    """kernels: the kernel family (asme_attention_fwd_kernels): 0 automatic (the product path); 1 streaming only and
    2 resident with the recomputing dQ pass for the kernel tests and A/B timing"""
    return _AttentionFn.apply(qkv, key_valid, heads, causal, p_drop, kernels)


def _strides(*ts):
    """the (batch, token, head) element strides of (B, L, heads, head_dim) tensors as a host array"""
    return (ctypes_i64 * (3 * len(ts)))(*(x for t in ts for x in t.stride()[:3]))


def _window_forward(q, k, v, valid, window, sinks, causal, scale, with_state):
    """(out, what the backward takes beside it: the rows' softmax state and, of bf16, what rounding took from out)"""
    B, L, H, D = q.shape
    out = torch.empty(B, L, H, D, device=q.device, dtype=q.dtype)
    state = torch.empty(B, H, L, 2, device=q.device, dtype=torch.float32) if with_state else None
    low = torch.empty_like(out) if with_state and out.dtype == torch.bfloat16 else None
    _call_on(q, "asme_window_attention_fwd", ptr(q), ptr(k), ptr(v), ptr(out), _strides(q, k, v, out), ptr(valid), B, H,
             k.shape[2], L, D, window, sinks, int(causal), scale, _dtype_code(q), ptr(low), ptr(state))
    return out, low, state


def _window_backward(q, k, v, valid, out, low, state, dout, grads, window, sinks, causal, scale):
    B, L, H, D = q.shape
    dout = _strided_heads(dout)
    ws, nb = _ws_bytes("asme_window_attention_bwd_workspace", B, H, k.shape[2], L, D, window, sinks, int(causal),
                       _dtype_code(q), device=q.device)
    _call_on(q, "asme_window_attention_bwd", ptr(q), ptr(k), ptr(v), ptr(out), ptr(dout), *(ptr(g) for g in grads),
             _strides(q, k, v, out, dout, *grads), ptr(valid), B, H, k.shape[2], L, D, window, sinks, int(causal), scale,
             _dtype_code(q), ptr(low), ptr(state), ptr(ws), nb)


class _WindowAttentionFn(torch.autograd.Function):
    """Sliding-window attention with sinks (csrc/window.hip) on separate q, k, v."""

    @staticmethod
    def forward(ctx, q, k, v, valid, *how):
        out, *kept = _window_forward(q, k, v, valid, *how, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(q, k, v, valid, out, *kept)
        ctx.how = how
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, valid, out, *kept = ctx.saved_tensors
        grads = [torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v)]
        _window_backward(q, k, v, valid, out, *kept, dout, grads, *ctx.how)
        return (*grads, *([None] * (1 + len(ctx.how))))


class _WindowAttentionQKVFn(torch.autograd.Function):
    """The same on one (B, L, heads + 2 kv_heads, head_dim) projection; its gradient is one buffer too."""

    @staticmethod
    def forward(ctx, qkv, valid, heads: int, *how):
        kv = (qkv.shape[2] - heads) // 2
        out, *kept = _window_forward(*qkv.split((heads, kv, kv), 2), valid, *how, ctx.needs_input_grad[0])
        ctx.save_for_backward(qkv, valid, out, *kept)
        ctx.how, ctx.parts = how, (heads, kv, kv)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, valid, out, *kept = ctx.saved_tensors
        grad = torch.empty(qkv.shape, device=qkv.device, dtype=qkv.dtype)
        _window_backward(*qkv.split(ctx.parts, 2), valid, out, *kept, dout, grad.split(ctx.parts, 2), *ctx.how)
        return (grad, None, None, *([None] * len(ctx.how)))


def _attention_scale(scale: Optional[float], D: int) -> float:
    if scale is not None and not 0.0 < scale < math.inf:
        raise ValueError(f"scale {scale}: expected a positive number")
    return D ** -0.5 if scale is None else float(scale)


def _check_window(q, heads: int, kv_heads: int, D: int, window: int, sinks: int, valid, scale):
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads for {kv_heads} key heads: expected a multiple")
    if D not in _HEAD_DIMS:
        raise ValueError(f"head_dim {D}: expected one of {_HEAD_DIMS}")
    if window < 1 or sinks < 0:
        raise ValueError(f"window {window}, sinks {sinks}: expected window >= 1, sinks >= 0")
    scale = _attention_scale(scale, D)
    if valid is not None and (valid.shape != q.shape[:2] or valid.dtype not in (torch.bool, torch.uint8)):
        raise ValueError(f"valid {tuple(valid.shape)} of {valid.dtype}: expected {tuple(q.shape[:2])} of bool")
    _dtype_code(q)
    _alike(q, valid=valid)
    return scale


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0,
                     causal: bool = True, valid: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None) -> torch.Tensor:
    """Attention over a sliding window with sinks: query i of a sequence sees key j iff 0 <= i - j < window or
    (j < sinks and j <= i); without `causal` iff |i - j| < window or j < sinks.  q (B, L, heads, head_dim), k and v
    (B, L, kv_heads, head_dim), heads a multiple of kv_heads, head_dim 16, 32, 64 or 128, float32 or bfloat16; views
    with adjacent head values are read in place.  valid (B, L): positions that are not valid (padding) are neither
    query nor key, whatever they hold; their rows of the output and of the gradients are 0.  scale: 1/sqrt(head_dim).
    Valid positions hold finite numbers (a NaN there reaches other rows of its tile).  Returns (B, L, heads, head_dim)."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: expected (B, L, heads, head_dim) "
                         "and twice (B, L, kv_heads, head_dim)")
    scale = _check_window(q, q.shape[2], k.shape[2], q.shape[3], window, sinks, valid, scale)
    _alike(q, q.dtype, k=k, v=v)
    if q.numel() == 0:
        return q * (1 + 0 * (k.sum() + v.sum()))  # (of every input, which all have a gradient)
    return _WindowAttentionFn.apply(*(_strided_heads(t) for t in (q, k, v)), None if valid is None else as_u8(valid),
                                    int(window), int(sinks), bool(causal), scale)


def window_attention_qkv(qkv: torch.Tensor, heads: int, window: int, sinks: int = 0, causal: bool = True,
                         valid: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """window_attention on a fused projection qkv (B, L, (heads + 2 kv_heads) * head_dim) with heads = kv_heads, the
    layout ops.attention takes; returns (B, L, heads * head_dim)."""
    if qkv.dim() != 3 or heads < 1 or qkv.shape[2] % (3 * heads):
        raise ValueError(f"qkv {tuple(qkv.shape)}: expected (B, L, 3 * {heads} * head_dim)")
    B, L = qkv.shape[:2]
    D = qkv.shape[2] // (3 * heads)
    scale = _check_window(qkv, heads, heads, D, window, sinks, valid, scale)
    if qkv.numel() == 0:
        return qkv[..., :heads * D] * 1
    out = _WindowAttentionQKVFn.apply(_strided_heads(qkv.view(B, L, 3 * heads, D) if qkv.is_contiguous() else
                                                     qkv.contiguous().view(B, L, 3 * heads, D)),
                                      None if valid is None else as_u8(valid), heads, int(window), int(sinks),
                                      bool(causal), scale)
    return out.view(B, L, heads * D)


def window_cache_fill(cache_k: torch.Tensor, cache_v: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      lengths: torch.Tensor, sinks: int = 0):
    """Lay prompts into ring caches (asme_window_cache_fill), in place: k, v (B, L, kv_heads, head_dim), of which
    sequence b has lengths[b] tokens from position 0; cache_k, cache_v (B, kv_heads, sinks + window, head_dim).  Slots
    that no position of a prompt falls on stay as they are (window_attention_step does not read them)."""
    _check_cache(cache_k, cache_v, sinks)
    B, KV, slots, D = cache_k.shape
    if k.dim() != 4 or k.shape != v.shape or k.shape[0] != B or k.shape[2:] != (KV, D):
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)}: expected (batch {B}, length, {KV}, {D})")
    _alike(cache_k, cache_k.dtype, k=k, v=v)
    _alike(cache_k, lengths=lengths)
    if lengths.shape != (B,):
        raise ValueError(f"lengths {tuple(lengths.shape)}: expected ({B},)")
    if torch.is_grad_enabled() and (cache_k.requires_grad or cache_v.requires_grad):
        raise RuntimeError("window_cache_fill has no gradient: the caches require none")
    if B == 0 or k.shape[1] == 0:
        return
    k, v = _strided_heads(k.detach()), _strided_heads(v.detach())
    _call_on(k, "asme_window_cache_fill", ptr(k), ptr(v), *k.stride()[:3], *v.stride()[:3], ptr(_i64(lengths)), B,
             k.shape[1], KV, D, slots, sinks, _dtype_code(cache_k), ptr(cache_k), ptr(cache_v))
    torch.autograd.graph.increment_version((cache_k, cache_v))


def window_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache_k: torch.Tensor,
                          cache_v: torch.Tensor, lengths: torch.Tensor, sinks: int = 0,
                          scale: Optional[float] = None) -> torch.Tensor:
    """One new token per sequence against its ring cache (asme_window_step): stores k, v (B, kv_heads, head_dim) as
    position lengths[b] -- the tokens before this one; negative: the sequence takes no step -- and returns the attention
    (B, heads, head_dim) of q to what the cache then holds, the row that window_attention gives that position.  The
    caches (B, kv_heads, sinks + window, head_dim) change in place; `lengths` does not (the layers of a model share it:
    add 1 once per token).  No gradients."""
    _check_cache(cache_k, cache_v, sinks)
    B, KV, slots, D = cache_k.shape
    if q.dim() != 3 or q.shape[0] != B or q.shape[2] != D or q.shape[1] == 0 or q.shape[1] % KV:
        raise ValueError(f"q {tuple(q.shape)}: expected ({B}, a multiple of {KV}, {D})")
    if k.shape != (B, KV, D) or v.shape != (B, KV, D):
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)}: expected ({B}, {KV}, {D})")
    _alike(cache_k, cache_k.dtype, q=q, k=k, v=v)
    _alike(cache_k, lengths=lengths)
    if lengths.shape != (B,):
        raise ValueError(f"lengths {tuple(lengths.shape)}: expected ({B},)")
    scale = _attention_scale(scale, D)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, cache_k, cache_v)):
        raise RuntimeError("window_attention_step has no gradient: call it under torch.no_grad()")
    q, k, v = (_aligned(t) for t in (q, k, v))
    out = torch.empty_like(q)
    if B == 0:
        return out
    ws, nb = _ws_bytes("asme_window_step_workspace", B, q.shape[1], KV, D, slots, device=q.device)
    _call_on(q, "asme_window_step", ptr(q), ptr(k), ptr(v), ptr(cache_k), ptr(cache_v), ptr(_i64(lengths)), B, q.shape[1],
             KV, D, slots, sinks, scale, _dtype_code(q), ptr(ws), nb, ptr(out))
    torch.autograd.graph.increment_version((cache_k, cache_v))
    return out


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t contiguous, from a 16-byte boundary on"""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _strided_heads(t: torch.Tensor) -> torch.Tensor:
    """(B, L, heads, head_dim) with adjacent head values and every row on a 16-byte boundary, copied only if it is not"""
    per = 16 // t.element_size()
    ok = (t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(s % per == 0 and s >= 0 for s in t.stride()[:3])
          and t.stride(1) < 2 ** 23)
    return t if ok else t.clone(memory_format=torch.contiguous_format)  # (whatever strides its axes of size 1 have)


_HEAD_DIMS = (16, 32, 64, 128)


def _check_cache(cache_k, cache_v, sinks: int):
    if cache_k.dim() != 4 or cache_k.shape != cache_v.shape:
        raise ValueError(f"caches {tuple(cache_k.shape)} and {tuple(cache_v.shape)}: expected two of (batch, kv_heads, "
                         "sinks + window, head_dim)")
    if cache_k.shape[3] not in _HEAD_DIMS:
        raise ValueError(f"head_dim {cache_k.shape[3]}: expected one of {_HEAD_DIMS}")
    if cache_k.shape[1] < 1:
        raise ValueError("caches of no heads")
    if not 0 <= sinks < cache_k.shape[2]:
        raise ValueError(f"sinks {sinks}: expected 0 <= sinks < {cache_k.shape[2]} slots")
    _dtype_code(cache_k)
    _alike(cache_k, cache_k.dtype, cache_v=cache_v)
    for c in (cache_k, cache_v):
        if not c.is_contiguous() or c.data_ptr() % 16:
            raise ValueError("the caches are contiguous, from a 16-byte boundary on")
    if cache_k.numel() and cache_k.data_ptr() == cache_v.data_ptr():
        raise ValueError("cache_k and cache_v are the same memory")


# ------------------------------------------------------------------------------------ heads / losses
class _SampledLogitsFn(torch.autograd.Function):
    """SASRecProjectionComponent.forward training branch (sasrec/components.py:34-44)."""

    @staticmethod
    def forward(ctx, hidden, table, pos_ids, neg_ids, table_grad: Optional[TableGrad]):
        shape = pos_ids.shape
        D = table.shape[1]
        h2 = _f32(hidden).reshape(-1, D)
        pos_ids, neg_ids = _i64(pos_ids), _i64(neg_ids)
        T = h2.shape[0]
        # the rows staged by this step's lazy Adam in slot order (SparseTablePlan.gather_source), else the table
        plan = table_grad.plan if table_grad is not None else None
        src, pos_src = plan.gather_source(table, pos_ids) if plan is not None else (table, pos_ids)
        neg_src = plan.gather_source(table, neg_ids)[1] if plan is not None and src is not table else neg_ids
        if src is not table and neg_src is neg_ids:
            src, pos_src, neg_src = table, pos_ids, neg_ids  # both id sets must read the same rows
        V = src.shape[0]
        po = torch.empty(T, device=hidden.device, dtype=torch.float32)
        no = torch.empty(T, device=hidden.device, dtype=torch.float32)
        call("asme_sampled_logits_fwd", ptr(h2), ptr(src), ptr(pos_src), ptr(neg_src), T, D, V, ptr(po), ptr(no),
             stream())
        ctx.save_for_backward(h2, table, src, pos_ids, neg_ids, pos_src, neg_src)
        ctx.table_grad = table_grad
        ctx.hshape = hidden.shape
        return po.view(shape), no.view(shape)

    @staticmethod
    def backward(ctx, g_pos, g_neg):
        h2, table, src, pos_ids, neg_ids, pos_src, neg_src = ctx.saved_tensors
        V, D = table.shape
        T = h2.shape[0]
        gp = torch.zeros(T, device=h2.device) if g_pos is None else _f32(g_pos).reshape(T)
        gn = torch.zeros(T, device=h2.device) if g_neg is None else _f32(g_neg).reshape(T)
        dh = torch.empty_like(h2) if ctx.needs_input_grad[0] else None
        g_table = None
        plan = ctx.table_grad.plan if ctx.table_grad is not None else None
        if ctx.needs_input_grad[1] and plan is not None:
            # dH pass with the rows the forward read; the table contributions go to the compact rows
            call("asme_sampled_logits_bwd", ptr(h2), ptr(src), ptr(pos_src), ptr(neg_src), T, D, src.shape[0],
                 ptr(gp), ptr(gn), ptr(dh), None, stream())
            # table rows: g_pos[t] * h[t] / g_neg[t] * h[t], summed per unique row by the plan (deterministic)
            plan.add_scaled(pos_ids, gp, h2)
            plan.add_scaled(neg_ids, gn, h2)
        else:
            if ctx.needs_input_grad[1]:
                g_table = torch.zeros_like(table)
            call("asme_sampled_logits_bwd", ptr(h2), ptr(table), ptr(pos_ids), ptr(neg_ids), T, D, V, ptr(gp),
                 ptr(gn), ptr(dh), ptr(g_table), stream())
        return (None if dh is None else dh.view(ctx.hshape)), g_table, None, None, None


def sampled_logits(hidden, table, pos_ids, neg_ids, table_grad: Optional[TableGrad] = None):
    return _SampledLogitsFn.apply(hidden, table, pos_ids, neg_ids, table_grad)


class _SASRecBCEFn(torch.autograd.Function):
    """sas_rec_binary_cross_entropy (core/losses/sasrec/sas_rec_losses.py:56-75)."""

    @staticmethod
    def forward(ctx, pos, neg, mask):
        pos_shape, neg_shape = pos.shape, neg.shape
        pos, neg = _f32(pos).reshape(-1), _f32(neg).reshape(-1)
        m = as_u8(mask.reshape(-1))
        T = pos.numel()
        nparts = max(1, min(1024, (T + 255) // 256))
        ws = torch.empty(nparts, 2, device=pos.device, dtype=torch.float32)
        out = torch.empty(2, device=pos.device, dtype=torch.float32)
        call("asme_sasrec_bce_fwd", ptr(pos), ptr(neg), ptr(m), T, ptr(ws), nparts, ptr(out), stream())
        ctx.save_for_backward(pos, neg, m, out)
        ctx.shapes = (pos_shape, neg_shape)
        return out[0]

    @staticmethod
    def backward(ctx, dloss):
        pos, neg, m, out = ctx.saved_tensors
        T = pos.numel()
        dl = _f32(dloss.reshape(1))
        gp, gn = torch.empty_like(pos), torch.empty_like(neg)
        call("asme_sasrec_bce_bwd", ptr(pos), ptr(neg), ptr(m), T, ptr(dl), ptr(out), ptr(gp), ptr(gn), stream())
        return gp.view(ctx.shapes[0]), gn.view(ctx.shapes[1]), None


def sasrec_bce(pos_logits, neg_logits, mask):
    loss = _SASRecBCEFn.apply(pos_logits, neg_logits, mask)
    return loss


class _CrossEntropyFn(torch.autograd.Function):
    """nn.CrossEntropyLoss(ignore_index=pad), mean over non-ignored rows."""

    @staticmethod
    def forward(ctx, logits, targets, ignore_index: int):
        C = logits.shape[-1]
        x = _f32(logits).reshape(-1, C)
        t = _i64(targets).reshape(-1)
        n = x.shape[0]
        if t.numel() != n:
            raise ValueError(f"logits rows ({n}) and targets ({t.numel()}) differ")
        lse = torch.empty(n, device=x.device, dtype=torch.float32)
        rl = torch.empty(n, device=x.device, dtype=torch.float32)
        out = torch.empty(2, device=x.device, dtype=torch.float32)
        call("asme_cross_entropy_fwd", ptr(x), C, ptr(t), ignore_index, n, C, ptr(lse), ptr(rl), ptr(out), stream())
        ctx.save_for_backward(x, t, lse, out)
        ctx.meta = (ignore_index, logits.shape)
        return out[0]

    @staticmethod
    def backward(ctx, dloss):
        x, t, lse, out = ctx.saved_tensors
        ignore_index, shape = ctx.meta
        n, C = x.shape
        dl = _f32(dloss.reshape(1))
        g = torch.empty_like(x)
        call("asme_cross_entropy_bwd", ptr(x), C, ptr(lse), ptr(t), ignore_index, n, C, ptr(dl), ptr(out), ptr(g), C,
             stream())
        return g.view(shape), None, None


def cross_entropy(logits, targets, ignore_index: int):
    return _CrossEntropyFn.apply(logits, targets, ignore_index)


def _capture_id(t: torch.Tensor) -> int:
    """the number of the graph capture that the current stream of t's device is in, 0 outside of one"""
    if not torch.cuda.is_current_stream_capturing():
        return 0
    return _lib.load().asme_stream_capture_id(torch._C._cuda_getCurrentRawStream(t.get_device()))


class _DistillFn(torch.autograd.Function):
    """tau^2 KL(teacher's list || softmax over the catalogue), mean over the rows with a list (csrc/distill.hip)."""

    @staticmethod
    def forward(ctx, logits, ids, teacher, temperature: float, weight: float):
        V, top = logits.shape[-1], ids.shape[-1]
        x = logits if logits.dim() == 2 and logits.stride(1) == 1 and logits.stride(0) >= V else logits.contiguous()
        kept, x = x, x if x.dim() == 2 else x.view(-1, V)
        ids, teacher = _i64(ids), teacher.to(torch.float32).contiguous()
        n, dev = x.shape[0], x.device
        state = torch.empty(n, 2, device=dev, dtype=torch.float32)
        prob = torch.empty(n, top, device=dev, dtype=torch.float32)
        out = torch.empty(2, device=dev, dtype=torch.float32)
        # out[0] as a tensor of its own: autograd lets no one change a view that a Function returns (loss += ...)
        loss = torch.empty(0, device=dev, dtype=torch.float32).set_(out.untyped_storage(), 0, ())
        ctx.meta, ctx.given = (temperature, weight, logits.shape), False
        code, grad = _dtype_code(x), None
        # the gradient with the forward (csrc/distill.hip, "together") where a workgroup holds a row: at 8192 x 26747 fp32
        # 375 us forward and backward in place of 580; 785 where an upstream factor other than 1 is left to apply (bf16 206,
        # and 404 with its gradient formed anew)
        if (ctx.needs_input_grad[0] and x.is_contiguous() and x.data_ptr() % 16 == 0
                and _lib.load().asme_distill_xent_grad_supported(n, V, code)):
            grad = torch.empty(logits.shape, device=dev, dtype=x.dtype)
            ws, nb = _ws_bytes("asme_distill_xent_grad_workspace", n, device=dev)
            _call_on(x, "asme_distill_xent_fwd_grad", ptr(x), V, n, V, ptr(ids), ptr(teacher), top, temperature, weight, code,
                     ptr(state), ptr(prob), ptr(grad), ptr(ws), nb, ptr(out))
            ctx.save_for_backward(kept, ids, state, prob, out, grad)
            ctx.capture = _capture_id(x)
            return loss
        ws, nb = _ws_bytes("asme_distill_xent_workspace", n, V, device=dev)
        _call_on(x, "asme_distill_xent_fwd", ptr(x), x.stride(0), n, V, ptr(ids), ptr(teacher), top, temperature, weight, code,
                 ptr(state), ptr(prob), ptr(ws), nb, ptr(out))
        ctx.save_for_backward(kept, ids, state, prob, out, grad)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        x, ids, state, prob, out, g = ctx.saved_tensors
        temperature, weight, shape = ctx.meta
        V = shape[-1]
        x = x if x.dim() == 2 else x.view(-1, V)
        n = x.shape[0]
        # A backward that is captured apart from its forward may be replayed more often than that, and would find the
        # gradient as its last replay left it: it forms its own.  (.data: the caller may change what it is given, which is
        # no change of a saved tensor)
        g, ctx.given = None if g is None or ctx.given or ctx.capture != _capture_id(x) else g.data, True
        if g is not None and g.dtype == torch.float32:
            _call_on(g, "asme_scale_by", ptr(g), g.numel(), _dtype_code(g), ptr(_f32(dloss)))
            return g, None, None, None, None
        if g is not None:  # (scaled, a bf16 gradient would be rounded twice)
            _call_on(x, "asme_distill_xent_bwd_again", ptr(x), V, n, V, ptr(ids), ids.shape[-1], temperature, weight,
                     _dtype_code(x), ptr(state), ptr(prob), ptr(out), ptr(_f32(dloss)), ptr(g))
            return g, None, None, None, None
        # (also a second backward of one forward: the first one gave its gradient away)
        g = torch.empty(shape, device=x.device, dtype=x.dtype)
        _call_on(x, "asme_distill_xent_bwd", ptr(x), x.stride(0), n, V, ptr(ids), ids.shape[-1], temperature, weight,
                 _dtype_code(x), ptr(state), ptr(prob), ptr(out), ptr(_f32(dloss)), ptr(g), V)
        return g, None, None, None, None


def distill_cross_entropy(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                          temperature: float = 1.0, weight: float = 1.0) -> torch.Tensor:
    """Distillation from a teacher's best items: for logits (..., V) and the teacher's lists teacher_ids,
    teacher_logits (..., k <= 1024; e.g. of catalog_topk), the scalar
        weight * temperature^2 * KL(softmax(teacher_logits / temperature) over the list || softmax(logits / temperature)
        over V),
    mean over the rows whose list is not empty (NaN when all are).  Entries whose id is not in [0, V) (-1 ends a shorter
    list) are absent, and a list of nothing but -inf is empty; an item twice on a list counts twice.  The gradient goes to `logits`; the teacher takes none.
    logits float32 or bfloat16, the loss float32.  A loss that is one part of another is cheapest with its `weight` here:
    the gradient is formed with the forward for that weight, and a factor other than 1 from above is one more pass."""
    V, top = logits.shape[-1], teacher_ids.shape[-1]
    if teacher_ids.shape != teacher_logits.shape or teacher_ids.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"logits {tuple(logits.shape)}, teacher_ids {tuple(teacher_ids.shape)} and teacher_logits "
                         f"{tuple(teacher_logits.shape)}: expected (..., V) and twice (..., k)")
    if not 1 <= top <= 1024 or V < 1:
        raise ValueError(f"{V} items and lists of {top}: expected at least one item and 1 to 1024 entries")
    if teacher_ids.is_floating_point() or teacher_ids.dtype == torch.bool:
        raise TypeError(f"teacher_ids are whole numbers, got {teacher_ids.dtype}")
    if not 0.0 < temperature < math.inf:
        raise ValueError(f"temperature {temperature}: expected a positive number")
    if not math.isfinite(weight):
        raise ValueError(f"weight {weight}: expected a finite number")
    if torch.is_grad_enabled() and teacher_logits.requires_grad:
        raise ValueError("distill_cross_entropy gives the teacher no gradient: detach teacher_logits")
    _dtype_code(logits)
    _alike(logits, teacher_ids=teacher_ids, teacher_logits=teacher_logits)
    if logits.numel() == 0:
        return logits.float().sum() * math.nan  # the mean over no rows
    return _DistillFn.apply(logits, teacher_ids, teacher_logits, float(temperature), float(weight))


def linear_xent_ok(hidden: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> bool:
    """shapes the logits kernels take (asme_linear_xent_*, asme_logits; csrc/logits.hip): hidden width a multiple of
    4 up to 128, weight rows contiguous and 16-B aligned"""
    d = hidden.shape[-1]
    # (the kernels read the weight / bias as fp32 in place: a bf16 / fp16 head, e.g. under autocast, is not taken)
    return (4 <= d <= 128 and d % 4 == 0 and weight.dim() == 2 and weight.shape[1] == d
            and weight.dtype == torch.float32 and (bias is None or bias.dtype == torch.float32)
            and weight.stride(1) == 1 and weight.stride(0) % 4 == 0 and weight.data_ptr() % 16 == 0)


class _LogitsFn(torch.autograd.Function):
    """H W^T + b materialised on asme_logits (evaluation / predict scores).  Its backward (only for callers that
    differentiate through materialised logits with a loss other than the fused cross-entropy) uses library
    GEMMs: dH = dS W, dW = dS^T H."""

    @staticmethod
    def forward(ctx, hidden, weight, bias):
        h = _f32(hidden).reshape(-1, hidden.shape[-1])
        n, d = h.shape
        V = weight.shape[0]
        out = torch.empty(n, V, device=h.device, dtype=torch.float32)
        nb = int(_lib.load().asme_logits_workspace(n, V, d))
        ws = torch.empty(max(4, nb // 4 + 1), device=h.device, dtype=torch.float32)
        call("asme_logits", ptr(h), d, n, d, ptr(weight), weight.stride(0), V, ptr(_f32(bias)) if bias is not None
             else None, ptr(out), V, ptr(ws), ws.numel() * 4, stream())
        ctx.save_for_backward(h, weight)
        ctx.meta = (bias is not None, hidden.shape)
        return out.view(*hidden.shape[:-1], V)

    @staticmethod
    def backward(ctx, ds):
        h, weight = ctx.saved_tensors
        has_bias, shape = ctx.meta
        ds2 = ds.reshape(-1, weight.shape[0])
        dh = (ds2 @ weight).view(shape) if ctx.needs_input_grad[0] else None
        dw = ds2.t() @ h if ctx.needs_input_grad[1] else None
        db = ds2.sum(0) if has_bias and ctx.needs_input_grad[2] else None
        return dh, dw, db


def logits(hidden, weight, bias=None):
    """full-catalogue scores hidden . weight^T (+ bias) on the bf16x6 logits kernel; widths above 128 (NARM's
    2H = 256) on the fp32-MFMA Linear kernel"""
    if linear_xent_ok(hidden, weight, bias) and hidden.is_cuda:
        return _LogitsFn.apply(hidden, weight, bias)
    return linear(hidden, weight, bias)


# the fused CE head's training form (dH accumulated in the forward pass, asme_linear_xent_fwd_dh / _bwd_dw); False
# runs the two-pass backward (asme_linear_xent_bwd), kept for same-process A/B timing (tools/xent_bench.py) and tests
XENT_TRAINING_FORM = True


class _LinearXentFn(torch.autograd.Function):
    """CrossEntropyLoss(ignore_index)(H W^T + b, targets), mean over non-ignored rows, without the (n, |V|)
    logits (csrc/logits.hip; layers.py:105-109,138-143 + losses.py:77-115)."""

    @staticmethod
    def forward(ctx, hidden, weight, bias, targets, ignore_index: int):
        h = _f32(hidden).reshape(-1, hidden.shape[-1])
        t = _i64(targets).reshape(-1)
        n, d = h.shape
        V = weight.shape[0]
        if t.numel() != n:
            raise ValueError(f"hidden rows ({n}) and targets ({t.numel()}) differ")
        lib = _lib.load()
        lse = torch.empty(n, device=h.device, dtype=torch.float32)
        out = torch.empty(2, device=h.device, dtype=torch.float32)
        dh_raw = None
        if ctx.needs_input_grad[0] and XENT_TRAINING_FORM:
            # training: dH (before the upstream scale) is accumulated in the same pass as the softmax statistics
            # (asme_linear_xent_fwd_dh), so the backward recomputes the logits once, for dW only
            ws = torch.empty(max(4, int(lib.asme_linear_xent_fwd_dh_workspace(n, V, d)) // 4 + 1), device=h.device,
                             dtype=torch.float32)
            dh_raw = torch.empty(n, d, device=h.device, dtype=torch.float32)
            call("asme_linear_xent_fwd_dh", ptr(h), d, n, d, ptr(weight), weight.stride(0), V, ptr(bias), ptr(t),
                 ignore_index, ptr(lse), ptr(dh_raw), d, ptr(ws), ws.numel() * 4, ptr(out), stream())
        else:
            ws = torch.empty(max(4, int(lib.asme_linear_xent_fwd_workspace(n, V, d)) // 4 + 1), device=h.device,
                             dtype=torch.float32)
            call("asme_linear_xent_fwd", ptr(h), d, n, d, ptr(weight), weight.stride(0), V, ptr(bias), ptr(t),
                 ignore_index, ptr(lse), ptr(ws), ws.numel() * 4, ptr(out), stream())
        ctx.save_for_backward(h, weight, bias, t, lse, out, dh_raw)
        ctx.meta = (ignore_index, hidden.shape)
        return out[0]

    @staticmethod
    def backward(ctx, dloss):
        h, weight, bias, t, lse, out, dh_raw = ctx.saved_tensors
        ignore_index, shape = ctx.meta
        n, d = h.shape
        V = weight.shape[0]
        lib = _lib.load()
        dh = torch.empty_like(h)
        dw = torch.empty(V, d, device=h.device, dtype=torch.float32)
        db = torch.empty(V, device=h.device, dtype=torch.float32) if bias is not None else None
        dl = _f32(dloss.reshape(1))
        if dh_raw is not None:
            ws = torch.empty(max(4, int(lib.asme_linear_xent_bwd_dw_workspace(n, V, d)) // 4 + 1), device=h.device,
                             dtype=torch.float32)
            call("asme_linear_xent_bwd_dw", ptr(h), d, n, d, ptr(weight), weight.stride(0), V, ptr(bias), ptr(t),
                 ignore_index, ptr(lse), ptr(out), ptr(dl), ptr(dh_raw), ptr(dh), ptr(dw), ptr(db), ptr(ws),
                 ws.numel() * 4, stream())
        else:
            ws = torch.empty(max(4, int(lib.asme_linear_xent_bwd_workspace(n, V, d)) // 4 + 1), device=h.device,
                             dtype=torch.float32)
            call("asme_linear_xent_bwd", ptr(h), d, n, d, ptr(weight), weight.stride(0), V, ptr(bias), ptr(t),
                 ignore_index, ptr(lse), ptr(out), ptr(dl), ptr(dh), ptr(dw), ptr(db), ptr(ws), ws.numel() * 4,
                 stream())
        return dh.view(shape), dw, db, None, None


def linear_cross_entropy(hidden, weight, bias, targets, ignore_index: int):
    """loss of CrossEntropyLoss(ignore_index)(F.linear(hidden, weight, bias), targets) on the fused kernels"""
    return _LinearXentFn.apply(hidden, weight, bias, targets, ignore_index)


def target_rank(scores: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """1-based rank of each target in its row (descending; ties -> lower id first)."""
    s = _f32(scores)
    t = _i64(targets)
    n, V = s.shape
    ranks = torch.empty(n, device=s.device, dtype=torch.int64)
    call("asme_target_rank", ptr(s), V, ptr(t), n, V, ptr(ranks), stream())
    return ranks


# ------------------------------------------------------------------------------------ full-catalogue eval
def catalog_planes(table: torch.Tensor) -> torch.Tensor:
    """the exact three-way bf16 split of a (V, d <= 128) catalogue (asme_catalog_split): the streamed operand of the
    ranking pass; split once and pass to catalog_rank / catalog_count_above to rank many query batches against it"""
    E = _f32(table)
    V, d = E.shape
    planes = torch.empty(int(_lib.load().asme_catalog_planes_bytes(V)), device=E.device, dtype=torch.uint8)
    call("asme_catalog_split", ptr(E), E.stride(0), V, d, ptr(planes), stream())
    return planes


# parameter updates the C-ABI optimizer kernels make through raw pointers (FusedAdam.step) do not move torch's
# version counter: every step bumps this instead, so a cached derivative of a parameter knows it is stale
_PARAM_WRITES = [0]


def note_param_write():
    _PARAM_WRITES[0] += 1


class CatalogPlanes:
    """catalog_planes(table) kept while the table is unchanged: a validation pass scores every batch against the same
    frozen catalogue, so the split (2.3 ms and 7.7 GB of planes at |V| = 10M) is made once per pass instead of once
    per batch.  The key is the table's storage, shape and torch version counter plus the count of optimizer steps
    taken through FusedAdam (whose kernels write parameters without touching the version counter); a table that
    _f32 had to copy (not contiguous) is never cached (its copy is new on every call)."""

    def __init__(self):
        self._key = None
        self._planes: Optional[torch.Tensor] = None
        self._table: Optional[torch.Tensor] = None  # held: its storage cannot be freed and reused under the same key

    def get(self, table: torch.Tensor) -> torch.Tensor:
        E = _f32(table)
        if E is not table and E.data_ptr() != table.data_ptr():
            return catalog_planes(E)
        key = (E.data_ptr(), tuple(E.shape), E.stride(0), E._version, _PARAM_WRITES[0])
        if key != self._key:
            self.clear()  # (the old planes are freed before the new ones are allocated)
            self._planes = catalog_planes(E)
            self._key, self._table = key, E.detach()
        return self._planes

    def clear(self):
        self._planes = self._key = self._table = None


def _catalog_ws(n: int, d: int, dev) -> Tuple[torch.Tensor, int]:
    nbytes = int(_lib.load().asme_catalog_x6_workspace(n, d))
    return torch.empty(nbytes, device=dev, dtype=torch.uint8), nbytes


def catalog_rank(hidden: torch.Tensor, table: torch.Tensor, targets: torch.Tensor,
                 bias: Optional[torch.Tensor] = None, planes: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rank (1-based, ties to the lower id) of each row's target among all |V| items scored as
    hidden . table^T (+ bias) -- the (rows, |V|) logits are never materialised (asme_catalog_rank_x6: the bf16x6
    score products asme_logits materialises, so the ranks are those of the materialised scores).  `planes`: a
    catalog_planes(table) split made earlier (else the table is split here).
    Reference: SASRecProjectionComponent inference + AllItemsSampler + argsort (sasrec/components.py:46-61,
    metrics/common.py:4-27)."""
    h = _f32(hidden)
    E = _f32(table)
    n, d = h.shape
    V = E.shape[0]
    tg = _i64(targets).reshape(n)
    counts = torch.empty(n, device=h.device, dtype=torch.int32)
    ranks = torch.empty(n, device=h.device, dtype=torch.int64)
    if planes is None:
        planes = catalog_planes(E)
    ws, nbytes = _catalog_ws(n, d, h.device)
    call("asme_catalog_rank_x6", ptr(h), h.stride(0), n, d, ptr(E), E.stride(0), ptr(planes), V,
         ptr(_f32(bias)) if bias is not None else None, ptr(tg), ptr(counts), ptr(ranks), ptr(ws), nbytes, stream())
    return ranks


def catalog_topk(hidden: torch.Tensor, table: torch.Tensor, k: int, bias: Optional[torch.Tensor] = None,
                 id_stride: int = 1, id_offset: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """The k (<= 16) best (score, item) per row over all |V| items, scores descending, ties to the lower id
    (asme_catalog_topk; no (rows, |V|) logits)."""
    h = _f32(hidden)
    E = _f32(table)
    n, d = h.shape
    V = E.shape[0]
    nbytes = int(_lib.load().asme_catalog_topk_workspace(n, V, d))
    ws = torch.empty(max(16, nbytes), device=h.device, dtype=torch.uint8)
    vals = torch.empty(n, k, device=h.device, dtype=torch.float32)
    idx = torch.empty(n, k, device=h.device, dtype=torch.int64)
    call("asme_catalog_topk", ptr(h), h.stride(0), n, d, ptr(E), E.stride(0), V,
         ptr(_f32(bias)) if bias is not None else None, id_stride, id_offset, k, ptr(ws), nbytes, ptr(vals), ptr(idx),
         stream())
    return vals, idx


def catalog_target_scores(hidden: torch.Tensor, target_rows: torch.Tensor,
                          target_bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """score of each row's target from its gathered table row, by the same products as the shard scan
    (asme_catalog_target_scores_x6: the owner's scan compares bit-identically against it)."""
    h, rows = _f32(hidden), _f32(target_rows)
    n, d = h.shape
    out = torch.empty(n, device=h.device, dtype=torch.float32)
    ws, nbytes = _catalog_ws(n, d, h.device)
    call("asme_catalog_target_scores_x6", ptr(h), h.stride(0), n, d, ptr(rows), rows.stride(0),
         ptr(_f32(target_bias)) if target_bias is not None else None, ptr(out), ptr(ws), nbytes, stream())
    return out


def catalog_count_above(hidden: torch.Tensor, table_shard: torch.Tensor, targets: torch.Tensor,
                        target_scores: torch.Tensor, id_stride: int, id_offset: int,
                        bias_shard: Optional[torch.Tensor] = None, planes: Optional[torch.Tensor] = None) -> torch.Tensor:
    """#items of this table shard (local row j = item j*id_stride + id_offset) ranked above each row's target
    (asme_catalog_count_above_x6; `planes`: catalog_planes(table_shard) made earlier)."""
    h, E = _f32(hidden), _f32(table_shard)
    n, d = h.shape
    counts = torch.empty(n, device=h.device, dtype=torch.int32)
    if planes is None:
        planes = catalog_planes(E)
    ws, nbytes = _catalog_ws(n, d, h.device)
    call("asme_catalog_count_above_x6", ptr(h), h.stride(0), n, d, ptr(planes), E.shape[0],
         ptr(_f32(bias_shard)) if bias_shard is not None else None, ptr(_i64(targets).reshape(n)),
         ptr(_f32(target_scores)), id_stride, id_offset, ptr(counts), ptr(ws), nbytes, stream())
    return counts

"""Low-rank adapters of many requests at once, on top of a shared projection's output:

    out[m] = base[m] + scale[i] * B[i] (A[i] x[m]),   i = ids[m];   out[m] = base[m] where ids[m] names no adapter

``Adapters`` holds a projection's adapters in slots; a slot is filled, replaced or emptied in place while others serve.
``Plan`` and ``route`` group a batch's rows by adapter once a step, for every projection of the step.  ``add`` is one
launch (``csrc/adapters.cu``); ``qmm.matmul``, ``qmm.prefill_matmul`` and ``Exl3Linear`` call it behind their product when
they are given ``adapters=`` and ``plan=``.  Sums are fp32, the low-rank row is kept to 16 bits or more (22 under fp32 rows), and a row's bits
depend neither on the other rows nor on their number.  No CPU path.
"""

from __future__ import annotations

import torch

from . import _lib
from . import experts as grouped

DTYPES = (torch.bfloat16, torch.float16)
ROW_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_RANK = 128
MAX_COUNT = 1024
ITEM = 64              # rows an item of a plan holds
# Up to this many rows each is an item of its own and nothing is sorted.  Measured on projections of 4096 x 4096, 64
# adapters of rank 16: 65 rows 7.7 us and 13.2 sorted, 128 rows 14.4 and 14.9, 256 rows 26.8 and 17.8; rank 64: 16.4 and
# 22.8 at 65 rows, 25.3 and 18.2 at 128.
DIRECT_ROWS = 96


class Adapters:
    """``count`` slots for adapters of rank ``rank`` or less on a projection of ``k`` inputs and ``n`` columns.  Empty slots
    add nothing."""

    def __init__(self, count: int, rank: int, k: int, n: int, dtype: torch.dtype = torch.bfloat16,
                 device: str | torch.device = "cuda") -> None:
        if dtype not in DTYPES:
            raise ValueError(f"adapters are bf16 or fp16, not {dtype}")
        if not 1 <= count <= MAX_COUNT or not 1 <= rank <= MAX_RANK:
            raise ValueError(f"1..{MAX_COUNT} adapters of rank 1..{MAX_RANK}, not {count} of {rank}")
        if k < 8 or k % 8 or n < 1:
            raise ValueError(f"a projection of {n} columns and {k} inputs (inputs in multiples of 8)")
        self.count, self.rank, self.k, self.n = count, rank, k, n
        padded = -(-rank // 8) * 8
        self.a = torch.zeros((count, padded, k), dtype=dtype, device=device)
        self.b = torch.zeros((count, n, padded), dtype=dtype, device=device)
        self.scale = torch.zeros((count,), dtype=torch.float32, device=device)

    @property
    def dtype(self) -> torch.dtype:
        return self.a.dtype

    @property
    def device(self) -> torch.device:
        return self.a.device

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.a, self.b, self.scale))

    def _slot(self, i: int) -> int:
        if not 0 <= i < self.count:
            raise ValueError(f"slot {i} of {self.count}")
        return i

    def put(self, i: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """Fill slot ``i``: a [r, k], b [n, r] with any r up to ``rank``; on the current stream, before any later ``add``."""

        i = self._slot(i)
        r = a.shape[0] if a.dim() == 2 else -1
        if a.dim() != 2 or b.dim() != 2 or not 1 <= r <= self.rank or a.shape[1] != self.k or tuple(b.shape) != (self.n, r):
            raise ValueError(f"a [r, {self.k}] and b [{self.n}, r] with r <= {self.rank}, not {tuple(a.shape)} and "
                             f"{tuple(b.shape)}")
        scale = float(scale)                                             # what is refused leaves the slot as it was
        self.a[i, :r].copy_(a)
        self.a[i, r:].zero_()
        self.b[i, :, :r].copy_(b)
        self.b[i, :, r:].zero_()
        self.scale[i:i + 1].fill_(scale)

    def clear(self, i: int) -> None:
        """Empty slot ``i``: its rows then come out as the base alone, whatever their inputs hold."""

        i = self._slot(i)
        self.a[i].zero_()
        self.b[i].zero_()
        self.scale[i:i + 1].zero_()


def make(a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor | float = 1.0) -> Adapters:
    """``Adapters`` from stacked matrices: a [count, r, k], b [count, n, r], scale [count] or one number."""

    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or a.dtype != b.dtype:
        raise ValueError(f"a [count, r, k] and b [count, n, r] of one type, not {tuple(a.shape)} and {tuple(b.shape)}")
    count, rank, k = a.shape
    if isinstance(scale, torch.Tensor) and scale.numel() != count:
        raise ValueError(f"one scale an adapter, not {tuple(scale.shape)}")
    ad = Adapters(count, rank, k, b.shape[1], a.dtype, a.device)
    ad.a[:, :rank].copy_(a)
    ad.b[:, :, :rank].copy_(b)
    if isinstance(scale, torch.Tensor):
        ad.scale.copy_(scale.reshape(count))
    else:
        ad.scale.fill_(float(scale))
    return ad


class Plan:
    """Scratch grouping up to ``rows`` rows by adapter, for projections with ``count`` slots."""

    def __init__(self, rows: int, count: int, device: str | torch.device) -> None:
        if rows < 1 or not 1 <= count <= MAX_COUNT:
            raise ValueError(f"a plan of at least one row and 1..{MAX_COUNT} adapters, not {rows} and {count}")
        self.rows, self.count = rows, count
        self.ids: torch.Tensor | None = None
        self.members = torch.zeros((rows,), dtype=torch.int32, device=device)
        self.items = torch.zeros((grouped.max_items(rows, count, ITEM), 3), dtype=torch.int32, device=device)
        self.counts = torch.zeros((2,), dtype=torch.int32, device=device)


def route(ids: torch.Tensor, plan: Plan) -> None:
    """``ids`` [M] int32, contiguous: each row's slot, or anything outside 0..count-1 for none.  The plan keeps the tensor and
    ``add`` reads it: route again after changing it."""

    if ids.dtype != torch.int32 or ids.dim() != 1 or not ids.is_contiguous():
        raise ValueError("ids must be contiguous int32 [rows]")
    if ids.shape[0] > plan.rows:
        raise ValueError(f"{ids.shape[0]} rows do not fit a plan of {plan.rows}")
    grouped._need_cuda(ids, "ids")
    if ids.device != plan.members.device:
        raise ValueError("ids must be on the plan's device")
    plan.ids = ids
    if ids.shape[0] > DIRECT_ROWS:
        with _lib.on(ids.device):
            _lib.call("tfb_plan", ids.data_ptr(), ids.shape[0], plan.count, ITEM, plan.members.data_ptr(),
                      plan.items.data_ptr(), plan.counts.data_ptr(), _lib.stream(ids.device))


def _end(t: torch.Tensor, m: int) -> int:
    """The address behind the last of ``m`` rows."""

    return t.data_ptr() + ((m - 1) * t.stride(0) + t.shape[1]) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor, m: int) -> bool:
    """Whether the first ``m`` rows of one may touch the other's; columns of their own of one buffer's rows do not."""

    if a.data_ptr() >= _end(b, m) or b.data_ptr() >= _end(a, m):
        return False
    step = a.stride(0) * a.element_size()
    if m == 1 or step != b.stride(0) * b.element_size() or step <= 0:
        return True
    at = (b.data_ptr() - a.data_ptr()) % step                                # b's columns within a's rows
    return at < a.shape[1] * a.element_size() or at + b.shape[1] * b.element_size() > step


def _rows_of(t: torch.Tensor, name: str, m: int, n: int, device: torch.device) -> tuple[int, int]:
    """The row type and the step between rows of [m, n] ``t``."""

    kind = ROW_TYPES.get(t.dtype)
    if kind is None or t.shape != (m, n):
        raise ValueError(f"{name}: [{m}, {n}] fp32, bf16 or fp16, not {t.dtype} {tuple(t.shape)}")
    row, one = t.stride()
    if one != 1 and n > 1:
        raise ValueError(f"{name}: [{m}, {n}] with unit-stride rows")
    if m > 1 and row < n:
        raise ValueError(f"{name}: rows must not overlap")
    if t.device != device:
        raise ValueError(f"{name} must be on x's device")
    return kind, row if m > 1 else n


def check(x: torch.Tensor, ad: Adapters, plan: Plan) -> None:
    """Refuses what ``add`` cannot take, before a projection in front of it is launched."""

    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor (this library has no CPU path)")
    ids, a = plan.ids, ad.a
    if x.dim() != 2 or x.dtype != a.dtype or x.shape[1] != ad.k or x.stride(1) != 1:
        raise ValueError(f"x: [M, {ad.k}] {ad.dtype} with unit-stride rows, as the adapters")
    if ids is None or ids.shape[0] != x.shape[0]:
        raise ValueError("route(ids, plan) comes first, with one id a row")
    if a.device != x.device or ids.device != x.device:
        raise ValueError("x, the adapters and the plan must be on one device")
    if plan.count != ad.count:
        raise ValueError(f"a plan of {plan.count} adapters for {ad.count}")


def add(x: torch.Tensor, ad: Adapters, plan: Plan, base: torch.Tensor, out: torch.Tensor | None = None, *,
        dtype: torch.dtype | None = None) -> torch.Tensor:
    """``base`` [M, n] (fp32, bf16 or fp16) plus each row's adapter on ``x`` [M, k], rounded once to ``out``'s type
    (``dtype``, or ``base``'s, where ``out`` is not given).  ``out`` may be ``base`` itself."""

    check(x, ad, plan)
    return add_checked(x, ad, plan, base, out, dtype)


def add_checked(x: torch.Tensor, ad: Adapters, plan: Plan, base: torch.Tensor, out: torch.Tensor | None,
                dtype: torch.dtype | None) -> torch.Tensor:
    """``add`` behind ``check``."""

    m, n, k, device = x.shape[0], ad.n, ad.k, x.device
    base_type, base_step = _rows_of(base, "base", m, n, device)
    if out is None:
        out = torch.empty_strided((m, n), (n, 1), dtype=dtype or base.dtype, device=device)   # a microsecond less than empty
        out_type, out_step = ROW_TYPES.get(out.dtype), n
        if out_type is None:
            raise ValueError(f"out: fp32, bf16 or fp16, not {out.dtype}")
    else:
        if dtype is not None and out.dtype != dtype:
            raise ValueError(f"out is {out.dtype}, not {dtype}")
        out_type, out_step = _rows_of(out, "out", m, n, device)
        same = out.data_ptr() == base.data_ptr() and out_type == base_type and out_step == base_step
        if m and (_overlap(out, x, m) or not same and _overlap(out, base, m)):
            raise ValueError("out may be base itself, but must not overlap x or a part of base (columns apart in one buffer's rows do not)")
    if m == 0:
        return out
    x_step = x.stride(0) if m > 1 else k
    if x_step % 8 or x_step < k or x.data_ptr() % 16:
        x, x_step = x.clone(memory_format=torch.contiguous_format), k        # rows are read in 16-byte pieces
    a, items, counts, members, most = ad.a, 0, 0, 0, 0
    if m > DIRECT_ROWS:
        items, counts, members = plan.items.data_ptr(), plan.counts.data_ptr(), plan.members.data_ptr()
        most = grouped.max_items(m, ad.count, ITEM)
    with _lib.on(device):
        _lib.call("tfb_adapters", a.dtype == torch.float16, x.data_ptr(), x_step, a.data_ptr(), ad.b.data_ptr(),
                  ad.scale.data_ptr(), a.shape[1], k, n, plan.ids.data_ptr(), m, ad.count, items, counts, members, most,
                  base.data_ptr(), base_type, base_step, out.data_ptr(), out_type, out_step, _lib.stream(device))
    return out

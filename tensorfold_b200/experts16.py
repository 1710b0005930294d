"""Grouped MoE experts on 16-bit weights (bf16 or fp16), for layers whose experts are not quantised.

The operators have the names, the plans and the argument order of ``experts`` (affine 4-bit): ``make``, ``unpack``,
``Plan``, ``gate_up``, ``down``; ``experts.route`` sorts the pairs.  ``moe.Routed`` takes either kind of experts.
One kernel serves every batch size (``csrc/experts16.cu``), and a (row, slot) pair's bits depend on nothing but its own
row.  The sums are fp32 and rounded once: gate and up are not rounded before the activation, unlike the 4-bit experts',
which follow their reference's bf16 steps.  No CPU path.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from . import experts as grouped

DTYPES = (torch.bfloat16, torch.float16)
ITEM = 256               # pairs an item holds at most: the tensor-core tile's N
# Up to so many pairs an expert on average: items of so many.  A smaller tile leaves more of the ring to the weights, a larger
# one reads them once for more pairs.  128 experts of 2048 x 768, top 8, gate/up + down in us with items of 32 / 128 / 256: 200
# rows 195 / 194 / 198, 400 rows 202 / 196 / 201, 800 rows 229 / 205 / 207; 1400 rows - / 214 / 218, 1999 rows - / 245 / 235.
SMALL_ITEMS = ((16, 32), (96, 128))


def _rows(mats: int, n: int) -> int:
    return mats * (-(-n // 16) * 16)


def _check_weight(w: torch.Tensor, name: str, like: torch.Tensor | None = None) -> None:
    if w.dim() != 3 or w.dtype not in DTYPES:
        raise ValueError(f"{name}: bf16 or fp16 [experts, columns, inputs], not {w.dtype} {tuple(w.shape)}")
    if min(w.shape) < 1 or w.shape[2] % 8:
        raise ValueError(f"{name}: inputs in multiples of 8, not {tuple(w.shape)}")
    if like is not None and (w.dtype != like.dtype or w.device != like.device):
        raise ValueError(f"{name}: every projection must share one dtype and device")


def pack(*mats: torch.Tensor) -> torch.Tensor:
    """One matrix [E, N, K], or gate and up: the kernel's layout [E, rows, K up to 64], its inner order the library's own."""

    if len(mats) not in (1, 2):
        raise ValueError("pack takes one matrix, or a gate and an up projection")
    for m in mats:
        _check_weight(m, "weights", mats[0])
        if m.shape != mats[0].shape:
            raise ValueError(f"gate and up differ: {tuple(mats[0].shape)} and {tuple(m.shape)}")
    grouped._need_cuda(mats[0], "weights")
    e, n, k = mats[0].shape
    mats = [m.contiguous() for m in mats]
    mats = [m if m.data_ptr() % 16 == 0 else m.clone() for m in mats]       # read in 16-byte pieces
    out = torch.empty((e, _rows(len(mats), n), -(-k // 64) * 64), dtype=mats[0].dtype, device=mats[0].device)
    with _lib.on(out.device):
        _lib.call("tfb_pack16", mats[0].data_ptr(), mats[1].data_ptr() if len(mats) == 2 else 0, out.data_ptr(), e, n, k,
                  _lib.stream(out.device))
    return out


def _unpack(packed: torch.Tensor, mats: int, n: int, k: int) -> list[torch.Tensor]:
    packed = packed.contiguous()
    out = [torch.empty((packed.shape[0], n, k), dtype=packed.dtype, device=packed.device) for _ in range(mats)]
    with _lib.on(packed.device):
        _lib.call("tfb_unpack16", packed.data_ptr(), out[0].data_ptr(), out[1].data_ptr() if mats == 2 else 0,
                  packed.shape[0], n, k, _lib.stream(packed.device))
    return out


@dataclass
class Experts16:
    """One layer's experts (the shared ones included) in bf16 or fp16: gate and up (SwiGLU) or up (relu^2), and down."""

    up: torch.Tensor          # [E, M * (NI up to 16), D up to 64] packed, M = 2 (gate and up) or 1
    down: torch.Tensor        # [E, D up to 16, NI up to 64] packed
    width: int                # NI: the expert's (or this rank's) intermediate width
    dims: int                 # D
    swiglu: bool
    limit: float = 0.0        # SwiGLU clip (0: none)

    @property
    def count(self) -> int:
        return self.up.shape[0]

    @property
    def dtype(self) -> torch.dtype:
        return self.up.dtype

    def bytes_per_expert(self) -> int:
        return (self.up[0].numel() + self.down[0].numel()) * 2


def make(up: list[torch.Tensor], down: torch.Tensor, *, limit: float = 0.0) -> Experts16:
    """``up`` [gate, up] (SwiGLU) or [up] (relu^2), each [E, NI, D]; ``down`` [E, D, NI]; NI and D multiples of 8."""

    if len(up) not in (1, 2):
        raise ValueError("experts take a gate and an up projection, or an up projection alone")
    for m in (*up, down):
        _check_weight(m, "experts", up[0])
    e, width, dims = up[0].shape
    if down.shape != (e, dims, width):
        raise ValueError(f"down must be [{e}, {dims}, {width}], not {tuple(down.shape)}")
    return Experts16(pack(*up), pack(down), width, dims, len(up) == 2, float(limit))


def _check_packed(w: torch.Tensor, name: str, experts: int, rows: int, k: int, like: torch.Tensor) -> None:
    """The kernel reads a packed tensor by its address alone: expert e's rows at e * rows * k."""

    want = (experts, rows, -(-k // 64) * 64)
    if tuple(w.shape) != want or w.dtype not in DTYPES or not w.is_contiguous() or w.data_ptr() % 16:
        raise ValueError(f"{name}: packed weights {list(want)} in bf16 or fp16, contiguous and 16-byte aligned, not {w.dtype} "
                         f"{tuple(w.shape)} with strides {w.stride()}")
    if w.dtype != like.dtype or w.device != like.device:
        raise ValueError(f"{name}: every projection must share one dtype and device")


def check_up(ex: Experts16) -> None:
    _check_packed(ex.up, "up", ex.count, _rows(2 if ex.swiglu else 1, ex.width), ex.dims, ex.up)


def check_down(ex: Experts16) -> None:
    """``down`` holds as many experts as ``up``, in its type and on its device."""

    _check_packed(ex.down, "down", ex.count, _rows(1, ex.dims), ex.width, ex.up)


def unpack(ex: Experts16) -> tuple[list[torch.Tensor], torch.Tensor]:
    """``make``'s inverse, bit for bit: ([gate, up] or [up], down)."""

    check_up(ex)
    check_down(ex)
    return (_unpack(ex.up, 2 if ex.swiglu else 1, ex.width, ex.dims), _unpack(ex.down, 1, ex.dims, ex.width)[0])


def item_pairs(pairs: int, experts: int) -> int:
    """Pairs an item of a plan holds; a pair's bits do not depend on it."""

    for most, item in SMALL_ITEMS:
        if pairs <= most * experts:
            return item
    return ITEM


class Plan(grouped.Plan):
    """``experts.Plan`` with the items of this kernel, for ``experts.route`` and ``moe.select``."""

    def __init__(self, rows: int, slots: int, experts: int, device: torch.device | str) -> None:
        super().__init__(rows, slots, experts, device)
        self.decode_tile = self.tile = item_pairs(rows * slots, experts)


def _run(epi: int, x: torch.Tensor, slots: int, w: torch.Tensor, k: int, n: int, plan: grouped.Plan, out: torch.Tensor,
         limit: float, rows: int) -> None:
    grouped._need_cuda(x, "x")
    pairs, device, dtype = rows * plan.slots, x.device, w.dtype
    need = rows if slots else pairs
    shape = x.shape
    if x.dtype != dtype or len(shape) != 2 or shape[1] != k or shape[0] < need:
        raise ValueError(f"x: at least {need} rows of {k} inputs in the experts' type, not {x.dtype} {tuple(shape)}")
    step, one = x.stride()
    if one != 1 or (step % 8 or step < k) and shape[0] > 1 or x.data_ptr() % 16:
        raise ValueError(f"x: at least {need} rows of {k} inputs, unit-stride and 16-byte aligned")
    want = torch.float32 if epi == 0 else dtype
    if out.dtype != want or not out.is_contiguous() or out.dim() < 1 or out.shape[-1] != n or out.numel() < pairs * n:
        raise ValueError(f"out: contiguous {want} rows of {n} columns, one a pair")
    if out.device != device or w.device != device or plan.members.device != device:
        raise ValueError("x, the experts, the plan and out must be on one device")
    if plan.hot or plan.prefill or not grouped.TILE <= plan.tile <= ITEM:
        raise ValueError(f"a plan with items of {grouped.TILE} to {ITEM} pairs (experts16.Plan)")
    if rows < 0 or rows > plan.rows:
        raise ValueError(f"{rows} rows do not fit a plan of {plan.rows}")
    with _lib.on(device):
        _lib.call("tfb_experts16", epi, dtype == torch.float16, x.data_ptr(), step if shape[0] > 1 else k, need, slots,
                  w.data_ptr(), w.shape[0], k, n, plan.items.data_ptr(), plan.counts.data_ptr(), plan.members.data_ptr(),
                  out.data_ptr(), limit, grouped.max_items(pairs, plan.experts, plan.tile), plan.tile, _lib.stream(device))


def _fits(ex: Experts16, plan: grouped.Plan) -> None:
    if plan.experts != ex.count:
        raise ValueError(f"a plan of {plan.experts} experts for {ex.count}")


def gate_up(x: torch.Tensor, ex: Experts16, plan: grouped.Plan, out: torch.Tensor, rows: int) -> None:
    """x [R, D] (the experts' type, unit-stride rows) -> out [R * slots, NI], each pair's activation in the same type."""

    _fits(ex, plan)
    check_up(ex)
    _run(2 if ex.swiglu else 1, x, plan.slots, ex.up, ex.dims, ex.width, plan, out, ex.limit, rows)


def down(act: torch.Tensor, ex: Experts16, plan: grouped.Plan, out: torch.Tensor, rows: int) -> None:
    """act [R * slots, NI] -> out [R * slots, D] per pair: fp32, or the experts' type when ``out`` has it."""

    _fits(ex, plan)
    check_down(ex)
    _run(0 if out.dtype == torch.float32 else 3, act, 0, ex.down, ex.width, ex.dims, plan, out, 0.0, rows)

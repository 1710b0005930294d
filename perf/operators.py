"""The operators on 16-bit weights whose speed is followed: what a serving program asks of them at decode and at prompt
sizes, through the entry points it would use, and their plain forms in elementary torch operations.

``experts``   one routed block on bf16 experts with the caller's routing: pairs sorted by expert, gate and up projections
              with their activation, down projection, weighted sum over a token's slots (``moe.picked``)
``gate_up``   its first half alone: the activations of every (token, slot) pair (``experts16.gate_up``)
``down``      its second half alone: every pair's row of the down projection (``experts16.down``)
``adapters``  low-rank adapters of many requests on top of a shared projection's output:
              out[m] = base[m] + scale[i] B[i] (A[i] x[m]) with i = ids[m], nothing added where ids[m] < 0 (``adapters.add``)
``affine``    a dense 4-bit projection together with its requests' adapters (``qmm.matmul``, ``qmm.prefill_matmul``)

``own`` false: the plain forms, in 32 bits, rounded once.  ``own`` true: the framework's entry points.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _experts(kind: str, rows: int, dims: int, count: int, width: int, top_k: int, dtype: str = "bf16", act: str = "swiglu",
             limit: float = 0.0, skew: float = 0.0) -> dict:
    return {"kind": kind, "rows": rows, "dims": dims, "experts": count, "width": width, "top_k": top_k, "dtype": dtype,
            "act": act, "limit": limit, "skew": skew}


def _adapters(rows: int, k: int, n: int, count: int, rank: int, dtype: str = "bf16", base: str = "fp32", out: str = "bf16",
              runs: bool = False, kind: str = "adapters") -> dict:
    return {"kind": kind, "rows": rows, "k": k, "n": n, "count": count, "rank": rank, "dtype": dtype, "base": base,
            "out": out, "runs": runs}


def listed() -> list[dict]:
    return [
        # one user's decode step through a layer of 128 experts: eight experts' weights, each read for one row
        {"name": "experts-1", **_experts("experts", 1, 2048, 128, 768, 8)},
        # a decode batch of 64 users: nearly every expert is read, for four rows each on average
        {"name": "experts-64", **_experts("experts", 64, 2048, 128, 768, 8)},
        # a prompt's chunk of odd length on the same layer, experts unevenly liked
        {"name": "experts-1999-skewed", **_experts("experts", 1999, 2048, 128, 768, 8, skew=1.0)},
        # many prompts' tokens at once through the larger layer: bound by the multiplications
        {"name": "experts-8192-wide", **_experts("experts", 8192, 4096, 160, 1536, 8)},
        # the first half in fp16 with ragged sizes, as a model of odd width with one matrix and a squared ReLU has it
        {"name": "gate-up-300-fp16-odd", **_experts("gate_up", 300, 1000, 60, 712, 6, "fp16", "relu2")},
        # the second half in fp16 for a small batch, fp32 rows for a caller that sums them itself
        {"name": "down-48-fp16", **_experts("down", 48, 2048, 128, 768, 8, "fp16")},
        # one user's decode step: one row, its adapter out of 32
        {"name": "adapters-1", **_adapters(1, 2048, 4096, 32, 16)},
        # a decode batch in which most users bring their own adapter, some none
        {"name": "adapters-64", **_adapters(64, 4096, 4096, 128, 32)},
        # a batch of middle size, fp16, onto rows that are already rounded, with odd sizes and a rank of 24
        {"name": "adapters-333-fp16-odd", **_adapters(333, 1544, 2001, 17, 24, "fp16", "fp16", "fp16")},
        # prompts of a few users behind one another
        {"name": "adapters-8192-runs", **_adapters(8192, 4096, 4096, 8, 16, runs=True)},
        # a 4-bit projection of a decode batch with its users' adapters
        {"name": "affine-16", **_adapters(16, 2048, 4096, 64, 16, kind="affine")},
        # and of two prompts
        {"name": "affine-1500-runs", **_adapters(1500, 2048, 4096, 8, 64, runs=True, kind="affine")},
    ]


def _log(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    top = 8192 * 8 * 4096 * 1536                       # rows x slots x sizes of the largest listed block
    weights = 160 * 4096 * 1536
    if rng.random() < 0.55:
        while True:
            count = _log(rng, 3, 256)
            kind = rng.choice(["experts", "experts", "gate_up", "down"])
            dtype = "bf16" if kind == "experts" else rng.choice(["bf16", "fp16"])
            case = _experts(kind, _log(rng, 1, 8192), 8 * _log(rng, 16, 512), count, 8 * _log(rng, 8, 256),
                            min(count, rng.randint(1, 8)), dtype, rng.choice(["swiglu", "swiglu", "relu2"]),
                            rng.choice([0.0, 0.0, 4.0]), rng.choice([0.0, 0.5, 1.5]))
            sizes = case["dims"] * case["width"]
            if case["rows"] * case["top_k"] * sizes <= top and count * sizes <= weights:
                return case
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    base = rng.choice(["fp32", dtype])
    rows = _log(rng, 1, 8192)
    if rng.random() < 0.25:
        return _adapters(min(rows, 4096), 64 * _log(rng, 4, 64), rng.randint(100, 4096), _log(rng, 1, 128),
                         _log(rng, 4, 64), runs=rng.random() < 0.5, kind="affine")
    return _adapters(rows, 8 * _log(rng, 32, 768), _log(rng, 256, 6000), _log(rng, 1, 160), _log(rng, 4, 64), dtype, base,
                     rng.choice([dtype, "fp32"]) if base == "fp32" else base, rng.random() < 0.5)


# ---- inputs -------------------------------------------------------------------------------------------------------
def _gen(seed: int, device=DEV) -> torch.Generator:
    return torch.Generator(device=device).manual_seed(seed)


def _normal(seed: int, shape, scale: float, dtype: torch.dtype) -> torch.Tensor:
    return (torch.randn(shape, generator=_gen(seed), device=DEV, dtype=torch.float32) * scale).to(dtype)


def _picks(case: dict, seed: int) -> torch.Tensor:
    """Each token's experts, distinct, as a router hands them out: a random order with some experts liked more."""

    g = _gen(seed, "cpu")
    liked = torch.randn((case["experts"],), generator=g) * case["skew"]
    score = liked - torch.log(-torch.log(torch.rand((case["rows"], case["experts"]), generator=g).clamp(1e-9, 1 - 1e-7)))
    return score.topk(case["top_k"], dim=1).indices.to(torch.int32)


def _ids(case: dict, seed: int) -> torch.Tensor:
    """Each row's adapter: a decode batch has one request a row, prompts have runs of rows; about a tenth bring none."""

    g = _gen(seed, "cpu")
    rows, count = case["rows"], case["count"]
    if not case["runs"]:
        ids = torch.randint(0, count, (rows,), generator=g)
        ids[torch.rand((rows,), generator=g) < 0.1] = -1
        return ids.to(torch.int32)
    cuts = torch.randint(0, rows + 1, (count,), generator=g).sort().values
    which = torch.randint(-1 if count > 4 else 0, count, (count + 1,), generator=g)
    return which[torch.searchsorted(cuts, torch.arange(rows), right=True)].to(torch.int32)


def _expert_inputs(case: dict, seed: int) -> dict:
    e, d, n, dtype = case["experts"], case["dims"], case["width"], TYPES[case["dtype"]]
    s = {"picks": _picks(case, seed).to(DEV)}
    if case["kind"] != "down":
        mats = 2 if case["act"] == "swiglu" else 1
        s["x"] = _normal(seed + 1, (case["rows"], d), 1.0, dtype)
        s["up"] = [_normal(seed + 2 + i, (e, n, d), d ** -0.5, dtype) for i in range(mats)]
    if case["kind"] != "gate_up":
        s["down"] = _normal(seed + 5, (e, d, n), n ** -0.5, dtype)
    if case["kind"] == "down":
        s["act"] = _normal(seed + 6, (case["rows"] * case["top_k"], n), 0.5, dtype)
    if case["kind"] == "experts":
        raw = torch.rand((case["rows"], case["top_k"]), generator=_gen(seed + 7), device=DEV) + 0.1
        s["wts"] = raw / raw.sum(-1, keepdim=True)
    return s


def _adapter_inputs(case: dict, seed: int) -> dict:
    rows, k, n, count, rank = (case[f] for f in ("rows", "k", "n", "count", "rank"))
    dtype = TYPES[case["dtype"]]
    s = {"ids": _ids(case, seed).to(DEV), "x": _normal(seed + 1, (rows, k), 1.0, dtype),
         "a": _normal(seed + 2, (count, rank, k), k ** -0.5, dtype), "b": _normal(seed + 3, (count, n, rank), 0.1, dtype),
         "scale": torch.rand((count,), generator=_gen(seed + 4), device=DEV) + 0.5}
    if case["kind"] == "adapters":
        s["base"] = _normal(seed + 5, (rows, n), 1.0, TYPES[case["base"]])
    else:
        s["words"] = torch.randint(-(2 ** 31), 2 ** 31, (n, k // 8), generator=_gen(seed + 6), device=DEV,
                                   dtype=torch.int64).to(torch.int32)
        s["scales"] = _normal(seed + 7, (n, k // 64), 0.01, torch.bfloat16).abs()
        s["biases"] = _normal(seed + 8, (n, k // 64), 0.01, torch.bfloat16)
    return s


def prepare(case: dict, seed: int) -> dict:
    """What the program holds before the call: its inputs, the weights as it keeps them, and its scratch."""

    if case["kind"] in ("experts", "gate_up", "down"):
        s = _expert_inputs(case, seed)
        rows, slots, d, n = case["rows"], case["top_k"], case["dims"], case["width"]
        s["limit"] = case["limit"]
        if own:
            from tensorfold_b200 import experts16, moe

            # a layer has both halves; a program that runs one alone still holds a layer's experts
            up = s.pop("up", None) or [torch.zeros((case["experts"], n, d), dtype=TYPES[case["dtype"]], device=DEV)]
            down = s.pop("down", None)
            if down is None:
                down = torch.zeros((case["experts"], d, n), dtype=TYPES[case["dtype"]], device=DEV)
            s["ex"] = experts16.make(up, down, limit=case["limit"])
            del up, down
            if case["kind"] == "experts":
                s["buf"] = moe.buffers(s["ex"], rows, slots, prefill=rows > 256)
            else:
                s["plan"] = experts16.Plan(rows, slots, case["experts"], DEV)
                s["out"] = torch.empty((rows * slots, n if case["kind"] == "gate_up" else d), device=DEV,
                                       dtype=TYPES[case["dtype"]] if case["kind"] == "gate_up" else torch.float32)
    else:
        s = _adapter_inputs(case, seed)
        if own:
            from tensorfold_b200 import adapters, qmm

            s["ad"] = adapters.make(s.pop("a"), s.pop("b"), s.pop("scale"))
            s["plan"] = adapters.Plan(case["rows"], case["count"], DEV)
            if case["kind"] == "affine":
                s["q"] = qmm.pack(s.pop("words"), s.pop("scales"), s.pop("biases"), 64)
    s["case"] = case
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------
def _activation(case: dict, parts: list[torch.Tensor]) -> torch.Tensor:
    if case["act"] == "relu2":
        return torch.relu(parts[0]) ** 2
    g, u = parts
    if case["limit"] > 0:
        g, u = g.clamp(max=case["limit"]), u.clamp(-case["limit"], case["limit"])
    return g / (1 + torch.exp(-g)) * u


def _plain_experts(s: dict) -> torch.Tensor:
    case = s["case"]
    picks = s["picks"].long()
    rows, slots = picks.shape
    order = torch.argsort(picks.reshape(-1), stable=True)
    counts = torch.bincount(picks.reshape(-1), minlength=case["experts"]).tolist()
    kind, dtype = case["kind"], TYPES[case["dtype"]]
    out = torch.empty((rows * slots, case["width"] if kind == "gate_up" else case["dims"]), dtype=torch.float32, device=DEV)
    at = 0
    for e, c in enumerate(counts):
        if c == 0:
            continue
        pairs = order[at:at + c]
        at += c
        if kind == "down":
            v = s["act"][pairs].float()
        else:
            v = s["x"][pairs // slots].float()
            v = _activation(case, [v @ w[e].float().t() for w in s["up"]])
        if kind != "gate_up":
            v = v @ s["down"][e].float().t()
        out[pairs] = v
    if kind == "gate_up":
        return out.to(dtype)
    if kind == "down":
        return out
    return (out.view(rows, slots, -1) * s["wts"][..., None]).sum(1).to(dtype)


def _plain_adapters(s: dict) -> torch.Tensor:
    case = s["case"]
    if case["kind"] == "affine":
        shifts = torch.arange(8, device=DEV, dtype=torch.int32) * 4
        q = ((s["words"][..., None] >> shifts) & 15).reshape(case["n"], case["k"] // 64, 64).float()
        w = q * s["scales"].float()[..., None] + s["biases"].float()[..., None]
        out = s["x"].float() @ w.reshape(case["n"], case["k"]).t()
    else:
        out = s["base"].float()
    ids = s["ids"].long()
    order = torch.argsort(ids, stable=True)
    counts = torch.bincount(ids + 1, minlength=case["count"] + 1).tolist()
    delta = torch.zeros_like(out)
    at = counts[0]
    for i, c in enumerate(counts[1:]):
        if c == 0:
            continue
        rows = order[at:at + c]
        at += c
        low = s["x"][rows].float() @ s["a"][i].float().t() * s["scale"][i]
        delta[rows] = low @ s["b"][i].float().t()
    return (out + delta).to(TYPES[case["out"]])


def run(s: dict):
    case = s["case"]
    if not own:
        return _plain_experts(s) if case["kind"] in ("experts", "gate_up", "down") else _plain_adapters(s)
    from tensorfold_b200 import adapters, experts, experts16, moe, qmm

    if case["kind"] == "experts":
        return moe.picked(s["x"], s["ex"], s["picks"], s["wts"], buf=s["buf"])
    if case["kind"] == "gate_up":
        experts.route(s["picks"], s["plan"])
        experts16.gate_up(s["x"], s["ex"], s["plan"], s["out"], case["rows"])
        return s["out"]
    if case["kind"] == "down":
        experts.route(s["picks"], s["plan"])
        experts16.down(s["act"], s["ex"], s["plan"], s["out"], case["rows"])
        return s["out"]
    adapters.route(s["ids"], s["plan"])
    if case["kind"] == "affine":
        product = qmm.prefill_matmul if case["rows"] > 128 else qmm.matmul
        return product(s["x"], s["q"], adapters=s["ad"], plan=s["plan"])
    return adapters.add(s["x"], s["ad"], s["plan"], s["base"], dtype=TYPES[case["out"]])


# ---- what a pass cannot do without, and what it should give -------------------------------------------------------
def work(case: dict) -> dict:
    """Weights of the experts or adapters that a batch of these sizes picks, rows in and rows out, each once."""

    rows = case["rows"]
    if case["kind"] in ("experts", "gate_up", "down"):
        d, n, pairs = case["dims"], case["width"], rows * case["top_k"]
        used = int(_picks(case, 0).unique().numel())
        mats = 2 if case["act"] == "swiglu" else 1
        up, down = case["kind"] != "down", case["kind"] != "gate_up"
        per = (mats if up else 0) + (1 if down else 0)
        moved = used * per * d * n * 2 + pairs * 4
        moved += rows * d * 2 if up else pairs * n * 2
        moved += {"experts": rows * d * 2 + pairs * 4, "gate_up": pairs * n * 2, "down": pairs * d * 4}[case["kind"]]
        return {"bytes": moved, "flops": 2 * pairs * per * d * n}
    k, n, rank = case["k"], case["n"], case["rank"]
    ids = _ids(case, 0)
    served, used = int((ids >= 0).sum()), int(ids[ids >= 0].unique().numel())
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    moved = used * rank * (k + n) * 2 + rows * (k * 2 + n * size[case["out"]] + 4)
    flops = 2 * served * rank * (k + n)
    if case["kind"] == "affine":
        return {"bytes": moved + n * k // 2 + n * (k // 64) * 4, "flops": flops + 2 * rows * n * k}
    return {"bytes": moved + rows * n * size[case["base"]], "flops": flops}


def exact(case: dict, seed: int):
    """The same in 64 bits, expert by expert and adapter by adapter over masks of the rows."""

    if case["kind"] in ("experts", "gate_up", "down"):
        s = _expert_inputs(case, seed)
        rows, slots = s["picks"].shape
        if case["kind"] == "experts":
            total = torch.zeros((rows, case["dims"]), dtype=torch.float64, device=DEV)
        else:
            total = torch.zeros((rows * slots, case["width"] if case["kind"] == "gate_up" else case["dims"]),
                                dtype=torch.float64, device=DEV)
        for e in range(case["experts"]):
            hit = s["picks"] == e
            if case["kind"] == "down":
                who = hit.reshape(-1).nonzero()[:, 0]
                total[who] = torch.einsum("pk,nk->pn", s["act"][who].double(), s["down"][e].double())
                continue
            who, slot = hit.nonzero(as_tuple=True)
            x = s["x"][who].double()
            up = torch.einsum("pk,nk->pn", x, s["up"][-1][e].double())
            if case["act"] == "relu2":
                act = up.clamp(min=0).square()
            else:
                gate = torch.einsum("pk,nk->pn", x, s["up"][0][e].double())
                if case["limit"] > 0:
                    gate = torch.minimum(gate, torch.full_like(gate, case["limit"]))
                    up = up.clamp(min=-case["limit"], max=case["limit"])
                act = gate * torch.sigmoid(gate) * up
            if case["kind"] == "gate_up":
                total[who * slots + slot] = act
            else:
                y = torch.einsum("pk,nk->pn", act, s["down"][e].double())
                total.index_add_(0, who, y * s["wts"][who, slot].double()[:, None])
        return total
    s = _adapter_inputs(case, seed)
    if case["kind"] == "affine":
        w = s["words"].long() & 0xFFFFFFFF
        q = torch.stack([(w >> (4 * i)) & 15 for i in range(8)], dim=-1).reshape(case["n"], case["k"]).double()
        q = q * s["scales"].double().repeat_interleave(64, 1) + s["biases"].double().repeat_interleave(64, 1)
        total = torch.einsum("mk,nk->mn", s["x"].double(), q)
    else:
        total = s["base"].double()
    for i in range(case["count"]):
        who = (s["ids"] == i).nonzero()[:, 0]
        low = torch.einsum("mk,rk->mr", s["x"][who].double(), s["a"][i].double())
        total[who] += s["scale"][i].double() * torch.einsum("mr,nr->mn", low, s["b"][i].double())
    return total

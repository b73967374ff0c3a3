"""Products of 8-bit floating point numbers with scales, and products grouped by expert: calls of a serving or training program.

A case is one of

* ``quantise``: a matrix to 8-bit floating point with a 32-bit scale for each block of 128, as it is or transposed;
* ``product``: rows of such codes times a weight of such codes, for all rows or by expert;
* ``experts``: 16-bit rows grouped by expert times their experts' weights, or the gradients of that to rows or weights;
* ``rows``: from the experts that each token chose, where each expert's rows begin, which token each row takes and where
  each choice went.
"""
from __future__ import annotations

import math

import torch

own = False

TORCH = {"F32": torch.float32, "Bf16": torch.bfloat16, "F16": torch.float16, "Fp8E4M3FN": torch.float8_e4m3fn,
         "Fp8E5M2": torch.float8_e5m2, "I32": torch.int32, "I64": torch.int64}
SIZE = {"F32": 4, "Bf16": 2, "F16": 2, "I32": 4, "I64": 8}
LARGEST = {"Fp8E4M3FN": 448.0, "Fp8E5M2": 57344.0}


# ---------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # The activations of a long prompt before a product.
        {"name": "quantise_prompt", "kind": "quantise", "rows": 16384, "cols": 8192, "dtype": "Bf16", "codes": "Fp8E4M3FN",
         "block_rows": 1, "transpose": False},
        # A weight after an optimiser's step, transposed for the product that gives its inputs' gradient.
        {"name": "quantise_weight", "kind": "quantise", "rows": 8192, "cols": 4096, "dtype": "F32", "codes": "Fp8E4M3FN",
         "block_rows": 128, "transpose": True},
        # One sequence's next token through a square layer: latency.
        {"name": "product_one", "kind": "product", "m": 1, "n": 4096, "k": 4096, "a": "Fp8E4M3FN", "b": "Fp8E4M3FN",
         "b_rows": 128, "out": "Bf16", "groups": 0},
        # A decode batch through a wide layer: the weight's bytes count.
        {"name": "product_step", "kind": "product", "m": 64, "n": 28672, "k": 8192, "a": "Fp8E4M3FN", "b": "Fp8E4M3FN",
         "b_rows": 128, "out": "Bf16", "groups": 0},
        # A long prompt through a square layer: the matrix products count.
        {"name": "product_prompt", "kind": "product", "m": 8192, "n": 8192, "k": 8192, "a": "Fp8E4M3FN", "b": "Fp8E4M3FN",
         "b_rows": 128, "out": "Bf16", "groups": 0},
        # A prompt's rows by expert.
        {"name": "product_experts", "kind": "product", "m": 16384, "n": 4096, "k": 2048, "a": "Fp8E4M3FN", "b": "Fp8E4M3FN",
         "b_rows": 128, "out": "Bf16", "groups": 32},
        # A decode batch's rows over many experts, a row or two each: the chosen experts' weights are read.
        {"name": "experts_step", "kind": "experts", "direction": "forward", "rows": 64, "n": 4096, "k": 2048, "groups": 64,
         "dtype": "Bf16", "out": "Bf16"},
        # A prompt's, an odd number of rows in all.
        {"name": "experts_prompt", "kind": "experts", "direction": "forward", "rows": 12001, "n": 8192, "k": 2048,
         "groups": 16, "dtype": "Bf16", "out": "Bf16"},
        # The gradients of the same: to the rows, and to the weights in 32 bits.
        {"name": "experts_input_gradient", "kind": "experts", "direction": "input", "rows": 12001, "n": 8192, "k": 2048,
         "groups": 16, "dtype": "Bf16", "out": "Bf16"},
        {"name": "experts_weight_gradient", "kind": "experts", "direction": "weight", "rows": 12001, "n": 8192, "k": 2048,
         "groups": 16, "dtype": "Bf16", "out": "F32"},
        # The choices of a decode batch: launch latency.
        {"name": "rows_step", "kind": "rows", "tokens": 64, "per": 4, "groups": 64, "index": "I32"},
        # And of a prompt.
        {"name": "rows_prompt", "kind": "rows", "tokens": 16384, "per": 8, "groups": 128, "index": "I32"},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    """One more case: any kind, over the range of sizes, types and options that the listed ones stand for."""
    kind = rng.choice(["quantise", "product", "product", "product", "experts", "experts", "experts", "rows"])
    if kind == "quantise":
        while True:
            rows, cols = _log(rng, 1, 28672), _log(rng, 16, 28672)
            if rows * cols <= 1 << 27:
                break
        return {"kind": kind, "rows": rows, "cols": cols if rng.random() < 0.3 else cols // 16 * 16,
                "dtype": rng.choice(["Bf16", "Bf16", "F16", "F32"]), "codes": rng.choice(["Fp8E4M3FN", "Fp8E4M3FN", "Fp8E5M2"]),
                "block_rows": rng.choice([1, 128]), "transpose": rng.random() < 0.4}
    if kind == "product":
        groups = rng.choice([0, 0, _log(rng, 1, 64)])
        while True:
            m = rng.choice([rng.randint(1, 64), _log(rng, 1, 16384)])
            n, k = _log(rng, 64, 28672), _log(rng, 64, 16384)
            if max(1, groups) * n * k <= 1 << 28 and m * n * k <= 1 << 38:
                break
        # Codes of 8 bits lie in rows of whole vectors: an odd length is padded (a gradient's sum over tokens).
        return {"kind": kind, "m": m, "n": n if rng.random() < 0.4 else max(64, n // 64 * 64), "k": k if rng.random() < 0.2 else k // 16 * 16,
                "a": rng.choice(["Fp8E4M3FN", "Fp8E4M3FN", "Fp8E5M2"]), "b": rng.choice(["Fp8E4M3FN", "Fp8E4M3FN", "Fp8E5M2"]),
                "b_rows": rng.choice([128, 128, 1]), "out": rng.choice(["Bf16", "Bf16", "F16"]), "groups": groups}
    if kind == "experts":
        while True:
            rows, groups = rng.choice([rng.randint(1, 128), _log(rng, 1, 16384)]), _log(rng, 1, 128)
            n, k = _log(rng, 64, 16384) // 8 * 8, _log(rng, 64, 16384) // 8 * 8
            if groups * n * k <= 1 << 29 and rows * n * k <= 1 << 37:
                break
        direction, dtype = rng.choice(["forward", "forward", "input", "weight"]), rng.choice(["Bf16", "Bf16", "F16"])
        return {"kind": kind, "direction": direction, "rows": rows, "n": n, "k": k, "groups": groups, "dtype": dtype,
                "out": rng.choice([dtype, dtype, "F32"])}
    per = rng.choice([1, 2, 2, 4, 6, 8])
    return {"kind": kind, "tokens": _log(rng, 1, 16384), "per": per, "groups": _log(rng, max(2, per), 256),
            "index": rng.choice(["I32", "I32", "I64"])}


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _counts(rows: int, groups: int, seed: int) -> list[int]:
    """Ragged groups: some experts are chosen several times as often as others, and some not at all."""
    gen = torch.Generator().manual_seed(int(seed))
    weight = torch.exp(torch.randn(groups, generator=gen) * 0.6)
    picks = torch.multinomial(weight, rows, replacement=True, generator=gen)
    return torch.bincount(picks, minlength=groups).tolist()


def _starts(counts: list[int]) -> torch.Tensor:
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    return torch.tensor(ends, device="cuda", dtype=torch.int32)


def _quantise(y: torch.Tensor, kind: str, block_rows: int):
    """Codes and scales of [..., rows, cols] 32-bit values: the largest magnitude of a block is the largest code."""
    r, c = y.shape[-2:]
    rb, cb = -(-r // block_rows), -(-c // 128)
    z = torch.nn.functional.pad(y, (0, cb * 128 - c, 0, rb * block_rows - r)).unflatten(-1, (cb, 128)).unflatten(-3, (rb, block_rows))
    scale = z.abs().amax((-3, -1)) / LARGEST[kind]
    step = torch.where(scale > 0, scale, torch.ones_like(scale))
    codes = (z / step[..., :, None, :, None]).flatten(-4, -3).flatten(-2)[..., :r, :c]
    return codes.to(TORCH[kind]), scale


def _padded(codes: torch.Tensor) -> torch.Tensor:
    """The same codes in rows of a whole number of 16 bytes."""
    c = codes.shape[-1]
    wide = torch.zeros((*codes.shape[:-1], -(-c // 16) * 16), device=codes.device, dtype=torch.uint8)
    wide[..., :c] = codes.view(torch.uint8)
    return wide.view(codes.dtype)[..., :c]


def _codes(case_kind: str, shape: tuple, block_rows: int, gen, spread: float):
    """Quantised values of unit variance, each row a little larger or smaller than the next."""
    y = torch.randn(shape, generator=gen, device="cuda")
    y *= torch.exp(spread * torch.randn((*shape[:-1], 1), generator=gen, device="cuda"))
    codes, scale = _quantise(y, case_kind, block_rows)
    return _padded(codes), scale


def prepare(case: dict, seed: int) -> dict:
    """The inputs, buffers and plan of a case, from the seed alone."""
    gen, kind = _gen(seed), case["kind"]
    if kind == "quantise":
        r, c = case["rows"], case["cols"]
        x = torch.randn((r, c), generator=gen, device="cuda")
        x = (x * torch.exp(torch.randn((r, 1), generator=gen, device="cuda"))).to(TORCH[case["dtype"]])
        tr, tc = (c, r) if case["transpose"] else (r, c)
        wide = torch.empty((tr, -(-tc // 16) * 16), device="cuda", dtype=torch.uint8).view(TORCH[case["codes"]])
        return {"case": case, "x": x, "codes": wide[:, :tc],
                "scales": torch.empty((-(-tr // case["block_rows"]), -(-tc // 128)), device="cuda", dtype=torch.float32)}
    if kind == "product":
        m, n, k, groups = case["m"], case["n"], case["k"], case["groups"]
        a, a_scale = _codes(case["a"], (m, k), 1, gen, 0.5)
        b, b_scale = _codes(case["b"], (max(1, groups), n, k), case["b_rows"], gen, 0.2)
        state = {"case": case, "a": a, "a_scale": a_scale, "b": b, "b_scale": b_scale,
                 "out": torch.empty((m, n), device="cuda", dtype=TORCH[case["out"]])}
        if groups:
            state["counts"] = _counts(m, groups, seed)
            state["starts"] = _starts(state["counts"])
        return state
    if kind == "experts":
        rows, n, k, groups = case["rows"], case["n"], case["k"], case["groups"]
        t, out, d = TORCH[case["dtype"]], TORCH[case["out"]], case["direction"]
        counts = _counts(rows, groups, seed)
        wide = k if d == "forward" else n
        state = {"case": case, "counts": counts, "starts": _starts(counts),
                 "x": torch.randn((rows, wide), generator=gen, device="cuda").to(t)}
        if d == "weight":
            state["y"] = torch.randn((rows, k), generator=gen, device="cuda").to(t)
            state["out"] = torch.empty((groups, n, k), device="cuda", dtype=out)
        else:
            state["w"] = (torch.randn((groups, n, k), generator=gen, device="cuda") / math.sqrt(wide)).to(t)
            state["out"] = torch.empty((rows, n if d == "forward" else k), device="cuda", dtype=out)
        return state
    tokens, per, groups = case["tokens"], case["per"], case["groups"]
    # A token's choices are different experts; some experts are chosen more often, and a few tokens are padding.
    likes = torch.randn((tokens, groups), generator=gen, device="cuda") + 0.6 * torch.randn(groups, generator=gen, device="cuda")
    ids = likes.topk(per, 1).indices.to(TORCH[case["index"]])
    ids[tokens // 2::89] = -1
    n = tokens * per
    return {"case": case, "ids": ids.contiguous(), "starts": torch.empty(groups + 1, device="cuda", dtype=torch.int32),
            "rows": torch.empty(n, device="cuda", dtype=torch.int32), "place": torch.empty(n, device="cuda", dtype=torch.int32)}


# ---------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------
_kept: dict = {}


def _executor(how: str, **form):
    """A program lowers a kernel once and keeps its executor."""
    import unpopped_amd as u

    key = (how, *form.values())
    if key not in _kept:
        _kept[key] = u.Executor(getattr(u.HipBackend(), how)(**form))
    return _kept[key]


def _held(t: torch.Tensor):
    """A tensor's memory as a launch argument."""
    import unpopped_amd as u

    return u.DeviceBuffer.held(t.data_ptr(), t.untyped_storage().nbytes() - t.storage_offset() * t.element_size(), t)


def _workspace(state: dict, ex, *shape: int) -> torch.Tensor:
    """A program keeps the workspace of a call that it makes again."""
    if "workspace" not in state:
        state["workspace"] = torch.empty(ex.workspace_bytes(*shape), device="cuda", dtype=torch.uint8)
    return state["workspace"]


def _run_own(state: dict):
    case, stream = state["case"], torch.cuda.current_stream().cuda_stream
    kind = case["kind"]
    if kind == "quantise":
        x, codes, scales = state["x"], state["codes"], state["scales"]
        ex = _executor("lower_quant8", dtype=case["dtype"], kind=case["codes"], block_rows=case["block_rows"],
                       transpose=case["transpose"])
        ex.launch(_held(x), _held(codes), _held(scales), x.shape[0], x.shape[1], x.stride(0), codes.stride(0),
                  scales.stride(0), stream=stream)
        return {"codes": codes, "scales": scales}
    if kind == "product":
        a, b, out, groups = state["a"], state["b"], state["out"], case["groups"]
        sa, sb = state["a_scale"], state["b_scale"]
        ex = _executor("lower_matmul8", a_kind=case["a"], b_kind=case["b"], out=case["out"], b_rows=case["b_rows"],
                       grouped=groups > 0)
        shape = (a.shape[0], b.shape[1], a.shape[1])
        strides = (a.stride(0), sa.stride(0), b.stride(1), sb.stride(1))
        if groups:
            ws = _workspace(state, ex, *shape, groups)
            ex.launch(_held(a), _held(sa), _held(b), _held(sb), _held(state["starts"]), _held(out), _held(ws), *shape, groups,
                      *strides, b.stride(0), sb.stride(0), out.stride(0), ws.numel(), stream=stream)
        else:
            ws = _workspace(state, ex, *shape)
            ex.launch(_held(a), _held(sa), _held(b), _held(sb), _held(out), _held(ws), *shape, *strides, out.stride(0),
                      ws.numel(), stream=stream)
        return out
    if kind == "experts":
        x, out = state["x"], state["out"]
        ex = _executor("lower_grouped_matmul", dtype=case["dtype"], out=case["out"], direction=case["direction"])
        shape = (case["rows"], case["n"], case["k"], case["groups"])
        ws = _workspace(state, ex, *shape)
        if case["direction"] == "weight":
            y = state["y"]
            ex.launch(_held(x), _held(y), _held(state["starts"]), _held(out), _held(ws), *shape, x.stride(0), y.stride(0),
                      out.stride(0), out.stride(1), ws.numel(), stream=stream)
        else:
            w = state["w"]
            ex.launch(_held(x), _held(w), _held(state["starts"]), _held(out), _held(ws), *shape, x.stride(0), w.stride(0),
                      w.stride(1), out.stride(0), ws.numel(), stream=stream)
        return out
    ids = state["ids"]
    ex = _executor("lower_group_rows", index_dtype=case["index"])
    shape = (ids.numel(), case["per"], case["groups"])
    ws = _workspace(state, ex, *shape)
    ex.launch(_held(ids), _held(state["starts"]), _held(state["rows"]), _held(state["place"]), _held(ws), *shape, ws.numel(),
              stream=stream)
    return {k: state[k] for k in ("starts", "rows", "place")}


# ---------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------
def _scaled(codes: torch.Tensor, scale: torch.Tensor, block_rows: int) -> torch.Tensor:
    """What codes [..., rows, cols] stand for, in 32 bits."""
    r, c = codes.shape[-2:]
    s = scale.repeat_interleave(128, -1)[..., :c]
    if block_rows > 1:
        s = s.repeat_interleave(block_rows, -2)[..., :r, :]
    return codes.float() * s


def _places(state: dict, rows: int):
    """Where the rows of each group lie when they are padded to the longest group: [groups, most], and whether there is one."""
    most = max(max(state["counts"]), 1)
    starts = state["starts"].long()
    row = torch.arange(most, device=starts.device)
    there = row[None, :] < (starts[1:] - starts[:-1])[:, None]
    return torch.where(there, starts[:-1, None] + row[None, :], rows), there


def _by_group(state: dict, x: torch.Tensor, w: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """Rows x [rows, a] times their groups' w [groups, a, b], all in 32 bits."""
    at, _ = _places(state, x.shape[0])
    wide = torch.cat([x, torch.zeros_like(x[:1])])[at]
    got = torch.empty((x.shape[0] + 1, w.shape[2]), device=x.device)
    got[at] = torch.matmul(wide, w.contiguous())
    return got[:-1].to(out.dtype)


def _rows_plain(state: dict):
    case, ids = state["case"], state["ids"].flatten().long()
    groups, per = case["groups"], case["per"]
    chosen = (ids[None, :] == torch.arange(groups, device=ids.device)[:, None]).int()
    before = chosen.cumsum(1, dtype=torch.int32) - chosen
    count = chosen.sum(1)
    starts = torch.cat([count.new_zeros(1), count.cumsum(0)])
    kept = (ids >= 0) & (ids < groups)
    safe = ids.clamp(0, groups - 1)
    place = torch.where(kept, starts[safe] + before.gather(0, safe[None, :])[0], -1)
    token = torch.arange(ids.numel(), device=ids.device) // per
    rows = torch.full((ids.numel() + 1,), -1, device=ids.device, dtype=torch.int64)
    rows[torch.where(kept, place, ids.numel())] = token
    return {"starts": starts.int(), "rows": rows[:-1].int(), "place": place.int()}


def run(state: dict):
    """One pass; the outputs of the framework's calls are the program's own buffers."""
    if own:
        return _run_own(state)
    case = state["case"]
    kind = case["kind"]
    if kind == "quantise":
        y = state["x"].float()
        codes, scales = _quantise(y.t() if case["transpose"] else y, case["codes"], case["block_rows"])
        return {"codes": codes, "scales": scales}
    if kind == "product":
        a = _scaled(state["a"], state["a_scale"], 1)
        b = _scaled(state["b"], state["b_scale"], case["b_rows"])
        if case["groups"]:
            return _by_group(state, a, b.transpose(1, 2), state["out"])
        return torch.matmul(a, b[0].t()).to(state["out"].dtype)
    if kind == "experts":
        x, d = state["x"].float(), case["direction"]
        if d != "weight":
            w = state["w"].float()
            return _by_group(state, x, w.transpose(1, 2) if d == "forward" else w, state["out"])
        at, there = _places(state, x.shape[0])
        y = state["y"].float()
        wide = [torch.cat([v, torch.zeros_like(v[:1])])[at] for v in (x, y)]
        return torch.matmul(wide[0].transpose(1, 2).contiguous(), wide[1]).to(state["out"].dtype)
    return _rows_plain(state)


# ---------------------------------------------------------------------------------------
# What the work is, and its results in 64 bits
# ---------------------------------------------------------------------------------------
def _used(case: dict) -> int:
    """About how many groups have rows: what a draw of this many rows leaves chosen."""
    g = max(1, case["groups"])
    return max(1, min(g, round(g * (1.0 - (1.0 - 1.0 / g) ** case.get("rows", case.get("m", 1))))))


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "quantise":
        n = case["rows"] * case["cols"]
        r, c = (case["cols"], case["rows"]) if case["transpose"] else (case["rows"], case["cols"])
        scales = -(-r // case["block_rows"]) * -(-c // 128)
        return {"bytes": n * (SIZE[case["dtype"]] + 1) + 4 * scales, "flops": 4 * n}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        blocks = -(-k // 128)
        weight = n * k + 4 * -(-n // case["b_rows"]) * blocks
        return {"bytes": m * k + 4 * m * blocks + _used(case) * weight + m * n * SIZE[case["out"]], "flops": 2 * m * n * k}
    if kind == "experts":
        rows, n, k = case["rows"], case["n"], case["k"]
        e, o = SIZE[case["dtype"]], SIZE[case["out"]]
        if case["direction"] == "weight":
            moved = rows * (n + k) * e + case["groups"] * n * k * o
        else:
            first, last = (k, n) if case["direction"] == "forward" else (n, k)
            moved = rows * first * e + _used(case) * n * k * e + rows * last * o
        return {"bytes": moved, "flops": 2 * rows * n * k}
    n = case["tokens"] * case["per"]
    return {"bytes": n * (SIZE[case["index"]] + 8) + 4 * (case["groups"] + 1), "flops": 2 * n}


def _exact_codes(v: torch.Tensor, kind: str) -> torch.Tensor:
    """64-bit values at the nearest number of an 8-bit type, ties to the even one, none past its largest."""
    bits, least = (3, -6) if kind == "Fp8E4M3FN" else (2, -14)
    _, e = torch.frexp(v.abs())
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=least) - bits)
    return (torch.round(v / step) * step).clamp(-LARGEST[kind], LARGEST[kind])


def _exact_product(a, sa, b, sb, b_rows):
    """Codes a [m, k] times b [n, k], a block of the sum at a time."""
    out = torch.zeros((a.shape[0], b.shape[0]), device=a.device, dtype=torch.float64)
    for i in range(sa.shape[1]):
        at = slice(128 * i, min(128 * (i + 1), a.shape[1]))
        col = sb[:, i].double()
        if b_rows > 1:
            col = col[torch.arange(b.shape[0], device=b.device) // b_rows]
        out += (a[:, at].double() @ b[:, at].double().t()) * sa[:, i].double()[:, None] * col[None, :]
    return out


def exact(case: dict, seed: int):
    """What `run` returns, from the definitions in 64 bits."""
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "rows":
        return None  # whole numbers
    if kind == "quantise":
        y = state["x"].t() if case["transpose"] else state["x"]
        codes = torch.zeros(y.shape, device="cuda", dtype=torch.float64)
        scales = torch.zeros(state["scales"].shape, device="cuda", dtype=torch.float64)
        for j in range(scales.shape[1]):
            part = y[:, 128 * j:128 * (j + 1)].double()
            most = part.abs().max(1).values
            group = torch.arange(y.shape[0], device="cuda") // case["block_rows"]
            top = torch.zeros(scales.shape[0], device="cuda", dtype=torch.float64).scatter_reduce_(0, group, most, "amax")
            scales[:, j] = top / LARGEST[case["codes"]]
            # The step that a code counts in is the 32-bit scale by definition.
            unit = (top.float() / LARGEST[case["codes"]]).double()
            unit = torch.where(unit == 0, torch.ones_like(unit), unit)[group]
            codes[:, 128 * j:128 * (j + 1)] = _exact_codes(part / unit[:, None], case["codes"])
        return {"codes": codes, "scales": scales}
    if kind == "product":
        a, sa, b, sb, rows = state["a"], state["a_scale"], state["b"], state["b_scale"], case["b_rows"]
        if not case["groups"]:
            return _exact_product(a, sa, b[0], sb[0], rows)
        out, at = [], 0
        for g, c in enumerate(state["counts"]):
            out.append(_exact_product(a[at:at + c], sa[at:at + c], b[g], sb[g], rows))
            at += c
        return torch.cat(out)
    out, at = [], 0
    for g, c in enumerate(state["counts"]):
        x = state["x"][at:at + c].double()
        if case["direction"] == "weight":
            out.append((x.t().contiguous() @ state["y"][at:at + c].double())[None])
        else:
            w = state["w"][g].double()
            out.append(x @ (w.t().contiguous() if case["direction"] == "forward" else w))
        at += c
    return torch.cat(out)

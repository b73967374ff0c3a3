"""Rotary positions and the 4-bit paged key/value cache: calls that a serving or training program makes.

A case is one of

* ``table``: the cosines and sines of a run of positions, scaled for long contexts;
* ``rotate``: the rotation of a batch's heads by their tokens' positions, or its gradient;
* ``append``: a step's keys (rotated on the way) and values quantised into their cache slots, then read back;
* ``attend``: a ragged batch's query rows against the pages of their sequences' cache.

The cache is one array of bytes: per page and key/value head a record of the key codes, the value codes and the
words of both (an f16 scale below a 16-bit zero point) per group and token.
"""
from __future__ import annotations

import math

import torch

own = False

TORCH = {"F32": torch.float32, "Bf16": torch.bfloat16, "F16": torch.float16}
INDEX = {"I32": torch.int32, "I64": torch.int64}
SIZE = {"F32": 4, "Bf16": 2, "F16": 2, "I32": 4, "I64": 8}
PLAIN = {"scaling": "none", "factor": 1.0, "low": 1.0, "high": 4.0, "original": 8192, "amplitude": 1.0}
STRETCHED = {"scaling": "ramp", "factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192, "amplitude": 1.0}


# ---------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # The positions of one context length, made when a model is loaded: a small call.
        {"name": "table_context", "kind": "table", "rot": 128, "base": 10000.0, "first": 0, "count": 8192, **PLAIN},
        # A long context's far positions with stretched frequencies.
        {"name": "table_far", "kind": "table", "rot": 128, "base": 500000.0, "first": 1 << 20, "count": 262144,
         **STRETCHED},
        # The query and key heads of a decode batch, one token each: launch latency.
        {"name": "rotate_step", "kind": "rotate", "tokens": 32, "heads": 40, "row_heads": 48, "head_dim": 128,
         "rot": 128, "layout": "halves", "dtype": "Bf16", "index": "I32", "inverse": False},
        # The query and key heads of a long prompt, inside the rows of a fused projection.
        {"name": "rotate_prompt", "kind": "rotate", "tokens": 16384, "heads": 40, "row_heads": 48, "head_dim": 128,
         "rot": 128, "layout": "halves", "dtype": "Bf16", "index": "I32", "inverse": False},
        # The gradient of a rotation of part of the head, interleaved pairs, 32-bit training, an odd count.
        {"name": "rotate_gradient", "kind": "rotate", "tokens": 4001, "heads": 24, "row_heads": 24, "head_dim": 128,
         "rot": 64, "layout": "pairs", "dtype": "F32", "index": "I64", "inverse": True},
        # A decode batch's new keys and values: one token per sequence.
        {"name": "append_step", "kind": "append", "tokens": 64, "kv_heads": 8, "head_dim": 128, "group": 128,
         "page": 16, "rot": 128, "layout": "halves", "dtype": "Bf16", "index": "I32"},
        # A whole prompt's.
        {"name": "append_prompt", "kind": "append", "tokens": 16384, "kv_heads": 8, "head_dim": 128, "group": 128,
         "page": 16, "rot": 128, "layout": "halves", "dtype": "Bf16", "index": "I32"},
        # Smaller groups, an odd head and token count, interleaved pairs over part of the head, 16-bit floats.
        {"name": "append_grouped", "kind": "append", "tokens": 4999, "kv_heads": 5, "head_dim": 96, "group": 32,
         "page": 64, "rot": 32, "layout": "pairs", "dtype": "F16", "index": "I64"},
        # A few sequences' next tokens over short contexts: latency.
        {"name": "attend_step_small", "kind": "attend", "batch": 4, "q": 1, "context": 1500, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "group": 128, "page": 16, "window": 0, "dtype": "Bf16"},
        # A full decode batch over ragged contexts: the cache's bytes count.
        {"name": "attend_step_batch", "kind": "attend", "batch": 64, "q": 1, "context": 16384, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "group": 128, "page": 16, "window": 0, "dtype": "Bf16"},
        # One sequence's next token over a very long context: the work has to be split along the keys.
        {"name": "attend_step_long", "kind": "attend", "batch": 1, "q": 1, "context": 262144, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "group": 64, "page": 64, "window": 0, "dtype": "Bf16"},
        # Prompts of three sequences, causal: the matrix products count.
        {"name": "attend_prompt", "kind": "attend", "batch": 3, "q": 4099, "context": 4099, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "group": 128, "page": 16, "window": 0, "dtype": "Bf16"},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    """One more case: any kind, over the range of sizes, types and options that the listed ones stand for."""
    kind = rng.choice(["table", "rotate", "append", "append", "attend", "attend", "attend"])
    if kind == "table":
        return {"kind": kind, "rot": 2 * rng.randint(8, 64), "base": rng.choice([10000.0, 500000.0, 1000000.0]),
                "first": rng.choice([0, _log(rng, 1, 1 << 22)]), "count": _log(rng, 1, 262144),
                "scaling": rng.choice(["none", "linear", "ramp"]), "factor": rng.choice([2.0, 4.0, 8.0, 32.0]),
                "low": 1.0, "high": rng.choice([4.0, 32.0]), "original": rng.choice([4096, 8192, 32768]),
                "amplitude": rng.choice([1.0, 1.1386])}
    if kind == "rotate":
        d = rng.choice([64, 80, 96, 128, 192, 256])
        rot = rng.choice([d, d, d // 2, d // 4])
        while True:
            tokens, heads = _log(rng, 1, 16384), rng.randint(1, 64)
            if tokens * heads * d <= 16384 * 40 * 128:
                break
        return {"kind": kind, "tokens": tokens, "heads": heads, "row_heads": heads + rng.choice([0, 0, rng.randint(1, 16)]),
                "head_dim": d, "rot": rot, "layout": rng.choice(["halves", "pairs"]),
                "dtype": rng.choice(["Bf16", "Bf16", "F16", "F32"]), "index": rng.choice(["I32", "I64"]),
                "inverse": rng.random() < 0.4}
    d = rng.choice([32, 64, 64, 96, 128, 128, 128, 160, 192, 256])
    group = rng.choice([g for g in (32, 64, 128, d, d) if d % g == 0])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    if kind == "append":
        while True:
            tokens, kv = _log(rng, 1, 16384), rng.randint(1, 16)
            if tokens * kv * d <= 16384 * 8 * 128:
                break
        return {"kind": kind, "tokens": tokens, "kv_heads": kv, "head_dim": d, "group": group, "page": page,
                "rot": rng.choice([0, d, d, d // 32 * 16]), "layout": rng.choice(["halves", "pairs"]),
                "dtype": rng.choice(["Bf16", "Bf16", "F16"]), "index": rng.choice(["I32", "I64"])}
    while True:
        kv, gqa = rng.randint(1, 8), rng.choice([1, 2, 4, 4, 5, 6, 7, 8, 16])
        batch = _log(rng, 1, 96)
        q = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 16, 2048)])
        context = max(q, _log(rng, 8, 131072))
        if batch * context * kv * d <= 1 << 29 and batch * q * kv * gqa * context <= 1 << 29:
            break
    return {"kind": kind, "batch": batch, "q": q, "context": context, "heads": kv * gqa, "kv_heads": kv, "head_dim": d,
            "group": group, "page": page, "window": rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
            "dtype": rng.choice(["Bf16", "Bf16", "F16"])}


def _spread(most: int, batch: int, phase: float = 0.0) -> list[int]:
    """Ragged lengths: the first is the longest, the others lie between three tenths of it and all of it."""
    return [max(1, round(most * (1.0 - 0.7 * math.fmod(b * 0.6180339887498949 + (phase if b else 0.0), 1.0))))
            for b in range(batch)]


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Each sequence's new rows and its whole context (the new rows are its end)."""
    rows = _spread(case["q"], case["batch"])
    ends = _spread(case["context"], case["batch"], 0.3)
    return rows, [max(n, e) if case["q"] < case["context"] else n for n, e in zip(rows, ends)]


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _angles(case: dict, positions: torch.Tensor) -> torch.Tensor:
    """positions x rot/2 angles in 64 bits."""
    i = torch.arange(case["rot"] // 2, device=positions.device, dtype=torch.float64)
    f = torch.exp(i * (-2.0 / case["rot"] * math.log(case["base"])))
    if case["scaling"] == "linear":
        f = f / case["factor"]
    if case["scaling"] == "ramp":
        turns = f * (case["original"] / (2.0 * math.pi))
        keep = ((turns - case["low"]) / (case["high"] - case["low"])).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / case["factor"])
    return positions.double()[:, None] * f[None, :]


def _table(case: dict, rows: int) -> torch.Tensor:
    """The table a program made once: [rows][rot / 2][cos, sin]."""
    a = _angles({"rot": case["rot"], "base": 10000.0, **PLAIN}, torch.arange(rows, device="cuda"))
    return torch.stack([a.cos(), a.sin()], 2).float()


def _words(scale: torch.Tensor, zero: torch.Tensor) -> torch.Tensor:
    """Words of an f16 scale and a zero point, as four bytes each (one more axis)."""
    return torch.stack([scale.view(torch.int16), zero.to(torch.int16)], -1).view(torch.uint8)


def _quantise(y: torch.Tensor, group: int):
    """Codes, scales and zero points of [..., head_dim] values of a 16-bit type: the range of each group, with 0 in
    it, in 15 steps of a 16-bit scale."""
    g = y.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1).clamp(max=0.0), g.amax(-1).clamp(min=0.0)
    scale = ((hi - lo) / 15.0).half()
    s = scale.float()
    step = torch.where(s > 0, s, torch.ones_like(s))
    zero = (-lo / step).round().clamp(0.0, 15.0)
    code = ((g / step[..., None]).round() + zero[..., None]).clamp(0.0, 15.0)
    return code.to(torch.uint8).flatten(-2), scale, zero.to(torch.uint8)


def _key_bytes(code: torch.Tensor) -> torch.Tensor:
    """[..., head_dim] codes as a token's key bytes: words of 8 codes, word w at place (w % 4) * (head_dim / 32) + w / 4."""
    two = code[..., 0::2] | (code[..., 1::2] << 4)
    return two.unflatten(-1, (-1, 4, 4)).transpose(-3, -2).flatten(-3)


def _value_bytes(code: torch.Tensor) -> torch.Tensor:
    """[..., head_dim] codes as a token's words of 8 value codes: [..., head_dim / 8, 4]."""
    two = code[..., 0::2] | (code[..., 1::2] << 4)
    return two.unflatten(-1, (-1, 4))


def _parts(case: dict, cache: torch.Tensor):
    """The cache's parts as views: key bytes [pages, heads, page, D/2], value bytes [.., page/4, D/8, 4, 4], key and
    value words [.., groups, page, 4]."""
    p, d, g = case["page"], case["head_dim"], case["head_dim"] // case["group"]
    half = p * d // 2
    lead = cache.shape[:-1]
    keys = cache[..., :half].unflatten(-1, (p, d // 2))
    values = cache[..., half:2 * half].unflatten(-1, (p // 4, d // 8, 4, 4))
    kw = cache[..., 2 * half:2 * half + 4 * p * g].unflatten(-1, (g, p, 4))
    vw = cache[..., 2 * half + 4 * p * g:].unflatten(-1, (g, p, 4))
    assert keys.shape[:-2] == lead
    return keys, values, kw, vw


def _record(case: dict) -> int:
    return case["page"] * (case["head_dim"] + 8 * (case["head_dim"] // case["group"]))


def _nibbles(two: torch.Tensor) -> torch.Tensor:
    return torch.stack([two & 15, two >> 4], -1).flatten(-2)


def _scaled(code: torch.Tensor, words: torch.Tensor, group: int) -> torch.Tensor:
    """(code - zero) * scale in 32 bits: codes [..., head_dim], words [..., groups, 4 bytes]."""
    w = words.contiguous().view(torch.int16)
    scale, zero = w[..., 0].view(torch.float16).float(), w[..., 1].float()
    return ((code.float().unflatten(-1, (-1, group)) - zero[..., None]) * scale[..., None]).flatten(-2)


def _page_values(case: dict, records: torch.Tensor):
    """The values that records [..., bytes] stand for: keys and values [..., page, head_dim] in 32 bits."""
    d, group = case["head_dim"], case["group"]
    keys, values, kw, vw = _parts(case, records)
    kc = _nibbles(keys.unflatten(-1, (4, d // 32, 4)).transpose(-3, -2).flatten(-3))
    vc = _nibbles(values.transpose(-3, -2).flatten(-2)).flatten(-3, -2)
    return _scaled(kc, kw.transpose(-3, -2), group), _scaled(vc, vw.transpose(-3, -2), group)


def _filled(case: dict, gen, pages: int) -> torch.Tensor:
    """Pages of a cache in use, every slot of them: keys and values of unit variance, quantised."""
    p, h, d = case["page"], case["kv_heads"], case["head_dim"]
    cache = torch.empty((pages, h, _record(case)), device="cuda", dtype=torch.uint8)
    at = max(1, (1 << 26) // (p * h * d))
    for i in range(0, pages, at):  # a part at a time: the 32-bit values of a large cache are many
        n = min(at, pages - i)
        keys, values, kw, vw = _parts(case, cache[i:i + n])
        for words, which in ((kw, 0), (vw, 1)):
            y = torch.randn((n, h, p, d), generator=gen, device="cuda").to(TORCH[case["dtype"]])
            code, scale, zero = _quantise(y, case["group"])
            words.copy_(_words(scale, zero).transpose(-3, -2))
            if which == 0:
                keys.copy_(_key_bytes(code))
            else:
                values.copy_(_value_bytes(code).unflatten(-3, (-1, 4)).transpose(-3, -2))
    return cache


def prepare(case: dict, seed: int) -> dict:
    """The inputs, buffers and plan of a case, from the seed alone."""
    gen, kind = _gen(seed), case["kind"]
    if kind == "table":
        # Another seed is another run of positions.
        first = case["first"] + int(seed) % 4096
        return {"case": case, "first": first,
                "out": torch.empty((case["count"], case["rot"] // 2, 2), device="cuda", dtype=torch.float32)}
    if kind == "rotate":
        t, d = case["tokens"], case["head_dim"]
        x = torch.randn((t, case["row_heads"], d), generator=gen, device="cuda").to(TORCH[case["dtype"]])
        pos = torch.randint(0, 32768, (t,), generator=gen, device="cuda", dtype=INDEX[case["index"]])
        return {"case": case, "x": x[:, :case["heads"]], "positions": pos, "table": _table(case, 32768),
                "out": torch.empty((t, case["heads"], d), device="cuda", dtype=x.dtype)}
    if kind == "append":
        t, h, d, p = case["tokens"], case["kv_heads"], case["head_dim"], case["page"]
        rows = torch.randn((t, 3 * h, d), generator=gen, device="cuda")  # a fused projection's queries, keys, values
        rows = rows.to(TORCH[case["dtype"]])
        pos = torch.randint(0, 32768, (t,), generator=gen, device="cuda", dtype=INDEX[case["index"]])
        pages = -(-2 * t // p) + 1
        slots = torch.randperm(pages * p, generator=gen, device="cuda")[:t]
        if t >= 256:  # long runs of one sequence lie in a row inside their pages
            order = torch.randperm(pages, generator=gen, device="cuda")
            slots = (order[:, None] * p + torch.arange(p, device="cuda")[None, :]).flatten()[:t].contiguous()
        slots[t // 2::97] = -1  # padded rows of the batch, which have no slot
        state = {"case": case, "k": rows[:, h:2 * h], "v": rows[:, 2 * h:], "slots": slots.to(INDEX[case["index"]]),
                 "cache": torch.zeros((pages, h, _record(case)), device="cuda", dtype=torch.uint8),
                 "ko": torch.empty((t, h, d), device="cuda", dtype=rows.dtype),
                 "vo": torch.empty((t, h, d), device="cuda", dtype=rows.dtype)}
        if case["rot"]:
            state |= {"positions": pos, "table": _table(case, 32768)}
        return state
    rows, ends = _lengths(case)
    p, b, h, d = case["page"], case["batch"], case["kv_heads"], case["head_dim"]
    need = [-(-e // p) for e in ends]
    width, pages = max(need), sum(need) + 3
    cache = _filled(case, gen, pages)
    order = torch.randperm(pages, generator=gen, device="cuda")
    table = torch.full((b, width), -1, device="cuda", dtype=torch.int32)
    filled = torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table[filled] = order[:sum(need)].to(torch.int32)
    t = sum(rows)
    q = torch.randn((t, case["heads"], d), generator=gen, device="cuda").to(TORCH[case["dtype"]])
    starts = [sum(rows[:i]) for i in range(b + 1)]
    return {"case": case, "q": q, "cache": cache, "pages": table, "most": max(rows),
            "starts": torch.tensor(starts, device="cuda", dtype=torch.int32),
            "lengths": torch.tensor(ends, device="cuda", dtype=torch.int32), "out": torch.empty_like(q)}


# ---------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------
_kept: dict = {}


def _executor(how: str, **form):
    """A program lowers a kernel once and keeps its executor."""
    import unpopped_amd as u

    key = (how, *sorted(form.items()))
    if key not in _kept:
        _kept[key] = u.Executor(getattr(u.HipBackend(), how)(**form))
    return _kept[key]


def _held(t: torch.Tensor):
    """A tensor's memory as a launch argument."""
    import unpopped_amd as u

    return u.DeviceBuffer.held(t.data_ptr(), t.untyped_storage().nbytes() - t.storage_offset() * t.element_size(), t)


def _run_own(state: dict):
    case = state["case"]
    kind, stream = case["kind"], torch.cuda.current_stream().cuda_stream
    if kind == "table":
        ex = _executor("lower_rope_table", **{k: case[k] for k in ("rot", "base", "scaling", "factor", "low", "high",
                                                                   "original", "amplitude")})
        ex.launch(_held(state["out"]), state["first"], case["count"], stream=stream)
        return state["out"]
    if kind == "rotate":
        x, out, table = state["x"], state["out"], state["table"]
        ex = _executor("lower_rope", dtype=case["dtype"], head_dim=case["head_dim"], rot=case["rot"],
                       layout=case["layout"], index_dtype=case["index"], inverse=case["inverse"])
        ex.launch(_held(x), _held(state["positions"]), _held(table), _held(out), case["tokens"], case["heads"],
                  x.stride(0), x.stride(1), out.stride(0), out.stride(1), 0, table.shape[0], stream=stream)
        return out
    form = {k: case[k] for k in ("dtype", "kv_heads", "head_dim", "group", "page")}
    if kind == "append":
        k, v, ko, vo, t = state["k"], state["v"], state["ko"], state["vo"], case["tokens"]
        slots, cache = _held(state["slots"]), _held(state["cache"])
        pages = state["cache"].shape[0]
        ex = _executor("lower_cache4_append", **form, rot=case["rot"], layout=case["layout"], index_dtype=case["index"])
        strides = (k.stride(0), k.stride(1), v.stride(0), v.stride(1))
        if case["rot"]:
            table = state["table"]
            ex.launch(_held(k), _held(v), slots, cache, _held(state["positions"]), _held(table), t, pages, *strides, 0,
                      table.shape[0], stream=stream)
        else:
            ex.launch(_held(k), _held(v), slots, cache, t, pages, *strides, stream=stream)
        ex = _executor("lower_cache4_read", **form, index_dtype=case["index"])
        ex.launch(slots, cache, _held(ko), _held(vo), t, pages, ko.stride(0), ko.stride(1), vo.stride(0), vo.stride(1),
                  stream=stream)
        return {"k": ko, "v": vo}
    q, out = state["q"], state["out"]
    ex = _executor("lower_cache4_attention", **form, heads=case["heads"], causal=True)
    shape = (q.shape[0], case["batch"], state["pages"].shape[1], state["cache"].shape[0])
    if "workspace" not in state:
        state["workspace"] = torch.empty(ex.workspace_bytes(*shape), device="cuda", dtype=torch.uint8)
    ws = state["workspace"]
    ex.launch(_held(q), _held(state["cache"]), _held(state["pages"]), _held(state["starts"]), _held(state["lengths"]),
              _held(out), _held(ws), *shape, q.stride(0), q.stride(1), out.stride(0), out.stride(1), case["window"],
              ws.numel(), stream=stream)
    return out


# ---------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------
def _turn(case: dict, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """The first rot elements of [tokens, heads, head_dim] rotated, in the type of x; cos and sin [tokens, 1, rot / 2]."""
    rot = case["rot"]
    a, rest = x[..., :rot], x[..., rot:]
    if case["layout"] == "halves":
        x0, x1 = a[..., :rot // 2], a[..., rot // 2:]
        y = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1)
    else:
        x0, x1 = a[..., 0::2], a[..., 1::2]
        y = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1).flatten(-2)
    return torch.cat([y, rest], -1)


def _append_plain(state: dict):
    case, cache = state["case"], state["cache"]
    k, v, p, group = state["k"], state["v"], case["page"], case["group"]
    if case["rot"]:
        # The codes' borders are met exactly: the rotation in 64 bits, then once to the keys' type.
        cs = state["table"][state["positions"].long()].double()[:, None]
        k = _turn(case, k.double(), cs[..., 0], cs[..., 1]).float().to(k.dtype)
    slots = state["slots"].long()
    kept = slots >= 0
    # A row without a slot writes to a page behind the cache's own.
    at = torch.where(kept, slots, torch.full_like(slots, cache.shape[0] * p))
    grown = torch.cat([cache, torch.zeros_like(cache[:1])])
    page, place = at // p, at % p
    keys, values, kw, vw = _parts(case, grown)
    kc, ks, kz = _quantise(k, group)
    vc, vs, vz = _quantise(v, group)
    keys[page, :, place] = _key_bytes(kc)
    values[page, :, place // 4, :, place % 4] = _value_bytes(vc)
    kw[page, :, :, place] = _words(ks, kz)
    vw[page, :, :, place] = _words(vs, vz)
    cache.copy_(grown[:-1])
    # Read back: the values of the rows' slots, rounded once.
    kq = _nibbles(keys[page, :, place].unflatten(-1, (4, case["head_dim"] // 32, 4)).transpose(-3, -2).flatten(-3))
    vq = _nibbles(values[page, :, place // 4, :, place % 4].flatten(-2))
    ko, vo = _scaled(kq, kw[page, :, :, place], group), _scaled(vq, vw[page, :, :, place], group)
    gone = ~kept[:, None, None]
    return {"k": ko.masked_fill(gone, 0.0).to(k.dtype), "v": vo.masked_fill(gone, 0.0).to(v.dtype)}


def _attend_plain(state: dict):
    case, q, table = state["case"], state["q"], state["pages"]
    b, h, d, most = case["batch"], case["kv_heads"], case["head_dim"], state["most"]
    gqa, dev = case["heads"] // case["kv_heads"], q.device
    starts, ends = state["starts"].long(), state["lengths"].long()
    # Every sequence's keys and values side by side, padded to the longest.
    k, v = _page_values(case, state["cache"][table.clamp(min=0).long()])
    k, v = (a.permute(0, 2, 1, 3, 4).reshape(b, h, -1, d) for a in (k, v))
    key = torch.arange(k.shape[2], device=dev)
    v = v.masked_fill((key[None, :] >= ends[:, None])[:, None, :, None], 0.0)
    # Their rows, padded to the most of any sequence; the padding goes to a row behind the last.
    row = torch.arange(most, device=dev)
    count = starts[1:] - starts[:-1]
    there = row[None, :] < count[:, None]
    at = torch.where(there, starts[:-1, None] + row[None, :], q.shape[0])
    rows = torch.cat([q.float(), torch.zeros((1, *q.shape[1:]), device=dev)])[at]
    rows = rows.unflatten(2, (h, gqa)).permute(0, 2, 1, 3, 4).reshape(b, h, most * gqa, d)
    place = (ends - count)[:, None] + row[None, :]
    seen = key[None, None, :] <= place[:, :, None]
    if case["window"]:
        seen &= key[None, None, :] > place[:, :, None] - case["window"]
    s = torch.matmul(rows, k.transpose(-2, -1)).mul_(1.0 / math.sqrt(d)).view(b, h, most, gqa, -1)
    s.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, h, most * gqa, -1), v).view(b, h, most, gqa, d).div_(total)
    o = o.permute(0, 2, 1, 3, 4).reshape(b, most, h * gqa, d)
    out = torch.zeros((q.shape[0] + 1, *q.shape[1:]), device=dev)
    out[at] = o
    return out[:-1].to(q.dtype)


def run(state: dict):
    """One pass; the outputs of the framework's calls are the program's own buffers."""
    if own:
        return _run_own(state)
    case = state["case"]
    if case["kind"] == "table":
        a = _angles(case, state["first"] + torch.arange(case["count"], device="cuda"))
        return (torch.stack([a.cos(), a.sin()], 2) * case["amplitude"]).float()
    if case["kind"] == "rotate":
        cs = state["table"][state["positions"].long()][:, None]
        sin = -cs[..., 1] if case["inverse"] else cs[..., 1]
        return _turn(case, state["x"].float(), cs[..., 0], sin).to(state["x"].dtype)
    return _append_plain(state) if case["kind"] == "append" else _attend_plain(state)


# ---------------------------------------------------------------------------------------
# What the work is, and its results in 64 bits
# ---------------------------------------------------------------------------------------
def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "table":
        # A sine and a cosine in 64 bits cost about 60 operations.
        return {"bytes": case["count"] * case["rot"] * 4, "flops": 60 * case["count"] * (case["rot"] // 2)}
    if kind == "rotate":
        n = case["tokens"] * case["heads"] * case["head_dim"]
        angles = min(case["tokens"], 32768) * case["rot"] * 4 + case["tokens"] * SIZE[case["index"]]
        return {"bytes": 2 * n * SIZE[case["dtype"]] + angles,
                "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    if kind == "append":
        n = case["tokens"] * case["kv_heads"]
        held = case["head_dim"] + 8 * (case["head_dim"] // case["group"])
        angles = min(case["tokens"], 32768) * case["rot"] * 4 + case["tokens"] * SIZE[case["index"]] * 3
        # Keys and values in, their codes out; the codes in, the values out.
        return {"bytes": n * (2 * held + 8 * case["head_dim"]) + angles, "flops": n * case["head_dim"] * 16}
    rows, ends = _lengths(case)
    w, d = case["window"], case["head_dim"]
    pairs = keys = 0
    for n, e in zip(rows, ends):
        first = e - n  # the place of the sequence's first row: it sees first + 1 keys, or the window's
        if w:
            short = max(0, min(n, w - 1 - first))  # rows that see less than a window
            pairs += short * first + short * (short + 1) // 2 + (n - short) * w
            keys += e - max(0, first - w + 1)
        else:
            pairs += n * first + n * (n + 1) // 2
            keys += e
    held = d + 8 * (d // case["group"])
    return {"bytes": keys * case["kv_heads"] * held + 2 * sum(rows) * case["heads"] * d * SIZE[case["dtype"]],
            "flops": 4 * d * case["heads"] * pairs}


def _exact_rotation(case: dict, x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, inverse: bool):
    y = x.double().clone()
    half = case["rot"] // 2
    cs = table.double()[positions.long()]
    for i in range(half):
        a, b = (i, i + half) if case["layout"] == "halves" else (2 * i, 2 * i + 1)
        c, s = cs[:, i, 0, None], cs[:, i, 1, None]
        s = -s if inverse else s
        x0, x1 = x[..., a].double(), x[..., b].double()
        y[..., a], y[..., b] = c * x0 - s * x1, s * x0 + c * x1
    return y


def _exact_codes(case: dict, y: torch.Tensor) -> torch.Tensor:
    """The values that a row's 4-bit codes stand for, in 64 bits; y in its 16-bit type."""
    out = torch.zeros(y.shape, device=y.device, dtype=torch.float64)
    for g in range(case["head_dim"] // case["group"]):
        part = slice(g * case["group"], (g + 1) * case["group"])
        x = y[..., part].double()
        low = torch.minimum(x.min(-1, keepdim=True).values, torch.zeros((), device=x.device, dtype=x.dtype))
        high = torch.maximum(x.max(-1, keepdim=True).values, torch.zeros((), device=x.device, dtype=x.dtype))
        # The scale is a 16-bit number by definition: the range in 32 bits, a fifteenth of it, then 16.
        s = ((high.float() - low.float()) / 15.0).half().double()
        unit = torch.where(s == 0, torch.ones_like(s), s)
        z = torch.clamp(torch.round(-low / unit), 0, 15)
        out[..., part] = (torch.clamp(torch.round(x / unit) + z, 0, 15) - z) * s
    return out


def exact(case: dict, seed: int):
    """What `run` returns, from the definitions in 64 bits."""
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "table":
        rows = []
        pos = (torch.arange(case["count"], device="cuda", dtype=torch.int64) + state["first"]).double()
        for i in range(case["rot"] // 2):
            f = case["base"] ** (-2.0 * i / case["rot"])
            if case["scaling"] == "linear":
                f /= case["factor"]
            elif case["scaling"] == "ramp":
                wave = 2.0 * math.pi / f
                blend = min(1.0, max(0.0, (case["original"] / wave - case["low"]) / (case["high"] - case["low"])))
                f = (1.0 - blend) * f / case["factor"] + blend * f
            rows.append(torch.stack([torch.cos(pos * f), torch.sin(pos * f)], 1) * case["amplitude"])
        return torch.stack(rows, 1)
    if kind == "rotate":
        return _exact_rotation(case, state["x"], state["table"], state["positions"], case["inverse"])
    if kind == "append":
        k, v = state["k"], state["v"]
        if case["rot"]:
            k = _exact_rotation(case, k, state["table"], state["positions"], False).float().to(k.dtype)
        lost = (state["slots"] < 0)[:, None, None]
        return {"k": _exact_codes(case, k).masked_fill(lost, 0.0), "v": _exact_codes(case, v).masked_fill(lost, 0.0)}
    rows, ends = _lengths(case)
    if sum(n * e for n, e in zip(rows, ends)) * case["heads"] > 1 << 31:
        return None
    q, p, gqa = state["q"], case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    at = 0
    for b, (n, e) in enumerate(zip(rows, ends)):
        used = state["cache"][state["pages"][b, :-(-e // p)].long()]
        for h in range(case["kv_heads"]):
            k, v = _exact_page(case, used[:, h])
            k, v = k[:e], v[:e]
            for g in range(gqa):
                x = q[at:at + n, h * gqa + g].double()
                s = x @ k.T / math.sqrt(case["head_dim"])
                place = torch.arange(e - n, e, device="cuda")[:, None]
                j = torch.arange(e, device="cuda")[None, :]
                seen = j <= place
                if case["window"]:
                    seen = seen & (place - j < case["window"])
                out[at:at + n, h * gqa + g] = torch.softmax(torch.where(seen, s, -math.inf), -1) @ v
        at += n
    return out


def _exact_page(case: dict, records: torch.Tensor):
    """Keys and values [tokens, head_dim] in 64 bits of one head's records [pages, bytes], byte by byte."""
    p, d, group = case["page"], case["head_dim"], case["group"]
    groups, half = d // group, p * d // 2
    t = torch.arange(p, device="cuda")[:, None]
    e = torch.arange(d, device="cuda")[None, :]
    word = e // 8
    low = (e % 8) // 2
    kb = t * (d // 2) + ((word % 4) * (d // 32) + word // 4) * 4 + low
    vb = half + (((t // 4) * (d // 8) + word) * 4 + t % 4) * 4 + low
    shift = (e % 2) * 4
    out = []
    for at, base in ((kb, 2 * half), (vb, 2 * half + 4 * p * groups)):
        code = (records[:, at].int() >> shift) & 15
        w = base + ((e // group) * p + t) * 4
        byte = [records[:, w + i].int() for i in range(4)]
        bits = byte[0] + 256 * byte[1]
        exponent, fraction = (bits >> 10) & 31, (bits & 1023).double()
        scale = torch.where(exponent == 0, fraction * 2.0 ** -24,
                            (1024.0 + fraction) * torch.pow(2.0, exponent.double() - 25.0))
        zero = byte[2] + 256 * byte[3]
        out.append(((code - zero).double() * scale).flatten(0, 1))
    return out

"""The 8-bit key/value cache operators: what is measured, and what they have to give.

Four operators over key/value caches held in 8 bits (signed integers or e4m3 floating point, one
fp32 scale for the 64 values of a head at a position), head dimension 64:

  append   rotate q and k, quantise k and v, and write them at their positions
  read     read a range of positions back into fp32
  attend   causal attention of each request's rows over its own cache (one token, several, a prompt)
  prefix   attention of a batch whose requests share a long prefix, computed once for all

``run`` computes them in plain torch operations where ``own`` is false and through the framework's
entry points where it is true. Sizes follow the framework's configurations: 14 query heads on 2
key/value heads (the language model), 512 cached positions, batches of 64 requests, prompts of 128
and 174 rows, the waveform decoder's four rows over a 65-position window in a ring of 128.
"""
import math

import numpy as np
import torch

own = False

DIM = 64
THETA = 1e6
LIMIT = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TINY = float(np.finfo(np.float32).tiny)


# ------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------
def _case(name, op, kind, requests, rows, lo, hi, capacity, *, hq=14, hkv=2, window=0, prefix=0, short=False):
    """`lo`..`hi`: the requests' first positions, spread evenly; `short`: row counts spread over 1..rows."""
    c = {"op": op, "kind": kind, "hq": hq, "hkv": hkv, "requests": requests, "rows": rows, "lo": lo, "hi": hi,
         "capacity": capacity, "window": window, "prefix": prefix, "short": short}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One request's next token in the engine's 512-position cache: the smallest call, latency only.
        _case("append one token", "append", "int8", 1, 1, 300, 300, 512),
        # The next token of a serving batch whose requests are at different places.
        _case("append batch of 64", "append", "e4m3", 64, 1, 128, 1999, 2048),
        # Padded prompts of a batch: 64 requests, 1 to 128 rows each, from position 0.
        _case("append padded prompts", "append", "int8", 64, 128, 0, 0, 512, short=True),
        # A 174-row prompt read back, as for handing it to an fp32 cache.
        _case("read one prompt", "read", "e4m3", 1, 174, 0, 0, 512),
        # A whole batch's caches read back.
        _case("read batch of 64", "read", "int8", 64, 500, 0, 0, 512, short=True),
        # One request's next token against the engine's cache: latency.
        _case("decode one", "attend", "int8", 1, 1, 300, 300, 512),
        # The next token of the engine's batch, lengths 130 to 500.
        _case("decode batch of 64", "attend", "e4m3", 64, 1, 130, 500, 512),
        # Long contexts of very different lengths.
        _case("decode 8 long", "attend", "int8", 8, 1, 4000, 32767, 32768),
        # The waveform decoder's step: four rows per request over 65 positions in a ring of 128.
        _case("windowed ring", "attend", "int8", 64, 4, 997, 1423, 128, window=65),
        # A long prompt in one call.
        _case("prompt of 4096", "attend", "e4m3", 1, 4096, 0, 0, 4096),
        # Eight requests that continue one 174-row voice prompt.
        _case("prefix 174, batch of 8", "prefix", "e4m3", 8, 1, 0, 320, 338, prefix=174),
        # A serving batch behind one long prompt.
        _case("prefix 8192, batch of 64", "prefix", "int8", 64, 1, 0, 500, 512, prefix=8192),
    ]


def _spread(rng, a, b):
    """A whole number of a..b, even over the logarithm."""
    return min(b, max(a, int(round(math.exp(rng.uniform(math.log(a), math.log(b + 0.999)))))))


def draw(rng):
    while True:
        op = rng.choice(["append", "read", "attend", "attend", "prefix"])
        kind = rng.choice(["int8", "e4m3"])
        hq, hkv = rng.choice([(14, 2), (14, 2), (2, 1), (16, 16), (16, 2), (8, 4)])
        requests = _spread(rng, 1, 64)
        rows = 1 if op in ("attend", "prefix") and rng.random() < 0.5 else _spread(rng, 1, 512 if op == "prefix" else 4096)
        window, prefix, short = 0, 0, rng.random() < 0.3
        hi = _spread(rng, 1, 32768) - 1
        lo = rng.randint(0, hi)
        capacity = hi + rows + rng.choice([0, 0, rng.randint(1, 100)])
        if op == "attend" and rng.random() < 0.25:
            window = _spread(rng, 1, 1024)
            capacity = max(window + rows - 1 + rng.randint(0, 64), 1)
        if op == "prefix":
            prefix = _spread(rng, 1, 16384)
            hi = _spread(rng, 1, 1024) - 1
            lo = rng.randint(0, hi)
            capacity = hi + rows
        c = _case("", op, kind, requests, rows, lo, hi, capacity, hq=hq, hkv=hkv, window=window, prefix=prefix, short=short)
        w = work(c)
        seen = prefix + capacity if op in ("attend", "prefix") else 1
        if w["flops"] <= 3.0e10 and w["bytes"] <= 1.2e8 and requests * hq * rows * seen <= 2.3e8 and \
                requests * hkv * capacity <= 6.0e5:
            return c


def _places(c):
    """First position and row count of each request (relative to the prefix's end)."""
    n = c["requests"]
    first = [c["lo"] + (c["hi"] - c["lo"]) * r // max(1, n - 1) for r in range(n)]
    count = [c["rows"] if not c["short"] else 1 + (c["rows"] - 1) * r // max(1, n - 1) for r in range(n)]
    return first, count


def _keys(c):
    """Per request: the keys that its rows see in its own cache, summed over the rows, and the number of different ones."""
    total, union = [], []
    for p, m in zip(*_places(c)):
        width = min(c["window"] or c["capacity"], c["capacity"])
        total.append(sum(min(p + i + 1, width) for i in range(m)))
        union.append(min(p + m, width + m - 1, c["capacity"]))
    return total, union


def work(c):
    rows = sum(_places(c)[1])
    pair = 2 * c["hkv"] * (DIM + 4)  # a position's codes and scales, keys and values
    if c["op"] == "append":
        return {"bytes": rows * ((2 * c["hq"] + 2 * c["hkv"]) * DIM * 4 + pair),
                "flops": rows * (3 * (c["hq"] + c["hkv"]) + 6 * c["hkv"]) * DIM}
    if c["op"] == "read":
        return {"bytes": rows * (pair + 2 * c["hkv"] * DIM * 4), "flops": rows * 2 * c["hkv"] * DIM}
    total, union = _keys(c)
    keys = sum(total) + rows * c["prefix"]
    return {"bytes": (sum(union) + c["prefix"]) * pair + rows * 2 * c["hq"] * DIM * 4, "flops": keys * c["hq"] * 4 * DIM}


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------
def _random_cache(kind, shape, gen):
    """Codes and scales of a cache whose rows have sizes spread over a factor of some ten."""
    if kind == "int8":
        codes = torch.randint(-127, 128, (*shape, DIM), generator=gen, device="cuda", dtype=torch.int8)
    else:
        codes = (torch.randn(*shape, DIM, generator=gen, device="cuda") * 110).clamp(-448, 448).to(CODE[kind])
    scale = torch.exp(0.5 * torch.randn(*shape, generator=gen, device="cuda")) * (2.0 / LIMIT[kind])
    return codes, scale


def prepare(case, seed):
    c, gen = case, torch.Generator(device="cuda")
    gen.manual_seed(seed)
    n, m, hq, hkv, cap = c["requests"], c["rows"], c["hq"], c["hkv"], c["capacity"]
    first, count = _places(c)
    order = torch.randperm(n, generator=gen, device="cuda")
    s = {"case": c, "kind": c["kind"], "n": n, "rows": m, "hq": hq, "hkv": hkv, "capacity": cap, "window": c["window"],
         "prefix_len": c["prefix"]}
    s["positions"] = (torch.tensor(first, dtype=torch.int32, device="cuda") + c["prefix"])[order].contiguous()
    s["counts"] = torch.tensor(count, dtype=torch.int32, device="cuda")[order].contiguous() if c["short"] else None
    s["inv_freq"] = torch.from_numpy((1.0 / THETA ** (np.arange(0, DIM, 2) / DIM)).astype(np.float32)).cuda()
    s["k"], s["k_scale"] = _random_cache(c["kind"], (n, hkv, cap), gen)
    s["v"], s["v_scale"] = _random_cache(c["kind"], (n, hkv, cap), gen)
    if c["op"] == "append":
        s["qkv"] = torch.randn(n * m, (hq + 2 * hkv) * DIM, generator=gen, device="cuda")
        s["qkv"] *= torch.exp(0.5 * torch.randn(n * m, 1, generator=gen, device="cuda"))
        s["q_out"] = torch.randn(n * m, hq * DIM, generator=gen, device="cuda")
    elif c["op"] == "read":
        s["k_out"] = torch.randn(n, hkv, m, DIM, generator=gen, device="cuda")
        s["v_out"] = torch.randn(n, hkv, m, DIM, generator=gen, device="cuda")
    else:
        s["q"] = torch.randn(n * m, hq * DIM, generator=gen, device="cuda")
        s["out"] = torch.randn(n * m, hq * DIM, generator=gen, device="cuda")
    if c["op"] == "prefix":
        s["pk"], s["pk_scale"] = _random_cache(c["kind"], (1, hkv, c["prefix"]), gen)
        s["pv"], s["pv_scale"] = _random_cache(c["kind"], (1, hkv, c["prefix"]), gen)
    return s


# ------------------------------------------------------------------------------------------------
# The framework's operators
# ------------------------------------------------------------------------------------------------
_framework = {}


def _context():
    """The framework's module and a context on this device, as a program holds them."""
    if not _framework:
        import importlib.util
        import os
        import sys
        name = "mingtts_b200"
        if name not in sys.modules:
            at = os.path.join(os.getcwd(), "ming-tts_b200")
            spec = importlib.util.spec_from_file_location(name, os.path.join(at, "__init__.py"), submodule_search_locations=[at])
            sys.modules[name] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules[name])
        _framework["mt"] = sys.modules[name]
        _framework["ctx"] = sys.modules[name].Context(torch.cuda.current_device())
    return _framework["mt"], _framework["ctx"]


def _run_own(s):
    mt, ctx = _context()
    if "cache" not in s:  # the handles of the caches, made with them
        s["cache"] = mt.KV8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"], base=s["prefix_len"])
        if s["prefix_len"]:
            s["prefix"] = mt.KV8Cache(s["pk"], s["pv"], s["pk_scale"], s["pv_scale"])
    n, m, hq, hkv, op = s["n"], s["rows"], s["hq"], s["hkv"], s["case"]["op"]
    if op == "append":
        ctx.rope_cache_kv8(s["qkv"], (hq + 2 * hkv) * DIM, n, m, hq, s["positions"], s["counts"], s["inv_freq"], s["cache"],
                           s["q_out"], hq * DIM)
    elif op == "read":
        ctx.kv8_read(s["cache"], n, m, s["positions"], s["counts"], s["k_out"], s["v_out"], m)
    elif op == "attend":
        ctx.attention_kv8(s["q"], hq * DIM, n, m, hq, s["positions"], s["counts"], s["window"], s["cache"], s["out"], hq * DIM)
    else:
        ctx.attention_prefix_kv8(s["q"], hq * DIM, n, m, hq, s["positions"], s["counts"], s["prefix"], s["prefix_len"],
                                 s["cache"], s["out"], hq * DIM)


# ------------------------------------------------------------------------------------------------
# The plain form
# ------------------------------------------------------------------------------------------------
def _row_positions(s):
    """Position of each row [n, rows], and whether the row is one of the request's (not padding)."""
    i = torch.arange(s["rows"], device="cuda")
    pos = s["positions"].long()[:, None] + i
    live = torch.ones_like(pos, dtype=torch.bool) if s["counts"] is None else i < s["counts"].long()[:, None]
    return pos, live


def _e4m3(x):
    """`x` (64 bits) rounded to the nearest e4m3 value, ties to even: steps of 2^(e-3), e >= -6."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _quantise(x, kind):
    """Codes and fp32 scales of rows of 64 fp32 values; a row whose scale is below fp32's normal range is zero."""
    scale = (x.abs().amax(-1).double() / LIMIT[kind]).float()
    scale = torch.where(scale < TINY, 0.0, scale)
    y = x.double() / torch.where(scale == 0, 1.0, scale).double()[..., None]
    y = torch.where((scale == 0)[..., None], 0.0, y)
    y = torch.round(y).clamp(-127, 127) if kind == "int8" else _e4m3(y)
    return y.float().to(CODE[kind]), scale


def _turn(x, pos):
    """NeoX rotation (pairs i, i + 32) of [n, rows, heads, 64] in 64 bits, rounded to 32."""
    inv = torch.from_numpy((1.0 / THETA ** (np.arange(0, DIM, 2) / DIM)).astype(np.float32)).cuda()
    a = pos.double()[..., None, None] * inv.double()
    x0, x1 = x[..., :32].double(), x[..., 32:].double()
    return torch.cat([x0 * a.cos() - x1 * a.sin(), x1 * a.cos() + x0 * a.sin()], -1).float()


def _append(s):
    n, m, hq, hkv = s["n"], s["rows"], s["hq"], s["hkv"]
    pos, live = _row_positions(s)
    x = s["qkv"].view(n, m, hq + 2 * hkv, DIM)
    turned = _turn(x[:, :, :hq + hkv], pos)
    q = s["q_out"].view(n, m, hq, DIM)
    q.copy_(torch.where(live[..., None, None], turned[:, :, :hq], q))
    request, row = live.nonzero(as_tuple=True)
    slot = (pos[request, row] - s["prefix_len"]) % s["capacity"]
    for name, new in (("k", turned[:, :, hq:]), ("v", x[:, :, hq + hkv:])):
        codes, scale = _quantise(new[request, row], s["kind"])
        s[name].view(torch.int8)[request, :, slot] = codes.view(torch.int8)
        s[name + "_scale"][request, :, slot] = scale


def _read(s):
    pos, live = _row_positions(s)
    slot = (pos % s["capacity"])[:, None, :].expand(-1, s["hkv"], -1)
    for name in ("k", "v"):
        values = s[name].float() * s[name + "_scale"][..., None]
        got = values.gather(2, slot[..., None].expand(-1, -1, -1, DIM))
        s[name + "_out"].copy_(torch.where(live[:, None, :, None], got, s[name + "_out"]))


def _attend(s):
    n, m, hq, hkv, cap, start = s["n"], s["rows"], s["hq"], s["hkv"], s["capacity"], s["prefix_len"]
    pos, live = _row_positions(s)
    last = s["positions"].long() + (m if s["counts"] is None else s["counts"].long()) - 1
    held = last[:, None] - (last[:, None] - start - torch.arange(cap, device="cuda")) % cap  # position in each slot
    sees = (held[:, None] <= pos[..., None]) & (held[:, None] >= start)
    if s["window"]:
        sees &= held[:, None] > pos[..., None] - s["window"]
    k = s["k"].float() * s["k_scale"][..., None]
    v = s["v"].float() * s["v_scale"][..., None]
    q = s["q"].view(n, m, hkv, hq // hkv, DIM).permute(0, 2, 3, 1, 4)  # [n, hkv, g, m, 64]
    score = torch.matmul(q.reshape(n, hkv, -1, DIM), k.transpose(2, 3)).view(n, hkv, -1, m, cap) * 0.125
    score = score.masked_fill(~sees[:, None, None], -math.inf)
    if start:
        pk = s["pk"].float() * s["pk_scale"][..., None]
        pv = s["pv"].float() * s["pv_scale"][..., None]
        ahead = torch.matmul(q.reshape(n, hkv, -1, DIM), pk.transpose(2, 3)).view(n, hkv, -1, m, start) * 0.125
        score = torch.cat([ahead, score], -1)
    score = score - score.amax(-1, keepdim=True)
    weight = torch.exp(score)
    weight = weight / weight.sum(-1, keepdim=True)
    weight = weight.view(n, hkv, -1, start + cap)
    out = torch.matmul(weight[..., start:], v)
    if start:
        out = out + torch.matmul(weight[..., :start], pv)
    out = out.view(n, hkv, hq // hkv, m, DIM).permute(0, 3, 1, 2, 4).reshape(n, m, hq * DIM)
    keep = s["out"].view(n, m, hq * DIM)
    keep.copy_(torch.where(live[..., None], out, keep))


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        _run_own(s)
    else:
        {"append": _append, "read": _read, "attend": _attend, "prefix": _attend}[op](s)
    if op == "append":
        return {"q": s["q_out"], "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if op == "read":
        return {"k": s["k_out"], "v": s["v_out"]}
    return {"out": s["out"]}


# ------------------------------------------------------------------------------------------------
# From the definitions, in 64 bits, one request at a time
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    positions = s["positions"].tolist()
    counts = s["counts"].tolist() if s["counts"] is not None else [s["rows"]] * s["n"]
    f = {"append": _exact_append, "read": _exact_read}.get(case["op"], _exact_attend)
    return f(s, positions, counts)


def _values(s, name, r):
    return s[name][r].float().double() * s[name + "_scale"][r].double()[..., None]


def _exact_append(s, positions, counts):
    m, hq, hkv, cap = s["rows"], s["hq"], s["hkv"], s["capacity"]
    inv = s["inv_freq"].double()
    q = s["q_out"].double()
    out = {"k": s["k"].float().double(), "v": s["v"].float().double(), "k_scale": s["k_scale"].double(),
           "v_scale": s["v_scale"].double()}
    grid = None
    if s["kind"] == "e4m3":  # every finite e4m3 value, and the borders between neighbours
        grid = torch.arange(256, dtype=torch.uint8, device="cuda").view(CODE["e4m3"]).float().double()
        grid = torch.unique(grid[~grid.isnan()])
    for r, (p, c) in enumerate(zip(positions, counts)):
        at = torch.arange(p, p + c, device="cuda")
        rows = s["qkv"][r * m:r * m + c].double().view(c, hq + 2 * hkv, DIM)
        z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), at.double()[:, None] * inv)[:, None]
        turned = torch.complex(rows[:, :hq + hkv, :32], rows[:, :hq + hkv, 32:]) * z
        turned = torch.cat([turned.real, turned.imag], -1)
        q[r * m:r * m + c] = turned[:, :hq].reshape(c, -1)
        for name, x in (("k", turned[:, hq:].float().double()), ("v", rows[:, hq + hkv:])):
            scale = (x.abs().amax(-1) / LIMIT[s["kind"]]).float().double()
            y = (x / scale[..., None]).clamp(-LIMIT[s["kind"]], LIMIT[s["kind"]])
            if grid is None:
                y = torch.round(y)
            else:
                above = torch.searchsorted(grid, y).clamp(1, len(grid) - 1)
                low, high = grid[above - 1], grid[above]
                even = above % 2 == 1  # neighbours alternate even and odd codes; zero, in the middle, is even
                if (len(grid) // 2) % 2 == 1:
                    even = ~even
                y = torch.where((y - low < high - y) | ((y - low == high - y) & even), low, high)
            out[name][r][:, at % cap] = y.transpose(0, 1)
            out[name + "_scale"][r][:, at % cap] = scale.transpose(0, 1)
    if s["kind"] == "int8":
        out = {n: x if n.endswith("scale") else None for n, x in out.items()}
    return {"q": q, **out}


def _exact_read(s, positions, counts):
    out = {"k": s["k_out"].double(), "v": s["v_out"].double()}
    for r, (p, c) in enumerate(zip(positions, counts)):
        for name in ("k", "v"):
            at = torch.arange(p, p + c, device="cuda") % s["capacity"]
            out[name][r, :, :c] = _values(s, name, r)[:, at]
    return out


def _exact_attend(s, positions, counts):
    m, hq, hkv, cap, start = s["rows"], s["hq"], s["hkv"], s["capacity"], s["prefix_len"]
    out = s["out"].double().view(s["n"], m, hkv, hq // hkv, DIM)
    for r, (p, c) in enumerate(zip(positions, counts)):
        first = max(start, p + c - cap, p - s["window"] + 1 if s["window"] else 0)
        at = torch.arange(first, p + c, device="cuda")
        k, v = (_values(s, name, r)[:, (at - start) % cap] for name in ("k", "v"))
        if start:
            k, v = (torch.cat([_values(s, "p" + name, 0), x], 1) for name, x in (("k", k), ("v", v)))
            at = torch.cat([torch.arange(start, device="cuda"), at])
        rows = torch.arange(p, p + c, device="cuda")
        sees = at <= rows[:, None]
        if s["window"]:
            sees &= at > rows[:, None] - s["window"]
        q = s["q"].view(s["n"], m, hkv, hq // hkv, DIM)[r, :c].double()
        for h in range(hkv):
            for g in range(hq // hkv):
                weight = torch.softmax((q[:, h, g] @ k[h].T / 8).masked_fill(~sees, -math.inf), -1)
                out[r, :c, h, g] = weight @ v[h]
    return {"out": out.reshape(s["n"] * m, hq * DIM)}

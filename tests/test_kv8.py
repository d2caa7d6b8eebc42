"""The 8-bit key/value cache: written (mt_rope_cache_kv8), read back (mt_kv8_read), attended to
(mt_attention_kv8) and behind a shared prefix (mt_attention_prefix_kv8), through the C ABI.

The plain implementation here is in 64 bits, one request at a time. Bounds, from the arithmetic:

* Codes and scales are equal: the rotated key is computed in 64 bits and rounded once to fp32, the
  scale is one rounded division, the code the nearest to the exact quotient.
* Rotated queries: the cosine and sine are rounded to fp32 (2^-24 each), two products and a sum
  (3 x 2^-24): |error| <= 4 x 2^-24 (|x0| + |x1|).
* Attention: a score is a sum of 64 exact codes times q in two fp16 planes (2^-22 relative) added in
  fp32 (128 terms, 2^-24 each) and scaled (4 roundings): |error| <= d = (4 + 128 + 4) 2^-24 A, A the
  row's largest sum_d |q_d k_d| / 8. A weight exp(s - m) is then off by 2 d and the exponential's own
  2^-21 (its argument is rounded: |s - m| 2^-24, below 2 A 2^-24, inside 2 d). A weight times the value's scale enters in two
  fp16 planes (2^-21), and the sums over n keys are fp32 in steps of 16 keys, then joined:
  (n / 8 + 64) 2^-24. Numerator and denominator both: |error| <= 2 (2 d + 2^-20 + (n / 8 + 64) 2^-24) V,
  V the largest |v| that the row sees.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

gpu = pytest.mark.gpu
LIMIT = {"int8": 127.0, "e4m3": 448.0}
KINDS = ["int8", "e4m3"]
INV_FREQ = (1.0 / 1e6 ** (np.arange(0, 64, 2) / 64)).astype(np.float32)


# ------------------------------------------------------------------------------------------------
# Refusals: host checks, no GPU (a null context is the last thing refused)
# ------------------------------------------------------------------------------------------------
def cache_struct(mt, kind=0, heads=2, capacity=64, base=0, stride=None, at=1 << 20, scale_at=1 << 20):
    return mt.KV8CacheStruct(kind, heads, capacity, base, heads * capacity if stride is None else stride, at, at, scale_at,
                             scale_at)


A = 1 << 20  # an aligned address that no refused call reads


def test_append_refusals(mt):
    def call(c=None, ldq=18 * 64, requests=1, rows=1, hq=14, ldqo=14 * 64, q_out=A, qkv=2 * A, positions=A, inv=A, **k):
        c = c if c is not None else cache_struct(mt, **k)
        return mt.lib().mt_rope_cache_kv8(None, None, qkv, ldq, requests, rows, hq, positions, None, inv, ctypes.byref(c), q_out,
                                          ldqo)

    assert call() == mt.MT_ERR_ARG  # only the context is missing
    assert mt.lib().mt_rope_cache_kv8(None, None, A, 1152, 1, 1, 14, A, None, A, None, A, 896) == mt.MT_ERR_ARG
    for bad in (dict(qkv=None), dict(positions=None), dict(inv=None), dict(q_out=None), dict(kind=2), dict(kind=-1),
                dict(at=A + 8), dict(scale_at=A + 2), dict(at=None), dict(scale_at=None)):
        assert call(**bad) == mt.MT_ERR_ARG, bad
    for bad in (dict(ldq=18 * 64 - 1), dict(ldqo=14 * 64 - 1), dict(hq=13), dict(hq=0), dict(requests=-1), dict(rows=-1),
                dict(heads=0), dict(capacity=0), dict(base=-1), dict(stride=127), dict(requests=2, stride=1 << 60),
                dict(q_out=2 * A, ldqo=14 * 64)):
        assert call(**bad) == mt.MT_ERR_SHAPE, bad
    assert call(rows=65) == mt.MT_ERR_CAPACITY


def test_read_refusals(mt):
    def call(requests=1, rows=1, positions=A, k=A, v=A, out_capacity=64, **kw):
        return mt.lib().mt_kv8_read(None, None, ctypes.byref(cache_struct(mt, **kw)), requests, rows, positions, None, k, v,
                                    out_capacity)

    assert call() == mt.MT_ERR_ARG
    assert call(rows=65, out_capacity=100) == mt.MT_ERR_CAPACITY
    assert call(rows=64, out_capacity=63) == mt.MT_ERR_CAPACITY
    assert call(requests=-1) == mt.MT_ERR_SHAPE
    for bad in (dict(k=None, v=None), dict(k=A + 4), dict(positions=None)):
        assert call(**bad) == mt.MT_ERR_ARG, bad


def test_attention_refusals(mt):
    def call(requests=1, rows=1, hq=14, ldq=896, ldo=896, window=0, q=A, out=A, positions=A, **kw):
        return mt.lib().mt_attention_kv8(None, None, q, ldq, requests, rows, hq, positions, None, window,
                                         ctypes.byref(cache_struct(mt, **kw)), out, ldo, None, 0)

    assert call() == mt.MT_ERR_ARG
    for bad in (dict(hq=15), dict(ldq=895), dict(ldo=895), dict(window=-1), dict(rows=-2), dict(stride=1)):
        assert call(**bad) == mt.MT_ERR_SHAPE, bad
    for bad in (dict(rows=65), dict(rows=2, window=64)):
        assert call(**bad) == mt.MT_ERR_CAPACITY, bad
    for bad in (dict(q=None), dict(out=None), dict(positions=None), dict(kind=7)):
        assert call(**bad) == mt.MT_ERR_ARG, bad


def test_prefix_refusals(mt):
    def call(prefix_len=16, base=16, prefix_base=0, prefix_capacity=16, prefix_heads=2, null=False, **kw):
        own, prefix = cache_struct(mt, base=base), cache_struct(mt, base=prefix_base, capacity=prefix_capacity, heads=prefix_heads)
        return mt.lib().mt_attention_prefix_kv8(None, None, A, 896, 1, 1, 14, A, None, None if null else ctypes.byref(prefix),
                                                prefix_len, ctypes.byref(own), A, 896, None, 0)

    assert call() == mt.MT_ERR_ARG
    assert call(null=True) == mt.MT_ERR_ARG
    assert call(prefix_len=0, base=0, null=True) == mt.MT_ERR_ARG  # no prefix: allowed, but for the context
    assert call(prefix_len=-1) == mt.MT_ERR_SHAPE
    assert call(base=15) == mt.MT_ERR_SHAPE
    assert call(prefix_heads=1) == mt.MT_ERR_SHAPE
    assert call(prefix_capacity=15) == mt.MT_ERR_CAPACITY
    assert call(prefix_base=1) == mt.MT_ERR_CAPACITY


def test_cache_object_refuses_other_layouts(mt):
    import torch
    k, s = torch.zeros(2, 2, 8, 64, dtype=torch.int8), torch.zeros(2, 2, 8)
    with pytest.raises(TypeError):
        mt.KV8Cache(k.float(), k.float(), s, s)
    with pytest.raises(TypeError):
        mt.KV8Cache(k, k, s.double(), s)
    with pytest.raises(ValueError):
        mt.KV8Cache(k[..., :32], k[..., :32], s, s)
    with pytest.raises(ValueError):  # not on a CUDA device
        mt.KV8Cache(k, k, s, s)


def test_calls_refuse_caches_of_fewer_requests_or_another_device(mt):
    from types import SimpleNamespace
    ctx = object.__new__(mt.Context)
    ctx.device = 0
    good = SimpleNamespace(requests=2, index=0, device="cuda:0")
    for bad, status in ((SimpleNamespace(requests=1, index=0, device="cuda:0"), mt.MT_ERR_SHAPE),
                        (SimpleNamespace(requests=2, index=1, device="cuda:1"), mt.MT_ERR_ARG)):
        for call in (lambda: ctx.rope_cache_kv8(None, 1152, 2, 1, 14, None, None, None, bad, None, 896),
                     lambda: ctx.kv8_read(bad, 2, 1, None, None, None, None, 1),
                     lambda: ctx.attention_kv8(None, 896, 2, 1, 14, None, None, 0, bad, None, 896),
                     lambda: ctx.attention_prefix_kv8(None, 896, 2, 1, 14, None, None, good, 3, bad, None, 896)):
            with pytest.raises(mt.MingError) as e:
                call()
            assert e.value.status == status
    with pytest.raises(mt.MingError):
        ctx.attention_prefix_kv8(None, 896, 2, 1, 14, None, None, SimpleNamespace(requests=1, index=1, device="cuda:1"), 3, good,
                                 None, 896)


def test_calls_refuse_positions_of_another_type(mt):
    import torch
    from types import SimpleNamespace
    ctx = object.__new__(mt.Context)
    ctx.device = 0
    cache = SimpleNamespace(requests=2, index=0, device="cuda:0")
    good = torch.zeros(2, dtype=torch.int32)
    for pos, counts in ((good.long(), None), (good[:1], None), (torch.zeros(4, dtype=torch.int32)[::2], None), (good, good.long()),
                        (good, good[:1])):
        for call in (lambda: ctx.rope_cache_kv8(None, 1152, 2, 1, 14, pos, counts, None, cache, None, 896),
                     lambda: ctx.kv8_read(cache, 2, 1, pos, counts, None, None, 1),
                     lambda: ctx.attention_kv8(None, 896, 2, 1, 14, pos, counts, 0, cache, None, 896),
                     lambda: ctx.attention_prefix_kv8(None, 896, 2, 1, 14, pos, counts, cache, 3, cache, None, 896)):
            with pytest.raises(TypeError):
                call()


# ------------------------------------------------------------------------------------------------
# The plain implementation, 64 bits
# ------------------------------------------------------------------------------------------------
def torch_kind(kind):
    import torch
    return torch.int8 if kind == "int8" else torch.float8_e4m3fn


def e4m3_grid():
    import torch
    g = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    return torch.unique(g[~g.isnan()])  # zero at an even index, neighbours alternate


def quantise(x, kind):
    """(codes as float64, scale fp32 as float64) of fp32 rows [..., 64] given in float64."""
    import torch
    top = x.abs().amax(-1)
    scale = torch.from_numpy((top.numpy().astype(np.float32) / np.float32(LIMIT[kind])).astype(np.float32)).double()
    scale = torch.where(scale < 2.0 ** -126, 0.0, scale)
    y = torch.where(scale[..., None] > 0, x / torch.where(scale > 0, scale, 1.0)[..., None], 0.0)
    if kind == "int8":
        codes = torch.round(y).clamp(-127, 127)
    else:
        grid = e4m3_grid()
        y = y.clamp(-448, 448)
        above = torch.searchsorted(grid, y).clamp(1, len(grid) - 1)
        low, high = grid[above - 1], grid[above]
        codes = torch.where((y - low < high - y) | ((y - low == high - y) & (above % 2 == 1)), low, high)
    bad = ~torch.isfinite(x).all(-1)
    codes = torch.where(bad[..., None], 0.0, codes)
    return codes, torch.where(bad, math.nan, scale)


def rotate(x, pos):
    """x [rows, heads, 64] float64 at positions pos [rows]."""
    import torch
    a = (pos.double()[:, None] * torch.from_numpy(INV_FREQ).double())[:, None]
    x0, x1 = x[..., :32], x[..., 32:]
    return torch.cat([x0 * a.cos() - x1 * a.sin(), x1 * a.cos() + x0 * a.sin()], -1)


def attend_reference(q, keys, values, sees):
    """q [rows, hq, 64], keys / values [hkv, n, 64], sees [rows, n]: (out, bound) per row and head."""
    import torch
    rows, hq, _ = q.shape
    hkv, n, _ = keys.shape
    g = hq // hkv
    out, bound = torch.zeros_like(q), torch.zeros(rows, hq, dtype=torch.float64)
    for h in range(hkv):
        for u in range(g):
            x = q[:, h * g + u]
            k = torch.where(torch.isnan(keys[h]), 0.0, keys[h])
            s = (x @ k.T / 8).masked_fill(~sees, -math.inf)
            a = (x.abs() @ k.abs().T / 8).masked_fill(~sees, 0.0).amax(-1)
            w = torch.softmax(s, -1)
            v = torch.where(torch.isnan(values[h]), 0.0, values[h])
            out[:, h * g + u] = w @ v
            top = torch.where(sees, v.abs().amax(-1)[None], 0.0).amax(-1)
            d = 136 * 2.0 ** -24 * a
            bound[:, h * g + u] = 2 * (2 * d + 2.0 ** -20 + (n / 8 + 64) * 2.0 ** -24) * top
    return out, bound


def live_rows(positions, rows, counts, base):
    """Rows of each request that are its own: none below the base or where positions reach 2^31 - 1."""
    counts = [rows] * len(positions) if counts is None else counts
    return [0 if p < base or p + rows > 2 ** 31 - 1 else min(max(c, 0), rows) for p, c in zip(positions, counts)]


class Cache:
    """A device cache with every slot poisoned, the positions of each request filled, and its values on the host."""

    def __init__(self, mt, kind, heads, capacity, spans, seed, base=0, layers=1, layer=0, spread=0.5):
        """spans: per request (first held position, one past the last)."""
        import torch
        g = torch.Generator().manual_seed(seed)
        n = len(spans)
        self.kind, self.base, self.capacity = kind, base, capacity
        codes, scales = [], []
        self.values = []
        for name in range(2):
            if kind == "int8":
                c = torch.full((n, heads, capacity, 64), -128, dtype=torch.int8)
            else:
                c = torch.full((n, heads, capacity, 64), 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn)
            s = torch.full((n, heads, capacity), math.nan)
            vals = []
            for r, (a, b) in enumerate(spans):
                m = max(0, b - a)
                if kind == "int8":
                    new = torch.randint(-127, 128, (heads, m, 64), generator=g, dtype=torch.int8)
                else:
                    new = (torch.randn(heads, m, 64, generator=g) * 110).clamp(-448, 448).to(torch.float8_e4m3fn)
                sc = torch.exp(spread * torch.randn(heads, m, generator=g)) * (2.0 / LIMIT[kind])
                at = (torch.arange(a, b) - base) % capacity
                c.view(torch.uint8)[r][:, at] = new.view(torch.uint8)
                s[r][:, at] = sc
                vals.append(new.double() * sc.double()[..., None])
            codes.append(c)
            scales.append(s)
            self.values.append(vals)
        self.spans = spans
        dev = [t.cuda() for t in (*codes, *scales)]
        if layers > 1:  # a slab of several layers, requests outermost
            wide = []
            for t in dev:
                big = torch.empty(n, layers, *t.shape[1:], dtype=t.dtype, device="cuda")
                big[:, layer] = t
                wide.append(big[:, layer])
            dev = wide
        self.kv = mt.KV8Cache(*dev, base=base)


def check_attention(ctx, mt, kind, hq, hkv, capacity, positions, rows, counts=None, window=0, base=0, prefix_len=0, pad_q=0,
                    pad_o=0, layers=1, seed=0, spread=0.5, q_scale=1.0, prefix_kind=None, run=None):
    """One call against the plain implementation; returns the output tensor."""
    import torch
    n = len(positions)
    base = prefix_len if prefix_len else base
    live = live_rows(positions, rows, counts, base)
    spans = [(max(base, p + c - capacity), p + c) if c else (0, 0) for p, c in zip(positions, live)]
    cache = Cache(mt, kind, hkv, capacity, spans, seed, base=base, layers=layers, layer=layers // 2, spread=spread)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(n * rows, hq * 64, generator=g) * q_scale
    for r in range(n):
        q[r * rows + live[r]:(r + 1) * rows] = math.nan  # padding rows are never read
    ldq, ldo = hq * 64 + pad_q, hq * 64 + pad_o
    qd = torch.full((n * rows, ldq), math.nan, device="cuda")
    qd[:, :hq * 64] = q.cuda()
    out = torch.full((n * rows, ldo), 7.0, device="cuda")
    pos = torch.tensor(positions, dtype=torch.int32, device="cuda")
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    if prefix_len:
        prefix = Cache(mt, prefix_kind or kind, hkv, prefix_len + 3, [(0, prefix_len)], seed + 2, spread=spread)

        def call():
            ctx.attention_prefix_kv8(qd, ldq, n, rows, hq, pos, cnt, prefix.kv, prefix_len, cache.kv, out, ldo)
    else:
        def call():
            ctx.attention_kv8(qd, ldq, n, rows, hq, pos, cnt, window, cache.kv, out, ldo)
    (run or (lambda f: f()))(call)
    ctx.check()
    got = out.cpu()
    for r in range(n):
        m, p = live[r], positions[r]
        block = got[r * rows:(r + 1) * rows]
        assert torch.equal(block[m:], torch.full_like(block[m:], 7.0)), f"padding of request {r} was written"
        assert torch.equal(block[:m, hq * 64:], torch.full_like(block[:m, hq * 64:], 7.0)), "columns past hq * 64"
        if m == 0:
            continue
        a, b = spans[r]
        at, mine = torch.arange(a, b), torch.arange(p, p + m)
        sees = at <= mine[:, None]
        if window:
            sees &= at > mine[:, None] - window
        k, v = cache.values[0][r], cache.values[1][r]
        if prefix_len:
            k, v = torch.cat([prefix.values[0][0], k], 1), torch.cat([prefix.values[1][0], v], 1)
            sees = torch.cat([torch.ones(m, prefix_len, dtype=torch.bool), sees], 1)
        want, bound = attend_reference(q[r * rows:r * rows + m].double().view(m, hq, 64), k, v, sees)
        err = (block[:m, :hq * 64].double().view(m, hq, 64) - want).abs().amax(-1)
        assert torch.all(err <= bound), (f"request {r}: worst error {float((err / bound).max()):.3g} of the bound at "
                                         f"{np.unravel_index(int((err / bound).argmax()), err.shape)}")
    return out


# ------------------------------------------------------------------------------------------------
# Writing
# ------------------------------------------------------------------------------------------------
def check_append(ctx, mt, kind, hq, hkv, capacity, positions, rows, counts=None, base=0, pad=0, pad_out=0, offset=0,
                 in_place=False, edit=None, seed=0):
    import torch
    n, width = len(positions), (hq + 2 * hkv) * 64
    live = live_rows(positions, rows, counts, base)
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n * rows, width, generator=g)
    x *= torch.exp(2 * torch.randn(n * rows, 1, generator=g))
    if edit:
        edit(x)
    cache = Cache(mt, kind, hkv, capacity, [(0, 0)] * n, seed, base=base)
    before = [t.clone() for t in cache.kv.tensors]
    ldq = width + pad
    store = torch.full((n * rows * ldq + offset,), 5.0, device="cuda")[offset:]  # offset: rows off 16-byte alignment
    qkv = store.view(n * rows, ldq)
    qkv[:, :width] = x.cuda()
    kept = qkv.clone()
    ldo = ldq if in_place else hq * 64 + pad_out
    q_out = qkv if in_place else torch.full((n * rows, ldo), 7.0, device="cuda")
    pos = torch.tensor(positions, dtype=torch.int32, device="cuda")
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    ctx.rope_cache_kv8(qkv, ldq, n, rows, hq, pos, cnt, torch.from_numpy(INV_FREQ).cuda(), cache.kv, q_out, ldo)
    ctx.check()
    if not in_place:
        assert torch.equal(qkv.view(torch.int32), kept.view(torch.int32)), "qkv was modified"
    got_q = q_out.cpu()
    want = [t.cpu().clone() for t in before]
    for r in range(n):
        m = live[r]
        at = torch.arange(positions[r], positions[r] + m)
        rows_x = x[r * rows:r * rows + m].double().view(m, hq + 2 * hkv, 64)
        turned = rotate(rows_x[:, :hq + hkv], at)
        new = got_q[r * rows:(r + 1) * rows]
        err = (new[:m, :hq * 64].double().view(m, hq, 64) - turned[:, :hq]).abs()
        size = rows_x[:, :hq].abs()
        tol = 4 * 2.0 ** -24 * (size[..., :32] + size[..., 32:]).repeat(1, 1, 2)
        fine = torch.isfinite(turned[:, :hq])
        assert torch.all((err <= tol) | ~fine), f"request {r}: rotated queries"
        rest = kept.cpu() if in_place else torch.full_like(got_q, 7.0)
        rest = rest[r * rows:(r + 1) * rows]
        assert torch.equal(new[m:], rest[m:]), "padding rows"
        assert torch.equal(new[:m, hq * 64:].view(torch.int32), rest[:m, hq * 64:].contiguous().view(torch.int32)), "other columns"
        slot = (at - base) % capacity
        for which, y in ((0, turned[:, hq:].float().double()), (1, rows_x[:, hq + hkv:])):
            codes, scale = quantise(y, kind)  # [m, hkv, 64], [m, hkv]
            want[which].view(torch.uint8)[r][:, slot] = codes.to(torch_kind(kind)).view(torch.uint8).transpose(0, 1)
            want[2 + which][r][:, slot] = scale.float().transpose(0, 1)
    for name, w, t in zip(("k", "v", "k_scale", "v_scale"), want, cache.kv.tensors):
        t = t.cpu()
        if w.dtype == torch.float32:
            assert torch.equal(torch.nan_to_num(t, nan=-1.0), torch.nan_to_num(w, nan=-1.0)), name
        else:  # codes as the values they stand for (-0 equals 0), poisoned ones by their bits
            same = (t.view(torch.uint8) == w.view(torch.uint8)) | (t.float() == w.float())
            assert torch.all(same), f"{name}: {int((~same).sum())} codes differ"
    return cache


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,capacity,positions,rows,counts,base", [
    (14, 2, 512, [300], 1, None, 0),
    (14, 2, 64, [0, 5, 63, 64, 200], 1, None, 0),            # the last two wrap
    (2, 1, 37, [0, 30, 100], 9, [9, 4, 0], 0),               # odd capacity, padding, an empty request
    (16, 16, 40, [7, -1, 3], 3, None, 3),                    # base, an idle request, one at the base
    (14, 2, 200000, [199990], 7, None, 0),                   # far positions: 64-bit angles
    (8, 4, 130, [0] * 33, 70, [1 + 2 * i for i in range(33)], 0),  # several rows a block
    (7, 7, 1, [0, 12], 1, None, 0),                          # one slot
    (6, 2, 16, [2 ** 31 - 9, 2 ** 31 - 8, 5], 8, None, 0),   # the last positions, and one too many: idle
])
def test_append(ctx, mt, kind, hq, hkv, capacity, positions, rows, counts, base):
    check_append(ctx, mt, kind, hq, hkv, capacity, positions, rows, counts, base)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pad,pad_out,offset,in_place", [(0, 0, 0, True), (12, 4, 0, False), (3, 1, 0, False), (0, 0, 1, False),
                                                          (5, 0, 3, True)])
def test_append_strides(ctx, mt, kind, pad, pad_out, offset, in_place):
    check_append(ctx, mt, kind, 14, 2, 50, [11, 0], 5, [5, 3], pad=pad, pad_out=pad_out, offset=offset, in_place=in_place)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_append_special_values(ctx, mt, kind):
    """Zeros, tiny rows, infinities, NaN, and values exactly between two codes."""
    import torch

    def edit(x):
        v = x.view(12, 4, 64)[:, 3]  # the value head of hq 2, hkv 1
        v[0] = 0.0
        v[1] = 0.0
        v[1, 5] = 1e-40
        v[2, 9] = math.inf
        v[3, 60] = math.nan
        v[4, 1] = -math.inf
        v[5] = torch.arange(64) - 31.5   # halves
        v[5, 0] = LIMIT[kind]
        v[6] = 2.0 ** -100 * v[6]
        v[7] = 2.0 ** 100 * v[7]
        v[8] = 0.0
        v[8, 63] = -3.4e38
        v[9] = LIMIT[kind] / 64 * torch.arange(64)
        v[10] = 2.0 ** (-torch.arange(64).float())
        v[11] = 1.17549435e-38 * LIMIT[kind]

    check_append(ctx, mt, kind, 2, 1, 12, [0], 12, edit=edit)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hkv,capacity,positions,rows,counts,out_capacity", [
    (2, 512, [100], 1, None, 1), (2, 512, [0, 3, 300], 174, [174, 1, 0], 200), (1, 37, [0, 35, 100], 37, None, 37),
    (3, 90, [-1, 4], 65, [65, 64], 65),
])
def test_read(ctx, mt, kind, hkv, capacity, positions, rows, counts, out_capacity):
    import torch
    n = len(positions)
    live = [0 if p < 0 else c for p, c in zip(positions, counts or [rows] * n)]
    cache = Cache(mt, kind, hkv, capacity, [(p, p + c) if c else (0, 0) for p, c in zip(positions, live)], 3)
    pos = torch.tensor(positions, dtype=torch.int32, device="cuda")
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    want = [torch.full((n, hkv, out_capacity, 64), 7.0) for _ in range(2)]
    for r in range(n):
        for t in range(2):
            want[t][r, :, :live[r]] = cache.values[t][r].float()  # one rounded product
    for which in ((True, True), (True, False), (False, True)):
        out = [torch.full((n, hkv, out_capacity, 64), 7.0, device="cuda") for _ in range(2)]
        ctx.kv8_read(cache.kv, n, rows, pos, cnt, out[0] if which[0] else None, out[1] if which[1] else None, out_capacity)
        ctx.check()
        for t in range(2):
            assert torch.equal(out[t].cpu(), want[t] if which[t] else torch.full_like(want[t], 7.0))


# ------------------------------------------------------------------------------------------------
# Attention
# ------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv", [(14, 2), (1, 1), (16, 2), (5, 5), (18, 2), (40, 1)])
def test_decode_lengths(ctx, mt, kind, hq, hkv):
    """One row a request: lengths around the sizes of every tile, in one batch and alone."""
    lengths = [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 300]
    check_attention(ctx, mt, kind, hq, hkv, 304, [n - 1 for n in lengths], 1)
    for n in (1, 16, 97, 301):
        check_attention(ctx, mt, kind, hq, hkv, 304, [n - 1], 1, seed=n)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("capacity,positions", [(5000, [4999]), (5001, [4999, 17]), (9000, [8999, 0, 4100]),
                                                (70000, [69990])])
def test_decode_long(ctx, mt, kind, capacity, positions):
    check_attention(ctx, mt, kind, 14, 2, capacity, positions, 1)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [2, 3, 4, 5, 8, 9, 16, 17, 33, 64, 65, 130])
def test_several_rows(ctx, mt, kind, rows):
    """Rows whose causal limits end inside tiles, behind cached positions and from the start."""
    check_attention(ctx, mt, kind, 14, 2, 333, [0, 200, 57], rows)
    check_attention(ctx, mt, kind, 4, 4, rows, [0], rows)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_prompt(ctx, mt, kind):
    check_attention(ctx, mt, kind, 14, 2, 1300, [0], 1237)
    check_attention(ctx, mt, kind, 2, 1, 2100, [1500], 600, seed=1)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,window,capacity,positions", [
    (1, 65, 128, [0, 64, 65, 127, 128, 1000]), (4, 65, 128, [0, 61, 124, 126, 997]), (4, 65, 68, [0, 66, 67, 500]),
    (1, 1, 1, [0, 9]), (3, 1, 7, [2, 5, 6]), (40, 100, 139, [0, 100, 1234]), (1, 1000, 1003, [5000, 1, 999]),
    (70, 3, 72, [0, 1, 71]), (130, 200, 333, [1, 1000]),
])
def test_window_and_ring(ctx, mt, kind, rows, window, capacity, positions):
    check_attention(ctx, mt, kind, 14, 2, capacity, positions, rows, window=window)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,capacity,positions", [(1, 16, [15, 16, 40]), (1, 37, [100]), (5, 24, [30, 22]), (50, 64, [40, 90])])
def test_cache_holds_the_last_positions(ctx, mt, kind, rows, capacity, positions):
    """Without a window, positions past the capacity replace the oldest."""
    check_attention(ctx, mt, kind, 6, 2, capacity, positions, rows)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_padding_idle_and_strides(ctx, mt, kind):
    check_attention(ctx, mt, kind, 14, 2, 90, [3, -1, 40, 0, 60], 6, counts=[6, 6, 0, 1, 4], pad_q=8, pad_o=4)
    check_attention(ctx, mt, kind, 14, 2, 91, [3, -1, 40, 0, 60], 1, counts=[1, 1, 0, 1, 9], pad_q=3, pad_o=1, layers=3)
    check_attention(ctx, mt, kind, 3, 1, 64, [10, 50], 20, counts=[-5, 20], pad_q=1, pad_o=5, layers=2)
    check_attention(ctx, mt, kind, 2, 1, 64, [12, 9, 40], 2, base=10, layers=2)
    check_attention(ctx, mt, kind, 2, 1, 80, [-1, -1], 2)  # nothing at all


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 40])
def test_scales_of_very_different_sizes(ctx, mt, kind, rows):
    """Value and key scales over many orders of magnitude, sharp and flat softmaxes."""
    check_attention(ctx, mt, kind, 14, 2, 700, [600], rows, spread=3.0)
    check_attention(ctx, mt, kind, 14, 2, 700, [600], rows, spread=0.1, q_scale=60.0)
    check_attention(ctx, mt, kind, 14, 2, 700, [600], rows, q_scale=1e-6)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 24])
def test_extreme_scales(ctx, mt, kind, rows):
    """All values tiny, all huge, and all zero: relative accuracy does not depend on the unit."""
    import torch
    n = 77 + rows
    g = torch.Generator().manual_seed(5)
    codes = torch.randint(-127, 128, (1, 1, n, 64), generator=g, dtype=torch.int8)
    codes = codes if kind == "int8" else (codes.float() * 3).to(torch.float8_e4m3fn)
    unit = torch.rand(1, 1, n, generator=g) + 0.5
    q = torch.randn(rows, 128, generator=g)
    pos = torch.tensor([77], dtype=torch.int32, device="cuda")
    outs = []
    for kf, vf, qf in ((2.0 ** -6, 1.0, 1.0), (2.0 ** -106, 2.0 ** -120, 2.0 ** 100), (2.0 ** 94, 2.0 ** 110, 2.0 ** -100),
                       (2.0 ** -6, 0.0, 1.0)):
        cache = mt.KV8Cache(codes.cuda(), codes.flip(2).contiguous().cuda(), (unit * kf).cuda(), (unit * vf).cuda())
        out = torch.empty(rows, 128, device="cuda")
        ctx.attention_kv8((q * qf).cuda(), 128, 1, rows, 2, pos, None, 0, cache, out, 128)
        ctx.check()
        outs.append(out.cpu().double())
    assert torch.isfinite(outs[0]).all() and torch.all(outs[3] == 0)
    top = outs[0].abs().amax()
    # powers of two commute with every rounding but those of the fp16 planes' tails: 2^-20 of the largest
    assert torch.all((outs[1] * 2.0 ** 120 - outs[0]).abs() <= 2.0 ** -20 * top)
    assert torch.all((outs[2] * 2.0 ** -110 - outs[0]).abs() <= 2.0 ** -20 * top)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_nan_reaches_only_rows_that_see_it(ctx, mt, kind):
    import torch
    n, rows, hq = 48, 48, 4
    for bad_at in (0, 20, 47):
        for which in (2, 3):
            cache = Cache(mt, kind, 2, n, [(0, n)], 9)
            cache.kv.tensors[which][0, 1, bad_at] = math.nan
            q = torch.randn(rows, hq * 64, device="cuda")
            q[30, :64] = math.nan
            out = torch.empty_like(q)
            pos = torch.zeros(1, dtype=torch.int32, device="cuda")
            ctx.attention_kv8(q, hq * 64, 1, rows, hq, pos, None, 0, cache.kv, out, hq * 64)
            ctx.check()
            bad = torch.isnan(out).view(rows, hq, 64).all(-1).cpu()
            some = torch.isnan(out).view(rows, hq, 64).any(-1).cpu()
            want = torch.zeros(rows, hq, dtype=torch.bool)
            want[bad_at:, 2:] = True
            want[30, 0] = True
            assert torch.equal(bad, want) and torch.equal(some, want)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("prefix_len", [1, 15, 16, 64, 174, 1000])
def test_prefix(ctx, mt, kind, prefix_len):
    own = [0, 1, 15, 16, 17, 63, 100]
    check_attention(ctx, mt, kind, 14, 2, 110, [prefix_len + p for p in own], 1, prefix_len=prefix_len)
    check_attention(ctx, mt, kind, 14, 2, 110, [prefix_len + p for p in own] + [-1], 5, counts=[5, 1, 0, 5, 3, 2, 5, 5],
                    prefix_len=prefix_len, pad_q=4, pad_o=8, layers=2)
    check_attention(ctx, mt, kind, 3, 3, 40, [prefix_len], 1, prefix_len=prefix_len)


@gpu
def test_prefix_shapes(ctx, mt):
    check_attention(ctx, mt, "int8", 14, 2, 70, [4000 + i for i in range(64)], 1, prefix_len=4000, prefix_kind="e4m3")
    check_attention(ctx, mt, "e4m3", 16, 2, 33, [900, 930], 37 - 4, prefix_len=900, prefix_kind="int8")
    check_attention(ctx, mt, "int8", 2, 1, 33, [333, 340, 350], 9, prefix_len=333, seed=3)
    check_attention(ctx, mt, "e4m3", 40, 1, 20, [77, 80], 3, prefix_len=77)
    check_attention(ctx, mt, "int8", 14, 2, 40, [0, 20], 3, prefix_len=0)
    check_attention(ctx, mt, "int8", 14, 2, 20, [50 + 30, 50 + 7], 2, prefix_len=50)  # the own part wraps


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_offsets_past_32_bits(ctx, mt, kind):
    """A slot more than 2^31 bytes (and 2^32 with the second request) into the codes."""
    import torch
    cap = (1 << 25) + 4096
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    small = 64
    p = cap - 100
    k = torch.zeros(2, 1, cap, 64, dtype=torch.uint8, device="cuda").view(torch_kind(kind))
    v = torch.zeros(2, 1, cap, 64, dtype=torch.uint8, device="cuda").view(torch_kind(kind))
    ks, vs = (torch.zeros(2, 1, cap, device="cuda") for _ in range(2))
    big = mt.KV8Cache(k, v, ks, vs)
    part = [torch.zeros(2, 1, small, 64, dtype=torch_kind(kind), device="cuda") for _ in range(2)]
    sc = [torch.zeros(2, 1, small, device="cuda") for _ in range(2)]
    ref = mt.KV8Cache(*part, *sc)
    inv = torch.from_numpy(INV_FREQ).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, hq, w = 12, 2, 16
    qkv = torch.randn(2 * rows, (hq + 2) * 64, device="cuda", generator=g)
    pos = torch.tensor([p, p + 7], dtype=torch.int32, device="cuda")
    outs, reads = [], []
    for cache in (big, ref):  # the same positions in a ring of 64 slots
        q = torch.empty(2 * rows, hq * 64, device="cuda")
        out = torch.empty_like(q)
        back = torch.empty(2, 1, rows, 64, device="cuda")
        ctx.rope_cache_kv8(qkv, (hq + 2) * 64, 2, rows, hq, pos, None, inv, cache, q, hq * 64)
        ctx.kv8_read(cache, 2, rows, pos, None, None, back, rows)
        ctx.attention_kv8(q, hq * 64, 2, rows, hq, pos, None, w, cache, out, hq * 64)
        ctx.check()
        outs.append(out)
        reads.append(back)
    assert torch.equal(reads[0], reads[1])
    assert torch.isfinite(outs[0]).all()
    # the same keys in tiles that start elsewhere: each within the header's bound, A <= |q| |k| / 8 (a code
    # is off by half a step of the largest, so |k| grows by 8 x 2^-4 / 2 at most)
    x = qkv.view(2 * rows, hq + 2, 64)
    a = float(x[:, :hq].norm(dim=-1).max() * x[:, hq].norm(dim=-1).max()) * 1.25 / 8
    tol = 2 * 2 * (2 * 136 * a + 16 + 66) * 2.0 ** -24 * float(reads[0].abs().max())
    assert float((outs[0] - outs[1]).abs().max()) <= tol


# Sizes at which calls of many rows, and long batches of different lengths, are laid out in their own ways.
@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,window,capacity,positions", [
    (500, 300, 900, [0, 1000, 333]), (300, 0, 500, [0, 450, 900]), (400, 1, 701, [0, 301, 302]), (513, 64, 1001, [3, 977]),
    (257, 1000, 1256, [999, 5000, 0]),
])
def test_many_rows_window_and_ring(ctx, mt, kind, rows, window, capacity, positions):
    check_attention(ctx, mt, kind, 14, 2, capacity, positions, rows, window=window)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv", [(14, 2), (5, 5), (40, 1)])
def test_many_rows_padding_idle_and_strides(ctx, mt, kind, hq, hkv):
    positions, counts = [3, -1, 140, 0, 260, 999], [400, 400, 0, 1, 377, 129]
    check_attention(ctx, mt, kind, hq, hkv, 1130, positions, 400, counts=counts, pad_q=8, pad_o=4)
    check_attention(ctx, mt, kind, hq, hkv, 1131, positions, 400, counts=counts, pad_q=3, pad_o=1, layers=3)
    check_attention(ctx, mt, kind, hq, hkv, 900, [200, 100, 150, 400, 99], 470, base=100, layers=2)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_many_rows_scales_of_very_different_sizes(ctx, mt, kind):
    check_attention(ctx, mt, kind, 14, 2, 1300, [800], 400, spread=3.0)
    check_attention(ctx, mt, kind, 14, 2, 1300, [800], 400, spread=0.1, q_scale=60.0)
    check_attention(ctx, mt, kind, 14, 2, 1300, [800], 400, q_scale=1e-6)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_many_rows_extreme_scales(ctx, mt, kind):
    """As test_extreme_scales."""
    import torch
    rows, hq, n = 600, 8, 1400
    g = torch.Generator().manual_seed(5)
    codes = torch.randint(-127, 128, (1, 1, n, 64), generator=g, dtype=torch.int8)
    codes = codes if kind == "int8" else (codes.float() * 3).to(torch.float8_e4m3fn)
    unit = torch.rand(1, 1, n, generator=g) + 0.5
    q = torch.randn(rows, hq * 64, generator=g)
    pos = torch.tensor([n - rows], dtype=torch.int32, device="cuda")
    outs = []
    for kf, vf, qf in ((2.0 ** -6, 1.0, 1.0), (2.0 ** -106, 2.0 ** -120, 2.0 ** 100), (2.0 ** 94, 2.0 ** 110, 2.0 ** -100),
                       (2.0 ** -6, 0.0, 1.0)):
        cache = mt.KV8Cache(codes.cuda(), codes.flip(2).contiguous().cuda(), (unit * kf).cuda(), (unit * vf).cuda())
        out = torch.empty(rows, hq * 64, device="cuda")
        ctx.attention_kv8((q * qf).cuda(), hq * 64, 1, rows, hq, pos, None, 0, cache, out, hq * 64)
        ctx.check()
        outs.append(out.cpu().double())
    assert torch.isfinite(outs[0]).all() and torch.all(outs[3] == 0)
    top = outs[0].abs().amax()
    assert torch.all((outs[1] * 2.0 ** 120 - outs[0]).abs() <= 2.0 ** -20 * top)
    assert torch.all((outs[2] * 2.0 ** -110 - outs[0]).abs() <= 2.0 ** -20 * top)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [900, 1500])
def test_many_rows_nan_reaches_only_rows_that_see_it(ctx, mt, kind, rows):
    import torch
    n, hq = rows, 8
    for bad_at in (0, 450, rows - 1):
        for which in (2, 3):
            cache = Cache(mt, kind, 2, n, [(0, n)], 9)
            cache.kv.tensors[which][0, 1, bad_at] = math.nan
            q = torch.randn(rows, hq * 64, device="cuda")
            q[600, :64] = math.nan
            out = torch.empty_like(q)
            pos = torch.zeros(1, dtype=torch.int32, device="cuda")
            ctx.attention_kv8(q, hq * 64, 1, rows, hq, pos, None, 0, cache.kv, out, hq * 64)
            ctx.check()
            bad = torch.isnan(out).view(rows, hq, 64).all(-1).cpu()
            some = torch.isnan(out).view(rows, hq, 64).any(-1).cpu()
            want = torch.zeros(rows, hq, dtype=torch.bool)
            want[bad_at:, 4:] = True
            want[600, 0] = True
            assert torch.equal(bad, want) and torch.equal(some, want)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,requests,rows", [(16, 16, 47, 2), (16, 16, 64, 8), (8, 8, 61, 9), (16, 16, 21, 17), (32, 32, 50, 1),
                                                  (9, 3, 37, 5), (16, 1, 300, 1)])
def test_many_small_requests(ctx, mt, kind, hq, hkv, requests, rows):
    """More requests and heads than blocks: several share one."""
    positions = [(13 * i) % 50 for i in range(requests)]
    counts = [rows - i % (rows + 1) if i % 3 else rows for i in range(requests)]
    check_attention(ctx, mt, kind, hq, hkv, 70, positions, rows)
    check_attention(ctx, mt, kind, hq, hkv, 41, positions, rows, counts=counts, window=20)
    check_attention(ctx, mt, kind, hq, hkv, 70, [p + 30 if i % 7 else -1 for i, p in enumerate(positions)], rows, counts=counts,
                    prefix_len=30, pad_q=1, pad_o=2)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_many_rows_prefix(ctx, mt, kind):
    """The rows of all requests in one pass over the prefix, padding and idle requests among them."""
    n = 22
    positions = [2000 + 7 * i for i in range(n - 2)] + [-1, 1999]
    counts = [9, 0, 4, 9, 1] * 4 + [9, 9]
    check_attention(ctx, mt, kind, 14, 2, 150, positions, 9, counts=counts, prefix_len=2000, pad_q=1, pad_o=3, layers=2)
    check_attention(ctx, mt, kind, 14, 2, 60, positions, 9, counts=counts, prefix_len=2000)  # own parts that wrap
    check_attention(ctx, mt, kind, 6, 3, 700, [1500, 1600], 600, prefix_len=1500)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,rows,base", [(14, 2, 1, 0), (20, 1, 2, 3), (14, 1, 1, 3)])
def test_long_batch_of_different_lengths(ctx, mt, kind, hq, hkv, rows, base):
    check_attention(ctx, mt, kind, hq, hkv, 40000, [39998, -1, 50, 12345, 3, 30000], rows, base=base)
    check_attention(ctx, mt, kind, hq, hkv, 40000, [39998, 2, 50, 12345, 3, 30000], rows, counts=[1, 0, 1, rows, 1, 0], base=base)
    check_attention(ctx, mt, kind, hq, hkv, 40000, [-1] * 6, rows, base=base)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_long_batch_of_many_requests(ctx, mt, kind):
    positions = [100 + 137 * i for i in range(40)]
    positions[3], positions[20], positions[33], positions[39] = 19999, 0, -1, 16000
    check_attention(ctx, mt, kind, 7, 1, 20000, positions, 1)
    check_attention(ctx, mt, kind, 7, 1, 20000, positions, 1, counts=[1] * 20 + [0] * 15 + [1] * 5)
    check_attention(ctx, mt, kind, 7, 1, 10001, [p + 8000 for p in positions], 2, window=10000)
    check_attention(ctx, mt, kind, 7, 1, 20000, [p + 100 for p in positions], 1, prefix_len=100)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("args", [(14, 2, 40000, [39000, 10, 1000, 0, 25000, 4000], 1), (14, 2, 1500, [0, 700], 600)])
def test_long_calls_repeat_bit_for_bit(ctx, mt, kind, args):
    import torch
    first = check_attention(ctx, mt, kind, *args)

    def both(call):
        s = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for t in s:
            with torch.cuda.stream(t):
                call()
        torch.cuda.synchronize()

    assert torch.equal(check_attention(ctx, mt, kind, *args, run=both), first)


# ------------------------------------------------------------------------------------------------
# As a program uses them
# ------------------------------------------------------------------------------------------------
def decode_loop(ctx, mt, cache, qkvs, hq, hkv, pos, inv, prefix=None, prefix_len=0):
    """Append and attend, a token a step; positions advance on the device."""
    import torch
    n = pos.numel()
    outs = []
    for x in qkvs:
        q, out = torch.empty(n, hq * 64, device="cuda"), torch.empty(n, hq * 64, device="cuda")
        ctx.rope_cache_kv8(x, (hq + 2 * hkv) * 64, n, 1, hq, pos, None, inv, cache, q, hq * 64)
        if prefix is not None:
            ctx.attention_prefix_kv8(q, hq * 64, n, 1, hq, pos, None, prefix, prefix_len, cache, out, hq * 64)
        else:
            ctx.attention_kv8(q, hq * 64, n, 1, hq, pos, None, 0, cache, out, hq * 64)
        pos += 1
        outs.append(out)
    return outs


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_prompt_then_decode_matches_the_fp32_cache(ctx, mt, kind):
    """Prompt and decode steps over the 8-bit cache equal mt_attention over what mt_kv8_read gives back."""
    import torch
    hq, hkv, rows, steps, cap = 14, 2, 53, 4, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    inv = torch.from_numpy(INV_FREQ).cuda()
    cache = mt.KV8Cache.allocate(1, hkv, cap, torch_kind(kind))
    prompt = torch.randn(rows, (hq + 2 * hkv) * 64, device="cuda", generator=g)
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, out = torch.empty(rows, hq * 64, device="cuda"), torch.empty(rows, hq * 64, device="cuda")
    ctx.rope_cache_kv8(prompt, (hq + 2 * hkv) * 64, 1, rows, hq, pos, None, inv, cache, q, hq * 64)
    ctx.attention_kv8(q, hq * 64, 1, rows, hq, pos, None, 0, cache, out, hq * 64)
    k, v = (torch.zeros(1, hkv, cap, 64, device="cuda") for _ in range(2))
    ctx.kv8_read(cache, 1, rows, pos, None, k, v, cap)
    want = torch.empty_like(out)
    ctx.attention(q, hq * 64, rows, hq, hkv, 0, 0, k, v, cap, want, hq * 64)
    ctx.check()
    # both sides are fp32 sums of at most 64 keys: twice the bound of the file's header, A <= 8 * 8 / 8 * 4
    tol = 4 * (2 * 136 * 32 + 16 + 72) * 2.0 ** -24 * float(v.abs().max())
    assert float((out - want).abs().max()) <= tol
    pos += rows
    xs = [torch.randn(1, (hq + 2 * hkv) * 64, device="cuda", generator=g) for _ in range(steps)]
    got = decode_loop(ctx, mt, cache, xs, hq, hkv, pos, inv)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    ctx.kv8_read(cache, 1, rows + steps, zero, None, k, v, cap)
    for i, (x, o) in enumerate(zip(xs, got)):
        p = torch.tensor([rows + i], dtype=torch.int32, device="cuda")
        qi, want = torch.empty(1, hq * 64, device="cuda"), torch.empty(1, hq * 64, device="cuda")
        scratch = mt.KV8Cache.allocate(1, hkv, cap, torch_kind(kind))
        ctx.rope_cache_kv8(x, (hq + 2 * hkv) * 64, 1, 1, hq, p, None, inv, scratch, qi, hq * 64)
        ctx.attention(qi, hq * 64, 1, hq, hkv, rows + i, 0, k, v, cap, want, hq * 64)
        ctx.check()
        assert float((o - want).abs().max()) <= tol


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_shared_prefix_equals_copies(ctx, mt, kind):
    """A batch behind a shared prefix computes what it computes with the prefix copied into every request's cache."""
    import torch
    hq, hkv, n, steps, plen = 14, 2, 5, 3, 174
    g = torch.Generator(device="cuda").manual_seed(4)
    inv = torch.from_numpy(INV_FREQ).cuda()
    prompt = torch.randn(plen, (hq + 2 * hkv) * 64, device="cuda", generator=g)
    zero = torch.zeros(n, dtype=torch.int32, device="cuda")
    prefix = mt.KV8Cache.allocate(1, hkv, plen, torch_kind(kind))
    q = torch.empty(n * plen, hq * 64, device="cuda")
    ctx.rope_cache_kv8(prompt, (hq + 2 * hkv) * 64, 1, plen, hq, zero, None, inv, prefix, q, hq * 64)
    full = mt.KV8Cache.allocate(n, hkv, 200, torch_kind(kind))
    ctx.rope_cache_kv8(prompt.repeat(n, 1), (hq + 2 * hkv) * 64, n, plen, hq, zero, None, inv, full, q, hq * 64)
    own = mt.KV8Cache.allocate(n, hkv, 16, torch_kind(kind), base=plen)
    xs = [torch.randn(n, (hq + 2 * hkv) * 64, device="cuda", generator=g) for _ in range(steps)]
    a = decode_loop(ctx, mt, full, xs, hq, hkv, zero + plen, inv)
    b = decode_loop(ctx, mt, own, xs, hq, hkv, zero + plen, inv, prefix, plen)
    ctx.check()
    tol = 4 * (2 * 136 * 32 + 16 + 90) * 2.0 ** -24 * 6
    for x, y in zip(a, b):
        assert float((x - y).abs().max()) <= tol


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,plen,cap", [(3, 40, 90), (40, 1500, 90), (64, 4000, 100)])
def test_steps_in_the_same_buffers(ctx, mt, kind, n, plen, cap):
    """Steps one behind the other without a pause, in buffers that every step writes again: no kernel starts
    on what an earlier step left there. The same as with the device idle between calls."""
    import torch
    hq, hkv, steps = 14, 2, 40
    g = torch.Generator(device="cuda").manual_seed(8)
    inv = torch.from_numpy(INV_FREQ).cuda()
    prefix = Cache(mt, kind, hkv, plen, [(0, plen)], 1).kv
    xs = torch.randn(steps, n, (hq + 2 * hkv) * 64, device="cuda", generator=g)
    x, q, out = torch.empty_like(xs[0]), torch.empty(n, hq * 64, device="cuda"), torch.empty(n, hq * 64, device="cuda")
    runs = []
    for pause in (False, True):
        cache = mt.KV8Cache.allocate(n, hkv, cap, torch_kind(kind), base=plen)
        pos = torch.full((n,), plen, dtype=torch.int32, device="cuda")
        outs = torch.zeros(steps, n, hq * 64, device="cuda")
        work = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        for i in range(steps):
            x.copy_(xs[i])
            ctx.rope_cache_kv8(x, (hq + 2 * hkv) * 64, n, 1, hq, pos, None, inv, cache, q, hq * 64)
            if pause:
                torch.cuda.synchronize()
            ctx.attention_prefix_kv8(q, hq * 64, n, 1, hq, pos, None, prefix, plen, cache, out, hq * 64, workspace=work)
            if pause:
                torch.cuda.synchronize()
            outs[i] = out
            pos += 1
        ctx.check()
        runs.append(outs)
    assert torch.equal(runs[0], runs[1])


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,plen", [(3, 700), (64, 4000)])
def test_captured_steps_replay(ctx, mt, kind, n, plen):
    """A captured step (append, attention behind a prefix) replayed as positions advance on the device; two
    graphs replayed at once on two streams; results equal the eager ones bit for bit."""
    import torch
    hq, hkv, steps = 14, 2, 5
    g = torch.Generator(device="cuda").manual_seed(6)
    inv = torch.from_numpy(INV_FREQ).cuda()
    prefix = Cache(mt, kind, hkv, plen, [(0, plen)], 1).kv
    xs = [torch.randn(n, (hq + 2 * hkv) * 64, device="cuda", generator=g) for _ in range(steps)]
    eager = mt.KV8Cache.allocate(n, hkv, 600, torch_kind(kind), base=plen)
    want = decode_loop(ctx, mt, eager, xs, hq, hkv, torch.full((n,), plen, dtype=torch.int32, device="cuda"), inv, prefix, plen)
    ctx.check()
    runs = []
    for _ in range(2):
        cache = mt.KV8Cache.allocate(n, hkv, 600, torch_kind(kind), base=plen)
        pos = torch.full((n,), plen, dtype=torch.int32, device="cuda")
        x, out = torch.zeros_like(xs[0]), torch.zeros(n, hq * 64, device="cuda")
        q = torch.zeros(n, hq * 64, device="cuda")
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            ctx.rope_cache_kv8(x, (hq + 2 * hkv) * 64, n, 1, hq, pos, None, inv, cache, q, hq * 64)
            ctx.attention_prefix_kv8(q, hq * 64, n, 1, hq, pos, None, prefix, plen, cache, out, hq * 64)
            pos += 1
        runs.append((graph, torch.cuda.Stream(), x, out, (cache, pos, q)))  # a graph keeps no tensor alive
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(steps):
        for j, (graph, stream, x, out, _) in enumerate(runs):
            with torch.cuda.stream(stream):
                x.copy_(xs[i])
                graph.replay()
                got[j].append(out.clone())
    torch.cuda.synchronize()
    for j in range(2):
        for i in range(steps):
            assert torch.equal(got[j][i], want[i]), f"graph {j} step {i}"


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_repeats_and_streams_agree_bit_for_bit(ctx, mt, kind):
    """The same call gives the same bits, also when two run at once on two streams."""
    import torch
    args = (14, 2, 3000, [2900, 10, 1000], 1)
    first = check_attention(ctx, mt, kind, *args)

    def both(call):
        s = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for t in s:
            with torch.cuda.stream(t):
                call()
        torch.cuda.synchronize()

    assert torch.equal(check_attention(ctx, mt, kind, *args, run=both), first)


@gpu
def test_workspace(ctx, mt):
    """A workspace of the size asked for is enough, its contents do not matter, a smaller one is refused."""
    import torch
    hq, hkv, cap = 14, 2, 20000
    cache = Cache(mt, "int8", hkv, cap, [(0, 15000)], 1).kv
    q = torch.randn(1, hq * 64, device="cuda")
    pos = torch.tensor([14999], dtype=torch.int32, device="cuda")
    need = mt.lib().mt_attention_kv8_workspace(ctx.handle, cache.ref, 1, 1, hq, 0)
    outs = []
    for fill in (0, 255):
        ws = torch.full((max(need, 16),), fill, dtype=torch.uint8, device="cuda")
        out = torch.empty_like(q)
        ctx.attention_kv8(q, hq * 64, 1, 1, hq, pos, None, 0, cache, out, hq * 64, workspace=ws)
        ctx.check()
        outs.append(out)
    assert torch.equal(outs[0], outs[1])
    if need:
        with pytest.raises(mt.MingError) as e:
            ctx.attention_kv8(q, hq * 64, 1, 1, hq, pos, None, 0, cache, out, hq * 64, workspace=ws[:need - 1])
        assert e.value.status == mt.MT_ERR_CAPACITY
    with pytest.raises(mt.MingError) as e:  # more requests than the cache has
        ctx.attention_kv8(q, hq * 64, 2, 1, hq, pos, None, 0, cache, out, hq * 64)
    assert e.value.status == mt.MT_ERR_SHAPE

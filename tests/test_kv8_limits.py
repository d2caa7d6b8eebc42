"""The 8-bit cache attention at the limits of its inputs, against the plain implementation in 64 bits of
test_kv8.py and within the bound derived there.

Caches are laid out by hand: `Keys` has the codes and scales of [requests, kv_heads, n, 64] for keys and values.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

import test_kv8 as base

gpu = base.gpu
KINDS = base.KINDS


class Keys:
    """Random codes, and the scales given (broadcast to [requests, heads, n])."""

    def __init__(self, kind, requests, heads, n, k_scale, v_scale, seed=0):
        import torch
        g = torch.Generator().manual_seed(seed)
        self.codes = []
        for _ in range(2):
            if kind == "int8":
                c = torch.randint(-127, 128, (requests, heads, n, 64), generator=g, dtype=torch.int8)
            else:
                c = (torch.randn(requests, heads, n, 64, generator=g) * 110).clamp(-448, 448).to(torch.float8_e4m3fn)
            self.codes.append(c)
        self.scales = [torch.as_tensor(s, dtype=torch.float32).expand(requests, heads, n).clone() for s in (k_scale, v_scale)]

    def values(self, which, r):
        return self.codes[which][r].double() * self.scales[which][r].double()[..., None]

    def cache(self, mt, start=0):
        return mt.KV8Cache(*(t.cuda() for t in (*self.codes, *self.scales)), base=start)


def attend(ctx, mt, keys, q, positions, window=0, prefix=None):
    """One call (rows from q [requests, rows, hq, 64]): the output, the plain one and its bound, per request."""
    import torch
    n, rows, hq, _ = q.shape
    plen = prefix.codes[0].shape[2] if prefix else 0
    qd = q.reshape(n * rows, hq * 64).float().cuda()
    out = torch.full_like(qd, 7.0)
    pos = torch.tensor([plen + p for p in positions], dtype=torch.int32, device="cuda")
    cache = keys.cache(mt, plen)
    if prefix:
        ctx.attention_prefix_kv8(qd, hq * 64, n, rows, hq, pos, None, prefix.cache(mt), plen, cache, out, hq * 64)
    else:
        ctx.attention_kv8(qd, hq * 64, n, rows, hq, pos, None, window, cache, out, hq * 64)
    ctx.check()
    out = out.cpu().double().view(n, rows, hq, 64)
    results = []
    for r, p in enumerate(positions):
        at, mine = torch.arange(p + rows), torch.arange(p, p + rows)
        sees = at <= mine[:, None]
        if window:
            sees &= at > mine[:, None] - window
        k, v = (keys.values(w, r)[:, :p + rows] for w in range(2))
        if prefix:
            k, v = torch.cat([prefix.values(0, 0), k], 1), torch.cat([prefix.values(1, 0), v], 1)
            sees = torch.cat([torch.ones(rows, plen, dtype=torch.bool), sees], 1)
        want, bound = base.attend_reference(q[r].float().double(), k, v, sees)
        results.append((out[r], want, bound))
    return results


def check(results):
    import torch
    for r, (got, want, bound) in enumerate(results):
        assert torch.isfinite(got).all(), f"request {r}: {int((~torch.isfinite(got)).sum())} outputs are not finite"
        err = (got - want).abs().amax(-1)
        assert torch.all(err <= bound), (f"request {r}: worst error {float((err / bound).max()):.3g} of the bound at "
                                         f"{np.unravel_index(int((err / bound).argmax()), err.shape)}")


# ------------------------------------------------------------------------------------------------
# Scores far below zero
# ------------------------------------------------------------------------------------------------
def against(kind, requests, heads, n, score, seed=0):
    """Keys whose codes are the largest against a query of ones: scores of about `score` ([n]) each."""
    import torch
    limit = base.LIMIT[kind]
    keys = Keys(kind, requests, heads, n, -torch.as_tensor(score, dtype=torch.float32) / (8 * limit), 2.0 / limit, seed)
    keys.codes[0] = torch.full_like(keys.codes[0].float(), -limit).to(base.torch_kind(kind))
    return keys


def ones(requests, rows, hq, seed=0):
    import torch
    g = torch.Generator().manual_seed(seed)
    return 1.0 + 0.05 * torch.rand(requests, rows, hq, 64, generator=g)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("low", [-85.0, -95.0, -300.0, -4e4])
def test_first_scores_far_below_zero(ctx, mt, kind, low):
    """Every key that a warp meets first scores below the range of 2^-x: one key, one tile, windows, many rows."""
    import torch
    spread = low + 3 * torch.rand(4096, generator=torch.Generator().manual_seed(1)) - 3
    check(attend(ctx, mt, against(kind, 1, 2, 1, spread[:1]), ones(1, 1, 14), [0]))
    check(attend(ctx, mt, against(kind, 2, 2, 300, spread[:300]), ones(2, 1, 14), [11, 299]))
    rising = torch.cat([spread[:70], spread[70:700] * 0.5])  # the largest scores come later
    check(attend(ctx, mt, against(kind, 1, 2, 700, rising), ones(1, 1, 14), [699]))
    check(attend(ctx, mt, against(kind, 1, 2, 700, rising), ones(1, 9, 6), [650]))
    check(attend(ctx, mt, against(kind, 1, 2, 64, spread[:64]), ones(1, 20, 4), [40], window=1))
    check(attend(ctx, mt, against(kind, 1, 2, 700, spread[:700]), ones(1, 40, 4), [600], window=200))
    check(attend(ctx, mt, against(kind, 1, 1, 4000, spread[:4000]), ones(1, 1, 7), [3999]))
    check(attend(ctx, mt, against(kind, 1, 2, 1024, spread[:1024]), ones(1, 500, 14), [500]))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("plen", [40, 1500])
def test_own_scores_far_below_zero_behind_a_prefix(ctx, mt, kind, plen):
    """A request's own keys score far below the prefix's, and far above them."""
    low, fair = against(kind, 3, 2, 20, [-300.0 - i for i in range(20)]), Keys(kind, 1, 2, plen, 0.5 / base.LIMIT[kind], 1.0, seed=2)
    check(attend(ctx, mt, low, ones(3, 1, 14), [0, 5, 19], prefix=fair))
    check(attend(ctx, mt, low, ones(3, 4, 14), [0, 5, 16], prefix=fair))
    deep = against(kind, 1, 2, plen, [-300.0 - i % 7 for i in range(plen)], seed=3)
    own = Keys(kind, 3, 2, 20, 0.5 / base.LIMIT[kind], 1.0, seed=4)
    check(attend(ctx, mt, own, ones(3, 1, 14), [0, 5, 19], prefix=deep))


# ------------------------------------------------------------------------------------------------
# Value scales of different sizes
# ------------------------------------------------------------------------------------------------
def value_scale_calls(ctx, mt, kind, scales, q_size=0.01, key_scale=None):
    """Calls of every layout over keys whose value scales are `scales(n)`. Queries are small, so that the
    scores' part of the bound is, and weights nearly equal."""
    import torch
    ks = 2.0 / base.LIMIT[kind] if key_scale is None else key_scale

    def q(*shape, seed=0):
        return q_size * torch.randn(*shape, 64, generator=torch.Generator().manual_seed(seed))

    def keys(requests, heads, n, seed=0):
        return Keys(kind, requests, heads, n, ks, scales(n), seed)

    check(attend(ctx, mt, keys(2, 2, 300), q(2, 1, 14), [40, 299]))
    check(attend(ctx, mt, keys(1, 2, 300), q(1, 9, 6), [291]))
    check(attend(ctx, mt, keys(1, 2, 4000), q(1, 1, 14), [3999]))
    check(attend(ctx, mt, keys(2, 2, 4000), q(2, 1, 14), [3999, 1000]))
    check(attend(ctx, mt, keys(1, 2, 1024), q(1, 500, 14), [524]))
    check(attend(ctx, mt, keys(1, 2, 700), q(1, 700, 14), [0]))
    fair = Keys(kind, 64, 2, 20, ks, float(scales(4000)[-1]), seed=5)
    check(attend(ctx, mt, fair, q(64, 1, 14), [i % 20 for i in range(64)], prefix=keys(1, 2, 4000)))
    check(attend(ctx, mt, Keys(kind, 3, 2, 20, ks, float(scales(174)[-1]), seed=5), q(3, 1, 14), [0, 7, 19], prefix=keys(1, 2, 174)))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("zeros", [1, 16, 64, 200])
@pytest.mark.parametrize("size", [4.0, 1e-2, 1e-4, 1e-6, 1e-30])
def test_zero_values_first(ctx, mt, kind, zeros, size):
    """The first value rows are zero (scale 0, as they are written), the rest of one size: errors are relative to it."""
    import torch

    def scales(n):
        s = size * (0.5 + torch.rand(n, generator=torch.Generator().manual_seed(7)))
        s[:zeros] = 0.0
        return s

    value_scale_calls(ctx, mt, kind, scales)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("first,small,large", [(16, -126, 0), (64, -126, 0), (64, -126, 110), (130, -100, 20), (300, -20, 100),
                                               (20, 105, -100), (300, 30, -126)])
def test_value_scales_of_any_ratio(ctx, mt, kind, first, small, large):
    """The first value scales 2^small, the others 2^large: each row is exact to the largest value that it sees itself."""
    import torch

    def scales(n):
        s = 1 + torch.rand(n, generator=torch.Generator().manual_seed(8), dtype=torch.float64)
        s[:first] *= 2.0 ** small
        s[first:] *= 2.0 ** large
        return s.float()

    value_scale_calls(ctx, mt, kind, scales)


# ------------------------------------------------------------------------------------------------
# Key scales near the largest and the smallest number
# ------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("power", [90, 112, 116, -100, -126])
def test_key_scales_of_any_size(ctx, mt, kind, power):
    """Scores of ordinary size from keys near either end of fp32 and queries near the other."""
    import torch
    value_scale_calls(ctx, mt, kind, lambda n: torch.full((n,), 0.01), q_size=2.0 ** (-power - 4), key_scale=2.0 ** power)


# ------------------------------------------------------------------------------------------------
# Scores of any size
# ------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [1e5, 3e7, 1e9, 1e12, 1e20, 1e30])
@pytest.mark.parametrize("v_power", [-6, -40, 40])
def test_scores_of_any_size(ctx, mt, kind, size, v_power):
    """Scores so large that fp32 holds no fraction of them: where one key is ahead by more than twice what the
    scores may be off, all others weigh nothing (e^-30 and less), and the output is its value."""
    import torch
    root = math.sqrt(size / 8)
    spread = torch.exp2(torch.randint(0, 12, (4000,), generator=torch.Generator().manual_seed(3)).float())
    seen = 0

    def run(requests, heads, n, rows, hq, positions, plen=0):
        nonlocal seen
        g = torch.Generator().manual_seed(n)
        q = root * torch.randn(requests, rows, hq, 64, generator=g)
        keys = Keys(kind, requests, heads, n, 2 * root / base.LIMIT[kind], 2.0 ** v_power * spread[:n], seed=n)
        prefix = Keys(kind, 1, heads, plen, 2 * root / base.LIMIT[kind], 2.0 ** v_power * spread[:plen], seed=n + 1) if plen else None
        results = attend(ctx, mt, keys, q, positions, prefix=prefix)
        check(results)
        for r, (got, want, _) in enumerate(results):
            p = positions[r]
            k, v = (torch.cat([prefix.values(w, 0), keys.values(w, r)], 1) if plen else keys.values(w, r) for w in range(2))
            for h in range(hq):
                kv = h // (hq // heads)
                s = q[r, :, h].double() @ k[kv].T / 8
                s = s.masked_fill(torch.arange(k.shape[1]) - plen > torch.arange(p, p + rows)[:, None], -math.inf)
                a = (q[r, :, h].double().abs() @ k[kv].abs().T / 8).amax(-1)
                top = s.topk(min(2, s.shape[1]), -1)
                ahead = top.values[:, 0] - top.values[:, -1] > 4 * 136 * 2.0 ** -24 * a + 30 if s.shape[1] > 1 else torch.ones(rows, dtype=torch.bool)
                value = v[kv][top.indices[:, 0]]
                err = (got[:, h] - value).abs().amax(-1)
                assert torch.all((err <= 2.0 ** -18 * value.abs().amax(-1)) | ~ahead), f"request {r} head {h}"
                seen += int(ahead.sum())

    run(2, 2, 300, 1, 14, [40, 299])
    run(1, 2, 60, 20, 6, [30])
    run(1, 2, 4000, 1, 14, [3999])
    run(1, 2, 1024, 500, 14, [524])
    run(1, 1, 1, 1, 3, [0])
    run(40, 2, 20, 1, 14, [i % 20 for i in range(40)], plen=3000)
    run(3, 2, 20, 1, 14, [0, 7, 19], plen=174)
    assert seen > 0


# ------------------------------------------------------------------------------------------------
# Workspace queries (on the CPU: of a context they read the number of SMs only)
# ------------------------------------------------------------------------------------------------
QUERIES = '''
import ctypes, sys
sys.path.insert(0, "tests")
import conftest
mt = conftest.load_package()
context = (ctypes.c_int * 1024)(*[148] * 1024)  # whatever a context's layout, its numbers of SMs is 148
ctx = ctypes.cast(context, ctypes.c_void_p)


def sizes(requests, rows, hq, window=0, prefix_len=16, kv_heads=2, capacity=512, base=0):
    c = mt.KV8CacheStruct(0, kv_heads, capacity, base, max(kv_heads * capacity, 0), None, None, None, None)
    return (mt.lib().mt_attention_kv8_workspace(ctx, ctypes.byref(c), requests, rows, hq, window),
            mt.lib().mt_attention_prefix_kv8_workspace(ctx, prefix_len, ctypes.byref(c), requests, rows, hq))


big = 2 ** 31 - 1
good = sizes(1, 1, 14, capacity=20000)
assert good[0] > 0 and good[1] > good[0], good
for bad in (dict(hq=1), dict(hq=3), dict(hq=0), dict(hq=-2), dict(hq=1026), dict(hq=2, kv_heads=0), dict(hq=2, kv_heads=-1),
            dict(hq=2, kv_heads=big), dict(requests=big, rows=big, capacity=1 << 30), dict(requests=-1), dict(rows=-1), dict(requests=0),
            dict(rows=0), dict(capacity=0), dict(capacity=-5), dict(capacity=big), dict(rows=513), dict(requests=big // 14 + 1)):
    got = sizes(**{**dict(requests=1, rows=1, hq=14), **bad})
    assert got == (0, 0), (bad, got)
assert sizes(1, 1, 14, window=-1)[0] == 0 and sizes(1, 1, 14, window=513)[0] == 0 and sizes(1, 1, 14, window=big)[0] == 0
assert sizes(1, 1, 14, prefix_len=-1)[1] == 0 and sizes(1, 1, 14, prefix_len=(1 << 30) + 1)[1] == 0
most = sizes(requests=1, rows=1 << 21, hq=1023, kv_heads=1, capacity=1 << 30, prefix_len=1 << 30)
assert most[1] >= (1 << 21) * 1023 * 66 * 4 * 2, most
print("sizes fine")
'''


def test_workspace_queries_refuse_in_a_process_of_their_own():
    """Sizes that the calls refuse need nothing; none of them ends the process."""
    import os
    import subprocess
    import sys
    got = subprocess.run([sys.executable, "-c", QUERIES], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                         capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and "sizes fine" in got.stdout, (got.returncode, got.stdout, got.stderr[-800:])


@gpu
def test_attention_refuses_head_counts(ctx, mt):
    """A head count that does not go with the cache is an error of the call, with and without a prefix."""
    import torch
    cache, prefix = mt.KV8Cache.allocate(1, 2, 64, base=16), mt.KV8Cache.allocate(1, 2, 16)
    q, pos = torch.zeros(1, 1024, device="cuda"), torch.full((1,), 20, dtype=torch.int32, device="cuda")
    for hq in (1, 3, 0, -2):
        for call in (lambda: ctx.attention_kv8(q, 1024, 1, 1, hq, pos, None, 0, cache, q.clone(), 1024),
                     lambda: ctx.attention_prefix_kv8(q, 1024, 1, 1, hq, pos, None, prefix, 16, cache, q.clone(), 1024)):
            with pytest.raises(mt.MingError) as e:
                call()
            assert e.value.status == mt.MT_ERR_SHAPE


# ------------------------------------------------------------------------------------------------
# Tensors of the Python calls (on the CPU: refused before anything reads them)
# ------------------------------------------------------------------------------------------------
def tensor_calls(mt, on="cpu"):
    """Per call of Context: its tensors by name (2 requests of 3 rows, 4 heads on 2), and the call itself with some replaced."""
    import torch
    from types import SimpleNamespace
    ctx = object.__new__(mt.Context)
    ctx.device = 0
    cache = SimpleNamespace(requests=2, kv_heads=2, index=0, device="cuda:0", ref=None)
    qkv, q, pos = torch.zeros(6, 512, device=on), torch.zeros(6, 256, device=on), torch.zeros(2, dtype=torch.int32, device=on)
    append = dict(qkv=qkv, positions=pos, counts=pos, inv_freq=torch.zeros(32, device=on), q_out=q)
    read = dict(positions=pos, counts=pos, k=torch.zeros(2, 2, 5, 64, device=on), v=torch.zeros(2, 2, 5, 64, device=on))
    attend = dict(q=q, positions=pos, counts=pos, out=q.clone())
    return [
        (append, lambda a: ctx.rope_cache_kv8(a["qkv"], 512, 2, 3, 4, a["positions"], a["counts"], a["inv_freq"], cache, a["q_out"], 256)),
        (read, lambda a: ctx.kv8_read(cache, 2, 3, a["positions"], a["counts"], a["k"], a["v"], 5)),
        (attend, lambda a: ctx.attention_kv8(a["q"], 256, 2, 3, 4, a["positions"], a["counts"], 0, cache, a["out"], 256)),
        (attend, lambda a: ctx.attention_prefix_kv8(a["q"], 256, 2, 3, 4, a["positions"], a["counts"], cache, 3, cache, a["out"], 256)),
    ]


def test_calls_refuse_tensors_of_the_host(mt, monkeypatch):
    """None of them reaches the library, with everything else in order."""
    import torch
    monkeypatch.setattr(mt, "lib", lambda: pytest.fail("the library was called"))
    real = torch.Tensor.get_device
    for args, call in tensor_calls(mt):
        for host in args:
            others = [id(t) for name, t in args.items() if name != host and t is not args[host]]
            monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0 if id(t) in others else real(t))
            with pytest.raises(mt.MingError) as e:
                call(args)
            assert e.value.status == mt.MT_ERR_ARG, host


def test_calls_refuse_tensors_of_another_type_or_size(mt, monkeypatch):
    import torch
    monkeypatch.setattr(mt, "lib", lambda: pytest.fail("the library was called"))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    for args, call in tensor_calls(mt):
        for name in args:
            if name in ("positions", "counts"):
                continue
            for dtype in (torch.bfloat16, torch.float16, torch.float64, torch.int32):
                with pytest.raises(TypeError):
                    call({**args, name: args[name].to(dtype)})
            short = args[name].flatten()
            gap = 128 if name in ("k", "v") else 0  # rows 3 and 4 of the last head are not part of the call
            spread = torch.zeros(4, 512)[:, ::2] if name != "inv_freq" else torch.zeros(20)[::2]
            for bad in (short[:len(short) - gap - 1], args[name][:1], spread[:0]) + ((spread,) if name in ("q", "out", "q_out") else ()) + (
                    (torch.zeros(2, 2, 5, 128)[..., :64],) if name in ("k", "v") else ()):
                with pytest.raises(mt.MingError) as e:
                    call({**args, name: bad})
                assert e.value.status == mt.MT_ERR_SHAPE, name


def test_workspaces_of_the_host_or_with_gaps_are_refused(mt):
    import torch
    ctx = object.__new__(mt.Context)
    ctx.device = 0
    with pytest.raises(mt.MingError) as e:
        ctx._workspace(64, torch.zeros(64, dtype=torch.uint8), None, None)
    assert e.value.status == mt.MT_ERR_ARG


@gpu
def test_calls_take_views(ctx, mt):
    """q as the first columns of qkv and rows of a larger buffer, as before."""
    import torch
    hq, hkv = 4, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(6, (hq + 2 * hkv) * 64, device="cuda", generator=g)
    pos, inv = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.from_numpy(base.INV_FREQ).cuda()
    outs = []
    for view in (False, True):
        cache = mt.KV8Cache.allocate(2, hkv, 8)
        x, out = qkv.clone(), torch.zeros(9, hq * 64 + 8, device="cuda")
        q = x[:, :hq * 64] if view else torch.empty(6, hq * 64, device="cuda")
        ld = x.shape[1] if view else hq * 64
        ctx.rope_cache_kv8(x, x.shape[1], 2, 3, hq, pos, None, inv, cache, q, ld)
        ctx.attention_kv8(q, ld, 2, 3, hq, pos, None, 0, cache, out[2:8, 8:], hq * 64 + 8)
        ctx.check()
        assert torch.all(out[:2] == 0) and torch.all(out[8:] == 0) and torch.all(out[:, :8] == 0)
        outs.append(out)
    assert torch.equal(outs[0], outs[1])


@gpu
@pytest.mark.parametrize("behind", [False, True])
def test_default_workspace_on_another_stream(ctx, mt, behind):
    """A call on a stream given by its handle, without a workspace: memory that the current stream allocates after
    the call does not share with the workspace that the call is still to use."""
    import torch
    hq, hkv, n, plen = 14, 2, 20000, 4000
    g = torch.Generator(device="cuda").manual_seed(5)
    full = Keys("int8", 1, hkv, n, 2.0 / 127, 2.0 / 127).cache(mt, plen if behind else 0)
    prefix = Keys("int8", 1, hkv, plen, 2.0 / 127, 2.0 / 127, seed=1).cache(mt)
    q = torch.randn(1, hq * 64, device="cuda", generator=g)
    pos = torch.tensor([n - 1 + (plen if behind else 0)], dtype=torch.int32, device="cuda")

    def call(out, **k):
        if behind:
            ctx.attention_prefix_kv8(q, hq * 64, 1, 1, hq, pos, None, prefix, plen, full, out, hq * 64, **k)
        else:
            ctx.attention_kv8(q, hq * 64, 1, 1, hq, pos, None, 0, full, out, hq * 64, **k)

    want, out = torch.empty_like(q), torch.empty_like(q)
    call(want)
    need = (mt.lib().mt_attention_prefix_kv8_workspace(ctx.handle, plen, full.ref, 1, 1, hq) if behind else
            mt.lib().mt_attention_kv8_workspace(ctx.handle, full.ref, 1, 1, hq, 0))
    assert need > 0
    call(out, stream=torch.cuda.default_stream().cuda_stream)
    assert torch.equal(out, want)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    for _ in range(5):
        with torch.cuda.stream(other):
            torch.cuda._sleep(4_000_000)  # some ms in which the call waits
        call(out, stream=other.cuda_stream)
        mine = [torch.full((need,), 255, dtype=torch.uint8, device="cuda") for _ in range(3)]  # NaN, as fp32
        while not other.query():  # for as long as the call may read and write
            for t in mine:
                t.fill_(255)
            torch.cuda.current_stream().synchronize()
        torch.cuda.synchronize()
        assert all(bool((t == 255).all()) for t in mine)
        assert torch.equal(out, want)
        del mine

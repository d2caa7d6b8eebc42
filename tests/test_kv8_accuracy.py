"""How exact the 8-bit cache attention is (relative to each output's own norm), and which kernels its calls launch.

The bounds of test_kv8.py are worst cases over all signs. Errors of independent roundings add up as their squares
do; with that, for an output of one row and head (64 dimensions) over n keys, S its largest |q.k| / 8:

* a score: queries in two planes (2^-22 at most, 2^-22.8 in the mean, of a sum of 64 terms that has the score's own
  deviation), four steps of the matrix unit that drop up to 2^-24 of it each, four roundings of 2^-24: a weight is off
  by at most 2^-20.6 S, and by 2^-22 for the exponential;
* a product of weight and value scale: 2^-22, and 2^-25 of the row's unit where it is far below that (keys behind one
  that has most of the weight): sqrt(n) 2^-25.8 of the output together;
* sums: eight steps of the matrix unit (2^-21 at most), weights added 16 keys at a time: sqrt(n / 16) 2^-24.

Together no more than 2^-21 (2 + S) + sqrt(n) 2^-24 of the output's norm, some 4e-6 at 300 keys. Queries or weights in
one plane would be 1e-4 off.
"""
from __future__ import annotations

import math

import pytest

import test_kv8 as base
import test_kv8_limits as limits

gpu = base.gpu
KINDS = base.KINDS


def check_norms(ctx, mt, keys, q, positions, window=0, prefix=None):
    import torch
    n, rows, hq, _ = q.shape
    worst = 0.0
    for r, (got, want, _) in enumerate(limits.attend(ctx, mt, keys, q, positions, window=window, prefix=prefix)):
        p = positions[r]
        k = keys.values(0, r)[:, :p + rows]
        at = torch.arange(p + rows)
        sees = at <= torch.arange(p, p + rows)[:, None]
        if window:
            sees &= at > torch.arange(p, p + rows)[:, None] - window
        if prefix:
            k = torch.cat([prefix.values(0, 0), k], 1)
            sees = torch.cat([torch.ones(rows, k.shape[1] - p - rows, dtype=torch.bool), sees], 1)
        for h in range(hq):
            s = (q[r, :, h].float().double() @ k[h // (hq // k.shape[0])].T / 8).abs().masked_fill(~sees, 0.0).amax(-1)
            tol = 2.0 ** -21 * (2 + s) + sees.sum(-1).double().sqrt() * 2.0 ** -24
            err = (got[:, h] - want[:, h]).norm(dim=-1) / want[:, h].norm(dim=-1)
            worst = max(worst, float((err / tol).max()))
    assert worst <= 1, f"worst error {worst:.3g} of the bound"


def some(kind, requests, heads, n, seed=0, spread=0.5):
    """Keys like those of the cases here and there: scales over a factor of some ten."""
    import torch
    g = torch.Generator().manual_seed(seed + 100)
    ks, vs = (torch.exp(spread * torch.randn(requests, heads, n, generator=g)) * (2.0 / base.LIMIT[kind]) for _ in range(2))
    return limits.Keys(kind, requests, heads, n, ks, vs, seed=seed)


def queries(requests, rows, hq, seed=0):
    import torch
    return torch.randn(requests, rows, hq, 64, generator=torch.Generator().manual_seed(seed))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("requests,n,rows,positions,window", [
    (1, 1, 1, [0], 0), (1, 2, 1, [1], 0), (3, 17, 1, [0, 8, 16], 0), (1, 301, 1, [300], 0), (8, 500, 1, [60 * i + 70 for i in range(8)], 0),
    (1, 5000, 1, [4999], 0), (3, 9000, 1, [8999, 100, 4000], 0), (4, 300, 4, [100, 200, 296, 0], 65), (2, 333, 9, [0, 300], 0),
    (1, 53, 53, [0], 0), (1, 1200, 600, [600], 0), (1, 1300, 1300, [0], 0), (2, 900, 500, [0, 400], 300),
])
def test_errors_are_those_of_fp32(ctx, mt, kind, requests, n, rows, positions, window):
    check_norms(ctx, mt, some(kind, requests, 2, n), queries(requests, rows, 14), positions, window)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("plen,requests,rows", [(174, 8, 1), (40, 3, 5), (4000, 64, 1), (1500, 2, 300)])
def test_errors_are_those_of_fp32_behind_a_prefix(ctx, mt, kind, plen, requests, rows):
    positions = [(37 * i) % 100 for i in range(requests)]
    check_norms(ctx, mt, some(kind, requests, 2, 100 + rows), queries(requests, rows, 14), positions, prefix=some(kind, 1, 2, plen, seed=1))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,rows", [(300, 1), (4096, 1), (16384, 1), (2000, 24), (4096, 300)])
@pytest.mark.parametrize("ahead,value", [(10.0, 1.0), (10.0, 1e-3), (16.0, 30.0)])
def test_a_first_key_with_most_of_the_weight(ctx, mt, kind, n, rows, ahead, value):
    """An attention sink: the first key is `ahead` of the others' mean score, its value of an ordinary size or not."""
    import torch
    g = torch.Generator().manual_seed(n)
    u = torch.randint(0, 2, (64,), generator=g) * 2.0 - 1
    keys = some(kind, 1, 2, n)
    keys.codes[0][:, :, 0] = (u * base.LIMIT[kind]).to(base.torch_kind(kind))
    keys.scales[0][:, :, 0] = ahead / 4 / base.LIMIT[kind]  # q.k / 8 = (u / 2).(u ahead / 4) / 8 and some
    keys.scales[1][:, :, 0] *= value
    check_norms(ctx, mt, keys, queries(1, rows, 14) * 0.8 + 0.5 * u, [n - rows])


# ------------------------------------------------------------------------------------------------
# Layouts
# ------------------------------------------------------------------------------------------------
def kernels(call):
    """Names of the kernels that a call launches, from a graph of it."""
    import torch
    driver = pytest.importorskip("cuda.bindings.driver")

    def ask(result):
        assert result[0] == driver.CUresult.CUDA_SUCCESS, result
        return result[1:]

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        call()
    raw = driver.CUgraph(graph.raw_cuda_graph())
    names = []
    nodes, count = ask(driver.cuGraphGetNodes(raw, 64))
    for node in nodes[:count]:
        if ask(driver.cuGraphNodeGetType(node))[0] == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            params = ask(driver.cuGraphKernelNodeGetParams(node))[0]
            names.append(ask(driver.cuFuncGetName(params.func))[0].decode())
    assert names
    return names


def layout(ctx, mt, hq, hkv, capacity, positions, rows, counts=None, window=0, prefix_len=0, at=0, kind="int8"):
    """{"wide", "warp", "shared", "passes", "join", "join_few"}: what a call of these sizes launches."""
    import torch
    n = len(positions)
    dtype = base.torch_kind(kind)
    cache = mt.KV8Cache.allocate(n, hkv, capacity, dtype, base=prefix_len or at)
    prefix = mt.KV8Cache.allocate(1, hkv, prefix_len, dtype) if prefix_len else None
    q = torch.zeros(n * rows, hq * 64, device="cuda")
    out, pos = torch.zeros_like(q), torch.tensor(positions, dtype=torch.int32, device="cuda")
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")

    def call():
        if prefix_len:
            ctx.attention_prefix_kv8(q, hq * 64, n, rows, hq, pos, cnt, prefix, prefix_len, cache, out, hq * 64)
        else:
            ctx.attention_kv8(q, hq * 64, n, rows, hq, pos, cnt, window, cache, out, hq * 64)

    found = set()
    for name in kernels(call):
        if "kv8_wide_kernel" in name:
            found.add("wide")
        elif "kv8_passes_kernel" in name:
            found.add("passes")
        elif "kv8_pass_kernel" in name:
            found.add("shared" if "Lb1" in name or "true" in name else "warp")
        elif "kv8_join_few_kernel" in name:
            found.add("join_few")
        elif "kv8_join_kernel" in name:
            found.add("join")
    ctx.check()
    return found


STAGGERED = [100 + 137 * i for i in range(40)]


@gpu
@pytest.mark.parametrize("found,args,options", [
    # Both sides of the rule between the kernels, and of the number of parts.
    ({"warp"}, (14, 2, 512, [300], 1), {}),
    ({"warp"}, (14, 2, 512, [60 * i + 70 for i in range(8)], 1), {}),
    ({"warp", "join_few"}, (14, 2, 4000, [3999], 1), {}),
    ({"warp", "join"}, (14, 2, 5000, [4999], 1), {}),
    ({"warp"}, (14, 2, 333, [0, 200, 57], 130), {}),
    ({"wide"}, (14, 2, 900, [0, 1000, 333], 500), {"window": 300}),
    ({"wide", "join_few"}, (14, 2, 1300, [0], 1237), {}),
    ({"warp"}, (8, 2, 900, [0], 900), {}),
    ({"wide", "join_few"}, (8, 2, 1500, [0], 1500), {}),
    ({"warp", "join_few"}, (14, 2, 2000, [1976], 24), {}),
    ({"wide", "join_few"}, (14, 2, 4096, [2000], 300), {}),
    # Sizes of the tests of many rows.
    ({"wide", "join_few"}, (14, 2, 500, [0, 450, 900], 300), {}),
    ({"wide", "join_few"}, (14, 2, 701, [0, 301, 302], 400), {"window": 1}),
    ({"wide", "join_few"}, (14, 2, 1001, [3, 977], 513), {"window": 64}),
    ({"wide", "join_few"}, (14, 2, 1256, [999, 5000, 0], 257), {"window": 1000}),
    ({"wide"}, (14, 2, 1130, [3, -1, 140, 0, 260, 999], 400), {}),
    ({"wide", "join_few"}, (5, 5, 1130, [3, -1, 140, 0, 260, 999], 400), {}),
    ({"wide"}, (40, 1, 900, [200, 100, 150, 400, 99], 470), {"at": 100}),
    ({"wide", "join_few"}, (14, 2, 1300, [800], 400), {}),
    ({"wide", "join_few"}, (8, 1, 1400, [800], 600), {}),
    ({"wide", "join_few"}, (14, 2, 1024, [524], 500), {}),
    ({"wide", "join_few"}, (14, 2, 700, [0], 700), {}),
    ({"warp"}, (16, 16, 70, [i % 50 for i in range(64)], 8), {}),
    # Slots shared out by length.
    ({"shared", "join"}, (14, 2, 40000, [39998, -1, 50, 12345, 3, 30000], 1), {}),
    ({"wide", "join"}, (20, 1, 40000, [39998, -1, 50, 12345, 3, 30000], 2), {"at": 3}),
    ({"shared", "join"}, (14, 1, 40000, [39998, -1, 50, 12345, 3, 30000], 1), {"at": 3}),
    ({"shared", "join"}, (7, 1, 20000, STAGGERED, 1), {}),
    ({"shared", "join"}, (7, 1, 10001, STAGGERED, 2), {"window": 10000}),
    # Behind a prefix: both passes in one launch, or beside one another.
    ({"passes", "join_few"}, (14, 2, 110, [174 + p for p in range(7)], 1), {"prefix_len": 174}),
    ({"passes", "join_few"}, (14, 2, 90, [1500] * 40, 1), {"prefix_len": 1500}),
    ({"wide", "warp", "join"}, (14, 2, 70, [4000 + i for i in range(64)], 1), {"prefix_len": 4000}),
    ({"wide", "warp", "join_few"}, (6, 3, 700, [1500, 1600], 600), {"prefix_len": 1500}),
    ({"shared", "warp", "join"}, (7, 1, 20000, [p + 100 for p in STAGGERED], 1), {"prefix_len": 100}),
    ({"shared", "wide", "join"}, (7, 1, 20000, [p + 16000 for p in STAGGERED], 1), {"prefix_len": 16000}),
])
def test_layouts(ctx, mt, found, args, options):
    """The layout that each test of that size is for (on 148 SMs; the rule goes by their number)."""
    import torch
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("layouts of 148 SMs")
    assert layout(ctx, mt, *args, **options) == found


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_shared_slots_beside_a_wide_prefix(ctx, mt, kind):
    base.check_attention(ctx, mt, kind, 7, 1, 20000, [p + 16000 for p in STAGGERED], 1, prefix_len=16000)


@gpu
def test_long_calls_need_a_workspace(ctx, mt):
    """Of the sizes at which test_kv8.py gives too small a one."""
    cache = mt.KV8Cache.allocate(1, 2, 20000)
    assert mt.lib().mt_attention_kv8_workspace(ctx.handle, cache.ref, 1, 1, 14, 0) > 0


# ------------------------------------------------------------------------------------------------
# What the bound would notice
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [17, 301, 5000])
@pytest.mark.parametrize("plane", ["queries", "weights"])
def test_the_bound_notices_a_missing_plane(n, plane):
    """On the CPU, in 64 bits but for queries or weights rounded to fp16 once."""
    import torch
    q = queries(1, 8, 7)[0].double()
    keys = some("int8", 1, 1, n)
    k, v = keys.values(0, 0)[0], keys.values(1, 0)[0]
    over = []
    for h in range(7):
        s = q[:, h] @ k.T / 8
        want = torch.softmax(s, -1) @ v
        if plane == "queries":
            got = torch.softmax(q[:, h].half().double() @ k.T / 8, -1) @ v
        else:
            w = torch.exp(s - s.amax(-1, keepdim=True))
            got = (w * keys.scales[1][0, 0]).half().double() @ (v / keys.scales[1][0, 0].double()[:, None]) / w.sum(-1, keepdim=True)
        tol = 2.0 ** -21 * (2 + s.abs().amax(-1)) + math.sqrt(n) * 2.0 ** -24
        over.append((got - want).norm(dim=-1) / want.norm(dim=-1) / tol)
    assert float(torch.stack(over).median()) > 8

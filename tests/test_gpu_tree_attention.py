"""Attention for trees of drafted tokens on the GPU against its definition in
64 bits (oracle/quant.py)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from litevllm import _hip, ops
from oracle import quant as oq
from test_gpu_quant_cache import (BS, CODES, DTYPES, cache_values, check, make_batch,
                                  pieces_written, rows, same)

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[case] {msg}", flush=True)


def random_parents(g, n):
    return [-1 if j == 0 else int(torch.randint(-1, j, (1,), generator=g)) for j in range(n)]


def make_trees(seed, device, heads, offs, nodes, dtype, code=None, fill=math.nan):
    """Trees of `nodes` drafted tokens behind `offs` committed ones; code None:
    a cache of dtype.  Rows of the cache that no context reaches hold NaN."""
    ctx = [o + n for o, n in zip(offs, nodes)]
    g = torch.Generator().manual_seed(seed + 1000)
    if code is not None:
        b = make_batch(seed, device, heads, ctx, nodes, dtype, code, fill=fill)
    else:
        H, Hkv, D = heads
        nb = [-(-c // BS) for c in ctx]
        pool = sum(nb) + 3
        k, v = (rows(g, pool * BS, Hkv, D).to(dtype) for _ in range(2))
        perm = torch.randperm(pool, generator=g).to(torch.int32)
        tables = torch.zeros(len(ctx), max(nb + [1]), dtype=torch.int32)
        used = torch.zeros(pool * BS, dtype=torch.bool)
        at = 0
        for i, (c, n) in enumerate(zip(ctx, nb)):
            tables[i, :n] = perm[at:at + n]
            at += n
            pos = torch.arange(c)
            used[tables[i].long()[pos // BS] * BS + pos % BS] = True
        k[~used], v[~used] = fill, fill
        b = dict(kv=[x.view(pool, BS, Hkv, D).to(device) for x in (k, v)], tables=tables,
                 ctx=torch.tensor(ctx, dtype=torch.int32),
                 cu=torch.tensor([0] + list(np.cumsum(nodes)), dtype=torch.int32),
                 q=torch.randn(sum(nodes), H, D, generator=g).to(dtype), heads=heads, lens=nodes,
                 scale=1 / math.sqrt(D))
    b["parents"] = [random_parents(g, n) for n in nodes]
    b["sees"] = [oq.ancestors(p) for p in b["parents"]]
    words = max(1, -(-max(nodes) // 64))
    b["mask"] = torch.from_numpy(np.concatenate([oq.mask_words(s, words) for s in b["sees"]]))
    return b


def reference(b):
    kv = cache_values(b["cache"]) if "cache" in b else [x.cpu().double() for x in b["kv"]]
    outs = []
    for i, n in enumerate(b["lens"]):
        c = int(b["ctx"][i])
        at = b["tables"][i].long()[:-(-c // BS)]
        k, v = (x[at].reshape(-1, *x.shape[2:])[:c] for x in kv)
        sees = np.ones((n, c), bool)
        base = c - n
        s = np.asarray(b["sees"][i])
        sees[:, max(base, 0):] = s[:, max(-base, 0):n]
        outs.append(oq.attention(b["q"][int(b["cu"][i]):int(b["cu"][i + 1])], k, v, sees,
                                 b["scale"]))
    return [torch.cat(x) for x in zip(*outs)]


def run(b, device, **kw):
    d = lambda t: t.to(device)
    args = (d(b["tables"]), d(b["ctx"]), d(b["cu"]), d(b["mask"]))
    kw = dict(scale=b["scale"], max_query_len=max(b["lens"]), **kw)
    if "cache" in b:
        return ops.tree_attention_quant(d(b["q"]), b["cache"], *args, **kw)
    return ops.tree_attention(d(b["q"]), *b["kv"], *args, **kw)


HEADS = [(16, 8, 128), (4, 2, 64), (8, 1, 128), (6, 2, 64), (2, 2, 128)]


@pytest.mark.parametrize("code", [None] + CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", HEADS)
def test_trees(device, code, dtype, heads):
    _say(f"trees {code} {dtype} {heads}")
    nodes = [1, 2, 7, 16, 17, 31, 5, 33, 64, 1, 13]
    offs = [0, 0, 1, 15, 300, 63, 64, 130, 500, 700, 3]
    b = make_trees(21, device, heads, offs, nodes, dtype, code)
    check(run(b, device), reference(b), dtype)


@pytest.mark.parametrize("code", [None, torch.int8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_small_trees_only(device, code, dtype):
    _say(f"small trees {code} {dtype}")
    b = make_trees(22, device, (16, 8, 128), [700, 200, 0], [4, 7, 3], dtype, code)
    check(run(b, device), reference(b), dtype)
    b = make_trees(23, device, (4, 2, 64), [100, 1000], [10, 16], dtype, code)
    check(run(b, device), reference(b), dtype)


@pytest.mark.parametrize("code", [None, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_trees(device, code, dtype):
    """More than one mask word, several row tiles, contexts split over many
    workgroups."""
    _say(f"large trees {code} {dtype}")
    b = make_trees(24, device, (8, 2, 64), [0, 30, 6000], [200, 130, 97], dtype, code)
    check(run(b, device), reference(b), dtype)


@pytest.mark.parametrize("code", [None, torch.int8])
def test_any_mask(device, code):
    """Masks that are no tree: rows that see nothing at all, rows that do not
    see themselves, bits past the drafted tokens."""
    _say(f"any mask {code}")
    for offs, nodes in (([0, 40, 0], [9, 30, 70]), ([0], [3])):
        b = make_trees(25, device, (4, 2, 128), offs, nodes, torch.bfloat16, code)
        g = torch.Generator().manual_seed(2)
        b["sees"] = [(torch.rand(n, n, generator=g) < 0.3).numpy() for n in nodes]
        b["sees"][0][1] = False
        b["sees"][-1][2] = False
        words = b["mask"].shape[1]
        b["mask"] = torch.from_numpy(np.concatenate([oq.mask_words(s, words) for s in b["sees"]]))
        b["mask"][2, words - 1] |= -(1 << 62)       # bits of no token of the first sequence
        got = run(b, device)
        check(got, reference(b), torch.bfloat16)
        assert not got[1].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_hidden_rows_that_are_not_finite(device, dtype, value):
    """NaN and infinities in drafted K and V do not reach the rows that do not
    see them."""
    _say(f"hidden {value} {dtype}")
    heads = (4, 2, 64)
    b = make_trees(26, device, heads, [50, 10, 1000], [40, 70, 12], dtype)
    want = reference(b)
    bad = {0: 3, 1: 66, 2: 0}                     # sequence: drafted token
    blind = torch.ones(sum(b["lens"]), dtype=torch.bool)
    for i, t in bad.items():
        p = int(b["ctx"][i]) - b["lens"][i] + t
        blk = int(b["tables"][i, p // BS])
        for x in b["kv"]:
            x[blk, p % BS] = value
        blind[int(b["cu"][i]):int(b["cu"][i + 1])] = torch.from_numpy(~b["sees"][i][:, t])
    got = run(b, device)
    check(got[blind.to(device)], [w[blind] for w in want], dtype)
    if math.isnan(value):
        assert torch.isnan(got[~blind.to(device)].float()).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_values_in_view(device, dtype):
    """An infinite V that a row sees is infinite in its output, in that dim."""
    _say(f"inf in view {dtype}")
    b = make_trees(27, device, (4, 2, 64), [30, 200], [10, 50], dtype)
    spots = {0: (3, 5), 1: (7, 60)}               # sequence: (drafted token, dim)
    for i, (t, dim) in spots.items():
        p = int(b["ctx"][i]) - b["lens"][i] + t
        b["kv"][1][int(b["tables"][i, p // BS]), p % BS, :, dim] = math.inf
    got = run(b, device).float().cpu()
    for i, (t, dim) in spots.items():
        r = got[int(b["cu"][i]):int(b["cu"][i + 1])]
        sees = torch.from_numpy(b["sees"][i][:, t])
        assert bool((r[sees][:, :, dim] == math.inf).all())
        others = torch.ones(64, dtype=torch.bool)
        others[dim] = False
        assert torch.isfinite(r[:, :, others]).all() and torch.isfinite(r[~sees]).all()


def test_strides_and_rows_past_the_batch(device):
    _say("tree strides")
    b = make_trees(28, device, (6, 2, 64), [50, 20], [12, 20], torch.float16)
    T = 32 + 4
    wide = torch.zeros(T, 10, 64, dtype=torch.float16, device=device)
    wide[:32, 2:8] = b["q"].to(device)
    out = torch.full((T, 8, 64), 3.0, dtype=torch.float16, device=device)
    mask = torch.full((T, 1), -1, dtype=torch.int64, device=device)
    mask[:32] = b["mask"].to(device)
    d = lambda t: t.to(device)
    ops.tree_attention(wide[:, 2:8], *b["kv"], d(b["tables"]), d(b["ctx"]), d(b["cu"]), mask,
                       scale=b["scale"], max_query_len=20, out=out[:, 1:7])
    check(out[:32, 1:7], reference(b), torch.float16)
    assert bool((out[32:] == 3.0).all()) and bool((out[:, [0, 7]] == 3.0).all())


def test_context_shorter_than_the_rows(device):
    """Fewer cached tokens than drafted rows: the first drafted ones are not in
    the cache and nobody sees them."""
    _say("short context")
    b = make_trees(29, device, (4, 2, 64), [40, 0], [10, 20], torch.bfloat16)
    b["ctx"][1] = 12
    check(run(b, device), reference(b), torch.bfloat16)
    b["ctx"][1] = 0
    got = run(b, device)
    check(got, reference(b), torch.bfloat16)
    assert not got[10:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("code", [None, torch.int8, torch.float8_e4m3fn])
def test_scores_of_huge_magnitude(device, dtype, code):
    """Scores near the end of the fp32 range: the larger one takes all, also
    where every score is far below zero."""
    _say(f"huge {dtype} {code}")
    b = make_trees(34, device, (4, 2, 64), [1, 40], [1, 40], dtype, fill=0.0)
    b["q"] = torch.full_like(b["q"], 1e18)
    k, v = (x.cpu() for x in b["kv"])
    k.fill_(-2e18)
    best = []
    for i in range(2):
        p = int(b["ctx"][i]) - b["lens"][i]       # the first drafted token: all see it
        at = int(b["tables"][i, p // BS]), p % BS
        k[at] = -1e18
        best.append(v[at])
    b["kv"] = [k.to(device), v.to(device)]
    if code is not None:
        n = k.shape[0]
        b["cache"] = ops.quant_kv_cache(n, BS, 2, 64, code, device)
        rows_ = [x.view(n * BS, 2, 64) for x in b["kv"]]
        ops.kv_scatter_quant(*rows_, b["cache"], torch.arange(n * BS, device=device))
        best = [oq.values(x, code) for x in best]
    b["sees"][1][:, 0] = True
    assert all(s[:, 0].all() for s in b["sees"])
    b["mask"][:, 0] |= 1
    got = run(b, device).double().cpu()
    for i in range(2):
        for j in range(int(b["cu"][i]), int(b["cu"][i + 1])):
            want = best[i].double().repeat_interleave(2, 0)
            # weights 1 and 0: the result's rounding, and three fp32 roundings
            # (a reciprocal of the scale, the quotient, the unit)
            tol = (torch.finfo(dtype).eps / 2 + 4 * 2.0 ** -23) * want.abs()
            assert bool(((got[j] - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_sequences(device, dtype):
    """More sequences than a launch takes, one of them with several row tiles."""
    _say(f"many trees {dtype}")
    n = 4200
    nodes = [1 + i % 2 for i in range(n)]
    nodes[4150] = 70
    b = make_trees(35, device, (4, 2, 64), [i % 5 for i in range(n)], nodes, dtype)
    check(run(b, device), reference(b), dtype)


def test_block_ids_outside_the_cache(device):
    _say("tree bad ids")
    b = make_trees(30, device, (4, 2, 64), [40], [10], torch.bfloat16)
    want = b["tables"].clone()
    want[0, 1] = 0
    b["tables"][0, 1] = 1 << 30
    ops.device_errors()
    got = run(b, device)
    assert ops.device_errors() == _hip.LV_DEVERR_BLOCK_ID
    b["tables"] = want
    for x in b["kv"]:
        x[0] = torch.nan_to_num(x[0])
    check(run(b, device), reference(b), torch.bfloat16)


def test_mask_of_parents(device):
    _say("tree_mask")
    g = torch.Generator().manual_seed(5)
    for nodes in ([1], [5, 0, 64, 65, 3], [130, 1, 200]):
        parents = [random_parents(g, n) for n in nodes]
        if nodes[0] == 130:
            parents[0][7] = 7                    # its own index and later ones: no parent
            parents[0][9] = 100
        words = max(1, -(-max(nodes) // 64))
        want = np.concatenate([oq.mask_words(oq.ancestors(p), words) if p else
                               np.zeros((0, words), np.int64) for p in parents])
        cu = torch.tensor([0] + list(np.cumsum(nodes)), dtype=torch.int32, device=device)
        flat = torch.tensor(sum(parents, []), dtype=torch.int32, device=device)
        got = ops.tree_mask(flat, cu, max(nodes))
        assert np.array_equal(got.cpu().numpy(), want)


@torch.inference_mode()
def test_streams_and_graphs(device):
    _say("tree streams and graphs")
    a = make_trees(31, device, (16, 8, 128), [2000, 90], [20, 64], torch.bfloat16)
    c = make_trees(32, device, (16, 8, 128), [1500, 9], [7, 5], torch.bfloat16, torch.int8)
    refs = [reference(a), reference(c)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(a, device)
    torch.cuda.current_stream().wait_stream(side)
    check(got, refs[0], torch.bfloat16)
    graphs, outs, keep = [], [], []
    for b in (a, c):
        d = {k: v.to(device) for k, v in b.items() if torch.is_tensor(v)}
        ws = torch.empty(max(256, ops.tree_attention_workspace_size(
            len(b["lens"]), b["q"].shape[0], max(b["lens"]), 16, 8, 128, d["tables"].shape[1],
            b["q"].dtype)), dtype=torch.uint8, device=device)
        out = torch.empty_like(d["q"])
        kv = (b["cache"],) if "cache" in b else tuple(b["kv"])
        op = ops.tree_attention_quant if "cache" in b else ops.tree_attention
        call = lambda: op(d["q"], *kv, d["tables"], d["ctx"], d["cu"], d["mask"],
                          scale=b["scale"], max_query_len=max(b["lens"]), out=out, workspace=ws)
        call()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            call()
        graphs.append(graph)
        outs.append(out)
        keep.append((d, ws))
    for _ in range(3):
        for graph, out in zip(graphs, outs):
            out.zero_()
            graph.replay()
            run(a, device)
        torch.cuda.synchronize()
        for out, ref in zip(outs, refs):
            check(out, ref, torch.bfloat16)


def test_same_call_same_bits(device):
    _say("tree repeatable")
    b = make_trees(33, device, (16, 2, 128), [5000, 700], [30, 64], torch.bfloat16)
    first = run(b, device)
    for _ in range(3):
        assert same(run(b, device), first)


@pytest.mark.parametrize("code,dtype,n", [
    (None, torch.bfloat16, 192), (None, torch.float16, 420), (torch.int8, torch.bfloat16, 200),
    (torch.float8_e4m3fn, torch.float16, 300), (None, torch.float32, 200)])
@pytest.mark.parametrize("longest,whole", [(1540, True), (6000, False)])
def test_units_whole_or_in_pieces(device, code, dtype, n, longest, whole):
    """Trees on both sides of the same choice: few and many, on eight and on four
    wavefronts."""
    _say(f"tree units {code} {dtype} {n} {longest}")
    heads = (2, 2, 64)
    offs = [1440 + 10 * (i // 50) if i % 20 == 3 else 850 + i % 60 for i in range(n)]
    offs[43] = longest
    nodes = [1 + i % 3 for i in range(n)]
    nodes[7], nodes[23], nodes[150], nodes[31] = 70, 66, 130, 0
    b = make_trees(36, device, heads, offs, nodes, dtype, code, fill=0.0)
    b["tables"] = torch.nn.functional.pad(b["tables"], (0, 400 - b["tables"].shape[1]))
    need = ops.tree_attention_workspace_size(n, sum(nodes), 130, *heads, 400, dtype)
    got = []
    split = pieces_written(lambda ws: got.append(run(b, device, workspace=ws)), need)
    assert split != whole
    check(got[0], reference(b), dtype)


@pytest.mark.parametrize("code", [None] + CODES)
@pytest.mark.parametrize("bad", [1 << 30, -2])
def test_rows_of_block_ids_outside_the_cache(device, code, bad):
    """Such an id reads block 0, in every row that sees its keys, and nothing else
    changes."""
    _say(f"tree bad ids {code} {bad}")
    b = make_trees(37, device, (4, 2, 64), [40, 3, 2000], [10, 70, 5], torch.bfloat16, code,
                   fill=0.0)
    at = ((0, 1), (1, 4), (2, 60))                # committed and drafted keys
    want = dict(b, tables=b["tables"].clone())
    for i, j in at:
        assert j * BS < int(b["ctx"][i])
        want["tables"][i, j] = 0
        b["tables"][i, j] = bad
    ops.device_errors()
    got = run(b, device)
    assert ops.device_errors() == _hip.LV_DEVERR_BLOCK_ID
    check(got, reference(want), torch.bfloat16)
    assert ops.device_errors() == 0

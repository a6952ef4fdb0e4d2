"""The 8-bit paged cache on the GPU: writers, reader and attention against the
definitions in 64 bits (oracle/quant.py)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from litevllm import _hip, ops
from oracle import quant as oq

pytestmark = pytest.mark.gpu

CODES = [torch.int8, torch.float8_e4m3fn]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
BS = 16


def _say(msg):
    print(f"[case] {msg}", flush=True)


def rows(g, *shape):
    """Normal values with a few wide channels and heads of unlike size."""
    x = torch.randn(*shape, generator=g)
    return x * (1 + 5 * (torch.rand(*shape[1:], generator=g) < 0.05)) \
        * (0.2 + torch.rand(shape[1], 1, generator=g))


def token_major(n, hkv, d, dtype, device):
    """A cache in the layout of the 16-bit one."""
    codes = torch.zeros((2, n, BS, hkv, d), dtype=torch.int8, device=device).view(dtype)
    scales = torch.zeros((2, n, BS, hkv), dtype=torch.float32, device=device)
    return ops.QuantKV(codes[0], codes[1], scales[0], scales[1])


def cache_values(cache):
    """float64 [N, bs, Hkv, D] of key and value codes * scales, on the CPU."""
    return [c.float().cpu().double() * s.cpu().double()[..., None]
            for c, s in ((cache.key, cache.key_scale), (cache.value, cache.value_scale))]


def same(a, b):
    """Bitwise, NaN included."""
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# -- writing and reading -----------------------------------------------------

@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,d,tokens,layout", [
    (8, 128, 61, "heads"), (1, 64, 1, "heads"), (3, 128, 77, "tokens"), (2, 256, 33, "heads"),
    (8, 64, 1000, "tokens")])
def test_scatter_and_gather(device, code, dtype, hkv, d, tokens, layout):
    """Codes and scales exactly as defined, only at their slots; padding skipped;
    values read back rounded once."""
    _say(f"scatter {code} {dtype} hkv={hkv} d={d} T={tokens} {layout}")
    g = torch.Generator().manual_seed(7)
    n = tokens // BS + 4
    k, v = rows(g, tokens, hkv, d).to(dtype), rows(g, tokens, hkv, d).to(dtype)
    k[0, 0] = 0
    if tokens > 40:
        k[5, 0] = 0
        k[7, 0] *= 1e-3 if dtype == torch.float16 else 1e-20
        v[9, hkv - 1, 3] = math.nan
        v[11, 0, 1] = math.inf
        k[12, 0, 2] = -math.inf
    slots = torch.randperm(n * BS, generator=g)[:tokens]
    slots[3::10] = -1
    qkv = torch.zeros(tokens, 3, hkv, d, dtype=dtype)      # rows inside a wider tensor
    qkv[:, 1], qkv[:, 2] = k, v
    qkv = qkv.to(device)
    make = token_major if layout == "tokens" else \
        (lambda *a: ops.quant_kv_cache(a[0], BS, *a[1:]))
    cache = make(n, hkv, d, code, device)
    for t in (cache.key, cache.value):
        t.view(torch.int8).fill_(5)
    cache.key_scale.fill_(-2.0)
    cache.value_scale.fill_(-2.0)
    ops.kv_scatter_quant(qkv[:, 1], qkv[:, 2], cache, slots.to(device))
    at = slots[slots >= 0]
    for x, codes, scale in ((k, cache.key, cache.key_scale), (v, cache.value, cache.value_scale)):
        want_c = torch.full((n * BS, hkv, d), 5, dtype=torch.int8).view(code).float().double()
        want_s = torch.full((n * BS, hkv), -2.0)
        c, s = oq.quantise(x[slots >= 0], code)
        want_c[at], want_s[at] = c, s
        assert torch.equal(codes.float().cpu().double().reshape(-1, hkv, d), want_c)
        assert torch.equal(torch.nan_to_num(scale.cpu().reshape(-1, hkv), nan=-7.0),
                           torch.nan_to_num(want_s, nan=-7.0))
    for out_dtype in DTYPES:
        got = ops.kv_gather_quant(cache, slots.to(device), out_dtype)
        for x, y in zip((k, v), got):
            c, s = oq.quantise(x, code)
            want = (c.float() * s[..., None]).to(out_dtype)    # one fp32 product, one rounding
            want[slots < 0] = 0
            assert torch.equal(torch.nan_to_num(y.cpu().float(), nan=-7.0),
                               torch.nan_to_num(want.float(), nan=-7.0)), out_dtype


@pytest.mark.parametrize("bs", [1, 12, 32])
def test_block_sizes(device, bs):
    """Slots of blocks of other sizes, no power of two among them."""
    _say(f"block size {bs}")
    g = torch.Generator().manual_seed(4)
    n, hkv, d, tokens = -(-200 // bs), 5, 64, 150
    k, v = (rows(g, tokens, hkv, d).to(torch.bfloat16) for _ in range(2))
    slots = torch.randperm(n * bs, generator=g)[:tokens]
    cache = ops.quant_kv_cache(n, bs, hkv, d, torch.int8, device)
    ops.kv_scatter_quant(k.to(device), v.to(device), cache, slots.to(device))
    for x, codes, scale in ((k, cache.key, cache.key_scale), (v, cache.value, cache.value_scale)):
        c, s = oq.quantise(x, torch.int8)
        want = torch.zeros(n * bs, hkv, d, dtype=torch.float64)
        want[slots] = c
        assert torch.equal(codes.cpu().double().reshape(-1, hkv, d), want)
        assert torch.equal(scale.cpu().reshape(-1, hkv)[slots], s)
    got = ops.kv_gather_quant(cache, slots.to(device), torch.float32)
    for x, y in zip((k, v), got):
        c, s = oq.quantise(x, torch.int8)
        assert torch.equal(y.cpu(), c.float() * s[..., None])


def test_gather_into_given_rows(device):
    """Strided outputs, unaligned rows, and slots past the cache."""
    _say("gather strided")
    g = torch.Generator().manual_seed(3)
    cache = ops.quant_kv_cache(4, BS, 2, 64, torch.int8, device)
    k = rows(g, 64, 2, 64).to(device)
    ops.device_errors()
    ops.kv_scatter_quant(k, k * 2, cache, torch.arange(64, device=device))
    slots = torch.tensor([5, -1, 64, 63, 5], device=device)
    buf = torch.full((5, 2 * 128 + 3), 9.0, device=device)
    a, b = buf[:, 1:129].view(5, 2, 64), buf[:, 130:258].view(5, 2, 64)
    out = ops.kv_gather_quant(cache, slots, torch.float32, out=(a, b))
    assert out[0] is a and out[1] is b
    assert ops.device_errors() == _hip.LV_DEVERR_SLOT
    want = ops.kv_gather_quant(cache, torch.tensor([5, 63, 5], device=device), torch.float32)
    for x, w in zip((a, b), want):
        assert torch.equal(x[[0, 3, 4]], w)
        assert not x[[1, 2]].any()
    assert bool((buf[:, [0, 129, 258]] == 9.0).all())


def test_scatter_slot_errors(device):
    _say("scatter past the cache")
    cache = ops.quant_kv_cache(2, BS, 2, 64, torch.int8, device)
    k = torch.ones(3, 2, 64, device=device)
    ops.device_errors()
    ops.kv_scatter_quant(k, k, cache, torch.tensor([31, 32, -5], device=device))
    assert ops.device_errors() == _hip.LV_DEVERR_SLOT
    assert int((cache.key_scale != 0).sum()) == 2      # the one row of two heads


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,tokens,norm,offset", [
    ((16, 8, 128), 37, True, 0), ((4, 2, 64), 130, False, 0), ((3, 1, 128), 5, True, 1),
    ((8, 8, 256), 9, True, 0)])
def test_prologue(device, code, dtype, heads, tokens, norm, offset):
    """q within its one rounding; K and V rows within half a code step (plus
    what fp32 leaves) of the rows in 64 bits."""
    H, Hkv, D = heads
    _say(f"prologue {code} {dtype} {heads} T={tokens} norm={norm} offset={offset}")
    g = torch.Generator().manual_seed(13)
    width = (H + 2 * Hkv) * D
    buf = torch.zeros(tokens, width + 8, dtype=dtype)
    qkv = rows(g, tokens, H + 2 * Hkv, D).view(tokens, width).to(dtype)
    buf[:, offset:offset + width] = qkv
    ang = torch.randn(300, D // 2, generator=g, dtype=torch.float64) * 3
    cos, sin = ang.cos().to(dtype), ang.sin().to(dtype)
    pos = torch.randint(0, 300, (tokens,), generator=g)
    qw = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype) if norm else None
    kw = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype) if norm else None
    n = tokens // BS + 2
    slots = torch.randperm(n * BS, generator=g)[:tokens]
    slots[2] = -1
    cache = ops.quant_kv_cache(n, BS, Hkv, D, code, device)
    dev = lambda t: None if t is None else t.to(device)
    q = ops.qk_norm_rope_cache_quant(dev(buf)[:, offset:offset + width], H, Hkv, D, dev(cos),
                                     dev(sin), dev(pos), dev(slots), cache, dev(qw), dev(kw),
                                     eps=1e-5)
    x = qkv.double().view(tokens, -1, D)
    parts = [x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]]
    for i, w in ((0, qw), (1, kw)):
        y = parts[i]
        if norm:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-5) * w.double()
        c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
        a, b = y[..., :D // 2], y[..., D // 2:]
        parts[i] = torch.cat([a * c - b * s, b * c + a * s], -1)
        # |a c| + |b s| bounds what the fp32 roundings act on: the norm's sum of D squares, its
        # root and three products, then two products and a sum of the rotation
        parts.append(torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
                     * (D / 2 + 8) * 2.0 ** -24)
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    err = (q.cpu().double() - parts[0]).abs()
    assert bool((err <= half * parts[0].abs() + 2 * parts[3] + tiny).all()), err.max()
    got = [t.cpu().double() for t in ops.kv_gather_quant(cache, dev(slots), torch.float32)]
    keep = slots >= 0
    for y, want, f32 in ((got[0], parts[1], parts[4]), (got[1], parts[2], torch.zeros(1))):
        top = want.abs().amax(-1, keepdim=True)
        if code == torch.int8:
            step = top / 127 / 2 * torch.ones_like(want)
        else:   # half a step of e4m3: 2^-4 of the value, at least 2^-10 of the scale
            step = torch.maximum(want.abs() * 2.0 ** -4, top / 448 * 2.0 ** -10)
        # the scale follows the largest value's fp32 error; a value near a tie may go to either
        # side of it: twice the fp32 error more
        room = step * (1 + 2.0 ** -16) + 3 * (f32 + f32.amax(-1, keepdim=True)) + 2.0 ** -20 * top
        bad = (y - want).abs() > room
        assert not bad[keep].any(), (y - want).abs()[keep].max()
        assert not y[~keep].any()


def test_prologue_far_positions(device):
    """Positions without a cos / sin row: NaN queries and NaN cached rows."""
    _say("prologue positions")
    cache = ops.quant_kv_cache(2, BS, 1, 64, torch.int8, device)
    qkv = torch.ones(3, 3 * 64, dtype=torch.bfloat16, device=device)
    cos = torch.ones(4, 32, dtype=torch.bfloat16, device=device)
    q = ops.qk_norm_rope_cache_quant(qkv, 1, 1, 64, cos, cos, torch.tensor([0, 4, -1], device=device),
                                     torch.arange(3, device=device), cache)
    assert torch.isfinite(q[0]).all() and torch.isnan(q[1:].float()).all()
    k, v = ops.kv_gather_quant(cache, torch.arange(3, device=device), torch.float32)
    assert torch.isfinite(k[0]).all() and torch.isnan(k[1:]).all() and torch.isfinite(v).all()


# -- attention -----------------------------------------------------------------

def make_batch(seed, device, heads, ctx, lens, dtype, code, layout="heads", fill=None, qscale=1.0):
    """A paged batch over a shuffled cache: ctx / lens of every sequence.  Rows
    of the cache that no context reaches hold `fill` scales and odd codes."""
    H, Hkv, D = heads
    g = torch.Generator().manual_seed(seed)
    nb = [-(-c // BS) for c in ctx]
    pool = sum(nb) + 3
    make = token_major if layout == "tokens" else \
        (lambda *a: ops.quant_kv_cache(a[0], BS, *a[1:]))
    cache = make(pool, Hkv, D, code, device)
    k, v = rows(g, pool * BS, Hkv, D), rows(g, pool * BS, Hkv, D)
    ops.kv_scatter_quant(k.to(device), v.to(device), cache, torch.arange(pool * BS, device=device))
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    tables = torch.zeros(len(ctx), max(nb + [1]), dtype=torch.int32)
    used = torch.zeros(pool * BS, dtype=torch.bool)
    at = 0
    for i, (c, n) in enumerate(zip(ctx, nb)):
        tables[i, :n] = perm[at:at + n]
        at += n
        pos = torch.arange(c)
        used[tables[i].long()[pos // BS] * BS + pos % BS] = True
    if fill is not None:
        # every code byte is a NaN of e4m3; all scales of unused rows are `fill`
        free = ~used.view(pool, BS).to(device)
        for t in (cache.key, cache.value):
            t.view(torch.int8)[free] = -1
        cache.key_scale[free] = fill
        cache.value_scale[free] = fill
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32)
    q = (torch.randn(int(cu[-1]), H, D, generator=g) * qscale).to(dtype)
    return dict(cache=cache, tables=tables, ctx=torch.tensor(ctx, dtype=torch.int32), cu=cu, q=q,
                heads=heads, lens=lens, scale=1 / math.sqrt(D))


def reference(b, sees_of=None):
    kv = cache_values(b["cache"])
    outs = []
    for i, n in enumerate(b["lens"]):
        c = int(b["ctx"][i])
        at = b["tables"][i].long()[:-(-c // BS)]
        k, v = (x[at].reshape(-1, *x.shape[2:])[:c] for x in kv)
        sees = np.tril(np.ones((n, c), bool), c - n) if sees_of is None else sees_of(i, n, c)
        q = b["q"][int(b["cu"][i]):int(b["cu"][i + 1])]
        outs.append(oq.attention(q, k, v, sees, b["scale"]))
    return [torch.cat(x) for x in zip(*outs)]


def run(b, device, num_decodes, **kw):
    d = lambda t: t.to(device)
    return ops.paged_attention_quant(d(b["q"]), b["cache"], d(b["tables"]), d(b["ctx"]),
                                     scale=b["scale"], cu_seqlens=d(b["cu"]),
                                     num_decodes=num_decodes,
                                     max_query_len=max(list(b["lens"]) + [1]), **kw)


def check(got, ref, dtype, what=""):
    err = (got.cpu().double() - ref[0]).abs()
    tol = oq.tolerance(*ref, dtype)
    assert torch.isfinite(got).all(), what
    worst = (err / tol).max()
    assert worst <= 1, f"{what}: {float(worst):.2f} of the tolerance, max-abs {float(err.max()):.2e}"


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 700]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(16, 8, 128), (4, 2, 64), (8, 1, 128), (32, 4, 64), (5, 1, 64),
                                   (6, 2, 128), (8, 8, 128)])
def test_decode(device, code, dtype, heads):
    _say(f"decode {code} {dtype} {heads}")
    b = make_batch(5, device, heads, EDGES, [1] * len(EDGES), dtype, code, fill=math.nan)
    got = run(b, device, len(EDGES))
    check(got, reference(b), dtype)
    assert not got[0].any()                       # context 0: zeros
    d = lambda t: t.to(device)
    again = ops.paged_attention_quant(d(b["q"]), b["cache"], d(b["tables"]), d(b["ctx"]),
                                      scale=b["scale"])
    assert same(again, got)                       # without cu_seqlens


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(16, 8, 128), (4, 2, 64), (8, 1, 128), (12, 4, 64), (7, 1, 128)])
def test_mixed(device, code, dtype, heads):
    """Decode rows, then chunks of odd lengths at odd offsets, from the first
    token on."""
    _say(f"mixed {code} {dtype} {heads}")
    lens = [1] * 6 + [1, 2, 5, 16, 17, 33, 64, 65, 100, 129, 257]
    offs = [0, 1, 40, 200, 300, 17] + [0, 0, 3, 16, 100, 31, 0, 64, 257, 500, 1]
    ctx = [o + n for o, n in zip(offs, lens)]
    b = make_batch(6, device, heads, ctx, lens, dtype, code, fill=math.nan)
    check(run(b, device, 6), reference(b), dtype)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_long_rows(device, code, dtype):
    """Contexts that are split over many workgroups."""
    _say(f"long {code} {dtype}")
    ctx = [20011, 3, 9000]
    b = make_batch(8, device, (8, 2, 128), ctx, [1, 1, 1], dtype, code, fill=math.nan)
    check(run(b, device, 3), reference(b), dtype)
    b = make_batch(9, device, (4, 1, 64), [9000, 5001], [70, 3], dtype, code, fill=math.nan)
    check(run(b, device, 0), reference(b), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("qscale", [30.0, 1e-3])
def test_sharp_and_flat_weights(device, dtype, qscale):
    """Scores of hundreds (one key takes all) and of nothing (all alike)."""
    _say(f"qscale {qscale} {dtype}")
    lens = [1, 1, 40]
    b = make_batch(10, device, (8, 4, 128), [900, 130, 300], lens, dtype, torch.int8,
                   qscale=qscale)
    check(run(b, device, 2), reference(b), dtype)


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-30, 7.0])
def test_odd_scales(device, scale):
    _say(f"scale {scale}")
    b = make_batch(11, device, (4, 2, 64), [300, 77], [1, 20], torch.bfloat16, torch.int8)
    b["scale"] = scale
    check(run(b, device, 1), reference(b), torch.bfloat16)


def test_scales_of_unlike_size(device):
    """Cached rows over thirty orders of magnitude, tiny before large and after."""
    _say("unlike scales")
    for flip in (False, True):
        b = make_batch(12, device, (4, 2, 128), [640, 640], [1, 50], torch.bfloat16, torch.int8)
        f = torch.logspace(-25, 5, b["cache"].value_scale.shape[0], device=device)
        b["cache"].value_scale.mul_((f.flip(0) if flip else f)[:, None, None])
        check(run(b, device, 1), reference(b), torch.bfloat16)


@pytest.mark.parametrize("layout", ["tokens", "heads"])
def test_layouts_strides_and_rows_past_the_batch(device, layout):
    """Strided queries and outputs, both cache layouts, rows of no sequence."""
    _say(f"layout {layout}")
    heads = (6, 2, 64)
    lens = [1, 1, 30]
    b = make_batch(13, device, heads, [50, 100, 200], lens, torch.bfloat16, torch.float8_e4m3fn,
                   layout)
    T = 32 + 5                                   # five rows behind the last sequence
    wide = torch.zeros(T, 10, 64, dtype=torch.bfloat16, device=device)
    wide[:32, 2:8] = b["q"].to(device)
    out = torch.full((T, 8, 64), 3.0, dtype=torch.bfloat16, device=device)
    d = lambda t: t.to(device)
    got = ops.paged_attention_quant(wide[:, 2:8], b["cache"], d(b["tables"]), d(b["ctx"]),
                                    scale=b["scale"], cu_seqlens=d(b["cu"]), num_decodes=2,
                                    max_query_len=30, out=out[:, 1:7])
    check(got[:32], reference(b), torch.bfloat16)
    assert bool((out[32:] == 3.0).all()) and bool((out[:, [0, 7]] == 3.0).all())


@pytest.mark.parametrize("code,dtype", [(torch.int8, torch.bfloat16),
                                        (torch.float8_e4m3fn, torch.float16)])
def test_whole_units(device, code, dtype):
    """Many sequences, none long against a workgroup's share: a workgroup takes
    whole units, longest contexts first; few and many rows side by side."""
    _say(f"whole units {code} {dtype}")
    ctx = [2100 + 7 * i if i % 20 == 3 else 850 + i % 60 for i in range(200)]
    lens = [1 + i % 3 for i in range(200)]
    lens[7], lens[23], lens[150] = 130, 128, 129
    b = make_batch(20, device, (2, 2, 64), ctx, lens, dtype, code)
    check(run(b, device, 0), reference(b), dtype)


def pieces_written(call, need):
    """Runs call(workspace) and tells whether any piece of a unit went to the
    workspace (behind its first part, 32 bytes for each of up to 512 ranges)."""
    ws = torch.full((need,), 0x5A, dtype=torch.uint8, device="cuda")
    call(ws)
    return bool((ws[512 * 32:] != 0x5A).any())


@pytest.mark.parametrize("code,dtype", [(torch.int8, torch.bfloat16),
                                        (torch.float8_e4m3fn, torch.float16),
                                        (torch.int8, torch.float32)])
@pytest.mark.parametrize("longest,whole", [(1540, True), (6000, False)])
@pytest.mark.parametrize("n", [200, 300])
def test_units_whole_or_in_pieces(device, code, dtype, longest, whole, n):
    """The two sides of what the kernel finds in the contexts: none is long against
    a workgroup's share, and every unit is one workgroup's (of eight wavefronts for
    16-bit queries), or one is, and units are split.  300 sequences are too many to
    rank."""
    _say(f"units {code} {dtype} {longest} {n}")
    ctx = [1440 + 10 * (i // 20) if i % 20 == 3 else 850 + i % 60 for i in range(n)]
    ctx[43] = longest
    lens = [1 + i % 3 for i in range(n)]
    lens[7], lens[23], lens[150], lens[31] = 130, 128, 129, 0
    heads = (2, 2, 64)
    b = make_batch(20, device, heads, ctx, lens, dtype, code)
    # tables wider than the longest context, as a graph's are
    b["tables"] = torch.nn.functional.pad(b["tables"], (0, 400 - b["tables"].shape[1]))
    need = ops.paged_attention_quant_workspace_size(n, 0, sum(lens), 130, *heads, 400, dtype)
    got = []
    split = pieces_written(lambda ws: got.append(run(b, device, 0, workspace=ws)), need)
    assert split != whole
    check(got[0], reference(b), dtype)


@pytest.mark.parametrize("seqs", [1, 700])
def test_no_blocks(device, seqs):
    """Tables without a column: no sequence has a key, every row is zeros."""
    _say(f"no blocks {seqs}")
    cache = ops.quant_kv_cache(1, BS, 2, 64, torch.int8, device)
    q = torch.ones(seqs, 4, 64, dtype=torch.bfloat16, device=device)
    tables = torch.zeros((seqs, 0), dtype=torch.int32, device=device)
    ctx = torch.full((seqs,), 5, dtype=torch.int32, device=device)
    cu = torch.arange(seqs + 1, dtype=torch.int32, device=device)
    got = ops.paged_attention_quant(q, cache, tables, ctx, scale=1.0, out=torch.ones_like(q))
    assert not got.any()
    mask = torch.ones((seqs, 1), dtype=torch.int64, device=device)
    got = ops.tree_attention_quant(q, cache, tables, ctx, cu, mask, scale=1.0, max_query_len=1,
                                   out=torch.ones_like(q))
    assert not got.any()


def test_block_ids_outside_the_cache(device):
    _say("bad block ids")
    b = make_batch(14, device, (4, 2, 64), [40, 40], [1, 20], torch.bfloat16, torch.int8)
    b["tables"][0, 1] = 10 ** 6
    b["tables"][1, 2] = -3
    ops.device_errors()
    got = run(b, device, 1)
    assert ops.device_errors() == _hip.LV_DEVERR_BLOCK_ID
    b["tables"][0, 1] = b["tables"][1, 2] = 0     # what such an id reads
    check(got, reference(b), torch.bfloat16)


def test_infinite_and_nan_rows_in_view(device):
    """A cached row of NaN makes NaN of the rows that see it, and only of them."""
    _say("nan rows")
    b = make_batch(15, device, (4, 2, 64), [100, 100, 100], [1, 1, 60], torch.bfloat16, torch.int8)
    blk = int(b["tables"][1, 2])
    b["cache"].value_scale[blk, 3, 1] = math.nan  # sequence 1, position 35, kv head 1
    blk = int(b["tables"][2, 5])
    b["cache"].key_scale[blk, 4, 0] = math.nan    # sequence 2, position 84: rows 44.. see it
    got = run(b, device, 2).float().cpu()
    nan = torch.isnan(got).all(-1)
    want = torch.zeros_like(nan)
    want[1, 2:] = True
    want[2 + 44:, :2] = True
    assert torch.equal(nan, want) and torch.equal(torch.isnan(got).any(-1), want)


def test_cache_past_32_bit_offsets(device):
    """Blocks whose codes lie past 2^32 bytes and whose scales past 2^31 ones."""
    _say("large cache")
    hkv, d = 8, 128
    n = (1 << 32) // (BS * hkv * d) + 40
    cache = ops.quant_kv_cache(n, BS, hkv, d, torch.int8, device)
    g = torch.Generator().manual_seed(16)
    ctx = [100, 37]
    tables = torch.tensor([[n - 1 - i for i in range(7)], [n - 20 - i for i in range(7)]],
                          dtype=torch.int32)
    b = dict(tables=tables, ctx=torch.tensor(ctx, dtype=torch.int32), lens=[1, 21],
             cu=torch.tensor([0, 1, 22], dtype=torch.int32), scale=0.1, heads=(16, 8, 128),
             q=torch.randn(22, 16, 128, generator=g).bfloat16(), cache=cache)
    slots = (tables.long()[..., None] * BS + torch.arange(BS)).reshape(-1)
    k, v = rows(g, slots.numel(), hkv, d), rows(g, slots.numel(), hkv, d)
    ops.kv_scatter_quant(k.to(device), v.to(device), cache, slots.to(device))
    got = run(b, device, 1)
    back = [t.double().cpu() for t in ops.kv_gather_quant(cache, slots.to(device), torch.float32)]
    for x, y in zip((k, v), back):
        assert torch.equal(y.float(), oq.values(x, torch.int8).float())
    outs = []
    for i, n_rows in enumerate(b["lens"]):
        kk, vv = (oq.values(x, torch.int8).view(2, -1, hkv, d)[i, :ctx[i]] for x in (k, v))
        sees = np.tril(np.ones((n_rows, ctx[i]), bool), ctx[i] - n_rows)
        q = b["q"][int(b["cu"][i]):int(b["cu"][i + 1])]
        outs.append(oq.attention(q, kk, vv, sees, 0.1))
    check(got, [torch.cat(x) for x in zip(*outs)], torch.bfloat16)


@torch.inference_mode()
def test_streams_and_graphs(device):
    """On another stream; and two captured graphs replayed in turn with eager
    work between, each owning its workspace."""
    _say("streams and graphs")
    heads = (16, 8, 128)
    a = make_batch(17, device, heads, [3000, 40, 800, 1], [1] * 4, torch.bfloat16, torch.int8)
    c = make_batch(18, device, heads, [2500, 900], [100, 33], torch.float16, torch.float8_e4m3fn)
    ref = [reference(a), reference(c)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(a, device, 4)
    torch.cuda.current_stream().wait_stream(side)
    check(got, ref[0], torch.bfloat16)
    graphs, outs, inputs = [], [], []
    for b, nd in ((a, 4), (c, 0)):
        d = {k: v.to(device) for k, v in b.items() if torch.is_tensor(v)}
        H, hkv, D = heads
        ws = torch.empty(max(256, ops.paged_attention_quant_workspace_size(
            len(b["lens"]), nd, b["q"].shape[0], max(b["lens"]), H, hkv, D, d["tables"].shape[1],
            b["q"].dtype)), dtype=torch.uint8, device=device)
        out = torch.empty_like(d["q"])
        call = lambda: ops.paged_attention_quant(
            d["q"], b["cache"], d["tables"], d["ctx"], scale=b["scale"], cu_seqlens=d["cu"],
            num_decodes=nd, max_query_len=max(b["lens"]), out=out, workspace=ws)
        call()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            call()
        graphs.append(graph)
        outs.append(out)
        inputs.append((d, ws))
    for _ in range(3):
        for graph, out in zip(graphs, outs):
            out.zero_()
            graph.replay()
            run(a, device, 4)
        torch.cuda.synchronize()
        check(outs[0], ref[0], torch.bfloat16)
        check(outs[1], ref[1], torch.float16)


def test_same_call_same_bits(device):
    _say("repeatable")
    b = make_batch(19, device, (16, 2, 128), [5000, 700, 300], [1, 1, 90], torch.bfloat16,
                   torch.int8)
    first = run(b, device, 2)
    for _ in range(3):
        assert same(run(b, device, 2), first)


@pytest.mark.parametrize("heads,dtype,width", [
    ((16, 8, 128), torch.bfloat16, 6),        # a wavefront a kv head, the largest stages
    ((4, 2, 64), torch.float16, 6),
    ((8, 8, 128), torch.float32, 6),          # 32-row tiles
    ((40, 1, 128), torch.bfloat16, 130)])     # tiles of two stages and eight wavefronts
def test_many_decode_rows(device, heads, dtype, width):
    """More decode rows than a launch takes, whose offsets would not fit the LDS
    beside the tiles; other sequences behind them."""
    _say(f"many decode rows {heads} {dtype} {width}")
    H, Hkv, D = heads
    n, pool = 8300, 64
    g = torch.Generator().manual_seed(21)
    cache = ops.quant_kv_cache(pool, BS, Hkv, D, torch.int8, device)
    k, v = rows(g, pool * BS, Hkv, D), rows(g, pool * BS, Hkv, D)
    ops.kv_scatter_quant(k.to(device), v.to(device), cache, torch.arange(pool * BS, device=device))
    edges = [0, 1, 4094, 4095, 4096, 4097, 8190, 8191, 8192, 8193, n - 2, n - 1]
    ctx = torch.randint(0, 33, (n,), generator=g, dtype=torch.int32)       # one tile
    ctx[edges] = 16 * width - 3 if width < 100 else 700
    lens = [1] * n
    lens[n - 1] = 9
    tables = torch.randint(0, pool, (n, width), generator=g, dtype=torch.int32)
    b = dict(cache=cache, tables=tables, ctx=ctx, lens=lens, scale=1 / math.sqrt(D), heads=heads,
             cu=torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32),
             q=torch.randn(n + 8, H, D, generator=g).to(dtype))
    got = run(b, device, n - 1)
    some = edges
    at = [r for i in some for r in range(int(b["cu"][i]), int(b["cu"][i + 1]))]
    part = dict(b, tables=tables[some], ctx=ctx[some], lens=[lens[i] for i in some], q=b["q"][at])
    part["cu"] = torch.tensor([0] + list(np.cumsum(part["lens"])), dtype=torch.int32)
    check(got[at], reference(part), dtype)
    # the others, of up to two blocks, side by side
    kv = cache_values(cache)
    for lo in range(0, n - 1, 1000):
        i = torch.tensor([i for i in range(lo, min(lo + 1000, n)) if i not in edges])
        kk, vv = (x[tables[i, :2].long()].reshape(len(i), 2 * BS, Hkv, D).transpose(1, 2) for x in kv)
        q = b["q"][i].double().view(len(i), Hkv, H // Hkv, D)
        sees = (torch.arange(2 * BS) < ctx[i, None])[:, None, None]        # [n, 1, 1, keys]
        x = (q @ kk.transpose(2, 3) * b["scale"]).masked_fill(~sees, -math.inf)
        w = torch.nan_to_num(torch.softmax(x, -1))                         # no key: zeros
        shown = vv.abs() * sees[:, 0, 0, None, :, None]
        reach = (b["scale"] * (q.abs() @ kk.abs().transpose(2, 3)) * sees).amax(-1)
        floor = (ctx[i, None] * shown.amax((2, 3)))[..., None].expand_as(reach)
        ref = [t.reshape(len(i), H, -1) for t in (w @ vv, w @ vv.abs())] \
            + [t.reshape(len(i), H) for t in (reach, floor)]
        check(got[i.to(device)], ref, dtype)

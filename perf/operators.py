"""Operators on an 8-bit paged K/V cache and on trees of drafted tokens, as measurable cases.

Kinds of case (``case["kind"]``):

* ``write``: K and V rows quantised into the paged cache at their slots and
  read back from there (a step's new tokens; rows swapped out again).
* ``prologue``: the attention prologue of one layer -- per-head RMSNorm (or
  none), rotary embedding, the query written out, K and V quantised into the
  cache -- and the new rows read back.
* ``attend``: one paged-attention call over the 8-bit cache for a step's
  decode rows (one query row per sequence), prompt chunks, or both.
* ``tree``: one attention call for the rows of drafted token trees (each row
  sees its sequence's cached prefix and its own ancestors), over a cache in
  the element type or in 8 bits.

A cached row is the D values of one token and kv head.  It is held as D codes
(whole numbers in [-127, 127], or e4m3 values) and one fp32 scale: the row's
largest magnitude over the code's largest, so value = code * scale.

Context, chunk and tree sizes are spread evenly over a case's range, so its
work does not depend on the seed; their order, the block tables and every
value do.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

BS = 16
MAX_POS = 40960
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"int8": (torch.int8, 127.0), "fp8": (torch.float8_e4m3fn, 448.0)}


# -- cases ---------------------------------------------------------------------

def _write(name, hkv, d, tokens, run, dtype, code):
    return dict(name=name, kind="write", Hkv=hkv, D=d, tokens=tokens, run=run, dtype=dtype,
                code=code)


def _prologue(name, heads, tokens, run, norm, dtype, code):
    h, hkv, d = heads
    return dict(name=name, kind="prologue", H=h, Hkv=hkv, D=d, tokens=tokens, run=run, norm=norm,
                dtype=dtype, code=code)


def _attend(name, heads, rows, lo, hi, dtype, code, chunks=0, len_lo=1, len_hi=1, off_lo=0,
            off_hi=0):
    h, hkv, d = heads
    return dict(name=name, kind="attend", H=h, Hkv=hkv, D=d, rows=rows, lo=lo, hi=hi,
                chunks=chunks, len_lo=len_lo, len_hi=len_hi, off_lo=off_lo, off_hi=off_hi,
                dtype=dtype, code=code)


def _tree(name, heads, trees, nodes_lo, nodes_hi, off_lo, off_hi, dtype, code):
    h, hkv, d = heads
    return dict(name=name, kind="tree", H=h, Hkv=hkv, D=d, chunks=trees, len_lo=nodes_lo,
                len_hi=nodes_hi, off_lo=off_lo, off_hi=off_hi, dtype=dtype, code=code)


def listed():
    return [
        # a decode step's new rows, one token per sequence
        _write("write_decode", 8, 128, 61, 1, "bf16", "int8"),
        # a whole step of prompt chunks under the 8192-token budget
        _write("write_chunks", 8, 128, 7872, 512, "bf16", "fp8"),
        # one layer's prologue of a 256-row decode step (Qwen3-0.6B heads)
        _prologue("prologue_decode", (16, 8, 128), 256, 1, True, "bf16", "int8"),
        # prompt chunks of a wide grouped-query model without q/k norms
        _prologue("prologue_chunks", (32, 8, 128), 4099, 500, False, "fp16", "fp8"),
        # interactive serving: a few short contexts
        _attend("decode_few", (32, 4, 64), 3, 40, 300, "fp16", "int8"),
        # a full decode batch (Qwen3-0.6B heads)
        _attend("decode_batch", (16, 8, 128), 256, 16, 2048, "bf16", "int8"),
        # few very long contexts: the keys of a row split over the chip
        _attend("decode_long", (32, 8, 128), 2, 60000, 131000, "bf16", "fp8"),
        # the mixed step: decode rows and prompt chunks in one call
        _attend("mixed_step", (16, 8, 128), 192, 256, 4096, "bf16", "int8", 15, 512, 512, 0,
                3071),
        # late chunks of long prompts, eight query heads to a kv head
        _attend("chunks_long", (16, 2, 128), 0, 0, 0, "fp16", "fp8", 2, 700, 1024, 15000, 19000),
        # speculative decoding for two users: small trees, short contexts
        _tree("tree_few", (16, 8, 128), 2, 7, 13, 200, 700, "bf16", "none"),
        # a batch of 64-node trees over the 16-bit cache
        _tree("tree_batch", (16, 8, 128), 48, 40, 64, 500, 4000, "bf16", "none"),
        # trees over the 8-bit cache, long contexts
        _tree("tree_codes", (32, 8, 128), 16, 25, 60, 2000, 16000, "fp16", "int8"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    half = rng.choice(["bf16", "fp16"])
    code = rng.choice(["int8", "fp8"])
    hkv, g, d = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    heads = (hkv * g, hkv, d)
    kind = rng.choice(["write", "prologue", "decode", "chunks", "mixed", "tree", "tree"])
    if kind == "write":
        return _write("", hkv, d, _log(rng, 1, 16000), rng.choice([1, 1, 100, 512]), dtype, code)
    if kind == "prologue":
        return _prologue("", heads, _log(rng, 1, 8000), rng.choice([1, 1, 100, 512]),
                         rng.random() < 0.5, half, code)
    hi = _log(rng, 30, 60000)
    lo = _log(rng, max(1, hi // 30), hi)
    if kind == "tree":
        n = _log(rng, 1, 100)
        return _tree("", heads, _log(rng, 1, 64), rng.randint(1, n), n, lo, hi, dtype,
                     rng.choice(["none", code]))
    rows = _log(rng, 1, 300) if kind != "chunks" else 0
    if kind == "decode":
        return _attend("", heads, rows, lo, hi, dtype, code)
    n = _log(rng, 2, 1500)
    chi = _log(rng, 30, 20000)
    return _attend("", heads, rows, lo, hi, dtype, code, _log(rng, 1, 16), rng.randint(1, n), n,
                   rng.randint(0, chi), chi)


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 3e14)


def _plain_bytes(case):
    """About what the plain form holds at once."""
    if case["kind"] in ("write", "prologue"):
        return 40 * case["tokens"] * case["D"] * (case["Hkv"] + case.get("H", 0))
    total = 0
    for seqs in _groups(case):
        if seqs:
            keys, q = max(c for c, _ in seqs), max(q for _, q in seqs)
            total = max(total, len(seqs) * keys * (20 * case["Hkv"] * case["D"]
                                                   + 20 * case["H"] * q))
    return total


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= most and _plain_bytes(case) <= 24e9:
            case.pop("name")
            return case


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _groups(case):
    """(context, query rows) of the decode sequences and of the others."""
    decodes = [(c, 1) for c in _spread(case["lo"], case["hi"], case["rows"])] \
        if case.get("rows") else []
    lens = _spread(case["len_lo"], case["len_hi"], case["chunks"])
    offs = _spread(case["off_lo"], case["off_hi"], case["chunks"])
    # long and short ones meet long and short offsets
    others = [(o + q, q) for o, q in zip(offs[::2] + offs[1::2], lens)]
    return decodes, others


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    hkv, d = case["Hkv"], case["D"]
    row = hkv * (d * es if case.get("code") == "none" else d + 4)      # cached K (or V) of a token
    if case["kind"] in ("write", "prologue"):
        t, h = case["tokens"], case.get("H", 0)
        rows = 2 * t * hkv * d * es                                    # K and V
        return {"bytes": 2 * rows + 2 * t * row + 2 * t * h * d * es + 16 * t
                + (t * d * es if h else 0),
                "flops": 6 * t * (h + 2 * hkv) * d}
    decodes, others = _groups(case)
    seqs = decodes + others
    rows = sum(q for _, q in seqs)
    pairs = sum(c for c, _ in decodes)
    if case["kind"] == "tree":   # the draft keys a row sees depend on the tree: the prefix alone
        pairs = sum(q * (c - q) for c, q in others)
    else:
        pairs += sum(q * (c - q) + q * (q + 1) // 2 for c, q in others)
    keys = sum(c for c, _ in seqs)
    return {"bytes": 2 * keys * row + 2 * rows * case["H"] * d * es + 4 * (keys // BS),
            "flops": 4 * pairs * case["H"] * d}


# -- inputs ----------------------------------------------------------------------

def _rows(gen, t, heads, d, dev):
    """K or V rows of t tokens: heads of unlike size, a few wide channels."""
    x = torch.randn(t, heads, d, generator=gen, device=dev)
    wide = 1 + 5 * (torch.rand(heads, d, generator=gen, device=dev) < 0.04)
    return x * wide * (0.5 + torch.rand(heads, 1, generator=gen, device=dev))


def _empty_cache(blocks, hkv, d, code, dev):
    """Key and value codes [blocks, BS, Hkv, D] and scales [blocks, BS, Hkv],
    each head's rows of a block in one run of memory."""
    ct = CODES[code][0]
    made = []
    for _ in range(2):
        made.append(torch.zeros(blocks, hkv, BS, d, dtype=torch.uint8, device=dev).view(ct)
                    .transpose(1, 2))
    for _ in range(2):
        made.append(torch.zeros(blocks, hkv, BS, device=dev).transpose(1, 2))
    return made


def _quantise(x, code):
    """Codes and scales of fp32 rows x[..., D]."""
    ct, top = CODES[code]
    top = torch.full((), top, device=x.device)
    scale = x.abs().amax(dim=-1) / top
    y = x / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    y = y.clamp(-top, top)
    return (y.round() if code == "int8" else y).to(ct), scale


def _slots(case, gen, rng, dev):
    """Distinct cache slots of the tokens, in runs of consecutive ones."""
    t, run = case["tokens"], case["run"]
    per = -(-(run + BS - 1) // BS)                   # blocks of a run at any first offset
    runs = -(-t // run)
    blocks = runs * per + 3
    order = torch.randperm(blocks, generator=gen, device=dev)[:runs * per].view(runs, per)
    first = torch.randint(0, BS, (runs, 1), generator=gen, device=dev)
    pos = first + torch.arange(run, device=dev)
    slots = torch.gather(order, 1, pos // BS) * BS + pos % BS
    return slots.reshape(-1)[:t].contiguous(), blocks


def _tree_masks(rng, nodes):
    """Rows of ancestor bits (each node's own among them), 64 to a word."""
    words = -(-max(nodes) // 64)
    rows = []
    for n in nodes:
        seen = []
        for j in range(n):
            up = rng.choice([-1, j - 1, rng.randrange(-1, j)]) if j else -1
            seen.append((seen[up] if up >= 0 else 0) | 1 << j)
        rows += seen
    signed = [[w - (w >> 63 << 64) for w in ((r >> 64 * k) & (1 << 64) - 1 for k in range(words))]
              for r in rows]
    return torch.tensor(signed, dtype=torch.int64)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    dtype, hkv, d = DTYPES[case["dtype"]], case["Hkv"], case["D"]
    s = dict(case=case, dtype=dtype)
    if case["kind"] in ("write", "prologue"):
        t = case["tokens"]
        s["slots"], blocks = _slots(case, gen, rng, dev)
        s["cache"] = _empty_cache(blocks, hkv, d, case["code"], dev)
        if case["kind"] == "write":
            s["key"] = _rows(gen, t, hkv, d, dev).to(dtype)
            s["value"] = _rows(gen, t, hkv, d, dev).to(dtype)
            return s
        s["qkv"] = _rows(gen, t, case["H"] + 2 * hkv, d, dev).to(dtype).view(t, -1)
        s["positions"] = torch.randint(0, MAX_POS, (t,), generator=gen, device=dev)
        freq = 1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=dev) / d)
        angle = torch.arange(MAX_POS, dtype=torch.float64, device=dev)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
        s["q_weight"] = s["k_weight"] = None
        if case["norm"]:
            w = 1 + 0.2 * torch.randn(2, d, generator=gen, device=dev)
            s["q_weight"], s["k_weight"] = w[0].to(dtype), w[1].to(dtype)
        return s
    decodes, others = _groups(case)
    rng.shuffle(decodes)
    rng.shuffle(others)
    seqs = decodes + others
    n_blocks = [-(-c // BS) for c, _ in seqs]
    pool = sum(n_blocks) + 5
    ids = torch.randperm(pool, generator=gen, device=dev).to(torch.int32)
    tables = torch.zeros(len(seqs), max(n_blocks), dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(n_blocks):
        tables[i, :n] = ids[at:at + n]
        at += n
    rows = sum(q for _, q in seqs)
    cu = [0]
    for _, q in seqs:
        cu.append(cu[-1] + q)
    s.update(tables=tables, ctx=torch.tensor([c for c, _ in seqs], dtype=torch.int32, device=dev),
             cu=torch.tensor(cu, dtype=torch.int32, device=dev), num_decodes=len(decodes),
             num_seqs=len(seqs), max_query=max(q for _, q in seqs),
             widths=[max([c for c, _ in g], default=0) for g in (decodes, others)],
             queries=[max([q for _, q in g], default=0) for g in (decodes, others)],
             scale=1 / math.sqrt(d))
    s["query"] = torch.randn(rows, case["H"], d, generator=gen, device=dev).to(dtype)
    if case["kind"] == "tree":
        s["mask"] = _tree_masks(rng, [q for _, q in seqs]).to(dev)
    if case["code"] == "none":
        s["cache"] = [_rows(gen, pool * BS, hkv, d, dev).to(dtype).view(pool, BS, hkv, d)
                      for _ in range(2)]
        return s
    s["cache"] = _empty_cache(pool, hkv, d, case["code"], dev)
    for k in range(2):
        codes, scale = _quantise(_rows(gen, pool * BS, hkv, d, dev).to(dtype).float(),
                                 case["code"])
        s["cache"][k].view(torch.uint8).copy_(codes.view(torch.uint8).view(pool, BS, hkv, d))
        s["cache"][2 + k].copy_(scale.view(pool, BS, hkv))
    return s


# -- the plain forms ---------------------------------------------------------------

def _put(cache, slots, key, value, code):
    """Quantise fp32 rows into the cache at their slots."""
    blk, off = slots // BS, slots % BS
    for k, x in enumerate((key, value)):
        codes, scale = _quantise(x, code)
        cache[k].view(torch.uint8)[blk, off] = codes.view(torch.uint8)
        cache[2 + k][blk, off] = scale


def _get(cache, slots):
    """fp32 values of the cached K and V rows at the slots."""
    blk, off = slots // BS, slots % BS
    return [cache[k].view(torch.uint8)[blk, off].view(cache[k].dtype).float()
            * cache[2 + k][blk, off][..., None] for k in range(2)]


def _read_back(s):
    return [x.to(s["dtype"]) for x in _get(s["cache"], s["slots"])]


def _plain_prologue(s):
    case = s["case"]
    h, hkv, d = case["H"], case["Hkv"], case["D"]
    x = s["qkv"].float().view(-1, h + 2 * hkv, d)
    q, k, v = x[:, :h], x[:, h:h + hkv], x[:, h + hkv:]
    if s["q_weight"] is not None:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["q_weight"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["k_weight"].float()
    cos = s["cos"][s["positions"]].float()[:, None]
    sin = s["sin"][s["positions"]].float()[:, None]
    q1, q2, k1, k2 = (*q.chunk(2, -1), *k.chunk(2, -1))
    q = torch.cat([q1 * cos - q2 * sin, q2 * cos + q1 * sin], -1)
    k = torch.cat([k1 * cos - k2 * sin, k2 * cos + k1 * sin], -1)
    _put(s["cache"], s["slots"], k, v, case["code"])
    return [q.to(s["dtype"])] + _read_back(s)


def _cached(s, k, tables):
    """fp32 rows [sequences, Hkv, keys, D] of the tables' blocks."""
    cache = s["cache"]
    if s["case"]["code"] == "none":
        x = cache[k][tables].float()
    else:
        x = cache[k].view(torch.uint8)[tables].view(cache[k].dtype).float()
        x = x * cache[2 + k][tables][..., None]
    n, blocks, _, hkv, d = x.shape
    return x.reshape(n, blocks * BS, hkv, d).transpose(1, 2).contiguous()


def _plain_attend(s, out, first, count, width, rows):
    """Rows of the sequences first .. first + count into out; width: their
    longest context, rows: their most query rows."""
    case = s["case"]
    h, hkv, d = case["H"], case["Hkv"], case["D"]
    dev = out.device
    tables = s["tables"][first:first + count, :-(-width // BS)].long()
    ctx = s["ctx"][first:first + count].long()
    cu = s["cu"].long()[first:first + count + 1]
    n_rows = cu[1:] - cu[:-1]
    j = torch.arange(rows, device=dev)
    real = j < n_rows[:, None]                                             # [n, rows]
    at = torch.where(real, cu[:-1, None] + j, cu[:-1, None])
    q = s["query"][at].float().view(count, rows, hkv, h // hkv, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(count, hkv, -1, d)
    keys = _cached(s, 0, tables)
    x = torch.matmul(q, keys.transpose(2, 3).contiguous()) * s["scale"]
    del keys
    pos = torch.arange(x.shape[-1], device=dev)
    if case["kind"] == "tree":
        drafted = pos - (ctx - n_rows)[:, None]                            # [n, keys]
        word = (drafted.clamp(0) // 64).clamp(max=s["mask"].shape[1] - 1)
        bits = torch.gather(s["mask"][at], 2, word[:, None].expand(-1, rows, -1))
        sees = (drafted < 0)[:, None] | ((bits >> (drafted % 64)[:, None]) & 1 == 1)
        sees = sees & (pos < ctx[:, None])[:, None]
    else:
        sees = pos <= (ctx - n_rows)[:, None, None] + j[:, None]           # [n, rows, keys]
    x = x.view(count, hkv, rows, h // hkv, -1)
    x = x.masked_fill(~sees[:, None, :, None], -torch.inf)
    x = x - x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    x = x.exp()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(count, hkv, -1, x.shape[-1]), _cached(s, 1, tables))
    o = o.view(count, hkv, rows, h // hkv, d) / torch.where(total > 0, total,
                                                            torch.ones_like(total))
    o = o.permute(0, 2, 1, 3, 4).reshape(count, rows, h, d)
    out[at[real]] = o[real].to(out.dtype)


def _plain(s):
    case = s["case"]
    if case["kind"] == "write":
        _put(s["cache"], s["slots"], s["key"].float(), s["value"].float(), case["code"])
        return _read_back(s)
    if case["kind"] == "prologue":
        return _plain_prologue(s)
    out = torch.empty_like(s["query"])
    nd = s["num_decodes"]
    if nd:
        _plain_attend(s, out, 0, nd, s["widths"][0], 1)
    if s["num_seqs"] > nd:
        _plain_attend(s, out, nd, s["num_seqs"] - nd, s["widths"][1], s["queries"][1])
    return out


# -- one pass ------------------------------------------------------------------------

def _ops():
    package = str(Path(__file__).resolve().parent.parent / "lite-vllm_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from litevllm import ops
    return ops


def _own(s):
    ops = _ops()
    case = s["case"]
    if case["code"] != "none":
        cache = ops.QuantKV(*s["cache"])
    if case["kind"] == "write":
        ops.kv_scatter_quant(s["key"], s["value"], cache, s["slots"])
        return list(ops.kv_gather_quant(cache, s["slots"], s["dtype"]))
    if case["kind"] == "prologue":
        q = ops.qk_norm_rope_cache_quant(
            s["qkv"], case["H"], case["Hkv"], case["D"], s["cos"], s["sin"], s["positions"],
            s["slots"], cache, s["q_weight"], s["k_weight"], eps=1e-6)
        return [q, *ops.kv_gather_quant(cache, s["slots"], s["dtype"])]
    if case["kind"] == "tree":
        if case["code"] == "none":
            return ops.tree_attention(s["query"], *s["cache"], s["tables"], s["ctx"], s["cu"],
                                      s["mask"], scale=s["scale"], max_query_len=s["max_query"])
        return ops.tree_attention_quant(s["query"], cache, s["tables"], s["ctx"], s["cu"],
                                        s["mask"], scale=s["scale"],
                                        max_query_len=s["max_query"])
    return ops.paged_attention_quant(s["query"], cache, s["tables"], s["ctx"], scale=s["scale"],
                                     cu_seqlens=s["cu"], num_decodes=s["num_decodes"],
                                     max_query_len=s["max_query"])


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# -- the definitions in 64 bits ----------------------------------------------------------

def _exact_row_values(x, code, dtype):
    """What rows x read back as.  The scale and x / scale are fp32 values by
    definition, so both are rounded to it."""
    top = CODES[code][1]
    scale = (x.abs().amax(-1, keepdim=True) / top).float().double()
    y = torch.where(scale > 0, x / scale, torch.zeros_like(x)).float().double()
    if code == "int8":
        y = y.round().clamp(-top, top)
    else:   # e4m3: 3 fraction bits, smallest exponent -6
        _, e = torch.frexp(y)
        step = torch.exp2(torch.clamp(e - 1, min=-6).double() - 3)
        y = (torch.round(y / step) * step).clamp(-top, top)
    return y * scale


def _exact_prologue(s):
    case = s["case"]
    h, hkv, d = case["H"], case["Hkv"], case["D"]
    x = s["qkv"].double().view(-1, h + 2 * hkv, d)
    parts = []
    for lo, hi, w in ((0, h, s["q_weight"]), (h, h + hkv, s["k_weight"])):
        y = x[:, lo:hi]
        if w is not None:
            y = y / ((y ** 2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * w.double()
        c = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, None]
        z = torch.complex(y[..., :d // 2].contiguous(), y[..., d // 2:].contiguous()) * c
        parts.append(torch.cat([z.real, z.imag], -1))
    return [parts[0]] + [_exact_row_values(r, case["code"], s["dtype"])
                         for r in (parts[1], x[:, h + hkv:])]


def _exact_attention(s):
    case = s["case"]
    h, hkv, d = case["H"], case["Hkv"], case["D"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=s["query"].device)
    ctx, cu = s["ctx"].tolist(), s["cu"].tolist()
    for i, c in enumerate(ctx):
        n = cu[i + 1] - cu[i]
        blocks = s["tables"][i, :-(-c // BS)].long()
        kv = []
        for k in range(2):
            if case["code"] == "none":
                x = s["cache"][k][blocks].double()
            else:
                codes = s["cache"][k].view(torch.uint8)[blocks].view(s["cache"][k].dtype)
                x = codes.float().double() * s["cache"][2 + k][blocks].double()[..., None]
            kv.append(x.reshape(-1, hkv, d)[:c])
        sees = torch.ones(n, c, dtype=torch.bool, device=out.device)
        if case["kind"] == "tree":
            m = s["mask"][cu[i]:cu[i + 1]].cpu().numpy().view("uint8")
            bits = torch.from_numpy(m).to(out.device)[:, :, None] >> torch.arange(
                8, dtype=torch.uint8, device=out.device)
            sees[:, c - n:] = (bits & 1).reshape(n, -1)[:, :n].bool()
        else:
            sees = sees.tril(c - n)
        for g in range(hkv):
            q = s["query"][cu[i]:cu[i + 1], g * (h // hkv):(g + 1) * (h // hkv)].double()
            x = (q.reshape(-1, d) @ kv[0][:, g].T.contiguous()).view(n, h // hkv, c) * s["scale"]
            p = torch.softmax(x.masked_fill(~sees[:, None], -math.inf), -1)
            o = p.view(-1, c) @ kv[1][:, g].contiguous()
            out[cu[i]:cu[i + 1], g * (h // hkv):(g + 1) * (h // hkv)] = o.view(n, h // hkv, d)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "write":
        return [_exact_row_values(s[k].double(), case["code"], s["dtype"])
                for k in ("key", "value")]
    if case["kind"] == "prologue":
        return _exact_prologue(s)
    if work(case)["flops"] > 4e12:
        return None
    return _exact_attention(s)

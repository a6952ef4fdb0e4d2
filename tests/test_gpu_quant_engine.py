"""The engine on an 8-bit cache, and a model's forward over drafted trees."""

from __future__ import annotations

import types

import pytest
import torch

from litevllm import LLM, SamplingParams, ops
from litevllm.layers.attention import Attention, AttentionMetadata, PagedAttention
from oracle import quant as oq
from oracle.model import OracleDecoder

pytestmark = pytest.mark.gpu

TINY = dict(model_type="llama", vocab_size=1000, hidden_size=128, num_hidden_layers=2,
            num_attention_heads=4, num_key_value_heads=2, head_dim=64, intermediate_size=256,
            max_position_embeddings=512)
TINY_QWEN = dict(TINY, model_type="qwen3", num_attention_heads=8, head_dim=128)


def _say(msg):
    print(f"[case] {msg}", flush=True)


class QuantisedKV(list):
    """A decoder's K/V list whose rows go through the 8-bit cache's rounding."""

    def __init__(self, code):
        super().__init__()
        self.code = code

    def _rounded(self, x, done=0):
        return torch.cat([x[:done], oq.values(x[done:], self.code).float()])

    def append(self, kv):
        super().append(tuple(self._rounded(x) for x in kv))

    def __setitem__(self, i, kv):
        done = self[i][0].shape[0]
        super().__setitem__(i, tuple(self._rounded(x, done) for x in kv))


def greedy(oracle, prompt, n, code):
    kv = QuantisedKV(code)
    logits = oracle.forward(prompt, 0, kv)
    out = []
    for i in range(n):
        top = torch.topk(logits, 2)
        out.append((int(logits.argmax()), float(top.values[0] - top.values[1])))
        logits = oracle.forward([out[-1][0]], len(prompt) + i, kv)
    return out


@pytest.mark.parametrize("code", ["int8", "fp8"])
@pytest.mark.parametrize("cfg,eager,prefix", [(TINY, True, False), (TINY, False, True),
                                              (TINY_QWEN, False, False)])
def test_engine_against_oracle(device, code, cfg, eager, prefix):
    """Greedy tokens of an fp32 model: chunked prompts, decode graphs and shared
    prefix blocks, against a decoder whose K/V take the same rounding.  (A code
    next to a tie may fall to either side: a step of it moves a logit by far less
    than the margin asked for.)"""
    _say(f"engine {code} {cfg['model_type']} eager={eager} prefix={prefix}")
    llm = LLM("tiny", dtype="float32", load_format="dummy", hf_overrides=cfg,
              skip_tokenizer_init=True, num_gpu_blocks=64, kv_cache_dtype=code, chunk_size=16,
              max_num_seqs=8, enforce_eager=eager, enable_prefix_caching=prefix)
    g = torch.Generator().manual_seed(3)
    shared = torch.randint(0, 1000, (33,), generator=g).tolist()
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (7, 1, 40)]
    prompts += [shared + [5], shared + [9, 8]]
    kv = llm.engine.model_runner.kv_cache
    assert isinstance(kv.get_kv(0), ops.QuantKV)
    assert kv.storage.dtype == ops.QUANT_DTYPES[code]
    params = SamplingParams(temperature=0.0, max_tokens=10, ignore_eos=True)
    outs = llm.generate(prompt_token_ids=prompts, sampling_params=params)
    if prefix:       # again, over cached blocks
        outs = llm.generate(prompt_token_ids=prompts, sampling_params=params)
    oracle = OracleDecoder(llm.engine.model_runner.model.state_dict(),
                           llm.engine.config.model_config,
                           use_qk_norm=cfg["model_type"] == "qwen3")
    compared = 0
    for o in outs:
        for got, (want, margin) in zip(o.output_token_ids,
                                       greedy(oracle, list(o.prompt_token_ids), 10,
                                              ops.QUANT_DTYPES[code])):
            if margin < 2e-3:
                break
            assert got == want, (o.prompt_token_ids[:4], o.output_token_ids)
            compared += 1
    assert compared >= 20


def test_engine_bf16_runs(device):
    """A bf16 model runs over every cache type, decode graphs on."""
    _say("engine bf16")
    prompts = [[3, 1, 4, 1, 5, 9, 2, 6] * 8, [2, 7, 1, 8]]
    for code in ("auto", "int8", "fp8"):
        llm = LLM("tiny", dtype="bfloat16", load_format="dummy", hf_overrides=TINY_QWEN,
                  skip_tokenizer_init=True, num_gpu_blocks=64, kv_cache_dtype=code,
                  max_num_seqs=4)
        o = llm.generate(prompt_token_ids=prompts,
                         sampling_params=SamplingParams(temperature=0.0, max_tokens=8,
                                                        ignore_eos=True))
        assert all(len(x.output_token_ids) == 8 for x in o) and len(o) == 2
    ops.check_device_errors()


def _runner(cfg, dtype, code):
    llm = LLM("tiny", dtype=dtype, load_format="dummy", hf_overrides=cfg, skip_tokenizer_init=True,
              num_gpu_blocks=64, kv_cache_dtype=code, enforce_eager=True)
    return llm.engine.model_runner


def _forward(runner, device, tokens, positions, slots, table, ctx, mask=None):
    i32 = dict(dtype=torch.int32, device=device)
    n = len(tokens)
    meta = AttentionMetadata(block_tables=torch.tensor([table], **i32),
                             context_lens=torch.tensor([ctx], **i32),
                             cu_seqlens=torch.tensor([0, n], **i32), num_decodes=0,
                             max_query_len=n, tree_mask=mask)
    kv = [runner.kv_cache.get_kv(i) for i in range(runner.kv_cache.num_layers)]
    with torch.inference_mode():
        return runner.model(torch.tensor(tokens, device=device),
                            torch.tensor(positions, device=device), kv,
                            slot_mapping=torch.tensor(slots, device=device), is_prefill=True,
                            attn_metadata=meta).float().cpu()


@pytest.mark.parametrize("code", ["auto", "int8", "fp8"])
@pytest.mark.parametrize("dtype,tol", [("float32", 2e-3), ("bfloat16", 6e-2)])
def test_tree_forward_equals_each_path(device, code, dtype, tol):
    """One forward over a drafted tree gives every node the logits of its own
    path fed as a plain chunk.  (fp32: rows in other batches round otherwise in
    their last bits, which may move a code by a step; bf16: every layer's
    roundings.)"""
    _say(f"tree forward {code} {dtype}")
    runner = _runner(TINY_QWEN, dtype, code)
    g = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, 1000, (37,), generator=g).tolist()
    parents = [-1, 0, 0, 1, 1, 2, -1, 6, 3]
    drafted = torch.randint(0, 1000, (len(parents),), generator=g).tolist()
    depth = []
    for p in parents:
        depth.append(depth[p] + 1 if p >= 0 else 0)
    n, table = len(prompt), [7, 3, 9, 12]
    slot = lambda p, t: t[p // 16] * 16 + p % 16
    _forward(runner, device, prompt, range(n), [slot(p, table) for p in range(n)], table, n)
    mask = ops.tree_mask(torch.tensor(parents, dtype=torch.int32, device=device),
                         torch.tensor([0, len(parents)], dtype=torch.int32, device=device),
                         len(parents))
    got = _forward(runner, device, drafted, [n + d for d in depth],
                   [slot(n + j, table) for j in range(len(drafted))], table, n + len(drafted),
                   mask)
    other = [20, 21, 22, 23]
    for j in range(len(parents)):
        path, at = [], j
        while at >= 0:
            path.insert(0, drafted[at])
            at = parents[at]
        seq = prompt + path
        want = _forward(runner, device, seq, range(len(seq)),
                        [slot(p, other) for p in range(len(seq))], other, len(seq))[-1]
        err = (got[j] - want).norm() / want.norm()
        assert err < tol, (j, float(err))
    ops.check_device_errors()


def test_attention_layer_paths(device):
    """Attention.forward with an 8-bit cache in place of the key cache: scatter
    and decode through the reference signature."""
    _say("Attention.forward over QuantKV")
    g = torch.Generator().manual_seed(2)
    attn = Attention(4, 64, 2)
    cache = ops.quant_kv_cache(8, 16, 2, 64, torch.int8, device)
    k, v = (torch.randn(20, 2, 64, generator=g).to(device) for _ in range(2))
    slots = torch.arange(48, 68, device=device)
    q = torch.randn(20, 4, 64, generator=g).to(device)
    out = attn(q, k, v, cache, None, None, slots, None, is_prefill=True)   # its own K and V
    assert torch.isfinite(out).all()
    back = ops.kv_gather_quant(cache, slots, torch.float32)
    for x, y in zip((k, v), back):
        assert torch.equal(y.cpu(), oq.values(x, torch.int8).float())
    table = torch.tensor([[3, 4]], dtype=torch.int32, device=device)
    ctx = torch.tensor([20], dtype=torch.int32, device=device)
    got = attn(q[:1], None, None, cache, None, table, None, ctx, is_prefill=False)
    want = ops.paged_attention_quant(q[:1], cache, table, ctx, scale=attn.scale)
    assert torch.equal(got, want)
    PagedAttention.write_to_cache(k[:2] * 2, v[:2], cache, None, slots[:2])
    assert torch.equal(ops.kv_gather_quant(cache, slots[:2], torch.float32)[0].cpu(),
                       oq.values(k[:2] * 2, torch.int8).float())


def test_native_and_python_paths_agree(device, monkeypatch):
    """The wrappers' own Python path gives the native path's bits."""
    _say("native against python")
    from test_gpu_quant_cache import make_batch
    from test_gpu_tree_attention import make_trees
    b = make_batch(41, device, (8, 2, 64), [300, 40, 90], [1, 1, 30], torch.bfloat16, torch.int8)
    t = make_trees(42, device, (8, 2, 64), [100, 9], [12, 40], torch.bfloat16)
    c = make_trees(43, device, (8, 2, 64), [100, 9], [12, 40], torch.float16, torch.float8_e4m3fn)
    d = lambda x: x.to(device)
    qkv = torch.randn(9, 12 * 64, device=device)
    cos = torch.randn(50, 32, device=device)

    def calls():
        cache = ops.quant_kv_cache(4, 16, 2, 64, torch.int8, device)
        slots = torch.arange(9, device=device) * 5
        x = qkv.view(9, 12, 64)
        ops.kv_scatter_quant(x[:, 8:10], x[:, 10:], cache, slots)
        out = list(ops.kv_gather_quant(cache, slots, torch.float16))
        out.append(ops.qk_norm_rope_cache_quant(qkv, 8, 2, 64, cos, cos,
                                                torch.arange(9, device=device), slots + 1, cache,
                                                q_norm_weight=cos[0].repeat(2)))
        out += [cache.key.view(torch.uint8), cache.key_scale]
        out.append(ops.paged_attention_quant(d(b["q"]), b["cache"], d(b["tables"]), d(b["ctx"]),
                                             scale=0.1, cu_seqlens=d(b["cu"]), num_decodes=2,
                                             max_query_len=30))
        for y, op, kv in ((t, ops.tree_attention, t.get("kv")),
                          (c, ops.tree_attention_quant, [c.get("cache")])):
            out.append(op(d(y["q"]), *kv, d(y["tables"]), d(y["ctx"]), d(y["cu"]), d(y["mask"]),
                          scale=0.1, max_query_len=40))
        return out
    native = calls()
    native = calls()                              # the scratch buffer exists now
    names = ("kv_scatter_quant", "kv_gather_quant", "qk_norm_rope_cache_quant",
             "paged_attention_quant", "tree_attention", "tree_attention_quant")
    none = types.SimpleNamespace(**{n: (lambda *a: None) for n in names})
    monkeypatch.setattr(ops, "_native_module", none)
    for x, y in zip(native, calls()):
        assert torch.equal(x, y)


def test_native_calls_serve_plain_arguments(device, monkeypatch):
    """Each wrapper's native call takes the arguments of a serving step itself: it
    returns a result, not None, which hands the call to the Python path."""
    _say("native calls")
    from test_gpu_quant_cache import make_batch
    from test_gpu_tree_attention import make_trees
    b = make_batch(41, device, (8, 2, 64), [300, 40, 90], [1, 1, 30], torch.bfloat16, torch.int8)
    t = make_trees(42, device, (8, 2, 64), [100, 9], [12, 40], torch.bfloat16)
    c = make_trees(43, device, (8, 2, 64), [100, 9], [12, 40], torch.float16, torch.float8_e4m3fn)
    b, t, c = ({k: v.to(device) if torch.is_tensor(v) else v for k, v in x.items()}
               for x in (b, t, c))
    # the stream's scratch buffer, which only the Python path makes
    ops._workspace(torch.device("cuda", torch.cuda.current_device()), 64 << 20)
    native, seen = ops._native_module or ops._native(), []
    names = ("kv_scatter_quant", "kv_gather_quant", "qk_norm_rope_cache_quant",
             "paged_attention_quant", "tree_attention", "tree_attention_quant")

    def watched(name):
        def call(*args):
            result = getattr(native, name)(*args)
            seen.append((name, result is not None))
            return result
        return call
    monkeypatch.setattr(ops, "_native_module",
                        types.SimpleNamespace(**{n: watched(n) for n in names}))
    slots = torch.arange(9, device=device)
    for code in (torch.int8, torch.float8_e4m3fn):
        for dtype in (torch.bfloat16, torch.float16, torch.float32):
            cache = ops.quant_kv_cache(4, 16, 2, 64, code, device)
            qkv = torch.ones(9, 12 * 64, dtype=dtype, device=device)
            x = qkv.view(9, 12, 64)
            cos = torch.ones(50, 32, dtype=dtype, device=device)
            ops.kv_scatter_quant(x[:, 8:10], x[:, 10:], cache, slots)
            ops.kv_gather_quant(cache, slots, dtype)
            ops.qk_norm_rope_cache_quant(qkv, 8, 2, 64, cos, cos, slots, slots, cache)
            ops.qk_norm_rope_cache_quant(qkv, 8, 2, 64, cos, cos, slots, slots, cache,
                                         q_norm_weight=cos.view(-1)[:64],
                                         k_norm_weight=cos.view(-1)[:64], eps=1e-5)
    for decodes, kw in ((2, {}), (0, dict(out=torch.empty_like(b["q"])))):
        ops.paged_attention_quant(b["q"], b["cache"], b["tables"], b["ctx"], scale=0.1,
                                  cu_seqlens=b["cu"], num_decodes=decodes, max_query_len=30, **kw)
    ops.paged_attention_quant(b["q"][:3], b["cache"], b["tables"], b["ctx"], scale=0.1)
    for y, op, kv in ((t, ops.tree_attention, t.get("kv")),
                      (c, ops.tree_attention_quant, [c.get("cache")])):
        op(y["q"], *kv, y["tables"], y["ctx"], y["cu"], y["mask"], scale=0.1, max_query_len=40)
    assert set(n for n, _ in seen) == set(names)
    assert all(served for _, served in seen), [n for n, served in seen if not served]

"""Host side of the 8-bit cache and of tree attention: refusals, sizes, layout
(no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from litevllm import _hip, ops
from litevllm.cache.kv_cache import KVCache
from litevllm.config import CacheConfig
from oracle import quant as oq

P = 0x1000          # pointers that are never dereferenced: the checks come first


def cache(**kw):
    v = dict(key=P, value=P, key_scale=P, value_scale=P, num_blocks=4, stride_block=2 * 16 * 64,
             stride_token=64, stride_head=16 * 64, scale_stride_block=32, scale_stride_token=1,
             scale_stride_head=16, block_size=16, num_kv_heads=2, head_dim=64, code=_hip.LV_INT8)
    v.update(kw)
    return _hip.QuantCache(**v)


def refused(rc, text, code=-1):
    msg = _hip.load().lv_last_error().decode()
    assert rc == code and text in msg, (rc, msg)


@pytest.mark.parametrize("change,text,code", [
    (dict(key=None), "null cache pointer", -1), (dict(value_scale=None), "null cache pointer", -1),
    (dict(code=2), "bad code type", -1), (dict(num_blocks=0), "bad cache geometry", -1),
    (dict(block_size=0), "bad cache geometry", -1), (dict(key=P + 8), "16-byte aligned", -1),
    (dict(key_scale=P + 2), "4-byte aligned", -1), (dict(stride_token=60), "strides", -1),
    (dict(stride_head=72), "strides", -1), (dict(stride_block=-2048), "strides", -1),
    (dict(scale_stride_head=0), "scale strides", -1), (dict(head_dim=32), "head_dim", -4)])
def test_cache_descriptions_are_checked(change, text, code):
    lib = _hip.load()
    c = cache(**change)
    refused(lib.lv_kv_scatter_quant(P, 128, P, 128, c, P, 4, _hip.LV_BF16, None), text, code)
    refused(lib.lv_kv_gather_quant(c, P, 4, P, 128, P, 128, _hip.LV_BF16, None), text, code)
    refused(lib.lv_qk_norm_rope_cache_quant(P, 512, None, None, P, P, 10, P, P, P, 256, c, 4, 4,
                                            1e-6, _hip.LV_BF16, None), text, code)
    if "head_dim" not in text:
        refused(lib.lv_paged_attention_quant(P, 256, c, P, 4, P, P, 2, 0, 4, 4, 4, 0.1, P, 256, P,
                                             1 << 40, _hip.LV_BF16, None), text, code)


def attend(c=None, q=P, qs=256, bt=P, mb=64, cu=P, ctx=P, B=2, nd=0, T=4, mq=4, H=4, out=P, os=256,
           ws=0x10000, wsb=1 << 40, dt=_hip.LV_BF16):
    return _hip.load().lv_paged_attention_quant(q, qs, c or cache(), bt, mb, cu, ctx, B, nd, T, mq,
                                                H, 0.1, out, os, ws, wsb, dt, None)


def test_attention_refusals():
    refused(attend(nd=3), "num_decodes")
    refused(attend(nd=-1), "num_decodes")
    refused(attend(dt=7), "bad dtype")
    refused(attend(H=3), "multiple of num_kv_heads")
    refused(attend(mq=-1), "negative")
    refused(attend(q=None), "null pointer")
    refused(attend(ctx=None), "null pointer")
    refused(attend(bt=None), "null pointer")
    refused(attend(cu=None), "one row")
    refused(attend(qs=200), "token stride")
    refused(attend(q=P + 2), "16-byte aligned")
    refused(attend(os=260), "16-byte aligned")
    refused(attend(mb=1 << 27), "32 bits")
    refused(attend(mb=1 << 26, B=64, cu=P, mq=4000, T=256000), "32-bit offsets")
    refused(attend(c=cache(head_dim=256, stride_token=256, stride_head=4096, stride_block=8192),
                   qs=1024, os=1024), "head_dim", -4)
    refused(attend(c=cache(block_size=32)), "block_size", -4)
    refused(attend(B=20000, T=20000, mq=1), "sequences", -4)
    lib = _hip.load()
    need = lib.lv_paged_attention_quant_workspace_size(2, 0, 4, 4, 4, 2, 64, 64, _hip.LV_BF16)
    assert need > 0 and need % 256 == 0
    refused(attend(wsb=need - 1), "workspace", -3)
    refused(attend(ws=None), "workspace", -3)
    refused(attend(ws=0x10010), "workspace", -3)
    assert attend(B=0, T=0) == 0 and attend(T=0) == 0          # nothing to do


def test_places_of_the_list_fit_32_bits():
    """A launch's tiles are counted in 32 bits, so as many as its own sequences can
    have are refused past them; those of the call's other launches do not count.
    (No workspace: what is accepted ends there.)"""
    wide = cache(num_kv_heads=8, stride_block=8 * 16 * 64, scale_stride_block=8 * 16)
    # one long chunk beside decode rows
    refused(attend(c=wide, qs=4096, os=4096, H=64, mb=8192, B=256, nd=255, T=255 + 8192, mq=8192,
                   wsb=0), "workspace", -3)
    # chunks alone, and decode rows of up to 8 heads a kv head, in tiles of 32 keys
    refused(attend(c=wide, qs=4096, os=4096, H=64, mb=1 << 20, B=256, T=256 * 8192, mq=8192,
                   wsb=0), "32-bit offsets")
    one = cache(num_kv_heads=1, stride_block=16 * 64, scale_stride_block=16)
    many = dict(c=one, qs=64, os=64, H=1, B=4096, nd=4096, T=4096, mq=1, wsb=0)
    refused(attend(mb=1 << 20, **many), "32-bit offsets")
    refused(attend(mb=1 << 19, **many), "workspace", -3)


def test_tree_refusals():
    lib = _hip.load()

    def tree(mask=P, words=1, kc=P, cu=P, T=4, mq=4, nb=4, H=4, D=64, bs=16):
        return lib.lv_tree_attention(P, 256, kc, P, nb, P, 4, cu, P, mask, words, 2, T, mq, H, 2, D,
                                     bs, 0.1, P, 256, 0x10000, 1 << 40, _hip.LV_BF16, None)
    refused(tree(mask=None), "tree_mask")
    refused(tree(mask=P + 4), "tree_mask")
    refused(tree(words=0), "mask_words")
    refused(tree(mq=65), "mask_words")
    refused(tree(kc=None), "cache")
    refused(tree(kc=P + 2), "cache")
    refused(tree(cu=None, T=2), "cu_seqlens")
    refused(tree(nb=0), "cache geometry")
    refused(tree(D=96), "head_dim", -4)
    refused(tree(bs=8), "block_size", -4)
    refused(lib.lv_tree_mask(None, P, 1, 4, P, 1, None), "null")
    refused(lib.lv_tree_mask(P, P, 1, 4, P, 17, None), "mask_words")
    refused(lib.lv_tree_mask(P, P, 1, 4, P, 0, None), "mask_words")
    refused(lib.lv_tree_mask(P, P, -1, 4, P, 1, None), "sizes")
    assert lib.lv_tree_mask(P, P, 1, 0, P, 1, None) == 0


def test_workspace_sizes_are_pure_host():
    lib = _hip.load()
    ws = lib.lv_paged_attention_quant_workspace_size
    big = ws(256, 256, 256, 1, 16, 8, 128, 128, _hip.LV_BF16)
    assert 0 < big < 64 << 20 and big % 256 == 0
    # a batch's need covers its decode rows and its chunks
    both = ws(20, 16, 16 + 4 * 512, 512, 16, 8, 128, 300, _hip.LV_BF16)
    assert both >= ws(16, 16, 16, 1, 16, 8, 128, 300, _hip.LV_BF16)
    assert both >= ws(4, 0, 4 * 512, 512, 16, 8, 128, 300, _hip.LV_BF16)
    assert ws(0, 0, 0, 1, 16, 8, 128, 128, _hip.LV_BF16) == 0
    assert ws(4, 0, 4, 1, 16, 8, 128, 0, _hip.LV_BF16) == 0    # no keys: nothing is split
    tree = lib.lv_tree_attention_workspace_size
    assert tree(4, 64, 16, 16, 8, 128, 100, _hip.LV_F16) % 256 == 0


def test_ops_refuse_cpu_tensors():
    c = ops.quant_kv_cache(4, 16, 2, 64, torch.int8, "cpu")
    k = torch.zeros(3, 2, 64)
    i64 = torch.zeros(3, dtype=torch.int64)
    for call in (lambda: ops.kv_scatter_quant(k, k, c, i64),
                 lambda: ops.kv_gather_quant(c, i64, torch.float32),
                 lambda: ops.paged_attention_quant(k, c, i64[None].int(), i64.int(), scale=1.0),
                 lambda: ops.tree_mask(i64.int(), i64.int(), 3),
                 lambda: ops.tree_attention(k, k, k, i64[None].int(), i64.int(), i64.int(),
                                            i64[:, None], scale=1.0, max_query_len=3)):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()
    with pytest.raises(RuntimeError, match="cache dtype"):
        ops.quant_kv_cache(4, 16, 2, 64, torch.bfloat16, "cpu")


def test_cache_layout():
    """Logical [num_blocks, block_size, num_kv_heads, head_dim], each head's
    rows of a block in one run."""
    c = ops.quant_kv_cache(5, 16, 3, 64, torch.float8_e4m3fn, "cpu")
    assert c.key.shape == c.value.shape == (5, 16, 3, 64)
    assert c.key_scale.shape == c.value_scale.shape == (5, 16, 3)
    assert c.key.stride() == (16 * 3 * 64, 64, 16 * 64, 1) and c.key_scale.stride() == (48, 1, 16)
    kv = KVCache(2, 5, 16, 3, 64, torch.bfloat16, "cpu", kv_cache_dtype="fp8")
    for i in range(2):
        q = kv.get_kv(i)
        assert isinstance(q, ops.QuantKV) and q.key.shape == (5, 16, 3, 64)
        assert q.key.stride() == c.key.stride() and q.key_scale.stride() == c.key_scale.stride()
    per_block = kv.total_bytes // 5
    assert per_block == 2 * 2 * 16 * 3 * 68
    assert KVCache.profile_num_blocks(10 * per_block, 2, 16, 3, 64, torch.bfloat16, "fp8") == 10
    plain = KVCache(2, 5, 16, 3, 64, torch.bfloat16, "cpu")
    assert isinstance(plain.get_kv(1), tuple) and not isinstance(plain.get_kv(1), ops.QuantKV)
    assert KVCache.profile_num_blocks(plain.total_bytes, 2, 16, 3, 64, torch.bfloat16) == 5


def test_config_refuses_other_cache_types():
    assert CacheConfig().kv_cache_dtype == "auto"
    assert CacheConfig(kv_cache_dtype="int8").kv_cache_dtype == "int8"
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        CacheConfig(kv_cache_dtype="int4")


def test_struct_matches_the_header():
    """4 pointers, 7 int64, 4 int32, no padding."""
    assert ctypes.sizeof(_hip.QuantCache) == 4 * 8 + 7 * 8 + 4 * 4


def test_oracle_codes():
    """The oracle's codes against torch's float8 conversion and by hand."""
    g = torch.Generator().manual_seed(0)
    y = (torch.rand(4000, generator=g) * 2 - 1) * 448
    y = torch.cat([y, y / 1000, torch.tensor([0.0, 448.0, -448.0, 2.0 ** -9, 2.0 ** -10,
                                              3 * 2.0 ** -10, 17.0, 19.0])])
    want = y.to(torch.float8_e4m3fn).double()
    assert torch.equal(torch.from_numpy(oq.e4m3(y.double().numpy())), want)
    x = torch.tensor([[1.0, -2.0, 0.5, 127.0], [0, 0, 0, 0], [1.5, 2.5, -0.5, 127]])
    codes, scale = oq.quantise(x, torch.int8)
    assert scale.tolist() == [1.0, 0.0, 1.0]
    assert codes.tolist() == [[1, -2, 0, 127], [0, 0, 0, 0], [2, 2, 0, 127]]
    codes, scale = oq.quantise(torch.tensor([[1.0, float("inf")], [float("nan"), 0]]), torch.int8)
    assert torch.isnan(scale).all() and not codes.any()
    assert oq.ancestors([-1, 0, 5, 1]).tolist() == [[True, False, False, False],
                                                    [True, True, False, False],
                                                    [False, False, True, False],
                                                    [True, True, False, True]]

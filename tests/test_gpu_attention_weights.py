"""How exactly attention over the 8-bit cache and over trees takes its weights:
outputs next to nothing show it where a weight is rounded to 16 bits, and scores
next to nothing leave no other error to hide it."""

from __future__ import annotations

import math

import pytest
import torch

import test_gpu_quant_cache as quant
import test_gpu_tree_attention as trees
from test_gpu_quant_cache import CODES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(16, 8, 128), (8, 1, 128), (4, 2, 64)])
@pytest.mark.parametrize("ctx,lens,decodes", [
    ([9, 30, 100, 250], [1] * 4, 4),                      # few short contexts
    ([12, 700, 33, 5000], [1] * 4, 4),                    # split ones
    ([20, 64, 150, 700], [20, 3, 140, 300], 0),           # chunks
    ([2500, 2600], [30, 290], 0)])                        # behind long contexts
def test_weights_over_codes(device, code, dtype, heads, ctx, lens, decodes):
    print(f"[case] weights {code} {dtype} {heads} {ctx} {lens}", flush=True)
    b = quant.make_batch(51, device, heads, ctx, lens, dtype, code, qscale=2.0 ** -9)
    quant.check(quant.run(b, device, decodes), quant.reference(b), dtype)


@pytest.mark.parametrize("code", [None] + CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(16, 8, 128), (8, 1, 128), (4, 2, 64)])
@pytest.mark.parametrize("offs,nodes", [
    ([0, 3, 40], [9, 13, 5]), ([5, 100, 900], [40, 64, 17]), ([2300, 0], [90, 130])])
def test_weights_of_trees(device, code, dtype, heads, offs, nodes):
    print(f"[case] tree weights {code} {dtype} {heads} {offs} {nodes}", flush=True)
    b = trees.make_trees(52, device, heads, offs, nodes, dtype, code, fill=math.nan)
    b["q"] = b["q"] * 2.0 ** -9
    quant.check(trees.run(b, device), trees.reference(b), dtype)

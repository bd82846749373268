"""DFlashGenerator over a hybrid target with 8-bit attention caches.  A drafter whose
drafts are always rejected: every verify mode keeps one token a block, so what it
generates must not depend on which drafts were rejected."""
from __future__ import annotations

import pytest
import torch

from dflash_mlx import DFlashGenerator
from dflash_mlx import runtime as rt
from tests.kv8_util import DTYPES
from tests.test_gpu_kv8_model import CFG, _model, weights  # noqa: F401

pytestmark = pytest.mark.gpu

PROMPT = torch.randint(0, CFG.vocab_size, (90,), generator=torch.Generator().manual_seed(7), dtype=torch.int32)
N_NEW = 60  # past position 128


class RandomDrafter:
    mask_token_id, target_layer_ids, block_size = 0, [3], 16

    def __init__(self, model, seed):
        self.model, self.gen = model, torch.Generator().manual_seed(seed)

    def make_cache(self):
        return []

    def __call__(self, noise_embedding, target_hidden, cache=None):
        toks = torch.randint(0, CFG.vocab_size, (noise_embedding.shape[1],), generator=self.gen)
        return (self.model.weights.lm_head[toks.to(self.model.device)] * 8)[None]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mode", rt.VERIFY_MODES)
def test_generate(weights, device, dtype, mode):  # noqa: F811
    model = _model(weights, device, dtype)
    runs = []
    for seed in (1, 2):
        res = DFlashGenerator(model, RandomDrafter(model, seed)).generate_from_tokens(
            PROMPT, max_new_tokens=N_NEW, verify_mode=mode, verify_chunk_size=4)
        acc = res.metrics["acceptance_lengths"]
        assert len(res.generated_tokens) == N_NEW
        assert f"3:kv={len(PROMPT) + sum(acc)}" in res.metrics["target_cache_summary"]
        runs.append((acc, res.generated_tokens))
    print(f"[kv8 generate] {dtype} {mode}: accepted {runs[0][0]}", flush=True)
    (a, ta), (b, tb) = runs
    n = next((i for i, (x, y) in enumerate(zip(a, b)) if x != y), min(len(a), len(b)))
    assert n >= 10 and ta[:sum(a[:n])] == tb[:sum(a[:n])]  # up to a draft that happened to be right

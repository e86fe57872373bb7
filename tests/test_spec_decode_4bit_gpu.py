"""Self-speculative decoding with 4-bit weights, dense and with experts: the
feed-forward operators run together on the step's path (CUDA graphs, padded
buckets, prefill chunks), around the same attention.

A step's kernels depend on its row count (few rows keep the unpacked weights
exact, more round them to bf16), as its attention's split does, so outputs are
compared as in the bf16 tests: every emitted token's logit is the maximum of
its teacher-forced row or within GAP_TOL of it."""

import numpy as np
import pytest
import torch

from aspire_b200.spec_decode import DenseModel, ModelConfig, SpecDecoder, synthetic_prompts, token_sha256

pytestmark = pytest.mark.gpu

B, P, G = 5, 300, 24
GAP_TOL = 0.25

CONFIGS = {
    "dense": ModelConfig("dense", 4, 1024, 8, 4, 2816, 4096, 1e6, True),
    "experts": ModelConfig("experts", 4, 1024, 8, 4, 384, 4096, 1e6, True, n_expert=12, top_k=3),
}


@pytest.mark.parametrize("name,group", [("dense", 64), ("dense", 128), ("experts", 32), ("experts", 128)])
def test_speculative_decoding(cuda_device, name, group):
    model = DenseModel(CONFIGS[name], cuda_device, seed=3, weight_bits=4, group=group)
    prompts = synthetic_prompts(B, P, model.cfg.vocab, seed=1)
    dec = SpecDecoder(model, batch=B, prompt_len=P, max_new=G, draft_len=(2, 4), budget_pages=12, recent_pages=4,
                      refresh_layer=-2)
    g0 = dec.prefill(prompts)
    a = dec.generate()
    dec.restart(g0)
    b = dec.generate()
    assert token_sha256(a["tokens"]) == token_sha256(b["tokens"])
    dec.restart(g0)
    dec.use_graphs = False
    assert np.array_equal(a["tokens"], dec.generate()["tokens"]), "CUDA-graph replay differs from eager steps"
    _, gaps = dec.teacher_forced_check(P, a["tokens"])
    assert gaps.max() <= GAP_TOL, float(gaps.max())


def test_weight_options_are_checked(cuda_device):
    with pytest.raises(ValueError):
        DenseModel(CONFIGS["dense"], cuda_device, weight_bits=8)
    with pytest.raises(ValueError):
        DenseModel(CONFIGS["experts"], cuda_device)

"""GPU checks of packed prefill over the forms in which prompts come."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def test_packed_prefill_of_prompts_with_a_leading_dimension(cuda):
    """Prompts as [1, P] tensors: the sequences stand at their P-th position, as for lists."""
    import torch
    from spark_b200.batch import BatchDecodeEngine
    from spark_b200.config import tiny_config
    from spark_b200.model import SyntheticWeights
    cfg = tiny_config(num_layers=1)
    w = SyntheticWeights(cfg, device="cuda", seed=5)
    prompts = [[(37 * i + 11 * b) % cfg.vocab_size for i in range(n)] for b, n in enumerate([30, 3])]
    engines = [BatchDecodeEngine(w, 2, max_seq_len=128, seed=5) for _ in range(2)]
    tokens = [engines[0].prefill(prompts, packed=True),
              engines[1].prefill([torch.tensor([p]) for p in prompts], packed=True)]
    torch.cuda.synchronize()
    assert torch.equal(*tokens) and all(e.pos.tolist() == [30, 3] for e in engines)

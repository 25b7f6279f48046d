"""CPU checks of the prefill entry points: token ids outside the vocabulary are refused before
any device work (looked up on the device they would end the CUDA context)."""
from __future__ import annotations

from types import SimpleNamespace

import pytest


@pytest.fixture
def engine(monkeypatch):
    """What the entry points look at before they touch the device."""
    from spark_b200 import prefill
    from spark_b200.config import tiny_config
    monkeypatch.setattr(prefill, "_projections", lambda *a: pytest.fail("went on to the device"))
    return SimpleNamespace(cfg=tiny_config(), w=None, device="cuda", max_seq_len=64)


@pytest.mark.parametrize("beyond", [-1, 0, 1 << 40])
def test_prefill_refuses_ids_outside_the_vocabulary(engine, beyond):
    import torch
    from spark_b200.prefill import prefill, prefill_packed
    bad = -1 if beyond < 0 else engine.cfg.vocab_size + beyond
    table = torch.zeros((2, 4), dtype=torch.int32)
    for prompts in ([[1, 2], [3, bad]], [torch.tensor([bad]), torch.tensor([5])]):
        with pytest.raises(ValueError, match="vocabulary"):
            prefill_packed(engine, prompts, table)
    for attn in ("sdpa", "paged"):
        with pytest.raises(ValueError, match="vocabulary"):
            prefill(engine, [3, bad], attn=attn)

"""A gradient that cannot be changed in place is refused before anything is, without a GPU (the check of the device left out)."""

from __future__ import annotations

import pytest
import torch

import torchure_amd as ta
from torchure_amd import embed


def test_inference_tensor(monkeypatch):
    monkeypatch.setattr(embed, "_on_gpu", lambda t, who, what: None)
    with torch.inference_mode():
        grad = torch.ones(4, 5)
    with pytest.raises(RuntimeError, match="embedding_grad_: grad is an inference tensor"):
        ta.embedding_grad_(grad, torch.arange(3), torch.ones(3, 5))
    with torch.inference_mode():  # where torch's own in-place operators take it
        assert ta.embedding_grad_(grad, torch.arange(0), torch.ones(0, 5)) is grad

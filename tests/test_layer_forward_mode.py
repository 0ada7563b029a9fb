"""A forward-mode tangent that a call would drop is refused, without a GPU (the check of the device left out)."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import torchure_amd as ta
from torchure_amd import embed


@pytest.mark.parametrize("tokens", [3, 0])
@pytest.mark.parametrize("dual", ["grad", "dy"])
def test_embedding_grad(monkeypatch, dual, tokens):
    monkeypatch.setattr(embed, "_on_gpu", lambda t, who, what: None)
    t = {"grad": torch.ones(4, 5), "dy": torch.ones(tokens, 5)}
    with forward_ad.dual_level():
        t[dual] = forward_ad.make_dual(t[dual], torch.ones_like(t[dual]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ta.embedding_grad_(t["grad"], torch.arange(tokens), t["dy"])

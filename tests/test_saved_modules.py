"""Modules saved whole (not as a state dict) by earlier versions of the package load and run; those of today keep what they have."""
import io

import pytest
import torch


def _reloaded(module):
    buf = io.BytesIO()
    torch.save(module, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)


def _earlier(module, *names):
    """The module without what its class did not have earlier."""
    for name in names:
        for held in (module.__dict__, module._buffers, module._modules, module._parameters):
            held.pop(name, None)
    return module


def test_a_router_without_other_rules(monkeypatch):
    import memory_b200 as M
    r = _reloaded(_earlier(M.ChapterRouter(8, 6, top_k=2), "selection", "by_logits", "last_load", "_last_shared", "balance_bias"))
    assert r.by_logits is False and r.balance_bias is None and r.last_load is None
    with pytest.raises(ValueError, match="CUDA"):
        r(torch.zeros(1, 3, 8))                                  # as far as it goes without a GPU
    with pytest.raises(ValueError, match="no balance bias"):
        r.bfloat16().update_balance()
    assert set(r.state_dict()) == {"router.weight", "router.bias"}


def test_a_block_without_a_norm_behind_it():
    import memory_b200 as M
    b = _reloaded(_earlier(M.MemorySubBlock(64, 1), "post_norm", "gate", "residual_scale"))
    with pytest.raises(ValueError, match="CUDA"):
        b(torch.zeros(1, 3, 64), torch.zeros(1, 4, 64))
    with pytest.raises(ValueError, match="post_norm"):
        b(torch.zeros(1, 3, 64), torch.zeros(1, 4, 64), gate=torch.zeros(1, 64))


def test_modules_of_today_keep_what_they_have():
    import memory_b200 as M
    r = _reloaded(M.ChapterRouter(8, 6, top_k=2, score="sigmoid", balance_bias=True))
    assert r.by_logits and r.selection["score"] == "sigmoid" and r.balance_bias.shape == (6,)
    b = _reloaded(M.MemorySubBlock(64, 1, post_norm=True, gate=True, residual_scale=0.5))
    assert isinstance(b.post_norm, M.RMSNorm) and isinstance(b.gate, torch.nn.Parameter) and b.residual_scale == 0.5
    assert "post_norm" not in b.__dict__ and "gate" not in b.__dict__

"""Attention over a projected-bank cache has no gradients and does not drop them silently."""
import pytest
import torch


@pytest.fixture
def calls(monkeypatch):
    """Cache and arguments on the CPU, and the calls that reach the operator."""
    import memory_b200 as M
    from memory_b200 import _lib as L, ops
    seen = []
    monkeypatch.setattr(L, "require_cuda", lambda *t: None)
    monkeypatch.setattr(ops, "decode_attn_cache", lambda q, *a: (seen.append(q), (q.detach(), None))[1])
    cache = M.ProjectedBankCache.from_rows(torch.zeros(64, 256, dtype=torch.bfloat16), 16)
    return cache, [torch.zeros(2, 1, 128, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3), 2], seen


def test_a_query_that_requires_a_gradient_is_refused(calls):
    cache, args, seen = calls
    args[0].requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradients"):
        cache.attend(*args)
    assert not seen
    with torch.no_grad():
        cache.attend(*args)
    args[0] = args[0].detach()
    cache.attend(*args)
    args[2].requires_grad_(True)               # a router's weights: numbers here
    assert not cache.attend(*args).requires_grad and len(seen) == 3


def test_rows_that_require_a_gradient_are_refused(calls):
    cache, args, _ = calls
    cache.kv_bank.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradients"):
        cache.attend(*args)


def test_forward_mode_gradients_are_refused(calls):
    from torch.autograd import forward_ad
    cache, args, _ = calls
    with forward_ad.dual_level():
        cache.attend(*args)                    # (no tangent among them)
        args[0] = forward_ad.make_dual(args[0], torch.ones_like(args[0]))
        with pytest.raises(RuntimeError, match="no gradients"):
            cache.attend(*args)


@pytest.mark.gpu
def test_a_decoder_with_trained_parameters_decodes():
    import memory_b200 as M
    torch.manual_seed(0)
    router = M.ChapterRouter(128, 9, top_k=3, score="sigmoid", balance_bias=True).cuda()
    bank, wk, wv, wq, wo = (torch.nn.Parameter(torch.randn(*s, device="cuda") * 0.1) for s in ((9 * 16, 128), *[(128, 128)] * 4))
    for dtype in (torch.bfloat16, torch.float8_e4m3fn):
        cache = M.ProjectedBankCache(bank, wk, wv, 16, cache_dtype=dtype)
        dec = M.MemoryDecoder(cache, None, None, wq, wo, num_heads=2, top_k=3, router=router)
        h = torch.randn(2, 1, 128, device="cuda").bfloat16().requires_grad_(True)
        out, _ = dec.step(h, torch.randn(2, 6, 128, device="cuda").bfloat16())
        assert out.isfinite().all() and not out.requires_grad

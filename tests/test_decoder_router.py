"""A decoder that is given a router of the reference's rules decodes by that router."""
import pytest
import torch


def _parts(seed=3):
    import memory_b200 as M
    torch.manual_seed(seed)
    cache = M.ProjectedBankCache(torch.randn(33 * 16, 256, device="cuda") * 0.2, *(torch.randn(256, 256, device="cuda") * 0.1 for _ in range(2)), 16)
    wq, wo = (torch.randn(256, 256, device="cuda") * 0.1 for _ in range(2))
    router = M.ChapterRouter(256, 33, top_k=5).cuda()
    with torch.no_grad():
        router.router.weight.normal_(0, 0.2)
        router.router.bias.normal_(0, 0.1)
    return cache, wq, wo, router


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 4, 20])
def test_its_weights_and_top_k_are_read(batch):
    import memory_b200 as M
    cache, wq, wo, router = _parts()
    own = M.MemoryDecoder(cache, router.router.weight.detach(), router.router.bias.detach(), wq, wo, num_heads=4, top_k=5)
    other = torch.randn(33, 256, device="cuda")                    # what is not to be read
    dec = M.MemoryDecoder(cache, other, None, wq, wo, num_heads=4, top_k=2, router=router)
    h, states = torch.randn(batch, 1, 256, device="cuda").bfloat16(), torch.randn(batch, 6, 256, device="cuda").bfloat16()
    for _ in range(2):
        (out, info), (want, ref) = dec.step(h, states), own.step(h, states)
        assert torch.equal(out, want) and all(torch.equal(info[k], ref[k]) for k in ref)
    router.top_k = own.top_k = 3                                   # a router may be changed between calls
    (out, info), (want, ref) = dec.step(h, states), own.step(h, states)
    assert info["indices"].shape == (batch, 3) and torch.equal(out, want)
    assert not out.requires_grad


def test_routers_of_either_kind_are_kept_without_a_gpu(monkeypatch):
    import memory_b200 as M
    from memory_b200 import ops
    seen = []
    monkeypatch.setattr(ops, "cast", lambda t, dt: t.to(dt))
    monkeypatch.setattr(ops, "decode_step", lambda h, s, w, b, *a, **k: (seen.append((w, b, k["top_k"])), (None,) * 5)[1])
    from types import SimpleNamespace
    cache = SimpleNamespace(kv_bank=torch.zeros(9 * 16, 256), tokens_per_chapter=16)
    router = M.ChapterRouter(128, 9, top_k=4)
    dec = M.MemoryDecoder(cache, torch.zeros(9, 128), None, torch.zeros(128, 128), torch.zeros(128, 128), num_heads=2, top_k=2, router=router)
    dec.step(torch.zeros(1, 1, 128), torch.zeros(1, 3, 128))
    w, b, k = seen[0]
    assert w.data_ptr() == router.router.weight.data_ptr() and b.data_ptr() == router.router.bias.data_ptr() and k == 4

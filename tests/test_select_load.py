"""Counts of the rows that take a chapter: with and without the places that were filled up for want of candidates."""
import pytest
import torch


def _masked(rows, c, seed):
    """Logits with one padding row in four and a masked chapter in seven."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(rows, c, generator=g, device="cuda")
    z[:, 3::7] = float("-inf")
    z[::4] = torch.finfo(torch.float32).min
    return z


@pytest.mark.gpu
@pytest.mark.parametrize("rows, c, k, shared, groups, keep", [
    (1, 33, 4, 1, 1, 1), (3, 40, 40, 0, 1, 1), (64, 65, 8, 1, 8, 2), (50, 700, 12, 0, 1, 1), (700, 2049, 16, 1, 4, 1), (9, 16400, 20, 16, 1, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_places_of_weight_zero_count_only_where_asked(rows, c, k, shared, groups, keep, score):
    import memory_b200 as M
    z = _masked(rows, c, rows).requires_grad_(rows % 2 == 0)
    b = torch.linspace(-0.05, 0.05, c, device="cuda")
    kw = dict(score=score, balance_bias=b, num_shared=shared, num_groups=groups, top_groups=keep)
    every, weighted = M.select_chapters(z, k, **kw), M.select_chapters(z, k, count_filled=False, **kw)
    for a, w in zip(every[:4], weighted[:4]):
        assert torch.equal(a, w)
    assert torch.equal(every.load, torch.bincount(every.indices.flatten(), minlength=c).int())
    live = every.indices[every.weights != 0]
    assert torch.equal(weighted.load, torch.bincount(live, minlength=c).int())
    assert weighted.load.sum() < every.load.sum()


@pytest.mark.gpu
def test_padding_does_not_move_the_balance_bias_of_a_router():
    """Padded rows list the lowest ids with weight 0; those chapters are not crowded."""
    import memory_b200 as M
    r = M.ChapterRouter(16, 24, top_k=4, score="sigmoid", balance_bias=True).cuda()
    z = torch.randn(256, 24, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    real = r.select(z, 0)
    load = r.last_load.clone()
    assert torch.equal(load, real.load)
    padded = torch.cat([z, torch.full((2000, 24), float("-inf"), device="cuda")])
    r.select(padded, 0)
    assert torch.equal(r.last_load, load)
    r.update_balance(0.5)
    assert torch.equal(r.balance_bias, 0.5 * torch.sign(load.double().mean() - load).float())


@pytest.mark.gpu
def test_a_captured_router_counts_anew_at_every_replay():
    import memory_b200 as M
    from memory_b200.graph import GraphedStep
    r = M.ChapterRouter(16, 24, top_k=4, score="sigmoid", balance_bias=True).cuda()
    z = _masked(100, 24, 3)
    graph = GraphedStep(lambda t: r.select(t, 1).load, [z])
    for seed in (4, 5):
        fresh = _masked(100, 24, seed)
        assert torch.equal(graph(fresh), M.select_chapters(fresh, 4, score="sigmoid", num_shared=1, balance_bias=r.balance_bias,
                                                           count_filled=False).load)


def test_the_count_refuses_without_a_gpu():
    from memory_b200 import _lib as L
    for idx, n, c, load in ((None, 4, 8, 4096), (4096, 4, 8, None), (4096, -1, 8, 4096), (4096, 4, 0, 4096), (4096, 4, 40000, 4096)):
        assert L.lib().moc_select_load(idx, None, n, c, load, None) == -1


@pytest.mark.gpu
def test_ids_from_elsewhere_stay_in_bounds():
    """The C entries take ids as they come: those of no chapter are neither counted nor read."""
    from memory_b200 import _lib as L, functional as F, ops
    rows, c, k = 50, 40, 4
    z = torch.randn(rows, c, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    s = L.SelectShape.from_buffer_copy(F._select_image(c, k, "sigmoid", 2, 1.0, 1, None, "max", True))
    s.rows, s.dtype, s.ld = rows, 0, c
    idx, w, _, cw, _, stats = ops.select_fwd(z, None, s, True)
    g = torch.randn_like(w)
    want = ops.select_bwd(z, s, idx, w, cw, stats, g, None)
    bad = idx.clone()
    bad[3, 0], bad[7, 1], bad[9, 2], bad[11, 3] = -1, c, 2 ** 40, 1          # (1 is a shared chapter)
    got = ops.select_bwd(z, s, bad, w, cw, stats, g, None)
    for r, j in ((3, 0), (7, 1), (9, 2), (11, 3)):
        want[r, idx[r, j]] = 0
    assert torch.equal(got, want)
    load = torch.empty(c, dtype=torch.int32, device="cuda")
    ops._issue("select_load", "f32", 1, z.device, (bad.data_ptr(), None, bad.numel(), c, load.data_ptr()))
    good = bad[(bad >= 0) & (bad < c)]
    assert torch.equal(load, torch.bincount(good, minlength=c).int())

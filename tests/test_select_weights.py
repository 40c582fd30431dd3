"""Renormalised weights are quotients: rounded once, not a product with a rounded reciprocal."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("rows, c", [(4000, 64), (3, 300), (2000, 1000), (500, 5000)])
def test_a_single_pick_weighs_one(rows, c, score):
    """w = s / s for k = 1, and 0.5 beside one shared chapter: exact."""
    import memory_b200 as M
    z = torch.randn(rows, c, device="cuda", generator=torch.Generator(device="cuda").manual_seed(c)) * 3
    got = M.select_chapters(z, 1, score=score, num_shared=1)
    assert (got.weights == 1).all() and (got.combined_weights == 0.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows, c, k, shared", [(4000, 64, 8, 0), (4000, 64, 8, 2), (2000, 1000, 31, 0), (300, 700, 100, 1)])
def test_weights_are_the_quotients_of_the_scores(rows, c, k, shared):
    """The same scores without renormalisation, divided by their sum: k - 1 additions of half a step each, one quotient, and the
    product with a scale of 2.5 and a second sum and quotient in the joint list."""
    import memory_b200 as M
    z = torch.randn(rows, c, device="cuda", generator=torch.Generator(device="cuda").manual_seed(k)) * 2
    kw = dict(score="sigmoid", num_shared=shared, routed_scale=2.5)
    s, w = M.select_chapters(z, k, renormalize=False, **kw), M.select_chapters(z, k, **kw)
    mass = s.weights.double().sum(1, keepdim=True)
    u, sums = 2.0 ** -24, 5 + -(-k // 32)                 # additions one after another: a lane's, then five across the warp
    assert ((w.weights.double() * mass / s.weights.double() - 1).abs() <= (sums + 1) * u * 1.001).all()
    if shared:
        joint = w.weights.double() * 2.5
        total = shared + joint.sum(1, keepdim=True)
        assert ((w.combined_weights[:, shared:].double() * total / joint - 1).abs() <= (sums + 4) * u * 1.001).all()

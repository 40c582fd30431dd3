"""Clipping writes tensors in place, and autograd can tell."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["dense", "strided", "twice"])
def test_a_graph_that_saved_a_gradient_refuses_the_clipped_one(layout):
    import memory_b200 as M
    p = torch.nn.Parameter(torch.randn(6, 4, device="cuda"))
    (p ** 3).sum().backward()
    if layout == "strided":
        p.grad = p.grad.t().contiguous().t()
    penalty = (p.grad * p).sum()                      # saves the gradient
    before = p.grad._version
    M.clip_grad_norm_([p, p] if layout == "twice" else [p], 1e-3)
    assert p.grad._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        penalty.backward()


@pytest.mark.gpu
def test_outputs_of_their_own_change_version_and_the_gradients_do_not():
    import memory_b200 as M
    grads, outs = [torch.randn(5, device="cuda") for _ in range(3)], [torch.empty(5, device="cuda") for _ in range(3)]
    M.clip_grad_norm_(grads, 1e-3, out=outs)
    versions = [g._version for g in grads]
    M.clip_grad_norm_(grads, 1e-3, out=outs)
    assert [g._version for g in grads] == versions and all(o._version >= 2 for o in outs)


@pytest.mark.gpu
def test_under_inference_mode():
    import memory_b200 as M
    with torch.inference_mode():
        g = torch.full((4,), 2.0, device="cuda")
        got = M.clip_grad_norm_([g], 1.0)
        assert float(got.total_norm) == 4.0 and torch.allclose(g, torch.full_like(g, 0.5), rtol=1e-6)

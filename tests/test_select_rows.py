"""Numbers of rows at the ends of what a selection takes."""
import pytest
import torch


@pytest.mark.parametrize("shape", [(2 ** 31, 1), (2 ** 32 + 5, 1), (2 ** 20, 2 ** 12, 2)])
def test_rows_that_32_bits_do_not_count_are_refused(shape):
    """The number of rows is 32 bits in the kernels: 2^32 + 5 of them were 5."""
    import memory_b200 as M
    with pytest.raises(ValueError, match="rows in one call"):
        M.select_chapters(torch.empty(shape, device="meta", dtype=torch.bfloat16), 1)
    with pytest.raises(ValueError, match="CUDA"):
        M.select_chapters(torch.empty(2 ** 31 - 1, 1, device="meta"), 1)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 12), (3, 0, 12)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows_give_empty_results_and_empty_gradients(shape, dtype):
    import memory_b200 as M
    z = torch.empty(shape, device="cuda", dtype=dtype, requires_grad=True)
    got = M.select_chapters(z, 4, num_shared=2)
    assert got.indices.shape == got.weights.shape == (*shape[:-1], 4) and got.combined_weights.shape == (*shape[:-1], 6)
    assert got.weights.dtype == torch.float32 and got.load.tolist() == [0] * 12
    for out in (got.weights, got.combined_weights):
        g, = torch.autograd.grad(out.sum(), z, retain_graph=True)
        assert g.shape == z.shape and g.dtype == dtype
    assert not M.select_chapters(z.detach(), 4).weights.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rms", "layernorm"])
@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_a_merge_of_no_rows_gives_every_parameter_a_zero_gradient(kind, types):
    import memory_b200 as M
    x, f = (torch.empty(2, 0, 16, device="cuda", dtype=t, requires_grad=True) for t in types)
    gate, *params = (torch.randn(s, device="cuda").requires_grad_(True) for s in ((2, 16), *[(16,)] * 4))
    w, nw, b, nb = params
    if kind == "rms":
        b = nb = None
    leaves = [t for t in (x, f, gate, w, b, nw, nb) if t is not None]
    y, n = M.gated_residual_norm(x, f, w, b, norm_type=kind, gate=gate, next_weight=nw, next_bias=nb)
    assert y.shape == n.shape == x.shape and (y.dtype, n.dtype) == types
    for out, reached in ((y, [t for t in leaves if t is not nw and t is not nb]), (n, leaves)):
        for t, g in zip(reached, torch.autograd.grad(out.sum(), reached, retain_graph=True)):
            assert g.shape == t.shape and (g == 0).all()

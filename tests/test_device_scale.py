"""Gradient scales of the bank's optimizer step in every form that a number has."""
import pytest
import torch


def _step(scale):
    import memory_b200 as M
    g = torch.Generator(device="cuda").manual_seed(0)
    param = torch.randn(10 * 8, 32, device="cuda", generator=g)
    sink = M.SparseBankGrad()
    sink.add(torch.tensor([2, 5, 7], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda"),
             torch.randn(24, 32, device="cuda", generator=g), 8)
    opt = M.SparseBankAdamW(param, 8, lr=1e-2)
    opt.step(sink, grad_scale=scale)
    assert opt.step_count == 1
    return param, opt.exp_avg, opt.exp_avg_sq


@pytest.mark.gpu
@pytest.mark.parametrize("make", [
    lambda: torch.tensor(0.375, device="cuda", dtype=torch.float64), lambda: torch.tensor(0.375, device="cuda", dtype=torch.bfloat16),
    lambda: torch.tensor([0.375], device="cuda", dtype=torch.float16), lambda: torch.tensor([[0.375]], device="cuda", dtype=torch.bfloat16),
    lambda: torch.tensor(0.375, device="cuda", requires_grad=True), lambda: torch.tensor([0.375], device="cuda"),
    lambda: torch.tensor(0.375, dtype=torch.float64), lambda: torch.tensor([0.375]), lambda: 0.375])
def test_one_number_in_any_type(make):
    """0.375 is exact in every type: the step is that of the plain number."""
    assert all(torch.equal(a, b) for a, b in zip(_step(make()), _step(0.375)))


@pytest.mark.gpu
def test_whole_numbers_scale_too():
    for one in (torch.tensor(2, device="cuda"), torch.tensor(True, device="cuda")):
        assert all(torch.equal(a, b) for a, b in zip(_step(one), _step(float(one))))


@pytest.mark.gpu
def test_more_than_a_number_is_refused_before_the_step_counts():
    import memory_b200 as M
    opt = M.SparseBankAdamW(torch.zeros(16, 32, device="cuda"), 8)
    sink = M.SparseBankGrad()
    sink.add(torch.zeros(1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"), torch.zeros(8, 32, device="cuda"), 8)
    for bad in (torch.ones(2, device="cuda"), torch.ones((), device="cuda", dtype=torch.complex64), torch.ones(0, device="cuda")):
        with pytest.raises(TypeError):
            opt.step(sink, grad_scale=bad)
    assert opt.step_count == 0

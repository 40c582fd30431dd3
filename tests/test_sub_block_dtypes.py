"""MemorySubBlock takes states of the same types with a norm behind the block as without one."""
import pytest
import torch


def _run(dtype, post, next_norm):
    import memory_b200 as M
    torch.manual_seed(0)
    block = M.MemorySubBlock(128, 2, wo_init_zero=False, compute_dtype=torch.bfloat16, post_norm=post, **(dict(gate=True) if post else {})).cuda()
    follow = M.RMSNorm(128).cuda() if next_norm else None
    g = torch.Generator(device="cuda").manual_seed(1)
    x, mem = (torch.randn(2, n, 128, device="cuda", generator=g).bfloat16().to(dtype).requires_grad_(True) for n in (64, 64))      # (bf16 training takes 64 positions at a time)
    got = block(x, mem, next_norm=follow) if next_norm else block(x, mem)
    outs = got if next_norm else (got,)
    weight = [torch.randn(o.shape, device="cuda", generator=g).bfloat16() for o in outs]
    torch.autograd.backward(outs, [w.to(o.dtype) for w, o in zip(weight, outs)])
    return outs, [x.grad, mem.grad] + [p.grad for p in block.parameters()]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
@pytest.mark.parametrize("next_norm", [False, True])
def test_states_of_other_types_pass_a_block_with_post_norm(dtype, next_norm):
    outs, grads = _run(dtype, True, next_norm)
    ref_outs, ref_grads = _run(torch.float32, True, next_norm)
    assert all(o.dtype == dtype for o in outs) and grads[0].dtype == grads[1].dtype == dtype
    # the states are bf16 numbers in every type; the branch leaves in bf16 (2^-8 of its own) instead of fp32, a norm makes it about 1 a
    # column, and y and its gradients carry that, the bf16 arithmetic between them a few such steps
    for got, want in zip([*outs, *grads], [*ref_outs, *ref_grads]):
        got, want = got.double(), want.double()
        assert (got - want).norm() <= 6 * 2.0 ** -8 * want.norm() + 1e-12


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float64, torch.float32, torch.bfloat16])
def test_both_blocks_take_them(dtype):
    for post in (False, True):
        outs, grads = _run(dtype, post, False)
        assert outs[0].dtype == dtype and all(g.isfinite().all() for g in grads)

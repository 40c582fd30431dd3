"""The fp32 sums that selection by softmax forms its keys with: within the bounds that its order rests on."""
import pytest
import torch

U = 2.0 ** -24


def _stats(z, k=8):
    """(largest logit, sum of the exponentials) of every row, as the selection kernels leave them."""
    from memory_b200 import functional as F, ops, _lib as L
    s = L.SelectShape.from_buffer_copy(F._select_image(z.shape[1], k, "softmax", 0, 1.0, 1, None, "max", True))
    s.rows, s.dtype, s.ld = z.shape[0], L.dtype_code(z.dtype), z.shape[1]
    stats = ops.select_fwd(z, torch.zeros(z.shape[1], device="cuda"), s, True)[5]
    return stats[:, 0].double(), stats[:, 1].double()


def _error(z):
    m, total = _stats(z)
    assert torch.equal(m, z.amax(1).double())
    return (total / torch.exp(z.double() - m[:, None]).sum(1) - 1).abs().max()


def _inputs(rows, n, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = torch.arange(n, device="cuda").float()
    each = torch.rand(rows, 1, device="cuda", generator=g)
    return {"normal": torch.randn(rows, n, device="cuda", generator=g) * 3, "rising": (each * 40 * c / n).contiguous(),
            "rising slowly": (each * 0.1 * c / n).contiguous(), "steps": (each * 1.3 * (c // 512)).contiguous(),
            "falling": (-each * 30 * c / n).contiguous(), "far": torch.randn(rows, n, device="cuda", generator=g) + 1e6 * each,
            "one large": torch.where(c == n - 1, 9.0, 0.0).expand(rows, n).contiguous()}


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 700])
@pytest.mark.parametrize("n", [40, 300, 512, 600, 2049, 4096, 8192, 16384])
def test_sums_are_within_their_bound(rows, n):
    """4 u of an exponential, 8 u of arguments, 19 + 4 + 6.5 u of references, 5 u of additions (or 26 of them and no references)."""
    for name, z in _inputs(rows, n).items():
        assert _error(z) <= 46.5 * U, name


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4096, 16384])
def test_rows_that_rise_slowly_do_not_collect_an_error_at_every_step(n):
    """All logits in one interval of whole numbers: no factor but the last, so 4 u of an exponential, 1 u of its argument, 5 u of
    additions, 6.5 u back to the largest logit, 1 u of each number of 32 bits: below 20 u."""
    assert _error(_inputs(2000, n)["rising slowly"].clamp(min=1e-6)) <= 20 * U


@pytest.mark.gpu
@pytest.mark.parametrize("n", [600, 16384])
def test_masked_and_infinite_logits_leave_the_other_rows_sums_alone(n):
    z = _inputs(700, n)["rising"]
    z[3], z[4, 1:], z[5, ::2] = float("-inf"), torch.finfo(torch.float32).min, float("-inf")
    z[6, 7], z[8, 9] = float("nan"), float("inf")
    m, total = _stats(z)
    real = torch.where(z <= torch.finfo(torch.bfloat16).min, float("-inf"), z.double())
    want = torch.exp(real - real.amax(1, keepdim=True)).sum(1)
    assert total[3] == 1 and total[4] == 1 and total[6].isnan() and total[8].isnan()
    rest = torch.ones(700, dtype=torch.bool, device="cuda")
    rest[[3, 6, 8]] = False
    assert ((total / want - 1)[rest].abs() <= 46.5 * U).all()

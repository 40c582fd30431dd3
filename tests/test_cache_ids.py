"""Chapter ids and counts of 64 bits: what 32 do not hold is out of range, not another chapter."""
import pytest
import torch

FAR = [2 ** 32, 2 ** 32 + 1, -(2 ** 32), 2 ** 31, -(2 ** 40) + 2, 2 ** 62, -(2 ** 63), 2 ** 63 - 1]


def test_numbers_are_clamped_not_wrapped():
    from memory_b200.decode import _whole
    got = _whole(torch.tensor(FAR + [5, -1, 2 ** 31 - 1]))
    assert got.dtype == torch.int32 and got.tolist()[8:] == [5, -1, 2 ** 31 - 1]
    assert all(v < 0 or v == 2 ** 31 - 1 for v in got.tolist()[:8])
    for dtype in (torch.int32, torch.int16, torch.uint8):
        t = torch.arange(6, dtype=dtype).view(2, 3).t()
        assert torch.equal(_whole(t), t.int()) and _whole(t).is_contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_ids_that_would_wrap_are_reported_and_left_out(dtype):
    import memory_b200 as M
    g = torch.Generator(device="cuda").manual_seed(0)
    cache = M.ProjectedBankCache.from_rows(torch.randn(10 * 16, 256, generator=g, device="cuda").bfloat16(), 16, cache_dtype=dtype)
    q = torch.randn(1, 1, 128, generator=g, device="cuda").bfloat16()
    w = torch.full((1, 3), 0.5, device="cuda")
    want = cache.attend(q, torch.tensor([[1, 4]], device="cuda"), w[:, :2].contiguous(), 2)
    for far in FAR:
        got = cache.attend(q, torch.tensor([[1, far, 4]], device="cuda"), w, 2)
        with pytest.raises(RuntimeError, match="chapter index"):
            M._lib.check_device_status(q.device)
        assert torch.equal(got, want), far
    # counts beyond 32 bits stand for the whole list, and below for none of it
    idx = torch.tensor([[1, 4]], device="cuda")
    for n, whole in ((2 ** 32 + 1, True), (2 ** 33, True), (-(2 ** 32) + 1, False)):
        got = cache.attend(q, idx, w[:, :2].contiguous(), 2, counts=torch.tensor([n], device="cuda"))
        assert torch.equal(got, want if whole else torch.zeros_like(want)), n
    M._lib.check_device_status(q.device)

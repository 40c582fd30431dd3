"""Attention over the 8-bit cache keeps its probabilities to fp32's bits: values that cancel, and chapters or blocks of rows whose values are
of very different size."""
import pytest
import torch

F8 = torch.float8_e4m3fn


def _definition(q, values, idx, w, heads, kv_heads, chapter):
    """Outputs in 64 bits and the sums of the magnitudes they are made of, both [B, n_q, H * 64]; ``values``: the cache's numbers."""
    b, n_q, _ = q.shape
    t = values.view(-1, chapter, 2, kv_heads, 64)[idx.long()]                      # [B, n, T, 2, HK, 64]
    t = t.flatten(1, 2).repeat_interleave(heads // kv_heads, 3)
    u = w.double().repeat_interleave(chapter, 1)
    s = torch.einsum("bqhd,brhd->bqhr", q.double().view(b, n_q, heads, 64), t[:, :, 0]) * u[:, None, None] / 8
    p = torch.softmax(s, -1) * u[:, None, None]
    return (torch.einsum("bqhr,brhd->bqhd", p, t[:, :, 1]).flatten(2),
            torch.einsum("bqhr,brhd->bqhd", p, t[:, :, 1].abs()).flatten(2))


def _attend(q, values, scales, idx, w, heads, kv_heads, chapter, block):
    import memory_b200 as M
    cache = M.ProjectedBankCache.from_quantized(values, scales, chapter, scale_rows=block)
    out = cache.attend(q, idx, w, heads, kv_heads)
    numbers = values.double() * scales.double().repeat_interleave(block, 0).repeat_interleave(64, 1)
    want, size = _definition(q, numbers, idx, w, heads, kv_heads, chapter)
    return out.double(), want, size


# queries on a KV head: 1, 4 (a column each), 6, 8 (a column each of 8), 9 and 16 (two tiles), 18 (two CTAs)
@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv_heads, n_q", [(2, 2, 1), (8, 2, 1), (12, 4, 2), (8, 1, 1), (9, 3, 3), (8, 1, 2), (6, 1, 3)])
@pytest.mark.parametrize("chapter, block", [(2, 2), (2, 1), (64, 64), (64, 8)])
def test_values_that_cancel(heads, kv_heads, n_q, chapter, block):
    """Rows in pairs with opposite values: what is left is the difference of nearly equal probabilities."""
    g = torch.Generator(device="cuda").manual_seed(heads * 100 + chapter + block)
    chapters, b, n = 40, 32, 2
    rows = torch.randn(chapters * chapter, 2 * kv_heads, 64, generator=g, device="cuda")
    rows[1::2, kv_heads:] = -rows[::2, kv_heads:]
    rows[1::2, :kv_heads] = rows[::2, :kv_heads] * 0.9
    values = (rows * 100).clamp(-448, 448).flatten(1).to(F8)          # (e4m3 has no infinity: past 448 it is NaN)
    scales = torch.full((chapters * chapter // block, 2 * kv_heads), 0.01, device="cuda")
    q = torch.randn(b, n_q, heads * 64, generator=g, device="cuda").bfloat16()
    idx = torch.rand(b, chapters, generator=g, device="cuda").argsort(1)[:, :n].int()
    w = torch.rand(b, n, generator=g, device="cuda") * 0.3
    out, want, size = _attend(q, values, scales, idx, w, heads, kv_heads, chapter, block)
    # |q||k| / 8 u: 64 products of below 10 x 0.3 / 8 in sum, so scores are off by 64 x 2^-23 x 0.4 = 3e-6 at most and probabilities by
    # as much, their two terms by 2^-21, sums of up to 128 of them by a few 2^-24: below 1e-5 of the magnitudes; then bf16's half step
    assert ((out - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * size).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv_heads", [(2, 2), (12, 2), (9, 1)])
@pytest.mark.parametrize("chapter, block", [(64, 64), (64, 16), (32, 8), (40, 8)])
@pytest.mark.parametrize("apart", [2.0 ** 12, 1.3 * 2.0 ** 20])
def test_large_values_of_unlikely_rows_leave_the_others_their_bits(heads, kv_heads, chapter, block, apart):
    """A block of rows with small keys' scores far below the others' and values far above them: the others make the result."""
    g = torch.Generator(device="cuda").manual_seed(int(apart) + chapter)
    chapters, b = 6, 8
    q = torch.randn(b, 1, heads * 64, generator=g, device="cuda").abs().bfloat16()          # (scores have the keys' sign)
    rows = torch.randn(chapters * chapter, 2 * kv_heads, 64, generator=g, device="cuda")
    rows[:, :kv_heads] = rows[:, :kv_heads].abs()
    values = (rows * 100).clamp(-448, 448).flatten(1).to(F8)          # (e4m3 has no infinity: past 448 it is NaN)
    scales = torch.full((chapters * chapter // block, 2 * kv_heads), 0.01, device="cuda")
    per = chapter // block
    scales[per - 1, :kv_heads] = -0.1                                                        # the last block of chapter 0
    scales[per - 1, kv_heads:] = 0.01 * apart
    idx = torch.arange(chapters, device="cuda").expand(b, chapters).int()
    w = torch.full((b, chapters), 1.0, device="cuda")
    out, want, size = _attend(q, values, scales, idx, w, heads, kv_heads, chapter, block)
    # scores up to 60: 64 products of 60 x 8 in sum, off by 64 x 2^-23 x 60 = 4.6e-4; the unlikely rows are e^-60 and less
    assert ((out - want).abs() <= (2.0 ** -8 + 1e-3) * size).all() and size.max() < 10


@pytest.mark.gpu
@pytest.mark.parametrize("apart", [1.1 * 2.0 ** 14, 1.3 * 2.0 ** 20])
def test_chapters_whose_values_differ_in_size(apart):
    """A chapter that weighs 1 / apart in the softmax with values `apart` times the other's: both count the same."""
    import math
    chapters, chapter, b = 2, 32, 16
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.ones(b, 1, 128, device="cuda").bfloat16()
    rows = torch.randn(chapters * chapter, 4, 64, generator=g, device="cuda").abs() + 0.1
    rows[:, :2] = 1.0
    values = (rows * 64).flatten(1).to(F8)
    scales = torch.full((chapters, 4), 1 / 64, device="cuda")
    scales[0, :2] = -math.log(apart) / 8 / 64                 # scores -ln(apart) and 0
    scales[1, :2] = 0.0
    scales[0, 2:] *= apart
    idx = torch.arange(2, device="cuda").expand(b, 2).int()
    w = torch.full((b, 2), 1.0, device="cuda")
    out, want, _ = _attend(q, values, scales, idx, w, 2, 2, chapter, chapter)
    # a score of 14 is off by 64 x 2^-23 x 14 = 1.1e-4 at most
    assert ((out - want).abs() <= (2.0 ** -8 + 3e-4) * want.abs()).all()

"""Selection where little is left to choose from: as many places as candidates, few groups that stay, masks that leave candidates to a
few threads of a row, fewer candidates than places.  And the numbers of rows at which another kernel takes a row."""
import os
import re

import pytest
import torch

from test_select_chapters import _bias, _compare, _logits

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "memory_b200", "csrc", "select.cu")


def _streaming_rows(k):
    """Rows from which a warp streams a row (the kernel's own constants)."""
    few, many = re.search(r"kStreamRows = (\d+), kStreamRowsManyPicks = (\d+);", open(SOURCE).read()).groups()
    return int(few if k <= 32 else many)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("c, k, groups, keep", [
    # as many places as the kept groups have chapters, or one fewer: a warp a row, a CTA a row
    (24, 24, 1, 1), (31, 31, 1, 1), (32, 31, 1, 1), (64, 16, 8, 2), (64, 15, 8, 2), (64, 8, 8, 1), (32, 8, 4, 1), (512, 31, 16, 1), (128, 31, 64, 16),
    (256, 64, 8, 2), (256, 63, 8, 2), (600, 100, 6, 1), (6000, 100, 60, 1), (2048, 128, 16, 1), (16384, 128, 64, 1)])
@pytest.mark.parametrize("top2", [False, True])
def test_as_many_places_as_candidates(c, k, groups, keep, biased, score, top2):
    z, b = _logits(37, c, c + k), _bias(c, c) if biased else None
    _compare(z, b, k, score, 0, groups, keep, top2)


@pytest.mark.gpu
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("c, k, groups", [(24, 24, 1), (64, 16, 8), (300, 31, 1), (256, 64, 8), (700, 40, 1), (4096, 128, 4), (9000, 50, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masks_that_leave_candidates_to_few_threads(c, k, groups, score, biased):
    """Candidates 32, 64 or 256 apart lie with one lane, or one thread, of a row."""
    z, b = _logits(24, c, 7), _bias(c, 3) if biased else None
    dead = torch.ones(24, c, dtype=torch.bool, device="cuda")
    for r, step in enumerate((1, 2, 3, 16, 31, 32, 33, 64, 128, 255, 256, 512)):
        dead[2 * r, r % step::step] = False                       # candidates `step` apart
        dead[2 * r + 1, : min(c, k + r - 5 if k > 5 else r)] = False      # about as many candidates as places, in a row
    z = torch.where(dead, float("-inf"), z)
    for renorm in (True, False):
        _compare(z, b, k, score, 0, groups, max(1, groups // 2), True, renorm)
    if biased:
        off = torch.where(dead[7], float("-inf"), b)              # a bias switches the same chapters off in every row
        _compare(_logits(9, c, 8), off, k, score, 0, 1, 1, True)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("c, k, shared, groups, keep, top2", [
    # k > 32; more than 32 groups; kept groups with few runs of candidates a lane; a bank of 513 to 600
    (514, 64, 1, 1, 1, False), (2049, 64, 1, 8, 3, False), (4097, 64, 1, 1, 1, True), (8200, 33, 8, 32, 7, True), (4097, 48, 1, 8, 2, True),
    (16384, 20, 0, 64, 9, True), (16385, 31, 1, 64, 33, False), (9984, 5, 0, 39, 2, True), (4097, 32, 1, 8, 1, False), (4097, 14, 1, 8, 1, True),
    (4096, 64, 0, 4, 1, False), (2048, 64, 0, 8, 1, True), (2048, 30, 0, 8, 1, False), (600, 40, 0, 2, 1, True)])
def test_rows_on_both_sides_of_the_streaming_kernels_line(c, k, shared, groups, keep, top2, biased, score):
    line = _streaming_rows(k)
    for rows in (line - 1, line, line + 37):
        z, b = _logits(rows, c, c + k), _bias(c, c) if biased else None
        z[5], z[6], z[7, 1:] = float("-inf"), 0.5, torch.finfo(torch.float32).min
        z[8, ::3], z[9, c // 2:], z[10] = float("-inf"), float("-inf"), z[10].bfloat16().float()
        z[11, torch.arange(c, device="cuda") % 512 > 7] = float("-inf")               # few runs with candidates
        z[12, : c - k // 2] = float("-inf")                                           # fewer candidates than places
        _compare(z, b, k, score, shared, groups, keep, top2, grad=rows == line)
        if biased and rows == line:
            _compare(z, torch.zeros(c, device="cuda"), k, score, shared, groups, keep, top2, grad=False)
            _compare(z.bfloat16(), b, k, score, shared, groups, keep, top2, False, grad=False)


@pytest.mark.gpu
def test_a_kernel_before_leaves_nothing_in_shared_memory_that_counts():
    """Columns behind the last chapter have no group: nothing of them is read (rows of NaN first leave NaN on the chip)."""
    import memory_b200 as M
    nan = torch.full((4000, 600), float("nan"), device="cuda")
    for c, k, groups, keep in ((183, 40, 3, 2), (600, 40, 6, 3), (1002, 33, 3, 1), (5000, 40, 50, 7)):
        M.select_chapters(nan, 40)
        for b in (None, _bias(c, 1)):
            _compare(_logits(300, c, c), b, k, "sigmoid", 0, groups, keep, True, grad=False)


def _time(rows, c, k, **kw):
    import memory_b200 as M
    z, b = _logits(rows, c, 1), _bias(c, 2)
    run = lambda: M.select_chapters(z, k, score="sigmoid", balance_bias=b, **kw)      # noqa: E731
    best = float("inf")
    for _ in range(8):
        run()
        torch.cuda._sleep(3_000_000)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(10):
            run()
        end.record()
        end.synchronize()
        best = min(best, start.elapsed_time(end))
    return best


@pytest.mark.gpu
@pytest.mark.parametrize("c, k, other, most, kw", [
    (64, 16, 4, 3, dict(num_groups=8, top_groups=2)), (64, 8, 4, 3, dict(num_groups=8, top_groups=1)), (256, 64, 40, 3, dict(num_groups=8, top_groups=2)),
    (2048, 64, 32, 5, dict(num_groups=8, top_groups=1)), (4096, 32, 8, 5, dict(num_groups=8, top_groups=1))])
def test_full_groups_cost_no_selection_of_another_kind(c, k, other, most, kw):
    """Every row in 64 bits took 4 to 8 times the time of the usual way.  More picks alone make 1.2 to 1.6 times; where they change from
    a warp that streams a row to a CTA a row, whose instructions are three times as many, up to 3 times (4,096 chapters: 36 us and 109)."""
    assert _time(4000, c, k, **kw) <= most * _time(4000, c, other, **kw)

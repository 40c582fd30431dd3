"""clip_grad_norm_ and the optimizer step that takes its coefficient from the device."""
import math

import pytest
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _check(grads, max_norm, banks=(), out=None, eps=1e-6):
    """Clips and compares with the definition in 64 bits."""
    import memory_b200 as M
    before = [g.detach().double().clone() for g in grads]
    total = sum(float((g * g).sum()) for g in before)
    for b in banks:
        for _, count, rows, t in b.entries:
            total += b.scale ** 2 * float((rows[: max(0, min(int(count), rows.shape[0] // t)) * t].double() ** 2).sum())
    got = M.clip_grad_norm_(grads, max_norm, bank_grads=banks, out=out, eps=eps)
    norm = math.sqrt(total)
    coef = min(1.0, max_norm / (norm + eps)) if norm + eps > 0 else float("nan")
    # 64-bit sums, then one rounding to fp32 each
    assert abs(float(got.total_norm) - norm) <= 2.0 ** -24 * norm * 1.001
    assert abs(float(got.coefficient) - coef) <= 2.0 ** -24 * 1.001
    for g, b, o in zip(grads, before, out or grads):
        step = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}[o.dtype]
        want = b * float(got.coefficient)
        # the product rounds to fp32, then to the result's type; fp16 results below 2^-14 are off by half of 2^-24
        assert ((o.double() - want).abs() <= (step + 2.0 ** -24) * want.abs() + (2.0 ** -25 if o.dtype == F16 else 1e-45)).all()
        if out is not None:
            assert torch.equal(g.double(), b)
    return got


def _grads(shapes, dtype, seed=0, std=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(*s, generator=g, device="cuda") * std).to(dtype) for s in shapes]


def _bank(count, spare, t, d, dtype=F32, scale=1.0, seed=1):
    import memory_b200 as M
    rows = _grads([((count + spare) * t, d)], dtype, seed)[0]
    rows[count * t:] = float("nan")                     # behind the count nothing stands
    sink = M.SparseBankGrad()
    sink.add(torch.arange(count + spare, dtype=torch.int32, device="cuda"), torch.full((1,), count, dtype=torch.int32, device="cuda"), rows, t)
    sink.scale = scale
    return sink


SHAPES = [(3, 5), (7,), (1,), (300, 257), (8192,), (8193,), (64, 64), (0, 4), (100000,)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("max_norm", [0.0, 1e-3, 1.0, 1e9, float("inf")])
def test_norm_and_clipping(dtype, max_norm):
    _check(_grads(SHAPES, dtype), max_norm)
    _check(_grads(SHAPES, dtype) + _grads(SHAPES, F32, 3), max_norm, [_bank(3, 2, 16, 33, scale=0.5)])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 64, 65, 680, 681, 1500])
def test_any_number_of_tensors(n):
    _check(_grads([(1 + i % 37,) for i in range(n)], F32), 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("src", [F32, BF16, F16])
@pytest.mark.parametrize("dst", [F32, BF16, F16])
def test_out_of_another_type_at_any_alignment(src, dst):
    shapes = [(5,), (1000,), (33, 17), (9000,), (3,)]
    grads = _grads(shapes, src)
    total = sum(g.numel() for g in grads)
    for shift in (0, 1, 3):
        flat = torch.full((total + shift + 2,), 7.0, dtype=dst, device="cuda")
        out = [p.view(g.shape) for p, g in zip(flat[shift:shift + total].split([g.numel() for g in grads]), grads)]
        _check(grads, 0.7, out=out)
        assert (flat[:shift] == 7).all() and (flat[shift + total:] == 7).all()
    unaligned = [torch.cat([g.flatten()[:1], g.flatten()])[1:].view(g.shape) for g in grads]
    _check(unaligned, 0.7)


@pytest.mark.gpu
def test_bank_gradients():
    import memory_b200 as M
    for count in (0, 1, 5):
        _check([], 0.1, [_bank(count, 3, 16, 64), _bank(2, 0, 8, 12, BF16, 0.25)])
    wrong = _bank(2, 1, 4, 8)
    wrong.entries[0][1].fill_(1000)                     # a count beyond the rows reads what there is
    wrong.entries[0][2].fill_(0.5)
    assert float(M.clip_grad_norm_([], 1.0, bank_grads=[wrong]).total_norm) == pytest.approx(0.5 * math.sqrt(3 * 4 * 8))
    assert float(_check(_grads([(4, 4)], F32), 1.0, [M.SparseBankGrad()]).total_norm) > 0


@pytest.mark.gpu
def test_extremes():
    import memory_b200 as M
    big = [torch.full((100,), 3e30, device="cuda"), torch.full((50,), 1e-30, device="cuda")]      # squares outside of fp32
    assert float(_check(big, 1.0).total_norm) == pytest.approx(3e31, rel=1e-6)
    tiny = [torch.full((100,), 1e-30, device="cuda")]
    assert float(_check(tiny, 1.0).total_norm) == pytest.approx(1e-29, rel=1e-6)
    zero = [torch.zeros(10, device="cuda")]
    assert float(_check(zero, 1.0).coefficient) == 1.0
    for bad, coefficient in ((float("nan"), "nan"), (float("inf"), "0")):
        grads = _grads([(50,), (40,)], F32)
        grads[0][3] = bad
        ref = [g.clone().requires_grad_(True) for g in grads]
        for r, g in zip(ref, grads):
            r.grad = g.clone()
        torch.nn.utils.clip_grad_norm_(ref, 1.0)
        got = M.clip_grad_norm_(grads, 1.0)
        assert math.isnan(float(got.coefficient)) if coefficient == "nan" else float(got.coefficient) == 0.0
        for g, r in zip(grads, ref):
            assert torch.equal(g.isnan(), r.grad.isnan()) and torch.equal(g[~g.isnan()], r.grad[~g.isnan()])


@pytest.mark.gpu
def test_parameters_layouts_and_repeats():
    import memory_b200 as M
    lin = torch.nn.Linear(33, 65).cuda()
    lin(torch.randn(5, 33, device="cuda")).square().sum().backward()
    frozen = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    ref = [p.grad.clone() for p in lin.parameters()]
    got = M.clip_grad_norm_([*lin.parameters(), frozen, lin.weight], 0.5)           # one without a gradient, one twice
    norm = math.sqrt(sum(float((r.double() ** 2).sum()) for r in ref))
    assert float(got.total_norm) == pytest.approx(norm, rel=1e-6)
    for p, r in zip(lin.parameters(), ref):
        assert torch.allclose(p.grad, r * (0.5 / (norm + 1e-6)), rtol=1e-6)
    wide = torch.randn(20, 30, device="cuda")
    keep = wide.clone()
    views = [wide.t()[3:9], torch.randn(4, 6, device="cuda").t()]
    _check(views, 0.1)
    assert torch.equal(wide[:, :3], keep[:, :3]) and torch.equal(wide[:, 9:], keep[:, 9:])
    a, b = _grads(SHAPES, BF16), _grads(SHAPES, BF16)
    ra, rb = M.clip_grad_norm_(a, 1.0), M.clip_grad_norm_(b, 1.0)
    assert torch.equal(ra.total_norm, rb.total_norm) and all(torch.equal(x, y) for x, y in zip(a, b))
    out = [torch.empty(8, 3, device="cuda").t()]
    _check(_grads([(3, 8)], F32), 0.2, out=out)


@pytest.mark.gpu
def test_two_captured_clips_replay_side_by_side():
    import memory_b200 as M
    sets = [_grads([(300, 41), (77,)], F32, s, 1.0) for s in (1, 2)]
    outs = [[torch.empty_like(g) for g in gs] for gs in sets]
    graphs, results = [], []
    for gs, os in zip(sets, outs):
        M.clip_grad_norm_(gs, 1.0, out=os)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(M.clip_grad_norm_(gs, 1.0, out=os))
        graphs.append(graph)
    for gs in sets:
        for g in gs:
            g.mul_(2.0)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for gs, os, r in zip(sets, outs, results):
        norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in gs))
        assert float(r.total_norm) == pytest.approx(norm, rel=1e-6)
        assert all(torch.equal(o, g * r.coefficient) for g, o in zip(gs, os))


@pytest.mark.gpu
def test_bank_step_takes_the_coefficient_from_the_device():
    import memory_b200 as M
    made = []
    for device in (True, False):
        torch.manual_seed(0)
        param = torch.randn(10 * 8, 32, device="cuda")
        sink = _bank(3, 2, 8, 32, scale=0.5)
        sink.entries[0][2][3 * 8:] = 0
        opt = M.SparseBankAdamW(param, 8, lr=1e-2)
        clip = M.clip_grad_norm_([], 0.05, bank_grads=[sink])
        assert float(clip.coefficient) < 0.1
        opt.step(sink, grad_scale=clip.coefficient if device else float(clip.coefficient))
        made.append((param, opt.exp_avg, opt.exp_avg_sq))
    # the scale is one fp32 product of two numbers more on the device: 0.5 is a power of two, so it is the same number
    assert all(torch.equal(a, b) for a, b in zip(*made))
    for bad in (torch.ones(2, device="cuda"), torch.ones(1, device="cuda", dtype=torch.float64)):
        with pytest.raises(TypeError):
            opt.step(sink, grad_scale=bad)


@pytest.mark.gpu
def test_other_types_and_layouts_are_refused():
    import memory_b200 as M
    g = torch.ones(4, 4, device="cuda")
    for grads, out, error in (([g.double()], None, TypeError), ([g], [g.double()], TypeError), ([g.to_sparse()], None, ValueError),
                              ([g, g.cpu()], None, ValueError), ([g], [g[:2]], ValueError), ([g], [g.cpu()], ValueError)):
        with pytest.raises(error):
            M.clip_grad_norm_(grads, 1.0, out=out)
    assert torch.equal(g, torch.ones_like(g))


@pytest.mark.gpu
def test_overlaps_are_refused():
    import memory_b200 as M
    t = torch.zeros(100, device="cuda")
    for grads, out in (([t[:60], t[50:]], None), ([t[:60], t[:30]], None), ([t[:50]], [t[20:70]]), ([t[:10], t[:10]], [t[50:60], t[70:80]]),
                       ([t[:20], t[30:50]], [t[50:70], t[60:80]])):
        with pytest.raises(ValueError):
            M.clip_grad_norm_(grads, 1.0, out=out)
    M.clip_grad_norm_([t[:50], t[50:]], 1.0)
    M.clip_grad_norm_([t[:50]], 1.0, out=[t[50:]])


def test_refusals():
    import memory_b200 as M
    g = torch.zeros(4)
    for kw, error in ((dict(max_norm=-1.0), ValueError), (dict(max_norm=float("nan")), ValueError), (dict(max_norm=1.0, eps=-1.0), ValueError),
                      (dict(max_norm=1.0), ValueError), (dict(max_norm=1.0, out=[]), ValueError)):
        with pytest.raises(error):
            M.clip_grad_norm_([g], **kw)
    with pytest.raises(ValueError, match="no gradients"):
        M.clip_grad_norm_([], 1.0)
    sink = M.SparseBankGrad()
    for _ in range(2):
        sink.add(torch.zeros(1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(4, 4), 4)
    with pytest.raises(NotImplementedError):
        M.clip_grad_norm_([], 1.0, bank_grads=[sink])


def test_c_entry_refuses_without_a_gpu():
    import ctypes as C
    from memory_b200 import _lib as L
    lib = L.lib()
    assert lib.moc_grad_clip_workspace_bytes(-1) == -1
    assert lib.moc_grad_clip_workspace_bytes(0) > 0 and lib.moc_grad_clip_workspace_bytes(681) > lib.moc_grad_clip_workspace_bytes(680) - 1
    p = 4096
    size = lib.moc_grad_clip_workspace_bytes(2)

    def call(count=2, dense=1, grads=(p, p), elems=(4, 8), dtypes=(0, 0), out=(p + 64,), out_dtypes=(0,), counts=(p,), units=(4,), max_norm=1.0,
             result=p, ws=size):
        ptrs, sizes, types = C.c_void_p * 2, C.c_int64 * 2, C.c_uint8 * 2
        return lib.moc_grad_clip(count, dense, ptrs(*grads), sizes(*elems), types(*dtypes), ptrs(*out), types(*out_dtypes), ptrs(*counts),
                                 (C.c_int32 * 2)(*units), (C.c_float * 2)(1.0), max_norm, 1e-6, result, p, ws, None)
    for change in (dict(count=-1), dict(dense=3), dict(dense=-1), dict(grads=(None, p)), dict(elems=(-1, 8)), dict(dtypes=(7, 0)), dict(dtypes=(0, 3)),
                   dict(out_dtypes=(3,)), dict(grads=(p + 2, p)), dict(out=(p + 3,)), dict(out=(p,), out_dtypes=(1,)), dict(counts=(None,)),
                   dict(units=(0,)), dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(result=None), dict(ws=size - 1),
                   dict(out=(p + 8,)), dict(out=(p,))):
        assert call(**change) == -1, change

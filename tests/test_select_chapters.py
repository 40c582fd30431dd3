"""Selection of chapters from logits: scores, balance bias, groups, order and gradients against plain forms in 64 bits, and what is
refused."""
import pytest
import torch

LOWEST = torch.finfo(torch.bfloat16).min
U32 = 2.0 ** -24          # half a step of fp32


def _plain(z, k, score, bias, shared, scale, groups, keep, top2, renorm):
    """The definition in 64 bits: (idx, weights, joint idx, joint weights, load), differentiable in z."""
    c = z.shape[1]
    n = c - shared
    t = z.double()[:, shared:]
    dead = t <= LOWEST
    t = torch.where(dead, torch.zeros_like(t), t)
    if score == "sigmoid":
        s = torch.sigmoid(t)
    else:
        top = torch.where(dead, torch.full_like(t, LOWEST), t).amax(1, keepdim=True).detach()
        e = torch.where(dead, torch.zeros_like(t), torch.exp(t - top))
        s = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    s = torch.where(dead, torch.zeros_like(s), s)
    none = float("-inf")
    sel = s.detach() + bias.double()[shared:] if bias is not None else t.detach()
    sel = torch.where(dead, none, sel)
    if keep < groups:
        judge = s.detach() if bias is None and top2 else sel
        best = torch.where(dead, none, judge).view(-1, groups, n // groups).sort(dim=2, descending=True).values
        value = best[:, :, 0]
        if top2 and n // groups > 1:
            value = value + torch.where(best[:, :, 1] == none, 0.0, best[:, :, 1])
        order = value.sort(dim=1, descending=True, stable=True).indices[:, :keep]
        stays = torch.zeros_like(value, dtype=torch.bool).scatter_(1, order, True)
        sel = torch.where(stays.repeat_interleave(n // groups, 1), sel, none)
    got, local = sel.sort(dim=1, descending=True, stable=True)
    got, local = got[:, :k], local[:, :k]
    w = torch.where(got == none, 0.0, s.gather(1, local))
    if renorm:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-12)
    idx = local + shared
    joint_idx, joint = idx, w
    if shared:
        lead = torch.arange(shared, device=z.device).expand(z.shape[0], -1)
        joint_idx, joint = torch.cat([lead, idx], 1), torch.cat([torch.ones_like(lead, dtype=w.dtype), scale * w], 1)
        joint = joint / joint.sum(1, keepdim=True)
    return idx, w, joint_idx.int(), joint, torch.bincount(idx.flatten(), minlength=c).int()


def _compare(z, bias, k, score="softmax", shared=0, groups=1, keep=None, top2=False, renorm=True, grad=True):
    import memory_b200 as M
    keep = groups if keep is None else keep
    z = z.detach().requires_grad_(grad)
    got = M.select_chapters(z, k, score=score, balance_bias=bias, num_shared=shared, routed_scale=2.5, num_groups=groups,
                            top_groups=keep, group_score="top2" if top2 else "max", renormalize=renorm)
    zr = z.detach().double().requires_grad_(grad)
    idx, w, joint_idx, joint, load = _plain(zr, k, score, bias, shared, 2.5, groups, keep, top2, renorm)
    assert torch.equal(got.indices, idx) and torch.equal(got.combined_indices, joint_idx) and torch.equal(got.load, load)
    # A score is off by the exponential (2 ulp of 2 U), its argument's rounding (|z - m| U, up to 16 here), the sum (a tree over
    # at most 64 terms a thread and 10 levels: 74 U) and quotients: below 128 U relative; the renormalised sums add as much again.
    tol = 256 * U32
    assert torch.allclose(got.weights.double(), w, rtol=tol, atol=1e-30)
    assert torch.allclose(got.combined_weights.double(), joint, rtol=tol, atol=1e-30)
    if not grad:
        return got
    g = torch.Generator(device=z.device).manual_seed(1)
    gw, gj = (torch.randn(t.shape, generator=g, device=z.device) for t in (got.weights, got.combined_weights))
    d, = torch.autograd.grad([got.weights, got.combined_weights], [z], [gw, gj])
    dr, = torch.autograd.grad([w, joint], [zr], [gw.double(), gj.double()])
    assert d.dtype == z.dtype
    # d_z = p (ds - lean): each factor within `tol` of its own size, differences of terms of the row's largest; bf16 rounds once more
    row = dr.abs().amax(1, keepdim=True) + 4 * gw.abs().amax() * w.detach().amax(1, keepdim=True)
    step = 2.0 ** -8 if z.dtype == torch.bfloat16 else 0.0
    assert ((d.double() - dr).abs() <= 4 * tol * row + step * dr.abs()).all()
    assert (d[:, :shared] == 0).all()
    return got


def _logits(rows, c, seed, dtype=torch.float32, std=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, c, generator=g, device="cuda") * std).to(dtype)


def _bias(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-60, 61, (c,), generator=g, device="cuda").float() * 0.001


CASES = [
    # rows, chapters, k, shared, groups, keep, top2
    (1, 5, 1, 0, 1, 1, False), (3, 33, 33, 0, 1, 1, False), (7, 65, 4, 1, 1, 1, False), (130, 129, 8, 1, 8, 3, True),
    (64, 257, 8, 1, 8, 4, True), (33, 512, 32, 0, 16, 2, False), (9, 152, 7, 2, 3, 1, True), (17, 513, 16, 1, 64, 5, False),
    (5, 120, 40, 0, 1, 1, False), (21, 1002, 3, 2, 4, 2, True), (19, 2050, 50, 2, 4, 3, True), (11, 4097, 64, 1, 1, 1, False),
    (40, 4097, 16, 1, 8, 4, True), (3, 8193, 128, 1, 2, 1, False), (2, 16384, 100, 0, 64, 9, True), (4, 600, 6, 0, 600 // 10, 7, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("rows, c, k, shared, groups, keep, top2", CASES)
def test_selection_and_gradient(rows, c, k, shared, groups, keep, top2, biased, score):
    z, b = _logits(rows, c, c + k), _bias(c, c) if biased else None
    for renorm in (True, False):
        _compare(z, b, k, score, shared, groups, keep, top2, renorm)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("c, k, shared, groups, keep, top2", [
    (513, 1, 0, 1, 1, False), (514, 64, 1, 1, 1, False), (1026, 16, 2, 4, 2, True), (2049, 64, 1, 8, 3, False), (2050, 8, 1, 1, 1, False),
    (4097, 16, 1, 8, 4, True), (4097, 64, 1, 1, 1, False), (4100, 5, 3, 17, 2, True), (8200, 33, 8, 32, 7, True), (16385, 64, 1, 64, 9, True),
    (16384, 20, 0, 1, 1, False), (700, 31, 0, 2, 1, True)])
def test_many_rows(c, k, shared, groups, keep, top2, biased, score):
    """Numbers of rows at which a warp takes a row of a large bank, some of them masked, equal, or with one candidate."""
    rows = 613
    z, b = _logits(rows, c, c + k), _bias(c, c) if biased else None
    z[5], z[6], z[7, 1:] = float("-inf"), 0.5, torch.finfo(torch.float32).min
    z[8, ::3] = float("-inf")
    z[9, c // 2:] = float("-inf")
    z[10] = z[10].bfloat16().float()
    _compare(z, b, k, score, shared, groups, keep, top2)
    _compare(z.bfloat16(), b, k, score, shared, groups, keep, top2, False, grad=False)
    if biased:
        _compare(z, torch.zeros(c, device="cuda"), k, score, shared, groups, keep, top2, grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("c, k, groups, keep", [(65, 8, 1, 1), (257, 8, 8, 4), (4097, 16, 8, 4), (4097, 64, 1, 1)])
def test_bf16_logits_with_ties(c, k, groups, keep):
    """bf16 logits hold equal values, so the order among them is that of the ids; the bias makes near ties that only 64 bits part."""
    z = _logits(200, c, 3, torch.bfloat16)
    for score in ("softmax", "sigmoid"):
        for b in (None, _bias(c, 5), torch.zeros(c, device="cuda")):
            _compare(z, b, k, score, 1, groups, keep, True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [50, 700])
@pytest.mark.parametrize("c", [64, 300, 1500, 4096, 6000])
def test_near_ties_are_told_apart(c, rows):
    """Sums that fp32 cannot order: scores and biases that cancel to differences around 1e-9."""
    g = torch.Generator(device="cuda").manual_seed(7)
    z = torch.randn(rows, c, generator=g, device="cuda")
    z[1:4] = z[0]
    for score in ("softmax", "sigmoid"):
        s = torch.sigmoid(z[0].double()) if score == "sigmoid" else torch.softmax(z[0].double(), 0)
        b = (0.9 - s + 1e-9 * torch.randn(c, generator=g, device="cuda", dtype=torch.float64)).float()
        _compare(z, b, 8, score, grad=False)
        _compare(z, b, 8, score, 0, 4, 2, True, grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("c, k", [(40, 6), (300, 12), (700, 20), (4096, 64), (9000, 33)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_equal_and_masked_rows(c, k, score):
    z = _logits(8, c, 11)
    z[0] = 0.25                                   # all equal
    z[1] = float("-inf")                          # nothing left
    z[2] = torch.finfo(torch.float32).min
    z[3] = LOWEST
    z[4] = float("-inf"); z[4, c // 2] = -3.0     # one left
    z[5, ::2] = float("-inf")
    z[6, k // 2:] = float("-inf")                 # fewer than k
    for b in (None, torch.zeros(c, device="cuda"), _bias(c, 2)):
        for renorm in (True, False):
            got = _compare(z, b, k, score, renorm=renorm)
            assert (got.weights[1:4] == 0).all()
            assert torch.equal(got.indices[1], torch.arange(k, device="cuda"))
        got = _compare(z, b, k, score, 0, 2, 1, True) if c % 2 == 0 else None
    off = torch.zeros(c, device="cuda")
    off[: c - k - 1] = float("-inf")              # a bias may switch chapters off
    _compare(z, off, k, score)


@pytest.mark.gpu
@pytest.mark.parametrize("c, rows", [(50, 3), (4096, 3), (4096, 700)])
def test_nan_and_infinite_logits_show_and_stay_in_range(c, rows):
    import memory_b200 as M
    z = _logits(rows, c, 1)
    z[0, 7], z[1, 9] = float("nan"), float("inf")
    for b in (None, _bias(c, 1)):
        got = M.select_chapters(z, 5, score="sigmoid", balance_bias=b)
        assert got.weights[0].isnan().all() and got.indices[0, 0] == 7
        assert got.weights[1].isfinite().all() and (b is not None or got.indices[1, 0] == 9)
        soft = M.select_chapters(z, 5, balance_bias=b)
        assert soft.weights[:2].isnan().all() and soft.weights[2:].isfinite().all()
        for s in (got, soft):
            assert ((s.indices >= 0) & (s.indices < c)).all()
            assert all(len(set(r.tolist())) == 5 for r in s.indices[:5])


@pytest.mark.gpu
def test_gradient_against_differences():
    import memory_b200 as M
    z, b = _logits(4, 40, 5).double(), _bias(40, 5)
    gw = torch.randn(4, 6, device="cuda", dtype=torch.float64)
    for score, renorm in (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)):
        leaf = z.float().requires_grad_(True)
        w = M.select_chapters(leaf, 6, score=score, balance_bias=b, num_shared=1, num_groups=3, top_groups=2, renormalize=renorm).weights
        w.backward(gw.float())
        v = torch.randn_like(z)
        h = 1e-5

        def at(t):
            return (_plain(t, 6, score, b, 1, 1.0, 3, 2, False, renorm)[1] * gw).sum()
        # central difference: h^2 / 6 of a third derivative of order 10, rounding 1e-16 / h
        slope = (at(z.float().double() + h * v) - at(z.float().double() - h * v)) / (2 * h)
        assert abs((leaf.grad.double() * v).sum() - slope) <= 1e-5 * (1 + slope.abs())


@pytest.mark.gpu
def test_strides_shapes_and_streams():
    import memory_b200 as M
    wide = _logits(48, 300, 9)
    _compare(wide[:, 17:282], None, 8, shared=1)                  # rows with a stride, a start off 16 bytes
    _compare(wide.t(), None, 5)                                   # columns
    three = wide.view(4, 12, 300)
    got = M.select_chapters(three, 8, score="sigmoid", num_groups=4, top_groups=2)
    flat = M.select_chapters(wide, 8, score="sigmoid", num_groups=4, top_groups=2)
    assert got.indices.shape == (4, 12, 8) and torch.equal(got.indices.view(48, 8), flat.indices)
    assert torch.equal(got.weights.view(48, 8), flat.weights) and torch.equal(got.load, flat.load)
    assert M.select_chapters(wide[:0], 8).load.sum() == 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = M.select_chapters(wide, 8, score="sigmoid", num_groups=4, top_groups=2)
    side.synchronize()
    assert torch.equal(other.indices, flat.indices)


@pytest.mark.gpu
def test_captured_forward_and_backward_replay_on_new_logits():
    import memory_b200 as M
    from memory_b200.graph import GraphedStep
    b = _bias(257, 4)
    z = _logits(100, 257, 1).requires_grad_(True)
    gw = _logits(100, 8, 2)

    def step(z, gw):
        s = M.select_chapters(z, 8, score="sigmoid", balance_bias=b, num_shared=1, num_groups=8, top_groups=4, group_score="top2")
        return s.indices, s.weights.detach(), s.load, torch.autograd.grad(s.weights, z, gw)[0]
    graph = GraphedStep(step, [z, gw])
    for seed in (5, 6):
        fresh = _logits(100, 257, seed).requires_grad_(True)
        for a, want in zip(graph(fresh, gw), step(fresh, gw)):
            assert torch.equal(a, want)


@pytest.mark.gpu
@pytest.mark.parametrize("token", [False, True])
@pytest.mark.parametrize("dtype, rows", [(torch.float32, 24), (torch.bfloat16, 24), (torch.bfloat16, 1000)])
def test_router_module(token, dtype, rows):
    """ChapterRouter with other rules: logits, selection and the gradients of states, weight and bias."""
    import memory_b200 as M
    torch.manual_seed(0)
    r = M.ChapterRouter(64, 97, top_k=5, score="sigmoid", balance_bias=True, num_groups=8, top_groups=3, group_score="top2").cuda()
    with torch.no_grad():
        r.router.weight.mul_(20)
        r.router.bias.normal_(0, 0.1)
        r.balance_bias.uniform_(-0.05, 0.05)
    h = (torch.randn(2, rows, 64, device="cuda") + torch.randn(2, 1, 64, device="cuda")).to(dtype).requires_grad_(True)
    idx, w, losses = (r.route_token_level if token else r)(h, exclude_prefix_chapters=1)
    assert losses == {} and float(M.compute_total_router_loss(losses, reference_tensor=h)) == 0.0
    hd, wd, bd = h.detach().double().requires_grad_(True), r.router.weight.detach().double().requires_grad_(True), r.router.bias.detach().double().requires_grad_(True)
    x = hd.reshape(-1, 64) if token else hd.mean(1)
    logits = x @ wd.t() + bd
    i2, w2, _, _, load = _plain(logits, 5, "sigmoid", r.balance_bias, 1, 1.0, 8, 3, True, True)
    # the logits are fp32 sums: rows whose order hangs on less than their error may differ
    same = (idx.view(-1, 5) == i2).all(1)
    assert same.float().mean() > 0.98 and r.last_load.sum() == idx.numel()
    assert torch.allclose(w.view(-1, 5).double()[same], w2[same], rtol=2e-5, atol=1e-7)
    if not same.all():
        return
    g = torch.randn_like(w2)
    w.backward(g.view(w.shape).float())
    w2.backward(g)
    eps = 2.0 ** -8 if dtype == torch.bfloat16 else 1e-5
    assert (h.grad.double() - hd.grad).norm() <= eps * hd.grad.norm()
    assert (r.router.weight.grad.double() - wd.grad).norm() <= 2e-5 * wd.grad.norm()
    assert (r.router.bias.grad.double() - bd.grad).norm() <= 2e-5 * bd.grad.norm()


@pytest.mark.gpu
def test_balance_bias_evens_the_load_out():
    import memory_b200 as M
    torch.manual_seed(1)
    r = M.ChapterRouter(32, 17, top_k=2, score="sigmoid", balance_bias=True).cuda()
    with torch.no_grad():
        r.router.bias.copy_(torch.linspace(-1, 1, 17))
    h = torch.randn(1, 500, 32, device="cuda")
    with pytest.raises(ValueError, match="no load"):
        r.update_balance()
    r.route_token_level(h, exclude_prefix_chapters=1)
    before, bias = r.last_load.clone(), r.balance_bias.clone()
    r.update_balance(0.01, num_shared=1)
    want = torch.sign(before[1:].double().mean() - before[1:]) * 0.01
    assert torch.equal(r.balance_bias[1:], want.float()) and r.balance_bias[0] == bias[0]
    for _ in range(200):
        r.route_token_level(h, exclude_prefix_chapters=1)
        r.update_balance(0.01, num_shared=1)
    assert r.last_load[1:].float().std() < 0.2 * before[1:].float().std()


def test_refusals():
    import memory_b200 as M
    z = torch.zeros(3, 12)
    for kw, text in ((dict(score="relu"), "softmax"), (dict(group_score="mean"), "group_score"), (dict(num_shared=12), "num_shared"),
                     (dict(num_groups=5), "divide"), (dict(num_groups=4, top_groups=5), "top_groups"),
                     (dict(num_groups=4, top_groups=1), "top_k"), (dict(num_groups=0), "num_groups")):
        with pytest.raises(ValueError, match=text):
            M.select_chapters(z, 4, **kw)
    with pytest.raises(ValueError, match="top_k must be > 0"):
        M.select_chapters(z, 0)
    with pytest.raises(ValueError, match="at most 128"):
        M.select_chapters(torch.zeros(2, 500), 129)
    with pytest.raises(ValueError, match="16384"):
        M.select_chapters(torch.zeros(2, 16390), 2)
    with pytest.raises(ValueError, match="num_chapters"):
        M.select_chapters(torch.zeros(12), 2)
    with pytest.raises(ValueError, match="CUDA"):
        M.select_chapters(z, 4)
    with pytest.raises(ValueError, match="no balance bias"):
        M.ChapterRouter(8, 6, top_k=2).update_balance()
    for kw in (dict(score="tanh"), dict(num_groups=3, top_groups=4), dict(group_score="sum")):
        with pytest.raises(ValueError):
            M.ChapterRouter(8, 6, top_k=2, **kw)
    assert "balance_bias" not in M.ChapterRouter(8, 6).state_dict()


def test_c_entry_refuses_bad_shapes_without_a_gpu():
    import ctypes as C
    from memory_b200 import _lib as L
    lib = L.lib()
    good = dict(rows=2, num_chapters=8, top_k=2, num_shared=0, score=0, num_groups=1, top_groups=1, group_top2=0, renormalize=1,
                dtype=0, ld=8, routed_scale=1.0)
    for change in (dict(rows=0), dict(num_shared=8), dict(num_chapters=20000, ld=20000), dict(num_groups=3), dict(top_groups=2),
                   dict(top_k=9), dict(score=2), dict(dtype=5), dict(ld=7), dict()):
        s = L.SelectShape(**dict(good, **change))
        assert lib.moc_select_fwd(C.byref(s), *([None] * 9)) == -1
        assert lib.moc_select_bwd(C.byref(s), *([None] * 9)) == -1
    assert lib.moc_balance_bias_step(None, None, 4, 0, 0.1, None) == -1

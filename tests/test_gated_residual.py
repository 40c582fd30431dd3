"""gated_residual_norm against its formulas in 64 bits, forward and backward, and what is refused."""
import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16


def _norm(kind, t, w, b, eps):
    if kind == "layernorm":
        t = t - t.mean(-1, keepdim=True)
    t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * w
    return t if b is None else t + b


def _make(shape, kind, gate, following, xt, ft, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s, std=1.0):
        return torch.randn(*s, generator=g, device="cuda") * std
    d = shape[-1]
    t = {"x": normal(*shape, std=2.0).to(xt), "f": normal(*shape, std=0.7).to(ft), "w": 1 + normal(d, std=0.2)}
    if kind == "layernorm":
        t["b"] = normal(d, std=0.3)
        t["f"] = (t["f"].float() + 3.0).to(ft)              # a mean to take away
    if gate != "none":
        t["gate"] = normal(*((d,) if gate == "channel" else (shape[0], d)))
    if following:
        t["nw"] = 1 + normal(d, std=0.2)
        if kind == "layernorm":
            t["nb"] = normal(d, std=0.3)
    return t, normal(*shape).to(xt), normal(*shape).to(ft)


def _plain(t, kind, scale, eps, next_eps):
    z = _norm(kind, t["f"], t["w"], t.get("b"), eps)
    if "gate" in t:
        z = z * (t["gate"] if t["gate"].dim() == 1 else t["gate"][:, None])
    y = scale * t["x"] + z
    return y, _norm(kind, y, t["nw"], t.get("nb"), next_eps) if "nw" in t else None


def _call(t, kind, scale, eps, next_eps):
    import memory_b200 as M
    got = M.gated_residual_norm(t["x"], t["f"], t["w"], t.get("b"), norm_type=kind, eps=eps, gate=t.get("gate"), residual_scale=scale,
                                next_weight=t.get("nw"), next_bias=t.get("nb"), next_eps=next_eps)
    return got if "nw" in t else (got, None)


def _step(t):
    return 2.0 ** -8 if t.dtype == BF16 else 2.0 ** -24


def _close(got, want, eps, what):
    """Elementwise: its own rounding, and ``eps`` (the fp32 arithmetic's relative error) against the tensor's typical size."""
    size = want.abs() + want.pow(2).mean().sqrt()
    worst = ((got.double() - want).abs() - _step(got) * want.abs() - eps * size).max()
    assert worst <= 0, (what, float(worst))


SHAPES = [(1, 1, 768), (1, 5, 64), (2, 3, 250), (3, 70, 256), (2, 1, 1), (5, 2, 7), (2, 33, 1000), (1, 9, 1023), (2, 3, 1028), (1, 4, 4099), (2, 2, 8192),
          (700, 1, 64), (2, 1200, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rms", "layernorm"])
@pytest.mark.parametrize("gate, following", [("none", False), ("none", True), ("channel", False), ("channel", True), ("sequence", False),
                                             ("sequence", True)])
@pytest.mark.parametrize("shape", SHAPES)
def test_values_and_gradients(shape, gate, following, kind):
    if kind == "layernorm" and shape[-1] == 1:
        pytest.skip("a LayerNorm of one column is its bias: its gradient is a difference of equal numbers")
    for xt, ft in ((F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)):
        t, gy, gn = _make(shape, kind, gate, following, xt, ft)
        for v in t.values():
            v.requires_grad_(True)
        ref = {k: v.detach().double().requires_grad_(True) for k, v in t.items()}
        y, n = _call(t, kind, 0.75, 1e-6, 1e-5)
        yr, nr = _plain(ref, kind, 0.75, 1e-6, 1e-5)
        assert y.dtype == xt and (n is None or n.dtype == ft)
        # fp32 sums of d terms in a tree: a few units of 2^-24, up to 16 a thread and 9 levels: 32; statistics enter twice
        eps = 64 * 2.0 ** -24
        _close(y, yr, eps, "y")
        if following:
            _close(n, nr, eps, "n")
        outs, gs = ([y, n], [gy, gn]) if following else ([y], [gy])
        outr = [yr, nr] if following else [yr]
        grads = torch.autograd.grad(outs, list(t.values()), gs)
        wants = torch.autograd.grad(outr, list(ref.values()), [g.double() for g in gs])
        mags = _magnitudes(ref, kind, gy, gn if following else None, 0.75, 1e-6, 1e-5)
        for (name, leaf), g, want in zip(t.items(), grads, wants):
            assert g.dtype == leaf.dtype and g.shape == leaf.shape
            # A gradient is a sum of terms, each off by at most eps (statistics and the row sums above) and a second eps for the other
            # norm it passed; so it is off by 2 eps times the sum of its terms' magnitudes, however much of them cancels (with
            # one column, 1 - fhat^2 = 1e-6 inv^2 is left of 1).
            assert ((g.double() - want).abs() <= _step(g) * want.abs() + 2 * eps * mags[name]).all(), (name, xt, ft)


def _magnitudes(r, kind, gy, gn, scale, eps, next_eps):
    """Sums of the magnitudes of the terms of every gradient, in 64 bits."""
    r = {k: v.detach() for k, v in r.items()}
    d = r["x"].shape[-1]
    gate = r.get("gate", torch.ones(d, dtype=torch.float64, device="cuda"))
    gate = (gate if gate.dim() == 1 else gate[:, None]).expand_as(r["x"]).abs()

    def hat(v, e):
        m = v.mean(-1, keepdim=True) if kind == "layernorm" else 0.0
        inv = 1 / torch.sqrt(((v - m) ** 2).mean(-1, keepdim=True) + e)
        # (a mean taken away leaves the rounding of what it was taken from)
        return (v.abs() + abs(m)) * inv, inv

    def back(g, h, inv):
        return inv * (g + g.mean(-1, keepdim=True) + h * (g * h).mean(-1, keepdim=True))
    fh, fi = hat(r["f"], eps)
    z = fh * r["w"].abs() + r.get("b", torch.zeros(1, device="cuda")).abs()
    y, _ = _plain(r, kind, scale, eps, next_eps)
    t = gy.double().abs()
    out = {}
    if gn is not None:
        g = gn.double().abs()
        yh, yi = hat(y, next_eps)
        yh = yh + yi * (scale * r["x"].abs() + gate * z)
        t = t + back(g * r["nw"].abs(), yh, yi)
        out["nw"], out["nb"] = (g * yh).sum((0, 1)), g.sum((0, 1))
    out["x"], out["f"] = scale * t, back(t * gate * r["w"].abs(), fh, fi)
    out["w"], out["b"] = (t * gate * fh).sum((0, 1)), (t * gate).sum((0, 1))
    if "gate" in r:
        out["gate"] = (t * z).sum((0, 1) if r["gate"].dim() == 1 else 1)
    return out


@pytest.mark.gpu
def test_one_output_used_alone():
    for keep in ("y", "n"):
        t, gy, gn = _make((3, 20, 96), "rms", "channel", True, F32, F32)
        for v in t.values():
            v.requires_grad_(True)
        ref = {k: v.detach().double().requires_grad_(True) for k, v in t.items()}
        out = dict(zip("yn", _call(t, "rms", 0.5, 1e-6, 1e-6)))[keep]
        want = dict(zip("yn", _plain(ref, "rms", 0.5, 1e-6, 1e-6)))[keep]
        g = gy if keep == "y" else gn
        out.backward(g)
        want.backward(g.double())
        for k in t:
            if ref[k].grad is None:
                assert t[k].grad is None
            else:
                _close(t[k].grad, ref[k].grad, 1e-4, (keep, k))


@pytest.mark.gpu
def test_gradient_against_differences():
    t, gy, gn = _make((2, 3, 40), "layernorm", "sequence", True, F32, F32)
    for v in t.values():
        v.requires_grad_(True)
    y, n = _call(t, "layernorm", 0.75, 1e-6, 1e-6)
    grads = torch.autograd.grad([y, n], list(t.values()), [gy, gn])
    base = {k: v.detach().double() for k, v in t.items()}

    def at(change):
        y, n = _plain({k: base[k] + change.get(k, 0.0) for k in base}, "layernorm", 0.75, 1e-6, 1e-6)
        return (y * gy).sum() + (n * gn).sum()
    for (k, v), g in zip(base.items(), grads):
        e = torch.randn_like(v)
        slope = (at({k: 1e-5 * e}) - at({k: -1e-5 * e})) / 2e-5
        assert abs((g.double() * e).sum() - slope) <= 1e-4 * (1 + slope.abs()), k


@pytest.mark.gpu
def test_extremes():
    """Rows of zeros, of large numbers, and with NaN or infinity: each row is its own."""
    import memory_b200 as M
    t, _, _ = _make((1, 6, 768), "rms", "channel", True, F32, F32)
    t["f"][0, 0] = 0
    t["x"][0, 0] = 0
    t["f"][0, 1] *= 1e15
    t["f"][0, 2, 5] = float("nan")
    t["x"][0, 3, 7] = float("inf")
    y, n = _call(t, "rms", 0.75, 1e-6, 1e-6)
    yr, nr = _plain({k: v.double() for k, v in t.items()}, "rms", 0.75, 1e-6, 1e-6)
    ok = [0, 1, 4, 5]
    _close(y[:, ok], yr[:, ok], 1e-5, "y")
    _close(n[:, ok], nr[:, ok], 1e-5, "n")
    assert y[0, 2].isnan().all() and n[0, 2].isnan().all() and y[0, 3, 7] == float("inf") and n[0, 3, 7].isnan()
    assert (y[0, 0] == 0).all() and (n[0, 0] == 0).all()
    empty, m = M.gated_residual_norm(t["x"][:, :0], t["f"][:, :0], t["w"], next_weight=t["nw"])
    assert empty.shape == (1, 0, 768) == m.shape
    leaf = t["x"][:, :0].clone().requires_grad_(True)
    M.gated_residual_norm(leaf, t["f"][:, :0], t["w"]).sum().backward()
    assert leaf.grad.shape == leaf.shape


@pytest.mark.gpu
def test_strided_and_unaligned_inputs_equal_dense_ones():
    t, gy, gn = _make((2, 9, 128), "rms", "channel", True, F32, BF16)
    wide = torch.randn(2, 9, 300, device="cuda")
    flat = torch.randn(2 * 9 * 128 + 1, device="cuda").bfloat16()
    wide[:, :, 5:133] = t["x"]
    flat[1:] = t["f"].flatten()
    other = dict(t, x=wide[:, :, 5:133], f=flat[1:].view(2, 9, 128))
    for v in list(t.values()) + [other["x"], other["f"]]:
        if v.is_leaf:
            v.requires_grad_(True)
    a, b = _call(t, "rms", 0.75, 1e-6, 1e-6), _call(other, "rms", 0.75, 1e-6, 1e-6)
    # (single columns instead of pieces of four: the sums run in another order)
    for u, v in zip(a, b):
        assert torch.allclose(u.float(), v.float(), rtol=2.0 ** -7 if u.dtype == BF16 else 1e-5, atol=1e-5)


@pytest.mark.gpu
def test_bf16_parameters_get_bf16_gradients_and_repeats_are_equal():
    t, gy, gn = _make((4, 30, 256), "layernorm", "sequence", True, BF16, BF16)
    t = {k: v.bfloat16().requires_grad_(True) for k, v in t.items()}
    runs = []
    for _ in range(2):
        y, n = _call(t, "layernorm", 0.75, 1e-6, 1e-6)
        runs.append([y, n] + list(torch.autograd.grad([y, n], list(t.values()), [gy, gn])))
    assert all(g.dtype == BF16 for g in runs[0]) and all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.gpu
def test_captured_step_replays_beside_eager_calls():
    from memory_b200.graph import GraphedStep
    t, gy, gn = _make((2, 50, 128), "rms", "sequence", True, F32, BF16)
    names = list(t)

    def step(*vals):
        u = dict(zip(names, vals))
        y, n = _call(u, "rms", 0.75, 1e-6, 1e-6)
        return [y.detach(), n.detach()] + list(torch.autograd.grad([y, n], list(vals), [gy, gn]))
    leaves = [t[k].requires_grad_(True) for k in names]
    first, second = GraphedStep(step, leaves), GraphedStep(step, leaves)
    for seed in (3, 4):
        u = _make((2, 50, 128), "rms", "sequence", True, F32, BF16, seed)[0]
        vals = [u[k].requires_grad_(True) for k in names]
        want = step(*vals)
        for graph in (first, second):
            assert all(torch.equal(a, b) for a, b in zip(graph(*vals), want))


@pytest.mark.gpu
@pytest.mark.parametrize("rms", [True, False])
def test_sub_block_with_post_norm(rms):
    """MemorySubBlock: attention branch, post-norm, gate, residual scale and the next block's norm, values and every gradient."""
    import memory_b200 as M
    torch.manual_seed(0)
    block = M.MemorySubBlock(64, 1, use_rms_norm=rms, wo_init_zero=False, compute_dtype=F32, post_norm=True, gate=True,
                             residual_scale=0.5).cuda()
    following = (M.RMSNorm(64) if rms else torch.nn.LayerNorm(64, eps=1e-6)).cuda()
    for p in [*block.parameters(), *following.parameters()]:
        torch.nn.init.normal_(p, 0.5 if p.dim() == 1 else 0.0, 0.2)
    h = torch.randn(2, 64, 64, device="cuda", requires_grad=True)
    memory = torch.randn(2, 48, 64, device="cuda", requires_grad=True)
    y, n = block(h, memory, next_norm=following)
    kind = "rms" if rms else "layernorm"
    ps = [h, memory, *block.parameters(), *following.parameters()]
    g = torch.Generator(device="cuda").manual_seed(2)
    gy, gn = torch.randn(y.shape, generator=g, device="cuda"), torch.randn(y.shape, generator=g, device="cuda")
    grads = torch.autograd.grad([y, n], ps, [gy, gn])

    ref = [p.detach().double().requires_grad_(True) for p in ps]
    names = ["h", "memory"] + [k for k, _ in block.named_parameters()] + ["next." + k for k, _ in following.named_parameters()]
    r = dict(zip(names, ref))
    a = _norm(kind, r["h"], r["memory_layernorm.weight"], r.get("memory_layernorm.bias"), 1e-6)
    q, k, v = a @ r["memory_attn.q_proj.weight"].t(), r["memory"] @ r["memory_attn.k_proj.weight"].t(), r["memory"] @ r["memory_attn.v_proj.weight"].t()
    o = torch.softmax(q @ k.transpose(1, 2) / 8, -1) @ v @ r["memory_attn.o_proj.weight"].t()
    yr = 0.5 * r["h"] + r["gate"] * _norm(kind, o, r["post_norm.weight"], r.get("post_norm.bias"), 1e-6)
    nr = _norm(kind, yr, r["next.weight"], r.get("next.bias"), 1e-6)
    wants = torch.autograd.grad([yr, nr], ref, [gy.double(), gn.double()])
    for name, got, want in [("y", y, yr), ("n", n, nr)] + list(zip(names, grads, wants)):
        assert (got.double() - want).norm() <= 1e-4 * want.norm() + 1e-6, name
    adaptive = torch.randn(2, 64, device="cuda")
    other = block(h, memory, gate=adaptive)
    want = 0.5 * r["h"] + adaptive.double()[:, None] * _norm(kind, o, r["post_norm.weight"], r.get("post_norm.bias"), 1e-6)
    assert (other.double() - want).norm() <= 1e-4 * want.norm()


def test_refusals():
    import memory_b200 as M
    x, w = torch.zeros(2, 3, 8), torch.zeros(8)
    call = M.gated_residual_norm
    for args, kw in (((x, x[:, :2], w), {}), ((x[0, 0], x[0, 0], w), {}), ((x, x, w[:7]), {}), ((x, x, w), dict(norm_type="batch")),
                     ((x, x, w, w), {}), ((x, x, w), dict(next_bias=w, norm_type="layernorm")), ((x, x, w), dict(gate=w[:4])),
                     ((x, x, w), dict(gate=torch.zeros(3, 8))), ((x[0], x[0], w), dict(gate=torch.zeros(3, 8))),
                     ((x, x, w), dict(next_weight=torch.zeros(4))), ((torch.zeros(1, 8193), torch.zeros(1, 8193), torch.zeros(8193)), {}),
                     ((x, x, w), {})):
        with pytest.raises(ValueError):
            call(*args, **kw)
    with pytest.raises(ValueError, match="post_norm"):
        M.MemorySubBlock(64, 1, gate=True)
    with pytest.raises(ValueError, match="post_norm"):
        M.MemorySubBlock(64, 1)(x, x, next_norm=M.RMSNorm(8))
    assert set(M.MemorySubBlock(64, 1).state_dict()) == {"memory_layernorm.weight"} | {
        f"memory_attn.{n}_proj.weight" for n in "qkvo"}


def test_c_entry_refuses_without_a_gpu():
    import ctypes as C
    from memory_b200 import _lib as L
    lib = L.lib()
    good = dict(rows=4, dim=64, kind=1, x_dtype=0, f_dtype=1, gate_seq=2, residual_scale=1.0, eps=1e-6, next_eps=1e-6)
    for change in (dict(rows=0), dict(dim=0), dict(dim=8193), dict(kind=0), dict(x_dtype=2), dict(gate_seq=3), dict(gate_seq=-1), dict()):
        s = L.ResidualShape(**dict(good, **change))
        assert lib.moc_gated_residual_fwd(C.byref(s), *([None] * 11)) == -1
        assert lib.moc_gated_residual_bwd(C.byref(s), *([None] * 18)) == -1
        if change:
            assert lib.moc_gated_residual_bwd_scratch_bytes(C.byref(s), 1) == -1

"""Training steps and generated tokens that run the operators together -- selection by other rules, post-norm with gate and next norm,
clipping with the bank's compact gradient, its optimizer step, the 8-bit cache -- against the same in 64 bits."""
import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16
B, L, D, HEADS, KV, T, C, K, RHO = 2, 48, 128, 2, 1, 16, 17, 3, 2.5


def _rms(t, w, eps=1e-6):
    return t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * w


def _select(logits, bias):
    """Sigmoid scores, the two best of four groups by the sum of their two largest, the K best; (ids, joint ids, joint weights)."""
    s = torch.sigmoid(logits[:, 1:])
    sel = s.detach() + bias[1:]
    groups = sel.view(-1, 4, 4).topk(2, -1).values.sum(-1).topk(2, -1).indices
    kept = torch.zeros_like(sel).view(-1, 4, 4).scatter_(1, groups[..., None].expand(-1, -1, 4), 1.0).view_as(sel)
    idx = sel.masked_fill(kept == 0, float("-inf")).topk(K, -1).indices
    w = s.gather(1, idx)
    w = w / w.sum(-1, keepdim=True)
    joint = torch.cat([torch.ones_like(w[:, :1]), RHO * w], -1)
    return idx + 1, torch.cat([torch.zeros_like(idx[:, :1]), idx + 1], -1), joint / joint.sum(-1, keepdim=True)


def _attend(q, k, v, heads, kv_heads):
    b, l, _ = q.shape
    q = q.view(b, l, heads, 64).transpose(1, 2)
    k, v = (t.view(b, -1, kv_heads, 64).transpose(1, 2).repeat_interleave(heads // kv_heads, 1) for t in (k, v))
    return (torch.softmax(q @ k.transpose(2, 3) / 8, -1) @ v).transpose(1, 2).reshape(b, l, heads * 64)


def _modules(compute):
    import memory_b200 as M
    torch.manual_seed(0)
    router = M.ChapterRouter(D, C, top_k=K, score="sigmoid", balance_bias=True, num_groups=4, top_groups=2, group_score="top2").cuda()
    block = M.MemorySubBlock(D, HEADS, num_kv_heads=KV, wo_init_zero=False, compute_dtype=compute, post_norm=True, gate=True,
                             residual_scale=0.7).cuda()
    following = M.RMSNorm(D).cuda()
    with torch.no_grad():
        for p in [*router.parameters(), *block.parameters(), *following.parameters()]:
            p.normal_(0.8 if p.dim() == 1 else 0.0, 0.2 if p.dim() == 1 else 0.12)
        router.router.bias.normal_()
        router.balance_bias.normal_(0.0, 0.05)
    return router, block, following, torch.nn.Parameter(torch.randn(C * T, D, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_training_steps(max_norm):
    import memory_b200 as M
    router, block, following, bank = _modules(F32)
    bank.moc_sparse_grad = M.SparseBankGrad()
    opt = M.SparseBankAdamW(bank, T, lr=1e-3, weight_decay=0.01)
    named = dict(router.named_parameters()) | {"block." + k: p for k, p in block.named_parameters()} | {
        "next." + k: p for k, p in following.named_parameters()}
    r = {k: p.detach().double().requires_grad_(True) for k, p in named.items()}
    ref_bank = bank.detach().double().requires_grad_(True)
    ref_opt = torch.optim.AdamW([ref_bank], lr=1e-3, betas=opt.betas, eps=opt.eps, weight_decay=0.01)
    bias = router.balance_bias.double()
    g = torch.Generator(device="cuda").manual_seed(1)
    for step in range(3):
        h = torch.randn(B, L, D, generator=g, device="cuda").requires_grad_(True)
        gy, gn = (torch.randn(B, L, D, generator=g, device="cuda") for _ in range(2))
        bank.moc_sparse_grad.clear()
        for p in named.values():
            p.grad = None
        idx, _, cidx, cw, _ = router.route_with_shared(h, 1, RHO)
        y, n = block(h, M.gather_chapters(bank, cidx, cw, T), next_norm=following)
        torch.autograd.backward([y, n], [gy, gn])
        clip = M.clip_grad_norm_(named.values(), max_norm, bank_grads=[bank.moc_sparse_grad])
        before = bank.detach().clone()
        opt.step(bank.moc_sparse_grad, grad_scale=clip.coefficient)
        router.update_balance(0.01)

        hr = h.detach().double().requires_grad_(True)
        ridx, rcidx, rcw = _select(hr.mean(1) @ r["router.weight"].t() + r["router.bias"], bias)
        assert torch.equal(idx, ridx) and torch.equal(cidx.long(), rcidx)
        memory = (ref_bank.view(C, T, D)[rcidx] * rcw[..., None, None]).reshape(B, -1, D)
        a = _rms(hr, r["block.memory_layernorm.weight"])
        o = _attend(a @ r["block.memory_attn.q_proj.weight"].t(), memory @ r["block.memory_attn.k_proj.weight"].t(),
                    memory @ r["block.memory_attn.v_proj.weight"].t(), HEADS, KV) @ r["block.memory_attn.o_proj.weight"].t()
        yr = 0.7 * hr + r["block.gate"] * _rms(o, r["block.post_norm.weight"])
        nr = _rms(yr, r["next.weight"])
        wants = torch.autograd.grad([yr, nr], [*r.values(), hr, ref_bank], [gy.double(), gn.double()])
        norm = torch.sqrt(sum(w.pow(2).sum() for w in (*wants[:-2], wants[-1])))
        coefficient = min(1.0, max_norm / (float(norm) + 1e-6))
        # fp32 throughout: a chain of about ten sums of up to 128 x 96 products, 2^-24 x sqrt(terms) each and cancellation of one to
        # two digits in the softmax's and norms' gradients; 1e-4 of a tensor's norm is ten times that
        def close(got, want, what):
            assert (got.double() - want).norm() <= 1e-4 * want.norm(), (step, what)
        close(y, yr, "y")
        close(n, nr, "n")
        close(h.grad, wants[-2], "h")
        close(clip.total_norm, norm, "norm")
        assert abs(float(clip.coefficient) - coefficient) <= 1e-4 * coefficient
        for name, want in zip(r, wants):
            close(named[name].grad, coefficient * want, name)
        close(bank.moc_sparse_grad.to_dense(bank), wants[-1], "bank")
        old = ref_bank.detach().clone()
        ref_bank.grad = coefficient * wants[-1]
        ref_opt.step()
        # a step is lr times g / (|g| + eps): elements whose gradient is within fp32's error of zero (1e-5 of its size: as large a part
        # of them) may differ by all of it, sqrt(1e-5) = 3e-3 of the step's norm; the parameter's own rounding is 2^-24 x 1 of 1e-3
        moved, want = bank.detach() - before, ref_bank.detach() - old
        assert (moved.double() - want).norm() <= 1e-2 * want.norm(), step
        load = torch.bincount(ridx.flatten(), minlength=C).double()
        bias[1:] += 0.01 * torch.sign(load[1:].mean() - load[1:])
        assert torch.allclose(router.balance_bias.double(), bias, rtol=0, atol=1e-6)          # three roundings of 2^-25


@pytest.mark.gpu
def test_generated_tokens():
    """Router on the window, attention over the 8-bit cache, the result merged into the stream: token by token."""
    import memory_b200 as M
    router, block, following, bank = _modules(BF16)
    a = block.memory_attn
    cache = M.ProjectedBankCache(bank, a.k_proj.weight, a.v_proj.weight, T, 1, None, cache_dtype=torch.float8_e4m3fn, scale_rows=8)
    dec = M.MemoryDecoder(cache, router.router.weight, router.router.bias, a.q_proj.weight, a.o_proj.weight, num_heads=HEADS,
                          num_kv_heads=KV, top_k=K, num_shared_chapters=1, routed_scaling_factor=RHO, router=router)
    window = M.RoutingWindow(8, "hybrid")
    g = torch.Generator(device="cuda").manual_seed(4)
    window.prefill(torch.randn(B, 5, D, generator=g, device="cuda").to(BF16))
    rows = (cache.kv_bank.double().view(C * T // 8, 8, 2 * KV, 64) * cache.kv_scale.double()[:, None, :, None]).view(C, T, 2 * KV * 64)
    for token in range(6):
        x = torch.randn(B, 1, D, generator=g, device="cuda").to(BF16)
        states = window.step(x)
        out, info = dec.step(block.memory_layernorm(x), states)
        y, n = M.gated_residual_norm(x, out, block.post_norm.weight, gate=block.gate, residual_scale=0.7,
                                     next_weight=following.weight)
        pooled = states.double().mean(1)
        idx, cidx, cw = _select(pooled @ router.router.weight.double().t() + router.router.bias.double(), router.balance_bias.double())
        assert torch.equal(info["indices"], idx)
        memory = (rows[cidx] * cw[..., None, None]).reshape(B, -1, 2 * KV * 64)
        q = _rms(x.double(), block.memory_layernorm.weight.double()) @ a.q_proj.weight.double().t()
        o = _attend(q, *memory.split(KV * 64, -1), HEADS, KV) @ a.o_proj.weight.double().t()
        yr = 0.7 * x.double() + block.gate.double() * _rms(o, block.post_norm.weight.double())
        nr = _rms(yr, following.weight.double())
        # roundings to bf16 on the way (2^-8 at worst, half that on average): the norm's result, the weights and q, the probabilities'
        # result, the projection's, y or n; they add up in squares to below 2^-8 x sqrt(8) / 2 = 2^-7.5, scores of size 1 to 3 double q's
        for got, want in ((y, yr), (n, nr)):
            assert (got.double() - want).norm() <= 2.0 ** -6 * want.norm(), token


def test_a_next_norm_of_another_kind_is_refused():
    import memory_b200 as M
    x = torch.zeros(1, 2, 64)
    for rms, other in ((True, torch.nn.LayerNorm(64)), (False, M.RMSNorm(64)), (False, torch.nn.LayerNorm(64, elementwise_affine=False)),
                       (True, torch.nn.Identity())):
        with pytest.raises(ValueError, match="next_norm"):
            M.MemorySubBlock(64, 1, use_rms_norm=rms, post_norm=True)(x, x, next_norm=other)

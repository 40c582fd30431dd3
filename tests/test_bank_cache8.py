"""The projected-bank cache in 8 bits: its values and scales, attention over it and over the bf16 cache, the decoder on it, and what
is refused."""
import pytest
import torch

T64 = 64


def _kv(rows, heads, seed, block=8):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv = torch.randn(rows, 2 * heads * 64, generator=g, device="cuda") * 0.5
    size = torch.exp(0.5 * torch.randn(rows // block, 2 * heads, generator=g, device="cuda"))
    return (kv * size.repeat_interleave(block, 0).repeat_interleave(64, 1)).bfloat16()


def _quantized(kv, block):
    t = kv.float().view(kv.shape[0] // block, block, -1, 64)
    scale = t.abs().amax((1, 3)) / 448.0
    s = scale[:, None, :, None]
    return torch.where(s > 0, t / s, torch.zeros_like(t)).to(torch.float8_e4m3fn).view(kv.shape), scale


@pytest.mark.gpu
@pytest.mark.parametrize("rows, heads, chapter, block", [(64, 12, 64, 64), (40, 1, 8, 1), (1040, 4, 16, 8), (120, 3, 40, 40), (96, 2, 32, 32),
                                                         (600, 5, 200, 100), (130, 1, 130, 130), (21, 2, 7, 7), (24, 1, 12, 3)])
def test_values_and_scales_are_the_definition_to_the_bit(rows, heads, chapter, block):
    import memory_b200 as M
    kv = _kv(rows, heads, rows, 1)
    kv[block:2 * block] = 0
    cache = M.ProjectedBankCache.from_rows(kv, chapter, cache_dtype=torch.float8_e4m3fn, scale_rows=block)
    values, scale = _quantized(kv, block)
    assert torch.equal(cache.kv_scale, scale)
    assert torch.equal(cache.kv_bank.view(torch.uint8), values.view(torch.uint8))
    # e4m3 is half a step of 2^-3 off above its subnormals, 2^-10 of the scale below 2^-6
    back = cache.kv_bank.float() * scale.repeat_interleave(block, 0).repeat_interleave(64, 1)
    err = (back - kv.float()).abs()
    assert (err <= 2.0 ** -4 * kv.float().abs() + 2.0 ** -10 * scale.repeat_interleave(block, 0).repeat_interleave(64, 1)).all()


@pytest.mark.gpu
def test_blocks_with_nan_or_infinity_stand_for_nan_and_leave_the_others_alone():
    import memory_b200 as M
    kv = _kv(128, 2, 1)
    kv[3, 5], kv[70, 130] = float("nan"), float("inf")
    cache = M.ProjectedBankCache.from_rows(kv, 64, cache_dtype=torch.float8_e4m3fn)
    back = cache.kv_bank.float().view(2, 64, 4, 64) * cache.kv_scale[:, None, :, None]
    bad = back.isnan().all(1).all(-1)
    assert torch.equal(bad.cpu(), torch.tensor([[True, False, False, False], [False, False, True, False]]))
    assert not back[~bad[:, None, :].expand(2, 64, 4)].isnan().any()


def _attention64(q, kv, idx, w, heads, kv_heads, chapter, counts, scale=0.125):
    """The definition in 64 bits over the cache's own numbers ``kv`` [rows, 2 * HK * 64]."""
    b, n_q, _ = q.shape
    t = kv.double().view(-1, chapter, 2, kv_heads, 64)
    out, lse = torch.zeros(b, n_q, heads, 64, dtype=torch.float64), torch.full((b, n_q, heads), float("-inf"), dtype=torch.float64)
    out, lse = out.cuda(), lse.cuda()
    for i in range(b):
        n = idx.shape[1] if counts is None else max(0, min(int(counts[i]), idx.shape[1]))
        if n == 0:
            continue
        rows = t[idx[i, :n].long()].reshape(n * chapter, 2, kv_heads, 64).repeat_interleave(heads // kv_heads, 2)
        u = w[i, :n].double().repeat_interleave(chapter)
        s = torch.einsum("qhd,rhd->qhr", q[i].double().view(n_q, heads, 64), rows[:, 0]) * u * scale
        lse[i] = s.logsumexp(-1)
        out[i] = torch.einsum("qhr,rhd->qhd", torch.softmax(s, -1) * u, rows[:, 1])
    return out.flatten(2), lse


def _lists(b, n, chapters, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    idx = torch.rand(b, chapters, generator=g, device="cuda").argsort(1)[:, :n].int()
    return idx, torch.rand(b, n, generator=g, device="cuda") * 0.3


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("b, n_q, heads, kv_heads, chapter, block, n, ragged", [
    (1, 1, 12, 12, 64, 64, 65, False), (3, 1, 12, 4, 64, 16, 9, True), (2, 3, 8, 1, 40, 8, 5, True), (5, 1, 10, 2, 16, 1, 1, False),
    (4, 2, 6, 3, 7, 7, 11, True), (64, 1, 2, 2, 16, 16, 33, True), (1, 1, 1, 1, 1, 1, 1, False), (2, 5, 4, 1, 130, 65, 3, False),
])
def test_attention_over_the_cache(b, n_q, heads, kv_heads, chapter, block, n, ragged, eight):
    import memory_b200 as M
    chapters = 70
    kv = _kv(chapters * chapter, kv_heads, n + b, 1)
    g = torch.Generator(device="cuda").manual_seed(b)
    q = (4 * torch.randn(b, n_q, heads * 64, generator=g, device="cuda")).bfloat16()
    idx, w = _lists(b, n, chapters, 3)
    counts = None
    if ragged:
        counts = torch.randint(0, n + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        counts[0], counts[-1] = 0, n
        idx[0] = -7                                # nothing of an empty list is read
        if b > 2:
            idx[1, int(counts[1]):] = 1 << 30      # ... nor what lies behind the count
    if eight:
        cache = M.ProjectedBankCache.from_rows(kv, chapter, cache_dtype=torch.float8_e4m3fn, scale_rows=block)
        real = cache.kv_bank.float() * cache.kv_scale.repeat_interleave(block, 0).repeat_interleave(64, 1)
    else:
        cache, real = M.ProjectedBankCache.from_rows(kv, chapter), kv
    out, lse = cache.attend(q, idx, w, heads, kv_heads, counts=counts, return_lse=True)
    want, want_lse = _attention64(q, real, idx, w, heads, kv_heads, chapter, counts)
    M._lib.check_device_status(q.device)
    # scores are fp32 dot products of 64 terms (|q||k| up to ~60 of them: 64 U 2^-24 relative to the sum of magnitudes, 1e-4 at
    # most), so probabilities within 2e-4; the output rounds to bf16 (2^-8 of the value, 2^-9 typical)
    top = want.abs().amax(-1, keepdim=True)
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 4e-4 * top).all()
    fine = torch.isfinite(want_lse)
    assert torch.equal(fine, torch.isfinite(lse)) and (lse[~fine] == float("-inf")).all()
    assert (lse.double() - want_lse)[fine].abs().max() <= 2e-4 if fine.any() else True
    if ragged:
        assert (out[0] == 0).all()
    again = cache.attend(q, idx, w, heads, kv_heads, counts=counts)
    assert torch.equal(again, out)


@pytest.mark.gpu
def test_far_chapters_pass_32_bits():
    """Rows whose bytes lie past 2^31 and 2^32 in the cache."""
    import memory_b200 as M
    chapters, width = 45000, 12 * 128                        # 45,000 x 64 x 1,536 = 4.4e9 bytes
    values = torch.zeros(chapters * 64, width, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(chapters, 24, device="cuda")
    far = [0, 21845, 43691, chapters - 1]
    g = torch.Generator(device="cuda").manual_seed(0)
    small = torch.randint(0, 120, (4, 64, width), generator=g, device="cuda", dtype=torch.uint8)
    for i, c in enumerate(far):
        values[c * 64:(c + 1) * 64] = small[i]
        scales[c] = 0.001 * (i + 1)
    q = torch.randn(2, 1, 768, generator=g, device="cuda").bfloat16()
    w = torch.tensor([[0.4, 0.3, 0.2, 0.1]], device="cuda").expand(2, 4).contiguous()
    cache = M.ProjectedBankCache.from_quantized(values.view(torch.float8_e4m3fn), scales, 64)
    near = M.ProjectedBankCache.from_quantized(small.reshape(-1, width).view(torch.float8_e4m3fn), scales[far].contiguous(), 64)
    ids = torch.tensor([far], dtype=torch.int64, device="cuda").expand(2, 4)
    a = cache.attend(q, ids, w, 12)
    b = near.attend(q, torch.arange(4, device="cuda").expand(2, 4), w, 12)
    assert torch.equal(a, b) and a.abs().sum() > 0


@pytest.mark.gpu
def test_bad_chapter_ids_are_reported_and_left_out():
    import memory_b200 as M
    kv = _kv(10 * 16, 2, 0)
    cache = M.ProjectedBankCache.from_rows(kv, 16, cache_dtype=torch.float8_e4m3fn)
    q = torch.randn(1, 1, 128, device="cuda").bfloat16()
    w = torch.full((1, 3), 0.5, device="cuda")
    got = cache.attend(q, torch.tensor([[1, 10, 4]], device="cuda"), w, 2)
    with pytest.raises(RuntimeError, match="chapter index"):
        M._lib.check_device_status(q.device)
    assert torch.equal(got, cache.attend(q, torch.tensor([[1, 4]], device="cuda"), w[:, :2].contiguous(), 2))


@pytest.mark.gpu
def test_a_nan_query_or_block_gives_nan():
    import memory_b200 as M
    kv = _kv(4 * 16, 2, 0)
    kv[20, 2 * 64 + 3] = float("nan")                     # a value row of head 0, chapter 1
    cache = M.ProjectedBankCache.from_rows(kv, 16, cache_dtype=torch.float8_e4m3fn)
    q = torch.randn(2, 1, 128, device="cuda").bfloat16()
    q[1, 0, 70] = float("nan")                            # head 1
    got = cache.attend(q, torch.tensor([[0, 1], [2, 3]], device="cuda"), torch.full((2, 2), 0.5, device="cuda"), 2).view(2, 2, 64)
    assert got[0, 0].isnan().all() and got[1, 1].isnan().all()
    assert got[0, 1].isfinite().all() and got[1, 0].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("chapters", [2, 40])
def test_nan_shows_over_either_cache(dtype, chapters):
    """A query, a key row or a value row with a NaN gives NaN and touches nothing else; one warp's unit among many, or all there is."""
    import memory_b200 as M
    kv = _kv(chapters * 16, 2, 1)
    kv[16 + 3, 5] = float("nan")                          # a key row of head 0, chapter 1
    kv[8, 3 * 64 + 7] = float("nan")                      # a value row of head 1, chapter 0
    cache = M.ProjectedBankCache.from_rows(kv, 16, cache_dtype=dtype)
    q = torch.randn(3, 2, 128, device="cuda").bfloat16()
    q[2, 1, 64 + 9] = float("nan")                        # sequence 2, token 1, head 1
    idx = torch.stack([torch.arange(chapters), torch.arange(chapters).clamp(min=1), torch.full((chapters,), 1)]).cuda()
    out, lse = cache.attend(q, idx, torch.full(idx.shape, 0.5, device="cuda"), 2, return_lse=True)
    out = out.view(3, 2, 2, 64)                           # [sequence, token, head, dim]
    assert out[:, :, 0].isnan().all() and lse[:, :, 0].isnan().all()
    assert out[0, :, 1].isnan().any(-1).all() and lse[0, :, 1].isfinite().all()
    assert out[1, :, 1].isfinite().all() and out[2, 0, 1].isfinite().all()
    assert out[2, 1, 1].isnan().all() and lse[2, 1, 1].isnan()


def _decoder(cache_kw, router=None, kv_heads=4):
    import memory_b200 as M
    torch.manual_seed(3)
    d, heads, chapters, t = 256, 4, 33, 16
    bank = torch.randn(chapters * t, d, device="cuda") * 0.2
    wk, wv = (torch.randn(kv_heads * 64, d, device="cuda") * 0.1 for _ in range(2))
    wq, wo = (torch.randn(d, d, device="cuda") * 0.1 for _ in range(2))
    rw, rb = torch.randn(chapters, d, device="cuda") * 0.2, torch.zeros(chapters, device="cuda")
    if router is not None:
        with torch.no_grad():
            router.router.weight.copy_(rw)
    cache = M.ProjectedBankCache(bank, wk, wv, t, 1, "rms", **cache_kw)
    return M.MemoryDecoder(cache, rw, rb, wq, wo, num_heads=heads, num_kv_heads=kv_heads, top_k=5, router=router), cache


@pytest.mark.gpu
@pytest.mark.parametrize("n_q", [1, 5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decoder_on_the_8_bit_cache(n_q, dtype):
    """The whole step is the step over a bf16 cache of the numbers that the 8 bits stand for."""
    import memory_b200 as M
    dec8, c8 = _decoder(dict(cache_dtype=torch.float8_e4m3fn, scale_rows=8))
    dec16, c16 = _decoder({})
    values, scale = _quantized(c16.kv_bank, 8)
    assert torch.equal(c8.kv_bank.view(torch.uint8), values.view(torch.uint8)) and torch.equal(c8.kv_scale, scale)
    window = M.RoutingWindow(6, "hybrid")
    states = window.prefill(torch.randn(3, 9, 256, device="cuda").to(dtype))
    for step in range(3):
        h = torch.randn(3, n_q, 256, device="cuda").to(dtype)
        states = window.step(torch.randn(3, 1, 256, device="cuda").to(dtype))
        out, info = dec8.step(h, states)
        ref, info16 = dec16.step(h, states)
        assert torch.equal(info["indices"], info16["indices"]) and torch.equal(info["combined_weights"], info16["combined_weights"])
        # an e4m3 value is within 2^-4 of its own, 0.6 x that in the mean square of uniform mantissas, and errors are independent
        assert (out.float() - ref.float()).norm() <= 0.06 * ref.float().norm()
        q = M.ops.gemm(h.view(-1, 256).bfloat16(), dec8.wq_c).view(3, n_q, 256)
        real = c8.kv_bank.float() * scale.repeat_interleave(8, 0).repeat_interleave(64, 1)
        want, _ = _attention64(q, real, info["combined_indices"], info["combined_weights"], 4, 4, 16, None)
        want = want.bfloat16().double() @ dec8.wo_c.double().t()
        assert (out.double() - want).norm() <= 2.0 ** -7 * want.norm()


@pytest.mark.gpu
def test_decoder_with_a_router_of_other_rules_captured_and_replayed():
    import memory_b200 as M
    from memory_b200.graph import GraphedStep
    torch.manual_seed(0)
    router = M.ChapterRouter(256, 33, top_k=5, score="sigmoid", balance_bias=True, num_groups=4, top_groups=2).cuda()
    dec, cache = _decoder(dict(cache_dtype=torch.float8_e4m3fn), router)
    h = torch.randn(2, 1, 256, device="cuda").bfloat16()
    states = torch.randn(2, 6, 256, device="cuda").bfloat16()
    out, info = dec.step(h, states)
    idx, w, cidx, cw, _ = router.route_with_shared(states, 1, 2.5)
    assert torch.equal(info["indices"], idx) and torch.equal(info["combined_weights"], cw)
    assert ((idx - 1) // 8).unique(dim=1).shape[1] >= 1 and all(len(set(((r - 1) // 8).tolist())) <= 2 for r in idx)
    q = M.ops.gemm(h.view(-1, 256), dec.wq_c).view(2, 1, 256)
    want = M.ops.gemm(cache.attend(q, cidx, cw, 4).view(2, 256), dec.wo_c).view(2, 1, 256)
    assert torch.equal(out, want)
    graph = GraphedStep(lambda h, s: dec.step(h, s)[0], [h, states])
    h2, s2 = torch.randn_like(h), torch.randn_like(states)
    assert torch.equal(graph(h2, s2), dec.step(h2, s2)[0])


def test_refusals():
    import memory_b200 as M
    kv = torch.zeros(64, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        M.ProjectedBankCache.from_rows(kv, 16)
    with pytest.raises(ValueError, match="CUDA"):
        M.ProjectedBankCache.from_quantized(kv.to(torch.float8_e4m3fn), torch.zeros(4, 4), 16)


@pytest.fixture
def on_cpu(monkeypatch):
    from memory_b200 import _lib as L
    monkeypatch.setattr(L, "require_cuda", lambda *t: None)

    def never():
        raise AssertionError("reached the library")
    monkeypatch.setattr(L, "lib", never)


def test_caches_whose_parts_contradict_are_refused(on_cpu):
    import memory_b200 as M
    kv, f8 = torch.zeros(64, 256, dtype=torch.bfloat16), torch.float8_e4m3fn
    make = M.ProjectedBankCache
    for call, error in ((lambda: make.from_rows(kv.float(), 16), TypeError), (lambda: make.from_rows(kv, 24), ValueError),
                        (lambda: make.from_rows(kv, 16, cache_dtype=torch.float16), TypeError),
                        (lambda: make.from_rows(kv, 16, scale_rows=8), ValueError),
                        (lambda: make.from_rows(kv, 16, cache_dtype=f8, scale_rows=5), ValueError),
                        (lambda: make.from_rows(kv, 16, head_dim=32, cache_dtype=f8), ValueError),
                        (lambda: make.from_quantized(kv, torch.zeros(4, 4), 16), TypeError),
                        (lambda: make.from_quantized(kv.to(f8), torch.zeros(4, 3), 16), ValueError),
                        (lambda: make.from_quantized(kv.to(f8), torch.zeros(4, 4).half(), 16), TypeError),
                        (lambda: make.from_quantized(kv.to(f8), torch.zeros(8, 4), 16, scale_rows=6), ValueError)):
        with pytest.raises(error):
            call()
    cache = make.from_quantized(kv.to(f8), torch.zeros(4, 4), 16)
    q, idx, w = torch.zeros(2, 1, 128, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3)
    for args, kw, error in (((q.float(), idx, w, 2), {}, TypeError), ((q, idx, w, 3), {}, ValueError), ((q, idx, w, 2, 1), {}, ValueError),
                            ((q, idx[:, :2], w, 2), {}, ValueError), ((q, idx[:1], w[:1], 2), {}, ValueError),
                            ((q, idx, w, 2), dict(counts=torch.zeros(3, dtype=torch.int32)), ValueError)):
        with pytest.raises(error):
            cache.attend(*args, **kw)


def test_c_entries_refuse_without_a_gpu():
    import ctypes as C
    from memory_b200 import _lib as L
    lib = L.lib()
    assert lib.moc_quantize_rows(None, 8, 2, 64, 4, None, None, None) == -1
    p = 4096
    for rows, heads, dim, block in ((8, 2, 32, 4), (8, 0, 64, 4), (9, 2, 64, 4), (0, 2, 64, 4), (8, 2, 64, 0)):
        assert lib.moc_quantize_rows(p, rows, heads, dim, block, p, p, None) == -1
    assert lib.moc_quantize_rows(p + 8, 8, 2, 64, 4, p, p, None) == -1
    s = L.DecodeShape(1, 1, 2, 2, 64, 3, 16, 0.125)
    assert lib.moc_decode_attn_cache(C.byref(s), p, p, p, 5, 64, p, p, None, p, None, p, None) == -1
    assert lib.moc_decode_attn_cache(C.byref(s), p, p, p, 0, 64, p, p, None, p, None, p, None) == -1

"""Cases of the operators around the memory layer: what a pass takes, in plain torch and through the package.

``select``    chapters (or experts) chosen from router logits: softmax or sigmoid scores, a balance bias that counts in the
              selection alone, groups of which only the best stay, top-k, renormalised weights, the joint list with the shared
              chapters in front, and how many rows took each chapter; forward, or forward with the gradient of the logits.
``attend``    attention of decoding queries over chapters of a projected-bank cache held in 8 bits (e4m3) with an fp32 scale for
              each block of rows, KV head, and K or V.
``build``     that cache from projected rows in bf16.
``residual``  a block's output merged into the residual stream: ``y = s x + gate * norm(f)``, and the next block's norm of y;
              forward, or forward with every gradient.
``clip``      the global gradient norm over many tensors and the bank's compact gradient, and the clipped tensors.

Sizes are those of the benchmark's layer (d 768, 12 heads of 64, 4,096 routed chapters of 64 rows and a shared one), of the
small parity configuration (d 256, 65 chapters of 16 rows), and the token-level variant's rows.
"""
import math

import torch

own = False

LOWEST = -3.3895313892515355e38          # the lowest finite value of bfloat16: a logit at or below it is masked
E4M3_MAX = 448.0
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
CLIP_EPS = 1e-6


def listed():
    return [
        # one sequence that decodes: a row of the whole bank, softmax scores, a balance bias
        dict(name="select_decode", kind="select", rows=1, chapters=4097, shared=1, topk=64, score="softmax", bias=True, groups=1,
             keep=1, group_score="max", renorm=True, dtype="fp32", train=False),
        # token-level routing of a batch over the whole bank: sigmoid scores, groups
        dict(name="select_tokens", kind="select", rows=8192, chapters=4097, shared=1, topk=16, score="sigmoid", bias=True, groups=8,
             keep=4, group_score="top2", renorm=True, dtype="fp32", train=False),
        # a training step's routing over 256 chapters, the usual number of experts, at an odd number of tokens
        dict(name="select_train", kind="select", rows=8191, chapters=257, shared=1, topk=8, score="sigmoid", bias=True, groups=8,
             keep=4, group_score="top2", renorm=True, dtype="fp32", train=True),
        # one generated token of one user, every head with its own K/V
        dict(name="attend_one", kind="attend", batch=1, queries=1, heads=12, kv_heads=12, chapters=4097, rows=64, block=64, topk=64,
             ragged=False),
        # a full batch of users
        dict(name="attend_batch", kind="attend", batch=64, queries=1, heads=12, kv_heads=12, chapters=4097, rows=64, block=64, topk=64,
             ragged=False),
        # grouped heads, several queries a sequence, lists of different lengths (one of them empty), finer scales
        dict(name="attend_grouped", kind="attend", batch=13, queries=3, heads=12, kv_heads=4, chapters=4097, rows=64, block=16, topk=47,
             ragged=True),
        # the whole bank's cache after the weights changed
        dict(name="build_bank", kind="build", chapters=4097, rows=64, kv_heads=12, block=64),
        # ... and the small configuration's, in blocks of 8 rows
        dict(name="build_small", kind="build", chapters=65, rows=16, kv_heads=4, block=8),
        # one generated token's merge into the stream
        dict(name="residual_token", kind="residual", batch=1, seq=1, d=768, norm="rms", gate="channel", following=True, x="bf16",
             f="bf16", train=False),
        # the training step's, fp32 stream and bf16 branch as under autocast
        dict(name="residual_train", kind="residual", batch=8, seq=1024, d=768, norm="rms", gate="channel", following=True, x="fp32",
             f="bf16", train=True),
        # the small configuration's few gradients
        dict(name="clip_small", kind="clip", layers=2, d=256, vocab=1000, dtype="fp32", touched=9, rows=16, max_norm=0.5),
        # every gradient of twelve blocks, an embedding and the bank's touched chapters
        dict(name="clip_model", kind="clip", layers=12, d=768, vocab=32768, dtype="fp32", touched=483, rows=64, max_norm=1.0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["select", "select", "select", "attend", "attend", "attend", "build", "residual", "residual", "residual",
                       "clip", "clip"])
    if kind == "select":
        per, groups = rng.choice([(8, 8), (32, 8), (50, 4), (61, 3), (64, 4), (512, 8), (1024, 4), (256, 16), (1000, 1), (4096, 1)])
        keep = rng.randint(1, groups)
        shared = rng.choice([0, 1, 2])
        return dict(kind=kind, rows=_log(rng, 1, 8192), chapters=per * groups + shared, shared=shared,
                    topk=rng.randint(1, min(64, per * keep)), score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.7,
                    groups=groups, keep=keep, group_score=rng.choice(["max", "top2"]), renorm=rng.random() < 0.7,
                    dtype=rng.choice(["fp32", "fp32", "bf16"]), train=rng.random() < 0.5)
    if kind == "attend":
        heads, kv_heads = rng.choice([(12, 12), (12, 4), (8, 1), (10, 2)])
        rows = rng.choice([16, 64, 64, 40])
        return dict(kind=kind, batch=_log(rng, 1, 64), queries=rng.choice([1, 1, 1, 2]), heads=heads, kv_heads=kv_heads,
                    chapters=rng.randint(200, 2000), rows=rows, block=rng.choice([8, rows]), topk=_log(rng, 1, 64),
                    ragged=rng.random() < 0.4)
    if kind == "build":
        rows = rng.choice([16, 64, 40, 128])
        return dict(kind=kind, chapters=_log(rng, 9, 2000), rows=rows, kv_heads=rng.choice([1, 3, 4, 12]), block=rng.choice([8, rows]))
    if kind == "residual":
        return dict(kind=kind, batch=rng.randint(1, 8), seq=_log(rng, 1, 1024), d=rng.choice([64, 250, 256, 768, 1000]),
                    norm=rng.choice(["rms", "layernorm"]), gate=rng.choice(["none", "channel", "sequence"]),
                    following=rng.random() < 0.6, x=rng.choice(["fp32", "bf16"]), f=rng.choice(["fp32", "bf16"]),
                    train=rng.random() < 0.6)
    d = rng.choice([64, 250, 256, 768])
    return dict(kind=kind, layers=rng.randint(1, 12), d=d, vocab=_log(rng, 100, 32768), dtype=rng.choice(["fp32", "bf16"]),
                touched=_log(rng, 1, 300), rows=rng.choice([16, 64]), max_norm=rng.choice([0.1, 1.0, 1e6]))


def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, _Inputs(seed))


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


def work(case):
    return globals()["_work_" + case["kind"]](case)


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](prepare(case, seed))


class _Inputs:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.g = torch.Generator(device=self.dev).manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=self.g, device=self.dev).mul_(std).to(dtype)

    def integers(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device=self.dev)

    def distinct(self, n, of, k):
        """[n, k] int32, each row k distinct ids below ``of``."""
        return torch.rand(n, of, generator=self.g, device=self.dev).argsort(1)[:, :k].to(torch.int32)


# ---- select ------------------------------------------------------------------------------------------------------
def _prepare_select(c, x):
    """Logits of trained routers spread over a few units; one row in 32 is padding (every logit at the type's lowest value) and
    one chapter in 100 is masked with -inf.  A balance bias has moved in steps of 0.001."""
    dtype = DTYPES[c["dtype"]]
    z = x.normal(c["rows"], c["chapters"], std=1.5, dtype=dtype)
    z = torch.where((x.integers(0, 100, c["chapters"]) == 0)[None], float("-inf"), z)
    if c["rows"] >= 32:
        z = torch.where((x.integers(0, 32, c["rows"]) == 0)[:, None], torch.finfo(dtype).min, z)
    st = {"case": c, "logits": z.contiguous()}
    st["bias"] = x.integers(-60, 61, c["chapters"]).float() * 0.001 if c["bias"] else None
    if c["train"]:
        st["logits"].requires_grad_(True)
        st["g_weights"] = x.normal(c["rows"], c["topk"])
        st["g_joint"] = x.normal(c["rows"], c["shared"] + c["topk"])
    return st


def _select(c, z, b, wide, scale):
    """Selection in ``wide`` bits, weights in those of ``z``."""
    s0, n, k = c["shared"], c["chapters"] - c["shared"], c["topk"]
    z = z[:, s0:]
    dead = z <= LOWEST

    def scores(t):
        t = torch.where(dead, 0.0, t)
        if c["score"] == "sigmoid":
            return torch.where(dead, 0.0, 1 / (1 + torch.exp(-t)))
        top = torch.where(dead, LOWEST, t).amax(1, keepdim=True).detach()
        e = torch.where(dead, 0.0, torch.exp(torch.where(dead, 0.0, t - top)))
        return e / e.sum(1, keepdim=True).clamp(min=1e-30)
    sw = scores(z.detach().to(wide))
    sel = z.detach().to(wide) if b is None else sw + b[s0:].to(wide)
    none = float("-inf")
    sel = torch.where(dead, none, sel)
    if c["groups"] > 1:
        of = (sel if b is not None or c["group_score"] == "max" else torch.where(dead, none, sw)).view(-1, c["groups"], n // c["groups"])
        best = of.sort(dim=2, descending=True).values[:, :, :2]
        value = best[:, :, 0]
        if c["group_score"] == "top2" and best.shape[2] > 1:
            value = value + torch.where(best[:, :, 1] == none, 0.0, best[:, :, 1])
        order = value.sort(dim=1, descending=True, stable=True).indices[:, :c["keep"]]
        kept = torch.zeros_like(value, dtype=torch.bool).scatter_(1, order, True)
        sel = torch.where(kept.repeat_interleave(n // c["groups"], 1), sel, none)
    got, local = sel.sort(dim=1, descending=True, stable=True)
    got, local = got[:, :k], local[:, :k]
    w = torch.where(got == none, 0.0, scores(z).gather(1, local))
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-12)
    idx = local + s0
    joint_idx, joint = idx, w
    if s0:
        lead = torch.arange(s0, device=z.device).expand(z.shape[0], -1)
        joint_idx = torch.cat([lead, idx], 1)
        joint = torch.cat([torch.ones_like(lead, dtype=w.dtype), w * scale], 1)
        joint = joint / joint.sum(1, keepdim=True).clamp(min=1e-12)
    load = torch.zeros(c["chapters"], dtype=torch.int32, device=z.device)
    load = load.scatter_add(0, idx.flatten(), torch.ones_like(idx.flatten(), dtype=torch.int32))
    return idx, w, joint_idx.to(torch.int32), joint, load


def _plain_select(st):
    c, z = st["case"], st["logits"]
    idx, w, joint_idx, joint, load = _select(c, z.float(), st["bias"], torch.float64, 2.5)
    out = {"indices": idx, "weights": w.detach(), "joint_indices": joint_idx, "joint_weights": joint.detach(), "load": load}
    if c["train"]:
        out["d_logits"], = torch.autograd.grad([w, joint], [z], [st["g_weights"], st["g_joint"]])
    return out


def _own_select(st):
    import memory_b200 as M
    c, z = st["case"], st["logits"]
    s = M.select_chapters(z, c["topk"], score=c["score"], balance_bias=st["bias"], num_shared=c["shared"], routed_scale=2.5,
                          num_groups=c["groups"], top_groups=c["keep"], group_score=c["group_score"], renormalize=c["renorm"])
    out = {"indices": s.indices, "weights": s.weights.detach(), "joint_indices": s.combined_indices,
           "joint_weights": s.combined_weights.detach(), "load": s.load}
    if c["train"]:
        out["d_logits"], = torch.autograd.grad([s.weights, s.combined_weights], [z], [st["g_weights"], st["g_joint"]])
    return out


def _work_select(c):
    size = {"fp32": 4, "bf16": 2}[c["dtype"]]
    table, lists = c["rows"] * c["chapters"], c["rows"] * (16 * c["topk"] + 8 * (c["shared"] + c["topk"]))
    back = c["rows"] * 4 * (c["shared"] + 2 * c["topk"]) + table * size if c["train"] else 0
    return {"bytes": table * size + lists + back + 8 * c["chapters"], "flops": table * (8 if c["train"] else 4)}


def _exact_select(st):
    c, z = st["case"], st["logits"].detach().double()
    b = None if st["bias"] is None else st["bias"].double()
    idx, w, joint_idx, joint, load = _select(c, z, b, torch.float64, 2.5)
    out = {"indices": idx, "weights": w, "joint_indices": joint_idx, "joint_weights": joint, "load": load}
    if not c["train"]:
        return out
    # the gradient by its formula: through the joint list, the renormalisation, then the scores
    s0, t = c["shared"], z[:, c["shared"]:]
    dead = t <= LOWEST
    g, gj = st["g_weights"].double(), st["g_joint"].double()
    if s0:
        mass = s0 + 2.5 * w.sum(1, keepdim=True)
        g = g + 2.5 * (gj[:, s0:] - (gj * joint).sum(1, keepdim=True)) / mass
    else:
        g = g + gj
    if c["score"] == "sigmoid":
        p = torch.where(dead, 0.0, torch.special.expit(torch.where(dead, 0.0, t)))
    else:
        p = torch.nan_to_num(torch.softmax(torch.where(dead, float("-inf"), t), 1))
    live = w > 0
    took = torch.where(live, p.gather(1, idx - s0), 0.0)
    if c["renorm"]:
        total = took.sum(1, keepdim=True)
        g = torch.where(total > 1e-12, (g - (g * w).sum(1, keepdim=True)) / total.clamp(min=1e-12), g / 1e-12)
    ds = torch.zeros_like(p).scatter_(1, idx - s0, torch.where(live, g, 0.0))
    dz = ds * p * (1 - p) if c["score"] == "sigmoid" else p * (ds - (ds * p).sum(1, keepdim=True))
    out["d_logits"] = torch.cat([torch.zeros_like(z[:, :s0]), torch.where(dead, 0.0, dz)], 1)
    return out


# ---- attend ------------------------------------------------------------------------------------------------------
def _prepare_attend(c, x):
    """A cache of projected rows whose magnitude differs from block to block; lists of distinct chapters, the shared one first,
    their weights as a router leaves them; ragged lists end anywhere, one of them before its first chapter."""
    heads = 2 * c["kv_heads"]
    total, width = c["chapters"] * c["rows"], heads * 64
    kv = x.normal(total, width, std=0.5, dtype=torch.bfloat16)
    kv *= torch.exp(x.normal(total // c["block"], heads, std=0.3)).to(kv.dtype).repeat_interleave(c["block"], 0).repeat_interleave(64, 1)
    data, scale = _quantize(kv, c["block"], heads)
    n = 1 + c["topk"]
    idx = torch.cat([torch.zeros(c["batch"], 1, dtype=torch.int32, device=x.dev), 1 + x.distinct(c["batch"], c["chapters"] - 1, n - 1)], 1)
    w = torch.cat([torch.ones(c["batch"], 1, device=x.dev), 2.5 * torch.softmax(x.normal(c["batch"], n - 1), 1)], 1) / 3.5
    counts = None
    if c["ragged"]:
        counts = x.integers(1, n + 1, c["batch"]).to(torch.int32)
        counts[c["batch"] // 2] = 0
    return {"case": c, "q": x.normal(c["batch"], c["queries"], c["heads"] * 64, std=4.0, dtype=torch.bfloat16), "data": data,
            "scale": scale, "idx": idx.contiguous(), "w": w.contiguous(), "counts": counts}


def _quantize(kv, block, heads):
    """(e4m3 values, fp32 scales [blocks, heads]) of [rows, heads * 64]."""
    t = kv.float().view(-1, block, heads, 64)
    scale = t.abs().amax((1, 3)) / E4M3_MAX
    s = scale[:, None, :, None]
    data = torch.where(s > 0, t / s, 0.0).to(torch.float8_e4m3fn)
    return data.view(kv.shape[0], -1), scale


def _attention(c, q, rows, scale, w, counts):
    """Joint softmax over the listed chapters' rows in the type of ``q``; ``rows`` [B, n, T, 2, HK, 64] as stored."""
    b, nq, n = q.shape[0], c["queries"], 1 + c["topk"]
    kv = (rows * scale).permute(3, 0, 4, 1, 2, 5).reshape(2, b, c["kv_heads"], 1, n * c["rows"], 64)
    u = w.repeat_interleave(c["rows"], 1).view(b, 1, 1, 1, -1)
    q = q.view(b, nq, c["kv_heads"], -1, 64).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q, kv[0].transpose(-1, -2)) * u * 0.125
    if counts is not None:
        live = torch.arange(n * c["rows"], device=q.device) < (counts * c["rows"]).view(b, 1, 1, 1, 1)
        s = torch.where(live, s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e * u, kv[1]) / torch.where(total > 0, total, 1.0)
    lse = torch.where(total > 0, torch.log(total) + top, float("-inf"))
    return out.permute(0, 3, 1, 2, 4).reshape(b, nq, -1), lse.squeeze(-1).permute(0, 3, 1, 2).reshape(b, nq, -1)


def _listed_rows(st, dtype):
    """The listed chapters' stored values and their scales, [B, n, T, 2, HK, 64] and [B, n, T, 2, HK, 1]."""
    c = st["case"]
    shape = (c["chapters"], c["rows"], 2, c["kv_heads"], 64)
    rows = st["data"].view(torch.uint8).view(shape)[st["idx"].long()].view(torch.float8_e4m3fn).to(dtype)
    scale = st["scale"].view(c["chapters"], -1, 2, c["kv_heads"], 1)[st["idx"].long()].to(dtype)
    return rows, scale.repeat_interleave(c["block"], 2)


def _plain_attend(st):
    rows, scale = _listed_rows(st, torch.float32)
    out, lse = _attention(st["case"], st["q"].float(), rows, scale, st["w"], st["counts"])
    return {"out": out.to(torch.bfloat16), "lse": lse}


def _own_attend(st):
    import memory_b200 as M
    c = st["case"]
    cache = M.ProjectedBankCache.from_quantized(st["data"], st["scale"], tokens_per_chapter=c["rows"], scale_rows=c["block"])
    out, lse = cache.attend(st["q"], st["idx"], st["w"], num_heads=c["heads"], num_kv_heads=c["kv_heads"], counts=st["counts"],
                            return_lse=True)
    return {"out": out, "lse": lse}


def _work_attend(c):
    # a chapter that several sequences list is read once
    routed = c["chapters"] - 1
    distinct = 1 + routed * (1 - (1 - c["topk"] / routed) ** c["batch"])
    share = 0.5 if c["ragged"] else 1.0
    row = 2 * c["kv_heads"] * (64 + 4 / c["block"])
    q = c["batch"] * c["queries"] * c["heads"]
    return {"bytes": distinct * (share if c["batch"] < 32 else 1.0) * c["rows"] * row + q * 64 * 4,
            "flops": 4 * 64 * q * (1 + c["topk"]) * c["rows"] * share}


def _exact_attend(st):
    c = st["case"]
    rows, scale = _listed_rows(st, torch.float64)
    kv = rows * scale
    q = st["q"].double().view(c["batch"], c["queries"], c["kv_heads"], -1, 64)
    s = torch.einsum("bqhgd,bnthd->bqhgnt", q, kv[:, :, :, 0]) * (st["w"].double()[:, None, None, None, :, None] / 8)
    if c["ragged"]:
        past = torch.arange(1 + c["topk"], device=q.device) >= st["counts"][:, None]
        s = s.masked_fill(past[:, None, None, None, :, None], float("-inf"))
    lse = s.flatten(-2).logsumexp(-1)
    p = torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[..., None, None]) * st["w"].double()[:, None, None, None, :, None]
    out = torch.einsum("bqhgnt,bnthd->bqhgd", p, kv[:, :, :, 1])
    return {"out": out.flatten(2), "lse": lse.flatten(2)}


# ---- build -------------------------------------------------------------------------------------------------------
def _prepare_build(c, x):
    kv = x.normal(c["chapters"] * c["rows"], 2 * c["kv_heads"] * 64, std=0.5, dtype=torch.bfloat16)
    kv[c["rows"]:2 * c["rows"]] = 0          # a chapter that was never written
    return {"case": c, "kv": kv}


def _plain_build(st):
    data, scale = _quantize(st["kv"], st["case"]["block"], 2 * st["case"]["kv_heads"])
    return {"values": data.to(torch.bfloat16), "scale": scale}


def _own_build(st):
    import memory_b200 as M
    c = st["case"]
    cache = M.ProjectedBankCache.from_rows(st["kv"], tokens_per_chapter=c["rows"], head_dim=64, cache_dtype=torch.float8_e4m3fn,
                                           scale_rows=c["block"])
    return {"values": cache.kv_bank.to(torch.bfloat16), "scale": cache.kv_scale}


def _work_build(c):
    n = c["chapters"] * c["rows"] * 2 * c["kv_heads"] * 64
    # (the bf16 copy of the stored values that a pass returns is written too)
    return {"bytes": n * 4 + n // (64 * c["block"]) * 4, "flops": 2 * n}


def _exact_build(st):
    # the stored values are what 8 bits leave of the quotient: no number of 64 bits stands for them
    c = st["case"]
    top = st["kv"].double().abs().view(-1, c["block"], 2 * c["kv_heads"], 64).amax(3).amax(1)
    return {"values": None, "scale": top / E4M3_MAX}


# ---- residual ----------------------------------------------------------------------------------------------------
def _prepare_residual(c, x):
    b, l, d = c["batch"], c["seq"], c["d"]
    st = {"case": c, "x": x.normal(b, l, d, std=2.0, dtype=DTYPES[c["x"]]), "f": x.normal(b, l, d, std=0.7, dtype=DTYPES[c["f"]])}
    st["w"], st["nw"] = 1 + x.normal(d, std=0.2), 1 + x.normal(d, std=0.2)
    st["b"], st["nb"] = x.normal(d, std=0.1), x.normal(d, std=0.1)
    if c["norm"] == "rms":
        st["b"] = st["nb"] = None
    if not c["following"]:
        st["nw"] = st["nb"] = None
    st["gate"] = None if c["gate"] == "none" else x.normal(*((d,) if c["gate"] == "channel" else (b, d)), std=0.5)
    st["g_y"] = x.normal(b, l, d, dtype=DTYPES[c["x"]])
    st["g_n"] = x.normal(b, l, d, dtype=DTYPES[c["f"]]) if c["following"] else None
    st["leaves"] = [k for k in ("x", "f", "w", "b", "gate", "nw", "nb") if st[k] is not None]
    if c["train"]:
        [st[k].requires_grad_(True) for k in st["leaves"]]
    return st


def _normed(kind, t, w, b):
    if kind == "layernorm":
        t = t - t.mean(-1, keepdim=True)
    t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w
    return t if b is None else t + b


def _residual_out(st, y, n):
    out = {"y": y.detach()}
    if n is not None:
        out["n"] = n.detach()
    if st["case"]["train"]:
        outs, gs = ([y, n], [st["g_y"], st["g_n"]]) if n is not None else ([y], [st["g_y"]])
        grads = torch.autograd.grad(outs, [st[k] for k in st["leaves"]], gs)
        out |= {"d_" + k: g for k, g in zip(st["leaves"], grads)}
    return out


def _plain_residual(st):
    c = st["case"]
    z = _normed(c["norm"], st["f"].float(), st["w"], st["b"])
    if st["gate"] is not None:
        z = z * (st["gate"] if c["gate"] == "channel" else st["gate"][:, None])
    y = 0.75 * st["x"].float() + z
    n = _normed(c["norm"], y, st["nw"], st["nb"]).to(DTYPES[c["f"]]) if c["following"] else None
    return _residual_out(st, y.to(DTYPES[c["x"]]), n)


def _own_residual(st):
    import memory_b200 as M
    c = st["case"]
    got = M.gated_residual_norm(st["x"], st["f"], st["w"], st["b"], norm_type=c["norm"], eps=1e-6, gate=st["gate"], residual_scale=0.75,
                                next_weight=st["nw"], next_bias=st["nb"])
    y, n = got if c["following"] else (got, None)
    return _residual_out(st, y, n)


def _work_residual(c):
    x, f = (4 if c["x"] == "fp32" else 2), (4 if c["f"] == "fp32" else 2)
    n = c["batch"] * c["seq"] * c["d"]
    size = x + f + x + (f if c["following"] else 0)
    if c["train"]:
        size += x + (f if c["following"] else 0) + x + f       # (x and f are counted once, with the forward pass)
    return {"bytes": n * size + 8 * 4 * c["d"], "flops": n * (40 if c["train"] else 12)}


def _exact_residual(st):
    c = st["case"]
    t = {k: st[k].detach().double() for k in st["leaves"]}
    rows, d = c["batch"] * c["seq"], c["d"]

    def stats(v):
        m = v.sum(1, keepdim=True) / d if c["norm"] == "layernorm" else torch.zeros_like(v[:, :1])
        return (v - m) / torch.sqrt(((v - m) ** 2).sum(1, keepdim=True) / d + 1e-6), 1 / torch.sqrt(((v - m) ** 2).sum(1, keepdim=True) / d + 1e-6)

    def back(g, hat, inv):
        g0 = g.sum(1, keepdim=True) / d if c["norm"] == "layernorm" else 0.0
        return inv * (g - g0 - hat * (g * hat).sum(1, keepdim=True) / d)
    fh, fi = stats(t["f"].reshape(rows, d))
    z = fh * t["w"] + t.get("b", 0.0)
    gate = t["gate"].expand(c["batch"], d).repeat_interleave(c["seq"], 0) if "gate" in t else torch.ones_like(z)
    y = 0.75 * t["x"].reshape(rows, d) + gate * z
    out = {"y": y.view(st["x"].shape)}
    yh, yi = stats(y)
    if c["following"]:
        out["n"] = (yh * t["nw"] + t.get("nb", 0.0)).view(st["x"].shape)
    if not c["train"]:
        return out
    g = st["g_y"].double().reshape(rows, d)
    if c["following"]:
        gn = st["g_n"].double().reshape(rows, d)
        g = g + back(gn * t["nw"], yh, yi)
        out["d_nw"], out["d_nb"] = (gn * yh).sum(0), gn.sum(0)
    gz = g * gate
    out["d_x"], out["d_f"] = (0.75 * g).view(st["x"].shape), back(gz * t["w"], fh, fi).view(st["x"].shape)
    out["d_w"], out["d_b"] = (gz * fh).sum(0), gz.sum(0)
    if "gate" in t:
        out["d_gate"] = (g * z).view(c["batch"], c["seq"], d).sum(1) if c["gate"] == "sequence" else (g * z).sum(0)
    names = ["y"] + (["n"] if c["following"] else []) + ["d_" + k for k in st["leaves"]]
    return {k: out[k] for k in names}


# ---- clip --------------------------------------------------------------------------------------------------------
def _prepare_clip(c, x):
    """Gradients of a stack of blocks (four attention and two MLP matrices, two norms each), an embedding, and the bank's compact
    gradient, whose rows behind the touched chapters hold nothing; a mean over two ranks is still to be taken of the bank's."""
    d = c["d"]
    shapes = [(d, d)] * 4 + [(4 * d, d), (d, 4 * d), (d,), (d,)]
    shapes = shapes * c["layers"] + [(c["vocab"], d), (d,)]
    dtype = DTYPES[c["dtype"]]
    st = {"case": c, "grads": [x.normal(*s, std=1e-3, dtype=dtype) for s in shapes]}
    # the clipped gradients go to one flat buffer, as an exchange or a flat optimizer has them
    st["flat"] = torch.empty(sum(g.numel() for g in st["grads"]), dtype=dtype, device=x.dev)
    st["out"] = [p.view(g.shape) for p, g in zip(st["flat"].split([g.numel() for g in st["grads"]]), st["grads"])]
    spare = c["touched"] // 8 + 1
    st["bank"] = x.normal((c["touched"] + spare) * c["rows"], d, std=2e-3)
    st["bank"][c["touched"] * c["rows"]:] = float("nan")
    st["ids"] = torch.arange(c["touched"] + spare, dtype=torch.int32, device=x.dev)
    st["count"] = torch.full((1,), c["touched"], dtype=torch.int32, device=x.dev)
    return st


def _plain_clip(st):
    c = st["case"]
    square = [g.float().square().sum(dtype=torch.float64) for g in st["grads"]]
    live = torch.arange(st["bank"].shape[0], device=st["bank"].device) < st["count"] * c["rows"]
    bank = torch.where(live[:, None], st["bank"], 0.0).square().sum(dtype=torch.float64) * 0.25
    norm = torch.sqrt(torch.stack(square + [bank]).sum())
    coef = (c["max_norm"] / (norm + CLIP_EPS)).clamp(max=1.0).float()
    return {"norm": norm.float(), "coefficient": coef, "grads": (torch.cat([g.flatten() for g in st["grads"]]).float() * coef).to(st["flat"].dtype)}


def _own_clip(st):
    import memory_b200 as M
    c = st["case"]
    bank = M.SparseBankGrad()
    bank.add(st["ids"], st["count"], st["bank"], c["rows"])
    bank.scale = 0.5
    got = M.clip_grad_norm_(st["grads"], c["max_norm"], bank_grads=[bank], out=st["out"])
    return {"norm": got.total_norm, "coefficient": got.coefficient, "grads": st["flat"]}


def _work_clip(c):
    d, size = c["d"], 4 if c["dtype"] == "fp32" else 2
    n = c["layers"] * (12 * d * d + 2 * d) + (c["vocab"] + 1) * d
    bank = c["touched"] * c["rows"] * d
    return {"bytes": 2 * n * size + 4 * bank, "flops": 3 * n + 2 * bank}


def _exact_clip(st):
    c = st["case"]
    total = sum(float((g.double() ** 2).sum()) for g in st["grads"])
    total += 0.25 * float((st["bank"][:c["touched"] * c["rows"]].double() ** 2).sum())
    norm = math.sqrt(total)
    coef = min(1.0, c["max_norm"] / (norm + CLIP_EPS))
    like = dict(dtype=torch.float64, device=st["bank"].device)
    return {"norm": torch.tensor(norm, **like), "coefficient": torch.tensor(coef, **like), "grads": torch.cat([g.flatten() for g in st["grads"]]).double() * coef}

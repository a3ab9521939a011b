"""What the serving operators are measured on: a paged key/value cache that grows and
shrinks on the GPU, rotary positions written into it, attention of drafted-token trees
over it, and the logits' penalties, biases and grammar masks.

`run` computes an operator in its plain form (elementary torch operations in 32 bits)
or, where `own` is true, calls this repository's operator.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # A decoding step of a busy server: one new token each for 64 requests.
        {"name": "grow_decode_64", "op": "grow", "requests": 64, "block": 16, "context": 4096,
         "new": 1, "pool": 1.0},
        # Prompts of odd lengths arriving at once, more than the pool can take.
        {"name": "grow_prompts_512", "op": "grow", "requests": 512, "block": 64, "context": 30000,
         "new": 255, "pool": 0.8},
        # Drafts taken back and finished requests freed.
        {"name": "release_1000", "op": "release", "requests": 1000, "block": 32, "context": 9000},
        # A decoding step's queries, keys and values, keys and values into the cache.
        {"name": "rope_append_decode_64", "op": "rope_append", "tokens": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "axes": 1, "cycled": False, "paired": False,
         "block": 16, "dtype": "bf16", "skip": 0.0},
        # A chunk of a prompt with images: three axes; some tokens were rejected by the pool.
        {"name": "rope_append_chunk_8192", "op": "rope_append", "tokens": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "axes": 3, "cycled": True, "paired": False,
         "block": 64, "dtype": "f16", "skip": 0.05},
        # The gradient through the rotation of a vision encoder: two axes, an odd token count.
        {"name": "rope_inverse_20001", "op": "rope", "tokens": 20001, "heads": 16,
         "kv_heads": 16, "dim": 80, "rotary": 80, "axes": 2, "cycled": False, "paired": True,
         "dtype": "f32", "inverse": True},
        # One request with a small tree of drafts over a short context: latency.
        {"name": "tree_one_request", "op": "attention", "requests": 1, "context": 700, "new": 12,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 16, "dtype": "bf16", "tree": True},
        # Plain decoding: 64 requests with contexts from nearly nothing to 8192.
        {"name": "decode_64_to_8192", "op": "attention", "requests": 64, "context": 8192, "new": 1,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 16, "dtype": "bf16", "tree": False},
        # Drafts over two very long contexts: the work is split over the keys.
        {"name": "tree_long_131072", "op": "attention", "requests": 2, "context": 131072, "new": 7,
         "heads": 64, "kv_heads": 8, "dim": 128, "block": 64, "dtype": "f16", "tree": True},
        # Wide trees for a batch: 256 rows and more share each key head.
        {"name": "tree_wide_64", "op": "attention", "requests": 24, "context": 6000, "new": 64,
         "heads": 32, "kv_heads": 4, "dim": 128, "block": 32, "dtype": "bf16", "tree": True},
        # A few requests' logits, odd vocabulary.
        {"name": "logits_3", "op": "logits", "rows": 3, "vocab": 50001, "history": 900,
         "biases": 40, "grammar": True, "dtype": "f32", "out": "f32"},
        # Every row of a large batch of drafts, long histories.
        {"name": "logits_256", "op": "logits", "rows": 256, "vocab": 131072, "history": 8192,
         "biases": 300, "grammar": True, "dtype": "bf16", "out": "f32"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["grow", "release", "rope_append", "rope", "attention", "attention",
                     "attention", "logits", "logits"])
    if op in ("grow", "release"):
        c = {"op": op, "requests": _log(rng, 1, 2048), "block": rng.choice([8, 16, 24, 32, 64, 128]),
             "context": _log(rng, 1, 40000)}
        if op == "grow":
            c.update(new=_log(rng, 1, max(1, 131072 // c["requests"])),
                     pool=rng.choice([0.3, 0.8, 1.0, 1.0]))
        return c
    if op in ("rope_append", "rope"):
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        rotary = rng.choice([dim, dim, dim // 2])
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * rng.choice([1, 2, 4, 7, 8])
        heads = min(heads, 64 // kv * kv)
        c = {"op": op, "tokens": _log(rng, 1, 12000), "heads": heads, "kv_heads": kv, "dim": dim,
             "rotary": rotary, "axes": rng.choice([1, 1, 2, 3, 4]),
             "cycled": rng.random() < 0.5, "paired": rng.random() < 0.3,
             "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
        if op == "rope_append":
            c.update(block=rng.choice([8, 16, 24, 64]), skip=rng.choice([0.0, 0.0, 0.1]))
        else:
            c["inverse"] = rng.random() < 0.5
        return c
    if op == "attention":
        kv = rng.choice([1, 2, 4, 8, 8, 16])
        group = rng.choice([1, 2, 4, 5, 8])
        new = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 160)])
        requests = _log(rng, 1, 128)
        # keys x (their bytes, and the rows that read them) bound the cost by the listed cases'
        most = min(2.2e6 / (requests * kv), 1.2e8 / (requests * kv * group * new), 100000)
        dim = rng.choice([64, 128, 128])
        dtype = rng.choice(["bf16", "bf16", "f16"])
        if rng.random() < 0.1:  # types and head sizes that are rare in serving
            dim, dtype, most = rng.choice([(80, "bf16", most / 16), (128, "f32", most / 16)])
        return {"op": op, "requests": requests, "context": _log(rng, min(20, most), most),
                "new": new, "heads": kv * group, "kv_heads": kv, "dim": dim,
                "block": rng.choice([8, 16, 16, 24, 32, 64, 128]), "dtype": dtype,
                "tree": rng.random() < 0.7}
    vocab = _log(rng, 1000, 160000)
    dtype = rng.choice(["bf16", "f16", "f32"])
    return {"op": op, "rows": _log(rng, 1, min(1024, 33000000 // vocab)), "vocab": vocab,
            "history": _log(rng, 1, 8192), "biases": rng.choice([0, 1, 20, 300]),
            "grammar": rng.random() < 0.6, "dtype": dtype, "out": rng.choice(["f32", dtype])}


# ---- inputs ------------------------------------------------------------------------------


def _ints(g, low, high, *shape):
    return torch.randint(low, high, shape, generator=g, device="cuda", dtype=torch.int32)


def _spread(g, low, high, n):
    """n whole numbers from low to high, evenly spread and shuffled: their sum is the same for
    every seed."""
    at = torch.arange(n, device="cuda", dtype=torch.float64) / max(1, n - 1)
    every = (high - (high - low) * at).round().to(torch.int32)
    return every[torch.randperm(n, generator=g, device="cuda")]


def _cu(lens):
    cu = torch.zeros(lens.numel() + 1, dtype=torch.int32, device="cuda")
    cu[1:] = torch.cumsum(lens, 0)
    return cu


def _tables(g, lens, block, columns):
    """A block table for requests of `lens` tokens (unused entries -1), and the number of blocks."""
    blocks = (lens + block - 1) // block
    total = int(blocks.sum())
    order = torch.randperm(max(1, total), generator=g, device="cuda").to(torch.int32)
    first = torch.cumsum(blocks, 0) - blocks
    col = torch.arange(columns, device="cuda")
    at = (first[:, None] + col).clamp(max=max(0, total - 1))
    return torch.where(col < blocks[:, None], order[at], -1).to(torch.int32), max(1, total)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op = case["op"]
    s = {"op": op, "case": case}
    if op in ("grow", "release"):
        n, block = case["requests"], case["block"]
        lens = _spread(g, 0, case["context"], n)
        if op == "grow":
            new = _spread(g, 1, 2 * case["new"] - 1, n)
            tokens = int(new.sum())
            columns = (case["context"] + 2 * case["new"]) // block + 2
            need = int(((lens + new + block - 1) // block - (lens + block - 1) // block).sum())
            count = int(math.ceil(need * case["pool"])) + 1
            s.update(new=new, tokens=tokens)
        else:
            keep = torch.minimum(lens, (lens * torch.rand(n, generator=g, device="cuda") * 1.3).int())
            columns = case["context"] // block + 2
            count = 100
            s.update(keep=keep)
        table, used = _tables(g, lens, block, columns)
        free = torch.full((count + used,), -1, dtype=torch.int32, device="cuda")
        free[:count] = used + torch.randperm(count, generator=g, device="cuda").int()
        s.update(lens=lens, table=table, free=free, block=block,
                 count=torch.full((1,), count, dtype=torch.int32, device="cuda"),
                 left=torch.zeros(1, dtype=torch.int32, device="cuda"))
        if op == "grow":
            s.update(slots=torch.zeros(tokens, dtype=torch.int32, device="cuda"),
                     positions=torch.zeros(tokens, dtype=torch.int32, device="cuda"),
                     cu=torch.zeros(n + 1, dtype=torch.int32, device="cuda"),
                     after=torch.zeros(n, dtype=torch.int32, device="cuda"))
        return s
    if op in ("rope_append", "rope"):
        t, h, hk, d, dt = (case["tokens"], case["heads"], case["kv_heads"], case["dim"],
                           DTYPES[case["dtype"]])
        # one packed projection's output: q, k and v are strided views of its rows
        packed = torch.randn(t, (h + 2 * hk) * d, generator=g, device="cuda").to(dt)
        q, k, v = packed.split([h * d, hk * d, hk * d], dim=1)
        pairs = case["rotary"] // 2
        last = 32768
        angle = (torch.arange(last, device="cuda", dtype=torch.float64)[:, None]
                 * 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs))
        s.update(q=q.unflatten(1, (h, d)), k=k.unflatten(1, (hk, d)), v=v.unflatten(1, (hk, d)),
                 cos_sin=torch.cat([angle.cos(), angle.sin()], 1).float(),
                 positions=_ints(g, 0, last, case["axes"], t))
        axes = case["axes"]
        if case["cycled"]:
            axis = [i % axes for i in range(pairs)]
        else:
            axis = sorted(i * axes // pairs for i in range(pairs))
        s.update(axis=axis, axis_gpu=torch.tensor(axis, device="cuda"), pairs=pairs,
                 paired=case["paired"], q_out=torch.empty(t, h, d, dtype=dt, device="cuda"))
        if op == "rope":
            s.update(inverse=case["inverse"], k_out=torch.empty(t, hk, d, dtype=dt, device="cuda"))
            return s
        block = case["block"]
        blocks = 2 * t // block + 2
        slots = torch.randperm(blocks * block, generator=g, device="cuda")[:t].int()
        skip = torch.rand(t, generator=g, device="cuda") < case["skip"]
        s.update(slots=torch.where(skip, -1, slots))
        for name in ("k_cache", "v_cache"):
            s[name] = torch.randn(blocks, block, hk, d, generator=g, device="cuda").to(dt)
        return s
    if op == "attention":
        n, block, hk, d, dt = (case["requests"], case["block"], case["kv_heads"], case["dim"],
                               DTYPES[case["dtype"]])
        new = _spread(g, (case["new"] + 1) // 2, case["new"], n)
        old = _spread(g, 0, case["context"], n)
        kv = old + new
        tokens, longest = int(new.sum()), int(kv.max())
        table, used = _tables(g, kv, block, (longest + block - 1) // block)
        cache = lambda: torch.randn(used, block, hk, d, generator=g, device="cuda").to(dt)  # noqa: E731
        s.update(q=torch.randn(tokens, case["heads"], d, generator=g, device="cuda").to(dt),
                 k_cache=cache(), v_cache=cache(), table=table, cu=_cu(new), kv=kv, mask=None,
                 scale=d ** -0.5, widest=case["new"], longest=longest, block=block,
                 out=torch.empty(tokens, case["heads"], d, dtype=dt, device="cuda"),
                 lse=torch.empty(tokens, case["heads"], device="cuda"))
        if case["tree"]:
            # each draft follows an earlier one of its request, often the one before it
            words = (case["new"] + 31) // 32
            at = torch.arange(tokens, device="cuda")
            i = at - torch.repeat_interleave(s["cu"][:-1].long(), new.long(), output_size=tokens)
            far = (torch.rand(tokens, generator=g, device="cuda") ** 3 * 6).long() + 1
            parent = torch.where(i == 0, -1, (i - far).clamp(min=0))
            seen = torch.zeros(tokens, words * 32, dtype=torch.bool, device="cuda")
            start = at - i
            for j in range(case["new"]):  # j-th drafts of all requests at once
                who = at[i == j]
                if j:
                    seen[who] = seen[start[who] + parent[who]]
                seen[who, j] = True
            bit = 1 << torch.arange(32, device="cuda", dtype=torch.int64)
            s["mask"] = (seen.view(tokens, words, 32) * bit).sum(2).to(torch.int32)
        return s
    r, v, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    lens = _spread(g, 0, case["history"], r)
    total = int(lens.sum())
    # tokens repeat as text does: a few are frequent
    tokens = (torch.rand(total, generator=g, device="cuda") ** 4 * v).int().clamp(max=v - 1)
    prompt = (lens * torch.rand(r, generator=g, device="cuda")).int()
    uniform = lambda lo, hi: lo + (hi - lo) * torch.rand(r, generator=g, device="cuda")  # noqa: E731
    s.update(logits=(4 * torch.randn(r, v, generator=g, device="cuda")).to(dt), tokens=tokens,
             cu=_cu(lens), prompt=prompt, repetition=uniform(1.0, 1.5), presence=uniform(-0.5, 1.0),
             frequency=uniform(0.0, 0.5), bias_ids=None, bias_values=None, bias_cu=None,
             allowed=None, out=torch.empty(r, v, dtype=DTYPES[case["out"]], device="cuda"),
             out_dtype=DTYPES[case["out"]])
    if case["biases"]:
        blens = _spread(g, 0, case["biases"], r)
        total = int(blens.sum())
        s.update(bias_ids=_ints(g, 0, v, total), bias_cu=_cu(blens),
                 bias_values=3 * torch.randn(total, generator=g, device="cuda"))
    if case["grammar"]:
        words = (v + 31) // 32
        a, b = (_ints(g, -2 ** 31, 2 ** 31 - 1, r, words) for _ in range(2))
        s["allowed"] = a & b
    return s


# ---- the operators -------------------------------------------------------------------------


def _grow(s):
    lens, new, block = s["lens"].long(), s["new"].long(), s["block"]
    had, need = (lens + block - 1) // block, (lens + new + block - 1) // block
    fits = need <= s["table"].shape[1]
    want = torch.where(fits, need - had, 0)
    end = torch.cumsum(want, 0)
    count = s["count"].long()
    ok = fits & ((want == 0) | (end <= count))
    s["cu"][1:] = torch.cumsum(new, 0)
    s["after"].copy_(torch.where(ok, lens + new, lens))
    s["left"].copy_(count - torch.where(ok & (want > 0), end, 0).max())
    col = torch.arange(s["table"].shape[1], device="cuda")
    fresh = ok[:, None] & (col >= had[:, None]) & (col < need[:, None])
    at = count - 1 - ((end - want)[:, None] + col - had[:, None])
    s["table"].copy_(torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1)], s["table"]))
    t = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(s["cu"][1:].long(), t, right=True).clamp(max=new.numel() - 1)
    pos = lens[b] + t - s["cu"][b]
    entry = s["table"][b, (pos // block).clamp(max=col.numel() - 1)].long()
    s["positions"].copy_(pos)
    s["slots"].copy_(torch.where(ok[b] & (entry >= 0), entry * block + pos % block, -1))
    return [s["table"], s["slots"], s["positions"], s["cu"], s["after"], s["left"]]


def _release(s):
    block = s["block"]
    first = (s["keep"].long() + block - 1) // block
    gone = (s["lens"].long() + block - 1) // block - first
    start = torch.cumsum(gone, 0) - gone
    col = torch.arange(s["table"].shape[1], device="cuda")
    which = (col >= first[:, None]) & (col < (first + gone)[:, None])
    at = s["count"] + start[:, None] + col - first[:, None]
    s["free"][at[which]] = s["table"][which]
    s["left"].copy_(s["count"] + gone.sum())
    return [s["free"], s["left"]]


def _rotate(x, cos, sin, paired, dtype):
    """x [tokens, heads, dim] with its first 2 * pairs elements rotated."""
    pairs = cos.shape[1]
    x = x.float()
    a, b = ((x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) if paired else
            (x[..., :pairs], x[..., pairs:2 * pairs]))
    cos, sin = cos[:, None], sin[:, None]
    y = x.clone()
    if paired:
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = a * cos - b * sin, b * cos + a * sin
    else:
        y[..., :pairs], y[..., pairs:2 * pairs] = a * cos - b * sin, b * cos + a * sin
    return y.to(dtype)


def _rope(s):
    at = s["positions"][s["axis_gpu"]].t().long()
    cos = s["cos_sin"][:, :s["pairs"]].gather(0, at)
    sin = s["cos_sin"][:, s["pairs"]:].gather(0, at)
    if s.get("inverse"):
        sin = -sin
    q = _rotate(s["q"], cos, sin, s["paired"], s["q"].dtype)
    k = _rotate(s["k"], cos, sin, s["paired"], s["k"].dtype)
    if s["op"] == "rope":
        return [q, k]
    keep = s["slots"] >= 0
    to = s["slots"][keep].long()
    s["k_cache"].flatten(0, 1)[to] = k[keep]
    s["v_cache"].flatten(0, 1)[to] = s["v"][keep]
    return [q, s["k_cache"], s["v_cache"]]


def _attention(s):
    q, cu, kv = s["q"], s["cu"].long(), s["kv"].long()
    hk = s["k_cache"].shape[2]
    n, tokens = kv.numel(), q.shape[0]
    new = cu[1:] - cu[:-1]
    i, pos = torch.arange(s["widest"], device="cuda"), torch.arange(s["longest"], device="cuda")
    rows = (cu[:-1, None] + i).clamp(max=tokens - 1)
    entry = s["table"][:, pos // s["block"]].long()
    slot = (entry * s["block"] + pos % s["block"]).clamp(min=0)
    k, v = (s[x].flatten(0, 1)[slot].float() for x in ("k_cache", "v_cache"))
    qs = q[rows].float().unflatten(2, (hk, -1))
    draft = pos - (kv - new)[:, None]
    if s["mask"] is None:
        inside = draft[:, None] <= i[:, None]
    else:
        j = draft.clamp(0, s["mask"].shape[1] * 32 - 1)
        word = s["mask"][rows].long().gather(2, (j >> 5)[:, None].expand(-1, i.numel(), -1))
        inside = (draft[:, None] < 0) | ((word >> (j & 31)[:, None]) & 1 == 1)
    visible = (inside & (pos < kv[:, None])[:, None])[:, None, None]
    scores = torch.einsum("bnhgd,blhd->bhgnl", qs, k) * s["scale"]
    scores = torch.where(visible, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1)
    o = torch.einsum("bhgnl,blhd->bnhgd", p, v)
    per = total.permute(0, 3, 1, 2)
    o = o / torch.where(per == 0, 1, per)[..., None]
    lse = (top[..., 0] + torch.log(total)).permute(0, 3, 1, 2)
    t = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(cu[1:], t, right=True)
    at = t - cu[b]
    return [o[b, at].flatten(1, 2).to(q.dtype), lse[b, at].flatten(1)]


def _logits(s):
    x = s["logits"].float()
    r, v = x.shape
    row = torch.arange(r, device="cuda")
    lens = (s["cu"][1:] - s["cu"][:-1]).long()
    total = s["tokens"].numel()
    of = torch.repeat_interleave(row, lens, output_size=total)
    at = of * v + s["tokens"]
    generated = torch.arange(total, device="cuda") - s["cu"][of] >= s["prompt"][of]
    seen = torch.zeros(r * v, dtype=torch.bool, device="cuda")
    seen[at] = True
    count = torch.zeros(r * v, device="cuda").index_add_(0, at, generated.float()).view(r, v)
    rep = s["repetition"][:, None]
    x = torch.where(seen.view(r, v), torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_ids"] is not None:
        total = s["bias_ids"].numel()
        of = torch.repeat_interleave(row, (s["bias_cu"][1:] - s["bias_cu"][:-1]).long(),
                                     output_size=total)
        entry = torch.full((r * v,), -1, dtype=torch.int64, device="cuda")
        entry.scatter_reduce_(0, of * v + s["bias_ids"], torch.arange(total, device="cuda"), "amax")
        entry = entry.view(r, v)
        x = x + torch.where(entry >= 0, s["bias_values"][entry.clamp(min=0)], 0)
    if s["allowed"] is not None:
        col = torch.arange(v, device="cuda")
        x = torch.where((s["allowed"][:, col >> 5] >> (col & 31).int()) & 1 == 1, x, -math.inf)
    return [x.to(s["out_dtype"])]


def run(s):
    op = s["op"]
    if not own:
        return {"grow": _grow, "release": _release, "rope": _rope, "rope_append": _rope,
                "attention": _attention, "logits": _logits}[op](s)
    import matcoredsl_b200 as mcb
    if op == "grow":
        mcb.paged_grow(s["table"], s["lens"], s["new"], s["free"], s["count"], s["block"],
                       out=(s["slots"], s["positions"], s["cu"], s["after"], s["left"]))
        return [s["table"], s["slots"], s["positions"], s["cu"], s["after"], s["left"]]
    if op == "release":
        mcb.paged_release(s["table"], s["lens"], s["keep"], s["free"], s["count"], s["block"],
                          out=s["left"])
        return [s["free"], s["left"]]
    if op == "rope":
        mcb.rope(s["q"], s["k"], s["cos_sin"], s["positions"], axis_map=s["axis"],
                 paired=s["paired"], inverse=s["inverse"], out=(s["q_out"], s["k_out"]))
        return [s["q_out"], s["k_out"]]
    if op == "rope_append":
        mcb.rope_append(s["q"], s["k"], s["v"], s["cos_sin"], s["positions"], s["slots"],
                        s["k_cache"], s["v_cache"], axis_map=s["axis"], paired=s["paired"],
                        out=s["q_out"])
        return [s["q_out"], s["k_cache"], s["v_cache"]]
    if op == "attention":
        mcb.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["kv"],
                           s["mask"], scale=s["scale"], out=s["out"], lse=s["lse"])
        return [s["out"], s["lse"]]
    mcb.adjust_logits(s["logits"], s["tokens"], s["cu"], s["prompt"], repetition=s["repetition"],
                      presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"],
                      bias_values=s["bias_values"], bias_cu=s["bias_cu"], allowed=s["allowed"],
                      out=s["out"])
    return [s["out"]]


# ---- work and exact values -----------------------------------------------------------------


def work(case):
    """Bytes and operations that a pass cannot do without, at the sizes' expected values (the
    ragged ones are uniform)."""
    op = case["op"]
    if op == "grow":
        n, tokens = case["requests"], case["requests"] * case["new"]
        blocks = case["pool"] * tokens / case["block"]
        return {"bytes": 16 * n + 8 * tokens + 8 * blocks + 4 * n, "flops": 0}
    if op == "release":
        n = case["requests"]
        return {"bytes": 8 * n + 8 * 0.45 * n * case["context"] / 2 / case["block"], "flops": 0}
    if op in ("rope", "rope_append"):
        t, h, hk, d, e = (case["tokens"], case["heads"], case["kv_heads"], case["dim"],
                          SIZE[case["dtype"]])
        ins = (h + hk * (2 if op == "rope_append" else 1)) * d * e
        read = t * (ins + 4 * case["axes"] + (4 if op == "rope_append" else 0))
        table = min(t * case["axes"], 32768) * case["rotary"] * 4 // case["axes"]
        kept = 1 - case.get("skip", 0.0)
        out = t * (h * d * e + kept * (ins - h * d * e))
        return {"bytes": read + table + out, "flops": 3 * t * (h + hk) * case["rotary"]}
    if op == "attention":
        n, d, e = case["requests"], case["dim"], SIZE[case["dtype"]]
        new = case["new"] + (n - 1) * ((case["new"] + 1) // 2 + case["new"]) / 2
        keys = case["context"] + (n - 1) * case["context"] / 2 + new
        rows = new * case["heads"]
        wide = 32 if not case["tree"] else (case["new"] + 31) // 32 * 32
        return {"bytes": 2 * keys * case["kv_heads"] * d * e + rows * (2 * d * e + 4) + 8 * n
                + 4 * keys / case["block"] + (new * wide / 8 if case["tree"] else 0),
                "flops": 4 * d * rows * keys / n}
    r, v = case["rows"], case["vocab"]
    history = case["history"] * (r + 1) / 2
    return {"bytes": r * v * (SIZE[case["dtype"]] + SIZE[case["out"]]) + 4 * history + 24 * r
            + 8 * case["biases"] * (r + 1) / 2 + (r * ((v + 31) // 32) * 4 if case["grammar"] else 0),
            "flops": 4 * r * v}


def exact(case, seed):
    op = case["op"]
    if op in ("grow", "release"):
        return None  # whole numbers: the plain form's are exact
    s = prepare(case, seed)
    if op in ("rope", "rope_append"):
        # as a complex product: (a + ib)(cos + i sin)
        turn = torch.zeros(case["tokens"], s["pairs"], dtype=torch.complex128, device="cuda")
        for i, axis in enumerate(s["axis"]):
            cs = s["cos_sin"].double()[s["positions"][axis].long()]
            turn[:, i] = torch.complex(cs[:, i], cs[:, s["pairs"] + i])
        if s.get("inverse"):
            turn = turn.conj()

        def turned(x):
            x = x.double()
            r = 2 * s["pairs"]
            if s["paired"]:
                z = torch.view_as_complex(x[..., :r].unflatten(-1, (-1, 2)).contiguous())
                y = torch.view_as_real(z * turn[:, None]).flatten(-2)
            else:
                z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * turn[:, None]
                y = torch.cat([z.real, z.imag], -1)
            return torch.cat([y, x[..., r:]], -1)

        if op == "rope":
            return [turned(s["q"]), turned(s["k"])]
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        keep = (s["slots"] >= 0).nonzero()[:, 0]
        kc.view(-1, *kc.shape[2:]).index_copy_(0, s["slots"][keep].long(), turned(s["k"])[keep])
        vc.view(-1, *vc.shape[2:]).index_copy_(0, s["slots"][keep].long(), s["v"].double()[keep])
        return [turned(s["q"]), kc, vc]
    if op == "attention":
        hk = case["kv_heads"]
        out, lse = [], []
        cu, kv = s["cu"].tolist(), s["kv"].tolist()
        for b in range(case["requests"]):
            n, length = cu[b + 1] - cu[b], kv[b]
            pages = s["table"][b, :(length + case["block"] - 1) // case["block"]].long()
            hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
            if s["mask"] is not None:
                for j in range(n):
                    hidden[:, j] = (s["mask"][cu[b]:cu[b + 1], j // 32] >> (j % 32)) & 1 == 0
            o, z = [], []
            for h in range(hk):
                k = s["k_cache"][pages, :, h].flatten(0, 1)[:length].double()
                v = s["v_cache"][pages, :, h].flatten(0, 1)[:length].double()
                q = s["q"][cu[b]:cu[b + 1]].double().unflatten(1, (hk, -1))[:, h]
                a = q @ k.t() * s["scale"]
                a[:, :, length - n:].masked_fill_(hidden[:, None], -math.inf)
                o.append(torch.softmax(a, -1) @ v)
                z.append(torch.logsumexp(a, -1))
            out.append(torch.stack(o, 1).flatten(1, 2))
            lse.append(torch.stack(z, 1).flatten(1))
        return [torch.cat(out), torch.cat(lse)]
    rows = []
    cu, prompt = s["cu"].tolist(), s["prompt"].tolist()
    bias_cu = s["bias_cu"].tolist() if case["biases"] else None
    rep, pre, fre = (s[x].double().tolist() for x in ("repetition", "presence", "frequency"))
    v = case["vocab"]
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        history = s["tokens"][cu[r]:cu[r + 1]].long()
        known = torch.unique(history)
        y = x[known]
        x[known] = torch.where(y > 0, y / rep[r], y * rep[r])
        count = torch.bincount(history[prompt[r]:], minlength=v).double()
        x = x - fre[r] * count - pre[r] * (count > 0)
        if bias_cu:
            ids = s["bias_ids"][bias_cu[r]:bias_cu[r + 1]].tolist()
            values = s["bias_values"][bias_cu[r]:bias_cu[r + 1]].tolist()
            last = dict(zip(ids, values))
            if last:
                where = torch.tensor(list(last), device="cuda")
                x[where] += torch.tensor(list(last.values()), dtype=torch.float64, device="cuda")
        if case["grammar"]:
            words = s["allowed"][r].long() & 0xFFFFFFFF
            bits = (words[:, None] >> torch.arange(32, device="cuda")) & 1
            x[bits.flatten()[:v] == 0] = -math.inf
        rows.append(x)
    return [torch.stack(rows)]

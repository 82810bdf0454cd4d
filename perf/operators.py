"""Cases and plain forms of the batched serving operators: the append to a paged KV cache with norm and rotation on
the way, attention of a batch over a shared prefix and each sequence's own pages, and the verification of drafted
tokens by sampling.  `own` selects the framework's kernels; otherwise everything is elementary torch."""
import math

import torch

own = False

GEOMS = [(24, 4, 256), (32, 8, 128), (8, 1, 256), (16, 16, 128), (40, 8, 128)]      # query heads, kv heads, head dim


def listed():
    def append(name, seqs, lo, hi, start, geom, rd, inter, scaling, norm, gated, fp8, page, base):
        return dict(name=name, op="append", seqs=seqs, lo=lo, hi=hi, start=start, hq=geom[0], hkv=geom[1], d=geom[2], rd=rd, inter=inter,
                    scaling=scaling, norm=norm, gated=gated, fp8=fp8, page=page, base=base)

    def attn(name, seqs, m, prefix, lo, hi, geom, fp8, page, pad=0):
        return dict(name=name, op="attn", seqs=seqs, m=m, prefix=prefix, lo=lo, hi=hi, hq=geom[0], hkv=geom[1], d=geom[2], fp8=fp8, page=page, pad=pad)

    def verify(name, seqs, k, vocab, agree, sampled, dtype):
        return dict(name=name, op="verify", seqs=seqs, k=k, vocab=vocab, agree=agree, sampled=sampled, dtype=dtype)

    a, b = GEOMS[0], GEOMS[1]
    return [
        # one new token of one conversation: latency
        append("append one token", 1, 1, 1, 4096, a, 64, False, "none", True, True, True, 64, 0),
        # four prompts of unequal length filled in one call
        append("append prompts", 4, 1024, 3000, 0, a, 64, False, "none", True, True, True, 64, 0),
        # a chunk for many conversations far into a context that was stretched, whole heads rotated in neighbouring pairs
        append("append far chunk", 37, 1, 40, 20000, b, 128, True, "yarn", False, False, False, 16, 1000000),
        # one conversation without a shared prompt
        attn("attend one", 1, 1, 0, 1000, 1000, a, True, 64),
        # a chat server: a long system prompt shared by the batch, conversations of every length
        attn("attend chats", 64, 1, 8192, 1, 2048, a, True, 64),
        # a verify step of drafts, one slot of the captured batch empty
        attn("attend drafts", 16, 5, 4099, 1, 1024, a, True, 32, 1),
        # small pages, 128-dim heads, a prefix that ends inside a tile
        attn("attend small pages", 33, 1, 1111, 1, 700, b, False, 16),
        # many readers of one book-length document
        attn("attend document", 128, 1, 65536, 1, 4096, a, False, 64),
        # one conversation's drafts
        verify("verify one", 1, 7, 131072, 0.7, True, "float32"),
        # drafts without probabilities (the most likely token of a draft model or a lookup), half-precision target, odd vocabulary
        verify("verify lookup", 24, 4, 50021, 0.6, False, "bfloat16"),
        verify("verify batch", 64, 5, 100352, 0.7, True, "float32"),
        verify("verify wide", 192, 3, 250000, 0.8, True, "float32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "verify"])
    if op == "verify":
        vocab = _log(rng, 1000, 250000)
        k = rng.randint(1, 8)
        seqs = min(_log(rng, 1, 192), int(192 * 4 * 250000 // (vocab * (k + 1))))
        return dict(op=op, seqs=seqs, k=k, vocab=vocab, agree=round(rng.uniform(0.2, 0.95), 3), sampled=rng.random() < 0.7,
                    dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]))
    hq, hkv, d = rng.choice(GEOMS)
    fp8, page = rng.random() < 0.6, rng.choice([16, 32, 64, 128])
    if op == "append":
        hi = _log(rng, 1, 2000)
        seqs = max(1, min(_log(rng, 1, 256), 8000 // hi))
        return dict(op=op, seqs=seqs, lo=rng.randint(1, hi), hi=hi, start=_log(rng, 1, 3000) - 1, hq=hq, hkv=hkv, d=d,
                    rd=rng.choice([d // 4, d // 2, d]), inter=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    norm=rng.random() < 0.6, gated=rng.random() < 0.5, fp8=fp8, page=page, base=rng.choice([0, _log(rng, 1, 2000000)]))
    seqs, m = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 4, 7])
    prefix = rng.choice([0, _log(rng, 1, 65536), _log(rng, 64, 65536)])
    hi = _log(rng, m, 4096)
    while seqs * hi * hkv * d > 128 * 4096 * 1024 or seqs * m * hq * prefix * d > 128 * 24 * 65536 * 256:
        seqs, prefix = max(1, seqs // 2), prefix // 2
    return dict(op=op, seqs=seqs, m=m, prefix=prefix, lo=rng.randint(m, hi), hi=hi, hq=hq, hkv=hkv, d=d, fp8=fp8, page=page,
                pad=rng.randint(0, 2) if seqs > 3 else 0)


def _spread(n, lo, hi):
    """n whole numbers over [lo, hi], the same for every seed: what a case costs does not depend on the seed."""
    return [lo + int((hi - lo + 1) * ((0.5 + 0.6180339887498949 * i) % 1.0)) for i in range(n)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 + seed)


def _table(rows, page, g):
    """Page table [len(rows), most pages] for sequences of that many rows in a shuffled pool, and the pool's pages."""
    counts = [-(-r // page) for r in rows]
    total = sum(counts) + 3
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    most = max(1, max(counts))
    at = torch.zeros(len(rows), most, dtype=torch.int64)
    first = 0
    for i, c in enumerate(counts):
        at[i, :c] = torch.arange(first, first + c)
        first += c
    return order[at.cuda()].contiguous(), total


def _quantise(x):
    """e4m3 codes and a scale for each row of the last dim."""
    scale = x.abs().amax(-1).float().clamp_min(1e-6) / 448.0
    return (x.float() / scale.unsqueeze(-1)).to(torch.float8_e4m3fn), scale


def _pool(pages, hkv, page, d, fp8, g, filled):
    shape = (pages, hkv, page, d)
    if not filled:
        x = torch.zeros(shape, device="cuda", dtype=torch.float8_e4m3fn if fp8 else torch.bfloat16)
        return x, torch.ones(shape[:3], device="cuda") if fp8 else None
    if not fp8:
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        return x.normal_(generator=g), None
    x, s = torch.empty(shape, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(shape[:3], device="cuda")
    step = max(1, (1 << 26) // (hkv * page * d))
    for i in range(0, pages, step):
        x[i:i + step], s[i:i + step] = _quantise(torch.randn((min(step, pages - i),) + shape[1:], device="cuda", generator=g).bfloat16())
    return x, s


def _frequencies(rd, scaling, theta=1e7, factor=4.0, trained=32768):
    """Radians a position of each pair and the factor on cos and sin, for a context stretched by `factor`."""
    i = torch.arange(rd // 2, dtype=torch.float64)
    if scaling == "ntk":
        theta = theta * factor ** (rd / (rd - 2))
    f = theta ** (-2.0 * i / rd)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling != "yarn":
        return f, 1.0
    low = max(math.floor(rd * math.log(trained / (32.0 * 2 * math.pi)) / (2 * math.log(theta))), 0)
    high = min(math.ceil(rd * math.log(trained / (2 * math.pi)) / (2 * math.log(theta))), rd - 1)
    ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    g, s = _gen(seed), dict(case)
    if case["op"] == "verify":
        b, k, v = case["seqs"], case["k"], case["vocab"]
        p = torch.randn(b, k + 1, v, device="cuda", generator=g).mul_(3.0).softmax(-1)
        other = torch.randn(b, k, v, device="cuda", generator=g).mul_(3.0).softmax(-1)
        q = other.mul_(1 - case["agree"]).add_(p[:, :k], alpha=case["agree"])       # drafts agree with the target about that often
        if case["sampled"]:
            s["drafts"] = torch.multinomial(q.view(b * k, v), 1, generator=g).view(b, k)
            s["q"] = q.to(getattr(torch, case["dtype"]))
        else:
            top = p[:, :k].argmax(-1)
            p[:, :k].scatter_add_(-1, top.unsqueeze(-1), torch.full((b, k, 1), 2.0, device="cuda"))   # a confident target
            p[:, :k] /= 3.0
            miss = torch.rand(b, k, device="cuda", generator=g) > case["agree"]
            s["drafts"] = torch.where(miss, torch.randint(0, v, (b, k), device="cuda", generator=g), top)
            s["q"] = None
        s["p"] = p.to(getattr(torch, case["dtype"]))
        s["u"] = torch.rand(b, k + 1, device="cuda", generator=g)
        return s
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    if case["op"] == "append":
        counts = _spread(case["seqs"], case["lo"], case["hi"])
        starts = _spread(case["seqs"], 0, case["start"])[::-1]
        s["table"], pages = _table([a + c for a, c in zip(starts, counts)], page, g)
        t, wide = sum(counts), hq * (2 if case["gated"] else 1)                     # [q | gate] of each head, or q alone
        qkv = torch.randn(t, (wide + 2 * hkv) * d, device="cuda", generator=g).bfloat16()
        s["q"] = qkv[:, :wide * d].view(t, hq, -1)[..., :d]
        s["k"] = qkv[:, wide * d:(wide + hkv) * d].view(t, hkv, d)
        s["v"] = qkv[:, (wide + hkv) * d:].view(t, hkv, d)
        s["lens"] = torch.tensor(starts, dtype=torch.int64, device="cuda")
        s["cu"] = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32) if case["hi"] > 1 else None
        s["k_pages"], s["k_scale"] = _pool(pages, hkv, page, d, case["fp8"], g, False)
        s["v_pages"], s["v_scale"] = _pool(pages, hkv, page, d, case["fp8"], g, False)
        s["q_w"] = s["k_w"] = None
        if case["norm"]:
            s["q_w"] = torch.randn(d, device="cuda", generator=g).mul_(0.1).bfloat16()
            s["k_w"] = torch.randn(d, device="cuda", generator=g).mul_(0.1).bfloat16()
        f, s["amplitude"] = _frequencies(case["rd"], case["scaling"])
        s["inv_freq"] = f.cuda()
        return s
    b, m = case["seqs"], case["m"]
    live = _spread(b, case["lo"], case["hi"])
    prefix_pages = -(-case["prefix"] // page)
    table, pages = _table(live + [case["prefix"]], page, g)
    most = max(1, -(-max(live) // page))
    s["table"] = table[:b, :most].contiguous()
    s["prefix_table"] = table[b, :prefix_pages].contiguous() if case["prefix"] else None
    lens = [n - m for n in live]
    for i in range(case["pad"]):
        lens[b - 1 - i] = -1                                                        # an empty slot of a captured batch
    s["lens"] = torch.tensor(lens, dtype=torch.int64, device="cuda")
    s["q"] = torch.randn(b, m, hq, d, device="cuda", generator=g).mul_(1.5).bfloat16()
    s["k_pages"], s["k_scale"] = _pool(pages, hkv, page, d, case["fp8"], g, True)
    s["v_pages"], s["v_scale"] = _pool(pages, hkv, page, d, case["fp8"], g, True)
    return s


def run(s):
    if own:
        from tokenrush_b200 import fused
        if s["op"] == "append":
            q = fused.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["k_scale"], s["v_scale"], q=s["q"],
                                   cu=s["cu"], base=s["base"], q_norm_w=s["q_w"], k_norm_w=s["k_w"], eps=1e-6, inv_freq=s["inv_freq"],
                                   interleaved=s["inter"], amplitude=s["amplitude"])
            return [q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]]
        if s["op"] == "attn":
            return fused.attn_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["k_scale"], s["v_scale"],
                                    prefix_table=s["prefix_table"], prefix_len=s["prefix"])
        return list(fused.spec_verify(s["p"], s["drafts"], s["u"], draft_probs=s["q"]))
    return {"append": _append_plain, "attn": _attend_plain, "verify": _verify_plain}[s["op"]](s)


def _norm_plain(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1 + w.float())


def _rotate_plain(x, cos, sin, rd, inter):
    r = x[..., :rd]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., :rd // 2], r[..., rd // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((a, b), -1).flatten(-2) if inter else torch.cat((a, b), -1)
    return torch.cat((r, x[..., rd:]), -1)


def _append_plain(s):
    t = torch.arange(s["k"].shape[0], device="cuda")
    if s["cu"] is None:
        seq, i = t, torch.zeros_like(t)
    else:
        seq = torch.bucketize(t, s["cu"][1:].long(), right=True)
        i = t - s["cu"].long()[seq]
    row = s["lens"][seq] + i
    angle = (row + s["base"]).double().unsqueeze(-1) * s["inv_freq"]               # far positions: 64 bits
    cos, sin = (angle.cos() * s["amplitude"]).float().unsqueeze(1), (angle.sin() * s["amplitude"]).float().unsqueeze(1)
    q = _rotate_plain(_norm_plain(s["q"], s["q_w"]), cos, sin, s["rd"], s["inter"]).bfloat16()
    k = _rotate_plain(_norm_plain(s["k"], s["k_w"]), cos, sin, s["rd"], s["inter"])
    page, at = s["table"][seq, row // s["page"]].long(), row % s["page"]
    for x, pages, scales in ((k, s["k_pages"], s["k_scale"]), (s["v"], s["v_pages"], s["v_scale"])):
        if scales is None:
            pages[page, :, at] = x.bfloat16()
        else:
            codes, scale = _quantise(x)
            pages.view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
            scales[page, :, at] = scale
    return [q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]]


def _rows_plain(pages, scales, table):
    """The rows of each table as [.., kv head, row, dim] in 32 bits."""
    x = pages.view(torch.uint8)[table.long()].view(pages.dtype).float() if scales is not None else pages[table.long()].float()
    if scales is not None:
        x = x * scales[table.long()].unsqueeze(-1)
    return x.transpose(-4, -3).flatten(-3, -2)


def _attend_plain(s):
    b, m, hq, d = s["q"].shape
    hkv, g, lens = s["hkv"], s["hq"] // s["hkv"], s["lens"]
    q = s["q"].float().view(b, m, hkv, g, d).permute(2, 0, 1, 3, 4).reshape(hkv, b * m * g, d) * d ** -0.5
    ko, vo = _rows_plain(s["k_pages"], s["k_scale"], s["table"]), _rows_plain(s["v_pages"], s["v_scale"], s["table"])
    qb = q.view(hkv, b, m * g, d).transpose(0, 1)
    so = (qb @ ko.transpose(-1, -2)).view(b, hkv, m, g, -1)
    at = torch.arange(so.shape[-1], device="cuda")
    last = lens.view(b, 1) + torch.arange(m, device="cuda")                        # the last own row that query row i sees
    seen = (at <= last.unsqueeze(-1)) & (lens >= 0).view(b, 1, 1)
    so = so.masked_fill(~seen.view(b, 1, m, 1, -1), -math.inf)
    top = so.amax(-1)
    if s["prefix_table"] is not None:
        n = s["prefix"]
        kp, vp = (_rows_plain(s[x + "_pages"], s[x + "_scale"], s["prefix_table"])[:, :n] for x in "kv")
        sp = (q @ kp.transpose(-1, -2)).view(hkv, b, m, g, n)
        sp = sp.masked_fill((lens < 0).view(1, b, 1, 1, 1), -math.inf)
        top = torch.maximum(top, sp.amax(-1).transpose(0, 1))
    top = top.clamp_min(-1e30).unsqueeze(-1)
    eo = (so - top).exp()
    total = eo.sum(-1, keepdim=True)
    o = (eo.view(b, hkv, m * g, -1) @ vo).view(b, hkv, m, g, d)
    if s["prefix_table"] is not None:
        ep = (sp - top.transpose(0, 1)).exp()
        total = total + ep.sum(-1, keepdim=True).transpose(0, 1)
        o = o + (ep.view(hkv, b * m * g, n) @ vp).view(hkv, b, m, g, d).transpose(0, 1)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 2, 1, 3, 4).reshape(b, m, hq, d).bfloat16()


def _verify_plain(s):
    p, x, u, q = s["p"], s["drafts"], s["u"], s["q"]
    b, k = x.shape
    px = p[:, :k].gather(-1, x.unsqueeze(-1)).squeeze(-1).double()
    qx = torch.ones_like(px) if q is None else q.gather(-1, x.unsqueeze(-1)).squeeze(-1).double()
    kept = u[:, :k].double() * qx < px                                             # 64 bits: the product is exact
    n = kept.long().cumprod(-1).sum(-1)
    rows = torch.arange(b, device="cuda")
    w = p[rows, n].double()
    at = n.clamp_max(k - 1)
    if q is None:
        less = torch.zeros_like(w).scatter_(-1, x[rows, at].unsqueeze(-1), math.inf)
    else:
        less = q[rows, at].double()
    left = (w - less).clamp_min(0)
    w = torch.where((n < k).unsqueeze(-1) & (left.sum(-1, keepdim=True) > 0), left, w)
    c = w.cumsum(-1)                                                               # 64 bits: long sums, values next to a border
    new = (c <= u[:, k:].double() * c[:, -1:]).sum(-1).clamp_max(w.shape[-1] - 1)
    i = torch.arange(k + 1, device="cuda")
    padded = torch.cat((x, x[:, :1]), -1)
    tokens = torch.where(i < n.unsqueeze(-1), padded, torch.where(i == n.unsqueeze(-1), new.unsqueeze(-1), -1))
    return [tokens, n]


def work(case):
    if case["op"] == "verify":
        size = 4 if case["dtype"] == "float32" else 2
        some = 1 - case["agree"] ** case["k"] if case["sampled"] else 0             # sequences that read a row of q too
        b, k, v = case["seqs"], case["k"], case["vocab"]
        return {"bytes": b * (v * size * (1 + some) + k * (8 + 4 + 2 * size) + (k + 2) * 8), "flops": b * v * 2}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    row = 2 * hkv * (d + 4 if case["fp8"] else 2 * d)                               # K and V of one position
    if case["op"] == "append":
        t = sum(_spread(case["seqs"], case["lo"], case["hi"]))
        return {"bytes": t * (4 * hq * d + 4 * hkv * d + row), "flops": t * (hq + hkv) * (6 * d if case["norm"] else 3 * case["rd"])}
    b, m = case["seqs"], case["m"]
    live = _spread(b, case["lo"], case["hi"])[:b - case["pad"]]
    keys = sum(live)
    seen = sum(m * n - m * (m - 1) // 2 for n in live) + len(live) * m * case["prefix"]
    return {"bytes": (case["prefix"] + keys) * row + 4 * len(live) * m * hq * d, "flops": 4 * d * hq * seen}


def exact(case, seed):
    """What run() returns, from the definitions in 64 bits, sequence by sequence."""
    if case["op"] == "verify":
        return None                                                                # whole numbers
    s = prepare(case, seed)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    if case["op"] == "attn":
        def rows(pages, scales, table, n, head):
            x = torch.cat([pages[int(t), head] for t in table[:-(-n // page)].tolist()])[:n].double()
            if scales is not None:
                x *= torch.cat([scales[int(t), head] for t in table[:-(-n // page)].tolist()])[:n].double().unsqueeze(-1)
            return x
        out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
        group = hq // hkv
        for h in range(hkv):
            kp = vp = torch.zeros(0, d, device="cuda", dtype=torch.float64)
            if case["prefix"]:
                kp, vp = (rows(s[x + "_pages"], s[x + "_scale"], s["prefix_table"], case["prefix"], h) for x in "kv")
            for b, before in enumerate(s["lens"].tolist()):
                if before < 0:
                    continue
                ko, vo = (rows(s[x + "_pages"], s[x + "_scale"], s["table"][b], before + case["m"], h) for x in "kv")
                for i in range(case["m"]):
                    n = before + i + 1
                    x = s["q"][b, i, h * group:(h + 1) * group].double()
                    z = torch.cat((x @ kp.T, x @ ko[:n].T), 1) / math.sqrt(d)
                    w = torch.softmax(z, 1)
                    out[b, i, h * group:(h + 1) * group] = w[:, :len(kp)] @ vp + w[:, len(kp):] @ vo[:n]
        return out
    shape = s["k_pages"].shape
    ks, vs = (torch.zeros(shape, device="cuda", dtype=torch.float64) for _ in range(2))
    kc, vc = (torch.ones(shape[:3], device="cuda", dtype=torch.float64) for _ in range(2))
    cu = s["cu"].tolist() if s["cu"] is not None else list(range(case["seqs"] + 1))
    q_out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    half = case["rd"] // 2
    pair = torch.arange(half, device="cuda")
    one = 2 * pair if case["inter"] else pair
    two = one + 1 if case["inter"] else pair + half

    def turned(x, w, position):
        x = x.double()
        if w is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * (1 + w.double())
        phase = torch.exp(1j * position.double().view(-1, 1, 1) * s["inv_freq"]) * s["amplitude"]
        z = torch.complex(x[..., one], x[..., two]) * phase
        y = x.clone()
        y[..., one], y[..., two] = z.real, z.imag
        return y

    for b, before in enumerate(s["lens"].tolist()):
        lo, hi = cu[b], cu[b + 1]
        row = before + torch.arange(hi - lo, device="cuda")
        q_out[lo:hi] = turned(s["q"][lo:hi], s["q_w"], row + case["base"])
        at = s["table"][b].long()[row // page], row % page
        for x, values, scales in ((turned(s["k"][lo:hi], s["k_w"], row + case["base"]), ks, kc), (s["v"][lo:hi].double(), vs, vc)):
            if case["fp8"]:
                top = x.abs().amax(-1).clamp_min(1e-6) / 448
                scales[at[0], :, at[1]] = top
                x = x / top.unsqueeze(-1)
            values[at[0], :, at[1]] = x
    return [q_out, ks, vs, kc, vc] if case["fp8"] else [q_out, ks, vs, None, None]

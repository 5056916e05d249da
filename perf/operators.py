"""Cases of the operators for sequences that grow from one prompt: attention over a shared prefix, the
normalised and rotated append, and copies of cache pages with the table rewrite of a compaction.

`run` computes each in plain torch operations in 32 bits (`own` false) or through pa_b200.ops (`own` true).
Lengths follow from a case's own numbers; values come from the seed alone."""
import math
import os
import sys

import torch

own = False

DT = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def _ops():
    path = os.path.abspath("gb10-attn_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from pa_b200 import ops
    return ops


# --------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------

def _shared(name, batch, groups, heads, kv_heads, head_dim, prefix, prefix_step, tail_lo, tail_hi, dtype,
            block=16, idle=0):
    """Attention of `batch` sequences in `groups` groups; group g shares prefix + g * prefix_step tokens and
    each member has tail_lo .. tail_hi tokens of its own; the last `idle` sequences are empty slots of the batch."""
    return {"name": name, "op": "shared", "batch": batch, "groups": groups, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "prefix": prefix, "prefix_step": prefix_step, "tail_lo": tail_lo,
            "tail_hi": tail_hi, "dtype": dtype, "block": block, "idle": idle}


def _append(name, seqs, len_lo, len_hi, start, heads, kv_heads, head_dim, rot, interleaved, norm, dtype, pool,
            block=16):
    """The append of `seqs` sequences of len_lo .. len_hi new tokens each, from position `start` on."""
    return {"name": name, "op": "append", "seqs": seqs, "len_lo": len_lo, "len_hi": len_hi, "start": start,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "rot": rot, "interleaved": interleaved,
            "norm": norm, "dtype": dtype, "pool": pool, "block": block}


def _pages(name, layers, blocks, moves, partial, kv_heads, head_dim, dtype, tables, width, block=16):
    """Copies of `moves` pages in every layer; partial: only a page's first rows (a fork's last page), else whole
    pages followed by the rewrite of a [tables, width] block table (a compaction)."""
    return {"name": name, "op": "pages", "layers": layers, "blocks": blocks, "moves": moves, "partial": partial,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "tables": tables, "width": width,
            "block": block}


def listed():
    return [
        # four samples of one short prompt, small heads: a call's fixed cost is what counts
        _shared("shared: 4 samples, 12 heads", 4, 1, 12, 12, 64, 512, 0, 1, 16, "float16"),
        # a batch of 64 behind one 2048-token instruction, as many kv heads as heads
        _shared("shared: 64 on one prompt", 64, 1, 12, 12, 64, 2048, 0, 1, 256, "float16"),
        # 128 requests behind an 8k system prompt, grouped heads
        _shared("shared: 128 on 8k, grouped heads", 128, 1, 32, 8, 128, 8192, 0, 1, 512, "bfloat16"),
        # seven prompts sampled a few times each, prefixes that end inside a page, two idle slots
        _shared("shared: 7 prompts, odd, idle", 61, 7, 32, 8, 128, 1003, 517, 0, 300, "bfloat16", 16, 2),
        # the largest: 256 sequences behind a 32k document, up to 1024 tokens each of their own
        _shared("shared: 256 on 32k", 256, 1, 32, 8, 128, 32768, 0, 256, 1024, "bfloat16"),
        # one decode step of a small batch: one token a sequence, launch latency
        _append("append: 8 tokens", 8, 1, 1, 1000, 32, 8, 128, 128, False, True, "bfloat16", "bfloat16"),
        # one decode step of a large batch
        _append("append: 256 tokens", 256, 1, 1, 4000, 32, 8, 128, 128, False, True, "bfloat16", "bfloat16"),
        # ragged chunks, half of each head rotated in neighbouring pairs, no norm
        _append("append: ragged, half rotated", 9, 1, 273, 5, 12, 12, 64, 32, True, False, "float16", "float16"),
        # four prompts of 4096 tokens
        _append("append: 4 x 4096 tokens", 4, 4096, 4096, 0, 32, 32, 128, 128, False, True, "bfloat16", "bfloat16"),
        # a fork into seven: seven copies of a last page, partly filled
        _pages("pages: fork, 7 part pages", 12, 512, 7, True, 12, 64, "float16", 8, 64),
        # many forks at once
        _pages("pages: fork, 250 part pages", 12, 1024, 250, True, 12, 64, "float16", 64, 64),
        # the compaction of a pool after a third of its sequences have ended
        _pages("pages: compaction", 16, 1024, 331, False, 8, 128, "bfloat16", 128, 200),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


HEADS = ((12, 12, 64), (32, 8, 128), (32, 32, 128), (16, 2, 64), (24, 8, 128), (8, 1, 128))


def draw(rng):
    op = rng.choice(("shared", "append", "pages"))
    heads, kv_heads, head_dim = rng.choice(HEADS)
    if op == "shared":
        batch = _log(rng, 1, 256)
        groups = min(batch, _log(rng, 1, 12))
        # what the largest listed case reads and multiplies is not passed
        row = kv_heads * head_dim
        prefix = _log(rng, 1, min(32768, 2 ** 28 // (batch * heads), 2 ** 26 // (groups * row)))
        tail = _log(rng, 1, min(1024, 2 ** 27 // (batch * row)))
        c = _shared("", batch, groups, heads, kv_heads, head_dim, prefix, rng.choice((0, 1, 37)), rng.choice((0, 1)),
                    tail, rng.choice(("float16", "bfloat16")), rng.choice((16, 16, 32)),
                    rng.choice((0, 0, 1)) if batch > groups else 0)
    elif op == "append":
        seqs = _log(rng, 1, 256)
        dtype = rng.choice(("float16", "bfloat16", "bfloat16", "float32"))
        width = (heads + 2 * kv_heads) * head_dim * (2 if dtype == "float32" else 1)
        hi = _log(rng, 1, max(1, 16384 * 96 * 128 // width // seqs))
        rot = rng.choice((head_dim, head_dim, head_dim // 2))
        c = _append("", seqs, rng.choice((1, hi)), hi, _log(rng, 1, 20000), heads, kv_heads, head_dim, rot,
                    rng.random() < 0.3, rng.random() < 0.7, dtype,
                    rng.choice(("float16", "bfloat16")))
    else:
        blocks = _log(rng, 64, 1024)
        partial = rng.random() < 0.5
        c = _pages("", _log(rng, 2, 24), blocks, _log(rng, 1, blocks // 3), partial, kv_heads if kv_heads < 32 else 8,
                   head_dim, rng.choice(("float16", "bfloat16")), _log(rng, 1, 256), _log(rng, 8, 200),
                   rng.choice((16, 16, 32)))
        if c["layers"] * c["blocks"] * c["block"] * c["kv_heads"] * c["head_dim"] > 16 * 1024 * 16 * 1024:
            c["layers"] = max(1, 16 * 1024 * 16 * 1024 // (c["blocks"] * c["block"] * c["kv_heads"] * c["head_dim"]))
    del c["name"]
    return c


# --------------------------------------------------------------------------------------------------
# lengths, from a case's numbers alone
# --------------------------------------------------------------------------------------------------

def _spread(lo, hi, i):
    """lo .. hi, scattered over i; the ends come up."""
    return hi if i == 0 else lo + (i * 7919) % (hi - lo + 1)


def _shared_lens(c):
    """(group starts, prefix lengths, context lengths)."""
    n, g = c["batch"], c["groups"]
    starts = [i * n // g for i in range(g + 1)]
    prefix = [c["prefix"] + i * c["prefix_step"] for i in range(g)]
    ctx = []
    for i in range(g):
        ctx += [prefix[i] + _spread(c["tail_lo"], c["tail_hi"], b) for b in range(starts[i], starts[i + 1])]
    for b in range(n - c["idle"], n):
        ctx[b] = 0
    return starts, prefix, ctx


def _append_lens(c):
    return [_spread(c["len_lo"], c["len_hi"], i) for i in range(c["seqs"])]


def _page_rows(c):
    return [1 + (i * 5 + 6) % c["block"] if c["partial"] else c["block"] for i in range(c["moves"])]


def work(c):
    if c["op"] == "shared":
        starts, prefix, ctx = _shared_lens(c)
        row = 2 * c["kv_heads"] * c["head_dim"] * 2
        tail = sum(ctx[b] - prefix[g] for g in range(c["groups"]) for b in range(starts[g], starts[g + 1]) if ctx[b])
        io = c["batch"] * c["heads"] * (2 * c["head_dim"] * 2 + 4)
        ids = 4 * sum(-(-x // c["block"]) for x in prefix) + 4 * -(-tail // c["block"])
        return {"bytes": (sum(prefix) + tail) * row + io + ids, "flops": 4 * c["head_dim"] * c["heads"] * sum(ctx)}
    if c["op"] == "append":
        lens = _append_lens(c)
        t, e, p = sum(lens), (4 if c["dtype"] == "float32" else 2), 2
        d = c["head_dim"]
        seen = max(lens) * c["rot"] * 4
        return {"bytes": t * d * ((2 * c["heads"] + 2 * c["kv_heads"]) * e + 2 * c["kv_heads"] * p) + seen + 8 * t,
                "flops": t * (c["heads"] + c["kv_heads"]) * d * 7}
    rows = sum(_page_rows(c))
    ids = 0 if c["partial"] else 4 * (2 * c["tables"] * c["width"] + c["blocks"])
    return {"bytes": 2 * 2 * c["layers"] * rows * c["kv_heads"] * c["head_dim"] * 2 + 12 * c["moves"] + ids, "flops": 0}


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return {"shared": _prepare_shared, "append": _prepare_append, "pages": _prepare_pages}[case["op"]](case, gen)


def _normal(shape, dtype, gen):
    return torch.randn(shape, dtype=torch.float32 if dtype == torch.float32 else dtype, device="cuda", generator=gen)


def _prepare_shared(c, gen):
    starts, prefix, ctx = _shared_lens(c)
    n, bs, dt = c["batch"], c["block"], DT[c["dtype"]]
    group = [g for g in range(c["groups"]) for _ in range(starts[g], starts[g + 1])]
    # a member's table: its group's whole prefix pages, then pages of its own (the page in which the prefix ends
    # is its own too: a fork copies it)
    shared = [p // bs for p in prefix]
    own_pages = [max(0, -(-ctx[b] // bs) - shared[group[b]]) for b in range(n)]
    width = max(max(-(-x // bs) for x in ctx), 1)
    used = sum(shared) + sum(own_pages)
    blocks = used + 8
    perm = torch.randperm(blocks, device="cuda", generator=gen).to(torch.int32)[:used]
    tables = torch.zeros((n, width), dtype=torch.int32, device="cuda")
    at = 0
    for g in range(c["groups"]):
        tables[starts[g]:starts[g + 1], :shared[g]] = perm[at:at + shared[g]]
        at += shared[g]
    for b in range(n):
        tables[b, shared[group[b]]:shared[group[b]] + own_pages[b]] = perm[at:at + own_pages[b]]
        at += own_pages[b]
    if c["idle"]:
        tables[n - c["idle"]:] = 0
    kc = _normal((blocks, bs, c["kv_heads"], c["head_dim"]), dt, gen)
    vc = _normal((blocks, bs, c["kv_heads"], c["head_dim"]), dt, gen)
    # the rows of a prefix's last, part-filled page are the same in every member's copy
    for g in range(c["groups"]):
        part = prefix[g] % bs
        if part:
            ids = tables[starts[g]:starts[g + 1], shared[g]].long()
            ids = ids[_ints([ctx[b] > 0 for b in range(starts[g], starts[g + 1])]).bool()]
            if len(ids):
                kc[ids, :part] = kc[ids[0], :part].clone()
                vc[ids, :part] = vc[ids[0], :part].clone()
    q = _normal((n, c["heads"], c["head_dim"]), dt, gen)
    return {"op": "shared", "q": q, "k": kc, "v": vc, "tables": tables, "ctx": _ints(ctx), "starts": _ints(starts),
            "prefix": _ints(prefix), "scale": c["head_dim"] ** -0.5, "sizes":
            (max(prefix), max([0] + [ctx[b] - prefix[group[b]] for b in range(n)]),
             max(starts[g + 1] - starts[g] for g in range(c["groups"])))}


def _prepare_append(c, gen):
    lens = _append_lens(c)
    t, bs, dt, h, hk, d = sum(lens), c["block"], DT[c["dtype"]], c["heads"], c["kv_heads"], c["head_dim"]
    # one projection's output, its q, k and v side by side
    qkv = _normal((t, h + 2 * hk, d), dt, gen) * 0.7
    first = c["start"] // bs
    pages = [-(-(c["start"] + x) // bs) - first for x in lens]
    width = first + max(pages)
    blocks = sum(pages) + 4
    perm = torch.randperm(blocks, device="cuda", generator=gen).to(torch.int32)
    tables = torch.zeros((len(lens), width), dtype=torch.int32, device="cuda")
    at = 0
    for i, p in enumerate(pages):
        tables[i, first:first + p] = perm[at:at + p]
        at += p
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), _ints(lens))
    ends = torch.cumsum(_ints(lens), 0)
    pos = torch.arange(t, device="cuda") - (ends - _ints(lens))[seq] + c["start"]
    top = c["start"] + max(lens)
    inv = 10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
    angle = torch.arange(top, dtype=torch.float64, device="cuda")[:, None] * inv
    cos_sin = torch.cat((angle.cos(), angle.sin()), 1).float()
    weights = [(1 + 0.1 * _normal((d,), torch.float32, gen)).to(dt) if c["norm"] else torch.empty(0, device="cuda")
               for _ in range(2)]
    shape = (blocks, bs, hk, d)
    return {"op": "append", "q": qkv[:, :h], "k": qkv[:, h:h + hk], "v": qkv[:, h + hk:], "wq": weights[0],
            "wk": weights[1], "eps": 1e-6, "cos_sin": cos_sin, "interleaved": c["interleaved"],
            "pos": pos.to(torch.int32), "seq": seq.to(torch.int32), "tables": tables,
            "kc": torch.zeros(shape, dtype=DT[c["pool"]], device="cuda"),
            "vc": torch.zeros(shape, dtype=DT[c["pool"]], device="cuda"), "none": torch.empty(0, device="cuda")}


def _prepare_pages(c, gen):
    pool = _normal((c["layers"], 2, c["blocks"], c["block"], c["kv_heads"], c["head_dim"]), DT[c["dtype"]], gen)
    n, nb = c["moves"], c["blocks"]
    free = torch.randperm(nb, device="cuda", generator=gen).to(torch.int32)
    if c["partial"]:
        # a few last pages, each copied to several pages of its own
        dst = free[:n].clone()
        src = free[n:n + max(1, n // 7)].repeat(8)[:n].clone()
        src = torch.cat((src, src[:1].expand(n - len(src)))) if len(src) < n else src
    else:
        # the highest pages in use go to the lowest free ones
        dst = torch.sort(free[free < nb - n][:n]).values
        src = torch.arange(nb - 1, nb - 1 - n, -1, device="cuda", dtype=torch.int32)
        if len(dst) < n:
            src = src[:len(dst)]
    to = torch.arange(nb, dtype=torch.int32, device="cuda")
    to[src.long()] = dst
    tables = torch.randint(0, nb, (c["tables"], c["width"]), dtype=torch.int32, device="cuda", generator=gen)
    # tables name no page that the compaction takes as free
    tables = torch.where(torch.isin(tables, dst), src[0], tables)
    rows = _ints(_page_rows(c))[:len(src)]
    return {"op": "pages", "pool": pool, "k_layers": [pool[i, 0] for i in range(c["layers"])],
            "v_layers": [pool[i, 1] for i in range(c["layers"])], "src": src, "dst": dst, "rows": rows,
            "partial": c["partial"], "map": to, "tables": tables, "none": torch.empty(0, device="cuda")}


# --------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------

def run(s):
    return {"shared": _run_shared, "append": _run_append, "pages": _run_pages}[s["op"]](s)


def _run_shared(s):
    if own:
        out, lse = _ops().paged_attention_shared(s["q"], s["k"], s["v"], s["tables"], s["ctx"], s["starts"],
                                                 s["prefix"], s["scale"])
        return {"out": out, "lse": lse}
    q, ctx, prefix = s["q"], s["ctx"].long(), s["prefix"].long()
    n, h, d = q.shape
    nb, bs, hk, _ = s["k"].shape
    longest, tail, most = s["sizes"]
    width = s["tables"].shape[1]
    k, v = s["k"].reshape(nb * bs, hk, d), s["v"].reshape(nb * bs, hk, d)
    tables, starts = s["tables"].long(), s["starts"].long()
    row = torch.arange(n, device=q.device)
    group = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    slot = row - starts[group]
    # the prefixes, once a group
    t = torch.arange(longest, device=q.device)
    flat = tables[starts[:-1]][:, torch.clamp(t // bs, max=width - 1)] * bs + t % bs
    kp, vp = k[flat].float(), v[flat].float()
    qg = torch.zeros((len(prefix), most, h, d), dtype=torch.float32, device=q.device)
    qg[group, slot] = q.float()
    qg = qg.view(len(prefix), most, hk, h // hk, d)
    sp = torch.einsum("gmkrd,gtkd->gmkrt", qg, kp)[group, slot] * s["scale"]
    seen = t < torch.minimum(prefix[group], ctx)[:, None]
    sp = sp.masked_fill(~seen[:, None, None], -math.inf)
    # each sequence's own tokens
    u = prefix[group][:, None] + torch.arange(tail, device=q.device)
    flat = torch.gather(tables, 1, torch.clamp(u // bs, max=width - 1)) * bs + u % bs
    ku, vu = k[flat].float(), v[flat].float()
    su = torch.einsum("bkrd,btkd->bkrt", q.float().view(n, hk, h // hk, d), ku) * s["scale"]
    su = su.masked_fill(~(u < ctx[:, None])[:, None, None], -math.inf)
    top = torch.cat((sp, su), -1).amax(-1, keepdim=True)
    base = torch.where(top.isinf(), torch.zeros_like(top), top)
    sp, su = torch.exp(sp - base), torch.exp(su - base)
    total = sp.sum(-1) + su.sum(-1)
    pg = torch.zeros((len(prefix), most, hk, h // hk, longest), dtype=torch.float32, device=q.device)
    pg[group, slot] = sp
    out = torch.einsum("gmkrt,gtkd->gmkrd", pg, vp)[group, slot] + torch.einsum("bkrt,btkd->bkrd", su, vu)
    out = (out / total[..., None]).view(n, h, d).to(q.dtype)
    return {"out": out, "lse": (base[..., 0] + torch.log(total)).view(n, h)}


def _run_append(s):
    if own:
        out = _ops().qk_norm_rope_append(s["q"], s["k"], s["v"], s["wq"], s["wk"], s["eps"], s["cos_sin"],
                                         s["interleaved"], s["pos"], s["seq"], s["kc"], s["vc"], s["tables"],
                                         s["none"], s["none"])
        return {"q": out, "k_cache": s["kc"], "v_cache": s["vc"]}
    pos, half, bs = s["pos"].long(), s["cos_sin"].shape[1] // 2, s["kc"].shape[1]
    cos, sin = s["cos_sin"][pos][:, None, :half], s["cos_sin"][pos][:, None, half:]

    def turned(x, w):
        x = x.float()
        if w.numel():
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * w.float()
        if s["interleaved"]:
            a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
            y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = x[..., :half], x[..., half:2 * half]
            y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((y, x[..., 2 * half:]), -1)

    block = s["tables"][s["seq"].long(), pos // bs].long()
    s["kc"][block, pos % bs] = turned(s["k"], s["wk"]).to(s["kc"].dtype)
    s["vc"][block, pos % bs] = s["v"].to(s["vc"].dtype)
    return {"q": turned(s["q"], s["wq"]).to(s["q"].dtype), "k_cache": s["kc"], "v_cache": s["vc"]}


def _run_pages(s):
    if own:
        ops = _ops()
        ops.copy_blocks(s["k_layers"], s["v_layers"], s["src"], s["dst"], s["rows"] if s["partial"] else s["none"])
        if s["partial"]:
            return {"pool": s["pool"]}
        return {"pool": s["pool"], "tables": ops.remap_block_tables(s["tables"], s["map"])}
    src, dst = s["src"].long(), s["dst"].long()
    if not s["partial"]:
        s["pool"][:, :, dst] = s["pool"][:, :, src]
        return {"pool": s["pool"], "tables": s["map"][s["tables"].long()]}
    keep = torch.arange(s["pool"].shape[3], device=src.device)[None] < s["rows"][:, None]
    keep = keep[None, None, :, :, None, None]
    s["pool"][:, :, dst] = torch.where(keep, s["pool"][:, :, src], s["pool"][:, :, dst])
    return {"pool": s["pool"]}


# --------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# --------------------------------------------------------------------------------------------------

def exact(case, seed):
    return {"shared": _exact_shared, "append": _exact_append, "pages": _exact_pages}[case["op"]](case, seed)


def _exact_shared(c, seed):
    s = prepare(c, seed)
    _, _, ctx = _shared_lens(c)
    n, h, d = s["q"].shape
    bs, hk = c["block"], c["kv_heads"]
    out = torch.full((n, h, d), math.nan, dtype=torch.float64, device="cuda")
    lse = torch.full((n, h), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(n):
        if not ctx[b]:
            continue
        ids = s["tables"][b, :-(-ctx[b] // bs)].long()
        kb = s["k"][ids].double().reshape(-1, hk, d)[:ctx[b]].transpose(0, 1)
        vb = s["v"][ids].double().reshape(-1, hk, d)[:ctx[b]].transpose(0, 1)
        logits = torch.matmul(s["q"][b].double().view(hk, h // hk, d), kb.transpose(1, 2)) / math.sqrt(d)
        lse[b] = torch.logsumexp(logits, -1).view(h)
        out[b] = torch.matmul(torch.softmax(logits, -1), vb).view(h, d)
    return {"out": out, "lse": lse}


def _exact_append(c, seed):
    s = prepare(c, seed)
    half = c["rot"] // 2
    z = torch.view_as_complex(torch.stack((s["cos_sin"][:, :half], s["cos_sin"][:, half:]), -1).double())
    z = z[s["pos"].long()][:, None]

    def turned(x, w):
        x = x.double()
        if c["norm"]:
            x = w.double() * x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + s["eps"])
        y = x.clone()
        one = slice(0, 2 * half, 2) if c["interleaved"] else slice(0, half)
        two = slice(1, 2 * half, 2) if c["interleaved"] else slice(half, 2 * half)
        r = torch.complex(x[..., one], x[..., two]) * z
        y[..., one], y[..., two] = r.real, r.imag
        return y

    at = s["pos"].long()
    flat = s["tables"].long()[s["seq"].long(), at // c["block"]] * c["block"] + at % c["block"]
    found = {"q": turned(s["q"], s["wq"])}
    for name, x in (("k_cache", turned(s["k"], s["wk"])), ("v_cache", s["v"].double())):
        cache = torch.zeros(s["kc"].shape, dtype=torch.float64, device="cuda")
        cache.view(-1, *cache.shape[2:]).index_copy_(0, flat, x)
        found[name] = cache
    return found


def _exact_pages(c, seed):
    s = prepare(c, seed)
    pool = s["pool"].double()
    for i, (a, b, r) in enumerate(zip(s["src"].tolist(), s["dst"].tolist(), s["rows"].tolist())):
        pool[:, :, b, :r] = s["pool"][:, :, a, :r].double()
    if c["partial"]:
        return {"pool": pool}
    to = s["map"].cpu()
    return {"pool": pool, "tables": torch.take(to, s["tables"].long().cpu()).to("cuda")}

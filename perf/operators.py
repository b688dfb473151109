"""Cases and plain forms of the serving operators: rotary positions (with the
write into a paged cache), causal attention over packed prompts, attention of
drafted token trees over the paged cache, and the compaction of the cache
after a draft was verified.

``run`` computes an operator either through ``akili_bench_b200.ops`` (``own``
true) or in its plain form: elementary torch operations in fp32, rounded once
at the end.  ``exact`` states the same definitions in fp64, sequence by
sequence.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # queries and keys of a long packed prompt before attention, grouped heads
        {"name": "rope_prompt_f16", "op": "rope", "dtype": "f16", "tokens": 8192, "hq": 32, "hk": 8, "d": 128,
         "rot": 128, "interleaved": False, "inverse": False, "max_pos": 16384},
        # a training step's gradient through a partial interleaved rotation, fp32
        {"name": "rope_grad_f32", "op": "rope", "dtype": "f32", "tokens": 2049, "hq": 16, "hk": 16, "d": 96, "rot": 64,
         "interleaved": True, "inverse": True, "max_pos": 4096},
        # a prompt's rotated keys and its values on their way into 16-token pages
        {"name": "append_prompt_bf16", "op": "append", "dtype": "bf16", "tokens": 4099, "hq": 32, "hk": 8, "d": 128,
         "rot": 128, "interleaved": False, "page": 16, "max_pos": 8192},
        # the new tokens of a small decode batch (a 7B llama2's heads): latency
        {"name": "append_decode_f16", "op": "append", "dtype": "f16", "tokens": 7, "hq": 32, "hk": 32, "d": 128,
         "rot": 128, "interleaved": True, "page": 16, "max_pos": 4096},
        # eight full prompts, every head with its own keys
        {"name": "prompt_full_f16", "op": "prompt", "dtype": "f16", "hq": 32, "hk": 32, "d": 128,
         "qlens": "4096,4096,4096,4096,4096,4096,4096,4096", "klens": "", "causal": True},
        # a packed batch of uneven prompts with grouped heads
        {"name": "prompt_ragged_bf16", "op": "prompt", "dtype": "bf16", "hq": 32, "hk": 8, "d": 128,
         "qlens": "1201,17,3999,1,500,2750", "klens": "", "causal": True},
        # many short requests, seven query heads to a key head; some continue an earlier part of their prompt
        {"name": "prompt_short_f16", "op": "prompt", "dtype": "f16", "hq": 14, "hk": 2, "d": 64,
         "qlens": "33,150,3,64,91,128,7,19,45,110,1,77,129,60,25,12,140,38,81,5,99,66,54,18",
         "klens": "33,150,3,300,91,128,7,19,245,110,90,77,129,60,25,12,140,38,81,5,199,66,54,18", "causal": True},
        # one new token of one sequence: latency
        {"name": "decode_one_f16", "op": "tree", "dtype": "f16", "hq": 32, "hk": 32, "d": 128, "ctx": "4001",
         "qlens": "1", "page": 16, "tree": False},
        # one new token each of a batch with uneven long contexts
        {"name": "decode_batch_bf16", "op": "tree", "dtype": "bf16", "hq": 32, "hk": 8, "d": 128,
         "ctx": "16383,900,12000,5111,8192,77,15001,9999,3333,14040,6007,11311,2048,7700,13500,10240,"
                "450,15800,1023,9001,16000,4100,8888,12345,650,14999,5005,10101,7070,11999,3210,13013",
         "qlens": ",".join(["1"] * 32), "page": 64, "tree": False},
        # drafted trees of a verification step
        {"name": "tree_draft_bf16", "op": "tree", "dtype": "bf16", "hq": 32, "hk": 8, "d": 128,
         "ctx": "700,5999,2048,3301,1500,4444,999,2777,3600,5120,1250,4001,810,2300,1900,3050",
         "qlens": "64,33,48,64,25,64,57,40,64,31,64,64,16,50,64,61", "page": 16, "tree": True},
        # the accepted branch of one verified sequence, all layers of a model
        {"name": "accept_one_f16", "op": "accept", "dtype": "f16", "layers": 32, "hk": 32, "d": 128, "ctx": "307",
         "qlens": "16", "accepted": "5", "page": 16},
        # the accepted branches of a verified batch
        {"name": "accept_batch_bf16", "op": "accept", "dtype": "bf16", "layers": 32, "hk": 8, "d": 128,
         "ctx": "100,511,250,64,333,480,15,210,409,128,77,300,460,199,350,31",
         "qlens": "64,64,64,64,64,64,64,64,64,64,64,64,64,64,64,64",
         "accepted": "9,1,4,0,12,7,3,5,2,8,6,11,1,4,10,3", "page": 16},
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def text(values):
    return ",".join(str(v) for v in values)


def draw(rng):
    op = rng.choice(["rope", "append", "prompt", "prompt", "tree", "tree", "tree", "accept"])
    group = rng.choice([1, 2, 3, 4, 7, 8])
    hk = rng.choice([1, 2, 4, 8]) if group > 1 else rng.choice([4, 8, 16, 32])
    hq = hk * group
    d = rng.choice([64, 80, 96, 128, 128])
    dtype = rng.choice(["f16", "bf16"])
    page = rng.choice([8, 16, 24, 32, 64, 128])
    if op in ("rope", "append"):
        c = {"op": op, "dtype": rng.choice(["f16", "bf16", "f32"]), "tokens": log_int(rng, 1, 8192), "hq": hq, "hk": hk,
             "d": d, "rot": rng.choice([d, d, d // 2]), "interleaved": rng.random() < 0.5, "max_pos": 16384}
        if op == "rope":
            c["inverse"] = rng.random() < 0.3
        else:
            c["page"] = page
        return c
    if op == "prompt":
        batch = log_int(rng, 1, 24)
        most = min(4096, 24576 // batch)
        qlens = [log_int(rng, 1, most) for _ in range(batch)]
        klens = [n + (rng.randint(1, 500) if rng.random() < 0.3 else 0) for n in qlens]
        causal = rng.random() < 0.85
        while sum(n * m for n, m in zip(qlens, klens)) * hq * (1 if causal else 2) > 8 * 4096 * 4096 * 32:
            qlens, klens = [(n + 1) // 2 for n in qlens], [(m + 1) // 2 for m in klens]
        return {"op": op, "dtype": dtype, "hq": hq, "hk": hk, "d": d, "qlens": text(qlens),
                "klens": text(klens) if klens != qlens else "", "causal": causal}
    batch = log_int(rng, 1, 48)
    if op == "tree":
        tree = rng.random() < 0.6
        most = min(16384, 200000 // batch)
        ctx = [log_int(rng, 1, most) for _ in range(batch)]
        top = rng.choice([4, 16, 64, 100])
        qlens = [rng.randint(1, top) if tree else 1 for _ in range(batch)]
        return {"op": op, "dtype": dtype, "hq": hq, "hk": hk, "d": d, "ctx": text(ctx), "qlens": text(qlens),
                "page": page, "tree": tree}
    batch = min(batch, 16)
    qlens = [rng.randint(1, 64) for _ in range(batch)]
    return {"op": op, "dtype": dtype, "layers": log_int(rng, 1, 32), "hk": hk, "d": d,
            "ctx": text(rng.randint(0, 500) for _ in range(batch)), "qlens": text(qlens),
            "accepted": text(rng.randint(0, min(12, n)) for n in qlens), "page": page}


def ints(s):
    return [int(x) for x in s.split(",")]


def prefix(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def work(case):
    e = SIZE[case["dtype"]]
    d = case["d"]
    if case["op"] in ("rope", "append"):
        t, hq, hk = case["tokens"], case["hq"], case["hk"]
        heads = hq + hk + (hk if case["op"] == "append" else 0)
        return {"bytes": 2 * t * heads * d * e + t * (4 * case["rot"] + (4 if case["op"] == "rope" else 12)),
                "flops": 3 * t * (hq + hk) * case["rot"]}
    if case["op"] == "accept":
        n = sum(ints(case["accepted"]))
        return {"bytes": 4 * n * case["layers"] * case["hk"] * d * e, "flops": 0}
    hq, hk = case["hq"], case["hk"]
    qlens = ints(case["qlens"])
    if case["op"] == "prompt":
        klens = ints(case["klens"]) if case["klens"] else qlens
        pairs = sum(sum(range(m - n + 1, m + 1)) if case["causal"] else n * m for n, m in zip(qlens, klens))
        keys = sum(klens)
    else:
        ctx = ints(case["ctx"])
        pairs = sum(n * c + (sum(len(a) for a in ancestors(case, b, n)) if case["tree"] else n * (n + 1) // 2)
                    for b, (n, c) in enumerate(zip(qlens, ctx)))
        keys = sum(ctx) + sum(qlens)
    return {"bytes": (2 * sum(qlens) * hq + 2 * keys * hk) * d * e, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------ inputs --
def parents_of(case, b, n):
    """The drafted tree of sequence b: node 0 is the newest sure token, the
    others hang from an earlier node, near ones more often (plain integers)."""
    state = 12345 + 7919 * b + n
    parents = [-1]
    for i in range(1, n):
        state = (1103515245 * state + 12345) % (1 << 31)
        parents.append(max(0, i - 1 - (state >> 16) % 6))
    return parents


def ancestors(case, b, n):
    rows = []
    for i, p in enumerate(parents_of(case, b, n)):
        rows.append((rows[p] if p >= 0 else set()) | {i})
    return rows


def tree_bits(case, qlens):
    words = (max(qlens) + 31) // 32
    rows = []
    for b, n in enumerate(qlens):
        for seen in ancestors(case, b, n):
            v = sum(1 << j for j in seen)
            w = [(v >> (32 * k)) & 0xFFFFFFFF for k in range(words)]
            rows.append([x - (1 << 32) if x >> 31 else x for x in w])
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


def rope_angles(max_pos, rot, base=10000.0):
    """cos | sin of position * base^(-2i/rot), the table a model keeps."""
    freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(max_pos, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat([a.cos(), a.sin()], 1).float()


def pages_for(gen, lens, page, extra=3):
    """A page table for sequences of these lengths over shuffled pages; unused entries are -1."""
    need = [(n + page - 1) // page for n in lens]
    total = sum(need) + extra
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        # one generated chunk is repeated over large buffers, so that inputs stay quick to make
        n = math.prod(shape)
        if n <= 1 << 27:
            return torch.randn(shape, generator=gen, device="cuda", dtype=dt)
        part = torch.randn((1 << 27) - 77, generator=gen, device="cuda", dtype=dt)
        return part.repeat(-(-n // part.numel()))[:n].view(shape)

    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"case": case}
    op, d = case["op"], case["d"]
    if op in ("rope", "append"):
        t = case["tokens"]
        s["q"], s["k"] = normal(t, case["hq"], d), normal(t, case["hk"], d)
        start = int(torch.randint(0, max(1, case["max_pos"] - t + 1), (1,), generator=gen, device="cuda"))
        s["pos"] = (torch.arange(t, device="cuda") + start).to(torch.int32)
        s["table"] = rope_angles(case["max_pos"], case["rot"])
        if op == "append":
            s["v"] = normal(t, case["hk"], d)
            n_pages = (t + case["page"] - 1) // case["page"] + 4
            s["k_pages"], s["v_pages"] = (normal(n_pages, case["page"], case["hk"], d) for _ in range(2))
            order = torch.randperm(n_pages, generator=gen, device="cuda")
            at = torch.arange(t, device="cuda") + case["page"] // 2
            s["slots"] = order[at // case["page"]] * case["page"] + at % case["page"]
        return s
    qlens = ints(case["qlens"])
    s["cu_q"] = i32(prefix(qlens))
    if op == "prompt":
        klens = ints(case["klens"]) if case["klens"] else qlens
        s["cu_k"] = i32(prefix(klens)) if case["klens"] else s["cu_q"]
        s["q"] = normal(sum(qlens), case["hq"], d)
        s["k"], s["v"] = normal(sum(klens), case["hk"], d), normal(sum(klens), case["hk"], d)
        s["max_q"], s["max_k"] = max(qlens), max(klens)
        return s
    ctx = ints(case["ctx"])
    s["ctx"] = i32(ctx)
    s["page_table"], n_pages = pages_for(gen, [c + n for c, n in zip(ctx, qlens)], case["page"])
    if op == "tree":
        s["q"] = normal(sum(qlens), case["hq"], d)
        s["k_pages"], s["v_pages"] = (normal(n_pages, case["page"], case["hk"], d) for _ in range(2))
        s["mask"] = tree_bits(case, qlens) if case["tree"] else None
        s["max_q"], s["max_k"] = max(qlens), max(c + n for c, n in zip(ctx, qlens))
        return s
    s["k_pages"], s["v_pages"] = (normal(case["layers"], n_pages, case["page"], case["hk"], d) for _ in range(2))
    took = ints(case["accepted"])
    picked = torch.zeros((len(ctx), max(max(took), 1)), dtype=torch.int32)
    cpu = torch.Generator().manual_seed(seed)
    for b, (n, a) in enumerate(zip(qlens, took)):
        picked[b, :a] = torch.randperm(n, generator=cpu)[:a].sort().values.to(torch.int32)
    s["accepted"], s["n_accepted"] = picked.cuda(), i32(took)
    return s


# ------------------------------------------------------------- plain forms --
def plain_rotate(x, pos, table, rot, interleaved, inverse):
    """(x1, x2) -> (x1 c - x2 s, x2 c + x1 s) over the first `rot` of each head's values, in fp32."""
    y = x.float()
    at = table[pos.long()]
    c, s = at[:, None, :rot // 2], at[:, None, rot // 2:]
    if inverse:
        s = -s
    head, rest = y[..., :rot], y[..., rot:]
    if interleaved:
        x1, x2 = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([x1 * c - x2 * s, x2 * c + x1 * s], -1).flatten(-2)
    else:
        x1, x2 = head[..., :rot // 2], head[..., rot // 2:]
        turned = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)
    return torch.cat([turned, rest], -1).to(x.dtype)


def plain_attention(q, k, v, seen, scale):
    """q [B, Hq, S, D], k/v [B, Hk, L, D] in fp32, seen [B, S, L]: rows that see nothing give 0."""
    b, hq, s, d = q.shape
    hk, n = k.shape[1], k.shape[2]
    scores = (q.reshape(b, hk, hq // hk * s, d) @ k.transpose(-1, -2)).view(b, hk, hq // hk, s, n)
    scores.mul_(scale).masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, hk, hq // hk * s, n) @ v).view(b, hk, hq // hk, s, d)
    return (o / torch.where(total == 0, torch.ones_like(total), total)).reshape(b, hq, s, d)


def padded(x, cu, most):
    """The packed rows of each sequence in a batch of `most` rows each, in fp32; rows past its end are 0."""
    at = torch.arange(most, device=x.device)
    inside = at[None] < (cu[1:] - cu[:-1])[:, None]
    y = x[(cu[:-1, None] + at[None]).clamp(max=x.shape[0] - 1).long()].float()
    return y.masked_fill_(~inside[..., None, None], 0.0).transpose(1, 2)


def packed(o, cu, rows):
    """The rows of each sequence of o [B, H, S, D], one after another."""
    t = torch.arange(rows, device=o.device)
    b = torch.searchsorted(cu[1:].contiguous(), t.to(torch.int32), right=True)
    return o.transpose(1, 2)[b, t - cu[b]]


def plain_prompt(s):
    q, cu_q, cu_k = s["q"], s["cu_q"], s["cu_k"]
    i = torch.arange(s["max_q"], device=q.device)[None, :, None]
    j = torch.arange(s["max_k"], device=q.device)[None, None, :]
    nq, nk = (cu_q[1:] - cu_q[:-1])[:, None, None], (cu_k[1:] - cu_k[:-1])[:, None, None]
    seen = j < nk
    if s["case"]["causal"]:
        seen = seen & (j <= i + (nk - nq))
    else:
        seen = seen & (i >= 0)
    o = plain_attention(padded(q, cu_q, s["max_q"]), padded(s["k"], cu_k, s["max_k"]), padded(s["v"], cu_k, s["max_k"]),
                        seen, q.shape[-1] ** -0.5)
    return packed(o, cu_q, q.shape[0]).to(q.dtype)


def plain_tree(s):
    q, cu_q, ctx, page = s["q"], s["cu_q"], s["ctx"], s["case"]["page"]
    j = torch.arange(s["max_k"], device=q.device)
    n = (cu_q[1:] - cu_q[:-1])
    at = s["page_table"].clamp(min=0).long()[:, j // page] * page + j % page
    inside = (j[None] < (ctx + n)[:, None])[..., None, None]
    k, v = ((p.flatten(0, 1)[at].float().masked_fill_(~inside, 0.0)).transpose(1, 2)
            for p in (s["k_pages"], s["v_pages"]))
    i = torch.arange(s["max_q"], device=q.device)
    node = j[None, None, :] - ctx[:, None, None]
    if s["mask"] is None:
        seen = node <= i[None, :, None]
    else:
        rows = s["mask"][(cu_q[:-1, None] + i[None]).clamp(max=q.shape[0] - 1).long()]
        words = rows.gather(2, (node.clamp(min=0) // 32).clamp(max=rows.shape[2] - 1).expand(-1, i.numel(), -1))
        seen = (node < 0) | ((words >> (node.clamp(min=0) % 32).int()) & 1).bool()
    seen = seen & (node < n[:, None, None])
    o = plain_attention(padded(q, cu_q, s["max_q"]), k, v, seen, q.shape[-1] ** -0.5)
    return packed(o, cu_q, q.shape[0]).to(q.dtype)


def plain_accept(s):
    took, ctx, page = s["n_accepted"], s["ctx"], s["case"]["page"]
    i = torch.arange(s["accepted"].shape[1], device=took.device)[None]
    live = i < took[:, None]
    src = ctx[:, None] + torch.where(live, s["accepted"], torch.zeros_like(s["accepted"]))
    dst = ctx[:, None] + torch.where(live, i, torch.zeros_like(i))
    where = lambda a: (s["page_table"].gather(1, (a // page).long()).long() * page + a % page)  # noqa: E731
    # rows that move nothing name node 0, which stays where it is unless it was replaced by the first that does
    first = torch.where(took > 0, s["accepted"][:, 0], torch.zeros_like(took))[:, None]
    src = where(torch.where(live, src, ctx[:, None] + first)).flatten()
    dst = where(dst).flatten()
    for pages in (s["k_pages"], s["v_pages"]):
        flat = pages.flatten(1, 2)
        flat[:, dst] = flat[:, src]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "lens": ctx + took}


def plain(s):
    c = s["case"]
    if c["op"] == "rope":
        return [plain_rotate(s[n], s["pos"], s["table"], c["rot"], c["interleaved"], c["inverse"]) for n in ("q", "k")]
    if c["op"] == "append":
        q, k = (plain_rotate(s[n], s["pos"], s["table"], c["rot"], c["interleaved"], False) for n in ("q", "k"))
        s["k_pages"].flatten(0, 1)[s["slots"]] = k
        s["v_pages"].flatten(0, 1)[s["slots"]] = s["v"]
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    return {"prompt": plain_prompt, "tree": plain_tree, "accept": plain_accept}[c["op"]](s)


# --------------------------------------------------------------------- run --
def run(s):
    if not own:
        return plain(s)
    from akili_bench_b200 import ops
    c = s["case"]
    if c["op"] == "rope":
        return list(ops.rope(s["q"], s["k"], s["pos"], s["table"], interleaved=c["interleaved"], inverse=c["inverse"]))
    if c["op"] == "append":
        q = ops.rope_append(s["q"], s["k"], s["v"], s["pos"], s["table"], s["slots"], s["k_pages"], s["v_pages"],
                            interleaved=c["interleaved"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if c["op"] == "prompt":
        return ops.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=c["causal"])
    if c["op"] == "tree":
        return ops.tree_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["ctx"], s["cu_q"], s["mask"])
    lens = ops.cache_accept(s["k_pages"], s["v_pages"], s["page_table"], s["ctx"], s["accepted"], s["n_accepted"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "lens": lens}


# ------------------------------------------------------------------- exact --
def exact_turn(x, pos, table, rot, interleaved, sign):
    """The rotation as a product of complex numbers in fp64."""
    y = x.double().clone()
    t = table.double()[pos.long()]
    w = torch.complex(t[:, :rot // 2], sign * t[:, rot // 2:])[:, None]
    if interleaved:
        z = torch.view_as_complex(y[..., :rot].reshape(*y.shape[:-1], rot // 2, 2).contiguous()) * w
        y[..., :rot] = torch.view_as_real(z).reshape(*y.shape[:-1], rot)
    else:
        z = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot]) * w
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    return y


def exact_heads(q, k, v, seen):
    """One sequence in fp64: q [n, Hq, D], k/v [m, Hk, D], seen [n, m] or None (all); a query head at a time where it is large."""
    n, hq, d = q.shape
    group = hq // k.shape[1]
    out = torch.empty(n, hq, d, dtype=torch.float64, device=q.device)
    step = max(1, min(hq, (1 << 28) // max(1, n * k.shape[0])))
    for h in range(0, hq, step):
        hs = torch.arange(h, min(hq, h + step), device=q.device)
        a = torch.einsum("nhd,mhd->hnm", q[:, hs].double(), k[:, hs // group].double()) / math.sqrt(d)
        if seen is not None:
            a = torch.where(seen[None], a, torch.full((), -math.inf, dtype=torch.float64, device=q.device))
        w = torch.nan_to_num(torch.softmax(a, -1), nan=0.0)
        out[:, hs] = torch.einsum("hnm,mhd->nhd", w, v[:, hs // group].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        sign = -1.0 if case["inverse"] else 1.0
        return [exact_turn(s[n], s["pos"], s["table"], case["rot"], case["interleaved"], sign) for n in ("q", "k")]
    if op == "append":
        q, k = (exact_turn(s[n], s["pos"], s["table"], case["rot"], case["interleaved"], 1.0) for n in ("q", "k"))
        out = {"q": q, "k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double()}
        page, row = s["slots"] // case["page"], s["slots"] % case["page"]
        out["k_pages"][page, row], out["v_pages"][page, row] = k, s["v"].double()
        return out
    qlens = ints(case["qlens"])
    cu = prefix(qlens)
    if op == "prompt":
        klens = ints(case["klens"]) if case["klens"] else qlens
        ck, parts = prefix(klens), []
        for b, (n, m) in enumerate(zip(qlens, klens)):
            seen = None
            if case["causal"]:
                seen = torch.ones(n, m, dtype=torch.bool, device="cuda").tril(m - n)
            parts.append(exact_heads(s["q"][cu[b]:cu[b + 1]], s["k"][ck[b]:ck[b + 1]], s["v"][ck[b]:ck[b + 1]], seen))
        return torch.cat(parts)
    ctx, page, table = ints(case["ctx"]), case["page"], s["page_table"].tolist()
    if op == "tree":
        parts = []
        for b, (n, c) in enumerate(zip(qlens, ctx)):
            ids = torch.tensor(table[b][:(c + n + page - 1) // page], device="cuda")
            k, v = (p[ids].reshape(-1, *p.shape[2:])[:c + n] for p in (s["k_pages"], s["v_pages"]))
            seen = torch.ones(n, c + n, dtype=torch.bool)
            for i, a in enumerate(ancestors(case, b, n) if case["tree"] else [range(i + 1) for i in range(n)]):
                seen[i, c:] = False
                seen[i, [c + x for x in a]] = True
            parts.append(exact_heads(s["q"][cu[b]:cu[b + 1]], k, v, seen.cuda()))
        return torch.cat(parts)
    out = {n: s[n].double() for n in ("k_pages", "v_pages")}
    for b, a in enumerate(s["accepted"].tolist()):
        for i in range(ints(case["accepted"])[b]):
            src, dst = ctx[b] + a[i], ctx[b] + i
            for n in ("k_pages", "v_pages"):
                out[n][:, table[b][dst // page], dst % page] = s[n][:, table[b][src // page], src % page].double()
    return {**out, "lens": None}

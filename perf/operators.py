"""The decode operators of l2domain_b200, as measurable cases: what a single-token decoding step reads.

Three operators that a decoding step runs one after the other:

* ``q4``      y = W.x for one or a few vectors, W held in 4 bits with group scales (Q4Matrix)
* ``append``  rotated keys, values and queries of new tokens; keys and values go to a paged cache (KvAppend)
* ``attn``    attention of one new token per sequence over that cache (PagedAttention)

``run`` computes each in its plain form (elementary torch operations in 32 bits, rounded once at
the end), or, where ``own`` is set, through the package.  ``exact`` is the definition in 64 bits.

Definitions (all sums over real numbers; out-of-range means no contribution):

    q4      y[b, i] = sum_j s[i, j // g] * (q[i, j] - z[i, j // g]) * x[b, j]       q in 0..15, z = 8 where not given
    append  (a, b) -> (a cos - b sin, b cos + a sin) for the pairs of the first rot elements of a head,
            the pair (i, i + rot/2), or (2i, 2i + 1) where interleaved; the token at position p of sequence s
            goes to slot p % page_size of page table[s, p // page_size]; p < 0 is padding and writes nothing
    attn    softmax(scale * q.k) . v over positions max(0, len - window) .. len - 1, query head h with
            key-value head h // (heads_q / heads_kv); no position at all gives 0, and -inf for the log-sum-exp
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
NO_PAGE = -1


def listed():
    return [
        # A square projection of the repository's L2-resident shape (4096 x 4096): the small call of a decoding
        # step, one vector, where launch and latency count.
        {"name": "q4 4096x4096 fp16", "op": "q4", "M": 4096, "N": 4096, "vectors": 1, "group": 128, "zeros": False, "type": "fp16"},
        # The repository's LLM-decode shape (28672 x 8192, an up-projection) in 4 bits with zero points.
        {"name": "q4 28672x8192 bf16 zeros", "op": "q4", "M": 28672, "N": 8192, "vectors": 1, "group": 128, "zeros": True, "type": "bf16"},
        # The repository's largest matrix, far above the L2: bandwidth alone.
        {"name": "q4 131072x16384 fp16", "op": "q4", "M": 131072, "N": 16384, "vectors": 1, "group": 64, "zeros": False, "type": "fp16"},
        # A small serving batch on fine groups: eight vectors share one pass over the weights.
        {"name": "q4 8 vectors 8192x8192 bf16", "op": "q4", "M": 8192, "N": 8192, "vectors": 8, "group": 32, "zeros": False, "type": "bf16"},
        # Rows of an odd length and no alignment, a short last group, 32-bit activations.
        {"name": "q4 3 vectors 1111x5003 fp32", "op": "q4", "M": 1111, "N": 5003, "vectors": 3, "group": 32, "zeros": True, "type": "fp32"},
        # The first steps of one conversation: a cache of two pages, latency alone.
        {"name": "attn 1 x 17 bf16", "op": "attn", "batch": 1, "length": 17, "ragged": False, "heads_q": 32, "heads_kv": 8, "dim": 128, "page": 16, "window": 0, "type": "bf16"},
        # A serving batch in the middle of its answers: lengths from nothing to 8192.
        {"name": "attn 64 x 8192 ragged bf16", "op": "attn", "batch": 64, "length": 8192, "ragged": True, "heads_q": 32, "heads_kv": 8, "dim": 128, "page": 16, "window": 0, "type": "bf16"},
        # One long document: few rows, so the work has to be split over the length.
        {"name": "attn 1 x 131072 fp16", "op": "attn", "batch": 1, "length": 131072, "ragged": False, "heads_q": 32, "heads_kv": 4, "dim": 128, "page": 64, "window": 0, "type": "fp16"},
        # 32-bit cache, one key-value head per query head, an odd page size and a sliding window.
        {"name": "attn 9 x 4000 window fp32", "op": "attn", "batch": 9, "length": 4000, "ragged": True, "heads_q": 12, "heads_kv": 12, "dim": 80, "page": 7, "window": 1000, "type": "fp32"},
        # One token for each of 32 sequences: the append of a decoding step.
        {"name": "append 32 tokens bf16", "op": "append", "tokens": 32, "prompt": False, "heads_q": 32, "heads_kv": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 16, "type": "bf16"},
        # A chunk of prompts: every token of a few sequences.
        {"name": "append 8192 tokens fp16", "op": "append", "tokens": 8192, "prompt": True, "heads_q": 32, "heads_kv": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 16, "type": "fp16"},
        # An odd number of tokens with padding among them, part of the head rotated, pairs side by side, 32 bits.
        {"name": "append 999 tokens fp32", "op": "append", "tokens": 999, "prompt": True, "heads_q": 12, "heads_kv": 12, "dim": 80, "rot": 32, "interleaved": True, "page": 7, "type": "fp32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["q4", "q4", "attn", "attn", "append"])
    kind = rng.choice(["fp16", "bf16", "bf16", "fp32"])
    if op == "q4":
        M, N = _log(rng, 1, 131072), _log(rng, 1, 28672)
        while M * N > 2 ** 31:
            M = max(1, M // 2)
        if rng.random() < 0.5:  # rows on 16-byte boundaries, as most weights have them
            N = max(32, N // 32 * 32)
        vectors = rng.choice([1, 1, 1, 2, 3, 4, 5, 8, 13, 16])
        return {"op": op, "M": M, "N": N, "vectors": vectors, "group": rng.choice([32, 64, 128, 128, 256]),
                "zeros": rng.random() < 0.5, "type": kind}
    heads_kv = rng.choice([1, 2, 4, 8, 12])
    heads_q = heads_kv * rng.choice([1, 2, 4, 5, 8, 16])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    page = rng.choice([1, 7, 16, 16, 32, 64, 128])
    if op == "attn":
        batch, length = _log(rng, 1, 96), _log(rng, 1, 131072)
        while batch * length * heads_kv * dim * BYTES[kind] > 2 ** 30:
            length = max(1, length // 2)
        return {"op": op, "batch": batch, "length": length, "ragged": rng.random() < 0.7, "heads_q": heads_q, "heads_kv": heads_kv,
                "dim": dim, "page": page, "window": rng.choice([0, 0, 0, 1 + length // 3]), "type": kind}
    tokens = _log(rng, 1, 8192)
    while tokens * (heads_q + 2 * heads_kv) * dim > 2 ** 26:
        tokens = max(1, tokens // 2)
    return {"op": op, "tokens": tokens, "prompt": rng.random() < 0.5, "heads_q": heads_q, "heads_kv": heads_kv, "dim": dim,
            "rot": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.4, "page": page, "type": kind}


# ------------------------------------------------------------------------------------------------
# Sizes that follow from a case alone
# ------------------------------------------------------------------------------------------------

def _lengths(c):
    """Keys of each sequence: one length for all, or lengths spread from none to the longest."""
    n, b = c["length"], c["batch"]
    if not c["ragged"]:
        return [n] * b
    at = [n, 0, 1, n // 2] + [(n * (7 * i % 64) + 31 * i) // 64 % (n + 1) for i in range(4, b)]
    return [min(n, v) for v in at[:b]]


def _tokens(c):
    """(sequence, position) of each token: one each at its own depth, or runs of a prompt with padding at their ends."""
    t = c["tokens"]
    if not c["prompt"]:
        return list(range(t)), [(37 * i * i + 11 * i) % 4000 for i in range(t)], t
    run = max(1, min(2048, t // 3))
    seq, pos = [i // run for i in range(t)], [(i % run) + 5 * (i // run) for i in range(t)]
    for i in range(run - 1, t, run):
        if run > 4:
            pos[i] = -1
    return seq, pos, seq[-1] + 1


def work(c):
    e = BYTES[c["type"]]
    if c["op"] == "q4":
        M, N, b, groups = c["M"], c["N"], c["vectors"], -(-c["N"] // c["group"])
        return {"bytes": M * ((N + 1) // 2) + M * groups * (2 + c["zeros"]) + b * (M + N) * e, "flops": 2 * M * N * b}
    if c["op"] == "attn":
        w = c["window"]
        keys = sum(min(n, w) if w else n for n in _lengths(c))
        heads = c["heads_q"] * c["batch"]
        return {"bytes": 2 * keys * c["heads_kv"] * c["dim"] * e + 2 * heads * c["dim"] * e + 4 * heads, "flops": 4 * keys * c["heads_q"] * c["dim"]}
    live = sum(p >= 0 for p in _tokens(c)[1])
    return {"bytes": live * (2 * (c["heads_q"] + 2 * c["heads_kv"]) * c["dim"] * e + 4 * c["rot"] + 12),
            "flops": 3 * live * (c["heads_q"] + c["heads_kv"]) * c["rot"]}


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------

def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[c["type"]]

    def normal(*shape):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=g).to(t)

    if c["op"] == "q4":
        M, N, groups = c["M"], c["N"], -(-c["N"] // c["group"])
        s = torch.empty(M, groups, device="cuda").uniform_(0.002, 0.02, generator=g)
        i = {"w": torch.randint(0, 256, (M, (N + 1) // 2), dtype=torch.uint8, device="cuda", generator=g),  # column 2j in the low half
             "s": s.to(torch.bfloat16 if c["type"] == "bf16" else torch.float16), "z": None, "x": normal(c["vectors"], N)}
        if c["zeros"]:
            i["z"] = torch.randint(5, 12, (M, groups), dtype=torch.uint8, device="cuda", generator=g)
        return i

    page, hk, d = c["page"], c["heads_kv"], c["dim"]
    if c["op"] == "attn":
        lens = _lengths(c)
        width = max(1, -(-max(lens) // page))
        need = [-(-n // page) for n in lens]
    else:
        seq, pos, seqs = _tokens(c)
        width = max(1, -(-(max(pos) + 1) // page))
        need = [width] * seqs
    total = sum(need)
    order = torch.randperm(total + 1, device="cuda", generator=g).to(torch.int32)  # one page is nobody's
    need_d = torch.tensor(need, device="cuda")
    first = torch.cumsum(need_d, 0) - need_d
    col = torch.arange(width, device="cuda")
    table = order[(first[:, None] + col[None, :]).clamp(max=total)]
    table = torch.where(col[None, :] < need_d[:, None], table, NO_PAGE).to(torch.int32).contiguous()
    if c["op"] == "attn":
        i = {"k": normal(total + 1, page, hk, d), "v": normal(total + 1, page, hk, d), "table": table,
             "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "q": normal(c["batch"], c["heads_q"], d)}
        for b, n in enumerate(lens):  # slots past a sequence's end hold whatever was there: not numbers, at worst
            if n % page and b < 8:
                last = int(table[b, n // page])
                i["k"][last, n % page:] = math.nan
                i["v"][last, n % page:] = math.nan
        return i
    depth = torch.arange(max(pos) + 1, dtype=torch.float64, device="cuda")
    freq = 10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
    angle = depth[:, None] * freq[None, :]
    n = c["tokens"]
    return {"k": normal(total + 1, page, hk, d), "v": normal(total + 1, page, hk, d), "table": table,
            "seq": torch.tensor(seq, dtype=torch.int32, device="cuda") if c["prompt"] else None,
            "pos": torch.tensor(pos, dtype=torch.int32, device="cuda"), "cos": angle.cos().float(), "sin": angle.sin().float(),
            "new_q": normal(n, c["heads_q"], d), "new_k": normal(n, hk, d), "new_v": normal(n, hk, d)}


def prepare(case, seed):
    c, i = case, _inputs(case, seed)
    s = {"case": c, **i}
    t = TYPES[c["type"]]
    if c["op"] == "q4":
        s["y"] = torch.empty(c["vectors"], c["M"], dtype=t, device="cuda")
    elif c["op"] == "attn":
        s["out"] = torch.empty_like(i["q"])
        s["lse"] = torch.empty(c["batch"], c["heads_q"], dtype=torch.float32, device="cuda")
    else:
        s["q_out"] = torch.zeros_like(i["new_q"])
    if own:  # the handle that a program keeps beside its weights, or beside its cache
        import l2domain_b200 as L
        kind = L.DTYPES[c["type"]]
        if c["op"] == "q4":
            s["handle"] = L.Q4Matrix(i["w"], i["s"], c["M"], c["N"], c["group"], zeros=i["z"], dtype_x=kind,
                                     dtype_s=L.BF16 if c["type"] == "bf16" else L.F16)
        else:
            cache = L.KvCache(i["k"], i["v"], kind, num_pages=i["k"].shape[0], page_size=c["page"], heads=c["heads_kv"], head_dim=c["dim"])
            seqs, width = i["table"].shape
            if c["op"] == "attn":
                s["handle"] = L.PagedAttention(cache, i["table"], num_seqs=seqs, table_width=width, heads_q=c["heads_q"],
                                               scale=1.0 / math.sqrt(c["dim"]), window=c["window"])
            else:
                s["handle"] = L.KvAppend(cache, i["table"], num_seqs=seqs, table_width=width, heads_q=c["heads_q"], cos=i["cos"], sin=i["sin"],
                                         max_pos=i["cos"].shape[0], rot_dim=c["rot"], interleaved=c["interleaved"])
    return s


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        if c["op"] == "q4":
            s["handle"].gemv(s["x"], s["y"], vectors=c["vectors"])
            return s["y"]
        if c["op"] == "attn":
            s["handle"].decode(s["q"], s["out"], s["lens"], batch=c["batch"], lse=s["lse"])
            return {"out": s["out"], "lse": s["lse"]}
        s["handle"].append(s["new_k"], s["new_v"], s["pos"], tokens=c["tokens"], seq=s["seq"], q=s["new_q"], q_out=s["q_out"])
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    return {"q4": _plain_q4, "attn": _plain_attn, "append": _plain_append}[c["op"]](s)


def _plain_q4(s):
    c = s["case"]
    M, N, g, w = c["M"], c["N"], c["group"], s["w"]
    q = torch.stack([w & 15, w >> 4], dim=-1).reshape(M, -1)[:, :N].float()
    if c["zeros"]:
        q -= s["z"].float().repeat_interleave(g, dim=1)[:, :N]
    else:
        q -= 8.0
    q *= s["s"].float().repeat_interleave(g, dim=1)[:, :N]
    return torch.matmul(s["x"].float(), q.t()).to(s["x"].dtype)


def _plain_attn(s):
    c = s["case"]
    b, hk, d, page = c["batch"], c["heads_kv"], c["dim"], c["page"]
    rows = s["table"].shape[1] * page
    at = torch.arange(rows, device="cuda")
    lens = s["lens"].long()
    live = at[None, :] < lens[:, None]
    if c["window"]:
        live &= at[None, :] >= lens[:, None] - c["window"]
    pages = s["table"].long().clamp(min=0)
    k = torch.where(live[:, :, None, None], s["k"][pages].reshape(b, rows, hk, d).float(), 0.0).permute(0, 2, 3, 1)
    v = torch.where(live[:, :, None, None], s["v"][pages].reshape(b, rows, hk, d).float(), 0.0).permute(0, 2, 1, 3)
    q = s["q"].float().reshape(b, hk, c["heads_q"] // hk, d)
    score = torch.matmul(q, k) * (1.0 / math.sqrt(d))
    score = torch.where(live[:, None, None, :], score, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0.0, 1.0, total)
    lse = (top + torch.log(total)).reshape(b, -1)
    return {"out": out.reshape(b, -1, d).to(s["q"].dtype), "lse": lse}


def _plain_append(s):
    c = s["case"]
    half, page = c["rot"] // 2, c["page"]
    live = torch.nonzero(s["pos"] >= 0)[:, 0]
    pos = s["pos"][live].long()
    seq = live if s["seq"] is None else s["seq"][live].long()
    cos, sin = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]

    def rotated(x):
        y = x[live].float()
        r = y[:, :, : c["rot"]]
        a, b = (r[:, :, 0::2], r[:, :, 1::2]) if c["interleaved"] else (r[:, :, :half], r[:, :, half:])
        u, w = a * cos - b * sin, b * cos + a * sin
        r = torch.stack([u, w], dim=-1).flatten(2) if c["interleaved"] else torch.cat([u, w], dim=-1)
        return torch.cat([r, y[:, :, c["rot"]:]], dim=-1).to(x.dtype)

    s["q_out"][live] = rotated(s["new_q"])
    where = (s["table"][seq, pos // page].long(), pos % page)
    s["k"][where] = rotated(s["new_k"])
    s["v"][where] = s["new_v"][live]
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------

def exact(case, seed):
    c, i = case, _inputs(case, seed)
    if c["op"] == "q4":
        N, g = c["N"], c["group"]
        x = i["x"].double()
        column = torch.arange(N, device="cuda")
        parts = []
        for lo in range(0, c["M"], 4096):
            byte = i["w"][lo: lo + 4096][:, column // 2].long()
            q = ((byte >> (4 * (column % 2))) & 15).double()
            z = i["z"][lo: lo + 4096].double()[:, column // g] if c["zeros"] else 8.0
            parts.append(x @ ((q - z) * i["s"][lo: lo + 4096].double()[:, column // g]).t())
        return torch.cat(parts, dim=1)
    if c["op"] == "attn":
        hk, d, page = c["heads_kv"], c["dim"], c["page"]
        out = torch.zeros(i["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.full(i["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lengths(c)):
            lo = max(0, n - c["window"]) if c["window"] else 0
            if n <= lo:
                continue
            at = torch.arange(lo, n, device="cuda")
            of = i["table"][b].long()[at // page]
            for h in range(hk):
                q = i["q"][b].double().reshape(hk, -1, d)[h]
                score = q @ i["k"][of, at % page, h].double().t() / math.sqrt(d)
                l = torch.logsumexp(score, dim=1)
                mine = slice(h * q.shape[0], (h + 1) * q.shape[0])
                out[b, mine] = torch.exp(score - l[:, None]) @ i["v"][of, at % page, h].double()
                lse[b, mine] = l
        return {"out": out, "lse": lse}
    seq, pos, _ = _tokens(c)
    live = [t for t, p in enumerate(pos) if p >= 0]
    at = torch.tensor([pos[t] for t in live], device="cuda")
    row = torch.tensor(live, device="cuda")
    turn = torch.complex(i["cos"].double()[at], i["sin"].double()[at])[:, None, :]

    def turned(x):
        y = x[row].double()
        r = y[..., : c["rot"]]
        # each pair as one complex number, turned by its angle
        pair = r.unflatten(-1, (-1, 2)) if c["interleaved"] else r.unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        y[..., : c["rot"]] = z.flatten(-2) if c["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return y

    q = torch.zeros(i["new_q"].shape, dtype=torch.float64, device="cuda")
    q[row] = turned(i["new_q"])
    k, v = i["k"].double(), i["v"].double()
    page_of = i["table"].long()[torch.tensor([seq[t] for t in live], device="cuda"), at // c["page"]]
    k[page_of, at % c["page"]] = turned(i["new_k"])
    v[page_of, at % c["page"]] = i["new_v"][row].double()
    return {"q": q, "k": k, "v": v}

"""More decode operators of l2domain_b200, as measurable cases: a cache held in 4 bits, other scores, a mixture of experts.

* ``append4``  rotated keys, values and queries of new tokens; keys and values go to a paged cache in 4 bits (KvCache4, KvAppend)
* ``attn``     attention of one new token per sequence over that cache, or over one in the queries' type, with capped
               scores, a bias by distance and starts of documents (PagedAttention)
* ``moe``      a whole mixture-of-experts layer for a few tokens: router, the chosen experts' products, their sum (MoeLayer)

``run`` computes each in its plain form (elementary torch operations in 32 bits, rounded once at the end, the router's
sums in 64 because they choose), or, where ``own`` is set, through the package.  ``exact`` is the definition in 64 bits.

Definitions (all sums over real numbers; out-of-range means no contribution):

    append4 rotation: (a, b) -> (a cos - b sin, b cos + a sin) for the pairs of the first rot elements of a head, the pair
            (i, i + rot/2), or (2i, 2i + 1) where interleaved; each product and each sum is rounded to fp32.  A group of
            elements, lo = min(0, least) and hi = max(0, largest), is held as s (n - z), n and z in 0..15:
            s = hi c - lo c with c = fp32(1/15), each rounded to fp32, then up to a number whose last four bits are zero;
            z = min(15, rint(-lo / s)), n = clamp(rint(x / s) + z, 0, 15), quotients rounded to fp32; s = 0 gives n = z = 0.
            The token at position p of sequence s goes to slot p % page of page table[s, p // page]; p < 0 is padding.
            A page: blocks of 16 slots, in each the heads, in each head the nibbles [32 elements][slot][16 bytes], element
            2j in the low half of byte j, and one word per group and slot: the bits of s, with z in the last four.
    attn    softmax(f(q.k)) . v over positions max(start, len - window, 0) .. len - 1, query head h with key-value head
            h // (heads_q / heads_kv); f(x) = scale x, then cap tanh(f / cap) where capped, then + slope[h] (p - (len - 1)).
            No position at all gives 0, and -inf for the log-sum-exp
    moe     the top largest of router.x, ties to the lowest expert; w = softmax over all experts, taken at the chosen ones
            and, where normalised, divided by their sum; y = sum_k w_k down_k (silu(gate_k x) * (up_k x))
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
NO_PAGE = -1
FIFTEENTH = float(torch.tensor(1.0 / 15.0, dtype=torch.float32))


def listed():
    return [
        # One token for each of 32 sequences: the append of a decoding step, latency alone.
        {"name": "append4 32 tokens bf16", "op": "append4", "tokens": 32, "prompt": False, "heads_q": 32, "heads_kv": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 16, "group": 128, "type": "bf16"},
        # A chunk of prompts: every token of a few sequences, whose own attention reads the values as stored.
        {"name": "append4 8192 tokens fp16", "op": "append4", "tokens": 8192, "prompt": True, "heads_q": 32, "heads_kv": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 16, "group": 32, "type": "fp16"},
        # An odd number of tokens with padding among them, part of the head rotated, pairs side by side, a short last group.
        {"name": "append4 999 tokens fp32", "op": "append4", "tokens": 999, "prompt": True, "heads_q": 12, "heads_kv": 12, "dim": 80, "rot": 32, "interleaved": True, "page": 32, "group": 64, "type": "fp32"},
        # The first steps of one conversation: two blocks of the cache, latency alone.
        {"name": "attn4 1 x 17 bf16", "op": "attn", "bits": 4, "batch": 1, "length": 17, "ragged": False, "heads_q": 32, "heads_kv": 8, "dim": 128, "page": 16, "group": 128, "window": 0, "cap": 0.0, "slopes": False, "starts": False, "type": "bf16"},
        # A serving batch in the middle of its answers: lengths from nothing to 8192.
        {"name": "attn4 64 x 8192 ragged bf16", "op": "attn", "bits": 4, "batch": 64, "length": 8192, "ragged": True, "heads_q": 32, "heads_kv": 8, "dim": 128, "page": 16, "group": 128, "window": 0, "cap": 0.0, "slopes": False, "starts": False, "type": "bf16"},
        # One long document on fine groups: few rows, so the work has to be split over the length.
        {"name": "attn4 1 x 131072 fp16", "op": "attn", "bits": 4, "batch": 1, "length": 131072, "ragged": False, "heads_q": 32, "heads_kv": 4, "dim": 128, "page": 64, "group": 32, "window": 0, "cap": 0.0, "slopes": False, "starts": False, "type": "fp16"},
        # 32-bit queries, one key-value head per query head, an odd head, a sliding window and capped scores.
        {"name": "attn4 9 x 4000 window cap fp32", "op": "attn", "bits": 4, "batch": 9, "length": 4000, "ragged": True, "heads_q": 12, "heads_kv": 12, "dim": 80, "page": 32, "group": 32, "window": 1000, "cap": 30.0, "slopes": False, "starts": False, "type": "fp32"},
        # Capped scores over a cache in the queries' type: a serving batch of equal lengths.
        {"name": "attn 16 x 4096 cap bf16", "op": "attn", "bits": 0, "batch": 16, "length": 4096, "ragged": False, "heads_q": 32, "heads_kv": 8, "dim": 128, "page": 16, "group": 0, "window": 0, "cap": 50.0, "slopes": False, "starts": False, "type": "bf16"},
        # A bias by distance and several documents in each sequence, heads of 64, ragged, pages of an odd size.
        {"name": "attn 5 x 3001 distance fp16", "op": "attn", "bits": 0, "batch": 5, "length": 3001, "ragged": True, "heads_q": 16, "heads_kv": 16, "dim": 64, "page": 7, "group": 0, "window": 0, "cap": 0.0, "slopes": True, "starts": True, "type": "fp16"},
        # One token: the experts' weights are read for it alone.
        {"name": "moe 1 token bf16", "op": "moe", "tokens": 1, "hidden": 4096, "inner": 1536, "experts": 32, "top": 4, "normalize": True, "type": "bf16"},
        # A serving batch: nearly every expert has a token or a few.
        {"name": "moe 32 tokens bf16", "op": "moe", "tokens": 32, "hidden": 4096, "inner": 1024, "experts": 64, "top": 4, "normalize": True, "type": "bf16"},
        # Odd sizes, rows off every alignment, weights that are not normalised, 32 bits.
        {"name": "moe 5 tokens 1001 x 333 fp32", "op": "moe", "tokens": 5, "hidden": 1001, "inner": 333, "experts": 10, "top": 3, "normalize": False, "type": "fp32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append4", "attn", "attn", "attn", "moe", "moe"])
    kind = rng.choice(["fp16", "bf16", "bf16", "fp32"])
    if op == "moe":
        tokens, hidden, inner = _log(rng, 1, 200), _log(rng, 16, 8192), _log(rng, 8, 4096)
        experts = rng.choice([1, 4, 8, 16, 32, 60, 64, 128])
        while experts * hidden * inner * BYTES[kind] > 2 ** 29:
            inner = max(1, inner // 2)
        if rng.random() < 0.6:  # rows on 16-byte boundaries, as most weights have them
            hidden, inner = max(8, hidden // 8 * 8), max(8, inner // 8 * 8)
        return {"op": op, "tokens": tokens, "hidden": hidden, "inner": inner, "experts": experts,
                "top": min(experts, rng.choice([1, 2, 2, 4, 6, 8])), "normalize": rng.random() < 0.6, "type": kind}
    heads_kv = rng.choice([1, 2, 4, 8, 12])
    heads_q = heads_kv * rng.choice([1, 2, 4, 5, 8, 16])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    if op == "attn":
        bits = rng.choice([0, 4, 4])
        page = rng.choice([16, 16, 32, 64, 128] if bits else [1, 7, 16, 16, 32, 64, 128])
        batch, length = _log(rng, 1, 96), _log(rng, 1, 131072)
        while batch * length * heads_kv * dim * (2 if bits else BYTES[kind]) > 2 ** 29:
            length = max(1, length // 2)
        cap = rng.choice([0.0, 20.0, 50.0])
        return {"op": op, "bits": bits, "batch": batch, "length": length, "ragged": rng.random() < 0.7, "heads_q": heads_q,
                "heads_kv": heads_kv, "dim": dim, "page": page, "group": rng.choice([32, 64, 128]) if bits else 0,
                "window": rng.choice([0, 0, 0, 1 + length // 3]), "cap": cap, "slopes": rng.random() < (0.4 if bits or cap else 0.8),
                "starts": rng.random() < 0.3, "type": kind}
    tokens = _log(rng, 1, 8192)
    while tokens * (heads_q + 2 * heads_kv) * dim > 2 ** 26:
        tokens = max(1, tokens // 2)
    return {"op": op, "tokens": tokens, "prompt": rng.random() < 0.5, "heads_q": heads_q, "heads_kv": heads_kv, "dim": dim,
            "rot": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.4, "page": rng.choice([16, 16, 32, 64, 128]),
            "group": rng.choice([32, 64, 128]), "type": kind}


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


def _starts(c):
    """Where each sequence's last document begins: at its front, in its middle, near its end, behind it."""
    return [(0, n // 3, n - n // 8, n + 1)[i % 4] if c["starts"] else 0 for i, n in enumerate(_lengths(c))]


def _keys(c):
    w = c["window"]
    return sum(max(0, n - max(s, n - w if w else 0, 0)) for n, s in zip(_lengths(c), _starts(c)))


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


def _row_bytes(c):
    """Of one key or value of one head: nibbles and a word per group, or elements."""
    if c["op"] == "attn" and not c["bits"]:
        return c["dim"] * BYTES[c["type"]]
    return (c["dim"] + 1) // 2 + 4 * -(-c["dim"] // c["group"])


def work(c):
    e = BYTES[c["type"]]
    if c["op"] == "moe":
        T, H, F, E, K = (c[k] for k in ("tokens", "hidden", "inner", "experts", "top"))
        # How many experts the tokens choose follows from the inputs; on average it is this many.
        chosen = E * (1.0 - (1.0 - K / E) ** T)
        return {"bytes": (chosen * 3 * H * F + E * H + 2 * T * H) * e + 8 * T * K, "flops": 6 * T * K * H * F + 2 * T * E * H}
    if c["op"] == "attn":
        heads, keys = c["heads_q"] * c["batch"], _keys(c)
        return {"bytes": 2 * keys * c["heads_kv"] * _row_bytes(c) + 2 * heads * c["dim"] * e + 4 * heads, "flops": 4 * keys * c["heads_q"] * c["dim"]}
    live = sum(p >= 0 for p in _tokens(c)[1])
    hq, hk, d = c["heads_q"], c["heads_kv"], c["dim"]
    return {"bytes": live * ((2 * hq + 4 * hk) * d * e + 2 * hk * _row_bytes(c) + 4 * c["rot"] + 12),
            "flops": live * (3 * (hq + hk) * c["rot"] + 8 * hk * d)}


# ------------------------------------------------------------------------------------------------
# The cache in 4 bits
# ------------------------------------------------------------------------------------------------

def _quantise(x, group):
    """(n, word) of the last axis: a number 0..15 of each element, and the word of each group."""
    d = x.shape[-1]
    groups, wide = -(-d // group), -(-d // group) * group
    x = torch.nn.functional.pad(x, (0, wide - d)).unflatten(-1, (groups, group))
    lo, hi = x.amin(-1).clamp(max=0.0), x.amax(-1).clamp(min=0.0)
    s = (hi * FIFTEENTH - lo * FIFTEENTH).contiguous().view(torch.int32)
    s = ((s + 15) & ~15).view(torch.float32)
    by = torch.where(s == 0.0, 1.0, s)
    z = torch.round(-lo / by).clamp(max=15.0)
    n = (torch.round(x / by[..., None]) + z[..., None]).clamp(0.0, 15.0)
    return n.to(torch.uint8).flatten(-2)[..., :d], s.view(torch.int32) | z.int()


def _stands_for(n, word, group):
    """The numbers that 4-bit ones and their groups' words stand for, in fp32 (exactly)."""
    s, z = (word & ~15).view(torch.float32), (word & 15).float()
    d = n.shape[-1]
    return s.repeat_interleave(group, -1)[..., :d] * (n.float() - z.repeat_interleave(group, -1)[..., :d])


def _views(buffer, c):
    """A cache's bytes as nibbles [page][block][head][32 elements][slot][16 bytes] and words [page][block][head][group][slot]."""
    chunks, groups = -(-c["dim"] // 32), -(-c["dim"] // c["group"])
    tile = buffer.view(buffer.shape[0], c["page"] // 16, c["heads_kv"], 256 * chunks + 64 * groups)
    return tile[..., : 256 * chunks].unflatten(-1, (chunks, 16, 16)), tile[..., 256 * chunks:].view(torch.int32).unflatten(-1, (groups, 16))


def _read(buffer, c):
    """[page][slot][head][dim] in fp32, of any number of pages."""
    nibbles, words = _views(buffer, c)
    n = nibbles.permute(0, 1, 4, 2, 3, 5).flatten(1, 2).flatten(-2)
    n = torch.stack([n & 15, n >> 4], -1).flatten(-2)[..., : c["dim"]]
    return _stands_for(n, words.permute(0, 1, 4, 2, 3).flatten(1, 2).contiguous(), c["group"])


def _packed(n, word):
    """Nibbles [..][dim] as bytes [..][32 elements][16], beside their words."""
    n = torch.nn.functional.pad(n, (0, -n.shape[-1] % 32))
    return (n[..., 0::2] | n[..., 1::2] << 4).unflatten(-1, (-1, 16)), word


def _filled(x, c):
    """A cache's bytes from values [page][slot][head][dim]."""
    chunks, groups = -(-c["dim"] // 32), -(-c["dim"] // c["group"])
    out = torch.empty(x.shape[0], c["page"] // 16 * c["heads_kv"] * (256 * chunks + 64 * groups), dtype=torch.uint8, device=x.device)
    nibbles, words = _views(out, c)
    n, word = _packed(*_quantise(x.float(), c["group"]))
    nibbles.copy_(n.unflatten(1, (-1, 16)).permute(0, 1, 3, 4, 2, 5))
    words.copy_(word.unflatten(1, (-1, 16)).permute(0, 1, 3, 4, 2))
    return out


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------

def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[c["type"]]

    def normal(*shape, scale=1.0):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=g).mul_(scale).to(t)

    if c["op"] == "moe":
        T, H, F, E = c["tokens"], c["hidden"], c["inner"], c["experts"]
        return {"x": normal(T, H), "router": normal(E, H, scale=1.5 / math.sqrt(H)), "gate": normal(E, F, H, scale=1.0 / math.sqrt(H)),
                "up": normal(E, F, H, scale=1.0 / math.sqrt(H)), "down": normal(E, H, F, scale=1.0 / math.sqrt(F))}

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
        i = {"table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "q": normal(c["batch"], c["heads_q"], d), "starts": None, "slopes": None}
        for name in ("k", "v"):
            x = normal(total + 1, page, hk, d)
            if c["bits"]:
                x = torch.cat([_filled(part, c) for part in x.split(max(1, 2 ** 25 // (page * hk * d)))])
            i[name] = x
            for b, n in enumerate(lens):  # slots past a sequence's end hold whatever was there: not numbers, at worst
                if n % page and b < 8:
                    last = int(table[b, n // page])
                    if c["bits"]:
                        at = torch.arange(n % page, page, device="cuda")
                        _views(x, c)[1].view(torch.float32)[last, at // 16, :, :, at % 16] = math.nan
                    else:
                        x[last, n % page:] = math.nan
        if c["starts"]:
            i["starts"] = torch.tensor(_starts(c), dtype=torch.int32, device="cuda")
        if c["slopes"]:  # a geometric row, from 2^(-8 / heads) to 2^-8
            h = torch.arange(1, c["heads_q"] + 1, device="cuda", dtype=torch.float64)
            i["slopes"] = torch.exp2(-8.0 * h / c["heads_q"]).float()
        return i
    depth = torch.arange(max(pos) + 1, dtype=torch.float64, device="cuda")
    freq = 10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
    angle = depth[:, None] * freq[None, :]
    n = c["tokens"]
    empty = torch.zeros(total + 1, page // 16 * hk * (256 * -(-d // 32) + 64 * -(-d // c["group"])), dtype=torch.uint8, device="cuda")
    return {"k": empty, "v": empty.clone(), "table": table, "seq": torch.tensor(seq, dtype=torch.int32, device="cuda") if c["prompt"] else None,
            "pos": torch.tensor(pos, dtype=torch.int32, device="cuda"), "cos": angle.cos().float(), "sin": angle.sin().float(),
            "new_q": normal(n, c["heads_q"], d), "new_k": normal(n, hk, d), "new_v": normal(n, hk, d)}


def prepare(case, seed):
    c, i = case, _inputs(case, seed)
    s = {"case": c, **i}
    if c["op"] == "moe":
        T, K = c["tokens"], c["top"]
        s["y"] = torch.empty_like(i["x"])
        s["ids"] = torch.empty(T, K, dtype=torch.int32, device="cuda")
        s["weights"] = torch.empty(T, K, dtype=torch.float32, device="cuda")
    elif c["op"] == "attn":
        s["out"] = torch.empty_like(i["q"])
        s["lse"] = torch.empty(c["batch"], c["heads_q"], dtype=torch.float32, device="cuda")
    else:
        s["q_out"], s["k_out"], s["v_out"] = (torch.zeros_like(i[name]) for name in ("new_q", "new_k", "new_v"))
    if own:  # the handle that a program keeps beside its weights, or beside its cache
        import l2domain_b200 as L
        kind = L.DTYPES[c["type"]]
        if c["op"] == "moe":
            s["handle"] = L.MoeLayer(i["router"], i["gate"], i["up"], i["down"], hidden=c["hidden"], inner=c["inner"], experts=c["experts"],
                                     top=c["top"], max_tokens=c["tokens"], dtype=kind, normalize=c["normalize"])
            return s
        four = c["op"] == "append4" or c["bits"]
        fields = dict(num_pages=i["k"].shape[0], page_size=c["page"], heads=c["heads_kv"], head_dim=c["dim"])
        cache = L.KvCache4(i["k"], i["v"], kind, group=c["group"], **fields) if four else L.KvCache(i["k"], i["v"], kind, **fields)
        seqs, width = i["table"].shape
        if c["op"] == "attn":
            s["handle"] = L.PagedAttention(cache, i["table"], num_seqs=seqs, table_width=width, heads_q=c["heads_q"],
                                           scale=1.0 / math.sqrt(c["dim"]), window=c["window"], cap=c["cap"], slopes=i["slopes"])
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
        if c["op"] == "moe":
            s["handle"].forward(s["x"], s["y"], tokens=c["tokens"], ids=s["ids"], weights=s["weights"])
            return {"y": s["y"], "ids": s["ids"], "weights": s["weights"]}
        if c["op"] == "attn":
            s["handle"].decode(s["q"], s["out"], s["lens"], batch=c["batch"], lse=s["lse"], starts=s["starts"])
            return {"out": s["out"], "lse": s["lse"]}
        s["handle"].append(s["new_k"], s["new_v"], s["pos"], tokens=c["tokens"], seq=s["seq"], q=s["new_q"], q_out=s["q_out"],
                           k_out=s["k_out"], v_out=s["v_out"])
        return {"q": s["q_out"], "k_out": s["k_out"], "v_out": s["v_out"], "k": s["k"], "v": s["v"]}
    return {"moe": _plain_moe, "attn": _plain_attn, "append4": _plain_append4}[c["op"]](s)


def _plain_moe(s):
    c, x = s["case"], s["x"].float()
    T, E, K = c["tokens"], c["experts"], c["top"]
    logits = torch.matmul(s["x"].double(), s["router"].double().t())
    ids = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :K]
    p = torch.softmax(logits, dim=-1).gather(1, ids)
    w = (p / p.sum(-1, keepdim=True) if c["normalize"] else p).float()
    if T * K <= E:  # the chosen experts alone, one after the other
        at = ids.flatten()
        each = x.repeat_interleave(K, 0)[:, :, None]
        gate, up = torch.matmul(s["gate"][at].float(), each), torch.matmul(s["up"][at].float(), each)
        y = torch.matmul(s["down"][at].float(), gate / (1.0 + torch.exp(-gate)) * up)
        y = (y.view(T, K, -1) * w[:, :, None]).sum(1)
    else:  # every expert for every token
        gate, up = torch.matmul(x, s["gate"].float().transpose(1, 2)), torch.matmul(x, s["up"].float().transpose(1, 2))
        y = torch.matmul(gate / (1.0 + torch.exp(-gate)) * up, s["down"].float().transpose(1, 2))  # [expert][token][hidden]
        of = torch.zeros(T, E, device="cuda").scatter_(1, ids, w)
        y = torch.where(of.t()[:, :, None] != 0.0, y * of.t()[:, :, None], 0.0).sum(0)
    return {"y": y.to(s["x"].dtype), "ids": ids.int(), "weights": w}


def _plain_attn(s):
    c = s["case"]
    b, hk, d, page = c["batch"], c["heads_kv"], c["dim"], c["page"]
    rows = s["table"].shape[1] * page
    at = torch.arange(rows, device="cuda")
    lens = s["lens"].long()
    live = at[None, :] < lens[:, None]
    if c["window"]:
        live &= at[None, :] >= lens[:, None] - c["window"]
    if c["starts"]:
        live &= at[None, :] >= s["starts"].long()[:, None]
    pages = s["table"].long().clamp(min=0)

    def rows_of(cache):
        x = _read(cache[pages.flatten()], c) if c["bits"] else cache[pages].float()
        return torch.where(live[:, :, None, None], x.reshape(b, rows, hk, d), 0.0)

    q = s["q"].float().reshape(b, hk, c["heads_q"] // hk, d)
    score = torch.matmul(q, rows_of(s["k"]).permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    if c["slopes"]:
        score = score + s["slopes"].view(1, hk, -1, 1) * (at[None, :] - (lens[:, None] - 1)).float()[:, None, None, :]
    score = torch.where(live[:, None, None, :], score, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p, rows_of(s["v"]).permute(0, 2, 1, 3)) / torch.where(total == 0.0, 1.0, total)
    lse = (top + torch.log(total)).reshape(b, -1)
    return {"out": out.reshape(b, -1, d).to(s["q"].dtype), "lse": lse}


def _plain_append4(s):
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
        return torch.cat([r, y[:, :, c["rot"]:]], dim=-1)

    def stored(x, cache, out):
        n, word = _quantise(x, c["group"])
        nibbles, words = _views(cache, c)
        of, slot = s["table"][seq, pos // page].long(), pos % page
        packed, _ = _packed(n, word)
        nibbles[of, slot // 16, :, :, slot % 16] = packed
        words[of, slot // 16, :, :, slot % 16] = word
        out[live] = _stands_for(n, word, c["group"]).to(out.dtype)

    s["q_out"][live] = rotated(s["new_q"]).to(s["new_q"].dtype)
    stored(rotated(s["new_k"]), s["k"], s["k_out"])
    stored(s["new_v"][live].float(), s["v"], s["v_out"])
    return {"q": s["q_out"], "k_out": s["k_out"], "v_out": s["v_out"], "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------

def exact(case, seed):
    c, i = case, _inputs(case, seed)
    return {"moe": _exact_moe, "attn": _exact_attn, "append4": _exact_append4}[c["op"]](c, i)


def _exact_moe(c, i):
    x = i["x"].double()
    logits = x @ i["router"].double().t()
    chance = torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True)).cpu()
    y = torch.zeros_like(x)
    weights = torch.zeros(c["tokens"], c["top"], dtype=torch.float64)
    users = {}
    for t, row in enumerate(logits.cpu().tolist()):
        best = sorted(range(c["experts"]), key=lambda e: (-row[e], e))[: c["top"]]
        weights[t] = chance[t, best]
        if c["normalize"]:
            weights[t] /= weights[t].sum()
        for k, e in enumerate(best):
            users.setdefault(e, []).append((t, k))
    for e, of in sorted(users.items()):
        rows = torch.tensor([t for t, _ in of], device="cuda")
        gate, up = x[rows] @ i["gate"][e].double().t(), x[rows] @ i["up"][e].double().t()
        part = (gate * torch.sigmoid(gate) * up) @ i["down"][e].double().t()
        y.index_add_(0, rows, part * torch.stack([weights[t, k] for t, k in of]).cuda()[:, None])
    return {"y": y, "ids": None, "weights": weights}


def _exact_attn(c, i):
    hk, d, page = c["heads_kv"], c["dim"], c["page"]
    out = torch.zeros(i["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(i["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")

    def head(cache, of, slot, h):
        if not c["bits"]:
            return cache[of, slot, h].double()
        nibbles, words = _views(cache, c)
        byte, word = nibbles[of, slot // 16, h, :, slot % 16].reshape(len(of), -1), words[of, slot // 16, h, :, slot % 16]
        j = torch.arange(d, device="cuda")
        number = (byte[:, j // 2].long() >> (4 * (j % 2))) & 15
        word = word[:, j // c["group"]]
        return (word - word % 16).view(torch.float32).double() * (number - word.long() % 16).double()

    for b, (n, start) in enumerate(zip(_lengths(c), _starts(c))):
        lo = max(start, n - c["window"] if c["window"] else 0, 0)
        if n <= lo:
            continue
        at = torch.arange(lo, n, device="cuda")
        of = i["table"][b].long()[at // page]
        for h in range(hk):
            q = i["q"][b].double().reshape(hk, -1, d)[h]
            score = q @ head(i["k"], of, at % page, h).t() / math.sqrt(d)
            mine = slice(h * q.shape[0], (h + 1) * q.shape[0])
            if c["cap"]:
                score = c["cap"] * torch.tanh(score / c["cap"])
            if c["slopes"]:
                score = score + i["slopes"][mine].double()[:, None] * (at - (n - 1)).double()[None, :]
            l = torch.logsumexp(score, dim=1)
            out[b, mine] = torch.exp(score - l[:, None]) @ head(i["v"], of, at % page, h)
            lse[b, mine] = l
    return {"out": out, "lse": lse}


def _exact_append4(c, i):
    seq, pos, _ = _tokens(c)
    live = [t for t, p in enumerate(pos) if p >= 0]
    at = torch.tensor([pos[t] for t in live], device="cuda")
    row = torch.tensor(live, device="cuda")
    cos, sin = i["cos"].double()[at][:, None, :], i["sin"].double()[at][:, None, :]

    def once(x):  # of one operation on fp32 numbers in 64 bits: as fp32 has it
        return x.float().double()

    def turned(x, rounded):
        r = (lambda v: v) if not rounded else once
        y = x[row].double()
        pair = y[..., : c["rot"]].unflatten(-1, (-1, 2)).movedim(-1, 0) if c["interleaved"] else y[..., : c["rot"]].unflatten(-1, (2, -1)).movedim(-2, 0)
        a, b = pair[0], pair[1]
        both = torch.stack([r(r(a * cos) - r(b * sin)), r(r(b * cos) + r(a * sin))], -1 if c["interleaved"] else -2)
        y[..., : c["rot"]] = both.flatten(-2)
        return y

    def held(x):
        parts = []
        for lo in range(0, c["dim"], c["group"]):
            g = x[..., lo: lo + c["group"]]
            least, most = g.amin(-1, keepdim=True).clamp(max=0.0), g.amax(-1, keepdim=True).clamp(min=0.0)
            s = once(once(most * FIFTEENTH) - once(least * FIFTEENTH))
            unit = torch.exp2(torch.floor(torch.log2(torch.where(s == 0, 1.0, s))) - 19.0)  # of a number of 20 bits
            s = torch.ceil(s / unit) * unit
            by = torch.where(s == 0, 1.0, s)
            z = torch.round(once(-least / by)).clamp(max=15.0)
            parts.append(s * ((torch.round(once(g / by)) + z).clamp(0.0, 15.0) - z))
        full = torch.zeros(c["tokens"], *x.shape[1:], dtype=torch.float64, device="cuda")
        full[row] = torch.cat(parts, -1)
        return full

    q = torch.zeros(i["new_q"].shape, dtype=torch.float64, device="cuda")
    q[row] = turned(i["new_q"], False)
    return {"q": q, "k_out": held(turned(i["new_k"], True)), "v_out": held(i["new_v"][row].double()), "k": None, "v": None}

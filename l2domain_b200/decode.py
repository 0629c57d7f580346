"""A layer's decoding step, from this package's operators: 4-bit projections, the append to the paged cache with its
rotation, attention over the cache, the 4-bit output projection, and a mixture of experts.

    python -m l2domain_b200.decode --batch 8 --length 4096 [--hidden 4096 --heads 32 --kv-heads 8 --head-dim 128]
                                   [--cache-bits 4 --cap 50 --slopes] [--experts 64 --top 4 --inner 1024]

runs steps of that shape on synthetic weights and an already filled cache, as one captured graph, and prints the
mean time of a step with the bytes it cannot do without.  Without --experts a step is the attention part alone.
"""
from __future__ import annotations

import argparse
import json

import l2domain_b200 as L


def pack_q4(weights, group: int, zero_points: bool = False, dtype_s: int = L.F16):
    """(bytes, scales, zeros) of a weight matrix [M][N] (a torch tensor), as :class:`Q4Matrix` takes them.

    Without zero points q is rounded to -8..7 of the group's largest magnitude / 7 (zeros is None); with them to
    0..15 of the group's range.  Rows of bytes are padded to 16 and rows of scales to 8, which are read fastest:
    pass ``bytes.stride(0)`` as ldw and ``scales.stride(0)`` as lds."""
    import torch

    M, N = weights.shape
    groups = -(-N // group)
    w = torch.zeros(M, groups * group, dtype=torch.float32, device=weights.device)
    w[:, :N] = weights.float()
    w = w.view(M, groups, group)
    if N % group:  # the short group's padding must not stretch its range
        w[:, -1, N % group:] = w[:, -1, :1]
    if zero_points:
        lo, hi = w.amin(-1).clamp(max=0.0), w.amax(-1).clamp(min=0.0)
        s = (hi - lo) / 15.0
    else:
        s = w.abs().amax(-1) / 7.0
    s = s.to({L.F32: torch.float32, L.F16: torch.float16, L.BF16: torch.bfloat16}[dtype_s])
    step = torch.where(s == 0, torch.ones_like(s), s).float()[..., None]
    z = torch.round(-lo[..., None] / step).clamp(0, 15) if zero_points else torch.full_like(step, 8.0)
    q = (torch.round(w / step) + z).clamp(0, 15).to(torch.uint8).view(M, -1)[:, :N]
    if N % 2:
        q = torch.cat([q, torch.zeros(M, 1, dtype=torch.uint8, device=q.device)], 1)
    packed = torch.zeros(M, -(-q.shape[1] // 32) * 16, dtype=torch.uint8, device=q.device)
    packed[:, : q.shape[1] // 2] = q[:, 0::2] | (q[:, 1::2] << 4)
    scales = torch.zeros(M, -(-groups // 8) * 8, dtype=s.dtype, device=s.device)
    scales[:, :groups] = s
    if not zero_points:
        return packed, scales, None
    zeros = torch.zeros(scales.shape, dtype=torch.uint8, device=s.device)
    zeros[:, :groups] = z[..., 0].to(torch.uint8)
    return packed, scales, zeros


class DecodeAttention:
    """One layer's attention for ``batch`` sequences of up to ``max_len`` tokens, in bf16 with 4-bit weights.

    ``w_qkv`` [(heads + 2 kv_heads) * head_dim][hidden] and ``w_out`` [hidden][heads * head_dim] are packed once.
    ``cache_bits`` is 16, or 4 with a scale per ``cache_group`` elements; ``cap`` and ``slopes`` as in :class:`PagedAttention`.
    :meth:`step` takes one new token per sequence; it allocates nothing and may be captured into a graph."""

    def __init__(self, w_qkv, w_out, heads: int, kv_heads: int, head_dim: int, batch: int, max_len: int, group: int = 128,
                 page_size: int = 16, theta: float = 10000.0, device: int = 0, cache_bits: int = 16, cache_group: int = 128,
                 cap: float = 0.0, slopes=None):
        import torch

        self.heads, self.kv_heads, self.head_dim, self.batch = heads, kv_heads, head_dim, batch
        hidden = w_out.shape[0]
        dev = torch.device("cuda", device)

        def matrix(w):
            packed, scales, zeros = pack_q4(w, group, dtype_s=L.BF16)
            return L.Q4Matrix(packed, scales, w.shape[0], w.shape[1], group, zeros=zeros, dtype_x=L.BF16, dtype_s=L.BF16,
                              ldw=packed.stride(0), lds=scales.stride(0), device=device)

        self.qkv_matrix, self.out_matrix = matrix(w_qkv), matrix(w_out)
        width = -(-max_len // page_size)
        pages = batch * width
        if cache_bits == 4:
            shape, kind = (pages, L.kv4_page_bytes(page_size, kv_heads, head_dim, cache_group)), torch.uint8
            self.key_bytes = (head_dim + 1) // 2 + 4 * -(-head_dim // cache_group)  # of one key or value of one head
        elif cache_bits == 16:
            shape, kind = (pages, page_size, kv_heads, head_dim), torch.bfloat16
            self.key_bytes = 2 * head_dim
        else:
            raise ValueError(f"a cache of {cache_bits} bits: 16 or 4")
        self.k, self.v = (torch.zeros(shape, dtype=kind, device=dev) for _ in range(2))
        # Pages in the order sequences get them, one after the other; any other order does as well.
        self.table = torch.arange(batch * width, dtype=torch.int32, device=dev).view(width, batch).t().contiguous()
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        if cache_bits == 4:
            cache = L.KvCache4(self.k, self.v, L.BF16, pages, page_size, kv_heads, head_dim, cache_group, device=device)
        else:
            cache = L.KvCache(self.k, self.v, L.BF16, pages, page_size, kv_heads, head_dim, device=device)
        row = (heads + 2 * kv_heads) * head_dim
        self.cos, self.sin = L.rotation_tables(max_len, head_dim, theta, device=dev)
        self.append = L.KvAppend(cache, self.table, batch, width, heads_q=heads, cos=self.cos, sin=self.sin, max_pos=max_len,
                                 rot_dim=head_dim, k_token=row, v_token=row, q_token=row, q_out_token=row, status=self.status)
        self.attention = L.PagedAttention(cache, self.table, batch, width, heads, q_token=row, status=self.status, cap=cap, slopes=slopes)
        self.qkv = torch.zeros(batch, row, dtype=torch.bfloat16, device=dev)
        self.mixed = torch.zeros(batch, heads * head_dim, dtype=torch.bfloat16, device=dev)
        self.hidden = hidden

    def prompt(self, qkv, pos, seq, tokens: int, k_out=None, v_out=None, stream=None) -> None:
        """Appends ``tokens`` tokens of prompts, rows of ``qkv`` [tokens][(heads + 2 kv_heads) * head_dim] at positions pos
        of sequences seq (int32), and rotates their queries in place.  ``k_out`` and ``v_out`` (a cache of 4 bits; bf16, strided as
        qkv): keys and values as the cache holds them, for the prompt's own attention."""
        import torch

        hd, kv = self.heads * self.head_dim, self.kv_heads * self.head_dim
        row, dev = hd + 2 * kv, self.status.device

        def rows_of(name, t, least):
            if t.dtype != torch.bfloat16 or t.dim() != 2 or t.shape[0] < tokens or t.shape[1] < least or t.device != dev or (
                    t.stride(1) != 1 or (tokens > 1 and t.stride(0) != row)):
                raise ValueError(f"{name} is {t.dtype} {list(t.shape)} strided {t.stride()} on {t.device}: bfloat16, {tokens} rows of "
                                 f"{least} elements and more, strided ({row}, 1), on {dev}")

        rows_of("qkv", qkv, row)
        for name, t in (("k_out", k_out), ("v_out", v_out)):
            if hasattr(t, "dtype"):  # a tensor, and not an address
                rows_of(name, t, kv)
        for name, t in (("pos", pos), ("seq", seq)):
            if hasattr(t, "dtype") and (t.dtype != torch.int32 or t.numel() < tokens or not t.is_contiguous() or t.device != dev):
                raise ValueError(f"{name} is {t.dtype} {list(t.shape)} on {t.device}: int32, {tokens} or more in a row, on {dev}")
        self.append.append(qkv[:, hd:], qkv[:, hd + kv:], pos, tokens, seq=seq, q=qkv, q_out=qkv, k_out=k_out, v_out=v_out, stream=stream)

    def step(self, x, pos, lens, out, stream=None, starts=None) -> None:
        """out[b] = W_out . attention of the token x[b] at position pos[b] over itself and the lens[b] - 1 before it, those from
        starts[b] on where given (pos, lens and starts int32 on the device; lens = pos + 1)."""
        n, hd = self.batch, self.heads * self.head_dim
        self.qkv_matrix.gemv(x, self.qkv, vectors=n, stream=stream)
        keys = self.qkv[:, hd:]
        values = self.qkv[:, hd + self.kv_heads * self.head_dim:]
        self.append.append(keys, values, pos, n, q=self.qkv, q_out=self.qkv, stream=stream)
        self.attention.decode(self.qkv, self.mixed, lens, n, stream=stream, starts=starts)
        self.out_matrix.gemv(self.mixed, out, vectors=n, stream=stream)


class DecodeExperts:
    """One layer's experts for up to ``batch`` tokens: ``router`` [experts][hidden], ``gate`` and ``up`` [experts][inner][hidden],
    ``down`` [experts][hidden][inner], of one type on one device (see :class:`MoeLayer`); rows and experts may be strided.
    :meth:`step` allocates nothing and may be captured."""

    def __init__(self, router, gate, up, down, top: int, batch: int, normalize: bool = True, device: int = 0):
        import torch

        kind = {torch.float32: L.F32, torch.float16: L.F16, torch.bfloat16: L.BF16}.get(gate.dtype)
        if kind is None or gate.dim() != 3:
            raise ValueError(f"gate is {gate.dtype} {list(gate.shape)}: [experts][inner][hidden] of 32 or 16 bits")
        experts, inner, hidden = gate.shape
        for name, t, shape in (("router", router, (experts, hidden)), ("gate", gate, (experts, inner, hidden)), ("up", up, (experts, inner, hidden)),
                               ("down", down, (experts, hidden, inner))):
            if t.dtype != gate.dtype:
                raise ValueError(f"{name} is {t.dtype}, gate {gate.dtype}: all of one type")
            if tuple(t.shape) != shape:
                raise ValueError(f"{name} has the shape {list(t.shape)}, not {list(shape)}")
            if t.shape[-1] > 1 and t.stride(-1) != 1:
                raise ValueError(f"{name}: the elements of a row must be next to each other (transposed?)")
            if any(n > 1 and step == 0 for n, step in zip(t.shape, t.stride())):
                raise ValueError(f"{name} is expanded: every row must be in memory")
        for name, t in (("router", router), ("gate", gate), ("up", up), ("down", down)):
            if t.device != torch.device("cuda", device):
                raise ValueError(f"{name} is on {t.device}, not on cuda:{device}")

        def step(t, dim):  # 0 (dense) where there is one, whose stride says nothing
            return t.stride(dim) if t.shape[dim] > 1 else 0

        self.layer = L.MoeLayer(router, gate, up, down, hidden, inner, experts, top, batch, kind, normalize, router_row=step(router, 0),
                                gate_row=step(gate, 1), up_row=step(up, 1), down_row=step(down, 1), gate_expert=step(gate, 0),
                                up_expert=step(up, 0), down_expert=step(down, 0), device=device)
        self.batch = batch
        self.ids = torch.zeros(batch, top, dtype=torch.int32, device=gate.device)

    def step(self, x, out, stream=None) -> None:
        """out[b] of the token x[b]; ``ids`` holds the experts that it chose."""
        self.layer.forward(x, out, self.batch, ids=self.ids, stream=stream)


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--length", type=int, default=4096)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--head-dim", type=int, default=128)
    ap.add_argument("--cache-bits", type=int, default=16, choices=(16, 4))
    ap.add_argument("--cap", type=float, default=0.0, help="of scores, by a tanh (0: none)")
    ap.add_argument("--slopes", action="store_true", help="a bias by distance")
    ap.add_argument("--experts", type=int, default=0)
    ap.add_argument("--top", type=int, default=4)
    ap.add_argument("--inner", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=200)
    args = ap.parse_args()

    import torch

    torch.cuda.set_device(0)
    g = torch.Generator(device="cuda").manual_seed(0)
    row = (args.heads + 2 * args.kv_heads) * args.head_dim

    def normal(*shape, scale=1.0):
        return (torch.empty(shape, device="cuda").normal_(generator=g) * scale).to(torch.bfloat16)

    layer = DecodeAttention(normal(row, args.hidden, scale=0.02), normal(args.hidden, args.heads * args.head_dim, scale=0.02),
                            args.heads, args.kv_heads, args.head_dim, args.batch, args.length + args.steps + 16, cache_bits=args.cache_bits,
                            cap=args.cap, slopes=L.distance_slopes(args.heads, device="cuda") if args.slopes else None)
    if args.cache_bits == 16:
        layer.k.normal_(generator=g)
        layer.v.normal_(generator=g)
    else:  # as a prompt of every sequence, some tokens at a time
        for first in range(0, args.length, 256):
            n = min(256, args.length - first)
            at = torch.arange(first, first + n, dtype=torch.int32, device="cuda").repeat(args.batch)
            of = torch.arange(args.batch, dtype=torch.int32, device="cuda").repeat_interleave(n)
            layer.prompt(normal(args.batch * n, row), at, of, args.batch * n, stream=torch.cuda.current_stream())
    experts = None
    if args.experts:
        e, f, h = args.experts, args.inner, args.hidden
        experts = DecodeExperts(normal(e, h, scale=h ** -0.5), normal(e, f, h, scale=h ** -0.5), normal(e, f, h, scale=h ** -0.5),
                                normal(e, h, f, scale=f ** -0.5), args.top, args.batch)
    x, out = normal(args.batch, args.hidden), torch.empty(args.batch, args.hidden, dtype=torch.bfloat16, device="cuda")
    pos = torch.full((args.batch,), args.length - 1, dtype=torch.int32, device="cuda")
    lens = pos + 1
    after = torch.empty_like(out)

    def step(stream):
        layer.step(x, pos, lens, out, stream=stream)
        if experts:
            experts.step(out, after, stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())  # which fills the cache, x, pos and lens
    with torch.cuda.stream(side):
        step(side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream())
        pos.add_(1)
        lens.add_(1)
    before = 10  # steps, each of which leaves the cache a token longer
    for _ in range(before):
        graph.replay()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(args.steps):
        graph.replay()
    end.record()
    end.synchronize()
    us = start.elapsed_time(end) / args.steps * 1e3
    keys = args.length + before + (args.steps - 1) / 2  # of a sequence in the timed steps, on average
    cache = int(2 * args.batch * keys * args.kv_heads * layer.key_bytes)
    weights = (row * args.hidden + args.hidden * args.heads * args.head_dim) * (0.5 + 2 / 128)
    if experts:  # those that the last step chose
        weights += 2 * (experts.ids.unique().numel() * 3 * args.inner + args.experts) * args.hidden
    print(json.dumps({"us_per_step": round(us, 2), "cache_bytes": cache, "weight_bytes": int(weights),
                      "gb_per_s": round((cache + weights) / us / 1e3, 1), "status": int(layer.status.item())}))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())

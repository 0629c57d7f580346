"""The attention part of a decoding step, from this package's operators: 4-bit projections, the append to the
paged cache with its rotation, attention over the cache, and the 4-bit output projection.

    python -m l2domain_b200.decode --batch 8 --length 4096 [--hidden 4096 --heads 32 --kv-heads 8 --head-dim 128]

runs steps of that shape on synthetic weights and an already filled cache, as one captured graph, and prints the
mean time of a step with the bytes it cannot do without.
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
    :meth:`step` takes one new token per sequence; it allocates nothing and may be captured into a graph."""

    def __init__(self, w_qkv, w_out, heads: int, kv_heads: int, head_dim: int, batch: int, max_len: int, group: int = 128,
                 page_size: int = 16, theta: float = 10000.0, device: int = 0):
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
        shape = (batch * width, page_size, kv_heads, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=torch.bfloat16, device=dev) for _ in range(2))
        # Pages in the order sequences get them, one after the other; any other order does as well.
        self.table = torch.arange(batch * width, dtype=torch.int32, device=dev).view(width, batch).t().contiguous()
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        cache = L.KvCache(self.k, self.v, L.BF16, shape[0], page_size, kv_heads, head_dim, device=device)
        row = (heads + 2 * kv_heads) * head_dim
        self.cos, self.sin = L.rotation_tables(max_len, head_dim, theta, device=dev)
        self.append = L.KvAppend(cache, self.table, batch, width, heads_q=heads, cos=self.cos, sin=self.sin, max_pos=max_len,
                                 rot_dim=head_dim, k_token=row, v_token=row, q_token=row, q_out_token=row, status=self.status)
        self.attention = L.PagedAttention(cache, self.table, batch, width, heads, q_token=row, status=self.status)
        self.qkv = torch.zeros(batch, row, dtype=torch.bfloat16, device=dev)
        self.mixed = torch.zeros(batch, heads * head_dim, dtype=torch.bfloat16, device=dev)
        self.hidden = hidden

    def step(self, x, pos, lens, out, stream=None) -> None:
        """out[b] = W_out . attention of the token x[b] at position pos[b] over itself and the lens[b] - 1 before it
        (pos and lens int32 on the device; lens = pos + 1)."""
        n, hd = self.batch, self.heads * self.head_dim
        self.qkv_matrix.gemv(x, self.qkv, vectors=n, stream=stream)
        keys = self.qkv[:, hd:]
        values = self.qkv[:, hd + self.kv_heads * self.head_dim:]
        self.append.append(keys, values, pos, n, q=self.qkv, q_out=self.qkv, stream=stream)
        self.attention.decode(self.qkv, self.mixed, lens, n, stream=stream)
        self.out_matrix.gemv(self.mixed, out, vectors=n, stream=stream)


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--length", type=int, default=4096)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--head-dim", type=int, default=128)
    ap.add_argument("--steps", type=int, default=200)
    args = ap.parse_args()

    import torch

    torch.cuda.set_device(0)
    g = torch.Generator(device="cuda").manual_seed(0)
    row = (args.heads + 2 * args.kv_heads) * args.head_dim

    def normal(*shape, scale=1.0):
        return (torch.empty(shape, device="cuda").normal_(generator=g) * scale).to(torch.bfloat16)

    layer = DecodeAttention(normal(row, args.hidden, scale=0.02), normal(args.hidden, args.heads * args.head_dim, scale=0.02),
                            args.heads, args.kv_heads, args.head_dim, args.batch, args.length + args.steps + 16)
    layer.k.normal_(generator=g)
    layer.v.normal_(generator=g)
    x, out = normal(args.batch, args.hidden), torch.empty(args.batch, args.hidden, dtype=torch.bfloat16, device="cuda")
    pos = torch.full((args.batch,), args.length - 1, dtype=torch.int32, device="cuda")
    lens = pos + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())  # which fills the cache, x, pos and lens
    with torch.cuda.stream(side):
        layer.step(x, pos, lens, out, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(x, pos, lens, out, stream=torch.cuda.current_stream())
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
    cache = int(2 * args.batch * keys * args.kv_heads * args.head_dim * 2)
    weights = (row * args.hidden + args.hidden * args.heads * args.head_dim) * (0.5 + 2 / 128)
    print(json.dumps({"us_per_step": round(us, 2), "cache_bytes": cache, "weight_bytes": int(weights),
                      "gb_per_s": round((cache + weights) / us / 1e3, 1), "status": int(layer.status.item())}))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())

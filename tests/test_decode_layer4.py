"""The decoding layer over a cache in 4 bits with other scores, its experts, and the command that times them (GPU)."""
import json
import math

import pytest

torch = pytest.importorskip("torch")

import l2domain_b200 as L  # noqa: E402
from l2domain_b200 import decode  # noqa: E402


def test_a_cache_of_other_bits_is_refused():
    w = torch.zeros(64, 32)
    with pytest.raises(ValueError, match="16 or 4"):
        decode.DecodeAttention(w, w, 1, 1, 16, 1, 16, cache_bits=8)


def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def values(buffer, page, slot, heads, D, group):
    """What a cache in 4 bits holds at (page, slot), one of each per row, from its bytes: [rows][heads][D] in 64 bits."""
    chunks, groups = -(-D // 32), -(-D // group)
    tile = buffer.unflatten(1, (-1, heads, 256 * chunks + 64 * groups))[page, slot // 16]
    at = torch.arange(len(slot), device=buffer.device)
    byte = tile[:, :, : 256 * chunks].unflatten(2, (chunks, 16, 16))[at, :, :, slot % 16].flatten(2).long()
    word = tile[:, :, 256 * chunks:].contiguous().view(torch.int32).unflatten(2, (groups, 16))[at, :, :, slot % 16]
    j = torch.arange(D, device=buffer.device)
    n = (byte[:, :, j // 2] >> (4 * (j % 2))) & 15
    word = word[:, :, j // group]
    return (word // 16 * 16).view(torch.float32).double() * (n - word % 16).double()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,heads,kv_heads,head_dim,hidden,group", [(3, 4, 2, 64, 256, 32), (2, 8, 1, 128, 384, 128)])
def test_layer_follows_its_definition(batch, heads, kv_heads, head_dim, hidden, group):
    """A prompt and thirty steps, attention and experts: each stage against 64-bit arithmetic on the bf16 inputs and the
    cache that it was given, so that an error is one rounding to bf16 (2^-8 relative to the row's largest terms)."""
    gpu()
    g = torch.Generator(device="cuda").manual_seed(heads)
    row = (heads + 2 * kv_heads) * head_dim
    half, cap = head_dim // 2, 4.0

    def normal(*shape, scale=1.0):
        return (torch.empty(shape, device="cuda").normal_(generator=g) * scale).to(torch.bfloat16)

    slopes = L.distance_slopes(heads, device="cuda")
    layer = decode.DecodeAttention(normal(row, hidden, scale=hidden ** -0.5), normal(hidden, heads * head_dim, scale=0.1), heads, kv_heads, head_dim, batch, 64,
                                   cache_bits=4, cache_group=group, cap=cap, slopes=slopes)
    experts, inner, top = 6, 96, 2
    router, gate, up, down = (normal(experts, hidden, scale=hidden ** -0.5), normal(experts, inner, hidden, scale=hidden ** -0.5),
                              normal(experts, inner, hidden, scale=hidden ** -0.5), normal(experts, hidden, inner, scale=0.1))
    moe = decode.DecodeExperts(router, gate, up, down, top, batch)
    out, after = (torch.empty(batch, hidden, dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def near(got, want):
        assert (got.double() - want).abs().max() <= 2.0 ** -7 * want.abs().max()

    first = 12
    prompt = normal(batch * first, row)
    at = torch.arange(first, dtype=torch.int32, device="cuda").repeat(batch)
    of = torch.arange(batch, dtype=torch.int32, device="cuda").repeat_interleave(first)
    held = torch.zeros_like(prompt)
    layer.prompt(prompt.clone(), at, of, batch * first, k_out=held, v_out=held[:, kv_heads * head_dim:])
    torch.cuda.synchronize()
    page, slot = layer.table[of.long(), (at // 16).long()].long(), at.long() % 16
    k = values(layer.k, page, slot, kv_heads, head_dim, group)
    v = values(layer.v, page, slot, kv_heads, head_dim, group)
    assert torch.equal(held[:, : kv_heads * head_dim], k.flatten(1).to(torch.bfloat16))
    assert torch.equal(held[:, kv_heads * head_dim: 2 * kv_heads * head_dim], v.flatten(1).to(torch.bfloat16))
    keys, vals = [k.unflatten(0, (batch, first))], [v.unflatten(0, (batch, first))]
    freq = 10000.0 ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device="cuda") / head_dim)
    starts = torch.arange(batch, dtype=torch.int32, device="cuda") * 5
    for t in range(first, first + 30):
        x, pos = normal(batch, hidden), torch.full((batch,), t, dtype=torch.int32, device="cuda")
        layer.step(x, pos, pos + 1, out, starts=starts)
        moe.step(out, after)
        torch.cuda.synchronize()
        got = layer.qkv.view(batch, -1, head_dim).double()
        page, slot = layer.table[:, t // 16].long(), pos.long() % 16
        k, v = values(layer.k, page, slot, kv_heads, head_dim, group), values(layer.v, page, slot, kv_heads, head_dim, group)
        # Keys and values as the projection left them, to a step of their group: at most a 15th of twice its largest.
        a, b = got[:, heads: heads + kv_heads, :half], got[:, heads: heads + kv_heads, half:]
        turned = torch.cat([a * (t * freq).cos() - b * (t * freq).sin(), b * (t * freq).cos() + a * (t * freq).sin()], -1)
        assert ((k - turned).abs() <= 0.14 * turned.abs().amax(-1, keepdim=True)).all()
        assert ((v - got[:, heads + kv_heads:]).abs() <= 0.14 * got[:, heads + kv_heads:].abs().amax(-1, keepdim=True)).all()
        keys.append(k[:, None])
        vals.append(v[:, None])
        kk, vv = (torch.cat(z, 1).repeat_interleave(heads // kv_heads, 2) for z in (keys, vals))
        s = torch.einsum("bhd,bnhd->bhn", got[:, :heads], kk) / math.sqrt(head_dim)
        p = torch.arange(t + 1, device="cuda")
        s = cap * torch.tanh(s / cap) + slopes.double()[:, None] * (p - t).double()
        s = torch.where(p[None, None, :] >= starts[:, None, None], s, -math.inf)
        near(layer.mixed.view(batch, heads, head_dim), torch.einsum("bhn,bnhd->bhd", torch.softmax(s, -1), vv))
        o = out.double()
        logits = o @ router.double().t()
        ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :top]
        assert torch.equal(moe.ids.long(), ids)
        w = torch.softmax(logits.gather(1, ids), 1)
        h = torch.einsum("bh,bkfh->bkf", o, gate.double()[ids])
        h = h * torch.sigmoid(h) * torch.einsum("bh,bkfh->bkf", o, up.double()[ids])
        near(after, torch.einsum("bk,bkf,bkhf->bh", w, h, down.double()[ids]))
    assert layer.status.item() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("more,key_bytes", [(["--cache-bits", "4"], 36), (["--cap", "20", "--slopes"], 128),
                                            (["--cache-bits", "4", "--slopes", "--experts", "5", "--top", "2", "--inner", "64"], 36)])
def test_command(monkeypatch, capsys, more, key_bytes):
    gpu()
    monkeypatch.setattr("sys.argv", ["decode", "--batch", "2", "--length", "300", "--hidden", "256", "--heads", "4", "--kv-heads", "2",
                                     "--head-dim", "64", "--steps", "5", *more])
    assert decode.main() == 0
    got = json.loads(capsys.readouterr().out)
    assert got["status"] == 0 and got["cache_bytes"] == 2 * 2 * (300 + 10 + 2) * 2 * key_bytes
    plain = int((512 * 256 + 256 * 256) * (0.5 + 2 / 128))
    if "--experts" in more:  # at least two of the five, at most four, are chosen by two tokens
        assert any(got["weight_bytes"] == plain + 2 * (n * 3 * 64 + 5) * 256 for n in (2, 3, 4))
    else:
        assert got["weight_bytes"] == plain

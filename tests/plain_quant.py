"""Quantised serving in plain 64-bit torch: rows in 8 bits, groups in 4 bits and their layout, attention over any keys, a Llama with both.
Shares no code with the package."""
import math

import torch

import plain_llama as P


def rows8(x):
    """(codes, scales) of rows: scale = float32(max |x| / 127), codes x / scale to the nearest integer, ties to even."""
    x = x.double()
    s = (x.abs().amax(dim=-1) / 127).float().double()
    bad = ~torch.isfinite(x).all(dim=-1)
    safe = torch.where((s > 0) & ~bad, s, 1.0)
    c = torch.round(torch.where(bad[:, None], 0.0, x) / safe[:, None]).clamp(-127, 127)
    c = torch.where(((s > 0) & ~bad)[:, None], c, 0.0)
    return c, torch.where(bad, math.nan, s)


def fake8(x):
    c, s = rows8(x)
    return c * s[:, None]


def groups4(x):
    """(codes [..., hd], scales [..., hd / 32]): m the number of largest magnitude (positive on a tie), scale bfloat16(m / -8)."""
    g = x.double().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(g).all(dim=-1)
    g = torch.where(bad[..., None], 0.0, g)
    hi, lo = g.amax(-1), g.amin(-1)
    d = (torch.where(hi >= -lo, hi, lo).float() / -8).bfloat16().double()
    c = torch.round(g / torch.where(d != 0, d, 1.0)[..., None]).clamp(-8, 7)
    c = torch.where((d != 0)[..., None], c, 0.0)
    return c.flatten(-2), torch.where(bad, math.nan, d)


def fake4(x):
    c, d = groups4(x)
    return (c.unflatten(-1, (-1, 32)) * d[..., None]).flatten(-2)


def pack4(c):
    """Codes [..., hd] -> bytes [..., hd / 2], one dimension after the other."""
    hd = c.shape[-1]
    out = torch.zeros(c.shape[:-1] + (hd // 2,), dtype=torch.int32)
    n = (c + 8).int()
    for dim in range(hd):
        blk, half, word, i = dim // 64, dim % 64 // 32, dim % 32 // 4, dim % 4
        out[..., 32 * blk + 4 * word + 2 * half + i // 2] |= n[..., dim] << (4 * (i % 2))
    return out.to(torch.uint8)


def unpack4(b, d):
    """Bytes and scales -> numbers (float64)."""
    hd = 2 * b.shape[-1]
    out = torch.empty(b.shape[:-1] + (hd,), dtype=torch.float64)
    for dim in range(hd):
        blk, half, word, i = dim // 64, dim % 64 // 32, dim % 32 // 4, dim % 4
        n = (b[..., 32 * blk + 4 * word + 2 * half + i // 2].int() >> (4 * (i % 2))) & 15
        out[..., dim] = (n - 8) * d[..., dim // 32].double()
    return out


def attention(q, k, v, scale, window=None):
    """q [n, nh, hd] at the last n of the positions of k, v [L, nkv, hd]; float64. Returns the output, sum_j p_j |v_j|, and each
    row's largest sum_d |q_d k_d| * scale over the keys it sees (what error bounds are made of)."""
    q, k, v = q.double(), k.double(), v.double()
    n, nh, hd = q.shape
    L, nkv = k.shape[:2]
    pos = torch.arange(L - n, L)[:, None]
    key = torch.arange(L)[None]
    seen = key <= pos
    if window:
        seen &= key > pos - window
    out, mag, big = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(n, nh, dtype=torch.float64)
    for h in range(nh):
        kh, vh = k[:, h // (nh // nkv)], v[:, h // (nh // nkv)]
        p = torch.softmax((q[:, h] @ kh.T * scale).masked_fill(~seen, -math.inf), dim=-1)
        out[:, h], mag[:, h] = p @ vh, p @ vh.abs()
        big[:, h] = (q[:, h].abs() @ kh.abs().T * scale).masked_fill(~seen, 0.0).amax(dim=-1)
    return out, mag, big


def llama(cfg, w, ids, kv4=False, int8=False, cuts=None):
    """Logits of a Llama in float64 with products in 8 bits and / or keys and values in 4 bits."""
    w = {n: t.double() for n, t in w.items()}
    lin = (lambda x, m: fake8(x) @ fake8(m).T) if int8 else (lambda x, m: x @ m.T)
    hold = fake4 if kv4 else (lambda x: x)
    ids = torch.as_tensor(ids)
    T, H = ids.numel(), cfg["hidden_size"]
    nh, nkv, hd = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"]
    eps, wins = cfg["rms_norm_eps"], P.layer_windows(cfg)
    f = P.rope_inv_freq(hd, cfg["rope_theta"], cfg.get("rope_scaling")).double()
    ang = torch.arange(T).double()[:, None] * f.float().double()
    cos, sin = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    norm = lambda x, g: x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * g

    def turn(x):
        a, b = x[..., : hd // 2], x[..., hd // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    h = w["model.embed_tokens.weight"][ids]
    for l in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{l}."
        n = norm(h, w[p + "input_layernorm.weight"])
        q, k, v = (lin(n, w[p + f"self_attn.{c}_proj.weight"]) + w.get(p + f"self_attn.{c}_proj.bias", 0.0) for c in "qkv")
        a, _, _ = attention(turn(q.view(T, nh, hd)), hold(turn(k.view(T, nkv, hd))), hold(v.view(T, nkv, hd)), hd ** -0.5, wins[l])
        h = h + lin(a.reshape(T, nh * hd), w[p + "self_attn.o_proj.weight"])
        n = norm(h, w[p + "post_attention_layernorm.weight"])
        g = lin(n, w[p + "mlp.gate_proj.weight"])
        h = h + lin(g / (1 + torch.exp(-g)) * lin(n, w[p + "mlp.up_proj.weight"]), w[p + "mlp.down_proj.weight"])
    out = w["model.embed_tokens.weight"] if cfg.get("tie_word_embeddings") else w["lm_head.weight"]
    return norm(h, w["model.norm.weight"]) @ out.T

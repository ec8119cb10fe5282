"""Oracle: the attention operators with positions in space, in 64 bits (TEST INFRASTRUCTURE, see oracle/__init__.py).

Plain restatements of the formulas in include/scgg.h; differentiable, so autograd in 64 bits gives the gradients' formulas.
The reference has no counterpart of these operators: parity unpinned."""
from __future__ import annotations

import torch


def axial_rope(x, positions, sections, theta=10000.0, interleaved=False):
    """x [B,N,H,D] float64, positions [B,N,A] or [N,A] of any type."""
    half = x.shape[-1] // 2
    out_a, out_b = [], []
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    pair = 0
    for axis, count in enumerate(sections):
        for j in range(count):
            t = positions[..., axis].double() * theta ** (-j / count)
            c, s = torch.cos(t)[..., None], torch.sin(t)[..., None]
            out_a.append(a[..., pair] * c - b[..., pair] * s)
            out_b.append(a[..., pair] * s + b[..., pair] * c)
            pair += 1
    ra = torch.cat((torch.stack(out_a, -1), a[..., pair:]), -1) if pair else a
    rb = torch.cat((torch.stack(out_b, -1), b[..., pair:]), -1) if pair else b
    return torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)


def head_norm(x, weight, eps=1e-6):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight


def qk_norm_rope(x, weight, positions=None, sections=(), theta=10000.0, interleaved=False, eps=1e-6):
    return axial_rope(head_norm(x, weight, eps), positions, sections, theta, interleaved)


def visible(B, N, M, key_mask=None, causal=False, device="cpu"):
    """[B,N,M] bool: which keys a query sees."""
    see = torch.ones(B, N, M, dtype=torch.bool, device=device)
    if key_mask is not None:
        see &= key_mask.bool()[:, None, :]
    if causal:
        see &= torch.arange(M, device=device)[None] <= torch.arange(N, device=device)[:, None] + (M - N)
    return see


def softmax_maps(q, k, see, scale):
    """P1, P2 [B,H,N,M]; rows that see nothing are zero."""
    group = q.shape[2] // k.shape[2]
    k = k.unflatten(2, (-1, 2)).repeat_interleave(group, 2).flatten(2, 3)
    s = torch.einsum("bnhd,bmhd->bhnm", q, k) * scale
    s = s.masked_fill(~see[:, None], float("-inf"))
    some = see.any(-1)[:, None, :, None]
    p = torch.softmax(torch.where(some, s, torch.zeros_like(s)), -1)
    p = torch.where(some, p, torch.zeros_like(p))
    return p[:, 0::2], p[:, 1::2]


def diff_attention(q, k, v, lam, key_mask=None, causal=False, scale=None):
    """q [B,N,2H,d], k [B,M,2Hkv,d], v [B,M,Hkv,dv] float64, lam [H].  Hidden keys hold zeros here."""
    B, N, M = q.shape[0], q.shape[1], k.shape[1]
    see = visible(B, N, M, key_mask, causal, q.device)
    p1, p2 = softmax_maps(q, k, see, q.shape[-1] ** -0.5 if scale is None else scale)
    v = v.repeat_interleave(p1.shape[1] // v.shape[2], 2)
    return torch.einsum("bhnm,bmhe->bnhe", p1 - lam[None, :, None, None] * p2, v)


def sit_differential(sd, x, t, mask, n_blocks, n_heads, theta=100.0):
    """The node-coordinate transformer with differential attention (node_coordinate_diffusion.SiT(attention="differential")) on a
    plain state_dict, in the type of its tensors (float64 in the tests)."""
    import math
    import torch.nn.functional as F

    def lin(name, v):
        return F.linear(v, sd[name + ".weight"], sd[name + ".bias"])

    def ln(v):
        return F.layer_norm(v, (v.shape[-1],), eps=1e-6)
    h = lin("pos_embedder", x)
    B, N, dim = h.shape
    half = sd["t_embedder.mlp.0.weight"].shape[1] // 2
    arg = t.to(x)[:, None] * torch.exp(torch.arange(half).to(x) * (-math.log(10000.0) / half))
    c = lin("t_embedder.mlp.2", F.silu(lin("t_embedder.mlp.0", torch.cat([arg.cos(), arg.sin()], -1))))
    d, H = dim // n_heads, n_heads // 2
    axes, pairs = x.shape[-1], d // 2
    sections = [pairs // axes + (1 if a < pairs % axes else 0) for a in range(axes)]
    for i in range(n_blocks):
        p = f"blocks.{i}."
        a = p + "attn."
        sh1, sc1, g1, sh2, sc2, g2 = lin(p + "adaLN_modulation.1", F.silu(c)).chunk(6, 1)
        qkv = lin(a + "qkv", ln(h) * (1 + sc1[:, None]) + sh1[:, None])
        q, k = (qkv[..., j * dim:(j + 1) * dim].reshape(B, N, 2 * H, d) for j in (0, 1))
        v = qkv[..., 2 * dim:].reshape(B, N, H, 2 * d)
        q = qk_norm_rope(q, sd[a + "q_norm"], x.detach(), sections, theta)
        k = qk_norm_rope(k, sd[a + "k_norm"], x.detach(), sections, theta)
        start = 0.8 - 0.6 * math.exp(-0.3 * i)
        lam = (sd[a + "lambda_q1"] @ sd[a + "lambda_k1"]).exp() - (sd[a + "lambda_q2"] @ sd[a + "lambda_k2"]).exp() + start
        o = head_norm(diff_attention(q, k, v, lam.expand(H), key_mask=mask), sd[a + "out_norm"]) * (1 - start)
        h = h + g1[:, None] * lin(a + "proj", o.reshape(B, N, dim))
        u = ln(h) * (1 + sc2[:, None]) + sh2[:, None]
        h = h + g2[:, None] * lin(p + "mlp.fc2", F.gelu(lin(p + "mlp.fc1", u), approximate="tanh"))
    sh, sc = lin("final_layer.adaLN_modulation.1", F.silu(c)).chunk(2, 1)
    return lin("final_layer.linear", ln(h) * (1 + sc[:, None]) + sh[:, None]) * mask[..., None]

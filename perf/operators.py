"""The attention operators with positions in space: what is measured, and their plain forms.

Operators (``semantically_consistent_graph_generation_amd.attention``):

  axial_rope      rotary positions with several axes on the heads of q and k
  qk_norm_rope    RMS norm of every head of q and k, with the rotation in the same pass
  diff_attention  differential attention: the difference of two softmax maps with a learned weight, times V

A case's ``way`` is "fwd" (the outputs) or "train" (the outputs and all gradients, through autograd).  ``own`` selects the
framework's kernels; otherwise ``run`` computes the same in elementary torch operations in 32 bits (angles in 64).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ITEM = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-6


def _rope(name, op, way, dtype, B, N, Hq, Hk, D, sections, pos, theta, interleaved=False, fused=False):
    return {"name": name, "op": op, "way": way, "dtype": dtype, "B": B, "N": N, "Hq": Hq, "Hk": Hk, "D": D, "sections": sections,
            "pos": pos, "theta": theta, "interleaved": interleaved, "fused": fused}


def _diff(name, way, dtype, B, N, M, H, Hkv, d, dv, causal=False, mask="none", fused=False):
    return {"name": name, "op": "diff", "way": way, "dtype": dtype, "B": B, "N": N, "M": M, "H": H, "Hkv": Hkv, "d": d, "dv": dv,
            "causal": causal, "mask": mask, "fused": fused}


def listed():
    return [
        # one step of a coordinate chain: 64 small graphs, heads of the small coordinate transformer, 3 real-valued axes
        _rope("axial coords fp32", "axial", "fwd", "fp32", 64, 40, 6, 6, 32, "6,5,5", "coords", 100.0),
        # training on the voxels of a volume: integer (z, y, x), grouped keys, interleaved pairs
        _rope("axial voxels bf16 train", "axial", "train", "bf16", 2, 13824, 12, 4, 64, "8,12,12", "grid", 10000.0, interleaved=True),
        # an odd number of tokens and heads, a head that is rotated in part only, q and k as views of one projection
        _rope("axial odd fp16", "axial", "fwd", "fp16", 3, 4093, 5, 5, 48, "7,9", "grid", 10000.0, fused=True),
        # serving: one new token of each sequence at a far position
        _rope("norm one token bf16", "norm", "fwd", "bf16", 32, 1, 16, 4, 64, "32", "far", 10000.0, fused=True),
        # training step of the small coordinate transformer
        _rope("norm coords fp32 train", "norm", "train", "fp32", 64, 64, 6, 6, 32, "6,5,5", "coords", 100.0),
        # training on long sequences
        _rope("norm long bf16 train", "norm", "train", "bf16", 4, 16384, 16, 4, 128, "64", "far", 10000.0, fused=True),
        # one step of a coordinate chain: ragged graphs of up to 40 nodes, 6 heads of 32 as 3 pairs
        _diff("diff coords fp32", "fwd", "fp32", 64, 40, 40, 3, 3, 32, 64, mask="ragged"),
        # training on graphs of 256 nodes in 32 bits
        _diff("diff graphs fp32 train", "train", "fp32", 4, 256, 256, 4, 4, 32, 64, mask="ragged"),
        # training on long causal sequences with grouped keys
        _diff("diff causal bf16 train", "train", "bf16", 1, 4096, 4096, 8, 4, 64, 128, causal=True, fused=True),
        # a long prompt, padded sequences
        _diff("diff long bf16", "fwd", "bf16", 2, 8192, 8192, 8, 8, 64, 128, mask="ragged"),
        # odd lengths and a head width between the powers of two; more keys than queries
        _diff("diff odd fp16 train", "train", "fp16", 2, 777, 1311, 5, 5, 48, 96),
        # serving: one new token of each sequence against a long cache
        _diff("diff one token bf16", "fwd", "bf16", 16, 1, 32768, 16, 4, 64, 128, mask="ragged"),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    """Sizes spread over the logarithm of the listed ranges, odd ones among them."""
    while True:
        op = rng.choice(["axial", "norm", "diff", "diff"])
        way, dtype = rng.choice(["fwd", "train"]), rng.choice(["fp32", "bf16", "fp16"])
        if op == "diff":
            one = rng.random() < 0.3
            d, dv = rng.choice([(16, 32), (32, 32), (32, 64), (48, 96), (64, 64), (64, 128), (40, 80)])
            Hkv = rng.choice([1, 2, 3, 4, 8])
            H = Hkv * rng.choice([1, 1, 2, 4])
            if one:
                way, N, M, causal = "fwd", rng.choice([1, 1, 2, 5]), _logint(rng, 64, 65536), False
            else:
                N, causal = _logint(rng, 1, 8192), rng.random() < 0.4
                M = N if rng.random() < 0.6 else _logint(rng, 1, 8192)
                if way == "train":  # a softmax over one key has no gradient: nothing but rounding to compare
                    N, M = (max(N, 8), max(N, 8)) if N == M else (N, max(M, 8))
            c = _diff("", way, dtype, _logint(rng, 1, 64), N, M, H, Hkv, d, dv, causal, rng.choice(["none", "ragged"]), rng.random() < 0.5 and N == M)
        else:
            D = rng.choice([32, 48, 64, 80, 128, 36])
            half = D // 2
            axes = rng.choice([1, 2, 3])
            used = half if rng.random() < 0.7 else max(axes, half - rng.randrange(1, half // 2))
            cut = [used // axes] * axes
            cut[0] += used - sum(cut)
            Hk = rng.choice([1, 2, 3, 4, 6, 8])
            c = _rope("", op, way, dtype, _logint(rng, 1, 64), _logint(rng, 1, 16384), Hk * rng.choice([1, 1, 2, 4]), Hk, D,
                      ",".join(map(str, cut)), rng.choice(["coords", "grid", "far"]), rng.choice([100.0, 10000.0, 500000.0]),
                      rng.random() < 0.4, rng.random() < 0.5)
        del c["name"]
        like = [_cost(x) for x in listed() if (x["op"] == "diff") == (op == "diff") and x["way"] == way]
        if _cost(c) <= max(like) and _held(c) <= 2.2e9:
            return c


def _held(c):
    """Values that a plain form holds at once: its two maps, or its keys and values in 32 bits for every head."""
    return max(2 * c["H"] * c["N"], c["H"] * (2 * c["d"] + c["dv"])) * c["B"] * c["M"] if c["op"] == "diff" else 0


def _lengths(c):
    """Valid keys of each sequence: a function of the case alone, so that its work is known.  Some sequences are empty."""
    if c["mask"] == "none":
        return [c["M"]] * c["B"]
    r = np.random.RandomState(c["B"] * 31 + c["M"])
    got = r.randint(c["M"] // 2, c["M"] + 1, c["B"])
    if c["B"] > 3:
        got[1] = 0
    got[0] = c["M"]
    return [int(v) for v in got]


def _pairs(c):
    """(query, key) pairs that see each other, over the batch, for one head."""
    n = 0
    for m in _lengths(c):
        if not c["causal"]:
            n += c["N"] * m
        else:
            seen = np.clip(np.arange(c["N"]) + c["M"] - c["N"] + 1, 0, m)
            n += int(seen.sum())
    return n


def work(case):
    c, it = case, ITEM[case["dtype"]]
    if c["op"] == "diff":
        keys = sum(_lengths(c))
        q, k, v = c["B"] * c["N"] * c["H"] * 2 * c["d"], keys * c["Hkv"] * 2 * c["d"], keys * c["Hkv"] * c["dv"]
        o = c["B"] * c["N"] * c["H"] * c["dv"]
        pairs = _pairs(c) * c["H"]
        full = c["B"] * c["M"] * c["Hkv"] * (2 * c["d"] + c["dv"])
        if c["way"] == "fwd":
            return {"bytes": (q + k + v + o) * it, "flops": pairs * (4 * c["d"] + 2 * c["dv"])}
        return {"bytes": (2 * q + k + v + full + 2 * o) * it, "flops": pairs * (4 * c["d"] + 2 * c["dv"] + 12 * c["d"] + 4 * c["dv"])}
    x = c["B"] * c["N"] * (c["Hq"] + c["Hk"]) * c["D"]
    pos = c["B"] * c["N"] * len(c["sections"].split(",")) * (4 if c["pos"] == "coords" else 8)
    steps = {("axial", "fwd"): 3, ("axial", "train"): 6, ("norm", "fwd"): 7, ("norm", "train"): 20}[c["op"], c["way"]]
    # forward: x in, y out; backward: dy in, dx out, and x again where its norm is needed (it cannot be kept on the chip)
    moves = {("axial", "fwd"): 2, ("axial", "train"): 4, ("norm", "fwd"): 2, ("norm", "train"): 5}[c["op"], c["way"]]
    return {"bytes": moves * x * it + pos, "flops": steps * x}


def _views(g, dev, dtype, fused, B, N, parts, scale=1.0):
    """One tensor [B, N, heads, width] for each (heads, width): views of one projection's output where ``fused``."""
    if fused:
        wide = sum(h * w for h, w in parts)
        base = (torch.randn(B, N, wide, generator=g, device=dev, dtype=torch.float32) * scale).to(dtype)
        out, at = [], 0
        for h, w in parts:
            out.append(base[..., at:at + h * w].unflatten(-1, (h, w)))
            at += h * w
        return out
    return [(torch.randn(B, N, h, w, generator=g, device=dev, dtype=torch.float32) * scale).to(dtype) for h, w in parts]


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype, train = DTYPES[c["dtype"]], c["way"] == "train"
    s = {"case": c}
    if c["op"] == "diff":
        # scores of unit variance and a little more, as normalised heads give them
        qp, kp, vp = (2 * c["H"], c["d"]), (2 * c["Hkv"], c["d"]), (c["Hkv"], c["dv"])
        if c["fused"]:
            s["q"], s["k"], s["v"] = _views(g, dev, dtype, True, c["B"], c["N"], [qp, kp, vp], 1.1)
        else:
            s["q"], = _views(g, dev, dtype, False, c["B"], c["N"], [qp], 1.1)
            s["k"], s["v"] = _views(g, dev, dtype, False, c["B"], c["M"], [kp, vp], 1.1)
        s["lam"] = 0.2 + 0.6 * torch.rand(c["H"], generator=g, device=dev)
        s["mask"] = None
        if c["mask"] != "none":
            s["mask"] = torch.arange(c["M"], device=dev)[None] < torch.tensor(_lengths(c), device=dev)[:, None]
        if train:
            s["dout"] = torch.randn(c["B"], c["N"], c["H"], c["dv"], generator=g, device=dev).to(dtype)
            for n in ("q", "k", "v", "lam"):
                s[n] = s[n].detach().requires_grad_()
        return s
    s["q"], s["k"] = _views(g, dev, dtype, c["fused"], c["B"], c["N"], [(c["Hq"], c["D"]), (c["Hk"], c["D"])], 1.7)
    sections = tuple(int(v) for v in c["sections"].split(","))
    s["sections"] = sections
    A = len(sections)
    if c["pos"] == "coords":
        s["pos"] = torch.randn(c["B"], c["N"], A, generator=g, device=dev) * 8
    else:
        lo, hi = (0, 256) if c["pos"] == "grid" else (100_000, 1_000_000)
        s["pos"] = torch.randint(lo, hi, (c["B"], c["N"], A), generator=g, device=dev)
    if c["op"] == "norm":
        s["wq"], s["wk"] = (1 + 0.2 * torch.randn(c["D"], generator=g, device=dev) for _ in range(2))
    if train:
        s["dq"], s["dk"] = (torch.randn(s[n].shape, generator=g, device=dev).to(dtype) for n in ("q", "k"))
        for n in ("q", "k") + (("wq", "wk") if c["op"] == "norm" else ()):
            s[n] = s[n].detach().requires_grad_()
    return s


def _plain_rotate(x, pos, sections, theta, interleaved):
    """x [B,N,H,D] in 32 bits."""
    half = x.shape[-1] // 2
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    freq = torch.tensor([theta ** (-j / n) for n in sections for j in range(n)], dtype=torch.float64, device=x.device)
    angle = pos.double()[..., axis] * freq
    pad = half - len(axis)
    cos = torch.nn.functional.pad(angle.cos().float(), (0, pad), value=1.0)[:, :, None]
    sin = torch.nn.functional.pad(angle.sin().float(), (0, pad), value=0.0)[:, :, None]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)


def _plain_norm(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _plain_diff(q, k, v, lam, mask, causal):
    B, N, H2, d = q.shape
    M, H, g = k.shape[1], H2 // 2, H2 // k.shape[2]
    dtype = q.dtype
    q, k, v = q.float(), k.float(), v.float()
    if g > 1:
        k = k.unflatten(2, (-1, 2)).repeat_interleave(g, 2).flatten(2, 3)
        v = v.repeat_interleave(g, 2)
    s = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1).contiguous()) * d ** -0.5
    seen = None
    if mask is not None:
        seen = mask[:, None, None, :]
    if causal:
        low = torch.arange(M, device=q.device)[None] <= torch.arange(N, device=q.device)[:, None] + (M - N)
        seen = low if seen is None else seen & low
    if seen is not None:
        s = s.masked_fill(~seen, float("-inf"))
    top = s.detach().amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(s - top)
    p = p / p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    p = p.unflatten(1, (H, 2))
    a = p[:, :, 0] - lam[:, None, None] * p[:, :, 1]
    return torch.matmul(a, v.transpose(1, 2).contiguous()).transpose(1, 2).to(dtype)


def run(state):
    s, c = state, state["case"]
    train = c["way"] == "train"
    with torch.set_grad_enabled(train):
        if own:
            from semantically_consistent_graph_generation_amd import attention
            if c["op"] == "diff":
                out = attention.diff_attention(s["q"], s["k"], s["v"], s["lam"], key_mask=s["mask"], causal=c["causal"])
            elif c["op"] == "axial":
                out = attention.axial_rope(s["q"], s["k"], s["pos"], s["sections"], theta=c["theta"], interleaved=c["interleaved"])
            else:
                out = attention.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["sections"], theta=c["theta"],
                                             interleaved=c["interleaved"], eps=EPS)
        elif c["op"] == "diff":
            out = _plain_diff(s["q"], s["k"], s["v"], s["lam"], s["mask"], c["causal"])
        else:
            out = []
            for x, w in ((s["q"], s.get("wq")), (s["k"], s.get("wk"))):
                y = x.float()
                y = y if w is None else _plain_norm(y, w)
                out.append(_plain_rotate(y, s["pos"], s["sections"], c["theta"], c["interleaved"]).to(x.dtype))
            out = tuple(out)
        if not train:
            return out
        if c["op"] == "diff":
            return (out,) + torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["lam"]), s["dout"])
        leaves = (s["q"], s["k"]) + ((s["wq"], s["wk"]) if c["op"] == "norm" else ())
        return tuple(out) + torch.autograd.grad(out, leaves, (s["dq"], s["dk"]))


def _exact_spin(pos, sections, theta, width):
    """The rotation of every token as unit complex numbers [B,N,1,width/2]."""
    turn = torch.zeros(pos.shape[0], pos.shape[1], width // 2, dtype=torch.float64, device=pos.device)
    at = 0
    for a, n in enumerate(sections):
        f = torch.exp(torch.arange(n, dtype=torch.float64, device=pos.device) * (-math.log(theta) / n))
        turn[..., at:at + n] = pos[..., a:a + 1].double() * f
        at += n
    return torch.polar(torch.ones_like(turn), turn)[:, :, None]


def _complex(x, interleaved):
    x = x.double()
    return torch.view_as_complex((x.unflatten(-1, (-1, 2)) if interleaved else x.unflatten(-1, (2, -1)).transpose(-1, -2)).contiguous())


def _real(z, interleaved):
    z = torch.view_as_real(z)
    return (z if interleaved else z.transpose(-1, -2)).flatten(-2)


@torch.no_grad()
def _exact_rope(s, c):
    outs, grads, weights = [], [], []
    il = c["interleaved"]
    spin = _exact_spin(s["pos"], s["sections"], c["theta"], c["D"])
    for x, w, dy in ((s["q"], s.get("wq"), s.get("dq")), (s["k"], s.get("wk"), s.get("dk"))):
        x = x.detach().double()
        r = torch.ones_like(x[..., :1]) if w is None else 1 / torch.sqrt(x.square().sum(-1, keepdim=True) / c["D"] + EPS)
        w1 = torch.ones(c["D"], dtype=torch.float64, device=x.device) if w is None else w.detach().double()
        outs.append(_real(_complex(x * r * w1, il) * spin, il))
        if dy is not None:
            t = _real(_complex(dy, il) * spin.conj(), il)
            if w is None:
                grads.append(t)
            else:
                h = x * r
                weights.append((t * h).sum((0, 1, 2)))
                t = t * w1
                grads.append(r * (t - h * (t * h).sum(-1, keepdim=True) / c["D"]))
    return tuple(outs + grads + weights)


@torch.no_grad()
def _exact_diff(s, c):
    q, k, v, lam = (s[n].detach() for n in ("q", "k", "v", "lam"))
    B, N, M, H, d, group = c["B"], c["N"], c["M"], c["H"], c["d"], c["H"] // c["Hkv"]
    train = c["way"] == "train"
    full = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)  # noqa: E731
    out = torch.zeros(B, N, H, c["dv"], dtype=torch.float64, device=q.device)
    dq, dk, dv, dl = full(q), full(k), full(v), full(lam)
    lengths = _lengths(c)
    for b in range(B):
        m = lengths[b]
        if m == 0:
            continue
        hide = torch.ones(N, m, dtype=torch.bool, device=q.device).triu(M - N + 1) if c["causal"] else None
        for h in range(H):
            kv = h // group
            maps, V = [], v[b, :m, kv].double()
            for i in (0, 1):
                e = q[b, :, 2 * h + i].double() @ k[b, :m, 2 * kv + i].double().t() / math.sqrt(d)
                if hide is not None:
                    e[hide] = -math.inf
                    e[hide.all(1)] = 0
                e = torch.exp(e - e.logsumexp(1, keepdim=True))
                if hide is not None:
                    e[hide] = 0
                maps.append(e)
            l = lam[h].double()
            out[b, :, h] = (maps[0] - l * maps[1]) @ V
            if train:
                g = s["dout"][b, :, h].double()
                dv[b, :m, kv] += (maps[0] - l * maps[1]).t() @ g
                gp = g @ V.t()
                dl[h] -= (gp * maps[1]).sum()
                for i, w in ((0, 1.0), (1, -l)):
                    e = w * maps[i] * (gp - (maps[i] * gp).sum(1, keepdim=True)) / math.sqrt(d)
                    dq[b, :, 2 * h + i] = e @ k[b, :m, 2 * kv + i].double()
                    dk[b, :m, 2 * kv + i] += e.t() @ q[b, :, 2 * h + i].double()
    return (out, dq, dk, dv, dl) if train else out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_diff(s, case) if case["op"] == "diff" else _exact_rope(s, case)

"""Drop-in for ``src/bootstrap/node_coordinate_diffusion`` of the reference: the ``SiT`` denoiser
(sit_model.py:157-247; ``SiT_models['SiT-T']``) as a parameter container with the reference's ``state_dict`` names, and
``NodeCoordsDiffusionModel`` (cow_ / atm_diff_nodes_with_3d_checks.py:22-81) with ``.model``, ``.to_cuda_device`` and
``.sample(pos, node_mask)``, which ``NoiseModel.sample_limit_dist`` calls once per sampled batch (noise_model.py:323-325;
here: ``NoiseModel(cfg, node_coord_model=NodeCoordsDiffusionModel(...).sample)``-style hook, see noise_model.py).

The arithmetic runs in libscgg.so (``scgg_sit_forward`` / ``scgg_sit_sample``, csrc/sit.hip); there is no eager fallback.
The reference's checkpoints (``cow_best_coord_model.pth``) are not in its repository: weights are whatever the caller loads.
Parity: the network is checked against outputs of the reference's own module (fixtures h1_sit_*, made with a stand-in for
the two ``timm`` constructors it imports); the sampler loop against ``NodeCoordsDiffusionModel.sample`` run from the
reference's real module with its normal draws recorded (fixtures h2_sit_sample_*).

``SiT(..., attention="differential")`` is a variant of the same network that the reference does not have: its heads are pairs of
softmax maps, q and k are normalised per head and rotated by the nodes' coordinates (attention.py).  It is differentiable, so it
is the one to train from scratch; its weights do not go with the other's.  ``attention="softmax"``, the default, is the
reference's network and runs as before."""
from __future__ import annotations

import ctypes as C
import math
import warnings

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib, attention as attn_ops


class _Attention(nn.Module):          # timm.models.vision_transformer.Attention's parameters (qkv with bias, proj)
    def __init__(self, dim):
        super().__init__()
        self.qkv, self.proj = nn.Linear(dim, 3 * dim), nn.Linear(dim, dim)


class _DiffAttention(nn.Module):
    """H pairs of heads of d: q, k [2H, d] and v [H, 2d] from one projection; q, k normalised per head and rotated by the node's
    coordinates (the pairs of a head dealt to the axes); differential attention; the result normalised per head.  The weight of the
    second map is exp(lambda_q1 . lambda_k1) - exp(lambda_q2 . lambda_k2) + its start value, which grows with the layer's number."""

    def __init__(self, dim, num_heads, layer, axes, theta):
        super().__init__()
        self.pairs, self.d, self.theta = num_heads // 2, dim // num_heads, theta
        self.lambda_init = 0.8 - 0.6 * math.exp(-0.3 * layer)
        half = self.d // 2
        self.sections = tuple(half // axes + (1 if a < half % axes else 0) for a in range(axes))
        self.qkv, self.proj = nn.Linear(dim, 3 * dim), nn.Linear(dim, dim)
        self.q_norm, self.k_norm, self.out_norm = (nn.Parameter(torch.ones(n)) for n in (self.d, self.d, 2 * self.d))
        self.lambda_q1, self.lambda_k1, self.lambda_q2, self.lambda_k2 = (nn.Parameter(0.1 * torch.randn(self.d)) for _ in range(4))

    def forward(self, u, pos, mask):
        dim = u.shape[-1]
        q, k, v = (t.unflatten(-1, s) for t, s in zip(self.qkv(u).split(dim, -1), ((2 * self.pairs, self.d),) * 2 + ((self.pairs, 2 * self.d),)))
        q, k = attn_ops.qk_norm_rope(q, k, self.q_norm, self.k_norm, pos, self.sections, theta=self.theta)
        lam = torch.exp((self.lambda_q1 * self.lambda_k1).sum()) - torch.exp((self.lambda_q2 * self.lambda_k2).sum()) + self.lambda_init
        o = attn_ops.diff_attention(q, k, v, lam, key_mask=mask)
        o, _ = attn_ops.qk_norm_rope(o, None, self.out_norm, None)
        return self.proj((o * (1.0 - self.lambda_init)).flatten(2))


class _Mlp(nn.Module):
    def __init__(self, dim, hidden):
        super().__init__()
        self.fc1, self.fc2 = nn.Linear(dim, hidden), nn.Linear(hidden, dim)


class _Block(nn.Module):
    def __init__(self, dim, hidden, attn=None):
        super().__init__()
        self.attn, self.mlp = attn or _Attention(dim), _Mlp(dim, hidden)
        self.adaLN_modulation = nn.Sequential(nn.Identity(), nn.Linear(dim, 6 * dim))


class _TEmb(nn.Module):
    def __init__(self, dim, freq=256):
        super().__init__()
        self.mlp = nn.Sequential(nn.Linear(freq, dim), nn.Identity(), nn.Linear(dim, dim))


class _Final(nn.Module):
    def __init__(self, dim, out):
        super().__init__()
        self.linear = nn.Linear(dim, out)
        self.adaLN_modulation = nn.Sequential(nn.Identity(), nn.Linear(dim, 2 * dim))


class SiT(nn.Module):
    """SiT(in_channels, hidden_size, num_transformer_blocks, num_heads, mlp_ratio) -- sit_model.py:161-187.

    ``attention``: "softmax" (the reference's) or "differential" (see the module's docstring; ``num_heads`` even, heads of a
    multiple of 8 up to 64 wide; ``rope_theta``: base of the rotation by coordinates)."""

    def __init__(self, in_channels=3, hidden_size=192, num_transformer_blocks=6, num_heads=6, mlp_ratio=4.0, noise_steps=1000,
                 beta_start=1e-4, beta_end=0.02, attention="softmax", rope_theta=100.0):
        super().__init__()
        if attention not in ("softmax", "differential"):
            raise _lib.ScggError(f"SiT: attention is 'softmax' or 'differential', got {attention!r}")
        self.attention = attention
        differential = attention == "differential"
        if differential and (num_heads % 2 or hidden_size % num_heads or (hidden_size // num_heads) % 8 or hidden_size // num_heads > 64):
            raise _lib.ScggError(f"SiT: {num_heads} heads on {hidden_size} channels: differential attention takes an even number of heads "
                                 "of a multiple of 8 up to 64 channels")
        if differential and not 1 <= in_channels <= attn_ops.MAX_AXES:
            raise _lib.ScggError(f"SiT: {in_channels} coordinates: differential attention rotates by 1 to {attn_ops.MAX_AXES} axes")
        if differential and not 0.0 < rope_theta < float("inf"):
            raise _lib.ScggError(f"SiT: rope_theta has to be positive and finite, got {rope_theta}")
        self.in_channels, self.hidden_size, self.num_heads = in_channels, hidden_size, num_heads
        self.mlp_hidden = int(hidden_size * mlp_ratio)
        self.noise_steps, self.beta_start, self.beta_end = noise_steps, beta_start, beta_end
        self.pos_embedder = nn.Linear(in_channels, hidden_size)
        self.t_embedder = _TEmb(hidden_size)
        self.blocks = nn.ModuleList([
            _Block(hidden_size, self.mlp_hidden, _DiffAttention(hidden_size, num_heads, i, in_channels, rope_theta) if differential else None)
            for i in range(num_transformer_blocks)])
        self.final_layer = _Final(hidden_size, in_channels)
        self._engine, self._key, self._versions, self._ws = None, None, None, {}

    def _release(self):
        if self._engine is not None:
            _lib.lib().scgg_sit_destroy(self._engine)
            self._engine = None

    def __del__(self):
        try:
            self._release()
        except Exception:
            pass

    def _ensure_engine(self, device):
        L = _lib.lib()
        sd = dict(self.state_dict(keep_vars=True))
        key = (str(device), tuple((k, v.data_ptr()) for k, v in sd.items()))
        versions = tuple(v._version for v in sd.values())
        if self._engine is None or key != self._key:
            self._release()
            for k, v in sd.items():
                if v.device != device or v.dtype != torch.float32 or not v.is_contiguous():
                    raise _lib.ScggError(f"parameter {k} must be contiguous fp32 on {device}")
            cfg = _lib.SitConfig(self.in_channels, self.hidden_size, len(self.blocks), self.num_heads, self.mlp_hidden,
                                 self.noise_steps, self.beta_start, self.beta_end)
            h = L.scgg_sit_create(C.byref(cfg))
            if not h:
                raise _lib.ScggError("scgg_sit_create: " + L.scgg_last_error().decode())
            self._engine = C.c_void_p(h)
            for k, v in sd.items():
                _lib.check(L.scgg_sit_set_param(self._engine, k.encode(), _lib.ptr(v.detach()), v.numel()), k)
            _lib.check(L.scgg_sit_finalize(self._engine, _lib.stream_ptr()), "sit finalize")
            self._key, self._versions = key, versions
        elif versions != self._versions:
            _lib.check(L.scgg_sit_finalize(self._engine, _lib.stream_ptr()), "sit finalize")
            self._versions = versions
        return self._engine

    def _workspace(self, B, n, device):
        k = (B, n, str(device))
        if k not in self._ws:
            nbytes = _lib.lib().scgg_sit_workspace_bytes(self._engine, B, n)
            self._ws = {k: torch.empty(nbytes + 256, dtype=torch.uint8, device=device)}
        ws = self._ws[k]
        off = (-ws.data_ptr()) % 256
        return C.c_void_p(ws.data_ptr() + off), ws.numel() - 256

    def forward(self, x, t, padding_mask):
        """x [B,N,3], t [B] timesteps, padding_mask [B,N] bool -> predicted noise [B,N,3] (valid rows; 0 on padded ones).
        Differentiable in the parameters with differential attention, forward only with the reference's.  The gradient of x goes through its
        embedding only: the rotation takes the coordinates as given, so it is not the derivative of the output (a warning says so)."""
        if not x.is_cuda:
            raise _lib.ScggError("SiT.forward runs on the MI355X only; move the inputs to the GPU")
        if self.attention == "differential":
            return self._forward_differential(x, t, padding_mask)
        return self._forward_engine(x, t, padding_mask)

    def _forward_differential(self, x, t, padding_mask):
        if x.requires_grad and torch.is_grad_enabled():
            warnings.warn("SiT(attention='differential'): the gradient of x leaves out its part through the rotation by coordinates", stacklevel=3)
        mask = padding_mask.to(torch.bool)
        x = x.float().masked_fill(~mask[..., None], 0.0)          # whatever padded rows hold: 0 times a NaN would reach the weights' gradients
        dim = self.hidden_size
        half = self.t_embedder.mlp[0].in_features // 2
        arg = t.float()[:, None] * torch.exp(torch.arange(half, device=x.device, dtype=torch.float32) * (-math.log(10000.0) / half))
        mlp = self.t_embedder.mlp
        c = F.silu(mlp[2](F.silu(mlp[0](torch.cat((arg.cos(), arg.sin()), -1)))))
        pos, h = x.detach(), self.pos_embedder(x)

        def modulated(h, shift, scale):
            return F.layer_norm(h, (dim,), eps=1e-6) * (1 + scale[:, None]) + shift[:, None]
        for blk in self.blocks:
            sh1, sc1, g1, sh2, sc2, g2 = blk.adaLN_modulation[1](c).chunk(6, -1)
            h = h + g1[:, None] * blk.attn(modulated(h, sh1, sc1), pos, mask)
            h = h + g2[:, None] * blk.mlp.fc2(F.gelu(blk.mlp.fc1(modulated(h, sh2, sc2)), approximate="tanh"))
        sh, sc = self.final_layer.adaLN_modulation[1](c).chunk(2, -1)
        return self.final_layer.linear(modulated(h, sh, sc)) * mask[..., None]

    @torch.no_grad()
    def _sample_differential(self, x_T, node_mask, steps, noise, seed, graph_id_base):
        """The reference's ancestral chain (cow_diff_nodes_with_3d_checks.py:63-81), one denoiser call and one update per step; the
        draws are those of ``scgg_sit_sample``: Philox normals keyed by (seed, global graph id, node, step), or ``noise``."""
        beta = torch.linspace(self.beta_start, self.beta_end, self.noise_steps, dtype=torch.float32)
        alpha = 1.0 - beta
        alpha_hat = torch.cumprod(alpha, 0)
        mask = node_mask.to(torch.bool)
        x = x_T.detach().float().masked_fill(~mask[..., None], 0.0).contiguous()
        B, n = x.shape[:2]
        z = torch.empty_like(x)
        for k, i in enumerate(range(self.noise_steps - 1, 0, -1)):
            if 0 <= steps <= k:
                break
            eps = self._forward_differential(x, torch.full((B,), i, device=x.device), mask)
            al, ah, be = float(alpha[i]), float(alpha_hat[i]), float(beta[i])
            x = (x - (1.0 - al) / math.sqrt(1.0 - ah) * eps) / math.sqrt(al)
            if i > 1:
                if noise is None and z.numel():
                    _lib.check(attn_ops._call(x.device, _lib.lib().scgg_philox_normal_rows, _lib.ptr(z), B, n, seed, graph_id_base, i), "philox_normal_rows")
                x = x + math.sqrt(be) * (z if noise is None else noise[k].float())
        return x.masked_fill(~mask[..., None], 0.0)

    @torch.no_grad()
    def _forward_engine(self, x, t, padding_mask):
        B, n = x.shape[0], x.shape[1]
        eng = self._ensure_engine(x.device)
        ws, nb = self._workspace(B, n, x.device)
        x = x.detach().float().contiguous()
        t32 = t.to(torch.int32).contiguous()
        m = padding_mask.to(torch.bool).contiguous()
        out = torch.empty(B, n, 3, device=x.device)
        _lib.check(_lib.lib().scgg_sit_forward(eng, _lib.ptr(x), _lib.ptr(t32), _lib.ptr(m.view(torch.uint8)), B, n, _lib.ptr(out),
                                               ws, nb, _lib.stream_ptr()), "sit_forward")
        return out

    @torch.no_grad()
    def sample(self, x_T, node_mask, steps=-1, noise=None, seed=0, graph_id_base=0):
        if self.attention == "differential":
            return self._sample_differential(x_T, node_mask, steps, noise, seed, graph_id_base)
        B, n = x_T.shape[0], x_T.shape[1]
        eng = self._ensure_engine(x_T.device)
        ws, nb = self._workspace(B, n, x_T.device)
        x_T = x_T.detach().float().contiguous()
        m = node_mask.to(torch.bool).contiguous()
        out = torch.empty(B, n, 3, device=x_T.device)
        nz = None if noise is None else noise.detach().float().contiguous()
        _lib.check(_lib.lib().scgg_sit_sample(eng, _lib.ptr(x_T), _lib.ptr(m.view(torch.uint8)), B, n, steps, _lib.ptr(nz), seed,
                                              graph_id_base, _lib.ptr(out), ws, nb, _lib.stream_ptr()), "sit_sample")
        return out


SiT_models = {"SiT-T": lambda **kw: SiT(num_transformer_blocks=6, hidden_size=192, num_heads=6, **kw),
              "SiT-VT": lambda **kw: SiT(num_transformer_blocks=4, hidden_size=192, num_heads=4, **kw),
              "SiT-S": lambda **kw: SiT(num_transformer_blocks=12, hidden_size=384, num_heads=6, **kw)}


class NodeCoordsDiffusionModel:
    """cow_diff_nodes_with_3d_checks.py:22-81 (sampling side): ``.model`` (SiT-T), ``.to_cuda_device``, ``.sample``."""

    takes_rng = True     # sample() accepts (seed, graph_id_base): NoiseModel.sample_limit_dist hands its Philox key on

    def __init__(self, noise_steps=1000, beta_start=1e-4, beta_end=0.02, coordinate_size=3, device="cuda", attention="softmax"):
        self.model = SiT_models["SiT-T"](in_channels=coordinate_size, noise_steps=noise_steps, beta_start=beta_start,
                                         beta_end=beta_end, attention=attention).to(device)
        self.noise_steps, self.beta_start, self.beta_end, self.device = noise_steps, beta_start, beta_end, device

    def to_cuda_device(self, device):
        if not next(self.model.parameters()).is_cuda:
            self.model.to(device)

    def sample(self, pos, node_mask, seed=None, graph_id_base=0):
        """``pos``: standard-normal start coordinates [B,n,3].  The reference ignores the values it is handed and draws
        torch.randn of the same shape again (:66); here the given draw IS x_T (same distribution, and the caller's
        generator decides it).  The per-step normals come from Philox keyed by (``seed``, ``graph_id_base`` + b, node, i);
        ``NoiseModel.sample_limit_dist`` passes the chain's own key, so a graph's coordinates depend on its global id only,
        not on the shard.  Called bare (the reference's signature), the seed is drawn from torch's global generator, which
        the reference consumes here too: ``torch.manual_seed`` reproduces a run and two calls never share a stream."""
        if seed is None:
            seed = int(torch.randint(0, 2 ** 31 - 1, (1,)))
        return self.model.sample(pos, node_mask, seed=seed, graph_id_base=graph_id_base)

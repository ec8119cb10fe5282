"""Attention with positions in space, for transformers over nodes with coordinates: three operators, each with its backward.

  axial_rope      rotary positions with several axes (x, y, z coordinates or voxel indices) on the heads of q and k
  qk_norm_rope    RMS norm of every head of q and k, and the rotation, in one pass
  diff_attention  differential attention: the difference of two softmax maps with a learned weight, times V

They are the attention of ``node_coordinate_diffusion.SiT(attention="differential")``.  The reference has no counterpart: its
coordinate transformer embeds positions by addition and takes one softmax map per head
(src/bootstrap/node_coordinate_diffusion/sit_model.py:80-103, :157-247).

Tensors are fp32, bf16 or fp16, [B, tokens, heads, width], on the GPU, with any strides: views of one projection's output are
read where they lie (a last axis that is not dense, or rows off the 16-byte grid in ``diff_attention``, cost a copy).  Outputs
and gradients are contiguous and of the inputs' type; statistics, sums and angles are held in 32 bits or more and rounded once.
Calls enqueue on the current stream of the tensors' device, never synchronise, give equal bits for equal inputs, and can be
captured into a HIP graph.  A tensor that another stream filled needs that stream's work to be waited for first, as with any
torch operation.  There is no CPU path (``_lib.ScggError``); second derivatives and forward-mode derivatives are not built, and
``torch.jit.trace`` and ``make_fx`` are refused.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_POSITIONS = {torch.float32: 0, torch.float64: 1, torch.int32: 2, torch.int64: 3}
MAX_AXES, MAX_ROPE_WIDTH = 8, 256


# ------------------------------------------------------------------------------------------------- shared checks
def _fail(what, why):
    raise _lib.ScggError(f"{what}: {why}")


def _check_heads(what, name, t, like=None):
    if not isinstance(t, torch.Tensor):
        _fail(what, f"{name} has to be a tensor")
    if t.dim() != 4:
        _fail(what, f"{name} has to be [B, tokens, heads, width], got {tuple(t.shape)}")
    if max(t.shape) > 2 ** 31 - 1:                             # the C side's extents are 32 bits and would take what is left of it
        _fail(what, f"{name} {tuple(t.shape)}: too many entries along an axis")
    if like is None or like is t:
        if t.dtype not in _DTYPES:
            _fail(what, f"{name} is {t.dtype}: float32, bfloat16 and float16 are supported")
    elif t.dtype != like.dtype or t.device != like.device:
        _fail(what, f"{name} is {t.dtype} on {t.device}, q is {like.dtype} on {like.device}")


try:                                                          # the mode in which make_fx records; None outside of one (0.1 us, get_proxy_mode takes 0.9)
    _recording = functools.partial(torch._C._get_dispatch_mode, torch._C._TorchDispatchModeKey.PROXY)
except AttributeError:
    from torch.fx.experimental.proxy_tensor import get_proxy_mode as _recording


def _check_mode(what, *ts):
    """The launches are seen by reverse-mode autograd and by stream capture, and by nothing else that records torch's operations."""
    if torch.jit.is_tracing() or _recording() is not None:
        _fail(what, "it cannot be traced (the trace would hold the empty outputs and not the kernels)")
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        _fail(what, "forward-mode derivatives are not built")


def _check_device(what, t):
    if not t.is_cuda:
        _fail(what, "the tensors have to be on the GPU (there is no CPU path)")


def _strides(t):
    """Strides of the first three axes in elements; an axis of one entry is never stepped along."""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape[:3])]


def _dense_rows(t):
    return t if t.shape[3] <= 1 or t.stride(3) == 1 else t.contiguous()


def _aligned_rows(t):
    """Dense rows that start at multiples of 16 bytes, 64 of them (and two heads) within 2 GiB; a copy where they do not."""
    t = _dense_rows(t)
    size, (b, n, h) = t.element_size(), _strides(t)
    if (t.data_ptr() | b * size | n * size | h * size) % 16 == 0 and (63 * n + h + t.shape[3]) * size < 2 ** 31 - 32:
        return t
    return t.clone(memory_format=torch.contiguous_format)


# the stream's handle without a Stream object around it, where this torch has it: 2 us of a call's 15
_stream_handle = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _new(t):
    """A contiguous tensor like t, not filled."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _call(device, fn, *args):
    """``fn(*args, stream)`` with the tensors' device current, on its current stream."""
    stream = _stream_handle(device.index)
    if torch.cuda.current_device() == device.index:
        return fn(*args, stream)
    with torch.cuda.device(device):
        return fn(*args, stream)


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ------------------------------------------------------------------------------------------------- rotation and head norm
def _rope_args(heads, weights, pos, cfg):
    """The argument block without its inputs; ``heads``: (q, k or None) or tensors of the same shapes."""
    sections, theta, interleaved, eps = cfg
    a = _lib.RopeArgs()
    q = heads[0]
    a.B, a.N, a.D = q.shape[0], q.shape[1], q.shape[3]
    a.dtype, a.interleaved, a.theta, a.eps = _DTYPES[q.dtype], int(interleaved), theta, eps
    for i, t in enumerate(heads):
        a.heads[i] = 0 if t is None else t.shape[2]
    for i, w in enumerate(weights):
        if w is not None:
            a.weight[i] = w.data_ptr()
            a.weight_f32 = int(w.dtype == torch.float32)
    a.n_sections = len(sections)
    a.sections[:len(sections)] = sections
    if pos is not None:
        a.positions, a.pos_type = pos.data_ptr(), _POSITIONS[pos.dtype]
        a.pos_stride_b, a.pos_stride_n, a.pos_stride_a = [s if n > 1 else 0 for s, n in zip(pos.stride(), pos.shape)]
    return a


def _rope_set(a, what, i, t):
    getattr(a, what)[i] = t.data_ptr()
    b, n, h = _strides(t)
    getattr(a, what + "_stride_b")[i], getattr(a, what + "_stride_n")[i], getattr(a, what + "_stride_h")[i] = b, n, h


def _rope_forward(q, k, wq, wk, pos, cfg):
    a = _rope_args((q, k), (wq, wk), pos, cfg)
    out = []
    for i, t in enumerate((q, k)):
        if t is None:
            out.append(None)
            continue
        y = _new(t)
        _rope_set(a, "x", i, t)
        a.y[i] = y.data_ptr()
        out.append(y)
    _lib.check(_call(q.device, _lib.lib().scgg_rope_forward, C.byref(a)), "rope")
    return out[0], out[1]


class _Rope(torch.autograd.Function):
    """Saves the inputs where a norm needs them again and nothing but the positions where not; one kernel each way (two in
    the backward of a norm: the weights' gradients are summed over the workgroups by a second one)."""

    @staticmethod
    def forward(ctx, q, k, wq, wk, pos, cfg):
        ctx.cfg, ctx.has_k, ctx.norm = cfg, k is not None, wq is not None
        ctx.save_for_backward(*((q, k, wq, wk, pos) if ctx.norm else (None, None, None, None, pos)))
        return _rope_forward(q, k, wq, wk, pos, cfg)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk, pos = ctx.saved_tensors
        gs = [_dense_rows(gq), _dense_rows(gk) if ctx.has_k else None]
        a = _rope_args(gs, (wq, wk), pos, ctx.cfg)
        grads, dw, ws = [None, None], [None, None], None
        for i, g in enumerate(gs):
            if g is None:
                continue
            grads[i] = _new(g)
            _rope_set(a, "g", i, g)
            a.y[i] = grads[i].data_ptr()
            if ctx.norm:
                _rope_set(a, "x", i, (q, k)[i])
                dw[i] = torch.empty_like((wq, wk)[i])
                a.dweight[i] = dw[i].data_ptr()
        size = 0
        if ctx.norm:
            size = _lib.lib().scgg_rope_workspace_bytes(C.byref(a))
            ws = torch.empty(size, dtype=torch.uint8, device=gq.device)
        _lib.check(_call(gq.device, _lib.lib().scgg_rope_backward, C.byref(a), ws.data_ptr() if ws is not None else None, size),
                   "rope (backward)")
        return grads[0], grads[1], dw[0], dw[1], None, None


def _rope(what, q, k, wq, wk, positions, sections, theta, interleaved, eps):
    _check_heads(what, "q", q)
    B, N, _, D = q.shape
    if k is not None:
        _check_heads(what, "k", k, q)
        if k.shape[0] != B or k.shape[1] != N or k.shape[3] != D:
            _fail(what, f"k {tuple(k.shape)} does not go with q {tuple(q.shape)}: only the number of heads may differ")
    if D < 2 or D % 2 or D > MAX_ROPE_WIDTH:
        _fail(what, f"heads of width {D}: even widths up to {MAX_ROPE_WIDTH} are supported")
    sections = tuple(int(s) for s in sections)
    if len(sections) > MAX_AXES or any(s < 0 for s in sections) or sum(sections) > D // 2:
        _fail(what, f"sections {sections}: at most {MAX_AXES} axes, with {D // 2} pairs of a head of width {D} in all")
    theta, eps = float(theta), float(eps)
    if not 0.0 < theta < float("inf"):
        _fail(what, f"theta has to be positive and finite, got {theta}")
    if not 0.0 <= eps < float("inf"):
        _fail(what, f"eps has to be finite and at least 0, got {eps}")
    if not sections:
        positions = None
    else:
        if not isinstance(positions, torch.Tensor) or positions.dtype not in _POSITIONS:
            _fail(what, "positions have to be a tensor of float32, float64, int32 or int64")
        if positions.dim() == 2:
            positions = positions[None].expand(B, -1, -1)
        if tuple(positions.shape) != (B, N, len(sections)):
            _fail(what, f"positions {tuple(positions.shape)}: [{B}, {N}, {len(sections)}] or [{N}, {len(sections)}] is needed")
        if positions.device != q.device:
            _fail(what, f"positions are on {positions.device}, q is on {q.device}")
        if positions.requires_grad and torch.is_grad_enabled():
            _fail(what, "positions take no gradient: detach them")
    for name, w in (("q_weight", wq), ("k_weight", wk)):
        if w is None:
            continue
        if not isinstance(w, torch.Tensor) or tuple(w.shape) != (D,) or w.dtype not in (torch.float32, q.dtype) or w.device != q.device:
            _fail(what, f"{name} has to be [{D}], float32 or {q.dtype}, on {q.device}")
    if wq is not None and wk is not None and wq.dtype != wk.dtype:
        _fail(what, f"q_weight is {wq.dtype}, k_weight is {wk.dtype}: one type is needed")
    _check_mode(what, q, k, wq, wk, positions)
    _check_device(what, q)
    q, k = _dense_rows(q), None if k is None else _dense_rows(k)
    wq, wk = (None if w is None else w.contiguous() for w in (wq, wk))
    cfg = (sections, theta, bool(interleaved), eps)
    return (_Rope.apply if _wants_grad(q, k, wq, wk) else _rope_forward)(q, k, wq, wk, positions, cfg)


def axial_rope(q, k, positions, sections, theta=10000.0, interleaved=False):
    """Rotary positions with several axes.

    q [B,N,Hq,D] and k [B,N,Hk,D] (or None), D even and at most 256; positions [B,N,A] or [N,A] with A = len(sections) <= 8,
    real (coordinates) or whole (voxel or token indices), float32 / float64 / int32 / int64.  ``sections[a]`` pairs of a head
    turn with axis a, the j-th of them by the angle ``positions[.., a] * theta ** (-j / sections[a])``; pairs behind the last
    section are left as they are.  A pair is (x[2i], x[2i+1]) if ``interleaved``, else (x[i], x[i + D/2]).  Angles are formed
    in two terms of 64 bits, so positions as far as 64 bits hold them keep theirs.  Returns (q', k'), contiguous; differentiable in q and k."""
    sections = tuple(sections)
    if not sections:
        _fail("axial_rope", "sections name no axis")
    return _rope("axial_rope", q, k, None, None, positions, sections, theta, interleaved, 0.0)


def qk_norm_rope(q, k, q_weight, k_weight, positions=None, sections=(), theta=10000.0, interleaved=False, eps=1e-6):
    """RMS norm of every head, ``x / sqrt(mean(x^2) + eps) * weight``, and ``axial_rope`` of the result, in one pass.

    ``q_weight`` and ``k_weight`` [D] are shared by the heads, float32 or of q's type.  ``sections=()`` gives the norm alone;
    k = None (with ``k_weight`` None) leaves k out.  Returns (q', k'), contiguous; differentiable in q, k and the weights."""
    if q_weight is None or (k_weight is None) != (k is None):
        _fail("qk_norm_rope", "q and k each need their weight")
    return _rope("qk_norm_rope", q, k, q_weight, k_weight, positions, sections, theta, interleaved, eps)


# ------------------------------------------------------------------------------------------------- differential attention
def _diff_set(a, name, t):
    setattr(a, name, t.data_ptr())
    for axis, s in zip("bnh", _strides(t)):
        setattr(a, f"{name}_stride_{axis}", s)


def _diff_args(q, k, v, lam, mask, cfg):
    causal, scale = cfg
    a = _lib.DiffAttentionArgs()
    _diff_set(a, "q", q)
    _diff_set(a, "k", k)
    _diff_set(a, "v", v)
    setattr(a, "lambda", lam.data_ptr())
    if mask is not None:
        a.key_mask, a.mask_stride_b = mask.data_ptr(), mask.stride(0) if mask.shape[0] > 1 else 0
    a.scale, a.causal, a.dtype = scale, int(causal), _DTYPES[q.dtype]
    a.B, a.N, a.M, a.H, a.Hkv, a.d, a.dv = q.shape[0], q.shape[1], k.shape[1], q.shape[2] // 2, v.shape[2], q.shape[3], v.shape[3]
    return a


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _diff_forward(q, k, v, lam, mask, cfg, with_stats=False):
    L = _lib.lib()
    a = _diff_args(q, k, v, lam, mask, cfg)
    out = torch.empty(q.shape[0], q.shape[1], a.H, a.dv, dtype=q.dtype, device=q.device)
    a.out = out.data_ptr()
    stats = torch.empty(a.B, a.H, 2, a.N, 2, dtype=torch.float32, device=q.device) if with_stats else None
    a.stats = stats.data_ptr() if with_stats else None
    nbytes = L.scgg_diff_attention_forward_workspace_bytes(C.byref(a))
    ws = _workspace(nbytes, q.device)
    _lib.check(_call(q.device, L.scgg_diff_attention_forward, C.byref(a), ws.data_ptr() if nbytes else None, nbytes), "diff_attention")
    return (out, stats) if with_stats else out


class _DiffAttention(torch.autograd.Function):
    """Saves its inputs and the softmax statistics of both maps (16 bytes per query and head); the backward forms the maps again."""

    @staticmethod
    def forward(ctx, q, k, v, lam, mask, cfg):
        out, stats = _diff_forward(q, k, v, lam, mask, cfg, with_stats=True)
        ctx.cfg = cfg
        ctx.save_for_backward(q, k, v, lam, mask, stats)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, lam, mask, stats = ctx.saved_tensors
        L = _lib.lib()
        a = _diff_args(q, k, v, lam, mask, ctx.cfg)
        dout = _aligned_rows(dout)
        _diff_set(a, "dout", dout)
        dq, dk, dv = _new(q), _new(k), _new(v)
        dlam = torch.empty_like(lam)
        a.stats, a.dq, a.dk, a.dv_out, a.dlambda = stats.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dlam.data_ptr()
        nbytes = L.scgg_diff_attention_backward_workspace_bytes(C.byref(a))
        ws = _workspace(nbytes, q.device)
        _lib.check(_call(q.device, L.scgg_diff_attention_backward, C.byref(a), ws.data_ptr() if nbytes else None, nbytes),
                   "diff_attention (backward)")
        return dq, dk, dv, dlam, None, None


def diff_attention(q, k, v, lam, key_mask=None, causal=False, scale=None):
    """Differential attention: head h gives ``(softmax(scale q1 k1^T) - lam[h] softmax(scale q2 k2^T)) v``.

    q [B,N,2H,d]: heads 2h and 2h + 1 are q1 and q2 of head h; k [B,M,2Hkv,d] likewise; v [B,M,Hkv,dv]; H a multiple of Hkv
    (query heads h share the key head ``h // (H / Hkv)``).  d and dv: multiples of 8, d <= 64, dv <= 128.  ``lam``: [H] or a
    scalar, a float32 tensor (differentiable) or a number.  ``key_mask`` [B,M], bool or uint8: True keys are seen; what hidden
    keys and their values hold does not matter.  ``causal``: query i sees the keys j <= i + M - N (the last query sees all of
    them); a key that ``causal`` hides from some queries only has to be finite, as its value is multiplied by their zeros.  ``scale`` > 0,
    default d ** -0.5.  A query that sees no key gives zeros, and no gradient, whatever it and its upstream gradient hold.  float32
    entries are split into terms: an infinity that is seen gives NaN.  Returns [B,N,H,dv].

    One or a few queries against many keys (a new token against a cache) split the keys over the GPU.  With N = M short or long
    the maps are never stored."""
    what = "diff_attention"
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_heads(what, name, t, q)
    B, N, H2, d = q.shape
    M, K2, Hkv, dv = k.shape[1], k.shape[2], v.shape[2], v.shape[3]
    if k.shape[0] != B or k.shape[3] != d or v.shape[0] != B or v.shape[1] != M:
        _fail(what, f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not go together")
    if H2 < 2 or H2 % 2 or Hkv < 1 or K2 != 2 * Hkv or (H2 // 2) % Hkv:
        _fail(what, f"{H2} heads of q, {K2} of k, {Hkv} of v: 2 H, 2 Hkv and Hkv are needed, H a multiple of Hkv")
    H = H2 // 2
    if d < 8 or dv < 8 or d % 8 or dv % 8 or d > 64 or dv > 128:
        _fail(what, f"d = {d}, dv = {dv}: multiples of 8 with d <= 64 and dv <= 128 are supported")
    if not isinstance(lam, torch.Tensor):
        lam = torch.full((H,), float(lam), dtype=torch.float32, device=q.device)
    if lam.dtype != torch.float32 or lam.device != q.device or tuple(lam.shape) not in ((), (1,), (H,)):
        _fail(what, f"lam has to be float32, [{H}] or a scalar, on {q.device}")
    lam = lam.expand(H).contiguous()
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        _fail(what, f"scale has to be positive and finite, got {scale}")
    if key_mask is not None:
        if not isinstance(key_mask, torch.Tensor) or key_mask.dtype not in (torch.bool, torch.uint8):
            _fail(what, "key_mask has to be a tensor of bool or uint8")
        if tuple(key_mask.shape) != (B, M) or key_mask.device != q.device:
            _fail(what, f"key_mask {tuple(key_mask.shape)} on {key_mask.device}: [{B}, {M}] on {q.device} is needed")
        if M > 1 and key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
    _check_mode(what, q, k, v, lam)
    _check_device(what, q)
    q, k, v = _aligned_rows(q), _aligned_rows(k), _aligned_rows(v)
    cfg = (bool(causal), scale)
    return (_DiffAttention.apply if _wants_grad(q, k, v, lam) else _diff_forward)(q, k, v, lam, key_mask, cfg)

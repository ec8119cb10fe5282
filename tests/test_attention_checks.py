"""What the attention operators refuse, without a GPU: the Python checks come before any launch, and so do those of the C ABI."""
import ctypes as C

import pytest
import torch

from semantically_consistent_graph_generation_amd import _lib, attention as A

Z = torch.zeros


def refused(fn, *args, match, **kw):
    with pytest.raises(_lib.ScggError, match=match):
        fn(*args, **kw)


def test_rope_refuses():
    q, k, pos = Z(2, 5, 4, 32), Z(2, 5, 2, 32), Z(2, 5, 3)
    ok = (6, 5, 5)
    for bad, why in (((q[0], k, pos, ok), r"B, tokens"), ((q.double(), None, pos, ok), "float64"), ((q, k.bfloat16(), pos, ok), "bfloat16"),
                     ((q, k[:, :4], pos, ok), "go with"), ((q, Z(2, 5, 2, 16), pos, ok), "go with"), ((Z(2, 5, 4, 31), None, pos, ok), "width 31"),
                     ((Z(2, 5, 1, 258), None, pos, ok), "width 258"), ((q, k, pos, (6, 6, 5)), "16 pairs"), ((q, k, pos, (-1, 5, 5)), "sections"),
                     ((q, k, Z(2, 5, 9), (1,) * 9), "8 axes"), ((q, k, pos[..., :2], ok), "is needed"), ((q, k, pos[:1], ok), "is needed"),
                     ((q, k, pos.half(), ok), "positions"), ((q, k, None, ok), "positions"), ((q, k, pos, ()), "no axis"),
                     ((q, k, pos.clone().requires_grad_(), ok), "no gradient"), (([1], k, pos, ok), "tensor"), ((q, k, pos, ok), "GPU")):
        refused(A.axial_rope, *bad, match=why)
    for theta in (0.0, -1.0, float("inf"), float("nan")):
        refused(A.axial_rope, q, k, pos, ok, theta=theta, match="theta")


def test_norm_refuses():
    q, k, w = Z(2, 5, 4, 32), Z(2, 5, 2, 32), Z(32)
    refused(A.qk_norm_rope, q, k, None, w, match="weight")
    refused(A.qk_norm_rope, q, k, w, None, match="weight")
    refused(A.qk_norm_rope, q, None, w, w, match="weight")
    refused(A.qk_norm_rope, q, k, Z(16), w, match=r"\[32\]")
    refused(A.qk_norm_rope, q, k, w.double(), w, match=r"\[32\]")
    refused(A.qk_norm_rope, q, k, w.bfloat16(), w, match=r"\[32\]")
    refused(A.qk_norm_rope, q.bfloat16(), k.bfloat16(), w.bfloat16(), w, match="one type")
    refused(A.qk_norm_rope, q, k, w, w, eps=-1.0, match="eps")
    refused(A.qk_norm_rope, q, k, w, w, eps=float("nan"), match="eps")
    refused(A.qk_norm_rope, q, k, w, w, match="GPU")


def rope_args(**kw):
    a = _lib.RopeArgs()
    a.B, a.N, a.D, a.heads[0], a.theta, a.n_sections, a.positions, a.sections[0] = 2, 3, 32, 4, 100.0, 1, 4096, 16
    a.x[0] = a.y[0] = a.g[0] = 4096
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,why", [(dict(dtype=3), "dtype"), (dict(D=33), "width"), (dict(D=258), "width"), (dict(D=0), "shape"), (dict(B=-1), "shape"),
                                    (dict(n_sections=9), "axes"), (dict(theta=0.0), "theta"), (dict(theta=float("nan")), "theta"),
                                    (dict(positions=None), "positions"), (dict(pos_type=4), "position type"), (dict(D=30), "pairs"),
                                    (dict(B=1 << 20, N=1 << 12), "too many")])
def test_rope_c_entry_refuses(kw, why):
    L, a = _lib.lib(), rope_args(**kw)
    assert L.scgg_rope_forward(C.byref(a), None) != 0 and why in L.scgg_last_error().decode()
    assert L.scgg_rope_backward(C.byref(a), None, 0, None) != 0
    assert L.scgg_rope_workspace_bytes(C.byref(a)) == 0


def test_rope_c_entry_refuses_missing_pointers():
    L = _lib.lib()
    assert L.scgg_rope_forward(None, None) != 0
    for name in ("x", "y"):
        a = rope_args()
        getattr(a, name)[0] = None
        assert L.scgg_rope_forward(C.byref(a), None) != 0 and "null" in L.scgg_last_error().decode()
    a = rope_args()
    a.g[0] = None
    assert L.scgg_rope_backward(C.byref(a), None, 0, None) != 0
    a = rope_args()
    a.heads[1], a.x[1], a.y[1] = 2, 4096, 4096
    a.weight[0] = 4096
    assert L.scgg_rope_forward(C.byref(a), None) != 0 and "weights" in L.scgg_last_error().decode()
    a.weight[1] = 4096
    a.g[1] = 4096
    assert L.scgg_rope_backward(C.byref(a), None, 0, None) != 0 and "workspace" in L.scgg_last_error().decode()
    a.eps = -1.0
    assert L.scgg_rope_forward(C.byref(a), None) != 0 and "eps" in L.scgg_last_error().decode()

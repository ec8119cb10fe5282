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
    assert L.scgg_rope_backward(C.byref(a), 4100, 1 << 30, None) != 0 and "aligned" in L.scgg_last_error().decode()
    a.eps = -1.0
    assert L.scgg_rope_forward(C.byref(a), None) != 0 and "eps" in L.scgg_last_error().decode()


def test_diff_attention_refuses():
    f = A.diff_attention
    q, k, v, lam = Z(2, 5, 4, 32), Z(2, 7, 4, 32), Z(2, 7, 2, 64), Z(2)
    for bad, why in (((q[0], k, v, lam), r"B, tokens"), ((q.double(), k, v, lam), "float64"), ((q, k.half(), v, lam), "float16"),
                     ((q, k[:1], v, lam), "go together"), ((q, k, v[:, :6], lam), "go together"), ((q, Z(2, 7, 4, 16), v, lam), "go together"),
                     ((q[:, :, :3], k, v, lam), "3 heads"), ((q, k, v[:, :, :1], lam), "heads"), ((Z(2, 5, 6, 32), k, v, lam), "multiple"),
                     ((q[:, :, :0], k, v, lam), "0 heads"), ((Z(2, 5, 4, 72), Z(2, 7, 4, 72), v, lam), "d = 72"), ((q[..., :4], k[..., :4], v, lam), "d = 4"),
                     ((q, k, Z(2, 7, 2, 136), lam), "dv = 136"), ((q, k, v[..., :12], lam), "dv = 12"), ((q, k, v, lam.double()), "lam"),
                     ((q, k, v, Z(3)), "lam"), ((q, k, v, Z(1, 2)), "lam"), ((q, k, v, lam), "GPU")):
        refused(f, *bad, match=why)
    refused(f, q, k, v, lam, key_mask=Z(2, 7), match="bool")
    refused(f, q, k, v, lam, key_mask=Z(2, 6, dtype=torch.bool), match="is needed")
    refused(f, q, k, v, lam, key_mask=[True], match="bool")
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        refused(f, q, k, v, lam, scale=scale, match="scale")


def diff_args(**kw):
    a = _lib.DiffAttentionArgs()
    a.B, a.N, a.M, a.H, a.Hkv, a.d, a.dv, a.scale = 2, 3, 4, 2, 1, 32, 64, 0.1
    for n in ("q", "k", "v", "lambda", "out", "stats", "dout", "dq", "dk", "dv_out", "dlambda"):
        setattr(a, n, 4096)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,why", [(dict(dtype=-1), "dtype"), (dict(N=-1), "shape"), (dict(H=3, Hkv=2), "heads"), (dict(Hkv=0), "heads"), (dict(d=72), "d = 72"),
                                    (dict(d=12), "d = 12"), (dict(dv=0), "dv = 0"), (dict(dv=136), "dv = 136"), (dict(scale=0.0), "scale"),
                                    (dict(scale=float("nan")), "scale"), (dict(M=2 ** 31 - 1), "too many"), (dict(B=2 ** 20, H=2 ** 12), "too many")])
def test_diff_c_entry_refuses(kw, why):
    L, a = _lib.lib(), diff_args(**kw)
    assert L.scgg_diff_attention_forward(C.byref(a), None, 0, None) != 0 and why in L.scgg_last_error().decode()
    assert L.scgg_diff_attention_backward(C.byref(a), None, 0, None) != 0
    assert L.scgg_diff_attention_forward_workspace_bytes(C.byref(a)) == 0 and L.scgg_diff_attention_backward_workspace_bytes(C.byref(a)) == 0


def test_diff_c_entry_refuses_pointers_alignment_and_workspace():
    L = _lib.lib()
    assert L.scgg_diff_attention_forward(None, None, 0, None) != 0
    for n in ("q", "k", "v", "lambda", "out"):
        assert L.scgg_diff_attention_forward(C.byref(diff_args(**{n: None})), None, 0, None) != 0 and "null" in L.scgg_last_error().decode()
    for n in ("dout", "dq", "dk", "dv_out", "dlambda", "stats"):
        assert L.scgg_diff_attention_backward(C.byref(diff_args(**{n: None})), 4096, 1 << 30, None) != 0 and "null" in L.scgg_last_error().decode()
    for kw in (dict(q=4104), dict(k_stride_n=2), dict(v_stride_b=1)):
        assert L.scgg_diff_attention_forward(C.byref(diff_args(**kw)), None, 0, None) != 0 and "16 bytes" in L.scgg_last_error().decode()
    assert L.scgg_diff_attention_backward(C.byref(diff_args(dout_stride_h=2)), 4096, 1 << 30, None) != 0 and "dout" in L.scgg_last_error().decode()
    a = diff_args(N=1, M=100000)
    need = L.scgg_diff_attention_forward_workspace_bytes(C.byref(a))
    assert need > 0
    assert L.scgg_diff_attention_forward(C.byref(a), 4096, need - 1, None) != 0 and "workspace" in L.scgg_last_error().decode()
    assert L.scgg_diff_attention_forward(C.byref(a), 4096 + 128, need, None) != 0 and "aligned" in L.scgg_last_error().decode()
    far = diff_args(k_stride_n=2 ** 24)
    assert L.scgg_diff_attention_forward(C.byref(far), None, 0, None) != 0 and "2 GiB" in L.scgg_last_error().decode()
    far = diff_args(dout_stride_n=2 ** 24)
    assert L.scgg_diff_attention_backward(C.byref(far), 4096, 1 << 30, None) != 0 and "2 GiB" in L.scgg_last_error().decode()
    assert L.scgg_diff_attention_backward(C.byref(a), None, 0, None) != 0 and "workspace" in L.scgg_last_error().decode()


def test_sit_refuses_heads_that_do_not_pair():
    from semantically_consistent_graph_generation_amd.node_coordinate_diffusion import SiT
    for kw in (dict(num_heads=3), dict(num_heads=5), dict(hidden_size=768, num_heads=4), dict(hidden_size=72, num_heads=6), dict(attention="other")):
        with pytest.raises(_lib.ScggError, match="SiT"):
            SiT(**{"attention": "differential", **kw})


def test_default_dtype_is_not_used(monkeypatch):
    """A number for lam, and the statistics that the kernels write in 32 bits, whatever torch's default type is."""
    made = []
    for name in ("full", "empty"):
        def kept(*a, _of=getattr(torch, name), **kw):
            made.append(_of(*a, **kw))
            return made[-1]
        monkeypatch.setattr(A.torch, name, kept)
    monkeypatch.setattr(A, "_call", lambda *a: 0)
    monkeypatch.setattr(A, "_check_device", lambda *a: None)
    q, k, v = (torch.zeros(1, 3, h, 8, dtype=torch.bfloat16) for h in (2, 2, 1))
    torch.set_default_dtype(torch.bfloat16)
    try:
        A.diff_attention(q.requires_grad_(), k, v, 0.5)
    finally:
        torch.set_default_dtype(torch.float32)
    lam, out, stats = made[:3]
    assert lam.dtype == torch.float32 and out.dtype == torch.bfloat16
    assert stats.dtype == torch.float32 and stats.numel() == 2 * 3 * 2


def test_diff_c_entry_refuses_outputs_off_the_grid_and_scales_out_of_range():
    """The kernels store 8 or 16 bytes at once, and take scale log2(e) in 32 bits."""
    L = _lib.lib()
    for n in ("out", "stats"):
        assert L.scgg_diff_attention_forward(C.byref(diff_args(**{n: 4104})), None, 0, None) != 0 and "aligned" in L.scgg_last_error().decode()
    for n in ("dq", "dk", "dv_out", "stats"):
        assert L.scgg_diff_attention_backward(C.byref(diff_args(**{n: 4104})), 4096, 1 << 30, None) != 0 and "aligned" in L.scgg_last_error().decode()
    a = diff_args(scale=3e38)
    assert L.scgg_diff_attention_forward(C.byref(a), None, 0, None) != 0 and "scale" in L.scgg_last_error().decode()


def calls():
    """(operator of its tensors, the tensors) of every entry point."""
    q, k, v = Z(1, 3, 2, 8), Z(1, 3, 2, 8), Z(1, 3, 1, 8)
    return [(lambda q, k, pos: A.axial_rope(q, k, pos, (4,))[0], (q, k, Z(1, 3, 1))),
            (lambda q, k, wq, wk, pos: A.qk_norm_rope(q, k, wq, wk, pos, (4,))[0], (q, k, Z(8), Z(8), Z(1, 3, 1))),
            (lambda q, k, v, lam: A.diff_attention(q, k, v, lam), (q, k, v, Z(1)))]


@pytest.mark.parametrize("which", range(3))
def test_forward_mode_and_traces_are_refused(which, monkeypatch):
    """A tangent would be dropped, and a trace would return memory that nothing wrote: both go past the operators' autograd function."""
    from torch.autograd import forward_ad as fw
    monkeypatch.setattr(A, "_check_device", lambda *a: None)
    monkeypatch.setattr(A, "_call", lambda *a: 0)
    f, ts = calls()[which]
    f(*ts)
    for i in range(len(ts)):
        with fw.dual_level():
            f(*ts)                                                    # no tangents: an ordinary call
            with pytest.raises(_lib.ScggError, match="forward-mode"):
                f(*ts[:i], fw.make_dual(ts[i], torch.ones_like(ts[i])), *ts[i + 1:])
    with pytest.raises(_lib.ScggError, match="traced"):
        torch.jit.trace(f, ts)


def test_differential_sampler_draws_on_its_tensors_device(monkeypatch):
    """The draws run on the stream and with the device of the tensors, which need not be the current ones."""
    from semantically_consistent_graph_generation_amd import node_coordinate_diffusion as N
    model = N.SiT(attention="differential", num_transformer_blocks=1, noise_steps=4)
    seen = []

    class Lib:
        @staticmethod
        def scgg_philox_normal_rows(*a):
            raise AssertionError("not on the tensors' device")
    monkeypatch.setattr(N._lib, "lib", lambda: Lib)
    monkeypatch.setattr(N._lib, "ptr", lambda t: t)
    monkeypatch.setattr(N._lib, "stream_ptr", lambda: None)
    monkeypatch.setattr(A, "_call", lambda device, fn, *a: seen.append((device, fn, a)) or 0)
    monkeypatch.setattr(model, "_forward_differential", lambda x, t, m: torch.zeros_like(x))
    x = Z(2, 3, 3)
    model.sample(x, torch.ones(2, 3, dtype=torch.bool), seed=5, graph_id_base=7)
    assert [(d, f is Lib.scgg_philox_normal_rows, a[1:]) for d, f, a in seen] == [(x.device, True, (2, 3, 5, 7, i)) for i in (3, 2)]


def test_diff_attention_refuses_types_that_all_tensors_share():
    q, k, v = Z(2, 5, 4, 32), Z(2, 7, 4, 32), Z(2, 7, 2, 64)
    for t in (torch.float64, torch.int32, torch.float8_e4m3fn):
        refused(A.diff_attention, q.to(t), k.to(t), v.to(t), Z(2), match="are supported")


def test_sections_from_an_iterator():
    """Counted once: an iterator that the check used up would leave no axis, and no rotation."""
    q, pos = Z(2, 5, 4, 32), Z(2, 5, 3)
    refused(A.axial_rope, q, None, pos, iter((6, 6, 5)), match="16 pairs")
    refused(A.axial_rope, q, None, pos, (n for n in (6, 5, 5)), match="GPU")
    refused(A.axial_rope, q, None, pos[..., :2], map(int, "655"), match="is needed")


def test_extents_past_32_bits_are_refused(monkeypatch):
    """2^32 + 5 tokens would be taken as 5: the rest of the output would keep what its memory held."""
    monkeypatch.setattr(A, "_check_device", lambda *a: None)
    monkeypatch.setattr(A, "_call", lambda *a: pytest.fail("launched"))
    far = 2 ** 32 + 5
    q = Z(1, 1, 2, 8)
    refused(A.axial_rope, q.expand(1, far, 2, 8), None, Z(1, 1).expand(far, 1), (4,), match="too many")
    refused(A.axial_rope, q, Z(1, 1, 1, 8).expand(1, 1, far, 8), Z(1, 1), (4,), match="too many")
    refused(A.qk_norm_rope, q.expand(far, 1, 2, 8), None, Z(8), None, match="too many")
    refused(A.diff_attention, q, q.expand(1, far, 2, 8), Z(1, 1, 1, 8).expand(1, far, 1, 8), 0.5, match="too many")
    refused(A.diff_attention, q.expand(1, far, 2, 8), q, Z(1, 1, 1, 8), 0.5, match="too many")


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up")
def test_diff_c_entry_refuses_grids_past_the_launch_limit():
    """Workgroups of 256 threads, 2^32 threads and more: refused before anything is set up or launched."""
    L = _lib.lib()
    lots = dict(B=2 ** 24, N=1, H=1, Hkv=1, d=8, dv=8)
    for kw in (dict(lots, M=4), dict(lots, M=600), dict(lots, B=2 ** 19, N=32, M=600)):
        a = diff_args(**kw)
        need = L.scgg_diff_attention_forward_workspace_bytes(C.byref(a))
        assert L.scgg_diff_attention_forward(C.byref(a), 4096, need, None) != 0 and "one launch" in L.scgg_last_error().decode()
    a = diff_args(**lots, M=4)
    assert L.scgg_diff_attention_backward(C.byref(a), 4096, 1 << 62, None) != 0 and "one launch" in L.scgg_last_error().decode()


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16])
def test_sit_differential_runs_in_32_bits_whatever_the_default_type(dtype, monkeypatch):
    """Network and sampler around the operators (which are replaced by ones that keep shapes): the same bits under another default type."""
    from semantically_consistent_graph_generation_amd import node_coordinate_diffusion as N
    monkeypatch.setattr(A, "qk_norm_rope", lambda q, k, *a, **kw: (q, k))
    monkeypatch.setattr(A, "diff_attention", lambda q, k, v, lam, key_mask: v * lam)
    torch.manual_seed(5)
    model = N.SiT(attention="differential", num_transformer_blocks=2, noise_steps=4)
    x, noise, mask = torch.randn(2, 3, 3), torch.randn(3, 2, 3, 3), torch.ones(2, 3, dtype=torch.bool)

    def run():
        with torch.no_grad():
            return model._forward_differential(x, torch.tensor([3, 1]), mask), model.sample(x, mask, noise=noise)
    want = run()
    torch.set_default_dtype(dtype)
    try:
        got = run()
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(a.dtype == torch.float32 and torch.equal(a, b) for a, b in zip(want, got))


def test_sit_refuses_what_every_forward_would():
    from semantically_consistent_graph_generation_amd.node_coordinate_diffusion import SiT
    for kw in (dict(in_channels=9), dict(in_channels=0), dict(rope_theta=0.0), dict(rope_theta=float("nan"))):
        with pytest.raises(_lib.ScggError, match="SiT"):
            SiT(attention="differential", num_transformer_blocks=1, **kw)
    SiT(attention="differential", num_transformer_blocks=1, in_channels=8)
    SiT(attention="softmax", num_transformer_blocks=1, in_channels=9)


def test_sit_differential_says_that_the_gradient_of_x_is_partial(monkeypatch):
    import warnings
    from semantically_consistent_graph_generation_amd import node_coordinate_diffusion as N
    monkeypatch.setattr(A, "qk_norm_rope", lambda q, k, *a, **kw: (q, k))
    monkeypatch.setattr(A, "diff_attention", lambda q, k, v, lam, key_mask: v * lam)
    model = N.SiT(attention="differential", num_transformer_blocks=1)
    x, t, mask = torch.randn(2, 3, 3), torch.tensor([3, 1]), torch.ones(2, 3, dtype=torch.bool)
    with pytest.warns(UserWarning, match="rotation"):
        model._forward_differential(x.clone().requires_grad_(), t, mask)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        model._forward_differential(x, t, mask).sum().backward()
        with torch.no_grad():
            model._forward_differential(x.clone().requires_grad_(), t, mask)


@pytest.mark.parametrize("which", range(3))
def test_make_fx_is_refused(which, monkeypatch):
    """The graph would hold the allocation of the output and no kernel, as a trace would."""
    from torch.fx.experimental.proxy_tensor import make_fx
    monkeypatch.setattr(A, "_check_device", lambda *a: None)
    monkeypatch.setattr(A, "_call", lambda *a: 0)
    f, ts = calls()[which]
    with pytest.raises(_lib.ScggError, match="traced"):
        make_fx(f)(*ts)
    f(*ts)

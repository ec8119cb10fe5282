"""The attention operators where tighter bounds or rarer inputs apply than in test_gpu_diff_attention.py and test_gpu_axial_rope.py, whose
references and tolerances are used here."""
import pytest
import torch

from test_gpu_diff_attention import DT, check, make, mask_of, reference, run_all

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", [
    (8, 201, 190, 64, 32, 64, 128, "none", True), (8, 190, 201, 64, 32, 48, 96, "ragged", False), (8, 201, 190, 64, 64, 64, 64, "random", False),
    (8, 201, 190, 64, 32, 32, 32, "none", True), (16, 201, 190, 32, 16, 32, 64, "ragged", False), (1, 2100, 2100, 4, 2, 64, 128, "none", True),
    (1, 2100, 2100, 4, 4, 32, 64, "none", False), (1, 1000, 4300, 4, 4, 48, 96, "ragged", False), (1, 1100, 8000, 2, 2, 64, 64, "rare", False),
    (1, 2200, 2200, 4, 4, 64, 128, "none", False), (1, 2200, 2200, 4, 4, 64, 128, "none", True)], ids=str)
def test_large_problems_round_outputs_only(case, dtype):
    """A and dS go into their products in two terms at every size, not on small problems alone: h^2 in the place of h."""
    B, N, M, H, Hkv, d, dv, kind, causal = case
    assert B * H * N * M > 2 ** 24
    q, k, v, lam, dout, g = make(B, N, M, H, Hkv, d, dv, dtype, N + M + d + 1)
    mask = mask_of(kind, B, M, g)
    check(run_all(q, k, v, lam, dout, key_mask=mask, causal=causal), reference(q, k, v, lam, dout, mask, causal, terms=2))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,N,M", [(0, 1024, 1024), (2, 0, 1024), (0, 5, 9000), (2, 0, 9000), (2, 1024, 0)])
def test_empty_with_many_keys(B, N, M, causal):
    """No queries or no keys, at sizes where the plans split: an empty output and gradients of zeros."""
    from semantically_consistent_graph_generation_amd.attention import diff_attention
    leaves = [torch.zeros(B, n, h, 32, device="cuda", requires_grad=True) for n, h in ((N, 4), (M, 4), (M, 2))]
    leaves.append(torch.full((2,), 0.3, device="cuda", requires_grad=True))
    out = diff_attention(*leaves, causal=causal)
    assert out.shape == (B, N, 2, 32) and not out.any()
    for t, gt in zip(leaves, torch.autograd.grad(out, leaves, torch.ones_like(out))):
        assert gt.shape == t.shape and not gt.any()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("N,M", [(1, 600), (2, 5000), (40, 300), (1, 40)])
def test_one_key_leads(N, M, dtype):
    """One key 17.5 above all others, with a value of zero: the output is the others' share, 2.5e-8 (2^-25.3, less than half of fp16's smallest
    step) of each value, and it has the accuracy that the entries of A have at any size."""
    q, k, v, lam, dout, g = make(1, N, M, 1, 1, 32, 64, dtype, N + M, size=1.0)
    q[:] = q[:, :1]
    k *= 0.02
    lead = q[0, 0, 0].double()
    k[0, M // 3, 0] = (lead * (17.5 * 32 ** 0.5 / float(lead @ lead))).to(k.dtype)
    v.abs_().mul_(1000.0)
    v[0, M // 3] = 0
    lam.zero_()
    want = reference(q, k, v, lam, dout, None, False, terms=1 if dtype == "fp32" else 2)[:1]
    assert float(want[0][0].max()) < 1.0 and float((want[0][1] / want[0][0]).max()) < 0.02
    check(run_all(q, k, v, lam, dout)[:1], want)


def empty_rows(B, N, M, mask):
    """[B,N]: causal queries that see no key."""
    first = torch.where(mask.any(1), mask.int().argmax(1), torch.full((B,), M, device="cuda"))
    return torch.arange(N, device="cuda")[None] + (M - N) < first[:, None]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("case", [(2, 300, 300, 2, 1, 64, 128), (2, 500, 400, 2, 2, 32, 64), (3, 70, 64, 4, 2, 48, 96), (2, 90, 1300, 1, 1, 64, 64),
                                  (2, 700, 2200, 2, 1, 64, 128), (2, 9, 600, 2, 1, 32, 32), (8, 200, 200, 64, 32, 64, 128)], ids=str)
def test_rows_that_see_nothing_may_hold_anything(case, dtype):
    """Causal sequences padded on the left (and N > M): what q and dO hold in the rows that see no key reaches no output and no gradient."""
    B, N, M, H, Hkv, d, dv = case
    q, k, v, lam, dout, g = make(B, N, M, H, Hkv, d, dv, dtype, N + M + 5)
    start = torch.randint(M // 2, M, (B,), generator=g, device="cuda")
    start[0] = max(2 * M // 3, M - N + 40 if M > N + 40 else 0)
    mask = torch.arange(M, device="cuda")[None] >= start[:, None]
    empty = empty_rows(B, N, M, mask)
    assert empty.any() and not empty.all()
    clean = run_all(q, k, v, lam, dout, key_mask=mask, causal=True)
    q2, dout2 = q.clone(), dout.clone()
    for i, x in enumerate((float("nan"), float("inf"), float("-inf"), torch.finfo(DT[dtype]).max)):
        spot = empty & (torch.arange(N, device="cuda") % 4 == i)
        q2[spot], dout2[spot] = x, x
    for name, a, b in zip(("out", "dq", "dk", "dv", "dlam"), clean, run_all(q2, k, v, lam, dout2, key_mask=mask, causal=True)):
        assert torch.isfinite(a).all() and torch.equal(a, b), name
    assert not clean[0][empty].any() and not clean[1][empty].any()
    # a value that other rows see and that is not finite does not change what such a row gives
    v2 = v.clone()
    v2[:, -1] = float("nan")
    lam2 = torch.full_like(lam, float("inf"))
    for got in (run_all(q, k, v2, lam, dout, key_mask=mask, causal=True), run_all(q, k, v, lam2, dout, key_mask=mask, causal=True)):
        assert not got[0][empty].any() and not got[1][empty].any()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("N,M,causal", [(40, 130, False), (150, 300, True), (20, 2000, False)])
def test_large_gradients_and_a_late_maximum(N, M, causal, dtype):
    """dP of 2^74 and, behind a first tile of scores near 0, keys whose scores are 45 (2^65 in the exponents) and 50 (2^72) larger."""
    q, k, v, lam, dout, g = make(1, N, M, 1, 1, 32, 64, dtype, N + M + 1, size=1.0)
    q[:] = q[:, :1]
    k *= 0.02
    for at, score in ((70, 45.0), (75, 45.0), (128, 50.0)):
        for i in range(2):
            lead = q[0, 0, i].double()
            k[0, at, i] = (lead * (score * 32 ** 0.5 / float(lead @ lead))).to(k.dtype)
    v, dout = v * 2.0 ** 35, dout * 2.0 ** 35
    want = reference(q, k, v, lam, dout, None, causal, terms=1 if dtype == "fp32" else 2)
    assert float(want[1][0].abs().max()) > 2.0 ** 48
    check(run_all(q, k, v, lam, dout, causal=causal), want)


def test_rope_over_more_tiles_than_a_launch_has_workgroups():
    """2^30 + 77 tokens of one pair (2^24 + 2 tiles of 64 tokens), all at the same position."""
    from semantically_consistent_graph_generation_amd.attention import axial_rope
    N = 2 ** 30 + 77
    q = torch.empty(1, N, 1, 2, dtype=torch.bfloat16, device="cuda")
    q[..., 0], q[..., 1] = 1.0, 0.5
    pos = torch.tensor([[0.7]], device="cuda")
    want, _ = axial_rope(q[:, :64], None, pos.expand(64, 1), (1,))
    got, _ = axial_rope(q, None, pos.expand(N, 1), (1,))
    assert bool((got.view(torch.int32) == want.view(torch.int32)[0, 0, 0, 0]).all())


@pytest.mark.parametrize("kind", ["i64", "f64", "f32"])
def test_far_whole_positions_keep_their_angle(kind):
    """Pairs of an angular step of 1 (sections of one pair), where the angle is the position itself: cos and sin of positions up to 2^62, of timestamps, of
    2^53 - 1.  The angle comes off the position to 2^-25 (its rounding to 32 bits, below pi / 4) and 2^-35 (2^60 turns times the 2^-106 that two terms
    leave, times 2 pi, and the series' end), cos and sin are formed in a few steps of 2^-24: the 8 u of the rotation."""
    import math
    from semantically_consistent_graph_generation_amd.attention import axial_rope
    at = [3, 10 ** 9 + 7, 10 ** 12 + 1, 2 ** 40 + 1, 2 ** 50 + 3, 2 ** 53 - 1, 1_700_000_000_123_456_768, 2 ** 62, -(2 ** 62) - 2 ** 12, -7, 0]
    pos = torch.tensor(at, device="cuda")
    pos = pos if kind == "i64" else pos.to(torch.float64 if kind == "f64" else torch.float32)
    n = len(at)
    q = torch.ones(1, n, 1, 4, device="cuda")
    q[..., 2:] = 0
    got = axial_rope(q, None, torch.stack((pos, pos.flip(0)), -1), (1, 1))[0].double().cpu()
    for i in range(n):
        for pair, x in ((0, float(pos[i])), (1, float(pos[n - 1 - i]))):
            assert abs(float(got[0, i, 0, pair]) - math.cos(x)) < 8 * 2.0 ** -24 and abs(float(got[0, i, 0, 2 + pair]) - math.sin(x)) < 8 * 2.0 ** -24, (x, pair)


def test_positions_past_every_angle_stay_bounded():
    """Where not even two terms hold the angle (1e25 and beyond) the rotation is some rotation: no length changes."""
    from semantically_consistent_graph_generation_amd.attention import axial_rope
    pos = torch.tensor([1e25, -3e30, 3e38], device="cuda")[:, None]
    q = torch.randn(1, 3, 2, 32, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    got, _ = axial_rope(q, None, pos, (16,), theta=100.0)
    length = [(t.double()[..., :16] ** 2 + t.double()[..., 16:] ** 2).sqrt() for t in (got, q)]
    assert float((length[0] - length[1]).abs().max()) < 1e-5


def test_weight_gradients_add_up_without_loss():
    """24576 terms t h of either sign for each channel.  Independent roundings, each of at most u / sqrt(3) rms of its value: t two products, a sum, and
    two for cos and sin; h three for the sum of squares, one step (two of u, four times the variance) of rsqrt and a product; the term's product and the
    partial sums' rounding: 15 in all, so the rms of the error over the root of the terms' square sum is at most sqrt(15 / 3) u = 1.33e-7; 512
    numbers scatter by 3 %, bound 1.5e-7.  (Sums of 32 bits in a row would add as much again.)"""
    from oracle import attention as O
    from semantically_consistent_graph_generation_amd.attention import qk_norm_rope
    square, count = 0.0, 0
    for seed in range(8):
        g = torch.Generator(device="cuda").manual_seed(seed)
        q, k, dq, dk = (torch.randn(64, 64, 6, 32, generator=g, device="cuda") for _ in range(4))
        pos = torch.randn(64, 64, 3, generator=g, device="cuda") * 8
        ws = [(1 + 0.2 * torch.randn(32, generator=g, device="cuda")).requires_grad_() for _ in range(2)]
        outs = qk_norm_rope(q, k, *ws, pos, (6, 5, 5), theta=100.0)
        for x, do, got in zip((q, k), (dq, dk), torch.autograd.grad(outs, ws, (dq, dk))):
            h = O.head_norm(x.double(), torch.ones(32, device="cuda").double()).requires_grad_()
            t, = torch.autograd.grad(O.axial_rope(h, pos, (6, 5, 5), 100.0), h, do.double())
            terms = (t * h.detach()).flatten(0, 2)
            square += float((((got.double() - terms.sum(0)) ** 2) / (terms ** 2).sum(0)).sum())
            count += 32
    assert count == 512 and (square / count) ** 0.5 < 1.5e-7, (square / count) ** 0.5


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("N,causal", [(20, False), (64, True), (65, False)])
def test_many_short_sequences(N, causal, dtype):
    """More than 512 workgroups whose queries are 64 at most (two waves share a tile), and just more."""
    q, k, v, lam, dout, g = make(300, N, N, 2, 2, 32, 64, dtype, N + 9)
    mask = mask_of("ragged", 300, N, g)
    check(run_all(q, k, v, lam, dout, key_mask=mask, causal=causal),
          reference(q, k, v, lam, dout, mask, causal, terms=1 if dtype == "fp32" else 2))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("N,M", [(70, 90), (3, 700), (130, 1300)])
def test_a_sequence_without_keys_may_hold_anything(N, M, dtype):
    """Whole sequences that the mask leaves nothing of, without `causal`: NaN in all of their rows."""
    q, k, v, lam, dout, g = make(3, N, M, 2, 1, 32, 64, dtype, N + M + 3)
    mask = mask_of("random", 3, M, g)
    mask[1] = False
    clean = run_all(q, k, v, lam, dout, key_mask=mask)
    dirty = [t.clone() for t in (q, k, v, dout)]
    for t in dirty:
        t[1] = float("nan")
    for a, b in zip(clean, run_all(*dirty[:3], lam, dirty[3], key_mask=mask)):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    assert not any(t[1].any() for t in clean[:4])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_two_streams_and_graphs_of_the_split_path(dtype):
    """Few queries against many keys on two streams at once, and as two captured graphs replayed in turn with eager work between."""
    from semantically_consistent_graph_generation_amd.attention import diff_attention
    q, k, v, lam, dout, g = make(4, 2, 6000, 4, 2, 64, 128, dtype, 31)
    q2 = (q * 0.5).contiguous()
    want, want2 = diff_attention(q, k, v, lam, causal=True), diff_attention(q2, k, v, lam)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(streams[0]):
            got[0].append(diff_attention(q, k, v, lam, causal=True))
        with torch.cuda.stream(streams[1]):
            got[1].append(diff_attention(q2, k, v, lam))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, want) for x in got[0]) and all(torch.equal(x, want2) for x in got[1])
    graphs, held = [], []
    for x, causal in ((q, True), (q2, False)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(diff_attention(x, k, v, lam, causal=causal))
        graphs.append(graph)
    for _ in range(3):
        k.mul_(1.01)
        for graph in graphs:
            graph.replay()
        eager = diff_attention(q, k, v, lam, causal=True), diff_attention(q2, k, v, lam)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))

"""The attention operators where tighter bounds or rarer inputs apply than in test_gpu_diff_attention.py and test_gpu_axial_rope.py, whose
references and tolerances are used here."""
import pytest
import torch

from test_gpu_diff_attention import check, make, mask_of, reference, run_all

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

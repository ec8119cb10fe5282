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

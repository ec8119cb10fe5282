"""SiT(attention="differential"): the model that uses the attention operators, against oracle/attention.py:sit_differential in 64 bits.
Tolerance 1e-4 of the scale (max |a - b| / max |b|), as for the other engines of the repository: fp32 products of 192 to 768 terms and
the operators' own bounds stay two orders below it."""
import pytest
import torch

from oracle import attention as O
from oracle import fixtures as fx
from oracle import sit as S

pytestmark = pytest.mark.gpu
REL = 1e-4


def build(name="SiT-T", seed=701, **kw):
    from semantically_consistent_graph_generation_amd.node_coordinate_diffusion import SiT_models
    model = SiT_models[name](in_channels=3, attention="differential", **kw)
    sd = fx.make_state_dict({k: tuple(v.shape) for k, v in model.state_dict().items()}, seed=seed)
    model.load_state_dict(sd)
    return model.cuda()


def rel(a, b):
    return float((a.detach().double().cpu() - b.detach().double().cpu()).abs().max() / b.detach().abs().max().clamp(min=1e-30))


def wide(model):
    return {k: v.detach().double().requires_grad_() for k, v in model.state_dict().items()}


@pytest.mark.parametrize("name,heads,n_nodes", [("SiT-T", 6, [40, 17, 1]), ("SiT-VT", 4, [33, 70]), ("SiT-S", 6, [9, 5, 12, 1])])
def test_forward_and_gradients(name, heads, n_nodes):
    model = build(name)
    m = fx.ragged_mask(n_nodes).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(*m.shape, 3, generator=g, device="cuda", requires_grad=True)
    t = torch.tensor([999, 500, 3, 1][: len(n_nodes)], device="cuda")
    out = model(x, t, m)
    sd = wide(model)
    x64 = x.detach().double().requires_grad_()
    want = O.sit_differential(sd, x64, t, m, len(model.blocks), heads)
    assert rel(out, want) < REL and not out[~m].any()
    do = torch.randn(out.shape, generator=g, device="cuda")
    params = dict(model.named_parameters())
    names = list(params)
    grads = torch.autograd.grad(out, [x] + [params[k] for k in names], do)
    wants = torch.autograd.grad(want, [x64] + [sd[k] for k in names], do.double())
    for k, a, b in zip(["x"] + names, grads, wants):
        assert rel(a, b) < 10 * REL, k                       # sums over all nodes of 12 sub-layers' rounding


def test_sampler():
    """Three steps with given draws and a whole short chain against the loop in 64 bits; Philox draws are the engine's."""
    model = build(noise_steps=6)
    m = fx.ragged_mask([9, 5, 12, 1]).cuda()
    g = torch.Generator(device="cuda").manual_seed(2)
    xT, noise = torch.randn(*m.shape, 3, generator=g, device="cuda"), torch.randn(5, *m.shape, 3, generator=g, device="cuda")
    sd = {k: v.detach() for k, v in wide(model).items()}
    beta, alpha, alpha_hat = S.schedule(6)
    for steps in (3, -1):
        out = model.sample(xT, m, steps=steps, noise=noise)
        x = xT.double()
        for k, i in enumerate([5, 4, 3, 2, 1][: steps if steps > 0 else 5]):
            eps = O.sit_differential(sd, x, torch.full((4,), i, device="cuda"), m, 6, 6)
            x = (x - float((1 - alpha[i]) / torch.sqrt(1 - alpha_hat[i])) * eps) / float(torch.sqrt(alpha[i]))
            x = x + (float(torch.sqrt(beta[i])) * noise[k].double() if i > 1 else 0)
        assert rel(out, x * m[..., None]) < REL
    a, b = model.sample(xT, m, seed=11), model.sample(xT, m, seed=11)
    one = model.sample(xT[2:3], m[2:3], seed=11, graph_id_base=2)
    assert torch.equal(a, b) and rel(one[0], a[2]) < 1e-5
    assert not torch.equal(a, model.sample(xT, m, seed=12)) and not a[~m].any()


def test_coordinate_model_and_default():
    """NodeCoordsDiffusionModel takes the variant; the default network has the reference's parameters and nothing else."""
    from semantically_consistent_graph_generation_amd.node_coordinate_diffusion import NodeCoordsDiffusionModel, SiT
    cm = NodeCoordsDiffusionModel(noise_steps=4, attention="differential")
    m = fx.ragged_mask([7, 3]).cuda()
    out = cm.sample(torch.randn(2, 7, 3, device="cuda"), m, seed=1)
    assert out.shape == (2, 7, 3) and torch.isfinite(out).all()
    assert not any("norm" in k or "lambda" in k for k in SiT().state_dict())


def test_padded_rows_may_hold_anything():
    """Output, sampler and gradients with NaN and infinities in the padded rows are those with zeros there, bit for bit, and 0 on them."""
    model = build()
    m = fx.ragged_mask([12, 5, 1]).cuda()
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(*m.shape, 3, generator=g, device="cuda").masked_fill(~m[..., None], 0.0)
    t = torch.tensor([999, 500, 3], device="cuda")
    do = torch.randn(x.shape, generator=g, device="cuda")
    params = list(model.parameters())

    def run(x):
        x = x.clone().requires_grad_()
        out = model(x, t, m)
        return (out.detach(),) + torch.autograd.grad(out, [x] + params, do)
    dirty = torch.where(m[..., None], x, torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda"))
    clean, got = run(x), run(dirty)
    assert all(torch.equal(a, b) for a, b in zip(clean, got)) and torch.isfinite(got[0]).all() and not got[0][~m].any() and not got[1][~m].any()
    chain = [model._sample_differential(y, m, 3, None, 7, 0) for y in (x, dirty)]
    assert torch.equal(*chain) and not chain[1][~m].any()


@pytest.mark.parametrize("attention", ["differential", "softmax"])
def test_draws_are_keyed_by_seed_graph_node_and_step(attention):
    """A seeded chain is the chain with the normals of scgg_philox_normal_rows for (seed, first graph's number, step i) handed in: the same bits
    with differential attention; the engine forms them inside its kernels, within REL."""
    from semantically_consistent_graph_generation_amd import _lib
    from semantically_consistent_graph_generation_amd.node_coordinate_diffusion import SiT_models
    model = SiT_models["SiT-T"](in_channels=3, attention=attention, noise_steps=6)
    model.load_state_dict(fx.make_state_dict({k: tuple(v.shape) for k, v in model.state_dict().items()}, seed=702))
    model = model.cuda()
    m = fx.ragged_mask([9, 5, 12, 1]).cuda()
    xT = torch.randn(*m.shape, 3, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    noise = torch.zeros(5, *m.shape, 3, device="cuda")
    for k, i in enumerate([5, 4, 3, 2, 1]):
        _lib.check(_lib.lib().scgg_philox_normal_rows(_lib.ptr(noise[k]), 4, m.shape[1], 21, 3, i, _lib.stream_ptr()), "philox_normal_rows")
    seeded, given = model.sample(xT, m, seed=21, graph_id_base=3), model.sample(xT, m, noise=noise)
    assert torch.equal(seeded, given) if attention == "differential" else rel(seeded, given) < REL
    assert rel(model.sample(xT, m, seed=21, graph_id_base=4), given) > 100 * REL

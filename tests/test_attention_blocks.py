"""The attention potential with normed features and gated feed-forward blocks: the operators together, as a model runs them, in MD and
in training, against the float64 oracle. Tolerances are those of the plain model's tests (a norm and a product more per layer), the
forces' of the largest force, which is below 1 here."""
import pytest
import torch

from oracle import blocks
from oracle import models as om
from fastmd_amd import systems
from fastmd_amd.config import InferenceConfig
from test_attention_model import _builder, _edges, _fn, _model

CONFIGS = [{"feed_forward": "gated", "norm_groups": 4}, {"feed_forward": "gated", "hidden": 344, "norm_groups": 1, "channels": 128},
           {"feed_forward": "gated", "hidden": 100, "channels": 48, "head_dim": 24, "heads": 2, "kv_heads": 1}, {"norm_groups": 8}]


def test_configs():
    m, params, _ = _model()
    assert "layers.0.W_1" in params and params["layers.0.W_1"].shape == (128, 64) and not any("norm_" in k for k in params)
    m, params, _ = _model(feed_forward="gated", hidden=100, norm_groups=2)
    assert params["layers.1.W_gate"].shape == (100, 64) and params["layers.1.W_down"].shape == (64, 100)
    assert params["layers.0.attention_norm_weight"].shape == (64,)
    with pytest.raises(ValueError, match="feed_forward"):
        _model(feed_forward="none")
    with pytest.raises(ValueError, match="norm_groups"):
        _model(norm_groups=5)


def test_oracle_forces():
    s = systems.perovskite(2)
    edges = _edges(s)
    _, params, cfg = _model(**CONFIGS[0])
    fn, pos = _fn(params, cfg, s, edges), edges[3]
    _, f, _ = om.energy_and_forces(fn, pos)
    d = torch.zeros_like(pos)
    d[7, 1] = 1e-5
    fd = -(fn(pos + d).sum() - fn(pos - d).sum()) / 2e-5
    assert float(f.abs().max()) > 0.0 and abs(float(fd - f[7, 1])) < 1e-6 * float(f.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("config", CONFIGS)
@pytest.mark.parametrize("n_cells", [3, 6])
def test_forces(device, n_cells, config):
    from fastmd_amd.engine.energy_derivative import EnergyDerivative
    from fastmd_amd.models.attention_like import AttentionAdapter

    s = systems.perovskite(n_cells, sigma=0.2)
    m, params, cfg = _model(**config)
    adapter = AttentionAdapter(m, device=device)
    builder = _builder(s, device)
    builder.build(torch.tensor(s.positions, device=device))
    out = EnergyDerivative(adapter)(builder.batch, adapter.prepare(builder.batch), n_real=s.n_atoms)
    torch.cuda.synchronize()
    edges = _edges(s)
    e, f, _ = om.energy_and_forces(_fn(params, cfg, s, edges), edges[3])
    assert abs(float(out["e"].item()) - float(e)) / s.n_atoms < 1e-5
    assert float((out["f"][0].cpu().double() - f).abs().max()) < 1e-4 * float(f.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("config", CONFIGS[:3])
def test_training_gradients(device, config):
    from fastmd_amd.models.attention_like import AttentionAdapter

    s = systems.perovskite(3, sigma=0.2)
    m, params, cfg = _model(**config)
    adapter = AttentionAdapter(m, device=device)
    adapter.module.requires_grad_(True)
    builder = _builder(s, device)
    builder.build(torch.tensor(s.positions, device=device))
    energies = adapter.node_energy(adapter.prepare(builder.batch), builder.batch.positions, builder.batch.cell)
    (energies[:s.n_atoms] ** 2).mean().backward()
    leaves = {k: v.double().requires_grad_(True) for k, v in params.items()}
    edges = _edges(s)
    (_fn(leaves, cfg, s, edges)(edges[3]) ** 2).mean().backward()
    for name, p in adapter.module.named_parameters():
        ref = leaves[name].grad
        err = float((p.grad.cpu().double() - ref).abs().max())
        assert err < 1e-4 * max(1e-3, float(ref.abs().max())), (name, err)


@pytest.mark.gpu
def test_md_eager_and_captured_agree(device):
    from fastmd_amd.execution.gpu_nhc import maxwell_boltzmann_momenta
    from fastmd_amd.interfaces.gpu_md import GPUResidentMolecularDynamics
    from fastmd_amd.models.attention_like import AttentionAdapter, AttentionConfig

    s = systems.perovskite(3)
    momenta = maxwell_boltzmann_momenta(s.masses, 500.0, 20)
    runs = []
    for execution in ("eager", "whole_step"):
        md = GPUResidentMolecularDynamics(s, model=AttentionAdapter(device=device, config=AttentionConfig(**CONFIGS[0])), device=device,
                                          temperature=500.0, timestep=0.25, tdamp=25.0, momenta=momenta,
                                          steps_per_launch=5 if execution == "whole_step" else 1,
                                          config=InferenceConfig(execution=execution))
        md.run(10)
        torch.cuda.synchronize()
        runs.append((md.integrator.positions.clone(), float(md.integrator.potential_energy.item())))
    assert float((runs[0][0] - runs[1][0]).abs().max()) < 1e-6
    assert abs(runs[0][1] - runs[1][1]) < 1e-5 * s.n_atoms


@pytest.mark.gpu
def test_a_block_with_weights_in_8_bits(device):
    """A block evaluated with its products on 8-bit weights, its features normed over systems: each step within the bounds of what
    it is given."""
    from fastmd_amd.ops.feed_forward import gated_feed_forward
    from fastmd_amd.ops.group_norm import group_norm
    from fastmd_amd.ops.int8 import linear_int8, quantize_rows

    g = torch.Generator().manual_seed(5)
    x = torch.randn(300, 64, generator=g) + 2.0
    w, wg, wu, wd = (torch.randn(*s, generator=g) * s[1] ** -0.5 for s in ((96, 64), (136, 96), (136, 96), (96, 136)))
    off = torch.tensor([0, 120, 290])
    gpu = lambda t: t.to(device)  # noqa: E731
    n = group_norm(gpu(x), 8, offsets=gpu(off), activation="silu")
    blocks.near(n, *blocks.group_norm(x, 8, None, None, off, name="silu")[0])
    y = linear_int8(n, quantize_rows(gpu(w)))
    blocks.near(y, *blocks.linear_int8(*blocks.quantize(n.cpu()), *blocks.quantize(w), None, torch.float32))
    z = gated_feed_forward(y, gpu(wg), gpu(wu), gpu(wd))
    blocks.near(z, *blocks.gated(y.cpu(), wg, wu, wd, "silu")[0])
    # and near the block in float32: 8 bits round values to 1/254 of a row's largest
    want = blocks.gated(torch.as_tensor(n.cpu() @ w.T), wg, wu, wd, "silu")[0][0]
    assert float((z.cpu().double() - want).norm() / want.norm()) < 0.03
    assert not z[290:].any()  # rows of no system

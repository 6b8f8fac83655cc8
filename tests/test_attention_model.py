"""The attention potential: the float64 oracle pinned by finite differences and invariances (CPU); the model on the HIP
kernels against it, in MD (one system, a union of systems, captured steps) and in training (GPU).

Tolerances are those of the package's other models (1e-5 eV per atom, 1e-4 of the largest force): a chain of about ten
float32 products of up to 128 terms, each within 2^-24 sqrt(128) ~ 7e-7 of its terms."""
import dataclasses

import numpy as np
import pytest
import torch

from oracle import models as om
from oracle import nl as onl
from fastmd_amd import systems
from fastmd_amd.adapters.protocol import PaddingRule
from fastmd_amd.config import InferenceConfig

F32 = np.float32


def _edges(s, cutoff=6.0):
    cell32 = s.cell.astype(F32)
    inv = np.linalg.inv(cell32.astype(np.float64)).astype(F32)
    _, wraps, wrapped = onl.wrap(s.positions, inv, cell32)
    cand = onl.candidates(wrapped, cell32, F32((cutoff + 1.0) ** 2), 1504)
    b = onl.build(s.positions, inv, cell32, cand, s.positions.astype(F32), wraps, F32(cutoff ** 2), F32(2.0),
                  (1, 0, 0), 10 ** 7)
    e = b.n_edges
    return (torch.tensor(b.center[:e].astype(np.int64)), torch.tensor(b.neighbor[:e].astype(np.int64)),
            torch.tensor(b.images[:e]), torch.tensor(b.wrapped.astype(np.float64)))


def _model(**config):
    from fastmd_amd.models.attention_like import AttentionConfig, AttentionLike

    cfg = AttentionConfig(**config)
    m = AttentionLike(cfg)
    return m, {k: v.detach().clone() for k, v in m.named_parameters()}, dataclasses.asdict(cfg)


def _elem(s, cfg):
    return torch.tensor([cfg["elements"].index(int(z)) for z in s.numbers])


def _fn(params, cfg, s, edges):
    return lambda pos: om.attention_like_node_energy(params, cfg, pos, torch.tensor(s.cell), _elem(s, cfg), *edges[:3])


def test_oracle_forces_and_invariances():
    """Forces are the energy's gradient, sum to zero, and atoms in another order give the same energies."""
    s = systems.perovskite(2)
    edges = _edges(s)
    _, params, cfg = _model()
    fn, pos = _fn(params, cfg, s, edges), edges[3]
    _, f, e = om.energy_and_forces(fn, pos)
    assert float(f.abs().max()) > 1e-2
    for atom, k in ((0, 0), (7, 1), (23, 2)):
        d = torch.zeros_like(pos)
        d[atom, k] = 1e-5
        fd = -(fn(pos + d).sum() - fn(pos - d).sum()) / 2e-5
        assert abs(float(fd - f[atom, k])) < 1e-6 * max(1.0, abs(float(fd)))
    assert float(f.sum(0).abs().max()) < 1e-10
    order = torch.randperm(s.n_atoms, generator=torch.Generator().manual_seed(1))
    place = torch.empty_like(order)
    place[order] = torch.arange(s.n_atoms)
    again = om.attention_like_node_energy(params, cfg, pos[order], torch.tensor(s.cell), _elem(s, cfg)[order],
                                          place[edges[0]], place[edges[1]], edges[2])
    assert float((again - e[order]).abs().max()) < 1e-11


def test_config_is_checked():
    with pytest.raises(ValueError, match="kv_heads"):
        _model(heads=3, kv_heads=2)


def _builder(s, device):
    from fastmd_amd.graph.fixed_capacity_builder import FixedCapacityGraphBuilder

    return FixedCapacityGraphBuilder(cell=torch.tensor(s.cell), atomic_numbers=torch.tensor(s.numbers),
                                     u_capacity=int(s.n_atoms * 18 / 2) + 100, t_capacity=0, atom_graph_cutoff=6.0,
                                     line_graph_cutoff=None, candidate_cutoff=8.0,
                                     padding=PaddingRule("far_self_loops"), device=device)


@pytest.mark.gpu
@pytest.mark.parametrize("n_cells,config", [(3, {}), (6, {}), (3, {"heads": 2, "kv_heads": 1, "head_dim": 64}),
                                            ((3, 3, 4), {"heads": 4, "kv_heads": 4, "head_dim": 24})])
def test_model_matches_oracle(device, n_cells, config):
    from fastmd_amd.engine.energy_derivative import EnergyDerivative
    from fastmd_amd.models.attention_like import AttentionAdapter

    print(f"[attention model] cells={n_cells} {config}", flush=True)
    s = systems.perovskite(n_cells, sigma=0.2)
    m, params, cfg = _model(**config)
    adapter = AttentionAdapter(m, device=device)
    builder = _builder(s, device)
    _, status = builder.build(torch.tensor(s.positions, device=device))
    assert not bool(status.overflow.item())
    inputs = adapter.prepare(builder.batch)
    deriv = EnergyDerivative(adapter)
    out = deriv(builder.batch, inputs, n_real=s.n_atoms)
    again = deriv(builder.batch, inputs, n_real=s.n_atoms)
    torch.cuda.synchronize()
    assert torch.equal(out["e"], again["e"]) and torch.equal(out["f"][0], again["f"][0])
    edges = _edges(s)
    e, f, _ = om.energy_and_forces(_fn(params, cfg, s, edges), edges[3])
    assert abs(float(out["e"].item()) - float(e)) / s.n_atoms < 1e-5
    assert float((out["f"][0].cpu().double() - f).abs().max()) < 1e-4 * max(1.0, float(f.abs().max()))


@pytest.mark.gpu
def test_training_gradients_match_oracle(device):
    """Gradients of a loss on the energies with respect to every parameter."""
    from fastmd_amd.models.attention_like import AttentionAdapter

    s = systems.perovskite(3, sigma=0.2)
    m, params, cfg = _model()
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
def test_md_eager_captured_and_union_agree(device):
    """Ten steps: the captured step follows the eager one, and each system of a union (two slots with vacant rows) its own
    run, to the float32 rounding of the forces (1e-4 of them moves an atom by 1e-4 F / m t^2 / 2 < 1e-6 A here)."""
    from fastmd_amd.execution.gpu_nhc import maxwell_boltzmann_momenta
    from fastmd_amd.execution.system_batch import SystemBatchedMD
    from fastmd_amd.interfaces.gpu_md import GPUResidentMolecularDynamics
    from fastmd_amd.models.attention_like import AttentionAdapter

    sys_list = [systems.perovskite(3), systems.perovskite((3, 3, 4), seed=1)]
    momenta = [maxwell_boltzmann_momenta(s.masses, 500.0, 20 + k) for k, s in enumerate(sys_list)]

    def run(k, execution):
        md = GPUResidentMolecularDynamics(sys_list[k], model=AttentionAdapter(device=device), device=device,
                                          temperature=500.0, timestep=0.25, tdamp=25.0, momenta=momenta[k],
                                          steps_per_launch=5 if execution == "whole_step" else 1,
                                          config=InferenceConfig(execution=execution))
        md.run(10)
        torch.cuda.synchronize()
        print(f"[attention model] system {k} {execution}", flush=True)
        return md.integrator.positions.clone(), float(md.integrator.potential_energy.item())

    captured = [run(k, "whole_step") for k in range(2)]
    q, e = run(0, "eager")
    assert float((q - captured[0][0]).abs().max()) < 1e-6
    assert abs(e - captured[0][1]) < 1e-5 * sys_list[0].n_atoms
    batch = SystemBatchedMD(sys_list, AttentionAdapter(device=device), ceilings=(140, 200), device=device,
                            temperature=500.0, timestep=0.25, tdamp=25.0, momenta=momenta, steps_per_launch=5)
    batch.run(10)
    torch.cuda.synchronize()
    for k, s in enumerate(sys_list):
        got = batch.system_state(k)
        assert float((got["positions"] - captured[k][0]).abs().max()) < 1e-6
        assert abs(float(got["potential_energy"].item()) - captured[k][1]) < 1e-5 * s.n_atoms

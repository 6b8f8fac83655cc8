"""The attention potential in replica batches: a replica's atoms attend to its own, whatever the others do.

Tolerances are those of test_attention_model.py (1e-5 eV per atom, 1e-4 of the largest force) and, for ten steps, 1e-6 A."""
import types

import numpy as np
import pytest
import torch

from oracle import models as om
from fastmd_amd import systems
from fastmd_amd.adapters.protocol import PaddingRule
from fastmd_amd.config import InferenceConfig
from test_attention_model import _edges, _fn, _model

REPLICAS = 3


def _batch(n_real, **fields):
    return types.SimpleNamespace(**{"positions": None, "n_real": n_real, "edge_offsets": torch.zeros(1), "systems": None,
                                    "edge_reverse": torch.zeros(1), "species": torch.full((n_real,), 55), **fields})


def test_each_replica_is_a_segment():
    from fastmd_amd.models.attention_like import AttentionAdapter

    adapter = AttentionAdapter(device="cpu")
    offsets = lambda batch: adapter._offsets(adapter.prepare(batch)).tolist()  # noqa: E731
    assert offsets(_batch(20, max_system_rows=5)) == [0, 5, 10, 15, 20]
    assert offsets(_batch(20, max_system_rows=20)) == offsets(_batch(20)) == offsets(_batch(20, max_system_rows=0)) == [0, 20]
    with pytest.raises(ValueError, match="replicas"):
        adapter.prepare(_batch(20, max_system_rows=6))


@pytest.mark.gpu
def test_energies_and_forces_of_unlike_replicas(device):
    """Copies with positions of their own against the float64 oracle of each alone."""
    from fastmd_amd.engine.energy_derivative import EnergyDerivative
    from fastmd_amd.graph.fixed_capacity_builder import FixedCapacityGraphBuilder
    from fastmd_amd.models.attention_like import AttentionAdapter

    copies = [systems.perovskite(3, sigma=0.2, seed=k) for k in range(REPLICAS)]
    n = copies[0].n_atoms
    m, params, cfg = _model()
    adapter = AttentionAdapter(m, device=device)
    builder = FixedCapacityGraphBuilder(
        cell=torch.tensor(copies[0].cell), atomic_numbers=torch.tensor(np.tile(copies[0].numbers, REPLICAS)),
        u_capacity=REPLICAS * (n * 9 + 100), t_capacity=0, atom_graph_cutoff=6.0, line_graph_cutoff=None,
        candidate_cutoff=8.0, padding=PaddingRule("far_self_loops"), device=device, system_size=n)
    _, status = builder.build(torch.tensor(np.concatenate([s.positions for s in copies]), device=device))
    assert not bool(status.overflow.item())
    out = EnergyDerivative(adapter, segments=REPLICAS)(builder.batch, adapter.prepare(builder.batch),
                                                       n_real=REPLICAS * n)
    for k, s in enumerate(copies):
        edges = _edges(s)
        e, f, _ = om.energy_and_forces(_fn(params, cfg, s, edges), edges[3])
        assert abs(float(out["e"][k].item()) - float(e)) / n < 1e-5, k
        err = float((out["f"][0][k * n:(k + 1) * n].cpu().double() - f).abs().max())
        assert err < 1e-4 * max(1.0, float(f.abs().max())), k


@pytest.mark.gpu
def test_replicas_follow_their_own_runs(device):
    from fastmd_amd.execution.gpu_nhc import maxwell_boltzmann_momenta
    from fastmd_amd.execution.replica_batch import ReplicaBatchedMD
    from fastmd_amd.interfaces.gpu_md import GPUResidentMolecularDynamics
    from fastmd_amd.models.attention_like import AttentionAdapter

    s = systems.perovskite(3)
    momenta = np.stack([maxwell_boltzmann_momenta(s.masses, 500.0, 11 + k) for k in range(REPLICAS)])
    batch = ReplicaBatchedMD(s, AttentionAdapter(device=device), replicas=REPLICAS, device=device, temperature=500.0,
                             timestep=0.25, tdamp=25.0, momenta=momenta, steps_per_launch=5)
    batch.run(10)
    torch.cuda.synchronize()
    for k in range(REPLICAS):
        one = GPUResidentMolecularDynamics(s, model=AttentionAdapter(device=device), device=device, temperature=500.0,
                                           timestep=0.25, tdamp=25.0, momenta=momenta[k], steps_per_launch=5,
                                           config=InferenceConfig(execution="whole_step"))
        one.run(10)
        torch.cuda.synchronize()
        got = batch.replica_state(k)
        assert float((got["positions"] - one.integrator.positions).abs().max()) < 1e-6, k
        assert abs(float(got["potential_energy"].item()) - float(one.integrator.potential_energy.item())) < 1e-5 * s.n_atoms

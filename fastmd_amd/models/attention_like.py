"""An attention interatomic potential: the atoms of a system look at each other through
``qk_norm_rotary`` and ``segment_attention``, in MD (forces by their VJPs) as in training.

The reference has no such model (parity unpinned: the oracle is this package's own float64 form).

Model (atom features x [N, C], H query heads on Hk key heads of width D):
  edge e = (centre i <- neighbour j): ef_n = sqrt(2/rc) sin(n pi r/rc)/r fc(r), n = 1..8, fc the polynomial cutoff
  d_i[z, n] = (1 / avg_neighbors) sum_{e: centre i, element of j = z} ef_n          (what surrounds an atom)
  x = d W_in^T + embedding[Z]
  per layer: q | k | v = x W_qkv^T; each head of q and k is normed over its columns and turned by its atom's element
             (position = element index: the scores of a pair depend on both elements, not on the atoms' order)
             x += attention(q, k, v over the atoms of the system) W_o^T;  x += silu(x W_1^T) W_2^T
  readout:   E_i = e0[Z_i] + x_i . wr
Sums over a system's atoms are softmax-weighted means, so the energy is extensive and does not depend on the order of the
atoms. Random init from ``torch.Generator().manual_seed(seed)``; parameters are frozen as those of the other models are, and
``module.requires_grad_()`` trains them (``node_energy`` is differentiable once: losses on energies, not on forces).

A union of systems, or of replicas of one, is one call: the systems are the segments, and the vacant rows of a slot are
segments of their own.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch import Tensor, nn
from torch.autograd import Function

from fastmd_amd import _abi
from fastmd_amd._autograd import first_derivatives
from fastmd_amd.adapters.protocol import (CapacityStep, GraphBatch, PaddingRule, TopologySpec, require_atom_rows,
                                         system_rows)
from fastmd_amd.ops.attention import segment_attention
from fastmd_amd.ops.csr_segment_sum import Csr, segment_sum_csr, segment_sum_t
from fastmd_amd.ops.qk_norm import qk_norm_rotary, rotary_tables
from fastmd_amd.ops.wide_gemm import linear

_ELEMENTS = 118


@dataclass(frozen=True)
class AttentionConfig:
    channels: int = 64
    heads: int = 4
    kv_heads: int = 2
    head_dim: int = 32
    num_layers: int = 2
    n_basis: int = 8
    cutoff: float = 6.0
    avg_num_neighbors: float = 15.0
    elements: tuple = (55, 50, 53)
    seed: int = 0


class AttentionLike(nn.Module):
    """Parameters (float32), matrices stored [out, in]."""

    def __init__(self, config: AttentionConfig = AttentionConfig()) -> None:
        super().__init__()
        self.config = config
        C, H, Hk, D = config.channels, config.heads, config.kv_heads, config.head_dim
        if H < 1 or Hk < 1 or H % Hk:
            raise ValueError(f"heads must be a multiple of kv_heads, got {H} and {Hk}")
        gen = torch.Generator().manual_seed(config.seed)

        def rnd(*shape, scale=1.0):
            return nn.Parameter(torch.randn(*shape, generator=gen) * scale / math.sqrt(shape[-1]), requires_grad=False)

        nel = len(config.elements)
        self.W_in = rnd(C, nel * config.n_basis)
        self.embedding = rnd(nel, C, scale=math.sqrt(C))
        self.layers = nn.ModuleList()
        for _ in range(config.num_layers):
            layer = nn.Module()
            layer.W_qkv = rnd((H + 2 * Hk) * D, C)
            layer.q_weight = nn.Parameter(1.0 + 0.1 * torch.randn(D, generator=gen), requires_grad=False)
            layer.k_weight = nn.Parameter(1.0 + 0.1 * torch.randn(D, generator=gen), requires_grad=False)
            layer.W_o = rnd(C, H * D)
            layer.W_1 = rnd(2 * C, C)
            layer.W_2 = rnd(C, 2 * C)
            self.layers.append(layer)
        self.wr = rnd(C)
        self.e0 = nn.Parameter(-1.0 - torch.rand(nel, generator=gen), requires_grad=False)
        cos, sin = rotary_tables(nel, D)
        self.register_buffer("cos", cos)
        self.register_buffer("sin", sin)
        table = torch.full((_ELEMENTS + 1,), -1, dtype=torch.int32)
        for k, z in enumerate(config.elements):
            table[z] = k
        self.register_buffer("z_table", table)

    def forward(self, surroundings: Tensor, elem: Tensor, offsets: Tensor) -> Tensor:
        """Energies [N] of atoms in packed systems: ``surroundings`` [N, elements * n_basis], element indices [N], and
        ``offsets`` [systems + 1] of the systems' rows."""
        cfg = self.config
        H, Hk, D = cfg.heads, cfg.kv_heads, cfg.head_dim
        x = linear(surroundings, self.W_in) + self.embedding[elem]
        for layer in self.layers:
            qkv = linear(x, layer.W_qkv).view(-1, H + 2 * Hk, D)
            q, k, v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]  # read in place
            q, k = qk_norm_rotary(q, k, layer.q_weight, layer.k_weight, self.cos, self.sin, elem)
            x = x + linear(segment_attention(q, k, v, offsets).view(-1, H * D), layer.W_o)
            x = x + linear(nn.functional.silu(linear(x, layer.W_1)), layer.W_2)
        return self.e0[elem] + (x * self.wr).sum(1)


@dataclass
class AttentionInput:
    batch: GraphBatch
    elem: Tensor  # [rows] int64
    columns: Tensor  # [elements, elements] float32 identity
    rows: Tensor  # offsets of the one system's rows, or of equal replicas'


class _Surroundings(Function):
    """[rows, elements * n_basis] from the positions, and their gradient by the edge-geometry VJP (fixed order)."""

    @staticmethod
    def forward(ctx, positions, cell, model: AttentionLike, inputs: AttentionInput):
        cfg, batch, dev = model.config, inputs.batch, positions.device
        ctx.save_for_backward(positions)
        positions = positions.detach().contiguous()
        cell = cell.detach().to(torch.float32).contiguous()
        e_cap, nb, n = batch.edge_index.shape[0], cfg.n_basis, positions.shape[0]
        geo = torch.empty(e_cap, 8, dtype=torch.float32, device=dev)
        ef = torch.empty(e_cap, nb, dtype=torch.float32, device=dev)
        de = torch.empty(e_cap, nb, dtype=torch.float32, device=dev)
        _abi.call("fmd_edge_geometry_f32", positions.data_ptr(), cell.data_ptr(), system_rows(batch),
                  batch.edge_index.data_ptr(), batch.edge_image.data_ptr(), batch.n_edges.data_ptr(), e_cap, cfg.cutoff,
                  nb, geo.data_ptr(), ef.data_ptr(), de.data_ptr(), _abi.stream_handle())
        # 1 in the column of the neighbour's element
        neighbour = inputs.columns[inputs.elem[batch.edge_index[:, 1].long()]]
        rows = (neighbour[:, :, None] * ef[:, None, :]).reshape(e_cap, -1)
        ctx.saved = geo, de, neighbour
        ctx.inputs, ctx.nb, ctx.n, ctx.inv_avg = inputs, nb, n, 1.0 / cfg.avg_num_neighbors
        return segment_sum_csr([(rows, Csr(batch.edge_offsets, None, e_cap), 0, ctx.inv_avg, None)], n, rows.shape[1])

    @staticmethod
    def backward(ctx, g):
        geo, de, neighbour = ctx.saved
        batch, nb = ctx.inputs.batch, ctx.nb
        e_cap = geo.shape[0]
        grow, _ = segment_sum_t(g * ctx.inv_avg, Csr(batch.edge_offsets, None, e_cap), e_cap)
        gef = (grow.view(e_cap, -1, nb) * neighbour[:, :, None]).sum(1)
        gpos = torch.empty(ctx.n, 3, dtype=torch.float32, device=g.device)
        _abi.call("fmd_edge_forces_f32", geo.data_ptr(), de.data_ptr(), nb, gef.data_ptr(), nb, None, 0, None,
                  batch.edge_offsets.data_ptr(), batch.edge_reverse.data_ptr(), batch.n_edges.data_ptr(), e_cap, ctx.n,
                  1.0, gpos.data_ptr(), None, _abi.stream_handle())
        (gpos,) = first_derivatives("the attention model's energy", (gpos,), g, *ctx.saved_tensors)
        return gpos, None, None, None


class AttentionAdapter:
    """The model behind the adapter protocol: an energy tap that the engine differentiates."""

    name = "attention_like"
    compiled = False

    def __init__(self, module: AttentionLike | None = None, device="cuda",
                 config: AttentionConfig = AttentionConfig()) -> None:
        self.module = (module or AttentionLike(config)).to(device)

    def topology_spec(self) -> TopologySpec:
        return TopologySpec(cutoff=self.module.config.cutoff, num_interactions=1, model_dtype="float32")

    def padding_rule(self) -> PaddingRule:
        return PaddingRule("far_self_loops")

    def capacity_step(self) -> CapacityStep:
        return CapacityStep(u_step=32, min_pad_u=32, u_thermal_factor=1.02)

    def isolated_atom_policy(self) -> str:
        return "model"

    def reference_energies(self):
        return None

    def prepare(self, batch: GraphBatch) -> AttentionInput:
        """Aliases of the batch, the element index of every row (host check of the species)."""
        if batch.edge_offsets is None or batch.edge_reverse is None:
            raise ValueError("the attention model needs an edges-only batch with its CSR")
        require_atom_rows(batch, "attention")
        species = batch.species.long()
        table = self.module.z_table.to(species.device)
        if bool(((species < 1) | (species > _ELEMENTS)).any()) or bool((table[species.clamp(1, _ELEMENTS)] < 0).any()):
            raise ValueError(f"the attention model supports atomic numbers {list(self.module.config.elements)}")
        columns = torch.eye(len(self.module.config.elements), dtype=torch.float32, device=species.device)
        size = getattr(batch, "max_system_rows", 0) or batch.n_real or 1  # of a replica, or of the one system
        if getattr(batch, "systems", None) is None and batch.n_real % size:
            raise ValueError(f"{batch.n_real} atom rows are not whole replicas of {size}")
        rows = torch.arange(0, batch.n_real + 1, size, dtype=torch.int64, device=species.device)
        return AttentionInput(batch, table[species].long(), columns, rows)

    @staticmethod
    def _offsets(inputs: AttentionInput) -> Tensor:
        """Of the systems' rows; a slot is its atoms, then its vacant rows (a captured step reads the slots' state)."""
        systems = getattr(inputs.batch, "systems", None)
        if systems is None:
            return inputs.rows
        starts = systems.row_ptr
        if systems.atoms is None:
            return starts
        return torch.cat((torch.stack((starts[:-1], starts[:-1] + systems.atoms), 1).flatten(), starts[-1:]))

    def node_energy(self, inputs: AttentionInput, positions: Tensor, cell: Tensor) -> Tensor:
        if cell.requires_grad:
            raise NotImplementedError("stress (a strained cell) is not supported by the attention model")
        surroundings = _Surroundings.apply(positions, cell, self.module, inputs)
        return self.module(surroundings, inputs.elem, self._offsets(inputs))

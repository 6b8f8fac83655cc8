"""Model oracle (test infrastructure and the timed CPU baseline; see oracle/__init__.py).

PyTorch-CPU eager restatements, differentiated by autograd exactly as the reference's
engine-owned derivative does (fastmd/engine/energy_derivative.py:110-140: positions leaf, FP64
energy sum over the real rows, one ``torch.autograd.grad``, F = -dE/dx), with the reference's
CPU op forms: ``index_select`` gathers, ``index_add_`` receiver sums
(triton_csr_segment_sum.py:463-479) and dense ``matmul`` GEMMs (triton_wide_gemm.py:488-489).

* ``morse_node_energy``: the configs[0] Morse pair potential (D, a, r0, cutoff), shifted to zero at
  the cutoff, E_i = 1/2 sum_j V(r_ij).
* ``mace_like_node_energy``: the MACE-like model specified in fastmd_amd/models/mace_like.py
  (its parameters are passed in as a dict of tensors; the oracle does not import the product).
* ``threebody_like_node_energy``: the three-body model of fastmd_amd/models/threebody_like.py, its
  triplets formed here by brute force (every ordered pair of distinct bonds at a centre) and its
  angle basis by torch's own acos / sin / cos (parity of the model's data path and kernels; the
  model itself is this package's, the reference's CHGNet / MatRIS weights being unavailable).
Edges are the real rows (centre, neighbour, image) of a neighbour list; vec = pos[neighbour] +
image @ cell - pos[centre].
"""
from __future__ import annotations

import math

import torch
from torch import Tensor


def edge_vectors(positions: Tensor, cell: Tensor, center: Tensor, neighbor: Tensor, images: Tensor) -> Tensor:
    img = images.to(positions.dtype)
    shift = img[:, 0:1] * cell[0] + img[:, 1:2] * cell[1] + img[:, 2:3] * cell[2]
    return (positions.index_select(0, neighbor) + shift) - positions.index_select(0, center)


def morse_node_energy(positions, cell, center, neighbor, images, *, D=0.3, a=1.5, r0=3.0, cutoff=6.0):
    vec = edge_vectors(positions, cell, center, neighbor, images)
    r = vec.norm(dim=1)
    vshift = D * ((1 - math.exp(-a * (cutoff - r0))) ** 2 - 1)
    v = D * ((1 - torch.exp(-a * (r - r0))) ** 2 - 1) - vshift
    v = torch.where(r < cutoff, v, torch.zeros_like(v))
    return 0.5 * torch.zeros(positions.shape[0], dtype=positions.dtype).index_add_(0, center, v)


def radial_basis(r: Tensor, cutoff: float, n_basis: int):
    n = torch.arange(1, n_basis + 1, dtype=r.dtype)
    bessel = math.sqrt(2.0 / cutoff) * torch.sin(n[None, :] * math.pi * r[:, None] / cutoff) / r[:, None]
    x = r / cutoff
    fcut = 1 - 21 * x ** 5 + 35 * x ** 6 - 15 * x ** 7
    fcut = torch.where(x < 1, fcut, torch.zeros_like(fcut))
    return bessel * fcut[:, None], fcut


def mace_like_node_energy(params: dict, config: dict, positions, cell, elem, center, neighbor, images):
    """Per-atom energies of the MACE-like model (see the module docstring)."""
    dt = positions.dtype
    p = {k: v.to(dt) for k, v in params.items()}
    C, nb = config["channels"], config["n_basis"]
    L = config["num_interactions"]
    n_atoms = positions.shape[0]
    vec = edge_vectors(positions, cell.to(dt), center, neighbor, images)
    r = vec.norm(dim=1)
    u = vec / r[:, None]
    ef, fcut = radial_basis(r, config["cutoff"], nb)
    elem = elem.long()
    h0 = p["embedding"].index_select(0, elem)
    h1 = torch.zeros(n_atoms, 3, C, dtype=dt)
    h_first = None
    for t in range(L):
        W = {k.split(".", 2)[2]: v for k, v in p.items() if k.startswith(f"layers.{t}.")}
        last = t == L - 1
        hj = h0.index_select(0, neighbor)
        a = torch.cat([hj, h0.index_select(0, center), ef], dim=1)
        z = a @ W["W1"]
        w = torch.nn.functional.silu(z) * fcut[:, None]
        wa, wb, wc, wd = w[:, :C], w[:, C:2 * C], w[:, 2 * C:3 * C], w[:, 3 * C:]
        h1j = h1.index_select(0, neighbor)
        proj = (h1j * u[:, :, None]).sum(1)
        m0 = wa * hj + wc * proj
        m1 = (wb * hj)[:, None, :] * u[:, :, None] + wd[:, None, :] * h1j
        A0 = torch.zeros(n_atoms, C, dtype=dt).index_add_(0, center, m0) / config["avg_num_neighbors"]
        A1 = torch.zeros(n_atoms, 3, C, dtype=dt).index_add_(0, center, m1) / config["avg_num_neighbors"]
        P0 = A0 @ W["Wm0"]
        P1 = A1 @ W["Wm1"]
        n1 = (P1 * P1).sum(1)
        c = W["Wc"].index_select(0, elem)
        B0 = c[:, 0] * P0 + c[:, 1] * P0 ** 2 + c[:, 2] * n1 + c[:, 3] * P0 ** 3 + c[:, 4] * P0 * n1
        h0n = B0 @ W["Wo0"] + h0 @ W["Wsc0"]
        if not last:
            d = W["Wd"].index_select(0, elem)
            q = d[:, 0] + d[:, 1] * P0 + d[:, 2] * P0 ** 2 + d[:, 3] * n1
            h1 = (q[:, None, :] * P1) @ W["Wo1"]
        if t == 0:
            h_first = h0n
        h0 = h0n
    y = h0 @ p["Wr2a"]
    e = h_first @ p["wr1"] + torch.nn.functional.silu(y) @ p["wr2b"]
    return p["e0"].index_select(0, elem) + config["scale"] * e + config["shift"]


def poly_cutoff(r: Tensor, rc: float) -> Tensor:
    x = r / rc
    f = 1 - 21 * x ** 5 + 35 * x ** 6 - 15 * x ** 7
    return torch.where(x < 1, f, torch.zeros_like(f))


def triplets_of(center: Tensor, bonds: Tensor):
    """Every ordered pair (b1, b2) of two distinct bonds (edge rows in ``bonds``) with a common
    centre, as (centre, b1, b2) int64 tensors; brute force by centre."""
    by_atom: dict = {}
    for e in bonds.tolist():
        by_atom.setdefault(int(center[e]), []).append(e)
    a, b1, b2 = [], [], []
    for i, rows in by_atom.items():
        for x in rows:
            for y in rows:
                if x != y:
                    a.append(i)
                    b1.append(x)
                    b2.append(y)
    as_t = lambda v: torch.tensor(v, dtype=torch.int64)  # noqa: E731
    return as_t(a), as_t(b1), as_t(b2)


def threebody_like_node_energy(params: dict, config: dict, positions, cell, elem, center, neighbor, images,
                               bond_rows=None):
    """Per-atom energies of the three-body model specified in fastmd_amd/models/threebody_like.py.
    Bonds are the edges shorter than the bond cutoff (``bond_rows`` to fix the set, e.g. to the
    builder's float32 decision; a row at the cutoff has a zero envelope either way)."""
    dt = positions.dtype
    p = {k: v.to(dt) for k, v in params.items()}
    C, nb, L, F = config["channels"], config["n_basis"], config["num_interactions"], config["n_freq"]
    rb = config["bond_cutoff"]
    n_atoms = positions.shape[0]
    vec = edge_vectors(positions, cell.to(dt), center, neighbor, images)
    r = vec.norm(dim=1)
    u = vec / r[:, None]
    ef, fc = radial_basis(r, config["cutoff"], nb)
    if bond_rows is None:
        bond_rows = torch.nonzero(r.detach() < rb).flatten()
    s = torch.zeros_like(r).index_copy(0, bond_rows, poly_cutoff(r.index_select(0, bond_rows), rb))
    atom, b1, b2 = triplets_of(center, bond_rows)
    cos = (u.index_select(0, b1) * u.index_select(0, b2)).sum(1) * (1 - 1e-6)
    theta = torch.arccos(cos)
    ph = theta[:, None] * torch.arange(1, F + 1, dtype=dt)[None, :]
    alpha = torch.cat([torch.full_like(theta[:, None], 2 ** -0.5), torch.sin(ph), torch.cos(ph)], 1) / math.sqrt(math.pi)
    elem = elem.long()
    h = p["embedding"].index_select(0, elem)
    eps = ef @ p["We"]
    w3 = s.index_select(0, b1) * s.index_select(0, b2)
    for t in range(L):
        W3, W2 = p[f"layers.{t}.W3"], p[f"layers.{t}.W2"]
        z3 = torch.cat([eps.index_select(0, b1), eps.index_select(0, b2), h.index_select(0, atom), alpha], 1) @ W3
        eps = eps.index_add(0, b1, torch.nn.functional.silu(z3) * w3[:, None] / config["avg_num_angles"])
        z2 = torch.cat([h.index_select(0, neighbor), h.index_select(0, center), eps], 1) @ W2
        h = h.index_add(0, center, torch.nn.functional.silu(z2) * fc[:, None] / config["avg_num_neighbors"])
    return p["e0"].index_select(0, elem) + h @ p["wr"]


def energy_and_forces(node_energy_fn, positions, *args, n_real=None, **kwargs):
    """The engine-owned derivative (energy_derivative.py:110-140): FP64 sum, one autograd.grad."""
    leaf = positions.detach().clone().requires_grad_(True)
    energies = node_energy_fn(leaf, *args, **kwargs)
    rows = energies.shape[0] if n_real is None else n_real
    energy = energies[:rows].to(torch.float64).sum()
    (grad,) = torch.autograd.grad(energy, leaf)
    return energy.detach(), -grad, energies.detach()


def energy_forces_stress(node_energy_fn, positions, cell):
    """The engine-owned derivative with its strain leaf (energy_derivative.py:110-140): a zero
    [3, 3] strain e, S = (e + e^T) / 2, the positions and the cell both deformed as x -> x + x S
    (the row-by-row ``_times`` of energy_derivative.py:76-79), FP64 energy sum, one autograd.grad
    over (positions, strain); F = -dE/dx and stress = dE/de / |c0 . (c1 x c2)| of the unstrained
    cell. ``node_energy_fn(positions, cell)`` returns per-atom energies."""
    leaf = positions.detach().clone().requires_grad_(True)
    cell = cell.detach().to(leaf.dtype)
    strain = torch.zeros((3, 3), dtype=leaf.dtype, requires_grad=True)
    sym = 0.5 * (strain + strain.transpose(0, 1))
    times = lambda rows: rows[:, 0:1] * sym[0] + rows[:, 1:2] * sym[1] + rows[:, 2:3] * sym[2]  # noqa: E731
    energies = node_energy_fn(leaf + times(leaf), cell + times(cell))
    energy = energies.to(torch.float64).sum()
    grad, gstrain = torch.autograd.grad(energy, (leaf, strain))
    volume = torch.dot(cell[0], torch.linalg.cross(cell[1], cell[2])).abs()
    return energy.detach(), -grad, gstrain / volume


def attention_like_node_energy(params: dict, config: dict, positions, cell, elem, center, neighbor, images, systems=None):
    """Per-atom energies of the attention model specified in fastmd_amd/models/attention_like.py. ``systems``: (first row,
    rows) of each system (None: one)."""
    dt = positions.dtype
    p = {k: v.to(dt) for k, v in params.items()}
    n, nb, nel = positions.shape[0], config["n_basis"], len(config["elements"])
    H, Hk, D = config["heads"], config["kv_heads"], config["head_dim"]
    vec = edge_vectors(positions, cell.to(dt), center, neighbor, images)
    ef, _ = radial_basis(vec.norm(dim=1), config["cutoff"], nb)
    elem = elem.long()
    d = torch.zeros(n * nel, nb, dtype=dt).index_add_(0, center * nel + elem[neighbor], ef)
    x = d.view(n, nel * nb) / config["avg_num_neighbors"] @ p["W_in"].T + p["embedding"][elem]
    turn = elem[:, None].to(dt) * 10000.0 ** (-torch.arange(0, D, 2, dtype=dt) / D)
    cos, sin = turn.cos()[:, None], turn.sin()[:, None]

    def head(t, weight):
        t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * weight
        a, b = t[..., :D // 2], t[..., D // 2:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    def normed(x, W, name):
        groups = config.get("norm_groups", 0)
        if not groups:
            return x
        y = x.view(n, groups, -1)
        y = (y - y.mean(-1, keepdim=True)) * torch.rsqrt(y.var(-1, correction=0, keepdim=True) + 1e-5)
        return y.reshape(n, -1) * W[name + "_norm_weight"] + W[name + "_norm_bias"]

    silu = torch.nn.functional.silu
    for t in range(config["num_layers"]):
        W = {k.split(".", 2)[2]: v for k, v in p.items() if k.startswith(f"layers.{t}.")}
        qkv = (normed(x, W, "attention") @ W["W_qkv"].T).view(n, H + 2 * Hk, D)
        q, k, v = head(qkv[:, :H], W["q_weight"]), head(qkv[:, H:H + Hk], W["k_weight"]), qkv[:, H + Hk:]
        k, v = k.repeat_interleave(H // Hk, 1), v.repeat_interleave(H // Hk, 1)
        out = []
        for a, m in systems or [(0, n)]:
            s = torch.einsum("ihd,jhd->hij", q[a:a + m], k[a:a + m]) / math.sqrt(D)
            out.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), v[a:a + m]))
        x = x + torch.cat(out).reshape(n, H * D) @ W["W_o"].T
        y = normed(x, W, "feed_forward")
        if "W_gate" in W:
            x = x + (silu(y @ W["W_gate"].T) * (y @ W["W_up"].T)) @ W["W_down"].T
        else:
            x = x + silu(y @ W["W_1"].T) @ W["W_2"].T
    return p["e0"][elem] + (x * p["wr"]).sum(1)

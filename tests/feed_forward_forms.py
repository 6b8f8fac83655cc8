"""Which of its three forms a call of the gated feed-forward block takes, from the sizes that the library asks for: "one" kernel, products
"straight" from memory, or "tiles" in LDS."""
from fastmd_amd import _abi


def _up(x, n):
    return -(-x // n) * n


def forms(bf16, rows, width, hidden, out):
    """(form of the forward pass, form of the VJP for x)"""
    lib = _abi.load()
    if not lib.fmd_gated_ffn_saves(bf16, rows, width, hidden, out):
        return "one", "one"
    forward = lib.fmd_gated_ffn_work_size(bf16, rows, width, hidden, out, 15, 1)  # tiles: the operands' layouts at least
    back = lib.fmd_gated_ffn_bwd_work_size(bf16, rows, width, hidden, out, 15, 1, 0)
    gradients = _up(2 * rows * _up(hidden, 8) * 2 * (2 if bf16 else 3), 256)  # straight: dg and du alone, in their planes
    assert back >= gradients
    return "tiles" if forward else "straight", "tiles" if back > gradients else "straight"

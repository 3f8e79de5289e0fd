"""The parts of long contractions, as the workspaces' sizes show them, without a GPU."""
import random

import pytest

pytest.importorskip("torch")

from moe_offload import _lib  # noqa: E402


def filled(nc, parts):
    """Whether every part of whole steps of 64 has something to sum."""
    steps = -(-nc // 64)
    return (parts - 1) * -(-steps // parts) < steps


def test_no_part_of_a_contraction_is_empty():
    lib = _lib.lib()
    rng = random.Random(5)
    sizes = [(64, 7744, 1040), (32, 4096, 4096), (100, 2560, 640), (40, 64, 100000), (64, 64, 100000)]
    sizes += [tuple(8 * int(2 ** rng.uniform(0, 14)) for _ in range(3)) for _ in range(4000)]
    forward = backward = 0
    for n_tok, n_in, n_out in sizes:
        parts, rest = divmod(lib.moe_linear_workspace_bytes(n_tok, n_in, n_out), 4 * n_tok * n_out)
        assert rest == 0
        if parts:
            assert parts > 1 and filled(n_in, parts), (n_tok, n_in, n_out, parts)
            forward += 1
    for n_in, n_out, n_tok in sizes:
        parts, rest = divmod(lib.moe_linear_grad_workspace_bytes(n_tok, n_in, n_out, 0, 0, 1, 0), 4 * n_in * n_out)
        assert rest == 0
        if parts:
            assert parts > 1 and filled(n_tok, parts), (n_tok, n_in, n_out, parts)
            backward += 1
    assert forward > 50 and backward > 50

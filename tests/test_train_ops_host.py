"""What the operators around the blocks of a training step refuse or compute without a GPU."""
import pytest
import torch

import asca_b200
from asca_b200 import ops


class Nothing:
    """Stands for a context on cuda:0 that must not be reached."""
    device = 0

    def _run(self, *args):
        raise AssertionError("the library was called")


def test_scratch_sizes():
    lib = asca_b200.load()
    assert lib.asca_embed_scaled_bwd_ws(0, 8, 10) > 0
    # sorted keys and tokens twice, at least; nothing that grows with vocabulary times tokens
    assert 4 * 4 * 100_000 < lib.asca_embed_scaled_bwd_ws(100_000, 64, 50_000) < 100_000 * 64 * 4
    assert lib.asca_embed_scaled_bwd_ws(-1, 8, 10) < 0 and lib.asca_embed_scaled_bwd_ws(1, 0, 10) < 0 and lib.asca_embed_scaled_bwd_ws(1, 8, 0) < 0
    assert lib.asca_moe_topk_dispatch_ws(1, 1, 2048) > 0 and lib.asca_moe_topk_dispatch_ws(1, 1, 2049) < 0 and lib.asca_moe_topk_dispatch_ws(1, 0, 4) < 0
    # without a context: refused, not followed
    assert lib.asca_gated_residual_rmsnorm_bwd_ws(None, 4, 4) < 0 and lib.asca_grad_norm_ws(None, 1) < 0


def test_entry_points_refuse_a_null_context():
    lib = asca_b200.load()
    for name, (_, args) in asca_b200._SIGNATURES.items():
        if not name.endswith("_ws"):
            assert getattr(lib, name)(*[None if a in (asca_b200._P,) else 0 for a in args]) == -1, name


def test_tensors_that_are_not_on_the_device_are_refused():
    t = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="cuda:0"):
        ops._need(Nothing(), "x", t)
    with pytest.raises(ValueError, match="x: expected"):
        ops._need(Nothing(), "x", None)

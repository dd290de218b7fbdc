"""What the operators around the blocks of a training step refuse or compute without a GPU."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import asca_b200
from asca_b200 import ops


class Closed:
    """Stands for a context that has been closed."""
    handle, device, bound_stream = 0, 0, 1


def test_scratch_sizes():
    lib = asca_b200.load()
    assert lib.asca_embed_scaled_bwd_ws(0, 8, 10) == 0 and lib.asca_embed_scaled_bwd_ws(2048, 64, 256) == 0   # few tokens need none
    # sorted keys and tokens twice, at least; nothing that grows with vocabulary times tokens
    assert 4 * 4 * 100_000 < lib.asca_embed_scaled_bwd_ws(100_000, 64, 50_000) < 100_000 * 64 * 4
    assert lib.asca_embed_scaled_bwd_ws(-1, 8, 10) < 0 and lib.asca_embed_scaled_bwd_ws(1, 0, 10) < 0 and lib.asca_embed_scaled_bwd_ws(1, 8, 0) < 0
    assert lib.asca_moe_topk_dispatch_ws(1, 1, 2048) == 0 and lib.asca_moe_topk_dispatch_ws(40_000, 1, 2048) > 0 and lib.asca_moe_topk_dispatch_ws(1, 1, 2049) < 0 and lib.asca_moe_topk_dispatch_ws(1, 0, 4) < 0
    # without a context: refused, not followed
    assert lib.asca_gated_residual_rmsnorm_bwd_ws(None, 4, 4) < 0 and lib.asca_grad_norm_ws(None, 1) < 0


def test_entry_points_refuse_a_null_context():
    lib = asca_b200.load()
    for name, (_, args) in asca_b200._SIGNATURES.items():
        if not name.endswith("_ws"):
            assert getattr(lib, name)(*[None if a in (asca_b200._P,) else 0 for a in args]) == -1, name


def test_a_closed_context_is_refused():
    t, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ops.embed_fwd(Closed(), t, ids), lambda: ops.grad_norm(Closed(), [t]), lambda: ops.moe_topk_dispatch(Closed(), ids.view(2, 2), 4),
                 lambda: ops.gated_residual_rmsnorm_fwd(Closed(), t, t)):
        with pytest.raises(ValueError, match="closed"):
            call()


def test_norm_and_largest_norm_belong_together():
    t = torch.zeros(8)
    for kw in (dict(norm=t), dict(max_norm=1.0)):
        with pytest.raises((ValueError, AssertionError)):
            ops.adamw_segmented(Closed(), t, t, t, t, [0, 8], [1e-3], [1e-8], 0.9, 0.95, 0.0, **kw)


def test_scratch_of_sizes_that_the_calls_refuse():
    lib = asca_b200.load()
    for bad in (1 << 31, 1 << 40, 1 << 62, (1 << 63) - 1):
        assert lib.asca_embed_scaled_bwd_ws(4, 8, bad) < 0 and lib.asca_embed_scaled_bwd_ws(bad, 8, 4) < 0 and lib.asca_embed_scaled_bwd_ws(4, bad, 4) < 0
        assert lib.asca_moe_topk_dispatch_ws(4, 1, bad) < 0 and lib.asca_moe_topk_dispatch_ws(bad, 1, 4) < 0 and lib.asca_moe_topk_dispatch_ws(4, bad, 4) < 0
    assert lib.asca_embed_scaled_bwd_ws(4, 8, (1 << 31) - 1) == 0 and lib.asca_embed_scaled_bwd_ws((1 << 31) - 1, 8, 4) > 0


WITHOUT = """
import sys, torch
{how}
from asca_b200 import ops
class Closed:
    handle, device, bound_stream = 0, 0, 1
assert all(callable(getattr(ops, f)) for f in ("gemm", "adamw", "rmsnorm_fwd", "moe_fwd", "DeltaHostPipeline"))
for call in (lambda: ops.embed_fwd(Closed(), None, None), lambda: ops.grad_norm(Closed(), []), lambda: ops.moe_sort_rows(Closed(), None, None)):
    try:
        call()
    except ImportError as e:
        assert "python -m asca_b200.build" in str(e)
    else:
        raise SystemExit("not refused")
"""


# not there, of another torch, one that does not say of which
@pytest.mark.parametrize("how", ["sys.modules['asca_b200._torch_ops'] = None", "torch.__version__ = '9.9.9'", "sys.modules['asca_b200._torch_ops'] = type(sys)('old')"])
def test_what_needs_the_library_alone_works_without_the_torch_binding(how):
    r = subprocess.run([sys.executable, "-c", WITHOUT.replace("{how}", how)], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_the_torch_binding_is_built_for_the_torch_at_hand(monkeypatch, tmp_path):
    from asca_b200 import _torch_ops, build

    assert torch.__version__ in _torch_ops.built_for
    commands = []

    def run(cmd, **_):
        commands.append(cmd)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    assert build.build_torch_ops() == build.TORCH_OPS and not commands   # as it is
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    for abi in (True, False):
        monkeypatch.setattr(torch, "compiled_with_cxx11_abi", lambda: abi)
        build.build_torch_ops()
        assert f"-D_GLIBCXX_USE_CXX11_ABI={int(abi)}" in commands[-1] and any("9.9.9" in word for word in commands[-1])
    monkeypatch.setattr("importlib.util.find_spec", lambda name: None)
    assert build.build_torch_ops() is None and len(commands) == 2

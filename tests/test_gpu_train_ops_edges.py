"""The operators around the blocks of a training step where their plans change: pairs of CTAs, strips and gate groups, columns one by
one, several contexts at once, what a graph keeps, what is refused. The statements in 64 bits and their bounds are those of
test_gpu_train_ops.py."""
import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest
import torch

import asca_b200
from asca_b200 import ops
from test_gpu_train_ops import DTYPES, U, join_case, rand, route, text, within
from test_gpu_train_ops import test_embedding_forward_and_gradient as check_embedding
from test_gpu_train_ops import test_gated_residual_forward_and_gradients as check_join
from test_gpu_train_ops import unaligned

pytestmark = pytest.mark.gpu


# Above 4096 columns two CTAs share a row of the backward pass. Up to 74 rows a pair has one row: every value rests on the first
# exchange between its CTAs.
@pytest.mark.parametrize("rows,cols,per", [(1, 4097, None), (1, 8192, None), (2, 4100, 1), (5, 8191, 2), (60, 5001, 7), (74, 8192, None), (73, 6144, 1)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_first_rows_of_a_pair(gpu, rows, cols, per, dtype):
    check_join(gpu, rows, cols, per, True, True, dtype)
    t, kw = join_case(rows, cols, per, True, True, dtype)
    args = dict(gate=t["gate"], w_post=t["w_post"], w_pre=t["w_pre"], **kw)
    d_xn, d_out = rand(7, rows, cols, dtype=dtype), rand(8, rows, cols)
    first = ops.gated_residual_rmsnorm_bwd(gpu, t["y"], t["x"], d_xn, d_out, **args)
    for _ in range(50):   # one behind the other: pairs that start while others leave
        again = ops.gated_residual_rmsnorm_bwd(gpu, t["y"], t["x"], d_xn, d_out, **args)
        assert all(torch.equal(v, again[k]) for k, v in first.items())


# Optimizer steps over more tensors than one launch's table holds. Offsets that are no multiples of four: a group of four elements on
# the border of two launches is done by both of them, each its own elements.
SEGMENTS = [128, 129, 200, 256, 400]


def adam_state(n_seg, seed=5):
    rng = np.random.default_rng(seed)
    sizes = rng.integers(0, 41, n_seg)
    sizes[n_seg // 2:n_seg // 2 + 9] = 0   # empty tensors
    off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)
    n = int(off[-1])
    lr, eps = rng.uniform(1e-4, 1e-2, n_seg).astype(np.float32), rng.uniform(1e-8, 1e-6, n_seg).astype(np.float32)
    return off, lr, eps, [rand(1, n), rand(2, n), rand(3, n, scale=0.1), rand(4, n).square()]


@pytest.mark.parametrize("n_seg", SEGMENTS)
@pytest.mark.parametrize("shift", [0, 1])   # on the 16-byte grid, off it
@pytest.mark.parametrize("clip", [False, True])
def test_adamw_of_many_tensors(gpu, n_seg, shift, clip):
    """Against 64 bits. Roundings: three of a moment (two products, their sum; 1 - beta is exact), four of the second; a root halves
    what its argument is off by, and it, the sum with eps and the quotient add one each, so the update is off by at most
    3 u M / D + 5 u |m| / D <= 8 u M / D, M the magnitudes in the first moment and D the denominator; the decay is off by 2 u |p|, the last
    product and sum by u (|p| + 2 lr M / D)."""
    off, lr, eps, (g, p, m, v) = adam_state(n_seg)
    place = lambda t: torch.cat([t.new_zeros(shift), t])[shift:]  # noqa: E731
    norm = ops.grad_norm(gpu, [g])
    got, gs = [place(t) for t in (p, m, v)], place(g)
    ops.adamw_segmented(gpu, got[0], gs, got[1], got[2], off, lr, eps, 0.9, 0.95, 1e-4, **(dict(norm=norm, max_norm=1.0) if clip else {}))
    assert torch.equal(gs, g)
    gc = (g * (1.0 / (norm + 1e-6)).clamp(max=1.0) if clip else g).double()   # (rounded to f32 before it enters, as the step does it)
    b1, b2, wd = (float(np.float32(x)) for x in (0.9, 0.95, 1e-4))
    per = torch.from_numpy(np.diff(off)).cuda()
    lr64, eps64 = (torch.from_numpy(x).cuda().double().repeat_interleave(per) for x in (lr, eps))
    m64, big_m = b1 * m.double() + (1 - b1) * gc, (b1 * m.double()).abs() + ((1 - b1) * gc).abs()
    v64 = b2 * v.double() + (1 - b2) * gc * gc
    d64 = v64.sqrt() + eps64
    within(got[1], m64, 3 * U * big_m, "m")
    within(got[2], v64, 4.01 * U * v64, "v")
    within(got[0], p.double() * (1 - wd) - lr64 * m64 / d64, 4 * U * p.double().abs() + 11 * U * lr64 * big_m / d64, "p")


@pytest.mark.parametrize("n_seg", SEGMENTS)
@pytest.mark.parametrize("clip", [False, True])
def test_a_captured_adamw_keeps_its_rates(gpu, n_seg, clip):
    """The host arrays belong to the caller again when the call returns."""
    off, lr, eps, (g, p, m, v) = adam_state(n_seg)
    want, got = ([t.clone() for t in (p, m, v)] for _ in range(2))
    kw = dict(norm=ops.grad_norm(gpu, [g]), max_norm=1.0) if clip else {}
    ops.adamw_segmented(gpu, want[0], g, want[1], want[2], off, lr, eps, 0.9, 0.95, 1e-4, **kw)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    try:
        with torch.cuda.stream(stream):
            gpu.use_torch_stream()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                ops.adamw_segmented(gpu, got[0], g, got[1], got[2], off, lr, eps, 0.9, 0.95, 1e-4, **kw)
            lr[:] = 7.0
            eps[:] = 1.0
            graph.replay()
            stream.synchronize()
    finally:
        gpu.use_torch_stream()
    assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_a_norm_among_what_is_written_is_refused(gpu):
    """It would be read by blocks that begin behind the first write."""
    flat = rand(1, 4000)
    before = flat.clone()
    for norm in (flat[:1], flat[3999:], flat[1000:1001]):
        with pytest.raises(asca_b200.AscaError) as err:
            ops.clip_grads(gpu, [flat[2000:], flat[:2000]], 1.0, norm=norm)
        assert err.value.code == -1
    off, lr, eps = np.array([0, 1000]), np.float32([1e-3]), np.float32([1e-8])
    p, g, m, v = flat.view(4, 1000)
    for t in (p, m, v):
        with pytest.raises(asca_b200.AscaError) as err:
            ops.adamw_segmented(gpu, p, g, m, v, off, lr, eps, 0.9, 0.95, 0.0, norm=t[500:501], max_norm=1.0)
        assert err.value.code == -1
    assert torch.equal(flat, before)
    room = torch.zeros(9, device="cuda")   # right behind them is apart
    norm = ops.grad_norm(gpu, [room[:8]], out=room[8:])
    ops.clip_grads(gpu, [room[:8]], 1.0, norm=norm)
    assert not room.any()


# Calls whose shared memory differs, of two contexts on two threads (the C boundary lets go of the interpreter's lock).
def dispatch_call(g, e):
    n = 5000
    experts, ws = route(e, n, 1, e, "any"), torch.empty(g.lib.asca_moe_topk_dispatch_ws(n, 1, e), dtype=torch.uint8, device="cuda")
    out = [torch.empty(size, dtype=torch.int32, device="cuda") for size in (n, e + 1, n)]
    call = lambda: g._run("asca_moe_topk_dispatch", experts.data_ptr(), n, 1, e, *[t.data_ptr() for t in out], ws.data_ptr(), ws.numel())  # noqa: E731
    return call, out, (experts, ws)


def few_tokens_call(g, n):
    d = 64
    dx, ids, table = rand(1, n, d), text(2, n, 50_000, "zipf"), torch.empty(50_000, d, device="cuda")
    call = lambda: g._run("asca_embed_scaled_bwd", dx.data_ptr(), ids.data_ptr(), n, d, 50_000, 1.0, 0, 0, table.data_ptr(), None, 0)  # noqa: E731
    return call, [table], (dx, ids)


def join_call(g, cols):
    y, x, d_xn, d_x, d_y = (rand(i, 8, cols) for i in range(5))
    ws = torch.empty(g.lib.asca_gated_residual_rmsnorm_bwd_ws(g._ctx, 8, cols), dtype=torch.uint8, device="cuda")
    call = lambda: g._run("asca_gated_residual_rmsnorm_bwd", y.data_ptr(), x.data_ptr(), d_xn.data_ptr(), None, None, None, 0, None, 1, 1.0, 1.0, 1e-6, 8, cols,  # noqa: E731
                          asca_b200.F32, 0, d_x.data_ptr(), d_y.data_ptr(), None, None, None, ws.data_ptr(), ws.numel())
    return call, [d_x, d_y], (y, x, d_xn, ws)


@pytest.mark.parametrize("make,sizes", [(dispatch_call, (2048, 1400)), (few_tokens_call, (4096, 3000)), (join_call, (2048, 1400)), (join_call, (8192, 4500))])
def test_two_contexts_on_two_threads(gpu, make, sizes):
    contexts = [asca_b200.Gpu(0) for _ in sizes]
    calls = [make(g, size) for g, size in zip(contexts, sizes)]
    torch.cuda.synchronize()
    want = []
    for g, (call, out, _) in zip(contexts, calls):
        call()
        g.sync()
        want.append([t.clone() for t in out])
    torch.cuda.synchronize()
    errors = []

    def work(g, call):
        for _ in range(1500):
            try:
                call()
            except asca_b200.AscaError as e:
                errors.append(str(e))
        g.sync()

    threads = [threading.Thread(target=work, args=(g, c[0])) for g, c in zip(contexts, calls)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, f"{len(errors)} calls, the first: {errors[0]}"
    for (_, out, _), w in zip(calls, want):
        assert all(torch.equal(a, b) for a, b in zip(out, w))
    for g in contexts:
        g.close()


def test_sizes_are_refused_before_memory_is_taken(gpu):
    experts, ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    for bad in (1 << 28, 1 << 31, 1 << 40, (1 << 63) - 1):
        with pytest.raises(asca_b200.AscaError) as err:
            ops.moe_topk_dispatch(gpu, experts, bad)
        assert err.value.code == -1 and "experts" in str(err.value)
    dx = torch.zeros(4, 1, device="cuda")
    for bad in (1 << 31, 1 << 40, (1 << 63) - 1):
        with pytest.raises(asca_b200.AscaError) as err:
            ops.embed_bwd(gpu, dx, ids, bad)
        assert err.value.code == -1 and "shape" in str(err.value)
    assert torch.cuda.max_memory_allocated() - held < 1 << 20
    # the C boundary's own scratch size: a call of that many rows is refused
    for bad in (1 << 31, (1 << 63) - 1):
        assert gpu.lib.asca_gated_residual_rmsnorm_bwd_ws(gpu._ctx, bad, 8) < 0


@pytest.mark.parametrize("rows", [0, 1, 300])
def test_gate_rows_beyond_the_rows(gpu, rows):
    """One gate for all rows, however many more rows it would serve."""
    t, kw = join_case(max(rows, 1), 96, None, True, True, torch.float32)
    t.update(y=t["y"][:rows], x=t["x"][:rows], gate=t["gate"][:min(rows, 1)])
    d_xn = rand(7, rows, 96)
    want = None
    for per in (max(rows, 1), 1000, 1 << 31, 1 << 40, (1 << 63) - 1):
        kw["gate_rows"] = per
        x_out, xn = ops.gated_residual_rmsnorm_fwd(gpu, **t, **kw)
        got = ops.gated_residual_rmsnorm_bwd(gpu, t["y"], x_out, d_xn, None, gate=t["gate"], w_post=t["w_post"], w_pre=t["w_pre"], **kw)
        got = [x_out, xn, *got.values()]
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))


WITHOUT = """
import sys
sys.modules["asca_b200._torch_ops"] = None   # not there
import torch, asca_b200
from asca_b200 import ops
gpu = asca_b200.Gpu(0)
gpu.use_torch_stream()
a, b = torch.ones(64, 96, device="cuda"), torch.full((96, 32), 2.0, device="cuda")
assert (ops.gemm(gpu, a, b) == 192).all()
"""


def test_products_without_the_torch_binding():
    r = subprocess.run([sys.executable, "-c", WITHOUT], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


@pytest.mark.parametrize("K", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("d", [4, 40, 77, 1028])
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_assignments_go_anywhere(gpu, K, d, dtype):
    """Tokens with no assignment, one or all of them, side by side: where an assignment goes nowhere, nothing of its row is used."""
    N, E = 160, 7
    experts = route(K, N, K, E, "any")
    at = torch.arange(N * K, device="cuda").view(N, K)
    keep = torch.where((torch.arange(N, device="cuda") // 20 % 2 == 0).unsqueeze(1), at % 7 == 3, at % 3 != 0)   # thin and thick stretches
    keep[32:48] = False   # whole batches of none
    experts[~keep] = -1
    _, offsets, slot = ops.moe_topk_dispatch(gpu, experts, E)
    n = int(keep.sum())
    assert int(offsets[-1]) == n
    ys, weights, d_out = rand(1, N * K, d, dtype=dtype), rand(2, N, K), rand(3, N, d)
    ys[n:] = float("nan")
    weights[~keep] = float("nan")
    token, k = keep.nonzero(as_tuple=True)
    rows, w = ys.double()[slot[token, k].long()], weights.double()[token, k].unsqueeze(1)
    z = lambda: torch.zeros(N, d, dtype=torch.float64, device="cuda")  # noqa: E731
    mass = z().index_add_(0, token, (w * rows).abs())
    within(ops.moe_unsort_rows(gpu, ys, slot, weights), z().index_add_(0, token, w * rows), (K + 2) * U * mass, "out")
    d_ys, d_w = ops.moe_unsort_rows_bwd(gpu, d_out, ys, slot, weights, d_ys=torch.full_like(ys, 7.0))
    want = w * d_out.double()[token]
    within(d_ys[slot[token, k].long()], want, want.abs() * (torch.finfo(dtype).eps / 2 + 2 * U), "d_ys")
    assert (d_ys[n:] == 7).all() and not d_w[~keep].any()
    prod = rows * d_out.double()[token]
    within(d_w[keep], prod.sum(1), (d + 2) * U * prod.abs().sum(1), "d_w")
    for _ in range(5):
        alias = ys.clone()
        got = ops.moe_unsort_rows_bwd(gpu, d_out, alias, slot, weights, d_ys=alias)
        assert torch.equal(alias[:n], d_ys[:n]) and torch.equal(got[1], d_w) and alias[n:].isnan().all()


@pytest.mark.parametrize("rows,cols", [(1, 5), (37, 64), (150, 100), (9500, 33), (4800, 193), (33, 256), (7, 300), (4, 5000)])   # teams without a row, and strips that end early
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_residual_over_its_inputs(gpu, rows, cols, dtype):
    code = asca_b200.BF16 if dtype == torch.bfloat16 else asca_b200.F32
    y, x, d_xn, d_out = rand(1, rows, cols, dtype=dtype), rand(2, rows, cols), rand(3, rows, cols, dtype=dtype), rand(4, rows, cols)
    x_out, xn = ops.gated_residual_rmsnorm_fwd(gpu, y, x)
    want = ops.gated_residual_rmsnorm_bwd(gpu, y, x_out, d_xn, d_out)
    ws = torch.empty(gpu.lib.asca_gated_residual_rmsnorm_bwd_ws(gpu._ctx, rows, cols), dtype=torch.uint8, device="cuda")
    for _ in range(5):
        a, b = y.clone(), x.clone()
        gpu._run("asca_gated_residual_rmsnorm_fwd", a.data_ptr(), b.data_ptr(), None, None, 0, None, 1, 1.0, 1.0, 1e-6, rows, cols, code, b.data_ptr(), a.data_ptr())
        assert torch.equal(b, x_out) and torch.equal(a, xn)   # x_out over x, xn over y
        a, b = y.clone(), d_out.clone()
        gpu._run("asca_gated_residual_rmsnorm_bwd", a.data_ptr(), x_out.data_ptr(), d_xn.data_ptr(), b.data_ptr(), None, None, 0, None, 1, 1.0, 1.0, 1e-6, rows, cols,
                 code, 0, b.data_ptr(), a.data_ptr(), None, None, None, ws.data_ptr(), ws.numel())
        assert torch.equal(b, want["d_x"]) and torch.equal(a, want["d_y"])   # d_x over d_out, d_y over y


# Strips of many rows: several shared gates in one (20,000 x 260 has strips of 17 rows on 148 SMs, rounded up to whole groups), groups
# over two strips and more, and the narrowest and widest teams alike.
@pytest.mark.parametrize("rows,cols,per", [(20_000, 260, 3), (20_000, 260, 7), (20_000, 260, 20), (20_000, 260, 33), (20_000, 260, 35), (20_000, 260, 90), (40_001, 64, 3),
                                           (40_001, 50, 11), (30_000, 100, 2), (30_000, 193, 5), (30_000, 193, 26), (603, 8192, 3), (603, 8192, 7), (603, 8191, 19)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_several_gates_in_a_strip(gpu, rows, cols, per, dtype):
    check_join(gpu, rows, cols, per, True, True, dtype)


@pytest.mark.parametrize("rows,cols", [(40, 64), (300, 260), (2500, 33), (9, 5000)])
@pytest.mark.parametrize("per", [1, 3, None])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_a_gate_and_gains_that_are_ones(gpu, rows, cols, per, dtype):
    """A null gate or gain is ones; its gradient may be asked for all the same."""
    per = per or rows
    groups = -(-rows // per)
    y, x, d_xn, d_out = rand(1, rows, cols, dtype=dtype), rand(2, rows, cols), rand(3, rows, cols, dtype=dtype), rand(4, rows, cols)
    ones, gates = torch.ones(cols, device="cuda"), torch.ones(groups, cols, device="cuda")
    x_out, xn = ops.gated_residual_rmsnorm_fwd(gpu, y, x, gate=gates, gate_rows=per, w_post=ones, w_pre=ones, branch_scale=0.5)
    plain = ops.gated_residual_rmsnorm_fwd(gpu, y, x, branch_scale=0.5)
    assert torch.equal(plain[0], x_out) and torch.equal(plain[1], xn)
    want = ops.gated_residual_rmsnorm_bwd(gpu, y, x_out, d_xn, d_out, gate=gates, gate_rows=per, w_post=ones, w_pre=ones, branch_scale=0.5)
    d_x, d_y = torch.empty_like(x), torch.empty_like(y)
    sums = {"d_w_post": torch.full((cols,), 7.0, device="cuda"), "d_gate": torch.full((groups, cols), 7.0, device="cuda"), "d_w_pre": torch.full((cols,), 7.0, device="cuda")}
    ws = torch.empty(gpu.lib.asca_gated_residual_rmsnorm_bwd_ws(gpu._ctx, rows, cols), dtype=torch.uint8, device="cuda")
    gpu._run("asca_gated_residual_rmsnorm_bwd", y.data_ptr(), x_out.data_ptr(), d_xn.data_ptr(), d_out.data_ptr(), None, None, per, None, 1, 1.0, 0.5, 1e-6, rows, cols,
             asca_b200.BF16 if dtype == torch.bfloat16 else asca_b200.F32, 0, d_x.data_ptr(), d_y.data_ptr(), *[t.data_ptr() for t in sums.values()], ws.data_ptr(), ws.numel())
    assert torch.equal(d_x, want["d_x"]) and torch.equal(d_y, want["d_y"])
    # the same terms, d being d_x here; a gate a row takes another form of the kernel, which may order them otherwise
    yd, xd = y.double(), x_out.double()
    branch = (0.5 * d_x.double() * yd / torch.sqrt((yd * yd).mean(1, keepdim=True) + 1e-6)).abs()
    pre = (d_xn.double() * xd / torch.sqrt((xd * xd).mean(1, keepdim=True) + 1e-6)).abs()
    index = torch.arange(rows, device="cuda") // per
    mass = {"d_w_post": branch.sum(0), "d_gate": torch.zeros(groups, cols, dtype=torch.float64, device="cuda").index_add_(0, index, branch), "d_w_pre": pre.sum(0)}
    for name, got in sums.items():
        within(got, want[name].double(), 2.1 * ((min(per, rows) if name == "d_gate" else rows) + 40) * U * mass[name], name)


# The embedding's gradient in several launches, columns one by one: short runs, runs over many pieces joined by one and by several
# lanes beside each other, rows without a token, ids and rows that begin anywhere.
@pytest.mark.parametrize("N,V,d,kind", [(6000, 300, 193, "zipf"), (5000, 40, 777, "zipf"), (9000, 3, 1031, "zipf"), (4500, 1, 131, "one"), (20_000, 2, 67, "past"),
                                        (4097, 5000, 65, "distinct"), (300, 20_000, 1001, "zipf"), (6000, 900, 130, "padding"), (30_000, 7, 5, "zipf"), (5000, 70_001, 33, "zipf")])
@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_gradient_by_single_columns(gpu, N, V, d, kind, dtype):
    check_embedding(gpu, N, V, d, kind, dtype)


@pytest.mark.parametrize("N,V,d", [(6000, 300, 192), (9000, 4, 1024), (5000, 3000, 64)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_gradient_off_the_16_byte_grid(gpu, N, V, d, dtype):
    ids, dx = text(N, N, V, "zipf"), rand(2, N, d, dtype=dtype)
    want = ops.embed_bwd(gpu, dx, ids, V)
    live = ids[(ids >= 0) & (ids < V)].long()
    mass = torch.zeros(V, d, dtype=torch.float64, device="cuda").index_add_(0, live, dx[(ids >= 0) & (ids < V)].double().abs())
    count = torch.zeros(V, 1, dtype=torch.float64, device="cuda").index_add_(0, live, torch.ones(len(live), 1, dtype=torch.float64, device="cuda"))
    for got in (ops.embed_bwd(gpu, unaligned(dx), ids, V), ops.embed_bwd(gpu, dx, ids, V, d_table=unaligned(want)), ops.embed_bwd(gpu, unaligned(dx), unaligned(ids), V)):
        within(got, want.double(), 2 * (count + 2) * U * mass, "d_table")   # both sides off by as much from the sum


LITTLE_MEMORY = """
import resource
import numpy as np, torch, asca_b200
gpu = asca_b200.Gpu(0)
gpu.use_torch_stream()
count = 20_000_000
flat, norm = torch.ones(count, device="cuda"), torch.ones(1, device="cuda")
at, n, dtype = flat.data_ptr() + 4 * np.arange(count, dtype=np.uint64), np.ones(count, np.int64), np.zeros(count, np.int32)
torch.cuda.synchronize()
held = int(next(line for line in open("/proc/self/status") if line.startswith("VmSize")).split()[1]) * 1024
resource.setrlimit(resource.RLIMIT_AS, (held + (100 << 20), resource.RLIM_INFINITY))
try:
    gpu._run("asca_clip_grads", at.ctypes.data, n.ctypes.data, dtype.ctypes.data, count, norm.data_ptr(), 1.0)   # 320 MB of places
except asca_b200.AscaError as e:
    assert e.code == -3, e
else:
    raise SystemExit("not refused")
resource.setrlimit(resource.RLIMIT_AS, (resource.RLIM_INFINITY, resource.RLIM_INFINITY))
torch.cuda.synchronize()
assert (flat == 1).all()   # the context is usable
"""


def test_clipping_more_tensors_than_the_host_has_memory_for():
    """An error, not an exception through the C boundary, which would end the process."""
    r = subprocess.run([sys.executable, "-c", LITTLE_MEMORY], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_ids_of_either_type_and_any_shape(gpu):
    table, dx = rand(1, 50, 24), rand(2, 60, 24)
    ids = text(3, 60, 50, "zipf")
    x, g = ops.embed_fwd(gpu, table, ids, scale=2.0), ops.embed_bwd(gpu, dx, ids, 50, scale=2.0)
    unsigned = ids.view(torch.uint32)   # -1 is 2^32 - 1 there
    for shape in ((60,), (3, 20), (1, 5, 12), (60, 1)):
        for t in (ids, unsigned):
            assert torch.equal(ops.embed_fwd(gpu, table, t.view(shape), scale=2.0), x.view(*shape, 24))
            assert torch.equal(ops.embed_bwd(gpu, dx.view(*shape, 24), t.view(shape), 50, scale=2.0), g)
    one = ids[ids >= 0][0].view(())   # a single id
    assert torch.equal(ops.embed_fwd(gpu, table, one), table[int(one)]) and torch.equal(ops.embed_bwd(gpu, dx[0], one, 50)[int(one)], dx[0])


def test_parameters_and_inference_mode(gpu):
    """Tensors that autograd knows are data here; outputs know nothing of it."""
    t, kw = join_case(40, 96, 10, True, True, torch.float32)
    d_xn = rand(7, 40, 96)

    def step(t):
        x_out, xn = ops.gated_residual_rmsnorm_fwd(gpu, **t, **kw)
        got = ops.gated_residual_rmsnorm_bwd(gpu, t["y"], x_out, d_xn, None, gate=t["gate"], w_post=t["w_post"], w_pre=t["w_pre"], **kw)
        return [x_out, xn, *got.values(), *ops.moe_topk_dispatch(gpu, route(1, 40, 2, 5, "any"), 5), ops.grad_norm(gpu, list(got.values()))]

    want = step(t)
    for got in (step({k: torch.nn.Parameter(v) for k, v in t.items()}),):
        assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, want))
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(step(t), want))
    part = want[4]   # a gradient that shares an allocation is a tensor like any other
    part.mul_(2.0).requires_grad_()
    (part * part).sum().backward()
    assert torch.equal(part.grad, 2 * part.detach())


def test_accumulated_and_clipped_in_a_graph(gpu):
    """Each replay adds once more, and clips what is there."""
    n, v, d = 5000, 90, 40
    ids, dx = text(1, n, v, "zipf"), rand(2, n, d)
    t, kw = join_case(n, d, 300, True, True, torch.float32)
    d_xn = rand(3, n, d)
    stream = torch.cuda.Stream()
    table, loose = torch.zeros(v, d, device="cuda"), rand(4, 1000)
    sums = {"d_gate": torch.zeros_like(t["gate"]), "d_w_post": torch.zeros(d, device="cuda"), "d_w_pre": torch.zeros(d, device="cuda")}

    def step():
        ops.embed_bwd(gpu, dx, ids, v, d_table=table, accumulate=True)
        ops.gated_residual_rmsnorm_bwd(gpu, t["y"], t["x"], d_xn, None, gate=t["gate"], w_post=t["w_post"], w_pre=t["w_pre"], grads=sums, **kw)
        ops.clip_grads(gpu, [table, *sums.values(), loose], 1.0)

    held = [table, loose, *sums.values()]
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(stream):
            gpu.use_torch_stream()
            start = [h.clone() for h in held]
            for _ in range(3):
                step()
            want = [h.clone() for h in held]
            for h, s in zip(held, start):
                h.copy_(s)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step()
            for _ in range(3):
                graph.replay()
            stream.synchronize()
    finally:
        gpu.use_torch_stream()
    assert all(torch.equal(a, b) for a, b in zip(held, want)) and not torch.equal(want[0], start[0])

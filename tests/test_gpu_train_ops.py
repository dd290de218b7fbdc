"""The operators around the blocks of a training step: scaled embedding, gated residual with its norms, rows sorted by expert, the
gradient norm and the clipped optimizer step. Each against a plain statement in 64 bits.

Tolerances are bounds of the arithmetic, element by element: u = 2^-24 is the largest relative error of an f32 rounding, half a
step of the output's type that of the last one (2^-8 for bf16), and a sum of n terms is off by at most n u times the sum of
their magnitudes whatever its order. A norm's statistic is a sum of positive terms of at most 48 roundings in a row (eight a
thread, five in a warp, 32 warps, the division and the root), so its inverse root is off by at most 30 u.
"""
import ctypes as C

import numpy as np
import pytest
import torch

import asca_b200
from asca_b200 import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rand(seed, *shape, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def within(got, want, bound, what):
    """|got - want| <= bound everywhere (64-bit tensors; bound not negative)."""
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all(), what
    bad = off > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values, worst {float((off / bound.clamp_min(1e-300)).max()):.2f} times the bound"


def unaligned(t):
    """The same values behind an address that is one element off the 16-byte grid."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.reshape(-1)
    return flat[1:].view(t.shape)


# ------------------------------------------------------------------ embedding
def text(seed, n, v, kind):
    rng = np.random.default_rng(seed)
    if kind == "one":            # the same token all over: a run over every piece
        ids = np.full(n, v - 1)
    elif kind == "distinct":     # no token twice
        ids = rng.permutation(v)[:n]
    elif kind == "padding":
        ids = np.full(n, -1)
    else:
        p = 1.0 / np.arange(1, v + 1)
        ids = rng.choice(v, n, p=p / p.sum())
        ids[rng.random(n) < 0.1] = -1 if kind == "zipf" else v
    return torch.from_numpy(ids.astype(np.int32)).cuda()


EMBED = [  # N, V, d, ids
    (1, 1, 1, "one"), (1, 256, 64, "zipf"), (12, 256, 768, "zipf"), (63, 300, 7, "zipf"), (64, 64, 32, "one"), (65, 70, 33, "distinct"),
    (777, 5, 130, "zipf"), (2048, 256, 64, "zipf"), (2049, 2047, 36, "past"), (5000, 70_001, 20, "zipf"), (4096, 4_200_000, 1, "zipf"),
    (129, 100, 1030, "one"), (40_000, 3, 12, "zipf"), (300, 1000, 8, "padding"), (140_000, 50_000, 4, "zipf"),
    (1_100_000, 70_000, 2, "zipf"), (9000, 40, 1032, "zipf"), (20_000, 900, 40, "zipf"), (400, 90, 700, "zipf"), (2048, 31, 128, "zipf"),
]


@pytest.mark.parametrize("N,V,d,kind", EMBED)
@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_forward_and_gradient(gpu, N, V, d, kind, dtype):
    ids = text(N + V, N, V, kind)
    scale = np.float32(np.sqrt(d)).item()
    live = ((ids >= 0) & (ids < V)).nonzero().squeeze(1)
    at = ids[live].long()
    for table_dtype in DTYPES:
        table = rand(1, V, d, dtype=table_dtype)
        x = ops.embed_fwd(gpu, table, ids, scale=scale, out_dtype=dtype)
        want = torch.zeros(N, d, dtype=torch.float64, device="cuda")
        want[live] = scale * table.double()[at]
        within(x, want, want.abs() * (half_step(dtype) + 2 * U), f"x from {table_dtype}")
    dx = rand(2, N, d, dtype=dtype)
    want, mass, count = (torch.zeros(V, w, dtype=torch.float64, device="cuda") for w in (d, d, 1))
    want.index_add_(0, at, scale * dx.double()[live])
    mass.index_add_(0, at, abs(scale) * dx.double()[live].abs())
    count.index_add_(0, at, torch.ones(len(at), 1, dtype=torch.float64, device="cuda"))
    got = ops.embed_bwd(gpu, dx, ids, V, scale=scale)
    within(got, want, (count + 2) * U * mass, "d_table")
    again = ops.embed_bwd(gpu, dx, ids, V, scale=scale)
    assert torch.equal(got, again)
    before = rand(3, V, d)
    acc = ops.embed_bwd(gpu, dx, ids, V, scale=scale, d_table=before.clone(), accumulate=True)
    met = torch.zeros(V, dtype=torch.bool, device="cuda")
    met[at] = True
    assert torch.equal(acc[~met], before[~met])   # rows of tokens that do not occur are left as they were
    within(acc, before.double() + want, (count + 3) * U * (mass + before.double().abs()), "accumulated d_table")


@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_off_the_16_byte_grid(gpu, dtype):
    ids = text(4, 333, 50, "zipf")
    table, dx = rand(1, 50, 64, dtype=dtype), rand(2, 333, 64, dtype=dtype)
    x, g = ops.embed_fwd(gpu, table, ids, scale=3.0), ops.embed_bwd(gpu, dx, ids, 50)
    assert torch.equal(ops.embed_fwd(gpu, unaligned(table), ids, scale=3.0), x)
    assert torch.equal(ops.embed_fwd(gpu, table, ids, scale=3.0, out=unaligned(x)), x)
    assert torch.equal(ops.embed_bwd(gpu, unaligned(dx), ids, 50), g)
    assert torch.equal(ops.embed_bwd(gpu, dx, ids, 50, d_table=unaligned(g)), g)
    assert torch.equal(ops.embed_bwd(gpu, dx.view(3, 111, 64), ids.view(3, 111), 50), g)   # ids of any shape


def test_embedding_without_tokens(gpu):
    ids = torch.empty(0, dtype=torch.int32, device="cuda")
    assert ops.embed_fwd(gpu, rand(1, 9, 8), ids).shape == (0, 8)
    assert not ops.embed_bwd(gpu, rand(1, 0, 8), ids, 9).any()
    kept = rand(2, 9, 8)
    assert torch.equal(ops.embed_bwd(gpu, rand(1, 0, 8), ids, 9, d_table=kept.clone(), accumulate=True), kept)


def test_embedding_values_that_are_not_numbers_stay_in_their_rows(gpu):
    ids = text(5, 400, 30, "zipf")
    dx = rand(1, 400, 16)
    row = int(ids[ids >= 0][0])
    dx[(ids == row).nonzero()[0]] = float("nan")
    dx[ids < 0] = float("inf")   # padding
    g = ops.embed_bwd(gpu, dx, ids, 30)
    bad = ~torch.isfinite(g).all(1)
    assert bad.nonzero().flatten().tolist() == [row]


# ------------------------------------------------------------------ gated residual with its norms
def join64(y, x, gate, per, w_post, w_pre, post, skip, branch, eps):
    n = y
    if post:
        n = y / torch.sqrt((y * y).mean(1, keepdim=True) + eps)
        if w_post is not None:
            n = n * w_post
    if gate is not None:
        n = n * gate[torch.arange(y.shape[0], device=y.device) // per]
    x_out = skip * x + branch * n
    xn = x_out / torch.sqrt((x_out * x_out).mean(1, keepdim=True) + eps)
    return x_out, xn if w_pre is None else xn * w_pre


JOIN = [  # rows, cols, rows a gate (None: all), norm after the block, gains
    (1, 1, None, True, True), (1, 768, None, True, True), (12, 768, None, True, True), (5, 33, 2, True, True), (7, 64, 1, True, True),
    (100, 128, 10, True, True), (333, 193, 111, True, True), (64, 256, None, False, True), (50, 257, 7, True, False), (1000, 512, 1000, True, True),
    (901, 516, 300, True, True), (2500, 96, 1250, True, True), (4700, 40, 900, False, True), (20, 2048, 3, True, True), (300, 2052, 299, True, True),
    (40, 4099, 13, True, True), (31, 8192, None, True, True), (9, 8191, 4, False, False), (3000, 64, 5, True, True), (1200, 260, 2, True, True),
    (33, 5000, 1, True, True), (200, 8192, 1, True, True), (300, 4100, 120, True, True), (150, 6001, 50, False, True),
]


def join_case(rows, cols, per, post, gains, dtype, seed=0):
    per = per or rows
    t = dict(y=rand(seed + 1, rows, cols, scale=0.7, dtype=dtype), x=rand(seed + 2, rows, cols, scale=1.5), gate=1 + rand(seed + 3, -(-rows // per), cols, scale=0.3),
             w_post=1 + rand(seed + 4, cols, scale=0.2) if post and gains else None, w_pre=1 + rand(seed + 5, cols, scale=0.2) if gains else None)
    return t, dict(gate_rows=per, post_norm=post, skip_scale=0.75, branch_scale=0.5, eps=1e-6)


@pytest.mark.parametrize("rows,cols,per,post,gains", JOIN)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_residual_forward_and_gradients(gpu, rows, cols, per, post, gains, dtype):
    t, kw = join_case(rows, cols, per, post, gains, dtype)
    per = kw["gate_rows"]
    w = {k: None if v is None else v.double() for k, v in t.items()}
    x_out, xn = ops.gated_residual_rmsnorm_fwd(gpu, t["y"], t["x"], gate=t["gate"], w_post=t["w_post"], w_pre=t["w_pre"], **kw)
    want_x, want_n = join64(w["y"], w["x"], w["gate"], per, w["w_post"], w["w_pre"], post, 0.75, 0.5, 1e-6)
    a = (0.75 * w["x"]).abs() + (want_x - 0.75 * w["x"]).abs()
    within(x_out, want_x, 40 * U * a, "x_out")
    kappa = (a.norm(dim=1) / (want_x.norm(dim=1) + 1e-30)).unsqueeze(1)
    r2 = 1 / torch.sqrt((want_x * want_x).mean(1, keepdim=True) + 1e-6)
    gain = 1.0 if w["w_pre"] is None else w["w_pre"].abs()
    within(xn, want_n, want_n.abs() * (half_step(dtype) + (40 * kappa + 34) * U) + 42 * U * a * r2 * gain, "xn")

    # the backward pass is a function of y and of the x_out that the forward has left
    d_xn, d_out = rand(7, rows, cols, dtype=dtype), rand(8, rows, cols)
    xo, y = x_out.double(), w["y"]
    ones = torch.ones(cols, dtype=torch.float64, device="cuda")
    w_post, w_pre = (ones if w[k] is None else w[k] for k in ("w_post", "w_pre"))
    g = w["gate"][torch.arange(rows, device="cuda") // per]
    i1 = 1 / torch.sqrt((y * y).mean(1, keepdim=True) + 1e-6) if post else torch.ones(rows, 1, dtype=torch.float64, device="cuda")
    yh = y * i1
    i2 = 1 / torch.sqrt((xo * xo).mean(1, keepdim=True) + 1e-6)
    xh = xo * i2

    def through(dn, do):
        td = dn * w_pre
        d = do + i2 * (td - xh * (td * xh).mean(1, keepdim=True))
        D = do.abs() + i2 * (td.abs() + xh.abs() * (td * xh).abs().mean(1, keepdim=True))
        ud, A = 0.5 * g * d * w_post, (0.5 * g * w_post).abs() * D
        dy, dy_bound = (i1 * (ud - yh * (ud * yh).mean(1, keepdim=True)), 300 * U * i1 * (A + yh.abs() * (A * yh.abs()).mean(1, keepdim=True))) if post else (ud, 130 * U * A)
        n = yh * w_post
        index = torch.arange(rows, device="cuda") // per
        groups = w["gate"].shape[0]
        fold = lambda v: torch.zeros(groups, cols, dtype=torch.float64, device="cuda").index_add_(0, index, v)  # noqa: E731
        return {"d_x": (0.75 * d, 121 * U * 0.75 * D), "d_y": (dy, dy_bound + half_step(dtype) * (dy.abs() + dy_bound)),
                "d_gate": (fold(0.5 * d * n), (min(per, rows) + 200) * U * fold((0.5 * n).abs() * D)),
                "d_w_pre": ((dn * xh).sum(0), (rows + 80) * U * (dn * xh).abs().sum(0)),
                "d_w_post": ((0.5 * g * d * yh).sum(0), (rows + 300) * U * ((0.5 * g * yh).abs() * D).sum(0))}

    args = dict(gate=t["gate"], w_post=t["w_post"], w_pre=t["w_pre"], **kw)
    zero = torch.zeros(rows, cols, dtype=torch.float64, device="cuda")
    for dn, do in ((d_xn, d_out), (d_xn, None), (None, d_out)):
        want = through(zero if dn is None else dn.double(), zero if do is None else do.double())
        got = ops.gated_residual_rmsnorm_bwd(gpu, t["y"], x_out, dn, do, **args)
        assert set(got) == {"d_x", "d_y", "d_gate"} | ({"d_w_pre"} if gains else set()) | ({"d_w_post"} if gains and post else set())
        for name, v in got.items():
            within(v, *want[name], f"{name} from {'d_xn' if dn is not None else ''} {'d_out' if do is not None else ''}")
    got = ops.gated_residual_rmsnorm_bwd(gpu, t["y"], x_out, d_xn, d_out, **args)
    again = ops.gated_residual_rmsnorm_bwd(gpu, t["y"], x_out, d_xn, d_out, **args)
    assert all(torch.equal(v, again[k]) for k, v in got.items())
    sums = {k: rand(9, *v.shape) for k, v in got.items() if k not in ("d_x", "d_y")}
    acc = ops.gated_residual_rmsnorm_bwd(gpu, t["y"], x_out, d_xn, d_out, grads={k: v.clone() for k, v in sums.items()}, **args)
    for k, v in sums.items():
        within(acc[k], v.double() + got[k].double(), 2 * U * (v.double().abs() + got[k].double().abs()), f"accumulated {k}")


def test_gated_residual_gradient_against_differences(gpu):
    rows, cols, per = 37, 70, 10
    t, kw = join_case(rows, cols, per, True, True, torch.float32)
    a, b = rand(11, rows, cols), rand(12, rows, cols)
    x_out, _ = ops.gated_residual_rmsnorm_fwd(gpu, **t, **{k: v for k, v in kw.items()})
    got = ops.gated_residual_rmsnorm_bwd(gpu, t["y"], x_out, b, a, gate=t["gate"], w_post=t["w_post"], w_pre=t["w_pre"], **kw)

    def loss(s):
        xo, xn = join64(s["y"], s["x"], s["gate"], per, s["w_post"], s["w_pre"], True, 0.75, 0.5, 1e-6)
        return float((xo * a.double()).sum() + (xn * b.double()).sum())

    s = {k: v.double() for k, v in t.items()}
    h = 1e-5
    for name, out in (("y", "d_y"), ("x", "d_x"), ("gate", "d_gate"), ("w_post", "d_w_post"), ("w_pre", "d_w_pre")):
        step = rand(13, *t[name].shape).double()
        slope = (loss({**s, name: s[name] + h * step}) - loss({**s, name: s[name] - h * step})) / (2 * h)
        # the difference is exact to h^2; the gradient to a few hundred u of the magnitudes it sums
        assert abs(slope - float((got[out].double() * step).sum())) < 1e-4 * float((got[out].double() * step).abs().sum()), name


def test_gated_residual_in_place_and_off_the_grid(gpu):
    t, kw = join_case(300, 260, 100, True, True, torch.float32)
    x_out, xn = ops.gated_residual_rmsnorm_fwd(gpu, **t, **kw)
    x = t["x"].clone()
    same, _ = ops.gated_residual_rmsnorm_fwd(gpu, **{**t, "x": x}, x_out=x, **kw)
    assert same.data_ptr() == x.data_ptr() and torch.equal(x, x_out)
    off = {k: unaligned(v) for k, v in t.items()}
    xo2, xn2 = ops.gated_residual_rmsnorm_fwd(gpu, **off, **kw)   # other columns a thread: sums that are off by other roundings
    assert torch.allclose(xo2, x_out, rtol=0, atol=80 * U * 20) and torch.allclose(xn2, xn, rtol=0, atol=250 * U * 20)   # no value passes 20
    only, none = ops.gated_residual_rmsnorm_fwd(gpu, **t, want_norm=False, **kw)
    assert none is None and torch.equal(only, x_out)


def test_gated_residual_of_zeros_and_of_what_is_no_number(gpu):
    t, kw = join_case(8, 96, None, True, True, torch.float32)
    t["y"][2] = 0
    t["y"][5, 7] = float("nan")
    t["x"][2] = 0
    x_out, xn = ops.gated_residual_rmsnorm_fwd(gpu, **t, **kw)
    assert not x_out[2].any() and not xn[2].any()
    assert torch.isnan(x_out).any(1).nonzero().flatten().tolist() == [5] and torch.isnan(xn).any(1).nonzero().flatten().tolist() == [5]
    empty = ops.gated_residual_rmsnorm_fwd(gpu, rand(1, 0, 96), rand(1, 0, 96), w_pre=t["w_pre"])
    assert empty[0].shape == (0, 96)
    got = ops.gated_residual_rmsnorm_bwd(gpu, rand(1, 0, 96), rand(1, 0, 96), rand(1, 0, 96), None, w_pre=t["w_pre"], w_post=t["w_post"])
    assert not got["d_w_pre"].any() and not got["d_w_post"].any()


# ------------------------------------------------------------------ rows by expert
MOE = [  # N, K, E, d
    (1, 1, 1, 1), (1, 2, 16, 768), (12, 2, 16, 768), (33, 8, 8, 31), (500, 3, 5, 64), (1500, 2, 8, 192), (2048, 1, 64, 36), (2049, 4, 255, 20), (700, 5, 256, 17),
    (900, 2, 2048, 8), (40_000, 8, 128, 4), (3, 6, 7, 1028), (1_060_000, 1, 40, 1), (30_000, 3, 2048, 5), (1300, 1, 4, 2048),
    (1190, 3, 5, 264),
]


def route(seed, n, k, e, kind):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "same":
        experts = torch.zeros(n, k, dtype=torch.int32, device="cuda") + (e - 1)
    elif kind == "none":
        experts = torch.full((n, k), -1, dtype=torch.int32, device="cuda")
    else:
        experts = torch.randint(0, e, (n, k), generator=g, device="cuda", dtype=torch.int32)   # the same expert twice is allowed
        if kind == "padded":
            drop = torch.rand(n, k, generator=g, device="cuda") < 0.2
            experts[drop] = -1
            experts[0, 0] = e + 5 if n > 1 else -1
    return experts


@pytest.mark.parametrize("N,K,E,d", MOE)
@pytest.mark.parametrize("kind", ["any", "padded", "same", "none"])
def test_rows_by_expert(gpu, N, K, E, d, kind):
    experts = route(N + E, N, K, E, kind)
    perm, offsets, slot = ops.moe_topk_dispatch(gpu, experts, E)
    flat = experts.reshape(-1).cpu().numpy()
    live = (flat >= 0) & (flat < E)
    order = np.argsort(np.where(live, flat, E), kind="stable")
    n_live = int(live.sum())
    assert np.array_equal(perm.cpu().numpy(), order)
    assert np.array_equal(offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(np.bincount(flat[live], minlength=E)[:E])]))
    where = np.empty(N * K, np.int64)
    where[order] = np.arange(N * K)
    assert np.array_equal(slot.cpu().numpy().reshape(-1), np.where(live, where, -1))
    at = torch.from_numpy(order[:n_live]).cuda()
    token = at // K
    weights = rand(1, N, K)
    for tok, row in ((torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)):
        x, ys, d_out, d_xs = rand(2, N, d, dtype=tok), rand(3, N * K, d, dtype=row), rand(4, N, d, dtype=tok), rand(5, N * K, d, dtype=row)
        ys[n_live:] = float("nan")   # what lies behind the last expert's rows is not looked at
        d_xs[n_live:] = float("inf")
        xs = ops.moe_sort_rows(gpu, x, slot, out=torch.full((N * K, d), 7.0, dtype=row, device="cuda"))
        assert torch.equal(xs[:n_live], x[token].to(row)) and (xs[n_live:] == 7).all()
        z = lambda: torch.zeros(N, d, dtype=torch.float64, device="cuda")  # noqa: E731
        w = weights.reshape(-1)[at].double().unsqueeze(1)
        yl = ys[:n_live].double()
        for wt, ww in ((weights, w), (None, torch.ones_like(w))):
            out = ops.moe_unsort_rows(gpu, ys, slot, weights=wt, out_dtype=tok)
            want, mass = z().index_add_(0, token, ww * yl), z().index_add_(0, token, (ww * yl).abs())
            within(out, want, (K + 1) * U * mass + half_step(tok) * (want.abs() + (K + 1) * U * mass), "out")
        dx = ops.moe_sort_rows_bwd(gpu, d_xs, slot, out_dtype=tok)
        want, mass = z().index_add_(0, token, d_xs[:n_live].double()), z().index_add_(0, token, d_xs[:n_live].double().abs())
        within(dx, want, K * U * mass + half_step(tok) * (want.abs() + K * U * mass), "dx")
        d_ys, d_w = ops.moe_unsort_rows_bwd(gpu, d_out, ys, slot, weights, d_ys=torch.full((N * K, d), 7.0, dtype=row, device="cuda"))
        want = w * d_out[token].double()
        within(d_ys[:n_live], want, want.abs() * (U + half_step(row) * (1 + U)), "d_ys")
        assert (d_ys[n_live:] == 7).all()
        want, mass = (torch.zeros(N * K, dtype=torch.float64, device="cuda") for _ in range(2))
        prod = d_out[token].double() * yl
        want[at], mass[at] = prod.sum(1), prod.abs().sum(1)
        within(d_w.reshape(-1), want, (d + 2) * U * mass, "d_w")
        plain, none = ops.moe_unsort_rows_bwd(gpu, d_out, ys, slot, None)
        assert none is None and torch.equal(plain[:n_live], d_out[token].to(row))
        again = ops.moe_unsort_rows_bwd(gpu, d_out, ys, slot, weights)
        assert torch.equal(again[0][:n_live], d_ys[:n_live]) and torch.equal(again[1], d_w)
        alias = ys.clone()
        got = ops.moe_unsort_rows_bwd(gpu, d_out, alias, slot, weights, d_ys=alias)   # the gradient over the rows it is of
        assert torch.equal(alias[:n_live], d_ys[:n_live]) and torch.equal(got[1], d_w)


def test_rows_by_expert_off_the_16_byte_grid(gpu):
    experts = route(3, 70, 2, 6, "padded")
    _, offsets, slot = ops.moe_topk_dispatch(gpu, experts, 6)
    n = int(offsets[-1])
    x, ys, weights = rand(1, 70, 64), rand(2, 140, 64), rand(3, 70, 2)
    xs, out = ops.moe_sort_rows(gpu, x, slot), ops.moe_unsort_rows(gpu, ys, slot, weights)
    d_ys, d_w = ops.moe_unsort_rows_bwd(gpu, x, ys, slot, weights)
    assert torch.equal(ops.moe_sort_rows(gpu, unaligned(x), slot)[:n], xs[:n])
    assert torch.equal(ops.moe_sort_rows(gpu, x, slot, out=unaligned(xs))[:n], xs[:n])
    assert torch.equal(ops.moe_unsort_rows(gpu, unaligned(ys), slot, weights), out)
    got = ops.moe_unsort_rows_bwd(gpu, unaligned(x), unaligned(ys), slot, weights, d_ys=unaligned(d_ys))
    assert torch.equal(got[0][:n], d_ys[:n])
    within(got[1], d_w.double(), 2 * 66 * U * (x.abs().max().double() * ys.abs().max().double()) * 64, "d_w")


def test_rows_by_expert_without_tokens(gpu):
    perm, offsets, slot = ops.moe_topk_dispatch(gpu, torch.empty(0, 2, dtype=torch.int32, device="cuda"), 4)
    assert perm.numel() == 0 and not offsets.any() and slot.shape == (0, 2)
    assert ops.moe_sort_rows(gpu, rand(1, 0, 8), slot).shape == (0, 8)
    assert ops.moe_unsort_rows(gpu, rand(1, 0, 8), slot).shape == (0, 8)


def test_rows_by_expert_gradients_against_differences(gpu):
    n, k, e, d = 40, 3, 5, 24
    _, _, slot = ops.moe_topk_dispatch(gpu, route(1, n, k, e, "any"), e)
    ys, weights, a = rand(1, n * k, d), rand(2, n, k), rand(3, n, d)
    d_ys, d_w = ops.moe_unsort_rows_bwd(gpu, a, ys, slot, weights)
    loss = lambda yy, ww: float((ops.moe_unsort_rows(gpu, yy, slot, ww).double() * a.double()).sum())  # noqa: E731
    # linear in each argument: a whole step is the derivative, to the roundings of two forward passes
    sy, sw = rand(4, n * k, d), rand(5, n, k)
    mass = 16 * U * float(a.abs().double().sum()) * 40
    assert abs(loss(ys + sy, weights) - loss(ys, weights) - float((d_ys.double() * sy).sum())) < mass
    assert abs(loss(ys, weights + sw) - loss(ys, weights) - float((d_w.double() * sw).sum())) < mass


# ------------------------------------------------------------------ gradient norm and clipping
def tensors(seed, sizes, dtypes, scale=1.0):
    return [rand(seed + i, n, scale=scale, dtype=dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


NORMS = [([1], 1.0), ([0, 5, 0], 1.0), ([7, 64, 16384, 16385, 3], 1.0), ([100_003] * 3, 1e-3), ([33] * 161, 1.0), ([1] * 400, 1.0), ([3_000_001, 2], 1e-2)]


@pytest.mark.parametrize("sizes,scale", NORMS)
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float32, torch.bfloat16]])
def test_gradient_norm_and_clipping(gpu, sizes, scale, dtypes):
    grads = tensors(1, sizes, dtypes, scale)
    want = float(torch.sqrt(sum((g.double() ** 2).sum() for g in grads)))
    norm = ops.grad_norm(gpu, grads)
    assert abs(float(norm) - want) <= want * (U + 1e-12)
    assert torch.equal(norm, ops.grad_norm(gpu, grads))
    for max_norm in (0.3 * want, 0.0):
        clipped = [g.clone() for g in grads]
        back = ops.clip_grads(gpu, clipped, max_norm)
        assert torch.equal(back, norm)
        c = max_norm / (want + 1e-6)
        for g, got in zip(grads, clipped):
            exact = c * g.double()
            within(got, exact, exact.abs() * (half_step(g.dtype) + 6 * U), "clipped")
    loose = [g.clone() for g in grads]
    ops.clip_grads(gpu, loose, 2 * want + 1, norm=norm)
    assert all(torch.equal(a, b) for a, b in zip(loose, grads))


def test_gradient_norm_of_views_far_values_and_nothing(gpu):
    flat = rand(1, 50_000)
    cuts = [0, 1, 6, 6, 777, 17_171, 50_000]   # views that begin anywhere
    views = [flat[a:b] for a, b in zip(cuts, cuts[1:])]
    want = float(flat.double().norm())
    assert abs(float(ops.grad_norm(gpu, views)) - want) <= want * (U + 1e-12)
    ops.clip_grads(gpu, views, 1.0)
    assert abs(float(ops.grad_norm(gpu, [flat])) - 1.0) < 8 * U + 2e-6 / want
    half = rand(2, 999, dtype=torch.bfloat16)
    want = float(half[1:].double().norm())
    assert abs(float(ops.grad_norm(gpu, [half[1:]])) - want) <= want * (U + 1e-12)
    for v in (1e30, 1e-30):   # squares beyond f32 on either side
        far = torch.full((1000,), v, device="cuda")
        want = float(far.double().norm())
        assert abs(float(ops.grad_norm(gpu, [far])) - want) <= want * (U + 1e-12)
    assert float(ops.grad_norm(gpu, [])) == 0.0
    assert float(ops.grad_norm(gpu, [torch.zeros(5, device="cuda")])) == 0.0
    assert np.isinf(float(ops.grad_norm(gpu, [torch.tensor([1.0, float("inf")], device="cuda")])))
    bad = torch.tensor([1.0, float("nan")], device="cuda")
    assert np.isnan(float(ops.clip_grads(gpu, [bad], 1.0))) and torch.isnan(bad).all()


@pytest.mark.parametrize("n_seg", [3, 200])
def test_clipped_adamw_is_adamw_on_the_clipped_gradient(gpu, n_seg):
    rng = np.random.default_rng(5)
    off = np.concatenate([[0], np.cumsum(rng.integers(1, 400, n_seg))]).astype(np.int64)
    n = int(off[-1])
    lr_t, eps_t = np.full(n_seg, 1e-3, np.float32), np.full(n_seg, 1e-8, np.float32)
    g, p, m = rand(1, n), rand(2, n), rand(3, n, scale=0.1)
    v = rand(4, n).square()
    norm = ops.grad_norm(gpu, [g])
    for max_norm in (0.5, 1e6):
        a, b = ([t.clone() for t in (p, m, v)] for _ in range(2))
        kept = g.clone()
        ops.adamw_segmented(gpu, a[0], g, a[1], a[2], off, lr_t, eps_t, 0.9, 0.95, 1e-4, norm=norm, max_norm=max_norm)
        c = (max_norm / (norm + 1e-6)).clamp(max=1.0)
        ops.adamw_segmented(gpu, b[0], g * c, b[1], b[2], off, lr_t, eps_t, 0.9, 0.95, 1e-4)
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(g, kept)


@pytest.mark.parametrize("compute", [asca_b200.F32, asca_b200.BF16])
def test_model_step_that_clips(gpu, compute):
    cfg = (256, 64, 2, 2, 4, 64)
    rng = np.random.default_rng(3)
    models = [asca_b200.Model(gpu, *cfg) for _ in range(2)]
    params = rng.normal(0, 0.05, models[0].n).astype(np.float32)
    ids, targets = (rng.integers(0, 256, 256).astype(np.uint32) for _ in range(2))
    for m in models:
        m.set_compute(compute)
        m.set_params(params)
        m.zero_grads()
        m.forward_backward(ids, targets, 4)
    grads = models[0].get()[1]
    want = np.sqrt((grads.astype(np.float64) ** 2).sum())
    assert abs(models[0].grad_norm() - want) <= want * (U + 1e-12)
    assert abs(models[0].adamw_step_clip(1e-3, 0.25 * want) - want) <= want * (U + 1e-12)
    assert np.array_equal(models[0].get()[1], grads)   # the buffer stays
    norm = np.float32(want)
    models[1].set_grads(grads * np.float32(np.float32(0.25 * want) / np.float32(norm + np.float32(1e-6))))
    models[1].adamw_step(1e-3)
    assert np.array_equal(models[0].get()[0], models[1].get()[0])
    assert models[0].adamw_step_clip(1e-3, 1e9, want_norm=False) is None
    for m in models:
        m.zero_grads()
    assert models[0].grad_norm() == 0.0
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(asca_b200.AscaError):
            models[0].adamw_step_clip(1e-3, bad)
    for m in models:
        m.free()


# ------------------------------------------------------------------ together, captured, refused
def test_a_training_step_of_a_mixture_of_experts(gpu):
    """ids -> scaled embedding -> join -> two experts a token -> join -> head -> loss, its gradients and the clipped update."""
    N, V, d, E, K, F = 96, 130, 64, 4, 2, 128
    ids, targets = text(1, N, V, "zipf"), (text(2, N, V, "distinct") % V)
    scale = 8.0
    P = dict(table=rand(1, V, d, scale=0.1), w1=rand(2, d, E * F, scale=0.1), b1=rand(3, E * F, scale=0.1), w2=rand(4, E * F, d, scale=0.1), b2=rand(5, d, scale=0.1),
             head=rand(6, d, V, scale=0.1), gate=1 + rand(7, 3, d, scale=0.1), w_post=1 + rand(8, d, scale=0.1), w_pre=1 + rand(9, d, scale=0.1))
    experts = route(5, N, K, E, "any")
    experts[ids < 0] = -1
    weights = torch.softmax(rand(10, N, K), 1).contiguous()
    ident = torch.arange(N * K, dtype=torch.int32, device="cuda")

    x0 = ops.embed_fwd(gpu, P["table"], ids, scale=scale)
    xn = ops.rmsnorm_fwd(gpu, x0)
    perm, offsets, slot = ops.moe_topk_dispatch(gpu, experts, E)
    xs = ops.moe_sort_rows(gpu, xn, slot, out=torch.zeros(N * K, d, device="cuda"))
    ys, pre, hid = ops.moe_fwd(gpu, xs, P["w1"], P["b1"], P["w2"], P["b2"], ident, offsets, F, E)
    y = ops.moe_unsort_rows(gpu, ys, slot, weights=weights)
    kw = dict(gate=P["gate"], gate_rows=32, w_post=P["w_post"], w_pre=P["w_pre"], skip_scale=0.9, branch_scale=0.5)
    x1, h = ops.gated_residual_rmsnorm_fwd(gpu, y, x0, **kw)
    logits = ops.gemm(gpu, h, P["head"])
    dlogits, loss = torch.empty_like(logits), torch.empty(1, device="cuda")
    gpu._call("asca_cross_entropy", gpu._ctx, *[C.c_void_p(t.data_ptr()) for t in (logits, targets)], C.c_int64(N), C.c_int64(V), C.c_void_p(dlogits.data_ptr()),
              C.c_void_p(loss.data_ptr()))
    got = {"head": ops.gemm(gpu, h, dlogits, mode=asca_b200.TN)}
    j = ops.gated_residual_rmsnorm_bwd(gpu, y, x1, ops.gemm(gpu, dlogits, P["head"], mode=asca_b200.NT), None, **kw)
    got.update(gate=j["d_gate"], w_post=j["d_w_post"], w_pre=j["d_w_pre"])
    d_ys, d_weights = ops.moe_unsort_rows_bwd(gpu, j["d_y"], ys, slot, weights, d_ys=torch.zeros_like(ys))
    got["w1"], got["b1"], got["w2"], got["b2"], d_xs = ops.moe_bwd(gpu, xs, P["w1"], P["w2"], pre, hid, d_ys, ident, offsets, F, E)
    d_x0 = j["d_x"] + ops.rmsnorm_bwd(gpu, x0, ops.moe_sort_rows_bwd(gpu, d_xs, slot))
    got["table"] = ops.embed_bwd(gpu, d_x0, ids, V, scale=scale)

    Q = {k: v.double().requires_grad_() for k, v in P.items()}
    wq = weights.double().requires_grad_()
    live = (ids >= 0).unsqueeze(1)
    x0q = torch.where(live, scale * Q["table"][ids.clamp_min(0).long()], 0.0)
    xnq = x0q / torch.sqrt((x0q ** 2).mean(1, keepdim=True) + 1e-6)
    yq = torch.zeros(N, d, dtype=torch.float64, device="cuda")
    for k in range(K):
        for e in range(E):
            t = (experts[:, k] == e).nonzero().squeeze(1)
            hidden = torch.nn.functional.silu(xnq[t] @ Q["w1"][:, e * F:(e + 1) * F] + Q["b1"][e * F:(e + 1) * F])
            yq = yq.index_add(0, t, wq[t, k:k + 1] * (hidden @ Q["w2"][e * F:(e + 1) * F] + Q["b2"]))
    _, hq = join64(yq, x0q, Q["gate"], 32, Q["w_post"], Q["w_pre"], True, 0.9, 0.5, 1e-6)
    lossq = torch.nn.functional.cross_entropy(hq @ Q["head"], targets.long())
    lossq.backward()

    def rel(a, b):
        return float((a.double() - b).abs().max() / b.abs().max())

    # the framework's bound of its f32 mode
    lossq = float(lossq.detach())
    assert abs(float(loss) - lossq) < 1e-5 * lossq
    assert rel(d_weights, wq.grad) < 1e-5
    for k, v in got.items():
        assert rel(v, Q[k].grad) < 1e-5, k

    names = list(P)
    flat, grad = torch.cat([P[k].reshape(-1) for k in names]), torch.cat([got[k].reshape(-1) for k in names])
    norm = ops.grad_norm(gpu, [got[k] for k in names])
    want = float(torch.sqrt(sum((Q[k].grad ** 2).sum() for k in names)))
    assert abs(float(norm) - want) < 1e-5 * want
    off = np.concatenate([[0], np.cumsum([P[k].numel() for k in names])]).astype(np.int64)
    m, v, before = torch.zeros_like(flat), torch.zeros_like(flat), flat.clone()
    ops.adamw_segmented(gpu, flat, grad, m, v, off, np.full(len(names), 1e-3, np.float32), np.full(len(names), 1e-8, np.float32), 0.9, 0.95, 0.0, norm=norm,
                        max_norm=0.1 * want)
    assert not torch.equal(flat, before) and abs(float(m.norm()) - 0.1 * 0.1 * want) < 1e-4 * want


def step_of(gpu, s):
    """Every operator once, on the tensors of `s`; outputs in `s["out"]`."""
    o = {"x": ops.embed_fwd(gpu, s["table"], s["ids"], scale=2.0), "d_table": ops.embed_bwd(gpu, s["x"], s["ids"], 500, scale=2.0)}
    o["x_out"], o["xn"] = ops.gated_residual_rmsnorm_fwd(gpu, s["y"], s["x"], gate=s["gate"], gate_rows=100, w_pre=s["w"])
    o.update(ops.gated_residual_rmsnorm_bwd(gpu, s["y"], o["x_out"], s["x"], s["y"], gate=s["gate"], gate_rows=100, w_pre=s["w"]))
    o["perm"], o["offsets"], o["slot"] = ops.moe_topk_dispatch(gpu, s["experts"], 8)
    o["xs"] = ops.moe_sort_rows(gpu, s["x"], o["slot"])
    o["back"] = ops.moe_unsort_rows(gpu, o["xs"], o["slot"], s["weights"])
    o["d_ys"], o["d_w"] = ops.moe_unsort_rows_bwd(gpu, s["y"], o["xs"], o["slot"], s["weights"])
    o["norm"] = ops.grad_norm(gpu, [o["d_table"], o["d_x"], o["d_gate"]])
    o["p"], o["m"], o["v"] = s["p"].clone(), torch.zeros_like(s["p"]), torch.zeros_like(s["p"])
    ops.adamw_segmented(gpu, o["p"], o["d_table"], o["m"], o["v"], np.array([0, 500 * 200]), np.float32([1e-3]), np.float32([1e-8]), 0.9, 0.95, 0.0, norm=o["norm"],
                        max_norm=1.0)
    s["out"] = o


def state_of(seed, n=700):
    d = 200
    return dict(table=rand(seed, 500, d), ids=text(seed, n, 500, "zipf"), x=rand(seed + 1, n, d), y=rand(seed + 2, n, d), gate=rand(seed + 3, n // 100, d), w=rand(seed + 4, d),
                experts=route(seed, n, 2, 8, "any"), weights=rand(seed + 5, n, 2), p=rand(seed + 6, 500, d))


@pytest.mark.parametrize("n", [700, 9000])   # sorted in one launch, in several
def test_captured_and_replayed_beside_each_other(gpu, n):
    """Two graphs of one context, replayed on two streams at once with new inputs: each has scratch of its own."""
    states, graphs, streams = [state_of(10, n), state_of(20, n)], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    try:
        for s, stream in zip(states, streams):
            with torch.cuda.stream(stream):
                gpu.use_torch_stream()
                step_of(gpu, s)   # loads the kernels
                stream.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    step_of(gpu, s)
                graphs.append(graph)
        gpu.use_torch_stream()
        for seed in (30, 40):
            fresh = [state_of(seed, n), state_of(seed + 5, n)]
            want = []
            for f in fresh:
                step_of(gpu, f)
                want.append(f["out"])
            for s, f in zip(states, fresh):
                for k, v in f.items():
                    if k != "out":
                        s[k].copy_(v)
            torch.cuda.synchronize()
            for _ in range(20):
                for graph, stream in zip(graphs, streams):
                    with torch.cuda.stream(stream):
                        graph.replay()
            torch.cuda.synchronize()
            for s, w in zip(states, want):
                for k, v in w.items():
                    assert torch.equal(s["out"][k], v), k
    finally:
        torch.cuda.synchronize()
        gpu.use_torch_stream()


def test_refusals(gpu):
    ids, x = text(1, 10, 20, "zipf"), rand(1, 10, 8)
    slot = torch.zeros(10, 2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        ops.embed_fwd(gpu, x.cpu(), ids)
    with pytest.raises(TypeError):
        ops.embed_fwd(gpu, x.half(), ids)
    with pytest.raises(TypeError):
        ops.embed_fwd(gpu, x, ids.long())
    with pytest.raises(ValueError):
        ops.embed_fwd(gpu, x.t(), ids)
    with pytest.raises(ValueError):
        ops.embed_bwd(gpu, x[:9], ids, 20)
    with pytest.raises(ValueError):
        ops.embed_bwd(gpu, x, ids, 20, accumulate=True)
    with pytest.raises(ValueError):
        ops.embed_bwd(gpu, x, ids, 20, d_table=rand(1, 19, 8))
    with pytest.raises(ValueError):
        ops.gated_residual_rmsnorm_fwd(gpu, x, x, gate=rand(1, 3, 8), gate_rows=2)
    with pytest.raises(ValueError):
        ops.gated_residual_rmsnorm_fwd(gpu, x, x, w_post=rand(1, 8), post_norm=False)
    with pytest.raises(TypeError):
        ops.gated_residual_rmsnorm_fwd(gpu, x, x.bfloat16())
    with pytest.raises(ValueError):
        ops.gated_residual_rmsnorm_bwd(gpu, x, x, None, None)
    with pytest.raises(asca_b200.AscaError) as err:
        ops.gated_residual_rmsnorm_fwd(gpu, rand(1, 1, 8193), rand(1, 1, 8193))
    assert err.value.code == -4 and "8192" in str(err.value)
    for e in (0, 2049):
        with pytest.raises(asca_b200.AscaError) as err:
            ops.moe_topk_dispatch(gpu, slot, e)
        assert err.value.code == -1 and "experts" in str(err.value)
    with pytest.raises(ValueError):
        ops.moe_sort_rows(gpu, x[:9], slot)
    with pytest.raises(ValueError):
        ops.moe_unsort_rows(gpu, x, slot)
    with pytest.raises(ValueError):
        ops.moe_unsort_rows(gpu, rand(1, 20, 8), slot, weights=rand(1, 10, 3))
    with pytest.raises(ValueError):
        ops.adamw_segmented(gpu, x, x, x, x, [0, 80], [1e-3], [1e-8], 0.9, 0.95, 0.0, norm=rand(1, 1))
    with pytest.raises(asca_b200.AscaError):
        ops.clip_grads(gpu, [x.view(-1), x.view(-1)[5:]], 1.0)
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(asca_b200.AscaError):
            ops.clip_grads(gpu, [x], bad)
    # scratch that is too small, through the C boundary
    n = 40_000
    many, rows, table, out = text(1, n, 20, "zipf"), rand(1, n, 8), rand(1, 20, 8), torch.empty(2 * n + 9, dtype=torch.int32, device="cuda")
    calls = {"asca_embed_scaled_bwd": (gpu.lib.asca_embed_scaled_bwd_ws(n, 8, 20), lambda at, size: gpu._run(
                 "asca_embed_scaled_bwd", rows.data_ptr(), many.data_ptr(), n, 8, 20, 1.0, asca_b200.F32, 0, table.data_ptr(), at, size)),
             "asca_moe_topk_dispatch": (gpu.lib.asca_moe_topk_dispatch_ws(n, 1, 8), lambda at, size: gpu._run(
                 "asca_moe_topk_dispatch", many.data_ptr(), n, 1, 8, out.data_ptr(), out.data_ptr() + 4 * n, out.data_ptr() + 4 * n + 36, at, size))}
    for nbytes, call in calls.values():
        ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        for at, size in ((ws.data_ptr(), nbytes - 1), (ws.data_ptr() + 4, nbytes), (0, 0), (0, nbytes)):
            with pytest.raises(asca_b200.AscaError) as err:
                call(at, size)
            assert err.value.code == -1
        call(ws.data_ptr(), nbytes)
    # a context on another stream than torch's current one
    with torch.cuda.stream(torch.cuda.Stream()):
        with pytest.raises(RuntimeError, match="use_torch_stream"):
            ops.embed_fwd(gpu, x, ids)
    assert torch.equal(ops.moe_unsort_rows(gpu, rand(1, 20, 8) * 0, slot), torch.zeros(10, 8, device="cuda"))   # the context is usable


def test_outputs_over_inputs(gpu):
    """In place where whoever writes an element has read it; refused elsewhere."""
    n, d = 12, 16
    buf, ids = rand(1, 4 * n * d), text(1, n, 8, "zipf")
    part = lambda at, rows: buf[at:at + rows * d].view(rows, d)  # noqa: E731
    _, _, slot = ops.moe_topk_dispatch(gpu, route(1, n, 1, 3, "any"), 3)
    w = rand(2, n, 1)
    refused = [
        lambda: ops.embed_fwd(gpu, part(0, n), ids, out=part(d, n)),
        lambda: ops.embed_bwd(gpu, part(0, n), ids, 8, d_table=part(5 * d, 8)),
        lambda: ops.moe_sort_rows(gpu, part(0, n), slot, out=part(0, n)),
        lambda: ops.moe_unsort_rows(gpu, part(0, n), slot, w, out=part(0, n)),
        lambda: ops.moe_unsort_rows_bwd(gpu, part(0, n), part(n * d, n), slot, w, d_ys=part(0, n)),
        lambda: ops.moe_unsort_rows_bwd(gpu, part(2 * n * d, n), part(0, n), slot, w, d_ys=part(d, n)),
        lambda: ops.gated_residual_rmsnorm_fwd(gpu, part(0, n), part(n * d, n), x_out=part(n * d + 4, n)),
        lambda: ops.gated_residual_rmsnorm_fwd(gpu, part(0, n), part(n * d, n), w_pre=buf[2 * n * d:][:d], x_out=part(2 * n * d, n)),
    ]
    gain, grad = rand(3, d), rand(4, d)   # one parameter in both places: its gradient would be added to by two sums at once
    refused.append(lambda: ops.gated_residual_rmsnorm_bwd(gpu, part(0, n), part(n * d, n), part(2 * n * d, n), None, w_post=gain, w_pre=gain,
                                                          grads={"d_w_post": grad, "d_w_pre": grad}))
    before = buf.clone()
    for call in refused:
        with pytest.raises(asca_b200.AscaError) as err:
            call()
        assert err.value.code == -1
    assert torch.equal(buf, before)
    both = ops.gated_residual_rmsnorm_bwd(gpu, part(0, n), part(n * d, n), part(2 * n * d, n), None, w_post=gain, w_pre=gain)
    y, x, d_xn = (part(i * n * d, n).clone() for i in range(3))
    gpu._run("asca_gated_residual_rmsnorm_bwd", y.data_ptr(), x.data_ptr(), d_xn.data_ptr(), None, gain.data_ptr(), None, 0, gain.data_ptr(), 1, 1.0, 1.0, 1e-6,
             n, d, asca_b200.F32, 0, x.data_ptr(), d_xn.data_ptr(), None, None, None,
             (ws := torch.empty(gpu.lib.asca_gated_residual_rmsnorm_bwd_ws(gpu._ctx, n, d), dtype=torch.uint8, device="cuda")).data_ptr(), ws.numel())
    assert torch.equal(x, both["d_x"]) and torch.equal(d_xn, both["d_y"])   # d_x over x_out, d_y over d_xn


def test_slots_that_are_none(gpu):
    slot = torch.tensor([[0, 99], [-7, 3], [1, 2]], dtype=torch.int32, device="cuda")   # six rows: 99 and -7 go nowhere
    x, ys, w = rand(1, 3, 8), rand(2, 6, 8), rand(3, 3, 2)
    xs = ops.moe_sort_rows(gpu, x, slot, out=torch.full((6, 8), 7.0, device="cuda"))
    assert torch.equal(xs[:4], x[[0, 2, 2, 1]]) and (xs[4:] == 7).all()
    out = ops.moe_unsort_rows(gpu, ys, slot, w)
    assert torch.equal(out[0], w[0, 0] * ys[0]) and torch.equal(out[1], w[1, 1] * ys[3])
    d_ys, d_w = ops.moe_unsort_rows_bwd(gpu, x, ys, slot, w, d_ys=torch.full((6, 8), 7.0, device="cuda"))
    assert torch.equal(d_ys[0], w[0, 0] * x[0]) and (d_ys[4:] == 7).all() and d_w[0, 1] == 0 and d_w[1, 0] == 0


def test_gradients_that_only_an_iterator_holds(gpu):
    grads = tensors(1, [50_000] * 40, [torch.float32])
    kept = [g * 2 for g in grads]
    assert torch.equal(ops.grad_norm(gpu, (g * 2 for g in grads)), ops.grad_norm(gpu, kept))
    norm = ops.clip_grads(gpu, iter(kept), 1.0)
    within(kept[3], grads[3].double() * 2 / float(norm), (6 * U) * grads[3].double().abs() * 2 / float(norm) + 1e-6 * 2 * grads[3].double().abs() / float(norm) ** 2, "clipped")


def test_matrices_of_more_than_2_31_elements(gpu):
    """What the last rows get is what they get alone."""
    cols, rows = 2048, (1 << 31) // 2048 + 70
    last = slice(rows - 50, rows)
    y = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_()
    x = torch.empty(rows, cols, device="cuda").normal_()
    kw = dict(w_post=rand(1, cols), w_pre=rand(2, cols), skip_scale=0.9, branch_scale=0.3)
    alone = ops.gated_residual_rmsnorm_fwd(gpu, y[last], x[last].clone(), **kw)
    x_out, xn = ops.gated_residual_rmsnorm_fwd(gpu, y, x, x_out=x, **kw)
    assert torch.equal(x_out[last], alone[0]) and torch.equal(xn[last], alone[1])
    got = ops.gated_residual_rmsnorm_bwd(gpu, y, x_out, xn, None, **kw)
    want = ops.gated_residual_rmsnorm_bwd(gpu, y[last], x_out[last], xn[last], None, **kw)
    assert torch.equal(got["d_x"][last], want["d_x"]) and torch.equal(got["d_y"][last], want["d_y"])
    del x, x_out, got, want
    # the same matrix as a table, as rows in expert order, and as rows of gradients
    ids = torch.randint(rows - 40, rows, (33,), dtype=torch.int32, device="cuda")
    assert torch.equal(ops.embed_fwd(gpu, y, ids), y[ids.long()])
    experts = torch.zeros(rows, 1, dtype=torch.int32, device="cuda")
    experts[:rows // 2] = 1
    _, _, slot = ops.moe_topk_dispatch(gpu, experts, 2)
    xs = ops.moe_sort_rows(gpu, y, slot, out=xn)
    half = rows - rows // 2
    assert torch.equal(xs[half:], y[:rows // 2]) and torch.equal(xs[:half], y[rows // 2:])
    back = ops.moe_unsort_rows(gpu, xs, slot, out_dtype=torch.bfloat16)
    assert torch.equal(back, y)
    del back
    d_ys, d_w = ops.moe_unsort_rows_bwd(gpu, y, xs, slot, torch.ones(rows, 1, device="cuda"), d_ys=xs)
    assert torch.equal(d_ys[:half], y[rows // 2:])
    square = (y[last].double() ** 2).sum(1)
    within(d_w[last, 0], square, (cols + 2) * U * square, "d_w")
    ids = torch.randint(0, 1000, (rows,), dtype=torch.int32, device="cuda")
    ids[:-50] = -1   # (padding: nothing but the last rows is summed)
    ids[-50:] = torch.arange(50, dtype=torch.int32, device="cuda")
    assert torch.equal(ops.embed_bwd(gpu, y, ids, 1000)[:50], y[last].float())
    norm = ops.grad_norm(gpu, [y])
    want = float(torch.sqrt(sum((part.double() ** 2).sum() for part in y.split(1 << 17))))
    assert abs(float(norm) - want) <= want * (U + 1e-10)


def test_another_context_on_another_stream(gpu):
    other, stream = asca_b200.Gpu(0), torch.cuda.Stream()
    a, b = state_of(50), state_of(60)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        other.use_torch_stream()
        step_of(other, b)
    step_of(gpu, a)
    torch.cuda.synchronize()
    for s in (a, b):
        got = s["out"]
        step_of(gpu, s)
        for k, v in s["out"].items():
            assert torch.equal(got[k], v), k
    other.close()

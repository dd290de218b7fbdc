"""The operators around the expert layer and the two ends of a training step, as cases that can be timed one by one.

``run`` is one pass. With ``own`` false it computes the operators from elementary torch operations in 32 bits; with ``own``
true it makes the calls that a user of asca_b200 makes. ``exact`` states the same results in 64 bits. Kinds of work:

* ``embed``  rows of a scaled embedding table by token, and the table's gradient by sorted tokens
* ``join``   norm after a block, its gate, the scaled residual and the norm before the next block, and their gradients
* ``moe``    tokens sorted by expert, the rows moved there and back with the router's weights, and the gradients
* ``clip``   the gradient norm over many tensors, and the AdamW step that clips by it

Padding tokens carry id -1 (``embed``) or expert -1 (``moe``).
"""
import math

import numpy as np
import torch

own = False

#: vocab, d, heads, blocks, experts, expert width
MODELS = {
    "331k": (256, 64, 4, 2, 4, 256),              # the CPU-runnable model
    "12.7m": (256, 192, 6, 6, 8, 640),            # the small training run
    "1.3b-block": (256, 2048, 16, 1, 64, 4096),   # one block of the training configuration
}
EPS = 1e-6
ADAM = dict(lr=3e-4, beta1=0.9, beta2=0.95, eps=1e-8, wd=0.01)


def listed():
    return [
        # a serving step of a dozen streams: one token each, pure latency
        {"name": "embed_decode_f32", "kind": "embed", "dtype": "f32", "N": 12, "V": 256, "d": 768, "pad": 0.0, "bwd": False},
        # the smallest training step: 16 sequences of 128 bytes, every row of the table met eight times
        {"name": "embed_train_331k_f32", "kind": "embed", "dtype": "f32", "N": 2048, "V": 256, "d": 64, "pad": 0.0, "bwd": True},
        # 8 sequences of 4096 tokens of a large vocabulary, frequent tokens by the thousand, one in twenty of them padding
        {"name": "embed_train_vocab_bf16", "kind": "embed", "dtype": "bf16", "N": 32768, "V": 48000, "d": 2048, "pad": 0.05, "bwd": True},
        # the join behind a block in a serving step
        {"name": "join_decode_bf16", "kind": "join", "dtype": "bf16", "B": 12, "T": 1, "d": 768, "per": 0, "post": True, "bwd": False},
        # three ragged sequences, an odd width, a gate of its own for each sequence
        {"name": "join_train_odd_f32", "kind": "join", "dtype": "f32", "B": 3, "T": 777, "d": 193, "per": 777, "post": True, "bwd": True},
        # a block of the training configuration: 8 sequences of 4096 tokens, one gate for all of them
        {"name": "join_train_bf16", "kind": "join", "dtype": "bf16", "B": 8, "T": 4096, "d": 2048, "per": 0, "post": True, "bwd": True},
        # a dozen tokens to two experts each in a serving step
        {"name": "moe_decode_bf16", "kind": "moe", "dtype": "bf16", "N": 12, "K": 2, "d": 768, "E": 16, "pad": 0.0, "bwd": False},
        # a small expert layer at a ragged size, a padded batch
        {"name": "moe_train_small_f32", "kind": "moe", "dtype": "f32", "N": 1500, "K": 2, "d": 192, "E": 8, "pad": 0.1, "bwd": True},
        # the isolated expert layer of the benchmark with two experts a token
        {"name": "moe_train_bf16", "kind": "moe", "dtype": "bf16", "N": 65536, "K": 2, "d": 1024, "E": 64, "pad": 0.0, "bwd": True},
        # the optimizer step of the smallest model, 22 tensors in one flat buffer
        {"name": "clip_step_331k", "kind": "clip", "dtype": "f32", "model": "331k", "step": True, "max_norm": 1.0},
        # the optimizer step of the small training run
        {"name": "clip_step_12.7m", "kind": "clip", "dtype": "f32", "model": "12.7m", "step": True, "max_norm": 1.0},
        # the norm alone over a block of the training configuration: large and tiny tensors, 1.07 G gradients in f32
        {"name": "norm_1.3b_block", "kind": "clip", "dtype": "f32", "model": "1.3b-block", "step": False, "max_norm": 1.0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["embed", "join", "moe", "clip"])
    dtype, bwd = rng.choice(["f32", "bf16"]), rng.random() < 0.7
    if kind == "clip":
        step = rng.random() < 0.5
        return {"kind": "clip", "dtype": "f32" if step else dtype, "model": rng.choice(["331k", "12.7m"] if step else ["331k", "12.7m", "1.3b-block"]),
                "step": step, "max_norm": round(rng.uniform(0.1, 2.0), 3)}
    d = _log(rng, 33, 2048)
    if rng.random() < 0.6:
        d = max(32, d - d % 32)
    rows = _log(rng, 1, max(1, 30_000_000 // d // (2 if dtype == "f32" else 1)))
    if kind == "embed":
        v = _log(rng, 100, max(100, min(200_000, 45_000_000 // d)))
        return {"kind": "embed", "dtype": dtype, "N": min(rows, 200_000), "V": v, "d": d, "pad": rng.choice([0.0, 0.0, 0.1]), "bwd": bwd}
    if kind == "join":
        t = _log(rng, 1, min(rows, 4096))
        per = rng.choice([0, 0, t, 1])
        return {"kind": "join", "dtype": dtype, "B": max(1, min(rows, 100_000) // t), "T": t, "d": d, "per": per, "post": rng.random() < 0.7, "bwd": bwd}
    k = rng.choice([1, 2, 4, 8])
    e = rng.choice([4, 8, 16, 64, 128])
    return {"kind": "moe", "dtype": dtype, "N": max(1, min(rows, 200_000) // k), "K": min(k, e), "d": d, "E": e, "pad": rng.choice([0.0, 0.0, 0.1]), "bwd": bwd}


# ------------------------------------------------------------------ inputs
_gpu_handle = None


def _gpu():
    """The process's one context, on torch's stream."""
    global _gpu_handle
    import asca_b200

    if _gpu_handle is None:
        _gpu_handle = asca_b200.Gpu(0)
    _gpu_handle.use_torch_stream()
    return _gpu_handle


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _zipf(v):
    """How often each of v tokens comes, the commonest first."""
    p = 1.0 / (np.arange(1, v + 1) + 2.7) ** 1.05
    return p / p.sum()


def _tokens(rng, n, v):
    """Token ids of a text; which id is common is a matter of the seed."""
    ids = np.searchsorted(np.cumsum(_zipf(v)), rng.random(n)).clip(0, v - 1)
    return rng.permutation(v)[ids]


def _sizes(model):
    v, d, h, blocks, e, f = MODELS[model]
    return [v * d, d * v] + blocks * [d * 3 * d, 3 * d, d * 2 * h, 2 * h, d * d, d, d * e * f, e * f, e * f * d, d]


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _dtype(case)

    def norm(*shape, scale=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dtype)

    s = {"case": case}
    if case["kind"] == "embed":
        n, v, d = case["N"], case["V"], case["d"]
        ids = _tokens(rng, n, v)
        ids[rng.random(n) < case["pad"]] = -1
        s.update(ids=torch.from_numpy(ids.astype(np.int32)).cuda(), table=norm(v, d, scale=0.02, dtype=dt), scale=math.sqrt(d))
        if case["bwd"]:
            s["dx"] = norm(n, d, scale=1e-2, dtype=dt)
    elif case["kind"] == "join":
        rows, d, per = case["B"] * case["T"], case["d"], case["per"] or case["B"] * case["T"]
        s.update(y=norm(rows, d, scale=0.7, dtype=dt), x=norm(rows, d, scale=1.5), gate=1.0 + norm(-(-rows // per), d, scale=0.3), per=per,
                 w_post=1.0 + norm(d, scale=0.1) if case["post"] else None, w_pre=1.0 + norm(d, scale=0.1), skip=0.9, branch=0.4)
        if case["bwd"]:
            s.update(d_xn=norm(rows, d, scale=1e-2, dtype=dt), d_out=norm(rows, d, scale=1e-2))
    elif case["kind"] == "moe":
        n, k, d, e = (case[key] for key in ("N", "K", "d", "E"))
        # a router's choice: k experts of each token, some experts liked better than others
        scores = torch.randn(n, e, generator=g, device="cuda") + torch.randn(e, generator=g, device="cuda")
        top, experts = scores.topk(k, dim=1)
        experts = experts.to(torch.int32)
        experts[torch.from_numpy(rng.random(n) < case["pad"]).cuda()] = -1
        s.update(x=norm(n, d, dtype=dt), experts=experts.contiguous(), weights=torch.softmax(top, dim=1).contiguous(),
                 # the expert layer's rows: what its products write, zeros behind the last expert's
                 ys=norm(n * k, d), xs=torch.zeros(n * k, d, dtype=dt, device="cuda"))
        if case["bwd"]:
            s.update(d_out=norm(n, d, scale=1e-2), d_xs=norm(n * k, d, scale=1e-2), d_ys=torch.zeros(n * k, d, device="cuda"))
    else:
        sizes = _sizes(case["model"])
        off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)
        scale = 1e-3 + torch.rand(1, generator=g, device="cuda").item() * 1e-3
        flat = norm(int(off[-1]), scale=scale, dtype=dt)
        s.update(flat=flat, grads=[flat[a:b] for a, b in zip(off[:-1], off[1:])], off=off)
        if case["step"]:
            # the moments of a run some hundred steps old; the counter advances once for each tensor
            count = 100 * len(sizes) + np.arange(1, len(sizes) + 1)
            c2 = np.sqrt(1.0 - ADAM["beta2"] ** count)
            s.update(p=norm(int(off[-1]), scale=0.02), m=norm(int(off[-1]), scale=1e-3), v=norm(int(off[-1]), scale=1e-3).square_(),
                     lr_t=(ADAM["lr"] * c2 / (1.0 - ADAM["beta1"] ** count)).astype(np.float32), eps_t=(ADAM["eps"] * c2).astype(np.float32))
    if own:
        s["gpu"] = _gpu()
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return {"embed": _embed, "join": _join, "moe": _moe, "clip": _clip}[s["case"]["kind"]](s)


def _embed(s):
    case, ids, table = s["case"], s["ids"], s["table"]
    if own:
        from asca_b200 import ops

        out = {"x": ops.embed_fwd(s["gpu"], table, ids, scale=s["scale"])}
        if case["bwd"]:
            out["d_table"] = ops.embed_bwd(s["gpu"], s["dx"], ids, case["V"], scale=s["scale"])
        return out
    live = ((ids >= 0) & (ids < case["V"])).unsqueeze(1)
    at = ids.clamp(0, case["V"] - 1).long()
    out = {"x": torch.where(live, table[at].float() * s["scale"], 0.0).to(table.dtype)}
    if case["bwd"]:
        rows = torch.where(live, s["dx"].float() * s["scale"], 0.0)
        out["d_table"] = torch.zeros(case["V"], case["d"], device="cuda").index_add_(0, at, rows)
    return out


def _join(s):
    case = s["case"]
    y, x, gate, w_post, w_pre, per, skip, branch = (s[key] for key in ("y", "x", "gate", "w_post", "w_pre", "per", "skip", "branch"))
    if own:
        from asca_b200 import ops

        x_out, xn = ops.gated_residual_rmsnorm_fwd(s["gpu"], y, x, gate=gate, gate_rows=per, w_post=w_post, w_pre=w_pre, post_norm=case["post"],
                                                   skip_scale=skip, branch_scale=branch, eps=EPS)
        out = {"x_out": x_out, "xn": xn}
        if case["bwd"]:
            out.update(ops.gated_residual_rmsnorm_bwd(s["gpu"], y, x_out, s["d_xn"], s["d_out"], gate=gate, gate_rows=per, w_post=w_post, w_pre=w_pre,
                                                      post_norm=case["post"], skip_scale=skip, branch_scale=branch, eps=EPS))
        return out
    rows, d = x.shape
    yf = y.float()
    if case["post"]:
        r1 = torch.rsqrt(yf.square().mean(1, keepdim=True) + EPS)
        yh = yf * r1
        n = yh * w_post
    else:
        n = yf
    gr = gate.expand(rows, d) if gate.shape[0] == 1 else gate.repeat_interleave(per, 0)[:rows]
    x_out = skip * x + branch * gr * n
    r2 = torch.rsqrt(x_out.square().mean(1, keepdim=True) + EPS)
    xh = x_out * r2
    out = {"x_out": x_out, "xn": (xh * w_pre).to(y.dtype)}
    if case["bwd"]:
        dn2 = s["d_xn"].float()
        out["d_w_pre"] = (dn2 * xh).sum(0)
        t = dn2 * w_pre
        dxo = s["d_out"] + r2 * (t - xh * (t * xh).mean(1, keepdim=True))
        out["d_x"] = skip * dxo
        dg = branch * dxo * n
        groups = gate.shape[0]
        if groups == 1:
            out["d_gate"] = dg.sum(0, keepdim=True)
        elif groups * per == rows:
            out["d_gate"] = dg.view(groups, per, d).sum(1)
        else:
            out["d_gate"] = torch.zeros_like(gate).index_add_(0, torch.arange(rows, device="cuda") // per, dg)
        dn1 = branch * gr * dxo
        if case["post"]:
            out["d_w_post"] = (dn1 * yh).sum(0)
            t = dn1 * w_post
            out["d_y"] = (r1 * (t - yh * (t * yh).mean(1, keepdim=True))).to(y.dtype)
        else:
            out["d_y"] = dn1.to(y.dtype)
    return out


def _moe(s):
    case, x, experts, weights, ys = s["case"], s["x"], s["experts"], s["weights"], s["ys"]
    n, k, e, d = (case[key] for key in ("N", "K", "E", "d"))
    if own:
        from asca_b200 import ops

        gpu = s["gpu"]
        perm, offsets, slot = ops.moe_topk_dispatch(gpu, experts, e)
        out = {"perm": perm, "offsets": offsets, "slot": slot, "xs": ops.moe_sort_rows(gpu, x, slot, out=s["xs"]),
               "out": ops.moe_unsort_rows(gpu, ys, slot, weights=weights)}
        if case["bwd"]:
            out["d_ys"], out["d_w"] = ops.moe_unsort_rows_bwd(gpu, s["d_out"], ys, slot, weights, d_ys=s["d_ys"])
            out["dx"] = ops.moe_sort_rows_bwd(gpu, s["d_xs"], slot)
        return out
    flat = experts.reshape(-1).long()
    live = (flat >= 0) & (flat < e)
    key = torch.where(live, flat, e)
    perm = torch.sort(key, stable=True).indices
    ends = torch.zeros(e + 1, dtype=torch.long, device="cuda").index_add_(0, key, torch.ones_like(key)).cumsum(0)
    offsets = torch.cat([ends.new_zeros(1), ends[:e]])
    place = torch.empty_like(perm)
    place[perm] = torch.arange(n * k, device="cuda")
    slot = torch.where(live, place, -1)
    behind = (torch.arange(n * k, device="cuda") >= offsets[e]).unsqueeze(1)
    out = {"perm": perm.int(), "offsets": offsets.int(), "slot": slot.int().view(n, k), "xs": torch.where(behind, 0.0, x[perm // k].float()).to(x.dtype)}
    rows = torch.where(live.unsqueeze(1), ys[place], 0.0).view(n, k, d)
    out["out"] = (rows * weights.unsqueeze(2)).sum(1)
    if case["bwd"]:
        d_out = s["d_out"]
        out["d_ys"] = torch.where(behind, 0.0, d_out[perm // k] * weights.reshape(-1)[perm].unsqueeze(1))
        out["d_w"] = (rows * d_out.unsqueeze(1)).sum(2)
        out["dx"] = torch.where(live.unsqueeze(1), s["d_xs"][place], 0.0).view(n, k, d).sum(1)
    return out


def _clip(s):
    case, grads = s["case"], s["grads"]
    if own:
        from asca_b200 import ops

        if not case["step"]:
            return {"norm": ops.grad_norm(s["gpu"], grads)}
        norm = ops.grad_norm(s["gpu"], [s["flat"]])
        ops.adamw_segmented(s["gpu"], s["p"], s["flat"], s["m"], s["v"], s["off"], s["lr_t"], s["eps_t"], ADAM["beta1"], ADAM["beta2"],
                            ADAM["lr"] * ADAM["wd"], norm=norm, max_norm=case["max_norm"])
        return {"norm": norm, "p": s["p"], "m": s["m"], "v": s["v"]}
    if not case["step"]:
        return {"norm": torch.stack([x.float().square().sum() for x in grads]).sum().sqrt().reshape(1)}
    p, m, v, flat = s["p"], s["m"], s["v"], s["flat"]
    norm = flat.square().sum().sqrt().reshape(1)
    gc = flat * (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    lengths = torch.from_numpy(np.diff(s["off"])).to("cuda", non_blocking=True)
    lr_t, eps_t = (torch.from_numpy(a).to("cuda", non_blocking=True).repeat_interleave(lengths, output_size=flat.numel()) for a in (s["lr_t"], s["eps_t"]))
    m.mul_(ADAM["beta1"]).add_((1 - ADAM["beta1"]) * gc)
    v.mul_(ADAM["beta2"]).add_((1 - ADAM["beta2"]) * gc * gc)
    p.sub_(ADAM["lr"] * ADAM["wd"] * p).sub_(lr_t * (m / (v.sqrt() + eps_t)))
    return {"norm": norm, "p": p, "m": m, "v": v}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "embed":
        n, v, d = case["N"], case["V"], case["d"]
        met = float(np.sum(1.0 - (1.0 - _zipf(v)) ** (n * (1.0 - case["pad"]))))   # rows of the table that a text of n tokens meets
        total = size * d * (met + n) + 4 * n
        if case["bwd"]:
            total += size * n * d + 4 * v * d
        return {"bytes": total, "flops": n * d * (2 if case["bwd"] else 1)}
    if case["kind"] == "join":
        rows, d = case["B"] * case["T"], case["d"]
        gates = -(-rows // (case["per"] or rows)) * d
        total = rows * d * (4 + 4 + 2 * size) + 4 * (gates + 2 * d)
        if case["bwd"]:
            # y and x_out again, both gradients in, both gradients out
            total += rows * d * (4 + size + size + 4 + 4 + size) + 4 * (gates + 2 * d) + 4 * gates
        return {"bytes": total, "flops": rows * d * (30 if case["bwd"] else 10)}
    if case["kind"] == "moe":
        n, k, d, e = (case[key] for key in ("N", "K", "d", "E"))
        rows = n * k * (1.0 - case["pad"])
        total = 12 * n * k + 4 * (e + 1) + size * d * (n + rows) + 4 * d * (n + rows) + 4 * n * k
        flops = 2 * rows * d
        if case["bwd"]:
            total += 4 * d * (n + 2 * rows) + 8 * n * k + 4 * d * (n + rows)
            flops += 4 * rows * d
        return {"bytes": total, "flops": flops}
    total = sum(_sizes(case["model"]))
    # a step reads the gradient and both moments and writes the weights and the moments, which it has read
    return {"bytes": total * (28 if case["step"] else size), "flops": total * (17 if case["step"] else 2)}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    w = {key: t.double() for key, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point() and key != "flat"}
    if case["kind"] == "embed":
        ids = s["ids"].long()
        live = (ids >= 0).nonzero().squeeze(1)
        x = torch.zeros(case["N"], case["d"], dtype=torch.float64, device="cuda")
        x[live] = s["scale"] * w["table"].index_select(0, ids[live])
        if not case["bwd"]:
            return {"x": x}
        table = torch.zeros(case["V"], case["d"], dtype=torch.float64, device="cuda")
        table.index_put_((ids[live],), s["scale"] * w["dx"][live], accumulate=True)
        return {"x": x, "d_table": table}
    if case["kind"] == "join":
        y, x, gate, w_pre = (w[key].requires_grad_() for key in ("y", "x", "gate", "w_pre"))
        row = torch.arange(x.shape[0], device="cuda") // s["per"]
        n, leaves = y, [y, x, gate, w_pre]
        if case["post"]:
            leaves.append(w["w_post"].requires_grad_())
            n = y / (y.pow(2).mean(1, keepdim=True) + EPS).sqrt() * leaves[-1]
        x_out = s["skip"] * x + s["branch"] * gate[row] * n
        xn = x_out / (x_out.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w_pre
        out = {"x_out": x_out.detach(), "xn": xn.detach()}
        if case["bwd"]:
            got = torch.autograd.grad([x_out, xn], leaves, [w["d_out"], w["d_xn"]])
            out.update(zip(("d_y", "d_x", "d_gate", "d_w_pre", "d_w_post"), got))
        return out
    if case["kind"] == "moe":
        n, k, e = case["N"], case["K"], case["E"]
        chosen = s["experts"].cpu().numpy().reshape(-1)
        order = [np.flatnonzero(chosen == i) for i in range(e)]
        valid = np.concatenate(order)
        perm = np.concatenate([valid, np.flatnonzero(chosen < 0)])
        slot = np.full(n * k, -1)
        slot[valid] = np.arange(valid.size)
        at = torch.from_numpy(valid).cuda()
        token = at // k
        xs = torch.zeros(n * k, case["d"], dtype=torch.float64, device="cuda")
        xs[: valid.size] = w["x"][token]
        weight = w["weights"].reshape(-1)[at].unsqueeze(1)
        out = torch.zeros(n, case["d"], dtype=torch.float64, device="cuda").index_add_(0, token, weight * w["ys"][: valid.size])
        whole = {"perm": torch.from_numpy(perm.astype(np.int32)), "slot": torch.from_numpy(slot.astype(np.int32)).view(n, k),
                 "offsets": torch.from_numpy(np.concatenate([[0], np.cumsum([len(o) for o in order])]).astype(np.int32))}
        res = {**whole, "xs": xs, "out": out}
        if case["bwd"]:
            res["d_ys"] = torch.zeros_like(xs)
            res["d_ys"][: valid.size] = weight * w["d_out"][token]
            res["d_w"] = torch.zeros(n * k, dtype=torch.float64, device="cuda")
            res["d_w"][at] = torch.linalg.vecdot(w["d_out"][token], w["ys"][: valid.size])
            res["d_w"] = res["d_w"].view(n, k)
            res["dx"] = torch.zeros(n, case["d"], dtype=torch.float64, device="cuda").index_add_(0, token, w["d_xs"][: valid.size])
        return res
    total = sum(float(torch.dot(x.double(), x.double())) for part in s["grads"] for x in part.split(1 << 26))
    norm = torch.tensor([math.sqrt(total)], dtype=torch.float64, device="cuda")
    if not case["step"]:
        return {"norm": norm}
    res = {key: torch.empty(int(s["off"][-1]), dtype=torch.float64, device="cuda") for key in "pmv"}
    c = min(1.0, case["max_norm"] / (math.sqrt(total) + 1e-6))
    for i, (a, b) in enumerate(zip(s["off"][:-1], s["off"][1:])):
        g = c * s["flat"][a:b].double()
        res["m"][a:b] = ADAM["beta1"] * w["m"][a:b] + (1 - ADAM["beta1"]) * g
        res["v"][a:b] = ADAM["beta2"] * w["v"][a:b] + (1 - ADAM["beta2"]) * g ** 2
        res["p"][a:b] = w["p"][a:b] * (1 - ADAM["lr"] * ADAM["wd"]) - float(s["lr_t"][i]) * res["m"][a:b] / (res["v"][a:b].sqrt() + float(s["eps_t"][i]))
    return {"norm": norm, **res}

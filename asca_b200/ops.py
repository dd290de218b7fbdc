"""Device-pointer entry points of libasca_b200 on torch CUDA tensors.

torch is used only to own device memory and streams; every function forwards raw pointers
to the C ABI (include/asca_b200.h) and launches the library's own kernels on the stream the
:class:`asca_b200.Gpu` context is bound to (call ``gpu.use_torch_stream()`` to share
torch's current stream).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import BF16, F32, NN, NT, TN, Gpu, _f, _i64, _p  # noqa: F401


class _Missing:
    """In the place of _torch_ops.so where it cannot be loaded: the functions that go through it refuse (there is no slower way in its
    place), those that need the library alone work."""

    def __init__(self, why):
        self._why = why

    def __getattr__(self, name):
        raise ImportError("asca_b200/_torch_ops.so is missing or was built for another torch: build it with `python -m asca_b200.build`") from self._why


try:
    from . import _torch_ops as _t

    _for = getattr(_t, "built_for", "a torch that it does not name")
    if not _for.startswith(f"torch {torch.__version__},"):   # (another torch's tensors may be laid out in another way)
        raise ImportError(f"built for {_for}; this is torch {torch.__version__}")
except ImportError as e:
    _t = _Missing(e)


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.bfloat16:
        return BF16
    raise TypeError(f"unsupported dtype {t.dtype}")


def _chk(*ts):
    for t in ts:
        if t is not None:
            assert t.is_cuda and t.is_contiguous(), "expected contiguous CUDA tensors"


def gemm(gpu: Gpu, a, b, mode=NN, bias=None, out=None, accumulate=False):
    """C = op(A) op(B) (+ bias) (+ C). a, b both f32 or both bf16; C f32."""
    _chk(a, b, bias, out)
    if mode == NN:
        m, k, n = a.shape[0], a.shape[1], b.shape[1]
    elif mode == TN:
        m, k, n = a.shape[1], a.shape[0], b.shape[1]
    else:
        m, k, n = a.shape[0], a.shape[1], b.shape[0]
    if out is None:
        out = torch.empty((m, n), dtype=torch.float32, device=a.device)
    gpu._call("asca_gemm", gpu._ctx, C.c_int(mode), _i64(m), _i64(n), _i64(k), _p(a), _i64(a.shape[1]), _p(b),
              _i64(b.shape[1]), _p(out), _i64(n), _p(bias), C.c_int(1 if accumulate else 0), C.c_int(_dt(a)))
    return out


def rmsnorm_fwd(gpu, x, eps=1e-6, want_inv=False):
    _chk(x)
    y = torch.empty_like(x)
    inv = torch.empty(x.shape[0], dtype=torch.float32, device=x.device) if want_inv else None
    gpu._call("asca_rmsnorm_fwd", gpu._ctx, _p(x), _p(y), _p(inv), _i64(x.shape[0]), _i64(x.shape[1]), _f(eps))
    return (y, inv) if want_inv else y


def rmsnorm_bwd(gpu, x, dy, eps=1e-6):
    _chk(x, dy)
    dx = torch.empty_like(x)
    gpu._call("asca_rmsnorm_bwd", gpu._ctx, _p(x), _p(dy), _p(dx), _i64(x.shape[0]), _i64(x.shape[1]), _f(eps))
    return dx


def residual_rmsnorm(gpu, x, y, eps=1e-6, want_norm=True):
    """x_mid = x + y and (optionally) xn = rmsnorm(x_mid) in one pass."""
    _chk(x, y)
    x_mid = torch.empty_like(x)
    xn = torch.empty_like(x) if want_norm else None
    gpu._call("asca_residual_rmsnorm", gpu._ctx, _p(x), _p(y), _p(x_mid), _p(xn), _i64(x.shape[0]), _i64(x.shape[1]),
              _f(eps))
    return x_mid, xn


def gather_rows(gpu, src, idx):
    _chk(src, idx)
    dst = torch.empty((idx.numel(), src.shape[1]), dtype=torch.float32, device=src.device)
    gpu._call("asca_gather_rows", gpu._ctx, _p(src), _p(idx), _i64(idx.numel()), _i64(src.shape[1]), _p(dst))
    return dst


def scatter_rows(gpu, src, idx, dst):
    _chk(src, idx, dst)
    gpu._call("asca_scatter_rows", gpu._ctx, _p(src), _p(idx), _i64(idx.numel()), _i64(src.shape[1]), _p(dst))


def adamw(gpu, p, g, m, v, lr_t, beta1, beta2, eps_t, wd_eff):
    _chk(p, g, m, v)
    gpu._call("asca_adamw", gpu._ctx, _p(p), _p(g), _p(m), _p(v), _i64(p.numel()), _f(lr_t), _f(beta1), _f(beta2),
              _f(eps_t), _f(wd_eff))


def adamw_segmented(gpu, p, g, m, v, seg_off, lr_t, eps_t, beta1, beta2, wd_eff, norm=None, max_norm=None):
    """seg_off: int64 numpy array (n_seg+1); lr_t, eps_t: float32 numpy arrays (n_seg). With ``norm`` (what :func:`grad_norm`
    returned) and ``max_norm`` the gradient enters as min(1, max_norm / (norm + 1e-6)) * g; g itself stays as it is."""
    import numpy as np

    _chk(p, g, m, v)
    if (norm is None) != (max_norm is None):
        raise ValueError("adamw_segmented: norm and max_norm belong together")
    seg_off = np.ascontiguousarray(seg_off, dtype=np.int64)
    lr_t = np.ascontiguousarray(lr_t, dtype=np.float32)
    eps_t = np.ascontiguousarray(eps_t, dtype=np.float32)
    if norm is not None:
        _t.adamw_clip(gpu.handle, gpu.device, gpu.bound_stream, p, g, m, v, seg_off, lr_t, eps_t, beta1, beta2, wd_eff, norm, max_norm)
        return
    gpu._call("asca_adamw_segmented", gpu._ctx, _p(p), _p(g), _p(m), _p(v), _p(seg_off), _p(lr_t), _p(eps_t),
              C.c_int(lr_t.size), _f(beta1), _f(beta2), _f(wd_eff))


# ------------------------------------------------------------------ a training step around the blocks
# These check their tensors (device, dtype, shape, contiguity) and that the context is on torch's current stream, because
# scratch and outputs come from torch's allocator in that stream's order: call gpu.use_torch_stream() after changing streams.
# A call that is captured into a CUDA graph has its scratch in the graph's own memory. The work of the wrappers is done in
# csrc/torch_ops.cpp.
def embed_fwd(gpu, table, ids, scale=1.0, out_dtype=None, out=None):
    """x[t] = scale * table[ids[t]]: table (V, d) f32 or bf16, ids int32 or uint32 of any shape; an id outside the table (-1, say) is
    padding and gives zeros. Returns ids.shape + (d,) in ``out_dtype`` (default: the table's)."""
    return _t.embed_fwd(gpu.handle, gpu.device, gpu.bound_stream, table, ids, scale, out_dtype, out)


def embed_bwd(gpu, dx, ids, vocab, scale=1.0, d_table=None, accumulate=False):
    """The gradient of :func:`embed_fwd` for a table of ``vocab`` rows: d_table[v] = scale * (sum of dx[t] over ids[t] == v), f32;
    with ``accumulate`` added to the given ``d_table``, of which only the rows of the tokens that occur are touched."""
    return _t.embed_bwd(gpu.handle, gpu.device, gpu.bound_stream, dx, ids, vocab, scale, d_table, accumulate)


def gated_residual_rmsnorm_fwd(gpu, y, x, gate=None, gate_rows=None, w_post=None, w_pre=None, post_norm=True, skip_scale=1.0, branch_scale=1.0,
                               eps=1e-6, want_norm=True, x_out=None):
    """The join behind a block whose output is y (rows, cols), f32 or bf16, on the f32 residual stream x:

    n = rmsnorm(y) * w_post (y itself without ``post_norm``), x_out = skip_scale * x + branch_scale * gate[r // gate_rows] * n,
    xn = rmsnorm(x_out) * w_pre in y's dtype. gate (ceil(rows / gate_rows), cols) f32, gate_rows None: one gate for all rows.
    Returns (x_out, xn); xn is None without ``want_norm``. ``x_out`` may be x."""
    return _t.join_fwd(gpu.handle, gpu.device, gpu.bound_stream, y, x, gate, gate_rows, w_post, w_pre, post_norm, skip_scale, branch_scale, eps,
                       want_norm, x_out)


def gated_residual_rmsnorm_bwd(gpu, y, x_out, d_xn, d_out, gate=None, gate_rows=None, w_post=None, w_pre=None, post_norm=True, skip_scale=1.0,
                               branch_scale=1.0, eps=1e-6, grads=None):
    """Gradients of :func:`gated_residual_rmsnorm_fwd`, from d_xn (y's dtype) and d_out (f32, what reaches x_out from further on);
    one of the two may be None. Returns a dict: d_x, d_y, and d_gate, d_w_post, d_w_pre for those of the three that are given.
    ``grads``: a dict with these tensors to add to instead of making new ones."""
    return _t.join_bwd(gpu.handle, gpu.device, gpu.bound_stream, y, x_out, d_xn, d_out, gate, gate_rows, w_post, w_pre, post_norm, skip_scale,
                       branch_scale, eps, grads)


def moe_topk_dispatch(gpu, experts, E):
    """experts (N, K) int32, a router's choice; one outside [0, E) (-1, say) sends the assignment nowhere. Returns perm (N*K: the
    assignments t*K + k by expert, ascending inside one, those that go nowhere last), offsets (E+1: the experts' bounds in perm) and
    slot (N, K: where each assignment lies in perm, -1 if it goes nowhere), all int32."""
    return _t.moe_dispatch(gpu.handle, gpu.device, gpu.bound_stream, experts, E)


def moe_sort_rows(gpu, x, slot, out_dtype=None, out=None):
    """xs[slot[t, k]] = x[t]: (N, d) -> (N*K, d) in expert order. Rows behind the last expert's are left as they were (in a new
    tensor: undefined)."""
    return _t.moe_sort(gpu.handle, gpu.device, gpu.bound_stream, x, slot, out_dtype, out)


def moe_sort_rows_bwd(gpu, d_xs, slot, out_dtype=torch.float32):
    """d_x[t] = sum over k of d_xs[slot[t, k]]."""
    return _t.moe_unsort(gpu.handle, gpu.device, gpu.bound_stream, d_xs, slot, None, out_dtype, None)


def moe_unsort_rows(gpu, ys, slot, weights=None, out_dtype=torch.float32, out=None):
    """out[t] = sum over k of weights[t, k] * ys[slot[t, k]]: (N*K, d) in expert order -> (N, d). weights (N, K) f32, None: ones.
    A given ``out`` has its own dtype."""
    return _t.moe_unsort(gpu.handle, gpu.device, gpu.bound_stream, ys, slot, weights, out_dtype, out)


def moe_unsort_rows_bwd(gpu, d_out, ys, slot, weights=None, d_ys=None):
    """Gradients of :func:`moe_unsort_rows`: (d_ys in ys' dtype, rows behind the last expert's left as they were; d_w (N, K) f32, or
    None without weights). ``d_ys`` may be ys."""
    return _t.moe_unsort_bwd(gpu.handle, gpu.device, gpu.bound_stream, d_out, ys, slot, weights, d_ys)


def grad_norm(gpu, grads, out=None):
    """The L2 norm over all elements of all tensors (f32 and bf16 may be mixed), as a device tensor (1,) f32; no wait."""
    return _t.grad_norm(gpu.handle, gpu.device, gpu.bound_stream, grads, out)


def clip_grads(gpu, grads, max_norm, norm=None):
    """Scales the tensors in place by min(1, max_norm / (norm + 1e-6)) and returns the norm (1,), taken here unless it is given.
    Tensors must not overlap, nor have the norm among their elements. An optimizer step that follows in :func:`adamw_segmented` can
    clip by itself, without this pass."""
    grads = list(grads)
    if norm is None:
        norm = grad_norm(gpu, grads)
    _t.clip_grads(gpu.handle, gpu.device, gpu.bound_stream, grads, max_norm, norm)
    return norm


def delta_ckpt_floats(gpu, B, T, H, dh, chunk):
    return int(gpu.lib.asca_delta_ckpt_floats(B, T, H, dh, chunk))


def delta_prep(gpu, qkv, gate, H, dh):
    _chk(qkv, gate)
    n, d = qkv.shape[0], H * dh
    f = dict(dtype=torch.float32, device=qkv.device)
    q, k, v = (torch.empty((n, d), **f) for _ in range(3))
    qn, kn, al, be = (torch.empty((n, H), **f) for _ in range(4))
    gpu._call("asca_delta_prep", gpu._ctx, _p(qkv), _p(gate), _i64(n), _i64(H), _i64(dh), _p(q), _p(k), _p(v), _p(qn),
              _p(kn), _p(al), _p(be))
    return q, k, v, qn, kn, al, be


def delta_fwd(gpu, q, k, v, alpha, beta, B, T, H, dh, chunk=64, s_init=None, want_final=False, want_ckpt=True,
              out=None, ckpt=None):
    _chk(q, k, v, alpha, beta, s_init)
    o = torch.empty_like(q) if out is None else out
    f = dict(dtype=torch.float32, device=q.device)
    s_final = torch.empty((B, H, dh, dh), **f) if want_final else None
    if want_ckpt and ckpt is None:
        ckpt = torch.empty(delta_ckpt_floats(gpu, B, T, H, dh, chunk), **f)
    gpu._call("asca_delta_fwd", gpu._ctx, _p(q), _p(k), _p(v), _p(alpha), _p(beta), _i64(B), _i64(T), _i64(H),
              _i64(dh), _i64(chunk), C.c_int(_dt(q)), _p(o), _p(s_init), _p(s_final), _p(ckpt if want_ckpt else None))
    return o, s_final, (ckpt if want_ckpt else None)


def delta_bwd(gpu, q, k, v, alpha, beta, qnorm, knorm, d_o, ckpt, B, T, H, dh, chunk=64, d_qkv=None, d_gate=None):
    _chk(q, k, v, alpha, beta, qnorm, knorm, d_o, ckpt)
    assert d_o.dtype == q.dtype
    n, d = B * T, H * dh
    f = dict(dtype=torch.float32, device=q.device)
    if d_qkv is None:
        d_qkv = torch.empty((n, 3 * d), **f)
    if d_gate is None:
        d_gate = torch.empty((n, 2 * H), **f)
    gpu._call("asca_delta_bwd", gpu._ctx, _p(q), _p(k), _p(v), _p(alpha), _p(beta), _p(qnorm), _p(knorm), _p(d_o),
              _p(ckpt), _i64(B), _i64(T), _i64(H), _i64(dh), _i64(chunk), C.c_int(_dt(q)), _p(d_qkv), _p(d_gate))
    return d_qkv, d_gate


def delta_step(gpu, q, k, v, alpha, beta, S, H, dh, fused=False, out=None):
    """In-place decode step on S (n_streams, H, dh, dh). fused: q = raw qkv (n, 3d), alpha = raw gate (n, 2H)."""
    _chk(q, k, v, alpha, beta, S)
    n = S.shape[0]
    o = torch.empty((n, H * dh), dtype=torch.float32, device=S.device) if out is None else out
    gpu._call("asca_delta_step", gpu._ctx, _p(q), _p(k), _p(v), _p(alpha), _p(beta), _p(S), _i64(n), _i64(H), _i64(dh),
              C.c_int(1 if fused else 0), _p(o))
    return o


def moe_dispatch(gpu, ids, E, want_route=False):
    _chk(ids)
    assert ids.dtype in (torch.int32, torch.uint32)
    n = ids.numel()
    perm = torch.empty(n, dtype=torch.int32, device=ids.device)
    offsets = torch.empty(E + 1, dtype=torch.int32, device=ids.device)
    route = torch.empty(n, dtype=torch.int32, device=ids.device) if want_route else None
    gpu._call("asca_moe_dispatch", gpu._ctx, _p(ids), _i64(n), _i64(E), _p(perm), _p(offsets), _p(route))
    return (perm, offsets, route) if want_route else (perm, offsets)


def moe_fwd(gpu, xn, w1, b1, w2, b2, perm, offsets, F, E, out=None, pre_p=None, hid_p=None):
    _chk(xn, w1, b1, w2, b2, perm, offsets)
    n, d = xn.shape
    dev = xn.device
    if out is None:
        out = torch.empty((n, d), dtype=torch.float32, device=dev)
    if pre_p is None:
        pre_p = torch.empty((n, F), dtype=torch.float32, device=dev)
    if hid_p is None:
        hid_p = torch.empty((n, F), dtype=xn.dtype, device=dev)
    gpu._call("asca_moe_fwd", gpu._ctx, _p(xn), _p(w1), _p(b1), _p(w2), _p(b2), _p(perm), _p(offsets), _i64(n), _i64(d),
              _i64(F), _i64(E), C.c_int(_dt(xn)), _p(out), _p(pre_p), _p(hid_p))
    return out, pre_p, hid_p


def moe_bwd(gpu, xn, w1, w2, pre_p, hid_p, dout, perm, offsets, F, E, grads=None):
    _chk(xn, w1, w2, pre_p, hid_p, dout, perm, offsets)
    n, d = xn.shape
    f = dict(dtype=torch.float32, device=xn.device)
    if grads is None:
        grads = (torch.empty((d, E * F), **f), torch.empty(E * F, **f), torch.empty((E * F, d), **f),
                 torch.empty(d, **f), torch.empty((n, d), **f))
    d_w1, d_b1, d_w2, d_b2, dxn = grads
    gpu._call("asca_moe_bwd", gpu._ctx, _p(xn), _p(w1), _p(w2), _p(pre_p), _p(hid_p), _p(dout), _p(perm), _p(offsets),
              _i64(n), _i64(d), _i64(F), _i64(E), C.c_int(_dt(xn)), _p(d_w1), _p(d_b1), _p(d_w2), _p(d_b2), _p(dxn))
    return grads


def moe_step(gpu, x, ids, w1, b1, w2, b2, F, E):
    _chk(x, ids, w1, b1, w2, b2)
    out = torch.empty_like(x)
    gpu._call("asca_moe_step", gpu._ctx, _p(x), _p(ids), _p(w1), _p(b1), _p(w2), _p(b2), _i64(x.shape[0]),
              _i64(x.shape[1]), _i64(F), _i64(E), C.c_int(_dt(w1)), _p(out))
    return out


class DeltaHostPipeline:
    """Delta-rule forward + BPTT for sequences that live in pinned host memory.

    The op is independent per sequence, so the step is cut into one stage per sequence and the
    stages are pipelined over three streams: the host->device copy of sequence s+1, the kernels
    of sequence s and the device->host copy of sequence s-1 run at the same time (PCIe is full
    duplex). ``depth`` device slots bound the memory held: each slot has room for one
    sequence's inputs, checkpoints and outputs.

    All host tensors must be pinned; q, k, v, d_o in one dtype (f32 or bf16), the rest f32.
    """

    def __init__(self, gpu: Gpu, T, H, dh, chunk=64, dtype=torch.bfloat16, depth=3):
        self.gpu, self.T, self.H, self.dh, self.chunk, self.depth = gpu, T, H, dh, chunk, depth
        dev = torch.device("cuda", gpu.device)
        self.dev = dev
        d = H * dh
        f = dict(dtype=torch.float32, device=dev)
        a = dict(dtype=dtype, device=dev)
        self.slots = []
        for _ in range(depth):
            self.slots.append(dict(
                q=torch.empty((T, d), **a), k=torch.empty((T, d), **a), v=torch.empty((T, d), **a),
                d_o=torch.empty((T, d), **a), alpha=torch.empty((T, H), **f), beta=torch.empty((T, H), **f),
                qn=torch.empty((T, H), **f), kn=torch.empty((T, H), **f), o=torch.empty((T, d), **a),
                ckpt=torch.empty(delta_ckpt_floats(gpu, 1, T, H, dh, chunk), **f),
                d_qkv=torch.empty((T, 3 * d), **f), d_gate=torch.empty((T, 2 * H), **f),
                computed=torch.cuda.Event(), drained=torch.cuda.Event()))
        self.s_in, self.s_run, self.s_out = (torch.cuda.Stream(dev) for _ in range(3))

    def run(self, q, k, v, alpha, beta, qnorm, knorm, d_o, o, d_qkv, d_gate, B):
        """Host in, host out; returns after every result has landed in o, d_qkv, d_gate."""
        T, H, dh, gpu = self.T, self.H, self.dh, self.gpu
        for x in (q, k, v, alpha, beta, qnorm, knorm, d_o, o, d_qkv, d_gate):
            assert not x.is_cuda and x.is_pinned() and x.shape[0] == B * T, "expected pinned host tensors of B*T rows"
        for s in range(B):
            sl = self.slots[s % self.depth]
            rows = slice(s * T, (s + 1) * T)
            with torch.cuda.stream(self.s_in):
                if s >= self.depth:
                    self.s_in.wait_event(sl["computed"])      # the slot's inputs have been consumed
                for name, src in (("q", q), ("k", k), ("v", v), ("alpha", alpha), ("beta", beta), ("qn", qnorm),
                                  ("kn", knorm), ("d_o", d_o)):
                    sl[name].copy_(src[rows], non_blocking=True)
                loaded = self.s_in.record_event()
            with torch.cuda.stream(self.s_run):
                self.s_run.wait_event(loaded)
                if s >= self.depth:
                    self.s_run.wait_event(sl["drained"])      # the slot's outputs have been copied out
                gpu.use_torch_stream()
                delta_fwd(gpu, sl["q"], sl["k"], sl["v"], sl["alpha"], sl["beta"], 1, T, H, dh, chunk=self.chunk,
                          out=sl["o"], ckpt=sl["ckpt"])
                delta_bwd(gpu, sl["q"], sl["k"], sl["v"], sl["alpha"], sl["beta"], sl["qn"], sl["kn"], sl["d_o"],
                          sl["ckpt"], 1, T, H, dh, chunk=self.chunk, d_qkv=sl["d_qkv"], d_gate=sl["d_gate"])
                sl["computed"].record(self.s_run)
            with torch.cuda.stream(self.s_out):
                self.s_out.wait_event(sl["computed"])
                o[rows].copy_(sl["o"], non_blocking=True)
                d_qkv[rows].copy_(sl["d_qkv"], non_blocking=True)
                d_gate[rows].copy_(sl["d_gate"], non_blocking=True)
                sl["drained"].record(self.s_out)
        self.s_out.synchronize()
        self.s_run.synchronize()
        gpu.use_torch_stream()   # back on the caller's stream

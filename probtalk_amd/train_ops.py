"""Autograd glue of the training path: every Function's forward AND backward run the library's HIP kernels through
the C ABI (`pt_conv1d_cl`, `pt_attention_cl`, `pt_embed_pe`, `pt_train_*`); torch.autograd is only the tape, torch
itself only moves memory (permute / pad / cat of weights and rows).  No CPU or PyTorch-kernel fallback exists: the ops
raise if the library or the GPU is missing.

All activations are channels-last 2-D fp32 tensors `[B*L, C]` with C a multiple of 32 (pad columns zero), the layout
of the inference library.  Conv `kind`: 0 = Linear / 1x1, 1 = k3 s1 p1, 2 = k7 s1 p3, 3 = k4 s2 p1, 4 = ConvTranspose
k4 s2 p1 (reference shapes: nets/spg/vqvae_modules.py:107-200, nets/inpainting/gated_pixelcnn_1d.py:39-83).
"""
import array
import contextlib
import ctypes as C

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, ptr, stream

_HERE = contextlib.nullcontext()
_KT = {0: 1, 1: 3, 2: 7, 3: 4, 4: 4}


def _ru(x, m):
    return (x + m - 1) // m * m


def _zeros(*shape):
    return torch.zeros(*shape, device="cuda", dtype=torch.float32)


def _empty(*shape):
    return torch.empty(*shape, device="cuda", dtype=torch.float32)


def pack_taps(w_nck):
    """(N, Cin, kt) -> contiguous [kt][Npad][Kpad] fp32 (the tap-GEMM's weight layout), zero padded."""
    N, Cin, kt = w_nck.shape
    Np, Kp = _ru(N, 128), _ru(Cin, 32)
    if kt == 1 and Np == N and Kp == Cin:
        return w_nck.reshape(1, N, Cin).contiguous(), Np, Kp
    out = _zeros(kt, Np, Kp)
    out[:, :N, :Cin] = w_nck.permute(2, 0, 1)
    return out, Np, Kp


def conv_raw(x2d, w_nck, bias, kind, B, Lin, act=0, slope=0.0, res=None):
    """y = act(conv(x) + bias + res) on channels-last rows through the fp32 tap-GEMM."""
    L = _lib.lib()
    N = w_nck.shape[0]
    wp, Np, Kp = pack_taps(w_nck)
    if x2d.shape[1] < Kp:
        raise RuntimeError(f"conv: input rows have {x2d.shape[1]} columns, packed K is {Kp}")
    Lout = {0: Lin, 1: Lin, 2: Lin, 3: (Lin - 2) // 2 + 1, 4: 2 * Lin}[kind]
    ldc = _ru(N, 32)
    y = _empty(B * Lout, ldc)
    bp = None
    if bias is not None:
        if Np == N and bias.is_contiguous() and bias.dtype == torch.float32:
            bp = bias                       # no padding to add: skips a fill and a copy launch per Linear
        else:
            bp = _zeros(Np)
            bp[:N] = bias
    check(L.pt_conv1d_cl(ptr(x2d), x2d.shape[1], ptr(wp), ptr(bp), N, Np, Kp, kind, B, Lin, ptr(y), ldc, act, slope,
                         ptr(res), 0 if res is None else res.shape[1], stream()))
    return y, Lout


class ConvCL(torch.autograd.Function):
    """Conv1d / ConvTranspose1d / Linear with optional fused residual and (leaky-)ReLU; weights in the reference layout
    ((N, Cin[, kt]) or, for kind 4, (Cin, N, kt))."""

    @staticmethod
    def forward(ctx, x, w, bias, res, kind, B, Lin, slope):
        w3 = w if w.dim() == 3 else w.unsqueeze(-1)
        w_nck = w3.permute(1, 0, 2) if kind == 4 else w3
        act = 0 if slope < 0 else 1
        y, Lout = conv_raw(x, w_nck.contiguous(), bias, kind, B, Lin, act, max(slope, 0.0), res)
        ctx.save_for_backward(x, w, y if act else None)
        ctx.meta = (kind, B, Lin, Lout, slope, bias is not None, res is not None, w.dim())
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, y = ctx.saved_tensors
        kind, B, Lin, Lout, slope, has_bias, has_res, wdim = ctx.meta
        L = _lib.lib()
        dy = dy.contiguous()
        N = w.shape[1] if kind == 4 else w.shape[0]
        Cin = w.shape[0] if kind == 4 else w.shape[1]
        if slope >= 0:
            dz = _empty(dy.shape)
            check(L.pt_train_act_bwd(ptr(dy), dy.shape[1], ptr(y), y.shape[1], slope, ptr(dz), dz.shape[1], dy.shape[0],
                                     dy.shape[1], stream()))
            dy = dz
        w3 = w if w.dim() == 3 else w.unsqueeze(-1)
        dx = dw = db = dres = None
        if ctx.needs_input_grad[0]:
            # input gradient = the same tap-GEMM on dY with re-laid-out weights (see train.hip header)
            if kind in (0, 1, 2):
                wt = w3.permute(1, 0, 2).flip(2).contiguous()            # (Cin, N, kt), taps reversed
                dx, _ = conv_raw(dy, wt, None, kind, B, Lout)
            elif kind == 3:
                wt = w3.permute(1, 0, 2).contiguous()                    # ConvTranspose form, W_k^T per tap
                if 2 * Lout < Lin:                                       # odd input length: one more (zero) output row
                    dyp = _zeros(B, Lout + 1, dy.shape[1])
                    dyp[:, :Lout] = dy.view(B, Lout, -1)
                    full, _ = conv_raw(dyp.view(B * (Lout + 1), -1), wt, None, 4, B, Lout + 1)
                    dx = full.view(B, 2 * (Lout + 1), -1)[:, :Lin].reshape(B * Lin, -1).contiguous()
                else:
                    dx, _ = conv_raw(dy, wt, None, 4, B, Lout)
                    if 2 * Lout > Lin:
                        dx = dx.view(B, 2 * Lout, -1)[:, :Lin].reshape(B * Lin, -1).contiguous()
            else:
                wt = w3.contiguous()                                     # (Cin, N, kt) is already (out=Cin, in=N, kt)
                dx, _ = conv_raw(dy, wt, None, 3, B, Lout)
            if dx.shape[1] != x.shape[1]:
                t = _zeros(x.shape)
                t[:, :min(dx.shape[1], x.shape[1])] = dx[:, :min(dx.shape[1], x.shape[1])]
                dx = t
        want_db = has_bias and ctx.needs_input_grad[2]
        if ctx.needs_input_grad[1]:
            kt = _KT[kind]
            dwp = _zeros(kt, N, Cin)
            if want_db:
                # the bias gradient rides on the weight-gradient kernel (it stages the dY tiles anyway)
                db = _zeros(N)
                check(L.pt_train_wgrad_bias(ptr(dy), dy.shape[1], ptr(x), x.shape[1], ptr(dwp), ptr(db), N, Cin, kind, B, Lin,
                                            stream()))
                want_db = False
            else:
                check(L.pt_train_wgrad(ptr(dy), dy.shape[1], ptr(x), x.shape[1], ptr(dwp), N, Cin, kind, B, Lin, stream()))
            dw = dwp.permute(2, 1, 0) if kind == 4 else dwp.permute(1, 2, 0)
            dw = dw.contiguous() if wdim == 3 else dw.reshape(N, Cin).contiguous()
        if want_db:
            db = _zeros(N)
            check(L.pt_train_colsum(ptr(dy), dy.shape[1], None, 0, dy.shape[0], N, ptr(db), stream()))
        if has_res and ctx.needs_input_grad[3]:
            dres = dy
        return dx, dw, db, dres, None, None, None, None


def conv(x, w, bias, kind, B, Lin, slope=-1.0, res=None):
    return ConvCL.apply(x, w, bias, res, kind, B, Lin, slope)


class LayerNormRes(torch.autograd.Function):
    """y = LayerNorm(x + res) over 512-wide rows (PTransformer.py:329-331 post-LN residual; norm_2 of the style block)."""

    @staticmethod
    def forward(ctx, x, res, gamma, beta):
        L = _lib.lib()
        rows = x.shape[0]
        y, stats = _empty(rows, 512), _empty(rows, 2)
        check(L.pt_train_ln_fwd(ptr(x), ptr(res), ptr(gamma), ptr(beta), ptr(y), ptr(stats), rows, stream()))
        ctx.save_for_backward(x, res, gamma, stats)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, res, gamma, stats = ctx.saved_tensors
        L = _lib.lib()
        rows = x.shape[0]
        dy = dy.contiguous()
        dx, dg, db = _empty(rows, 512), _zeros(512), _zeros(512)
        check(L.pt_train_ln_bwd(ptr(dy), ptr(x), ptr(res), ptr(stats), ptr(gamma), ptr(dx), ptr(dg), ptr(db), rows, stream()))
        return dx, (dx if res is not None else None), dg, db


def layer_norm(x, gamma, beta, res=None):
    if x.shape[1] != 512:
        raise RuntimeError("layer_norm: the path's LayerNorms are 512 wide")
    return LayerNormRes.apply(x, res, gamma, beta)


def _forward_mode():
    """Whether tensors may carry tangents, which autograd refuses for its functions without a forward rule: a raw call would drop them."""
    return forward_ad._current_level >= 0


class _Last(torch.autograd.Function):
    """Gradients inside a graph of their own (create_graph): a gradient of these is refused, not left out.  `anchor`: a tensor that requires one."""

    @staticmethod
    def forward(ctx, what, anchor, *grads):
        ctx.what = what
        return tuple(None if g is None else g.clone() for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.what}: no second derivatives")


def _row_major(v):
    return v if v.stride(1) == 1 and v.stride(0) >= v.shape[1] else v.contiguous()


def _row_stride(v):
    return 0 if v is None else v.stride(0) if v.shape[0] > 1 else v.shape[1]


def _at(t):
    return None if t is None else t.data_ptr()


def _gated_norm(x, t, gate, res_scale, post_w, post_b, pre_w, pre_b, clip, kind, eps, grad):
    rows, cols = x.shape
    device, dtype = x.device, x.dtype
    y = None if t is None else torch.empty(rows, cols, device=device, dtype=dtype)
    h = None if pre_w is None else torch.empty(rows, cols, device=device, dtype=dtype)
    stats = torch.empty(rows, 4, device=device, dtype=torch.float32) if grad else None
    at = [None if v is None else v.data_ptr() for v in (x, t, gate, res_scale, post_w, post_b, pre_w, pre_b, y, h, stats)]
    with _on(device):
        check(_lib.lib().pt_train_gated_norm_fwd(at[0], _row_stride(x), at[1], _row_stride(t), *at[2:], rows, cols, clip, kind, eps,
                                                 int(dtype is torch.bfloat16), stream()))
    return y, h, stats


class GatedNorm(torch.autograd.Function):
    """y = x + res_scale * gate * N(t; post), h = N(y; pre) (see gated_norm)."""

    @staticmethod
    def forward(ctx, x, t, gate, res_scale, post_w, post_b, pre_w, pre_b, clip, kind, eps):
        y, h, stats = _gated_norm(x, t, gate, res_scale, post_w, post_b, pre_w, pre_b, clip, kind, eps, True)
        ctx.save_for_backward(x, t, gate, res_scale, post_w, post_b, pre_w, stats)
        ctx.meta = (clip, kind, int(x.dtype is torch.bfloat16))
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        x, t, gate, res_scale, post_w, post_b, pre_w, stats = ctx.saved_tensors
        clip, kind, bf = ctx.meta
        if dy is None and dh is None:
            return (None,) * 11
        rows, cols = x.shape
        need = ctx.needs_input_grad
        dy, dh = (None if d is None else d.contiguous() for d in (dy, dh))
        device, dtype = x.device, x.dtype
        dx = torch.empty(rows, cols, device=device, dtype=dtype)
        dt = torch.empty(rows, cols, device=device, dtype=dtype) if need[1] else None
        dgate = torch.empty_like(gate) if need[2] else None
        vec = [torch.empty(cols, device=device, dtype=torch.float32) if n else None for n in need[3:8]]
        L = _lib.lib()
        with _on(device):
            size = L.pt_train_gated_norm_workspace_bytes(rows, cols, clip if gate is not None else 0)
            ws = torch.empty(size, dtype=torch.uint8, device=device)
            at = [None if v is None else v.data_ptr() for v in (x, t, gate, res_scale, post_w, post_b, pre_w, stats, dy, dh, dx, dt, dgate, *vec, ws)]
            check(L.pt_train_gated_norm_bwd(at[0], _row_stride(x), at[1], _row_stride(t), *at[2:], size, rows, cols, clip, kind, bf, stream()))
        if torch.is_grad_enabled():
            dx, dt, dgate, *vec = _Last.apply("gated_norm", torch.zeros((), requires_grad=True), dx, dt, dgate, *vec)
        return dx, dt, dgate, *vec, None, None, None


def gated_norm(x, t=None, gate=None, res_scale=None, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None, rows_per_clip=None,
               kind="layer", eps=1e-5):
    """The norm of a block's output, its gate and residual scale, the residual sum and the norm in front of the next block:

        y = x + res_scale * gate * u,   u = N(t) * post_weight + post_bias,   h = N(y) * pre_weight + pre_bias      -> (y, h)

    x, t: rows (R, C) of fp32 or bf16, 1 <= C <= 8192.  gate (R / rows_per_clip, C) of x's type: a row for every rows_per_clip rows
    (by default as many as it has rows for).  Vectors of C values in fp32.  kind: 'layer' (mean and variance) or 'rms'.  Left out:
    t (y is x itself), gate, res_scale, post_weight (u = t), pre_weight (h is None).  Statistics and sums are fp32; h is taken from y
    before that is rounded to bf16.  No forward-mode and no second derivatives.  To capture the backward pass into a HIP graph, make
    the leaves inside the capture (x.detach().requires_grad_()): an eager graph of the same leaves must not be alive."""
    if x.dim() != 2 or not x.is_cuda or x.dtype not in (torch.float32, torch.bfloat16) or not 1 <= x.shape[1] <= 8192 or x.shape[0] < 1:
        raise RuntimeError(f"gated_norm: rows (R, C) of fp32 or bf16 on the GPU with C up to 8192, got {tuple(x.shape)} {x.dtype} on {x.device}")
    if kind != "layer" and kind != "rms":
        raise ValueError(f"gated_norm: kind must be 'layer' or 'rms', got {kind!r}")
    rows, cols = x.shape
    gpu = x.get_device()
    if t is None:
        if gate is not None or res_scale is not None or post_weight is not None or pre_weight is None:
            raise RuntimeError("gated_norm: without t there is nothing to gate, scale or norm but x: pass pre_weight alone")
    elif t.shape != x.shape or t.dtype is not x.dtype or t.get_device() != gpu:
        raise RuntimeError(f"gated_norm: t must be {tuple(x.shape)} {x.dtype} on {x.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if (post_bias is not None and post_weight is None) or (pre_bias is not None and pre_weight is None):
        raise RuntimeError("gated_norm: a bias comes with its weight")
    vectors = (res_scale, post_weight, post_bias, pre_weight, pre_bias)
    for name, v in zip(("res_scale", "post_weight", "post_bias", "pre_weight", "pre_bias"), vectors):
        if v is not None and (v.shape != (cols,) or v.dtype is not torch.float32 or v.get_device() != gpu):
            raise RuntimeError(f"gated_norm: {name} must be ({cols},) torch.float32 on {x.device}, got {tuple(v.shape)} {v.dtype} on {v.device}")
    clip = rows
    if gate is not None:
        if gate.dim() != 2 or gate.shape[1] != cols or gate.dtype is not x.dtype or gate.get_device() != gpu:
            raise RuntimeError(f"gated_norm: gate must be (clips, {cols}) {x.dtype} on {x.device}, got {tuple(gate.shape)} {gate.dtype} on {gate.device}")
        clip = int(rows_per_clip) if rows_per_clip is not None else rows // max(gate.shape[0], 1)
        if clip < 1 or gate.shape[0] * clip != rows:
            raise RuntimeError(f"gated_norm: {rows} rows are not {gate.shape[0]} clips of {clip}")
        gate = gate.contiguous()
    own = x
    if not x.is_contiguous():
        x = _row_major(x)
    if t is not None and not t.is_contiguous():
        t = _row_major(t)
    given = (x, t, gate, *[v if v is None or v.is_contiguous() else v.contiguous() for v in vectors])
    mode = 0 if kind == "layer" else 1
    if _forward_mode() or (torch.is_grad_enabled() and any([v is not None and v.requires_grad for v in given])):
        y, h = GatedNorm.apply(*given, clip, mode, eps)
    else:
        y, h, _ = _gated_norm(*given, clip, mode, eps, False)
    return (own if t is None else y), h


class ModSiLU(torch.autograd.Function):
    """h = SiLU(y * (1 + scale[c]) + shift[c]) with table (n_classes, 1024) = scale | shift (PTransformer.py:134-139)."""

    @staticmethod
    def forward(ctx, y, table, label, rows_per_clip):
        L = _lib.lib()
        h = _empty(y.shape)
        check(L.pt_train_modsilu_fwd(ptr(y), ptr(table), ptr(label), label.numel(), rows_per_clip, table.shape[0], ptr(h),
                                     y.shape[0], stream()))
        ctx.save_for_backward(y, table, label)
        ctx.rpc = rows_per_clip
        return h

    @staticmethod
    def backward(ctx, dh):
        y, table, label = ctx.saved_tensors
        L = _lib.lib()
        dh = dh.contiguous()
        dy, dt = _empty(y.shape), _zeros(table.shape)
        check(L.pt_train_modsilu_bwd(ptr(dh), ptr(y), ptr(table), ptr(label), label.numel(), ctx.rpc, table.shape[0], ptr(dy),
                                     ptr(dt), y.shape[0], stream()))
        return dy, dt, None, None


class Attention(torch.autograd.Function):
    """softmax(QK^T/8)V per (clip, head), 8 heads x 64, on row tensors: q [B*Nq, ldq], kv rows [B*Nk, ldk] with K at
    column k_off and V at v_off.  Self-attention passes the packed in-proj output (q | k | v) as both tensors.
    p > 0: dropout on the attention weights (nn.MultiheadAttention(dropout) in train mode), mask replayed from the seed."""

    @staticmethod
    def forward(ctx, q, kv, q_off, k_off, v_off, B, Nq, Nk, p, seed):
        L = _lib.lib()
        o = _empty(B * Nq, 512)
        qb, kb = q.data_ptr() + 4 * q_off, kv.data_ptr()
        if p > 0:
            check(L.pt_train_attention_fwd(C.c_void_p(qb), q.shape[1], C.c_void_p(kb + 4 * k_off), kv.shape[1],
                                           C.c_void_p(kb + 4 * v_off), kv.shape[1], ptr(o), 512, B, Nq, Nk, 8, p, seed, stream()))
        else:
            check(L.pt_attention_cl(C.c_void_p(qb), q.shape[1], C.c_void_p(kb + 4 * k_off), kv.shape[1],
                                    C.c_void_p(kb + 4 * v_off), kv.shape[1], ptr(o), 512, B, Nq, Nk, 8, stream()))
        ctx.save_for_backward(q, kv)
        ctx.meta = (q_off, k_off, v_off, B, Nq, Nk, p, seed, q.data_ptr() == kv.data_ptr())
        return o

    @staticmethod
    def backward(ctx, do):
        q, kv = ctx.saved_tensors
        q_off, k_off, v_off, B, Nq, Nk, p, seed, packed = ctx.meta
        L = _lib.lib()
        do = do.contiguous()
        dq = _zeros(q.shape)
        dkv = dq if packed else _zeros(kv.shape)
        lse, delta = _empty(B * 8 * Nq), _empty(B * 8 * Nq)
        qb, kb, dqb, dkb = q.data_ptr() + 4 * q_off, kv.data_ptr(), dq.data_ptr() + 4 * q_off, dkv.data_ptr()
        check(L.pt_train_attention_bwd(C.c_void_p(qb), q.shape[1], C.c_void_p(kb + 4 * k_off), kv.shape[1],
                                       C.c_void_p(kb + 4 * v_off), kv.shape[1], ptr(do), 512, C.c_void_p(dqb), dq.shape[1],
                                       C.c_void_p(dkb + 4 * k_off), dkv.shape[1], C.c_void_p(dkb + 4 * v_off), dkv.shape[1],
                                       ptr(lse), ptr(delta), B, Nq, Nk, 8, p, seed, stream()))
        return dq, (None if packed else dkv), None, None, None, None, None, None, None, None


def attention_self(qkv, B, N, p=0.0, seeds=None):
    p = float(p) if seeds is not None else 0.0
    return Attention.apply(qkv, qkv, 0, 512, 1024, B, N, N, p, seeds.next() if p > 0 else 0)


def attention_cross(q, kv, B, Nq, Nk, p=0.0, seeds=None):
    p = float(p) if seeds is not None else 0.0
    return Attention.apply(q, kv, 0, 0, 512, B, Nq, Nk, p, seeds.next() if p > 0 else 0)


def _strides(*tensors):
    """Strides of all but the last dimension, as the C entries take them (a dimension of one value has none)."""
    return array.array("q", [s if n > 1 else 0 for t in tensors for s, n in zip(t.stride()[:-1], t.shape)])


def _has_vectors(t):
    """Whether rows of channels can be read in 16-byte vectors."""
    if t.is_contiguous() and t.shape[-1] % 8 == 0:
        return t.data_ptr() % 16 == 0
    strides, per = t.stride(), 16 // t.element_size()
    return strides[-1] == 1 and t.data_ptr() % 16 == 0 and all([n == 1 or s % per == 0 for s, n in zip(strides[:-1], t.shape)])


def _vectors(t):
    """t itself if it can be read in vectors, else a contiguous copy."""
    if _has_vectors(t):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _window_attention(q, k, v, lengths, meta, grad):
    B, Nq, _, H, _, D = meta[:6]
    o = torch.empty(B, Nq, H, D, device=q.device, dtype=q.dtype)
    L, stats = _lib.lib(), None
    if grad:
        stats = torch.empty(L.pt_attention_window_stats_bytes(B, Nq, H, D, meta[10]), device=q.device, dtype=torch.uint8)
    with _on(q.device):
        check(L.pt_attention_window_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _at(stats), _address(_strides(q, k, v)), _at(lengths),
                                        *meta, stream()))
    return o, stats


class WindowAttention(torch.autograd.Function):
    """softmax over a window of keys and a few first ones (see window_attention)."""

    @staticmethod
    def forward(ctx, q, k, v, lengths, meta):
        o, stats = _window_attention(q, k, v, lengths, meta, True)
        ctx.meta = meta
        ctx.save_for_backward(q, k, v, lengths, o, stats)
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, lengths, o, stats = ctx.saved_tensors
        L = _lib.lib()
        do = _vectors(do.contiguous())
        dq, dk, dv = (torch.empty(t.shape, device=q.device, dtype=q.dtype) for t in (q, k, v))
        with _on(q.device):
            ws = torch.empty(L.pt_attention_window_bwd_workspace_bytes(*ctx.meta[:9]), dtype=torch.uint8, device=q.device)
            check(L.pt_attention_window_bwd(_at(q), _at(k), _at(v), _at(o), _at(do), _at(stats), _at(dq), _at(dk), _at(dv), _address(_strides(q, k, v)),
                                            _at(lengths), *ctx.meta, _at(ws), ws.numel(), stream()))
        if torch.is_grad_enabled():
            dq, dk, dv = _Last.apply("window_attention", torch.zeros((), requires_grad=True), dq, dk, dv)
        return dq, dk, dv, None, None


def _check_window(what, q, k, v, heads, batch, lengths, left, right, sinks, scale):
    shape, d, dtype = k.shape, q.shape[-1], q.dtype
    if len(shape) != 4 or v.shape != shape or shape[0] != batch or shape[3] != d or shape[1] < 1:
        raise RuntimeError(f"{what}: shapes {tuple(q.shape)}, {tuple(shape)} and {tuple(v.shape)} do not go together")
    gpu = q.get_device()
    if gpu < 0 or k.get_device() != gpu or v.get_device() != gpu:
        raise RuntimeError(f"{what}: tensors must be on one GPU, got {q.device}, {k.device} and {v.device}")
    if (dtype is not torch.bfloat16 and dtype is not torch.float32) or k.dtype is not dtype or v.dtype is not dtype:
        raise RuntimeError(f"{what}: fp32 or bf16, one type for all, got {dtype}, {k.dtype} and {v.dtype}")
    if d % 8 or not 8 <= d <= 128 or shape[2] < 1 or heads < 1 or heads % shape[2]:
        raise RuntimeError(f"{what}: {heads} query heads over {shape[2]} key heads of {d} channels (a multiple of 8 up to 128)")
    if lengths is not None and (lengths.dtype is not torch.int32 or lengths.shape != (batch,) or lengths.get_device() != gpu or not lengths.is_contiguous()):
        raise RuntimeError(f"{what}: lengths must be ({batch},) torch.int32 on {q.device}")
    left, right = -1 if left is None else int(left), -1 if right is None else int(right)
    if left < -1 or right < -1 or not 0 <= sinks <= 128:
        raise RuntimeError(f"{what}: a window of {left} to the left and {right} to the right with {sinks} first keys (up to 128)")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise RuntimeError(f"{what}: scale must be positive, got {scale}")
    return min(left, 1 << 30), min(right, 1 << 30), int(sinks), scale


def window_attention(q, k, v, left=None, right=0, sinks=0, lengths=None, scale=None):
    """Attention of q (B, Nq, H, D) over k, v (B, Nk, Hk, D), fp32 or bf16 -> (B, Nq, H, D); H is a multiple of Hk (heads of a
    group share a key head), D a multiple of 8 up to 128, any strides.  Row i stands at position t = i + Nk - Nq and sees key j where

        j <= t + right   and   (j >= t - left or j < sinks)   and   j < lengths[b]

    left, right: None for no limit (right = 0 is causal); sinks: first keys that stay visible, up to 128; lengths: int32 (B,), the
    keys of each sequence of a padded batch (what lies behind is not read; all of them by default).  A row that sees nothing gives
    zeros and no gradient.  Softmax and sums are fp32, probabilities and their gradients 16 bits or more, results are rounded once;
    scale is 1 / sqrt(D) by default.  Keys and values inside a sequence must be finite, with gradients q and the output's gradient too.
    With gradients, bf16 keeps a byte more of every output value for them.  The backward pass is free of atomics: the same inputs give
    the same bits.  No forward-mode and no second derivatives.  To capture it into a HIP graph, make the leaves inside the capture
    (q.detach().requires_grad_()): an eager graph of the same leaves must not be alive."""
    if q.dim() != 4 or q.shape[0] < 1 or q.shape[1] < 1:
        raise RuntimeError(f"window_attention: q is (B, Nq, H, D), got {tuple(q.shape)}")
    B, Nq, H, D = q.shape
    left, right, sinks, scale = _check_window("window_attention", q, k, v, H, B, lengths, left, right, sinks, scale)
    _, Nk, Hk, _ = k.shape
    if Nk < Nq:
        raise RuntimeError(f"window_attention: {Nq} rows for {Nk} keys")
    meta = (B, Nq, Nk, H, Hk, D, left, right, sinks, scale, int(q.dtype is torch.bfloat16))
    q, k, v = [_vectors(t if t.shape[1] == 1 or 0 <= t.stride(1) <= 1 << 20 else t.contiguous()) for t in (q, k, v)]
    if _forward_mode() or (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        return WindowAttention.apply(q, k, v, lengths, meta)
    return _window_attention(q, k, v, lengths, meta, False)[0]


def window_attention_step(q, k, v, lengths, left=None, sinks=0, scale=None):
    """window_attention for one new token per sequence over a cache: q (B, H, D), k, v (B, N, Hk, D) with room for N tokens, of
    which the first lengths[b] (int32) are filled and the last of these is the token's own -> (B, H, D).  Reads the visible keys
    only, whatever else the cache holds; a sequence of length 0 gives zeros.  No gradient."""
    if q.dim() != 3 or q.shape[0] < 1:
        raise RuntimeError(f"window_attention_step: q is (B, H, D), got {tuple(q.shape)}")
    if lengths is None:
        raise RuntimeError("window_attention_step: lengths are needed")
    if _forward_mode() and any([forward_ad.unpack_dual(t).tangent is not None for t in (q, k, v)]):
        raise NotImplementedError("window_attention_step: no forward mode differentiation")
    B, H, D = q.shape
    left, _, sinks, scale = _check_window("window_attention_step", q, k, v, H, B, lengths, left, 0, sinks, scale)
    if not _has_vectors(k) or not _has_vectors(v):
        raise RuntimeError("window_attention_step: a cache's channels must be neighbours, its address and strides multiples of 16 bytes")
    q = _vectors(q)
    _, N, Hk, _ = k.shape
    device, dtype = q.device, q.dtype
    o = torch.empty(B, H, D, device=device, dtype=dtype)
    L = _lib.lib()
    with _on(device):
        size = L.pt_attention_window_step_workspace_bytes(B, N, H, Hk, D, left, sinks)
        ws = o if size <= 16 else torch.empty(size, dtype=torch.uint8, device=device)         # up to 16 bytes: nothing is kept there
        check(L.pt_attention_window_step(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _address(_strides(q, k, v)), lengths.data_ptr(), B, N,
                                         H, Hk, D, left, sinks, scale, int(dtype is torch.bfloat16), ws.data_ptr(), size, stream()))
    return o


class CrossEntropy(torch.autograd.Function):
    """F.cross_entropy(logits [rows, V], target [rows]) with mean reduction (predictor.py:261)."""

    @staticmethod
    def forward(ctx, logits, target):
        L = _lib.lib()
        rows, V = logits.shape
        loss, dl = _zeros(1), _empty(rows, V)
        check(L.pt_train_cross_entropy(ptr(logits), ptr(target), V, rows, ptr(loss), ptr(dl), stream()))
        ctx.save_for_backward(dl)
        return loss[0]

    @staticmethod
    def backward(ctx, g):
        (dl,) = ctx.saved_tensors
        return dl * g, None


class BNTrain(torch.autograd.Function):
    """y = act(BatchNorm1d_train(x) + res) on channels-last rows, batch statistics over all rows; running statistics
    are updated in place like nn.BatchNorm1d (momentum 0.1, unbiased running variance)."""

    @staticmethod
    def forward(ctx, x, gamma, beta, res, slope, run_mean, run_var, momentum):
        L = _lib.lib()
        rows, cols = x.shape[0], gamma.numel()
        y = _zeros(rows, x.shape[1]) if x.shape[1] != cols else _empty(rows, cols)
        mr = _empty(2, cols)
        acc = torch.empty(2 * cols, device="cuda", dtype=torch.float64)
        check(L.pt_train_bn_fwd(ptr(x), x.shape[1], rows, cols, ptr(gamma), ptr(beta), ptr(res),
                                0 if res is None else res.shape[1], slope, ptr(y), y.shape[1], ptr(mr), ptr(acc), ptr(run_mean),
                                ptr(run_var), momentum, stream()))
        ctx.save_for_backward(x, gamma, y, mr)
        ctx.meta = (slope, res is not None)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, gamma, y, mr = ctx.saved_tensors
        slope, has_res = ctx.meta
        L = _lib.lib()
        rows, cols = x.shape[0], gamma.numel()
        dy = dy.contiguous()
        dz = _zeros(dy.shape) if dy.shape[1] != cols else _empty(dy.shape)
        dx = _zeros(x.shape) if x.shape[1] != cols else _empty(x.shape)
        sums = _empty(2, cols)
        check(L.pt_train_bn_bwd(ptr(dy), dy.shape[1], ptr(y), y.shape[1], slope, ptr(x), x.shape[1], ptr(mr), ptr(gamma), ptr(dz),
                                dz.shape[1], ptr(dx), dx.shape[1], ptr(sums), rows, cols, stream()))
        return dx, sums[1].clone(), sums[0].clone(), (dz if has_res else None), None, None, None, None


def bn_train(x, gamma, beta, run_mean, run_var, slope=-1.0, res=None, momentum=0.1):
    return BNTrain.apply(x, gamma, beta, res, slope, run_mean, run_var, momentum)


class Gate(torch.autograd.Function):
    """tanh(a) * sigmoid(b) on hv = [a | b] (gated_pixelcnn_1d.py:74-76)."""

    @staticmethod
    def forward(ctx, hv):
        L = _lib.lib()
        rows, C2 = hv.shape
        out = _empty(rows, C2 // 2)
        check(L.pt_train_gate_fwd(ptr(hv), rows, C2 // 2, ptr(out), stream()))
        ctx.save_for_backward(hv)
        return out

    @staticmethod
    def backward(ctx, dout):
        (hv,) = ctx.saved_tensors
        L = _lib.lib()
        dhv = _empty(hv.shape)
        check(L.pt_train_gate_bwd(ptr(dout.contiguous()), ptr(hv), hv.shape[0], hv.shape[1] // 2, ptr(dhv), stream()))
        return dhv


class EmbedPE(torch.autograd.Function):
    """x[row] = float(double(tok_emb[id]) + (PE[t+1] + PPE[g+1])) (PTransformer.py:447-474); gradient to tok_emb only
    (the sinusoid tables are frozen, PTransformer.py:243-245)."""

    @staticmethod
    def forward(ctx, ids32, tok, pe, ppe, N, G):
        L = _lib.lib()
        rows = ids32.numel()
        x = _empty(rows, 512)
        check(L.pt_embed_pe(ptr(ids32), ptr(tok), ptr(pe), ptr(ppe), ptr(x), rows, N, G, tok.shape[0], stream()))
        ctx.save_for_backward(ids32)
        ctx.vocab = tok.shape[0]
        return x

    @staticmethod
    def backward(ctx, dx):
        (ids32,) = ctx.saved_tensors
        L = _lib.lib()
        dE = _zeros(ctx.vocab, 512)
        check(L.pt_train_embed_bwd(ptr(dx.contiguous()), ptr(ids32), ids32.numel(), ctx.vocab, ptr(dE), stream()))
        return None, dE, None, None, None, None


class Dropout(torch.autograd.Function):
    """Inverted dropout with a counter-based mask that the backward pass replays from the seed."""

    @staticmethod
    def forward(ctx, x, p, seed):
        L = _lib.lib()
        y = _empty(x.shape)
        check(L.pt_train_dropout(ptr(x), ptr(y), x.numel(), p, seed, stream()))
        ctx.meta = (p, seed)
        return y

    @staticmethod
    def backward(ctx, dy):
        p, seed = ctx.meta
        L = _lib.lib()
        dy = dy.contiguous()
        dx = _empty(dy.shape)
        check(L.pt_train_dropout(ptr(dy), ptr(dx), dy.numel(), p, seed, stream()))
        return dx, None, None


class _Seeds:
    """Per-step dropout seed stream (host counter; the device never sees torch's RNG).  The rank of the process is folded
    into every seed when it is drawn, so data-parallel replicas draw independent masks (as nn.DataParallel's replicas do)
    whenever the process group was initialised; the position `n` is checkpointed by the wrappers."""

    def __init__(self, seed=0):
        self.base, self.n = int(seed) & 0xFFFFFFFF, 0

    def next(self):
        import torch.distributed as dist
        self.n += 1
        rank = dist.get_rank() if dist.is_available() and dist.is_initialized() else 0
        return (((self.base ^ (rank << 16)) & 0xFFFFFFFF) << 20) + self.n

    def state_dict(self):
        return {"base": self.base, "n": self.n}

    def load_state_dict(self, sd):
        self.base, self.n = int(sd["base"]), int(sd["n"])


def dropout(x, p, seeds):
    if p <= 0.0 or seeds is None:
        return x
    return Dropout.apply(x.contiguous(), float(p), seeds.next())


def ncl_to_rows(x_ncl, width=None):
    """(B, C, L) fp32 CUDA -> rows [B*L, round_up(C,32)] (pad columns zero); no gradient (inputs)."""
    L = _lib.lib()
    B, C, Ln = x_ncl.shape
    ld = width or _ru(C, 32)
    out = _empty(B * Ln, ld)
    check(L.pt_ncl_to_cl(ptr(x_ncl.contiguous()), ptr(out), B, C, Ln, ld, stream()))
    return out


class NCLToRows(torch.autograd.Function):
    """(B, C, L) -> rows [B*L, ld] (pad columns zero) with a gradient: the module API's tensors are channels-first, the
    kernels' are channels-last rows."""

    @staticmethod
    def forward(ctx, x, ld):
        B, C, Ln = x.shape
        out = _empty(B * Ln, ld)
        check(_lib.lib().pt_ncl_to_cl(ptr(x.contiguous()), ptr(out), B, C, Ln, ld, stream()))
        ctx.meta = (B, C, Ln, ld)
        return out

    @staticmethod
    def backward(ctx, dy):
        B, C, Ln, ld = ctx.meta
        dx = _empty(B, C, Ln)
        check(_lib.lib().pt_cl_to_ncl(ptr(dy.contiguous()), ld, ptr(dx), B, C, Ln, stream()))
        return dx, None


class RowsToNCL(torch.autograd.Function):
    """rows [B*L, ld] -> (B, C, L) (the first C columns) with a gradient."""

    @staticmethod
    def forward(ctx, rows, B, C, Ln):
        out = _empty(B, C, Ln)
        ld = rows.shape[1]
        check(_lib.lib().pt_cl_to_ncl(ptr(rows.contiguous()), ld, ptr(out), B, C, Ln, stream()))
        ctx.meta = (B, C, Ln, ld)
        return out

    @staticmethod
    def backward(ctx, dy):
        B, C, Ln, ld = ctx.meta
        d = _empty(B * Ln, ld)
        check(_lib.lib().pt_ncl_to_cl(ptr(dy.contiguous()), ptr(d), B, C, Ln, ld, stream()))
        return d, None, None, None


def to_rows(x_ncl, width=None):
    """ncl_to_rows for tensors that may carry a gradient."""
    ld = width or _ru(x_ncl.shape[1], 32)
    x = x_ncl.to(torch.float32)
    return NCLToRows.apply(x, ld) if x.requires_grad else ncl_to_rows(x, ld)


class PQQuantizeTrain(torch.autograd.Function):
    """ProductQuantization.forward in train mode, the differentiable part (vqvae_modules.py:470-487,536-544): nearest
    codes per sub-codebook (same fp32 search kernel as inference), commitment loss cc * mse(z, q), straight-through
    estimator.  z rows [B*W, G*D]; returns (q rows, loss, indices (B*W, G) int64)."""

    @staticmethod
    def forward(ctx, z, codebooks, commitment_cost):
        L = _lib.lib()
        rows, Cc = z.shape
        G, K, D = codebooks.shape
        q = _empty(rows, Cc)
        idx = torch.empty(rows, G, dtype=torch.int64, device=z.device)
        check(L.pt_pq_search_cl(ptr(z), Cc, ptr(codebooks), rows, G, D, K, ptr(idx), ptr(q), Cc, stream()))
        ss = _zeros(1)
        check(L.pt_train_sqdiff(ptr(z), ptr(q), z.numel(), ptr(ss), stream()))
        ctx.save_for_backward(z, q)
        ctx.cc = float(commitment_cost)
        ctx.mark_non_differentiable(idx)
        return q, ss[0] * (ctx.cc / z.numel()), idx

    @staticmethod
    def backward(ctx, dq, dloss, _didx):
        z, q = ctx.saved_tensors
        L = _lib.lib()
        dz = _empty(z.shape)
        g = dloss.reshape(1).contiguous() if dloss is not None else None
        dqc = dq.contiguous() if dq is not None else None
        check(L.pt_train_commit_bwd(ptr(dqc), ptr(z), ptr(q), ptr(g), 2.0 * ctx.cc / z.numel(), z.numel(), ptr(dz), stream()))
        return dz, None, None


def _tile_args(tile_noise, shape, need):
    """(noise pointer tensor or None, seed) for `_tile`'s noise (vqvae_modules.py:573-577): injected N(0,1) draws in the
    parity mode, else a seed for the kernel's own generator drawn from torch's CPU generator."""
    if tile_noise is not None:
        tn = tile_noise.to(device="cuda", dtype=torch.float32).contiguous()
        if tuple(tn.shape) != tuple(shape):
            raise RuntimeError(f"_tile noise must have shape {tuple(shape)}, got {tuple(tn.shape)}")
        return tn, 0
    return None, (int(torch.randint(0, 2 ** 62, (1,)).item()) if need else 0)


def pq_ema_update(z, idx, cs_hidden, dw_hidden, emb, decay, eps, counter, tile_noise=None):
    """EMA codebook update + dead-code re-seeding (vqvae_modules.py:513-534) in place on the stacked buffers
    cs_hidden [G,K], dw_hidden [G,K,D], emb [G,K,D]; z rows are the encoder output of this step, idx its codes.
    Fewer rows than codes: the seed rows are the noise-tiled batch (`_tile`); tile_noise [G,K,D] injects its N(0,1)."""
    L = _lib.lib()
    G, K, D = emb.shape
    counts, dw = _empty(G, K), _empty(G, K, D)
    tn, seed = _tile_args(tile_noise, (G, K, D), z.shape[0] < K)
    check(L.pt_train_pq_ema(ptr(z), z.shape[1], ptr(idx), z.shape[0], G, D, K, ptr(counts), ptr(dw), ptr(cs_hidden),
                            ptr(dw_hidden), ptr(emb), float(decay), float(eps), int(counter), ptr(tn), seed, stream()))


def pq_ema_update_shared(z, idx, G, cs_hidden, dw_hidden, emb, decay, eps, counter, tile_noise=None):
    """share_code=True (vqvae_modules.py:496-512): the chunks of all G groups update the ONE code book in place:
    cs_hidden [K], dw_hidden [K,D], emb [K,D]; z rows [B*W, G*D], idx (B*W, G)."""
    L = _lib.lib()
    K, D = emb.shape
    counts, dw = _empty(K), _empty(K, D)
    tn, seed = _tile_args(tile_noise, (K, D), z.shape[0] * G < K)
    check(L.pt_train_pq_ema_shared(ptr(z), z.shape[1], ptr(idx), z.shape[0], G, D, K, ptr(counts), ptr(dw), ptr(cs_hidden),
                                   ptr(dw_hidden), ptr(emb), float(decay), float(eps), int(counter), ptr(tn), seed, stream()))


def vq_ema_update(z, idx, cs_hidden, dw_hidden, emb, decay, eps, counter):
    """VectorQuantizerEMA's EMA codebook update (vqvae_modules.py:323-334, no re-seeding) in place on cs_hidden [K],
    dw_hidden [K,D], emb [K,D]; z rows [B*W, ld] are the encoder output of this step, idx (B*W, 1) its codes."""
    L = _lib.lib()
    K, D = emb.shape
    counts, dw = _empty(1, K), _empty(1, K, D)
    check(L.pt_train_vq_ema(ptr(z), z.shape[1], ptr(idx), z.shape[0], D, K, ptr(counts), ptr(dw), ptr(cs_hidden), ptr(dw_hidden),
                            ptr(emb), float(decay), float(eps), int(counter), stream()))


class VQLosses(torch.autograd.Function):
    """vq_teacher.get_loss (vq_teacher.py:184-232) without the commitment term: weighted smooth-L1 part losses +
    velocity L1.  Returns (total, sums) with sums = part means | velocity mean | total (device tensor, no gradient)."""

    @staticmethod
    def forward(ctx, pred, gt, B, Tn, bounds, weights, vel_cols, beta):
        L = _lib.lib()
        nparts = len(weights)
        sums = _zeros(nparts + 2)
        dpred = _zeros(pred.shape)
        check(L.pt_train_vq_losses(ptr(pred), pred.shape[1], ptr(gt), gt.shape[1], B, Tn, nparts,
                                   (C.c_int * (nparts + 1))(*bounds), (C.c_float * nparts)(*weights), vel_cols, beta,
                                   ptr(sums), ptr(dpred), dpred.shape[1], stream()))
        ctx.save_for_backward(dpred)
        ctx.mark_non_differentiable(sums)
        return sums[nparts + 1].clone(), sums

    @staticmethod
    def backward(ctx, g, _gs):
        (dpred,) = ctx.saved_tensors
        return dpred * g, None, None, None, None, None, None, None


class MaskedL1Losses(torch.autograd.Function):
    """refiner.get_loss (refiner.py:313-391): per-part L1 over the unmasked frames, weighted, + velocity L1.
    nmask: (B*T,) = 1 - mask per frame row.  Returns (total, sums) like VQLosses."""

    @staticmethod
    def forward(ctx, pred, gt, nmask, t_nmask, B, Tn, bounds, weights, vel_cols):
        L = _lib.lib()
        nparts = len(weights)
        sums = _zeros(nparts + 2)
        dpred = _zeros(pred.shape)
        check(L.pt_train_masked_l1_losses(ptr(pred), pred.shape[1], ptr(gt), gt.shape[1], ptr(nmask), float(t_nmask), B, Tn,
                                          nparts, (C.c_int * (nparts + 1))(*bounds), (C.c_float * nparts)(*weights),
                                          vel_cols, ptr(sums), ptr(dpred), dpred.shape[1], stream()))
        ctx.save_for_backward(dpred)
        ctx.mark_non_differentiable(sums)
        return sums[nparts + 1].clone(), sums

    @staticmethod
    def backward(ctx, g, _gs):
        (dpred,) = ctx.saved_tensors
        return dpred * g, None, None, None, None, None, None, None, None


# ---------------------------------------------------------------------------------------------------------------
# optimizer side: torch.nn.utils.clip_grad_norm_ + torch.optim.AdamW semantics on HIP kernels
# ---------------------------------------------------------------------------------------------------------------
MOMENT_BLOCK = 256      # values of an 8-bit moment that share a scale


def _on(device):
    """Launches go to the current stream of the tensors' device."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _same(what, tensors, dtypes, device=None):
    """The device of `tensors`, checked with their types and layout."""
    for t in tensors:
        if not torch.is_tensor(t) or not t.is_cuda:
            raise RuntimeError(f"{what}: tensors must be on the GPU")
        device = device or t.device
        if t.device != device:
            raise RuntimeError(f"{what}: tensors on {device} and {t.device}")
        if t.dtype not in dtypes:
            raise RuntimeError(f"{what}: {t.dtype} where {' or '.join(map(str, dtypes))} is taken")
        if not t.is_contiguous():
            raise RuntimeError(f"{what}: tensors must be contiguous")
    return device


def _addresses(tensors):
    return array.array("Q", map(torch.Tensor.data_ptr, tensors))


def _address(a):
    """An array.array as a pointer argument; the argument holds the array, which may have no other reference."""
    return None if a is None else (C.c_char * (len(a) * a.itemsize)).from_buffer(a)


def _grad_norm(pointers, sizes, is_bf16, n, max_norm, device, ws_bytes=None):
    """A device tensor [norm, coef]; pointers and sizes from _address."""
    L = _lib.lib()
    if ws_bytes is None:
        ws_bytes = L.pt_train_grad_norm_workspace_bytes(sizes, n)
    out = torch.empty(2, device=device, dtype=torch.float32)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    at = out.data_ptr()
    check(L.pt_train_grad_norm(pointers, sizes, is_bf16, n, max_norm, at, at + 4, ws.data_ptr(), ws_bytes, stream()))
    return out


def grad_norm(grads, max_norm):
    """(norm, coef), two device tensors of one float: the norm over all of `grads` (fp32 or bf16) and the factor
    min(1, max_norm / (norm + 1e-6)) of torch.nn.utils.clip_grad_norm_, NaN where the norm is.  The sum runs in fp64 in a fixed order."""
    grads = [g.contiguous() for g in grads]
    device = _same("grad_norm", grads, (torch.float32, torch.bfloat16)) if grads else torch.device("cuda", torch.cuda.current_device())
    kinds = None
    if any(g.dtype is torch.bfloat16 for g in grads):
        kinds = bytes(g.dtype is torch.bfloat16 for g in grads)
    with _on(device):
        out = _grad_norm(_address(_addresses(grads)), _address(array.array("q", [g.numel() for g in grads])), kinds, len(grads), float(max_norm), device)
    return out[:1], out[1:]


def clip_grad_norm(params, max_norm):
    """Scales the gradients' effect by min(1, max_norm / (total_norm + 1e-6)); returns (total_norm tensor, coef tensor).
    The coefficient stays on the device and is applied inside the AdamW kernel (no extra pass over the gradients)."""
    return grad_norm([p.grad for p in params if p.grad is not None], max_norm)


def _overlap(tensors):
    """Whether two of these contiguous tensors share memory."""
    at = sorted((t.data_ptr(), t.numel() * t.element_size()) for t in tensors if t.numel())
    return any([a + n > b for (a, n), (b, _) in zip(at, at[1:])])


class AdamWList:
    """AdamW over a fixed list of tensors, a few launches a step whatever their number.

    params: fp32, or bf16 (then rounded stochastically).  exp_avgs, exp_avg_sqs: fp32 tensors of the parameters' sizes; or, with
    `scales`, uint8 tensors of these sizes (8-bit moments) and one fp32 tensor (ceil(n / 256), 2) each: the scales of every block
    of 256 values for the first and the second moment.  Zeros everywhere stand for moments of zero.  `moment_values` gives what
    8-bit moments stand for.  All are updated in place; the list keeps their memory, so it does not follow a tensor whose
    `.data` is exchanged afterwards.  Two steps of one list must not run at the same time on two streams."""

    def __init__(self, params, exp_avgs, exp_avg_sqs, scales=None):
        lists = [[t.detach() for t in x] for x in ((params, exp_avgs, exp_avg_sqs) if scales is None else
                                                   (params, exp_avgs, exp_avg_sqs, scales))]
        params, exp_avgs, exp_avg_sqs = lists[:3]
        if not params or any(len(x) != len(params) for x in lists):
            raise RuntimeError(f"AdamWList: lists of {', '.join(str(len(x)) for x in lists)} tensors")
        self.dtype = params[0].dtype
        self.device = _same("AdamWList", params, (torch.float32, torch.bfloat16))
        _same("AdamWList", params, (self.dtype,))
        _same("AdamWList", exp_avgs + exp_avg_sqs, (torch.float32 if scales is None else torch.uint8,), self.device)
        for i, p in enumerate(params):
            if not p.numel() == exp_avgs[i].numel() == exp_avg_sqs[i].numel():
                raise RuntimeError(f"AdamWList: tensor {i} has {p.numel()} values, its moments {exp_avgs[i].numel()} and {exp_avg_sqs[i].numel()}")
        if scales is not None:
            _same("AdamWList", lists[3], (torch.float32,), self.device)
            for p, s in zip(params, lists[3]):
                if tuple(s.shape) != (-(-p.numel() // MOMENT_BLOCK), 2):
                    raise RuntimeError(f"AdamWList: {p.numel()} values have scales of shape {(-(-p.numel() // MOMENT_BLOCK), 2)}, not {tuple(s.shape)}")
        self._lists = lists                  # holds the memory behind the addresses
        self._arrays = [_addresses(x) for x in lists] + ([None] if scales is None else [])
        for a in self._arrays:
            used = [x for x in a or () if x]
            if len(set(used)) != len(used):
                raise RuntimeError("AdamWList: the same tensor twice")
        if _overlap([t for x in lists for t in x]):
            raise RuntimeError("AdamWList: two tensors share memory")
        self.sizes = [p.numel() for p in params]
        self._n = array.array("q", self.sizes)
        self._bf16 = int(self.dtype is torch.bfloat16)
        self._kinds = b"\1" * len(params) if self._bf16 else None
        self._pointers = [*map(_address, self._arrays), _address(self._n)]
        self._norm_ws = _lib.lib().pt_train_grad_norm_workspace_bytes(self._pointers[-1], len(params))

    def __reduce__(self):                    # a copy has memory, and so addresses, of its own
        return type(self), tuple(self._lists)

    def step(self, grads, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, coef=None, max_norm=None, seed=0):
        """One step with `grads` (of the parameters' type and sizes).  coef: device scalar that scales the gradients; max_norm
        instead: the coefficient of this list's own gradient norm, which is then returned.  step: the count of this step, from
        1; or a CUDA int32 tensor of one value that holds it, read when the step runs (a captured step needs that: the
        caller adds 1 to it inside the capture).  seed: of the random bits of stochastic roundings."""
        if not torch.is_tensor(step):
            with _on(self.device):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("AdamWList.step: a captured step would repeat one step count: pass `step` as a CUDA int32 tensor")
        return self._step(grads, step, lr, betas, eps, weight_decay, coef, max_norm, seed)

    def _step(self, grads, step, lr, betas, eps, weight_decay, coef=None, max_norm=None, seed=0):
        if len(grads) != len(self.sizes):
            raise RuntimeError(f"AdamWList.step: {len(grads)} gradients for {len(self.sizes)} parameters")
        if not all(map(torch.Tensor.is_contiguous, grads)):
            grads = [g.contiguous() for g in grads]
        if list(map(torch.Tensor.numel, grads)) != self.sizes:
            raise RuntimeError("AdamWList.step: a gradient has another size than its parameter")
        if set(map(torch.Tensor.get_device, grads)) != {self.device.index} or not all([g.dtype is self.dtype for g in grads]):
            raise RuntimeError(f"AdamWList.step: gradients must be {self.dtype} on {self.device}")
        if coef is not None and max_norm is not None:
            raise RuntimeError("AdamWList.step: coef or max_norm, not both")
        on_device = torch.is_tensor(step)
        if on_device:
            _same("AdamWList.step", [step], (torch.int32,), self.device)
            if step.numel() != 1:
                raise RuntimeError("AdamWList.step: step is one value")
        elif step < 1:
            raise RuntimeError(f"AdamWList.step: steps count from 1, got {step}")
        if coef is not None:
            _same("AdamWList.step", [coef], (torch.float32,), self.device)
            if coef.numel() != 1:
                raise RuntimeError("AdamWList.step: coef is one value")
        norm = dyn = None
        scale = _at(coef)
        with _on(self.device):
            g = _address(_addresses(grads))
            if max_norm is not None:
                out = _grad_norm(g, self._pointers[-1], self._kinds, len(grads), float(max_norm), self.device, self._norm_ws)
                norm, scale = out[:1], out.data_ptr() + 4
            if on_device:
                dyn = torch.empty(3, device=self.device, dtype=torch.float32)
            check(_lib.lib().pt_train_adamw_multi(self._pointers[0], g, *self._pointers[1:], len(grads), self._bf16, scale, lr, *betas, eps,
                                                  weight_decay, 0 if on_device else step, _at(step) if on_device else None, _at(dyn),
                                                  seed & 0xFFFFFFFF, stream()))
        return norm


def moment_values(exp_avg, exp_avg_sq, scale):
    """The fp32 values that the 8-bit moments of one tensor stand for (see AdamWList)."""
    device = _same("moment_values", [exp_avg, exp_avg_sq], (torch.uint8,))
    _same("moment_values", [scale], (torch.float32,), device)
    n = exp_avg.numel()
    if exp_avg_sq.numel() != n or tuple(scale.shape) != (-(-n // MOMENT_BLOCK), 2):
        raise RuntimeError(f"moment_values: {n} and {exp_avg_sq.numel()} codes with scales of shape {tuple(scale.shape)}")
    m, v = (torch.empty(t.shape, device=device, dtype=torch.float32) for t in (exp_avg, exp_avg_sq))
    with _on(device):
        check(_lib.lib().pt_train_moment_values(ptr(exp_avg), ptr(exp_avg_sq), ptr(scale), n, ptr(m), ptr(v), stream()))
    return m, v


class AdamW:
    """torch.optim.AdamW (amsgrad off) on the library's kernel; state_dict()/load_state_dict() use torch's layout.
    state_bits = 8 holds the moments in a byte each (AdamWList), with a third state tensor 'scale'; its stochastic rounding
    draws from `seed`.  A captured step keeps the step count that it was captured with, in every replay (AdamWList.step takes a
    count that lives on the device); where it would round stochastically it is refused, for its random bits would repeat."""

    def __init__(self, param_groups, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32, got {state_bits!r}")
        self.param_groups = [dict(params=list(g["params"]), lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay)
                             for g in param_groups]
        self.state = {}
        self.state_bits, self.seed = state_bits, int(seed)
        self._lists = {}

    def __getstate__(self):                  # lists are made anew where they are needed
        return self.__dict__ | {"_lists": {}}

    def __setstate__(self, state):
        self.__dict__.update({"state_bits": 32, "seed": 0, "_lists": {}} | state)

    def zero_grad(self):
        for g in self.param_groups:
            for p in g["params"]:
                p.grad = None

    def _names(self):
        return ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else ("exp_avg", "exp_avg_sq", "scale")

    def _state(self, p):
        st = self.state.get(p)
        if st is None:
            if self.state_bits == 32:
                st = {k: torch.zeros(p.shape, device=p.device, dtype=torch.float32) for k in ("exp_avg", "exp_avg_sq")}
            else:
                st = {k: torch.zeros(p.shape, device=p.device, dtype=torch.uint8) for k in ("exp_avg", "exp_avg_sq")}
                st["scale"] = torch.zeros(-(-p.numel() // MOMENT_BLOCK), 2, device=p.device, dtype=torch.float32)
            st = self.state[p] = {"step": 0} | st
        if not p.is_cuda:
            raise RuntimeError("AdamW.step: parameters must be on the GPU")
        for k in self._names():                    # state restored before the module moved to the GPU
            if st[k].device != p.device:
                st[k] = st[k].to(p.device)
        return st

    def _list(self, ps, sts):
        """The AdamWList of these parameters: made once, and anew where a parameter's or a moment's memory is another.  None where
        parameters share memory."""
        key = tuple(map(id, ps))
        held = [x for k in self._names() for x in map(torch.Tensor.data_ptr, [st[k] for st in sts])] + list(map(torch.Tensor.data_ptr, ps))
        made = self._lists.get(key)
        if made is None or made[1] != held:
            if len(self._lists) >= 32 + 4 * len(self.param_groups):      # more than the lists that steps come back to
                self._lists.clear()
            apart = len(ps) == 1 or not _overlap(ps)
            made = self._lists[key] = (AdamWList(ps, *([st[k] for st in sts] for k in self._names())) if apart else None, held, ps)
        return made[0]

    def step(self, coefs=None):
        """coefs: optional {param: device scalar} of clip coefficients."""
        for gi, g in enumerate(self.param_groups):
            parts = {}
            for p in g["params"]:
                if p.grad is None:
                    continue
                st = self._state(p)
                c = None if coefs is None else coefs.get(p)
                part = parts.setdefault((id(c), st["step"], p.dtype, p.device), (c, [], []))
                part[1].append(p)
                part[2].append(st)
            for k, ((_, done, dtype, device), (c, ps, sts)) in enumerate(parts.items()):
                with _on(device):
                    if (self.state_bits == 8 or dtype is torch.bfloat16) and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("AdamW.step: a captured step would repeat its random bits: use AdamWList.step with a step count on the device")
                hyper = (g["lr"], g["betas"], g["eps"], g["weight_decay"], c, None, self.seed + 0x10001 * gi + 0x1000003 * k)
                whole = self._list(ps, sts)
                if whole is not None:
                    whole._step([p.grad for p in ps], done + 1, *hyper)
                    for st in sts:
                        st["step"] = done + 1
                    continue
                for p, st in zip(ps, sts):         # parameters that share memory: one after the other, as they come
                    self._list([p], [st])._step([p.grad], st["step"] + 1, *hyper)
                    st["step"] += 1

    def state_dict(self):
        idx, packed, groups = {}, {}, []
        for g in self.param_groups:
            ids = []
            for p in g["params"]:
                idx[p] = len(idx)
                ids.append(idx[p])
            groups.append({k: v for k, v in g.items() if k != "params"} | {"params": ids})
        for p, st in self.state.items():
            packed[idx[p]] = {"step": torch.tensor(float(st["step"]))} | {k: st[k] for k in self._names()}
        return {"state": packed, "param_groups": groups}

    def load_state_dict(self, sd):
        flat = [p for g in self.param_groups for p in g["params"]]
        self._lists.clear()                        # they hold the moments that are replaced
        for i, st in sd.get("state", {}).items():
            p = flat[int(i)]
            if self.state_bits == 8:
                if "scale" not in st:
                    raise RuntimeError("AdamW: a state with moments in 32 bits cannot be loaded with state_bits=8")
                new = {k: st[k].to(p.device).clone(memory_format=torch.contiguous_format) for k in self._names()}
            elif "scale" in st:                    # moments saved in 8 bits: what they stand for
                m, v = moment_values(*(st[k].to("cuda") for k in ("exp_avg", "exp_avg_sq", "scale")))
                new = {"exp_avg": m.to(p.device), "exp_avg_sq": v.to(p.device)}
            else:
                new = {k: st[k].to(p.device).float().clone(memory_format=torch.contiguous_format) for k in self._names()}
            self.state[p] = {"step": int(float(st["step"]))} | new
        for g, sg in zip(self.param_groups, sd.get("param_groups", [])):
            for k in ("lr", "betas", "eps", "weight_decay"):
                if k in sg:
                    g[k] = tuple(sg[k]) if k == "betas" else sg[k]

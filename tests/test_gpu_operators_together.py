"""gated_norm, windowed attention and the optimizer's list as a block of a network uses them: norm, projection, attention, projection,
gated residual sum with the next norm; gradients, clipping, one step with 8-bit moments, and the same block token by token over a cache."""
import math

import pytest
import torch

from probtalk_amd import train_ops as T

pytestmark = pytest.mark.gpu

C, H, HK, D = 128, 4, 2, 32
LEFT, SINKS, EPS = 24, 3, 1e-5


def parameters(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s, scale=1.0, shift=0.0: torch.randn(*s, device="cuda", generator=g) * scale + shift  # noqa: E731
    return {"pre.weight": n(C, scale=0.1, shift=1.0), "pre.bias": n(C, scale=0.1), "qkv.weight": n((H + 2 * HK) * D, C, scale=C ** -0.5),
            "qkv.bias": n((H + 2 * HK) * D, scale=0.1), "out.weight": n(C, H * D, scale=(H * D) ** -0.5), "out.bias": n(C, scale=0.1),
            "scale": n(C, scale=0.1, shift=0.5), "post.weight": n(C, scale=0.1, shift=1.0), "post.bias": n(C, scale=0.1),
            "next.weight": n(C, scale=0.1, shift=1.0), "next.bias": n(C, scale=0.1)}


def block(P, x, gate, B, N, lengths):
    _, h = T.gated_norm(x, pre_weight=P["pre.weight"], pre_bias=P["pre.bias"], eps=EPS)
    qkv = T.conv(h, P["qkv.weight"], P["qkv.bias"], 0, B, N).view(B, N, H + 2 * HK, D)
    q, k, v = qkv.split((H, HK, HK), 2)
    o = T.window_attention(q, k, v, LEFT, sinks=SINKS, lengths=lengths)
    t = T.conv(o.reshape(B * N, H * D), P["out.weight"], P["out.bias"], 0, B, N)
    y, h2 = T.gated_norm(x, t, gate, P["scale"], P["post.weight"], P["post.bias"], P["next.weight"], P["next.bias"], rows_per_clip=N, eps=EPS)
    return y, h2, q, k, v, o


def plain(P, x, gate, B, N, lengths):
    norm = lambda r, w, b: (r - r.mean(1, keepdim=True)) / (r.var(1, correction=0, keepdim=True) + EPS).sqrt() * w + b  # noqa: E731
    qkv = (norm(x, P["pre.weight"], P["pre.bias"]) @ P["qkv.weight"].T + P["qkv.bias"]).view(B, N, H + 2 * HK, D)
    q, k, v = (u.transpose(1, 2).repeat_interleave(H // u.shape[2], 1) for u in qkv.split((H, HK, HK), 2))
    i = torch.arange(N, device=x.device)
    see = (i[None] <= i[:, None]) & ((i[None] >= i[:, None] - LEFT) | (i[None] < SINKS))
    see = see[None, None] & (i < lengths.view(-1, 1, 1, 1))
    s = (q @ k.transpose(2, 3).contiguous() / math.sqrt(D)).masked_fill(~see, -math.inf)
    e = (s - s.detach().amax(-1, keepdim=True).clamp_min(-1e30)).exp()
    o = (e / e.sum(-1, keepdim=True).clamp_min(1e-30)) @ v
    t = o.transpose(1, 2).reshape(B * N, H * D) @ P["out.weight"].T + P["out.bias"]
    y = x + P["scale"] * gate.repeat_interleave(N, 0) * norm(t, P["post.weight"], P["post.bias"])
    return y, norm(y, P["next.weight"], P["next.bias"])


def leaves(P, x, gate, to=lambda t: t):
    return {n: to(t.detach()).requires_grad_() for n, t in {**P, "x": x, "gate": gate}.items()}


def inputs(B, N):
    g = torch.Generator(device="cuda").manual_seed(5)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return n(B * N, C), 1.0 + 0.2 * n(B, C), n(B * N, C), n(B * N, C)


@pytest.mark.parametrize("B,N,lengths", [(2, 150, [150, 61]), (1, 1, [1]), (3, 33, [33, 0, 5])])
def test_a_block_its_gradients_and_a_step(B, N, lengths):
    P, (x, gate, gy, gh) = parameters(1), inputs(B, N)
    lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def both(f, to):
        p = leaves(P, x, gate, to)
        y, h = f(p, p["x"], p["gate"], B, N, lengths.to(p["x"].device))[:2]
        grads = torch.autograd.grad((y * to(gy)).sum() + (h * to(gh)).sum(), list(p.values()))
        return {"y": y.detach(), "h": h.detach(), **dict(zip(p, grads))}

    got, want, rough = both(block, lambda t: t.clone()), both(plain, lambda t: t.double()), both(plain, lambda t: t.cpu())
    for n in want:
        # the plain form in fp32 makes the same roundings and others in the order of its sums: four times its error, and 2^-21 of the
        # whole for values that it happens to hit
        far = lambda a: float((a[n].double().to("cuda") - want[n]).norm())  # noqa: E731
        assert far(got) <= 4 * far(rough) + 2.0 ** -21 * float(want[n].norm()) + 1e-12, (n, far(got), far(rough), float(want[n].norm()))

    # clipping and a first step with 8-bit moments: p - lr (wd p + g / (|g| + eps)) with g the clipped gradient
    ps = [torch.nn.Parameter(P[n].clone()) for n in P]
    for p, n in zip(ps, P):
        p.grad = got[n]
    lr, wd, eps = 1e-2, 0.1, 1e-8
    opt = T.AdamW([{"params": ps}], lr=lr, weight_decay=wd, eps=eps, state_bits=8)
    norm, coef = T.clip_grad_norm(ps, 0.5)
    total = math.sqrt(sum(float(got[n].double().square().sum()) for n in P))
    assert abs(float(norm) - total) <= 2.0 ** -23 * total
    assert abs(float(coef) - min(1.0, 0.5 / (total + 1e-6))) <= 2.0 ** -21
    opt.step({p: coef for p in ps})
    for p, n in zip(ps, P):
        g = got[n].double() * float(coef)
        # m / (1 - b1) and v / (1 - b2) are g and g^2 but for a few roundings (1 - b2 is 2^-14 off its own value in fp32); where eps matters the
        # quotient is between 0 and 1 all the same
        step = g / (g.abs() + eps)
        err = (p.detach().double() - (P[n].double() * (1 - lr * wd) - lr * step)).abs()
        assert bool((err <= 2.0 ** -22 * P[n].abs() + lr * 2.0 ** -12).all()), (n, float(err.max()))


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused_not_dropped(grad):
    from torch.autograd import forward_ad
    x, w = torch.randn(8, 64, device="cuda"), torch.ones(64, device="cuda")
    q, lengths = torch.randn(1, 4, 2, 32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for f in (lambda: T.gated_norm(dual(x), pre_weight=w), lambda: T.gated_norm(x, x.clone(), post_weight=dual(w), pre_weight=w),
                  lambda: T.window_attention(dual(q), q, q), lambda: T.window_attention(q, q, dual(q)),
                  lambda: T.window_attention_step(q[:, 0], q, dual(q), lengths)):
            with pytest.raises(NotImplementedError, match="forward mode"):
                f()
        T.gated_norm(x, pre_weight=w)                      # without tangents they run
        T.window_attention(q, q, q)
        T.window_attention_step(q[:, 0], q, q, lengths)


def test_second_derivatives_are_refused_not_left_out():
    x, b = (torch.randn(s, device="cuda", requires_grad=True) for s in ((8, 64), (64,)))
    q = torch.randn(1, 4, 2, 32, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda")
    for leaf, f in ((x, lambda: T.gated_norm(x, pre_weight=w)[1]), (b, lambda: T.gated_norm(x.detach(), pre_weight=w, pre_bias=b)[1]),
                    (q, lambda: T.window_attention(q, q.detach(), q.detach()))):
        first = torch.autograd.grad(f().square().sum(), leaf)[0]
        loss = f().square().sum()
        d, = torch.autograd.grad(loss, leaf, create_graph=True)
        assert torch.equal(d, first)
        with pytest.raises(RuntimeError, match="second derivatives"):
            (loss + d.square().sum()).backward()
        leaf.grad = None                                   # the part of `loss` may have arrived before
        f().square().sum().backward(create_graph=True)     # without them nothing is refused
        assert torch.equal(leaf.grad, first)
        leaf.grad = None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_by_token_over_a_cache(dtype):
    """The block's attention for the last token of growing sequences: what window_attention gives for that row."""
    B, N = 2, 90
    P, (x, gate, _, _) = parameters(2), inputs(2, 90)
    full = torch.full((B,), N, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        q, k, v, o = block(P, x, gate, B, N, full)[2:]
        if dtype is torch.bfloat16:
            q, k, v = (t.to(dtype) for t in (q, k, v))
            o = T.window_attention(q, k, v, LEFT, sinks=SINKS)
        cache = torch.full((2, B, N + 7, HK, D), math.nan, device="cuda", dtype=dtype)
        lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
        # both round: fp32 their sums of up to 28 products of D terms, bf16 a probability and the result (half a step of 2^-8 each)
        tol = 2.0 ** -17 if dtype is torch.float32 else 4 * 2.0 ** -8
        most = float(v.abs().max())
        for i in range(N):
            cache[0, :, i], cache[1, :, i] = k[:, i], v[:, i]
            lengths += 1
            got = T.window_attention_step(q[:, i], cache[0], cache[1], lengths, LEFT, sinks=SINKS)
            err = float((got.float() - o[:, i].float()).abs().max())
            assert err <= tol * most, (i, err)

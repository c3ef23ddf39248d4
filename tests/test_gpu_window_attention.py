"""window_attention (pt_attention_window_fwd / _bwd) and window_attention_step against the definition in 64 bits, with bounds that
follow every rounding of the kernels."""
import math

import pytest
import torch

from probtalk_amd import train_ops as T

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                                  # half a step of fp32
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
# batch, rows, keys, heads, key heads, channels, left, right, sinks, lengths
CASES = {
    "one": (1, 1, 1, 1, 1, 8, 0, 0, 0, None),
    "itself only": (2, 33, 33, 2, 1, 64, 0, 0, 0, None),
    "sinks in the window's tile": (2, 33, 33, 2, 1, 64, 8, 0, 2, None),
    "two row tiles": (1, 130, 130, 4, 2, 128, 40, 0, 4, None),
    "both sides, padded": (3, 200, 200, 2, 2, 40, 16, 16, 0, [200, 77, 1]),
    "a new part of a sequence": (1, 5, 77, 8, 2, 96, 30, 0, 3, None),
    "everything": (2, 64, 64, 1, 1, 64, None, None, 0, None),
    "causal, no limit": (1, 300, 300, 2, 1, 32, None, 0, 0, None),
    "far rows": (1, 700, 700, 2, 1, 64, 50, 0, 5, None),
    "many chunks of far rows, two blocks of sinks": (1, 1500, 1500, 2, 2, 128, 100, 3, 40, None),
    "far rows of a new part": (2, 600, 900, 4, 1, 64, 20, 0, 7, [900, 450]),
    "as many sinks as allowed, an empty sequence": (3, 300, 300, 4, 4, 64, 10, 10, 128, [300, 0, 129]),
    "more sinks than keys": (1, 20, 20, 2, 2, 8, 3, 0, 64, None),
    "group of 8": (1, 260, 260, 8, 1, 80, 64, 0, 4, [259]),
    "window of whole tiles": (1, 512, 512, 1, 1, 128, 127, 0, 0, None),
    "padded rows see sinks only or nothing": (2, 256, 256, 2, 1, 64, 5, 0, 1, [3, 0]),
}


# sinks in two blocks of keys and rows far behind them; key heads that share out over the chip evenly, sequences of all lengths
MORE = {
    "many sinks, far rows": (1, 900, 900, 2, 1, 64, 70, 0, 100, None),
    "sinks beyond a block, a new part": (2, 700, 1000, 4, 2, 48, 30, 5, 65, [1000, 333]),
    "eight key heads, padded": (4, 300, 300, 4, 2, 64, 90, 90, 0, [300, 1, 170, 64]),
    "a whole sequence in view": (1, 800, 800, 8, 8, 32, None, 0, 0, None),
}


def make(case, dtype, seed=0):
    B, Nq, Nk, H, Hk, D, left, right, sinks, lengths = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s, scale=1.0: (torch.randn(*s, device="cuda", generator=g) * scale).to(dtype).requires_grad_()  # noqa: E731
    q, k, v, do = n(B, Nq, H, D, scale=1.5), n(B, Nk, Hk, D), n(B, Nk, Hk, D), n(B, Nq, H, D).detach()
    return q, k, v, do, None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")


def oracle(q, k, v, do, left, right, sinks, lengths, scale=None):
    """The outputs by matrix products in 64 bits, and how far the kernels' roundings can move each of them."""
    half = HALF[q.dtype]
    B, Nq, H, D = q.shape
    Nk, Hk = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    big = lambda t: t.detach().double().transpose(1, 2).repeat_interleave(H // t.shape[2], 1)  # noqa: E731   (B, H, N, D)
    Q, K, V, G = big(q), big(k), big(v), big(do)
    t = torch.arange(Nk - Nq, Nk, device="cuda")[:, None]
    j = torch.arange(Nk, device="cuda")[None]
    far = 1 << 30
    see = (j <= t + (far if right is None else right)) & ((j >= t - (far if left is None else left)) | (j < sinks))
    see = see[None, None] if lengths is None else see[None, None] & (j[None, None] < lengths.view(-1, 1, 1, 1))
    s = (Q @ K.transpose(2, 3) * scale).masked_fill(~see, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(-1e300)
    e = (s - top).exp()
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    o = p @ V
    # relative errors of p: the products of a score (its sum passes D additions), the exponent's own rounding and 2^-22 of exp2, the sum
    size = (Q.abs() @ K.abs().transpose(2, 3) * scale).masked_fill(~see, 0.0)
    ep = U * (2 * (D + 4) * size.amax(-1, keepdim=True) + Nk / 8 + 64)
    if q.dtype is torch.float32:
        half_p = U
    else:
        half_p = 2.0 ** -8
    pv = p @ V.abs()
    eo = (ep + half_p + Nk * U) * pv
    out = {"o": o, "q": None, "k": None, "v": None}
    tol = {"o": eo + half * (o.abs() + eo)}
    dp, delta = G @ V.transpose(2, 3), (G * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    g_abs = G.abs()
    e_delta = (g_abs * tol["o"]).sum(-1, keepdim=True) + D * U * (g_abs * o.abs()).sum(-1, keepdim=True)
    e_dp = (D + 4) * U * (g_abs @ V.abs().transpose(2, 3))
    e_ds = p * ((1 + ep) * (e_dp + e_delta) + (ep + 4 * U) * (dp.abs() + delta.abs())) + half_p * ds.abs()
    join = lambda x: x.view(B, Hk, H // Hk, Nk, D).sum(2)  # noqa: E731
    out["q"], e_q = scale * ds @ K, scale * (e_ds + Nk * U * ds.abs()) @ K.abs()
    rows = Nq * (H // Hk) * U
    dsT, e_dsT, pT = ds.transpose(2, 3), (e_ds + rows * ds.abs()).transpose(2, 3), p.transpose(2, 3)
    out["k"], e_k = scale * join(dsT @ Q), scale * join(e_dsT @ Q.abs())
    out["v"], e_v = join(pT @ G), join((pT * 0 + (p * (ep + half_p + rows)).transpose(2, 3)) @ g_abs)
    for n, e in (("q", e_q), ("k", e_k), ("v", e_v)):
        tol[n] = e + half * (out[n].abs() + e) + 1e-30
    tol["o"] = tol["o"] + 1e-30
    return {n: x.transpose(1, 2) for n, x in out.items()}, {n: x.transpose(1, 2) for n, x in tol.items()}, see


def grads(q, k, v, do, case, lengths, scale=None):
    o = T.window_attention(q, k, v, case[6], case[7], sinks=case[8], lengths=lengths, scale=scale)
    return dict(zip("oqkv", (o.detach(), *torch.autograd.grad(o, (q, k, v), do))))


def check(got, want, tol):
    for n in want:
        err = (got[n].double() - want[n]).abs()
        assert got[n].shape == want[n].shape and bool(torch.isfinite(got[n]).all()), n
        assert bool((err <= tol[n]).all()), (n, float((err - tol[n]).max()), float((err / tol[n]).max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", sorted(CASES | MORE))
def test_forward_and_gradients(name, dtype):
    case = (CASES | MORE)[name]
    q, k, v, do, lengths = make(case, dtype)
    want, tol, see = oracle(q, k, v, do, *case[6:9], lengths)
    got = grads(q, k, v, do, case, lengths)
    check(got, want, tol)
    blind = ~see.any(-1).any(1).expand(q.shape[0], -1)            # (B, Nq): rows that see nothing
    assert bool((got["o"][blind] == 0).all()) and bool((got["q"][blind] == 0).all())
    if lengths is not None:                                       # keys behind a sequence get no gradient
        behind = torch.arange(k.shape[1], device="cuda")[None] >= lengths[:, None]
        assert bool((got["k"][behind] == 0).all()) and bool((got["v"][behind] == 0).all())
    again = grads(q, k, v, do, case, lengths)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("left", [2, 8, 100])
def test_gradients_of_few_keys_do_not_feel_the_rounding_of_the_output(left):
    """bf16.  Two roundings reach dQ and dK: of the factors in front of keys and queries, and of the result; delta is taken from an
    output that is rounded to 24 bits.  Each rounding is uniform within half a step, so its mean square is at most
    (2^-8)^2 / 3 of the value's; the roundings are independent, and a mean over 50,000 values is within a tenth of its expectation
    (delta from the rounded output: 1.6 times the bound for left = 2)."""
    case = (2, 400, 400, 2, 1, 64, left, 0, 0, None)
    q, k, v, do, _ = make(case, torch.bfloat16)
    got = grads(q, k, v, do, case, None)
    big = lambda t: t.detach().double().transpose(1, 2).repeat_interleave(2 // t.shape[2], 1)  # noqa: E731
    Q, K, V, G = big(q), big(k), big(v), big(do)
    i = torch.arange(400, device="cuda")
    far = (i[None] > i[:, None]) | (i[None] < i[:, None] - left)
    p = (Q @ K.transpose(2, 3) / 8).masked_fill(far, -math.inf).softmax(-1)
    ds = p * (G @ V.transpose(2, 3) - (G * (p @ V)).sum(-1, keepdim=True)) / 8
    e = (2.0 ** -8) ** 2 / 3
    join = lambda x: x.view(2, 1, 2, 400, 64).sum(2)  # noqa: E731
    for n, want, square in (("q", ds @ K, ds.square() @ K.square()),
                            ("k", join(ds.transpose(2, 3) @ Q), join(ds.square().transpose(2, 3) @ Q.square()))):
        err = (got[n].double().transpose(1, 2) - want).square().sum()
        assert float(err) <= 1.1 * e * float(square.sum() + want.square().sum()), (n, float(err / (e * (square.sum() + want.square().sum()))))


@pytest.mark.parametrize("D", [32, 128])
def test_gradients_of_short_sequences_are_rounded_once(D):
    """bf16, at most 32 keys: the factors of the second products are held in 16 bits, so that only the results' rounding is left; its mean
    square is at most (2^-8)^2 / 3 of the value's, and what comes before is 2^-8 of it."""
    case = (5, 29, 29, 4, 2, D, 6, 0, 2, None)
    q, k, v, do, _ = make(case, torch.bfloat16)
    want = oracle(q, k, v, do, *case[6:9], None)[0]
    got = grads(q, k, v, do, case, None)
    for n in "oqkv":
        err, size = (got[n].double() - want[n]).square().sum(), want[n].square().sum()
        assert float(err) <= 1.02 * (2.0 ** -8) ** 2 / 3 * float(size), (n, float(err / size) ** 0.5)


def rounded_once(got, want, what):
    """bf16: results that are off by d before their one rounding are off by |round(x) - x| + 2 |d| at most after it.  d is 2^-14 of the whole:
    the factors of the second products and the output in delta are held in 16 bits or more (2^-17 and 2^-16 of each), fp32 sums add less."""
    size, ideal = float(want.norm()), float((want.to(torch.bfloat16).double() - want).norm())
    err = float((got.double() - want).norm())
    assert err <= ideal + 2 * 2.0 ** -14 * size, (what, err, ideal, size)


ONCE = {
    "many keys": (1, 1500, 1500, 4, 1, 128, 1023, 0, 4, None),
    "sinks and far rows": (1, 900, 900, 4, 2, 64, 300, 0, 40, None),
    "short sequences in a padded batch": (4, 200, 200, 2, 1, 64, None, 0, 0, [20, 200, 3, 32]),
    "short sequences, wide heads": (3, 130, 130, 4, 2, 128, 40, 40, 0, [7, 130, 31]),
}


@pytest.mark.parametrize("sharp", [1.0, 6.0])
@pytest.mark.parametrize("name", sorted(ONCE))
def test_results_are_rounded_once(name, sharp):
    """bf16: outputs and gradients of every sequence, whatever its length and that of its neighbours, as far from 64 bits as one rounding.
    sharp: scores that leave most of a row's weight to a few of its many keys, so that roundings of probabilities do not average out."""
    case = ONCE[name]
    q, k, v, do, lengths = make(case, torch.bfloat16)
    with torch.no_grad():
        q.mul_(sharp)
    want, _, see = oracle(q, k, v, do, *case[6:9], lengths)
    got = grads(q, k, v, do, case, lengths)
    for b in range(case[0]):
        for n in "oqkv":
            rounded_once(got[n][b], want[n][b], (name, b, n))


def test_gradients_against_differences():
    case = CASES["a new part of a sequence"]
    q, k, v, do, _ = make(case, torch.float32)
    got = grads(q, k, v, do, case, None)
    def loss(x):
        with torch.no_grad():
            return float((T.window_attention(*x, case[6], case[7], sinks=case[8]).double() * do).sum())
    # the loss is a sum of 3840 terms below 10 with errors below 1e-5 of them in all, over 2 e; the third derivative's part is below e^2 * 100
    e = 2.0 ** -7
    for i, n in enumerate("qkv"):
        x = [q.detach(), k.detach(), v.detach()]
        d = torch.randn_like(x[i])
        d /= d.norm()
        up, down = (loss([t + s * e * d if j == i else t for j, t in enumerate(x)]) for s in (1, -1))
        assert abs((up - down) / (2 * e) - float((got[n].double() * d).sum())) <= 3840 * 10 * 1e-7 / (2 * e) + 100 * e * e, n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_lies_behind_a_sequence_is_not_read(dtype):
    case = CASES["both sides, padded"]
    q, k, v, do, lengths = make(case, dtype)
    want = grads(q, k, v, do, case, lengths)
    with torch.no_grad():
        for b, n in enumerate(case[9]):
            k[b, n:], v[b, n:] = math.nan, math.inf
    got = grads(q, k, v, do, case, lengths)
    assert all(torch.equal(got[n], want[n]) for n in got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_scale(dtype):
    """One packed projection's columns, heads in front of rows, and an address that is no multiple of 16: the same bits."""
    B, N, H, D = 2, 150, 4, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn(B * N, 3 * H * D, device="cuda", generator=g).to(dtype).requires_grad_()
    q, k, v = (x.unflatten(1, (H, D)).unflatten(0, (B, N)) for x in rows.split(H * D, 1))
    do = torch.randn(B, N, H, D, device="cuda", generator=g).to(dtype)
    case = (B, N, N, H, H, D, 20, 4, 2, None)
    o = T.window_attention(q, k, v, 20, 4, sinks=2, scale=0.3)
    packed = torch.autograd.grad(o, rows, do)[0]
    c = [x.detach().contiguous().requires_grad_() for x in (q, k, v)]
    want = grads(*c, do, case, None, scale=0.3)
    assert torch.equal(o, want["o"]) and torch.equal(packed, torch.cat([want[n].reshape(B * N, H * D) for n in "qkv"], 1))
    t = [x.detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for x in c]
    u = [torch.zeros(x.numel() + 1, device="cuda", dtype=dtype)[1:].view(x.shape).copy_(x.detach()).requires_grad_() for x in c]
    for x in (t, u):
        got = grads(*x, do, case, None, scale=0.3)
        assert all(torch.equal(got[n], want[n]) for n in got)
    check(want, *oracle(*c, do, 20, 4, 2, None, scale=0.3)[:2])
    d = torch.randn(B, H, N, D, device="cuda", generator=g).to(dtype).transpose(1, 2)      # a gradient with other strides
    got, same = (torch.autograd.grad(T.window_attention(*c, 20, 4, sinks=2), c, x) for x in (d, d.contiguous()))
    assert all(torch.equal(a, b) for a, b in zip(got, same))


def test_more_shares_of_first_keys_than_a_grid_has_threads():
    """2^28 values of first keys' gradients to add up: the same bits as of a few sequences alone."""
    case = (1024, 131, 131, 8, 8, 128, 0, 0, 128, None)
    q, k, v, do, _ = make(case, torch.bfloat16)
    got = grads(q, k, v, do, case, None)
    for b in (0, 511, 1022):
        few = [x.detach()[b:b + 2].clone().requires_grad_() for x in (q, k, v)]
        want = grads(*few, do[b:b + 2], case, None)
        assert all(torch.equal(got[n][b:b + 2], want[n]) for n in want), b


def test_no_gradient_wanted_and_scores_of_any_size():
    q, k, v, do, _ = make(CASES["two row tiles"], torch.float32)
    o = T.window_attention(q, k, v, 40)
    with torch.no_grad():
        assert torch.equal(T.window_attention(q, k, v, 40), o)
        # scores in the thousands: a softmax that has one key for each row, up to exp(-difference)
        huge = T.window_attention(q * 1e3, k, v, 40)
        want, _, _ = oracle(q * 1e3, k, v, do, 40, 0, 0, None)
        size = float((q.detach().double() * 1e3).norm(dim=-1).max() * k.detach().double().norm(dim=-1).max() / 128 ** 0.5)
        assert float((huge.double() - want["o"]).abs().max()) <= 2 * (2 * 132 * U * size) * float(v.abs().max()) + 1e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_forward_and_backward(dtype):
    case = CASES["many chunks of far rows, two blocks of sinks"]
    q, k, v, do, _ = (None if x is None else x.detach() for x in make(case, dtype))
    lengths = torch.tensor([1400], dtype=torch.int32, device="cuda")
    leaves = lambda: [x.detach().requires_grad_() for x in (q, k, v)]  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(*leaves(), do, case, lengths)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = grads(*leaves(), do, case, lengths)
    for n in (1500, 900, 1):
        lengths.fill_(n)
        q.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        want = grads(*leaves(), do, case, lengths)
        torch.cuda.synchronize()
        assert all(torch.equal(got[x], want[x]) for x in got), n


def test_two_streams():
    case = CASES["far rows"]
    q, k, v, do, _ = make(case, torch.bfloat16)
    want = grads(q, k, v, do, case, None)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            got.append(grads(*(x.detach().requires_grad_() for x in (q, k, v)), do, case, None))
    torch.cuda.synchronize()
    assert all(torch.equal(g[n], want[n]) for g in got for n in want)


# ------------------------------------------------------------------------------------------------------------- one token
# batch, room, heads, key heads, channels, left, sinks, lengths
STEPS = {
    "one token": (1, 1, 1, 1, 8, 0, 0, [1]),
    "short": (2, 40, 4, 2, 64, 10, 2, [40, 7]),
    "nothing in the cache": (3, 50, 2, 2, 32, 8, 1, [0, 50, 1]),
    "no limit": (2, 1000, 8, 8, 64, None, 0, [1000, 333]),
    "long, few sequences": (1, 9000, 2, 1, 128, 5000, 4, [8999]),
    "group of 3": (2, 300, 6, 2, 80, 100, 16, [300, 299]),
    "group of 16": (2, 513, 16, 1, 96, 512, 0, [513, 400]),
    "sinks only beside itself": (1, 700, 4, 4, 40, 0, 128, [600]),
    "lengths beyond the room": (2, 64, 2, 2, 64, 31, 3, [70, -5]),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", sorted(STEPS))
def test_step(name, dtype):
    B, N, H, Hk, D, left, sinks, lens = STEPS[name]
    g = torch.Generator(device="cuda").manual_seed(2)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    q, k, v = n(B, H, D) * 1.5, n(B, N, Hk, D), n(B, N, Hk, D)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for b, size in enumerate(lens):              # what a token does not see may hold anything
        size = min(max(size, 0), N)
        k[b, size:], v[b, size:] = math.nan, math.nan
        if left is not None:
            k[b, sinks:max(size - 1 - left, sinks)], v[b, sinks:max(size - 1 - left, sinks)] = math.inf, math.nan
    o = T.window_attention_step(q, k, v, lengths, left, sinks=sinks)
    assert bool(torch.isfinite(o).all())
    for b, size in enumerate(lens):
        size = min(max(size, 0), N)
        if size == 0:
            assert bool((o[b] == 0).all())
            continue
        kk, vv = (torch.nan_to_num(x[b:b + 1, :size], 0.0, 0.0, 0.0) for x in (k, v))
        want, tol, _ = oracle(q[b:b + 1, None], kk, vv, q[b:b + 1, None], left, 0, sinks, None)
        err = (o[b].double() - want["o"][0, 0]).abs()
        assert bool((err <= tol["o"][0, 0]).all()), (b, float((err / tol["o"][0, 0]).max()))
    assert torch.equal(T.window_attention_step(q, k, v, lengths, left, sinks=sinks), o)


# two to eight slices, more heads of a group than a tile has columns, and caches that are read past the caches
MORE_STEPS = {
    "few slices": (40, 300, 16, 4, 64, None, 0, [300 - 7 * b for b in range(40)]),
    "group of 40": (2, 200, 80, 2, 40, 150, 2, [200, 33]),
    "a large cache": (8, 4096, 16, 8, 128, None, 0, [4096, 1, 4095, 31, 2048, 0, 33, 4000]),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", sorted(MORE_STEPS))
def test_step_cuts(name, dtype):
    B, N, H, Hk, D, left, sinks, lens = MORE_STEPS[name]
    g = torch.Generator(device="cuda").manual_seed(5)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    q, k, v = n(B, H, D), n(B, N, Hk, D), n(B, N, Hk, D)
    for b, size in enumerate(lens):
        k[b, size:], v[b, size:] = math.nan, math.inf
    o = T.window_attention_step(q, k, v, torch.tensor(lens, dtype=torch.int32, device="cuda"), left, sinks=sinks)
    for b, size in enumerate(lens):
        if size == 0:
            assert bool((o[b] == 0).all())
            continue
        want, tol, _ = oracle(q[b:b + 1, None], k[b:b + 1, :size], v[b:b + 1, :size], q[b:b + 1, None], left, 0, sinks, None)
        err = (o[b].double() - want["o"][0, 0]).abs()
        assert bool((err <= tol["o"][0, 0]).all()), (b, float((err / tol["o"][0, 0]).max()))


@pytest.mark.parametrize("name", ["few slices", "many slices", "one workgroup", "wide heads"])
def test_step_results_are_rounded_once(name):
    """bf16: the probabilities of the single-token form are held in 16 bits or more, in one slice and in many.  Scores of a few units, so that many
    keys share a row's weight (a weight next to 1 is held exactly by any type)."""
    B, N, H, Hk, D, left, sinks, lens = {"few slices": MORE_STEPS["few slices"], "many slices": (2, 6000, 16, 2, 64, None, 0, [6000, 3333]),
                                         "one workgroup": (3, 900, 4, 4, 64, 700, 4, [900, 20, 801]),
                                         "wide heads": (4, 3000, 32, 4, 128, 2000, 4, [3000, 1, 2100, 300])}[name]
    g = torch.Generator(device="cuda").manual_seed(6)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    q, k, v = n(B, H, D), n(B, N, Hk, D), n(B, N, Hk, D)
    o = T.window_attention_step(q, k, v, torch.tensor(lens, dtype=torch.int32, device="cuda"), left, sinks=sinks)
    for b, size in enumerate(lens):
        want = oracle(q[b:b + 1, None], k[b:b + 1, :size], v[b:b + 1, :size], q[b:b + 1, None], left, 0, sinks, None)[0]
        rounded_once(o[b], want["o"][0, 0], (name, b))


def test_step_strides_and_growing_cache_in_a_graph():
    """A cache with heads in front of rows, the step captured once and replayed while the sequences grow."""
    B, N, H, Hk, D = 3, 2100, 8, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = torch.randn(2, B, Hk, N, D, device="cuda", generator=g).to(torch.bfloat16)
    k, v = (c.transpose(1, 2) for c in cache)
    q = torch.randn(B, 2 * H, D, device="cuda", generator=g).to(torch.bfloat16)[:, ::2]
    lengths = torch.tensor([1, 1000, 2095], dtype=torch.int32, device="cuda")
    T.window_attention_step(q, k, v, lengths, 300, sinks=4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lengths.add_(1)
        o = T.window_attention_step(q, k, v, lengths, 300, sinks=4)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, T.window_attention_step(q.contiguous(), k.contiguous(), v.contiguous(), lengths, 300, sinks=4)), i
        assert lengths.tolist() == [2 + i, 1001 + i, 2096 + i]


def test_offsets_that_pass_32_bits():
    """A cache of more than 2^32 values: the last sequence's keys lie behind them."""
    B, N, Hk, D = 3, 1 << 21, 8, 128
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 26 GB")
    k = torch.empty(B, N, Hk, D, device="cuda", dtype=torch.bfloat16)
    v = torch.empty_like(k)
    g = torch.Generator(device="cuda").manual_seed(4)
    lens = [N, 5, N - 3]
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    parts = []
    for b, n in enumerate(lens):
        lo = max(n - 101, 0)
        for c in (k, v):
            c[b, :2] = torch.randn(2, Hk, D, device="cuda", generator=g)
            c[b, lo:n] = torch.randn(n - lo, Hk, D, device="cuda", generator=g)
        parts.append((lo, n))
    q = torch.randn(B, 16, D, device="cuda", generator=g).to(torch.bfloat16)
    o = T.window_attention_step(q, k, v, lengths, 100, sinks=2)
    for b, (lo, n) in enumerate(parts):
        pick = lambda c: torch.cat([c[b:b + 1, :min(2, lo)], c[b:b + 1, lo:n]], 1)  # noqa: E731
        want, tol, _ = oracle(q[b:b + 1, None], pick(k), pick(v), q[b:b + 1, None], None, 0, 0, None)
        assert bool(((o[b].double() - want["o"][0, 0]).abs() <= tol["o"][0, 0]).all()), b


def test_refusals():
    n = lambda *s, dtype=torch.float32: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    q, k = n(2, 8, 4, 64), n(2, 10, 2, 64)
    T.window_attention(q, k, k, 3)
    bad = lambda *a, **kw: pytest.raises(RuntimeError, match="window_attention")  # noqa: E731
    for args, kw in (((q[0], k, k), {}), ((q, k, k[:, :9]), {}), ((q, k[:1], k[:1]), {}), ((q, k[..., :56], k[..., :56]), {}), ((q, k.bfloat16(), k.bfloat16()), {}),
                     ((q.half(), k.half(), k.half()), {}), ((q, k.cpu(), k.cpu()), {}), ((q[:, :, :3], k, k), {}), ((q[..., :60], k[..., :60], k[..., :60]), {}),
                     ((n(1, 2, 1, 136), n(1, 2, 1, 136), n(1, 2, 1, 136)), {}), ((q, k[:, :7], k[:, :7]), {}), ((q[:, :0], k, k), {}), ((q, k, k), dict(left=-2)),
                     ((q, k, k), dict(sinks=129)), ((q, k, k), dict(sinks=-1)), ((q, k, k), dict(scale=0.0)), ((q, k, k), dict(scale=float("nan"))),
                     ((q, k, k), dict(lengths=torch.ones(2, device="cuda"))), ((q, k, k), dict(lengths=torch.ones(3, device="cuda", dtype=torch.int32)))):
        with bad():
            T.window_attention(*args, **kw)
    lens = torch.ones(2, device="cuda", dtype=torch.int32)
    T.window_attention_step(q[:, 0], k, k, lens)
    for args, kw in (((q, k, k, lens), {}), ((q[:, 0], k, k, None), {}), ((q[:, 0], k, k, lens.cpu()), {}), ((q[:, 0], k, k, lens.long()), {}),
                     ((q[:, 0, :, ::2], k[..., ::2], k[..., ::2], lens), {}), ((q[:1, 0], k, k, lens), {}), ((q[:, 0], k, k, lens), dict(sinks=200))):
        with bad():
            T.window_attention_step(*args, **kw)

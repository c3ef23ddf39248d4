"""AdamW over a list of tensors (pt_train_adamw_multi), the global gradient norm (pt_train_grad_norm) and the 8-bit moments
against plain implementations: 64 bits for the 32-bit form, numpy's IEEE fp32 one operation at a time for the codes, which
have to be equal."""
import math

import numpy as np
import pytest
import torch

from probtalk_amd import train_ops as T

pytestmark = pytest.mark.gpu

E = 2.0 ** -24                                       # half a step of fp32
LISTS = {"one": [1], "edges": [255, 256, 257, 0, 3], "units": [4096, 4097, 12_345, 1], "many": [7 + 37 * i for i in range(200)],
         "large": [3_000_001, 5]}
H = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=1e-2)


def tensors(sizes, seed, scale=1.0, dtype=torch.float32, odd=False):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        t = torch.randn(n + 1, generator=g).mul(scale).to(dtype)
        t = t.cuda()[1:] if odd else t[1:].cuda()     # odd: one value behind an aligned address
        out.append(t)
    return out


def f64(ts):
    return [t.detach().cpu().double().numpy() for t in ts]


@pytest.mark.parametrize("name", sorted(LISTS))
@pytest.mark.parametrize("odd", [False, True])
def test_norm_of_a_list(name, odd):
    gs = tensors(LISTS[name], 1, 0.3, odd=odd)
    gs[0] = gs[0].to(torch.bfloat16)                  # mixed types in one list
    want = math.sqrt(sum(float((g * g).sum()) for g in f64(gs)))
    norm, coef = T.grad_norm(gs, 0.7 * want)
    assert abs(float(norm) - want) <= 1.01 * E * want                       # the sum is exact to fp64, rounded once
    assert abs(float(coef) - 0.7 * want / (want + 1e-6)) <= 6 * E           # norm, its sum with 1e-6, max_norm and the quotient: a rounding each
    assert float(T.grad_norm(gs, 1e9)[1]) == 1.0
    again = T.grad_norm(gs, 0.7 * want)
    assert torch.equal(again[0], norm) and torch.equal(again[1], coef)


def test_norm_of_nothing_and_of_non_finite():
    norm, coef = T.grad_norm([], 1.0)
    assert float(norm) == 0.0 and float(coef) == 1.0
    norm, coef = T.grad_norm([torch.zeros(0, device="cuda"), torch.zeros(5, device="cuda")], 1.0)
    assert float(norm) == 0.0 and float(coef) == 1.0
    g = torch.ones(1000, device="cuda")
    g[3] = math.inf
    norm, coef = T.grad_norm([g], 1.0)
    assert math.isinf(float(norm)) and float(coef) == 0.0
    g[3] = math.nan
    assert math.isnan(float(T.grad_norm([g], 1.0)[0]))


def pair_of_calls(gs, max_norm):
    """Norm and coefficient by the entries for one tensor."""
    from probtalk_amd import _lib
    L, p, s = _lib.lib(), _lib.ptr, _lib.stream()
    total, coef, norm = (torch.zeros(1, device="cuda") for _ in range(3))
    for g in gs:
        _lib.check(L.pt_train_sumsq(p(g), g.numel(), p(total), s))
    _lib.check(L.pt_train_clip_coef(p(total), max_norm, p(coef), p(norm), s))
    return norm, coef


@pytest.mark.parametrize("name", ["units", "many", "one"])
def test_norm_of_a_list_is_that_of_the_entries_for_one_tensor(name):
    gs = tensors(LISTS[name], 21, 0.3)
    want, got = pair_of_calls(gs, 0.7), T.grad_norm(gs, 0.7)
    # fp32 sums of squares: a thread passes n / 262,144 + 1 values, then 6 lanes, 4 waves and as many workgroups as there are, once per tensor; the
    # root halves what they lose, the quotient keeps it
    n = sum(1 + 6 + 4 + min(-(-s // 1024), 1024) + s // 262_144 for s in LISTS[name])
    for a, b in zip(want, got):
        assert abs(float(a) - float(b)) <= (n / 2 + 8) * E * float(b)


@pytest.mark.parametrize("size", [1000, 300_000])                          # one launch, and a launch of partial sums
def test_a_norm_that_is_no_number_is_not_taken_for_one(size):
    """As torch.nn.utils.clip_grad_norm_ has it: the factor is NaN, and no tensor takes an unclipped step."""
    gs = [torch.ones(size, device="cuda"), torch.ones(7, device="cuda")]
    gs[0][3] = math.nan
    for norm, coef in (T.grad_norm(gs, 1.0), pair_of_calls(gs, 1.0)):
        assert math.isnan(float(norm)) and math.isnan(float(coef))
    ps = [torch.nn.Parameter(torch.ones_like(g)) for g in gs]
    qs = [torch.nn.Parameter(torch.ones_like(g)) for g in gs]
    for p, q, g in zip(ps, qs, gs):
        p.grad, q.grad = g.clone(), g.clone()
    torch.nn.utils.clip_grad_norm_(ps, 1.0)
    torch.optim.AdamW(ps).step()
    norm, coef = T.clip_grad_norm(qs, 1.0)
    T.AdamW([{"params": qs}]).step({q: coef for q in qs})
    assert all(torch.equal(torch.isnan(p), torch.isnan(q)) and bool(torch.isnan(q).all()) for p, q in zip(ps, qs))


def reference(p, g, m, v, coef, step, lr, betas, eps, weight_decay):
    """64 bits, with the constants that the kernel is given (fp32)."""
    b1, b2, lr, eps, wd = (float(np.float32(x)) for x in (*betas, lr, eps, weight_decay))
    g = g * coef
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    upd = lr / (1 - b1 ** step) * m / (np.sqrt(v) / math.sqrt(1 - b2 ** step) + eps)
    # roundings: 1 - b^t loses what pow rounds, relative to the small difference; 14 more in m, v, the root, the quotients
    off = 14 * E + E / (1 - b1 ** step) + 0.5 * E / (1 - b2 ** step)
    return p * (1 - lr * wd) - upd, m, v, np.abs(upd) * off + 3 * E * np.abs(p)


@pytest.mark.parametrize("name", sorted(LISTS))
@pytest.mark.parametrize("odd", [False, True])
def test_step_with_32_bit_moments(name, odd):
    sizes = LISTS[name]
    p, g = tensors(sizes, 2, odd=odd), tensors(sizes, 3, 0.1, odd=odd)
    m, v = tensors(sizes, 4, 0.05, odd=odd), [t.square_() for t in tensors(sizes, 5, 0.05, odd=odd)]
    coef = torch.tensor([0.37], device="cuda")
    before = [f64(x) for x in (p, g, m, v)]
    lst = T.AdamWList(p, m, v)
    assert lst.step(g, 3, coef=coef, **H) is None
    for i in range(len(sizes)):
        P, G, M, V = (b[i] for b in before)
        wp, wm, wv, tol = reference(P, G, M, V, float(coef), 3, **H)
        assert (np.abs(f64([p[i]])[0] - wp) <= tol).all()
        assert (np.abs(f64([m[i]])[0] - wm) <= 4 * E * (np.abs(0.9 * M) + np.abs(0.1 * G))).all()
        assert (np.abs(f64([v[i]])[0] - wv) <= 6 * E * wv).all()
        assert np.array_equal(f64([g[i]])[0], G)


def test_step_equals_the_one_tensor_kernel():
    """The same update as pt_train_adamw, and the same clipping as the two calls."""
    from probtalk_amd import _lib
    sizes = LISTS["units"]
    p, g, m = (tensors(sizes, s, 0.1) for s in (6, 7, 8))
    v = [t.square_() for t in tensors(sizes, 9, 0.1)]
    q, m1, v1 = ([t.clone() for t in x] for x in (p, m, v))
    norm, coef = T.grad_norm(g, 0.5)
    for i in range(len(sizes)):
        _lib.check(_lib.lib().pt_train_adamw(_lib.ptr(q[i]), _lib.ptr(g[i]), _lib.ptr(m1[i]), _lib.ptr(v1[i]), sizes[i], _lib.ptr(coef), 1e-3, 0.9, 0.99,
                                             1e-8, 1e-2, 7, _lib.stream()))
    n2 = T.AdamWList(p, m, v).step(g, 7, max_norm=0.5, **H)
    assert torch.equal(n2, norm)
    for a, b in ((p, q), (m, m1), (v, v1)):
        for x, y in zip(a, b):
            assert torch.equal(x, y)                                        # the list's kernel writes out the same contraction


# --------------------------------------------------------------------------------------------------------- 8-bit moments
U32, F = np.uint32, np.float32


def hashed(pos, seed, step):
    with np.errstate(over="ignore"):
        x = (U32(step) * U32(0x9E3779B9)) ^ U32(seed)
        x = (x ^ (x >> U32(16))) * U32(0x6A09E667)
        key = x ^ (x >> U32(15))
        x = (pos.astype(U32) ^ key) * U32(0x9E3779B9)
        x ^= x >> U32(15)
        x *= U32(0x6A09E667)
        return x ^ (x >> U32(14))


def values(c, mant, scale):
    c = c.astype(np.int64)
    n = np.where(c < 2 ** mant, c, (2 ** mant + c % 2 ** mant) * 2.0 ** (c // 2 ** mant - 1)).astype(F)
    return n * np.repeat(scale, 256)[:len(n)]


def codes(x, mant, top, r):
    n = len(x)
    a = np.zeros(-(-n // 256) * 256, F)
    a[:n] = np.abs(x)
    big = a.reshape(-1, 256).max(1)
    scale = np.where(big < F(2.0 ** -100), F(0), big / F(top)).astype(F)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(scale > 0, F(1) / scale, F(0)).astype(F)
    z = np.minimum(a * np.repeat(inv, 256), F(top))[:n]
    low = np.floor(z + r.astype(F) * F(2.0 ** -16)).astype(np.int64)
    high = ((z.view(U32).astype(np.int64) + (r.astype(np.int64) << (7 - mant))) >> (23 - mant)) - ((126 + mant) << mant)
    return np.where(z < 2 ** mant, low, high), z, scale


def step8(P, G, m8, v8, s, coef, step, seed, block0):
    """numpy fp32, one operation at a time -> (p in 64 bits from the fp32 moments, codes, scales)."""
    b1, b2 = F(0.9), F(0.99)
    gr = G.astype(F) * F(coef)
    m = values(m8 & 127, 3, s[:, 0])
    m = np.where(m8 >= 128, -m, m)
    v = values(v8, 4, s[:, 1])
    m = b1 * m + (F(1) - b1) * gr
    v = b2 * v + ((F(1) - b2) * gr) * gr
    r = hashed(np.arange(len(P)) + block0 * 256, seed, step)
    cm, _, sm = codes(m, 3, 245760, r & U32(0xFFFF))
    cv, z, sv = codes(v, 4, 507904, r >> U32(16))
    cv = np.where(z > 0, np.maximum(cv, 1), cv)
    m64, v64 = m.astype(np.float64), v.astype(np.float64)
    lr, wd = float(F(1e-3)), float(F(1e-2))
    upd = lr / (1 - float(b1) ** step) * m64 / (np.sqrt(v64) / math.sqrt(1 - float(b2) ** step) + float(F(1e-8)))
    tol = np.abs(upd) * (10 * E + E / (1 - float(b1) ** step) + 0.5 * E / (1 - float(b2) ** step)) + 3 * E * np.abs(P)
    return P.astype(np.float64) * (1 - lr * wd) - upd, tol, cm | ((m < 0) << 7), cv, np.stack([sm, sv], 1)


def state8(sizes, seed, odd=False):
    """Codes over the whole range, among them the smallest, and scales of every size."""
    r = np.random.RandomState(seed)
    m, v, s = [], [], []
    for n in sizes:
        off = 1 if odd else 0
        m.append(torch.from_numpy(r.randint(0, 256, n + off).astype(np.uint8)).cuda()[off:])
        v.append(torch.from_numpy(r.randint(0, 256, n + off).astype(np.uint8)).cuda()[off:])
        s.append(torch.from_numpy((10.0 ** r.uniform(-12, -5, (-(-n // 256), 2))).astype(np.float32)).cuda())
    return m, v, s


@pytest.mark.parametrize("name", sorted(LISTS))
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_with_8_bit_moments(name, odd, dtype):
    sizes = LISTS[name]
    p, g = tensors(sizes, 2, 1.0, dtype, odd), tensors(sizes, 3, 1e-3, dtype, odd)
    for t in g:
        t[::7] = 0
    m, v, s = state8(sizes, 4, odd)
    s[0].zero_()                                       # a tensor whose moments are zero: the first step
    before = [[t.float().cpu().numpy() if t.dtype != torch.uint8 else t.cpu().numpy() for t in x] for x in (p, g, m, v, s)]
    coef = torch.tensor([0.37], device="cuda")
    T.AdamWList(p, m, v, s).step(g, 5, coef=coef, seed=11, **H)
    block = 0
    for i, n in enumerate(sizes):
        P, G, m8, v8, sc = (b[i] for b in before)
        wp, tol, cm, cv, ws = step8(P, G, m8, v8, sc, np.float32(0.37), 5, 11, block)
        block += -(-n // 256)
        assert np.array_equal(m[i].cpu().numpy(), cm) and np.array_equal(v[i].cpu().numpy(), cv), (i, n)
        assert np.array_equal(s[i].cpu().numpy(), ws)
        if dtype == torch.bfloat16:
            tol = tol + 2.0 ** -7 * np.abs(wp)         # a stochastic rounding is off by less than one bf16 step
        assert (np.abs(p[i].float().cpu().numpy() - wp) <= tol).all()
        got = T.moment_values(m[i], v[i], s[i])
        mm = values(cm & 127, 3, ws[:, 0])
        assert np.array_equal(got[0].cpu().numpy(), np.where(cm >= 128, -mm, mm)) and np.array_equal(got[1].cpu().numpy(), values(cv, 4, ws[:, 1]))


@pytest.mark.parametrize("name", sorted(LISTS))
@pytest.mark.parametrize("odd", [False, True])
def test_step_of_bf16_parameters_with_32_bit_moments(name, odd):
    """numpy's fp32, one operation at a time: the same bits of moments and of parameters, whose rounding takes 16 bits of the value's hash."""
    sizes = LISTS[name]
    bf = torch.bfloat16
    p, g = tensors(sizes, 2, 1.0, bf, odd), tensors(sizes, 3, 0.1, bf, odd)
    m, v = tensors(sizes, 4, 0.05, odd=odd), [t.square_() for t in tensors(sizes, 5, 0.05, odd=odd)]
    before = [[t.float().cpu().numpy() for t in x] for x in (p, g, m, v)]
    T.AdamWList(p, m, v).step(g, 3, coef=torch.tensor([0.37], device="cuda"), seed=11, **H)
    b1, b2, lr, eps, wd = F(0.9), F(0.99), F(1e-3), F(1e-8), F(1e-2)
    bc1, bc2 = F(1) - F(float(b1) ** 3), F(1) - F(float(b2) ** 3)
    decay, size, root = F(1 - float(lr) * float(wd)), lr / bc1, np.sqrt(bc2)
    block = 0
    for i, n in enumerate(sizes):
        P, G, M, V = (b[i] for b in before)
        gr = G * F(0.37)
        M = b1 * M + (F(1) - b1) * gr
        V = b2 * V + ((F(1) - b2) * gr) * gr
        want = P * decay - size * (M / (np.sqrt(V) / root + eps))
        assert np.array_equal(m[i].cpu().numpy(), M) and np.array_equal(v[i].cpu().numpy(), V), (i, n)
        with np.errstate(over="ignore"):
            r = (hashed(np.arange(n) + block * 256, 11, 3) * U32(0xBB67AE85)) >> U32(16)
        block += -(-n // 256)
        codes16 = (want.view(U32) + r) >> U32(16)
        assert np.array_equal(p[i].view(torch.int16).cpu().numpy().view(np.uint16), codes16.astype(np.uint16)), (i, n)


def test_stochastic_roundings_have_no_bias():
    """Zero gradients and no decay: m and v only shrink, by less than a code step.  Over many values the mean of what is stored is
    the mean of what was to be stored: a rounding has a standard deviation of at most half a step, 1/16 and 1/32 of the value.
    bf16 parameters with a step far below a bf16 step move by it in the mean."""
    n = 1 << 20
    m = torch.randint(64, 128, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).to(torch.uint8)
    v = m + 100
    s = torch.full((n // 256, 2), 1e-6, device="cuda")
    m0, v0 = (x.double() for x in T.moment_values(m, v, s))
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    T.AdamWList([p], [m], [v], [s]).step([g], 1, lr=0.0, weight_decay=0.0, betas=(0.99, 0.999))
    m1, v1 = (x.double() for x in T.moment_values(m, v, s))
    sd_m, sd_v = (m0.square().mean().sqrt() / 16 / math.sqrt(n)), (v0.square().mean().sqrt() / 32 / math.sqrt(n))
    assert abs(float(m1.mean() - 0.99 * m0.mean())) < 5 * float(sd_m)
    assert abs(float(v1.mean() - 0.999 * v0.mean())) < 5 * float(sd_v)
    assert not torch.equal(m1, m0)
    p = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    mom = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    T.AdamWList([p], [mom[0]], [mom[1]]).step([torch.ones(n, device="cuda", dtype=torch.bfloat16)], 1, lr=1e-5, weight_decay=0.0)
    # the first step of AdamW is lr; below 1 a bf16 step is 2^-8, of which 1e-5 / 2^-8 = 0.26 % of the values move
    sd = 2.0 ** -8 * math.sqrt(0.0026 / n)
    assert abs(float(1.0 - p.double().mean()) - 1e-5) < 5 * sd


def test_a_block_that_is_not_finite():
    n = 1024
    for bad in (math.inf, math.nan):
        p, g = torch.ones(n, device="cuda"), torch.full((n,), 1e-3, device="cuda")
        g[300] = bad
        m, v, s = torch.zeros(n, device="cuda", dtype=torch.uint8), torch.zeros(n, device="cuda", dtype=torch.uint8), torch.zeros(4, 2, device="cuda")
        T.AdamWList([p], [m], [v], [s]).step([g], 1, **H)
        mv = T.moment_values(m, v, s)
        for x in mv:
            assert bool(torch.isnan(x[256:512]).all()) and bool(torch.isfinite(x[:256]).all()) and bool(torch.isfinite(x[512:]).all())
        ok = torch.ones(n, dtype=torch.bool, device="cuda")
        ok[300] = False
        assert bool(torch.isfinite(p[ok]).all())      # this step's parameters come from the moments before rounding


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on_the_device(bits):
    sizes = [5000, 17, 256]
    def fresh():
        p = tensors(sizes, 2)
        if bits == 32:
            return p, [[torch.zeros_like(t) for t in p], [torch.zeros_like(t) for t in p]]
        return p, [[torch.zeros_like(t, dtype=torch.uint8) for t in p], [torch.zeros_like(t, dtype=torch.uint8) for t in p],
                   [torch.zeros(-(-t.numel() // 256), 2, device="cuda") for t in p]]
    g = tensors(sizes, 3, 0.1)
    p, st = fresh()
    lst = T.AdamWList(p, *st)
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, st2 = fresh()
    eager = T.AdamWList(q, *st2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="int32"):
            lst.step(g, 1, **H)
        count.add_(1)
        norm = lst.step(g, count, max_norm=0.5, seed=3, **H)
    torch.cuda.synchronize()
    for k in range(1, 5):
        for t in g:
            t.mul_(0.9)
        graph.replay()
        want = eager.step(g, k, max_norm=0.5, seed=3, **H)
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and int(count) == k
        for a, b in zip(st, st2):
            for x, y in zip(a, b):
                assert torch.equal(x, y), k
        for x, y in zip(p, q):                         # pow on the device and on the host may differ in the last bit of 1 - b^t
            assert float((x - y).abs().max()) <= 1e-3 * 40 * E * k + 4 * E * float(y.abs().max())
    del graph


def test_optimizer_class_in_8_bits_resumes_bit_for_bit():
    sizes = [(30, 17), (512,), (1000, 3)]
    def model():
        return [torch.nn.Parameter(t.view(s)) for t, s in zip(tensors([math.prod(s) for s in sizes], 2), sizes)]
    ps = model()
    opt = T.AdamW([{"params": ps[:2]}, {"params": ps[2:]}], lr=1e-2, state_bits=8, seed=5)
    def steps(opt, ps, a, b):
        for k in range(a, b):
            for i, p in enumerate(ps):
                p.grad = None if (k, i) == (1, 1) else tensors([p.numel()], 100 + 10 * k + i)[0].view_as(p)    # one parameter misses a step
            norm, coef = T.clip_grad_norm(ps, 3.0)
            opt.step({ps[0]: coef, ps[2]: coef})
    steps(opt, ps, 0, 3)
    sd = opt.state_dict()
    assert set(sd["state"][0]) == {"step", "exp_avg", "exp_avg_sq", "scale"} and sd["state"][0]["exp_avg"].dtype == torch.uint8
    assert float(sd["state"][1]["step"]) == 2 and float(sd["state"][0]["step"]) == 3
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt2 = T.AdamW([{"params": qs[:2]}, {"params": qs[2:]}], lr=1e-2, state_bits=8, seed=5)
    opt2.load_state_dict(sd)
    opt3 = T.AdamW([{"params": [torch.nn.Parameter(p.detach().clone()) for p in ps]}])
    opt3.load_state_dict(sd)                           # 8 bits into 32: what the codes stand for
    assert torch.equal(opt3.state[opt3.param_groups[0]["params"][2]]["exp_avg_sq"],
                       T.moment_values(*(sd["state"][2][k] for k in ("exp_avg", "exp_avg_sq", "scale")))[1])
    with pytest.raises(RuntimeError, match="32 bits"):
        opt2.load_state_dict(opt3.state_dict())
    steps(opt, ps, 3, 5)
    steps(opt2, qs, 3, 5)
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and torch.equal(opt.state[p]["exp_avg"], opt2.state[q]["exp_avg"])


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_class_loads_moments_in_any_order_of_memory(bits):
    """A checkpoint's tensors keep the strides that they were saved with."""
    def model():
        return torch.nn.Parameter(tensors([30 * 40], 2)[0].view(30, 40))
    p, q = model(), model()
    opt, other = (T.AdamW([{"params": [x]}], state_bits=bits) for x in (p, q))
    p.grad, q.grad = (tensors([1200], 3)[0].view(30, 40) for _ in range(2))
    opt.step()
    with torch.no_grad():
        q.copy_(p)
    sd = opt.state_dict()
    for k in ("exp_avg", "exp_avg_sq"):
        sd["state"][0][k] = sd["state"][0][k].t().contiguous().t()
    other.load_state_dict(sd)
    opt.step()
    other.step()
    assert torch.equal(p, q) and torch.equal(opt.state[p]["exp_avg_sq"], other.state[q]["exp_avg_sq"])


def test_optimizer_class_follows_exchanged_memory():
    p = torch.nn.Parameter(torch.ones(100, device="cuda"))
    opt = T.AdamW([{"params": [p]}], lr=0.1, weight_decay=0.0)
    p.grad = torch.ones(100, device="cuda")
    opt.step()
    old = p.data
    p.data = torch.full((100,), 5.0, device="cuda")
    opt.step()
    assert bool((p < 4.95).all()) and bool((old > 0.89).all())


def one_by_one(ps, grads, states, step, **h):
    """The entry for one tensor, parameter by parameter."""
    from probtalk_amd import _lib
    p = _lib.ptr
    for x, g, (m, v) in zip(ps, grads, states):
        _lib.check(_lib.lib().pt_train_adamw(p(x), p(g), p(m), p(v), x.numel(), None, h["lr"], *h["betas"], h["eps"], h["weight_decay"], step, _lib.stream()))


@pytest.mark.parametrize("shared", ["same", "part", "twice"])
def test_optimizer_class_steps_parameters_that_share_memory_in_turn(shared):
    def model():
        flat = tensors([3000], 2)[0].clone()
        if shared == "twice":
            p = torch.nn.Parameter(flat[:1000])
            return flat, [p, torch.nn.Parameter(flat[1000:]), p]
        return flat, [torch.nn.Parameter(x) for x in ((flat, flat, flat[64:128]) if shared == "same" else (flat[:2000], flat[1024:], flat[:512]))]
    (a, ps), (b, qs) = model(), model()
    opt = T.AdamW([{"params": ps}], lr=H["lr"], betas=H["betas"], eps=H["eps"], weight_decay=H["weight_decay"])
    states = {id(q): [torch.zeros_like(q) for _ in range(2)] for q in qs}
    steps = 0
    for k in range(2):
        for i, p in enumerate(ps):
            p.grad = tensors([p.numel()], 30 + 10 * k + i)[0]
        opt.step()
        gs = [p.grad for p in ps]
        for q, g in zip(qs, gs):
            steps += 1
            count = k + 1 if shared != "twice" or q is qs[1] else (2 * k + 1 if steps % 3 == 1 else 2 * k + 2)
            one_by_one([q.detach()], [g], [states[id(q)]], count, **H)
        assert torch.equal(a, b), k
    for p, q in zip(ps, qs):
        assert torch.equal(opt.state[p]["exp_avg"], states[id(q)][0]) and torch.equal(opt.state[p]["exp_avg_sq"], states[id(q)][1])
    assert opt.state[ps[0]]["step"] == (4 if shared == "twice" else 2) and opt.state[ps[1]]["step"] == 2


def test_list_refuses_tensors_that_share_memory():
    flat = torch.zeros(4000, device="cuda")
    t = lambda: torch.zeros(1000, device="cuda")  # noqa: E731
    for p, m, v in (([flat[:1000], flat[999:1999]], [t(), t()], [t(), t()]), ([flat[:1000]], [flat[500:1500]], [t()]), ([t()], [flat[:1000]], [flat[4:1004]])):
        with pytest.raises(RuntimeError, match="share memory"):
            T.AdamWList(p, m, v)
    T.AdamWList([flat[:1000], flat[3000:]], [flat[1000:2000], t()], [flat[2000:3000], t()])


def test_optimizer_class_makes_the_lists_of_many_groups_once(monkeypatch):
    ps = [torch.nn.Parameter(t) for t in tensors([64 + i for i in range(90)], 2)]
    opt = T.AdamW([{"params": ps[i:i + 2]} for i in range(0, 90, 2)])
    made = []
    monkeypatch.setattr(T, "AdamWList", lambda *a, of=T.AdamWList: made.append(1) or of(*a))
    for k in range(3):
        for p in ps:
            p.grad = torch.ones_like(p)
        opt.step()
        assert len(made) == 45, k


@pytest.mark.parametrize("bits", [32, 8])
def test_copies_of_an_optimizer_are_apart(bits):
    """copy.deepcopy and pickle after steps, as a sweep or a whole-object checkpoint makes them."""
    import copy
    import io
    ps = [torch.nn.Parameter(t) for t in tensors([300, 17], 2)]
    opt = T.AdamW([{"params": ps}], state_bits=bits, seed=4)

    def step(o):
        for i, p in enumerate(o.param_groups[0]["params"]):
            p.grad = tensors([p.numel()], 40 + i)[0]
        o.step()

    step(opt)
    held, file = [p.detach().clone() for p in ps], io.BytesIO()
    torch.save(opt, file)
    file.seek(0)
    others = [copy.deepcopy(opt), torch.load(file, weights_only=False)]
    for o in others:
        step(o)
    assert all(torch.equal(p, h) for p, h in zip(ps, held))
    step(opt)
    for o in others:
        for p, q in zip(ps, o.param_groups[0]["params"]):
            assert torch.equal(p, q) and torch.equal(opt.state[p]["exp_avg"], o.state[q]["exp_avg"])
    lists = T.AdamWList([torch.zeros(300, device="cuda")], [torch.zeros(300, device="cuda")], [torch.zeros(300, device="cuda")])
    twin = copy.deepcopy(lists)
    twin.step([torch.ones(300, device="cuda")], 1)
    assert all(bool((t[0] == 0).all()) for t in lists._lists) and bool((twin._lists[0][0] != 0).all())


def test_optimizer_class_in_a_graph_keeps_its_step_count():
    """fp32 with 32-bit moments: what a captured step did when it launched a kernel for every tensor."""
    sizes = [5000, 17]
    ps, qs = ([torch.nn.Parameter(t) for t in tensors(sizes, 2)] for _ in range(2))
    gs = tensors(sizes, 3, 0.1)
    opt = T.AdamW([{"params": ps}], **H)
    states = [[torch.zeros_like(q) for _ in range(2)] for q in qs]
    for p, g in zip(ps, gs):
        p.grad = g
    opt.step()
    one_by_one([q.detach() for q in qs], gs, states, 1, **H)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        for g in gs:
            g.mul_(0.8)
        graph.replay()
        torch.cuda.synchronize()
        one_by_one([q.detach() for q in qs], gs, states, 2, **H)
        assert all(torch.equal(p, q) and torch.equal(opt.state[p]["exp_avg_sq"], s[1]) for p, q, s in zip(ps, qs, states))
    low = T.AdamW([{"params": qs}], state_bits=8)
    for q, g in zip(qs, gs):
        q.grad = g
    low.step()
    torch.cuda.synchronize()
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        with pytest.raises(RuntimeError, match="random bits"):
            low.step()
        gs[0].mul_(1.0)
    del graph, other


def test_refusals():
    p, m, v = (torch.zeros(300, device="cuda") for _ in range(3))
    u, w, s = torch.zeros(300, device="cuda", dtype=torch.uint8), torch.zeros(300, device="cuda", dtype=torch.uint8), torch.zeros(2, 2, device="cuda")
    for args, word in ((([p], [m], []), "lists"), (([p, p], [m, torch.zeros_like(m)], [v, torch.zeros_like(v)]), "twice"), (([p], [m], [v[:299]]), "values"),
                       (([p], [m], [v.double()]), "float64"), (([p[::2]], [m[:150]], [v[:150]]), "contiguous"), (([p.half()], [m], [v]), "float16"),
                       (([p], [u], [w]), "uint8"), (([p], [u], [w], [s[:1]]), "shape"), (([p], [m], [v], [s]), "float32"), (([p, p.bfloat16()], [m, m.clone()], [v, v.clone()]), "float"),
                       (([p], [m.cpu()], [v]), "GPU")):
        with pytest.raises(RuntimeError, match=word):
            T.AdamWList(*args)
    lst, g = T.AdamWList([p], [m], [v]), torch.zeros(300, device="cuda")
    for args, kw in ((([g, g], 1), {}), (([g[:299]], 1), {}), (([g.bfloat16()], 1), {}), (([g.cpu()], 1), {}), (([g], 0), {}),
                     (([g], torch.ones(1, device="cuda")), {}), (([g], 1), dict(coef=torch.ones(1, device="cuda"), max_norm=1.0)),
                     (([g], 1), dict(coef=torch.ones(2, device="cuda"))), (([g], 1), dict(coef=torch.ones(1)))):
        with pytest.raises(RuntimeError):
            lst.step(*args, **kw)
    with pytest.raises(RuntimeError):
        T.grad_norm([g.half()], 1.0)
    with pytest.raises(RuntimeError):
        T.moment_values(u, w, s[:1])
    with pytest.raises(ValueError):
        T.AdamW([{"params": [p]}], state_bits=16)

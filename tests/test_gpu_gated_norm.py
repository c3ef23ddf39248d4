"""gated_norm (pt_train_gated_norm_fwd / _bwd) against its definition in 64 bits, differentiated by torch."""
import pytest
import torch

from probtalk_amd import train_ops as T

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                     # half a step of fp32
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
NAMES = ("x", "t", "gate", "res_scale", "post_weight", "post_bias", "pre_weight", "pre_bias")
# rows, columns, rows per clip: one value; lanes and waves that are partly empty; each number of waves per row; a clip of one row, clips
# that a worker takes whole and clips that several share
SHAPES = [(1, 1, 1), (5, 3, 5), (44, 512, 44), (7, 513, 1), (24, 1024, 8), (33, 2047, 11), (12, 4100, 3), (9, 8192, 9), (2000, 96, 125),
          (5000, 512, 1250), (4096, 8, 4)]


def make(rows, cols, clip, dtype, without=(), seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s, scale=1.0, shift=0.0: torch.randn(*s, device="cuda", generator=g) * scale + shift  # noqa: E731
    v = {"x": n(rows, cols, scale=1.5).to(dtype), "t": n(rows, cols, scale=0.7, shift=0.3).to(dtype), "gate": n(rows // clip, cols, shift=0.5).to(dtype),
         "res_scale": n(cols, scale=0.2, shift=0.5), "post_weight": n(cols, scale=0.2, shift=1.0), "post_bias": n(cols, scale=0.2),
         "pre_weight": n(cols, scale=0.2, shift=1.0), "pre_bias": n(cols, scale=0.2)}
    v = {k: (None if k in without else x.requires_grad_()) for k, x in v.items()}
    return v, n(rows, cols).to(dtype), n(rows, cols).to(dtype)


def norm(x, w, b, kind, eps):
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    r = 1 / (x.square().mean(1, keepdim=True) + eps).sqrt()
    return (x * r * w if b is None else x * r * w + b), r


def oracle(v, clip, kind, eps, dy, dh):
    """Outputs, gradients, and for each the size of what is summed and multiplied up in it (64 bits)."""
    w = {k: None if x is None else x.detach().double().requires_grad_() for k, x in v.items()}
    rows, cols = w["x"].shape
    one = torch.ones((), device="cuda", dtype=torch.float64)
    a = one if w["res_scale"] is None else w["res_scale"]
    g = one if w["gate"] is None else w["gate"].repeat_interleave(clip, 0)
    y, u, rt = w["x"], None, one
    if w["t"] is not None:
        u, rt = (w["t"], one) if w["post_weight"] is None else norm(w["t"], w["post_weight"], w["post_bias"], kind, eps)
        y = y + a * g * u
    h, ry = (None, one) if w["pre_weight"] is None else norm(y, w["pre_weight"], w["pre_bias"], kind, eps)
    outs = [(o, d.double()) for o, d in ((y if u is not None else None, dy), (h, dh)) if o is not None]
    leaves = [k for k in NAMES if w[k] is not None]
    if u is None:
        outs = outs[-1:]
    grads = dict(zip(leaves, torch.autograd.grad([o for o, _ in outs], [w[k] for k in leaves], [d for _, d in outs])))
    # sizes: the largest term of each row, through both norms
    row = lambda x: x.detach().abs().amax(1, keepdim=True).expand(rows, cols)  # noqa: E731
    w1 = one if w["post_weight"] is None else w["post_weight"].abs().max()
    w2 = one if w["pre_weight"] is None else w["pre_weight"].abs().max()
    big_t = 0 if u is None else row(w["t"]) * rt * w1 + (0 if w["post_bias"] is None else w["post_bias"].abs().max())
    ag = (a * g).abs().amax() if u is not None else 0
    big_y = row(w["x"]) + ag * big_t
    big_h = big_y * ry * w2 + (0 if w["pre_bias"] is None else w["pre_bias"].abs().max())
    yh = big_y * ry + 1
    d_in = (row(dy.double()) if u is not None else 0) + (0 if h is None else ry * row(dh.double()) * w2 * yh * yh)
    th = 1 if u is None or w["post_weight"] is None else row(w["t"]) * rt + 1
    size = {"y": big_y, "h": big_h, "x": d_in}
    if u is not None:
        size["t"] = d_in * ag * w1 * rt * th * th
        gg = g.abs() if g.dim() else g
        size["gate"] = (d_in * a.abs() * big_t).reshape(-1, clip, cols).sum(1)
        size["res_scale"], size["post_weight"], size["post_bias"] = ((d_in * gg * f).sum(0) for f in (big_t, a.abs() * th, a.abs()))
    if h is not None:
        size["pre_weight"], size["pre_bias"] = ((row(dh.double()) * f).expand(rows, cols).sum(0) for f in (yh, 1))
    return {"y": y.detach(), "h": None if h is None else h.detach()}, grads, {k: s.detach() for k, s in size.items()}


def check(got, want, size, dtype, roundings, what):
    """A sum over a row passes at most 8 + 6 + 16 additions; a norm has two of them, a root and a product, the backward pass six
    sums in all: `roundings` half steps of fp32 relative to the largest terms, and the rounding of the result."""
    err = (got.double() - want).abs()
    tol = roundings * U * size.double() + HALF[dtype] * want.abs() * 1.01
    assert bool((err <= tol).all()), (what, float((err - tol).max()), float(err.max()))


def run(v, clip, kind, dy, dh, **kw):
    y, h = T.gated_norm(*(v[k] for k in NAMES), rows_per_clip=clip, kind=kind, eps=1e-5, **kw)
    outs = [(o, d) for o, d in ((y if v["t"] is not None else None, dy), (h, dh)) if o is not None]
    leaves = [k for k in NAMES if v[k] is not None]
    return y, h, dict(zip(leaves, torch.autograd.grad([o for o, _ in outs], [v[k] for k in leaves], [d for _, d in outs])))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradients(shape, kind, dtype):
    rows, cols, clip = shape
    v, dy, dh = make(rows, cols, clip, dtype)
    y, h, grads = run(v, clip, kind, dy, dh)
    out, want, size = oracle(v, clip, kind, 1e-5, dy, dh)
    check(y, out["y"], size["y"], dtype, 100, "y")
    check(h, out["h"], size["h"], dtype, 200, "h")
    for k in NAMES:
        assert grads[k].dtype == v[k].dtype and grads[k].shape == v[k].shape
        # a column's sum passes at most rows / 512 + 32 additions on top
        check(grads[k], want[k], size[k], v[k].dtype, 600 + rows / 512, k)
    again = run(v, clip, kind, dy, dh)
    assert all(torch.equal(again[2][k], grads[k]) for k in NAMES)


# each number of lanes a row, one clip that all workers share, rows that are no multiples of 16 bytes, and 16 values a lane
MORE = [(3000, 33, 3000), (700, 64, 1), (900, 100, 450), (1000, 250, 1000), (2, 7, 1), (400, 3, 100), (50, 4097, 50), (64, 6812, 32), (40, 7354, 20), (300, 8191, 300)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("shape", MORE, ids=str)
def test_row_lengths(shape, bias, dtype):
    rows, cols, clip = shape
    v, dy, dh = make(rows, cols, clip, dtype, () if bias else ("post_bias", "pre_bias"), seed=1)
    kind = "layer" if bias else "rms"
    y, h, grads = run(v, clip, kind, dy, dh)
    out, want, size = oracle(v, clip, kind, 1e-5, dy, dh)
    check(y, out["y"], size["y"], dtype, 100, "y")
    check(h, out["h"], size["h"], dtype, 200, "h")
    for k in grads:
        check(grads[k], want[k], size[k], v[k].dtype, 600 + rows / 512, k)
    again = run(v, clip, kind, dy, dh)
    assert all(torch.equal(again[2][k], grads[k]) for k in grads)
    # rows of a wider tensor, at odd addresses: the same bits, and what lies beside them is not touched
    wide = torch.full((rows + 1, cols + 5), float("nan"), device="cuda", dtype=dtype)
    shifted = wide.flatten()[1:1 + rows * (cols + 5)].view(rows, cols + 5)[:, 2:2 + cols]
    shifted.copy_(v["x"].detach())
    same = run({**v, "x": shifted.requires_grad_()}, clip, kind, dy, dh)
    assert torch.equal(same[0], y) and torch.equal(same[1], h) and all(torch.equal(same[2][k], grads[k]) for k in grads)
    assert int(torch.isnan(wide).sum()) == wide.numel() - rows * cols


PARTS = [("gate",), ("res_scale",), ("gate", "res_scale"), ("post_weight", "post_bias"), ("post_bias", "pre_bias"), ("pre_weight", "pre_bias"),
         ("gate", "res_scale", "post_weight", "post_bias", "pre_weight", "pre_bias"), ("t", "gate", "res_scale", "post_weight", "post_bias"),
         ("t", "gate", "res_scale", "post_weight", "post_bias", "pre_bias")]


@pytest.mark.parametrize("without", PARTS, ids="-".join)
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_parts_that_are_left_out(without, kind):
    rows, cols, clip = 60, 200, 20
    v, dy, dh = make(rows, cols, clip, torch.float32, without)
    y, h, grads = run(v, None if "gate" in without else clip, kind, dy, dh)
    out, want, size = oracle(v, clip, kind, 1e-5, dy, dh)
    if "t" in without:
        assert y is v["x"]
    else:
        check(y, out["y"], size["y"], torch.float32, 100, "y")
    assert (h is None) == ("pre_weight" in without)
    if h is not None:
        check(h, out["h"], size["h"], torch.float32, 200, "h")
    for k in grads:
        check(grads[k], want[k], size[k], torch.float32, 600, k)


def test_gradients_against_differences():
    rows, cols, clip = 6, 40, 3
    v, dy, dh = make(rows, cols, clip, torch.float32)
    _, _, grads = run(v, clip, "layer", dy, dh)
    def loss(w):
        y, h = T.gated_norm(*(w[k] for k in NAMES), rows_per_clip=clip)
        return float((y.double() * dy).sum() + (h.double() * dh).sum())
    # central differences of size e: the sum of 480 fp32 values of size up to 10 is off by 480 * 200 U * 10 at most, over 2 e; the third derivative's
    # part is below e^2 * 100 times the direction's size cubed (unit directions here)
    e = 2.0 ** -6
    for k in NAMES:
        d = torch.randn_like(v[k], dtype=torch.float32)
        d /= d.norm()
        with torch.no_grad():
            up, down = ({n: (x + s * e * d if n == k else x) for n, x in v.items()} for s in (1, -1))
            num = (loss(up) - loss(down)) / (2 * e)
        assert abs(num - float((grads[k].double() * d).sum())) <= 480 * 200 * U * 10 / (2 * e) + 100 * e * e, k


def test_one_output_used_and_no_gradient_wanted():
    v, dy, dh = make(30, 100, 10, torch.float32)
    y, h = T.gated_norm(*(v[k] for k in NAMES), rows_per_clip=10)
    zero = torch.zeros_like(dy)
    for o, d, pair in ((y, dy, (dy, zero)), (h, dh, (zero, dh))):
        got = torch.autograd.grad(o, [v["x"], v["gate"]], d, retain_graph=True)
        y2, h2 = T.gated_norm(*(v[k] for k in NAMES), rows_per_clip=10)
        want = torch.autograd.grad((y2, h2), [v["x"], v["gate"]], pair)
        assert all(torch.allclose(a, b, rtol=8 * U, atol=1e-7) for a, b in zip(got, want))
    with torch.no_grad():
        y3, h3 = T.gated_norm(*(v[k] for k in NAMES), rows_per_clip=10)
    assert torch.equal(y3, y) and torch.equal(h3, h) and not y3.requires_grad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_rows_and_odd_addresses(dtype):
    """Rows that are columns of a wider tensor, an address between two vectors, columns apart: the same bits as contiguous rows."""
    rows, cols, clip = 40, 264, 8
    v, dy, dh = make(rows, cols, clip, dtype)
    want = run(v, clip, "layer", dy, dh)
    def wide(x, off, step=1):
        big = torch.full((rows, (cols + 16) * step), 7.0, device="cuda", dtype=dtype)
        w = big[:, off:off + cols * step:step]
        with torch.no_grad():
            w.copy_(x)
        return w.detach().requires_grad_()
    for off, step in ((8, 1), (3, 1), (0, 2)):
        w = dict(v, x=wide(v["x"], off, step), t=wide(v["t"], off, step))
        got = run(w, clip, "layer", dy, dh)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert all(torch.equal(got[2][k], want[2][k]) for k in NAMES), (off, step)


def test_rows_of_zeros_infinities_and_nan_stay_in_their_rows():
    v, dy, dh = make(12, 64, 4, torch.float32)
    with torch.no_grad():
        v["x"][2], v["t"][2] = 0, 0
        v["x"][5, 3], v["t"][9, 1] = float("inf"), float("nan")
    y, h, grads = run(v, 4, "layer", dy, dh)
    ok = [i for i in range(12) if i not in (5, 9)]
    assert bool(torch.isfinite(h[ok]).all()) and bool(torch.isfinite(grads["x"][ok]).all()) and bool(torch.isfinite(grads["t"][ok]).all())
    assert bool(torch.isnan(h[5]).all()) and bool(torch.isnan(h[9]).all())
    assert bool(torch.isfinite(grads["gate"][0]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(40_002, 8, 20_001), (6002, 512, 3001), (8190, 4096, 4095)], ids=str)
@pytest.mark.parametrize("bad", ["x", "t"])
def test_a_row_that_is_not_finite_reaches_its_own_clip_only(bad, shape, dtype):
    """Long clips that many workers share, with rows over: the workers behind a clip's end look at the next clip's rows."""
    rows, cols, clip = shape
    v, dy, dh = make(rows, cols, clip, dtype)
    want = run(v, clip, "layer", dy, dh)[2]
    with torch.no_grad():
        v[bad][clip, cols // 2] = float("nan")
    got = run(v, clip, "layer", dy, dh)[2]
    assert torch.equal(got["gate"][0], want["gate"][0]) and bool(torch.isnan(got["gate"][1]).all())
    ok = torch.arange(rows, device="cuda") != clip
    assert all(torch.equal(got[k][ok], want[k][ok]) and bool(torch.isfinite(got[k][ok]).all()) for k in ("x", "t"))


def test_without_t_nothing_else_of_the_first_norm_counts():
    """The C entries take res_scale, post_w and post_b without t: y is x then, in the backward pass too."""
    from probtalk_amd import _lib
    L, p, rows, cols = _lib.lib(), _lib.ptr, 30, 72
    v, _, dh = make(rows, cols, 10, torch.float32)
    d = {k: x.detach() for k, x in v.items()}
    got = []
    for first in ((None, None, None), (d["res_scale"], d["post_weight"], d["post_bias"])):
        h, stats, dx = torch.empty_like(d["x"]), torch.empty(rows, 4, device="cuda"), torch.empty_like(d["x"])
        dw, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
        ws = torch.empty(L.pt_train_gated_norm_workspace_bytes(rows, cols, 0), dtype=torch.uint8, device="cuda")
        _lib.check(L.pt_train_gated_norm_fwd(p(d["x"]), cols, None, 0, None, *map(p, first), p(d["pre_weight"]), p(d["pre_bias"]), None, p(h), p(stats), rows, cols,
                                             rows, 0, 1e-5, 0, _lib.stream()))
        _lib.check(L.pt_train_gated_norm_bwd(p(d["x"]), cols, None, 0, None, *map(p, first), p(d["pre_weight"]), p(stats), None, p(dh), p(dx), None, None, None, None,
                                             None, p(dw), p(db), p(ws), ws.numel(), rows, cols, rows, 0, 0, _lib.stream()))
        got.append((h, dx, dw, db))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    y, h = T.gated_norm(v["x"], pre_weight=v["pre_weight"], pre_bias=v["pre_bias"])
    assert y is v["x"] and torch.equal(got[0][0], h)
    assert torch.equal(got[0][1], torch.autograd.grad(h, v["x"], dh)[0])


def test_as_many_rows_as_32_bits_hold():
    """Rows of one value (RMS): 2^31 - 1 of them forward, where a row's number behind the last one passes 32 bits; and one gate for more than
    2^30 rows with gradients.  The same rows in a small call give the same bits."""
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 60 GB")
    g = torch.Generator(device="cuda").manual_seed(7)
    part, dt = 1 << 20, torch.bfloat16
    n = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dt)  # noqa: E731
    w = torch.tensor([0.9], device="cuda")
    gate = n(1, 1) + 1
    small = [n(part, 1) for _ in range(4)]
    f = lambda x, t, q: T.gated_norm(x, t, q, None, w, None, w, kind="rms", rows_per_clip=x.shape[0])  # noqa: E731
    rows = (1 << 31) - 1
    big = [x.repeat(1 << 11, 1)[:rows] for x in small[:2]]
    with torch.no_grad():
        y, h = f(*big, gate)
        want = f(*small[:2], gate)
    for got, e in zip((y, h), want):
        assert torch.equal(got[:part], e) and torch.equal(got[-part + 1:], e[:-1]) and torch.equal(got[rows // 2 // part * part:][:part], e)
    del big, y, h, got
    times = (1 << 10) + 1
    x, t, dy, dh = (v.repeat(times, 1) for v in small)
    leaves = [v.requires_grad_() for v in (x, t, gate.clone())]
    dx, dtt, dg = torch.autograd.grad(f(*leaves), leaves, (dy, dh))
    same = [v.clone().requires_grad_() for v in (*small[:2], gate)]
    ex, et, _ = torch.autograd.grad(f(*same), same, small[2:])
    for got, e in ((dx, ex), (dtt, et)):
        assert torch.equal(got[:part], e) and torch.equal(got[-part:], e)
    s = [v.detach().double().requires_grad_() for v in same]
    norm = lambda v: v / (v.square() + 1e-5).sqrt() * w.double()  # noqa: E731
    u = norm(s[1])
    yy = s[0] + s[2] * u
    d = torch.autograd.grad((yy, norm(yy)), [s[0], s[2]], [v.double() for v in small[2:]])
    # a worker adds up 65,600 rows one after the other, 16,384 workers are added up after that; a bf16 result
    size = float((d[0] * u.detach()).abs().sum()) * times
    assert abs(float(dg) - float(d[1]) * times) <= (65_600 + 16_400) * U * size + 2.0 ** -8 * abs(float(d[1]) * times)


def test_captured_forward_and_backward():
    v, dy, dh = make(300, 520, 100, torch.bfloat16)
    base = {k: x.detach() for k, x in v.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w = {k: x.detach().requires_grad_() for k, x in base.items()}
        run(w, 100, "rms", dy, dh)
        del w
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        w = {k: x.detach().requires_grad_() for k, x in base.items()}     # leaves of the capture
        y, h, grads = run(w, 100, "rms", dy, dh)
    for k in range(3):
        with torch.no_grad():
            base["x"].add_(0.25)
            dy.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        e = {n: x.detach().clone().requires_grad_() for n, x in base.items()}
        want = run(e, 100, "rms", dy, dh)
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(h, want[1]) and all(torch.equal(grads[n], want[2][n]) for n in NAMES), k


def test_two_streams():
    v, dy, dh = make(2000, 512, 100, torch.float32)
    want = run(v, 100, "layer", dy, dh)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run({k: x.detach().requires_grad_() for k, x in v.items()}, 100, "layer", dy, dh))
    torch.cuda.synchronize()
    for r in got:
        assert torch.equal(r[1], want[1]) and all(torch.equal(r[2][k], want[2][k]) for k in NAMES)


def test_refusals():
    v, _, _ = make(12, 64, 4, torch.float32)
    a = [v[k].detach() for k in NAMES]
    f = lambda **kw: T.gated_norm(**dict(zip(NAMES, a)) | kw)  # noqa: E731
    f()
    for kw in (dict(x=a[0].half()), dict(x=a[0][0]), dict(t=a[1][:11]), dict(t=a[1].bfloat16()), dict(gate=a[2][:, :60]), dict(gate=a[2].bfloat16()), dict(rows_per_clip=5),
               dict(rows_per_clip=0), dict(res_scale=a[3].bfloat16()), dict(post_weight=a[4][:60]), dict(post_weight=None), dict(pre_weight=None), dict(t=None),
               dict(pre_bias=a[7].cpu()), dict(x=torch.zeros(2, 8200, device="cuda")), dict(x=a[0][:0], t=a[1][:0], gate=a[2][:0])):
        with pytest.raises(RuntimeError, match="gated_norm"):
            f(**kw)
    with pytest.raises(ValueError):
        f(kind="batch")

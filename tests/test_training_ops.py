"""The training operators (rebel_amd.training, rbl_layer_norm_* / rbl_grad_* of the C ABI) against their definitions in 64 bits.

Tolerances are bounds, element by element, from the roundings of the computation: u = 2^-24 is half a step of f32, a sum of n terms
whose longest chain of additions has D members is off by at most D u sum|terms| (first order; the constants are rounded up), and the
result is rounded once to its type (half a step, eps / 2 relative; half a subnormal step absolute)."""
import ctypes as C
import math

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from rebel_amd import capi, training
from rebel_amd.models import Net2

U = 2.0 ** -24
EPS = 1e-5
gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rounding(v, dtype):
    """Half a step of `dtype` at v: relative for normal numbers, half the subnormal step below them."""
    info = torch.finfo(dtype)
    return v.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def make(rows, cols, dtype, params, seed=0, affine=(True, True), offset=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + rows * 31 + cols)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x = (rnd(rows, cols) * (0.2 + 2 * torch.rand(rows, 1, generator=g, device="cuda")) + offset * rnd(rows, 1)).to(dtype)
    w = (1 + 0.3 * rnd(cols)).to(params) if affine[0] else None
    b = (0.3 * rnd(cols)).to(params) if affine[1] else None
    return x, w, b, rnd(rows, cols).to(dtype)


def oracle(x, w, b, dy=None, gelu=False, eps=EPS):
    """The definition in 64 bits, with a bound for each output's error before its last rounding."""
    x = x.double()
    n = x.shape[-1]
    w = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b.double()
    depth = n / 16 + 16  # terms one lane adds up (16 lanes at least share a row) and the joins behind
    m = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((x - m).square().mean(-1, keepdim=True) + eps)
    h = (x - m) * r
    z = h * w + b
    # mean: rounded once, u |m|; before that it is corrected by the sum of the deviations from the first estimate, whose chain of D
    # additions is off by D u sum|x - m|, so the mean by D u mean|x - m| (the first estimate's own error drops out); variance: D u
    # relative, of which r has half; the subtraction, the product and 1 / sqrt a rounding each
    em = depth * U * (x - m).abs().mean(-1, keepdim=True)
    eh = h.abs() * (depth + 8) * U + (2 * U * (m.abs() + x.abs()) + em) * r
    ez = w.abs() * eh + 3 * U * ((h * w).abs() + b.abs())
    if gelu:
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        pdf = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        y, slope = z * cdf, cdf + z * pdf
        # |slope| <= 1.13, |d slope / dz| <= 0.8; the normal distribution: 5e-7 relative on its tail, exp(-z^2/2) 2 u z^2 more
        ey = 1.13 * ez + z.abs() * (torch.minimum(cdf, 1 - cdf) * (5e-7 + 2 * U * z * z) + 2 * U * cdf)
        es = 0.8 * ez + torch.minimum(cdf, 1 - cdf) * (5e-7 + 2 * U * z * z) + (z * pdf).abs() * (4 * U + 2 * U * z * z) + 2 * U * slope.abs()
    else:
        y, slope, ey, es = z, torch.ones_like(z), ez, torch.zeros_like(z)
    out = {"y": (y, ey), "mean": (m[:, 0], (U * m.abs() + em)[:, 0]), "r": (r[:, 0], r[:, 0] * (depth + 4) * U)}
    if dy is None:
        return out
    dy = dy.double()
    g = dy * slope
    eg = dy.abs() * es + U * g.abs()
    gw = g * w
    egw = w.abs() * eg + U * gw.abs()
    mean = lambda t: t.mean(-1, keepdim=True)
    c1, c2 = mean(gw), mean(gw * h)
    e1 = mean(egw) + (depth + 2) * U * mean(gw.abs())
    e2 = mean(egw * h.abs() + gw.abs() * eh) + (depth + 2) * U * mean((gw * h).abs())
    inner = gw.abs() + c1.abs() + (h * c2).abs()
    out["dx"] = (r * (gw - c1 - h * c2), r * (egw + e1 + h.abs() * e2 + eh * c2.abs() + (depth + 8) * U * inner))
    rows_deep = x.shape[0] / 4 + 32  # at least four partial sums over the rows
    out["dw"] = ((g * h).sum(0), (eg * h.abs() + g.abs() * eh).sum(0) + rows_deep * U * (g * h).abs().sum(0))
    out["db"] = (g.sum(0), eg.sum(0) + rows_deep * U * g.abs().sum(0))
    return out


def near(got, want, what=""):
    v, e = want
    got64 = got.double().reshape(v.shape)
    over = (got64 - v).abs() / (1.01 * e + rounding(v, got.dtype) * 1.01 + 1e-300)
    assert bool((over <= 1).all()), (what, "worst", over.max().item(), "at", int(over.argmax()), got64.reshape(-1)[over.argmax()].item(),
                                     v.reshape(-1)[over.argmax()].item())


def run(x, w, b, dy, act, eps=EPS):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = training.layer_norm(*leaves, eps=eps, activation=act)
    want = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, want, dy))
    return y.detach(), *[next(grads) if t is not None else None for t in leaves]


SIZES = [(1, 1), (3, 1), (5, 2), (1, 7), (2, 8), (33, 9), (7, 16), (65, 63), (4, 64), (9, 65), (130, 127), (1, 128), (17, 129), (1, 256),
         (512, 256), (77, 255), (6, 257), (50, 511), (40, 512), (3, 513), (33, 1000), (20, 1023), (16, 1024), (9, 1025), (5, 2048),
         (7, 2049), (11, 4095), (4, 4096), (3, 4097), (5, 8192), (2, 8199), (3, 16384), (2, 16391), (2, 32768), (1, 32775), (3, 65536),
         (2, 65537), (1, 200003), (4099, 5), (4096, 64), (3001, 200), (2500, 1030)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_layer_norm_against_64_bits(rows, cols, dtype):
    t = TYPES[dtype]
    for act in (None, "gelu"):
        for params in {torch.float32, t}:
            x, w, b, dy = make(rows, cols, t, params)
            want = oracle(x, w, b, dy, act == "gelu")
            y, dx, dw, db = run(x, w, b, dy, act)
            assert torch.equal(training.layer_norm(x, w, b, activation=act), y)  # with and without a gradient to come: the same bits
            assert y.dtype == dx.dtype == t and dw.dtype == db.dtype == params
            for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
                near(got, want[name], (name, act, params))


@gpu
@pytest.mark.parametrize("rows,cols", [(5, 40), (300, 256), (33, 1023), (6, 20000)])
@pytest.mark.parametrize("affine", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_a_parameter(rows, cols, affine):
    x, w, b, dy = make(rows, cols, torch.float32, torch.float32, affine=affine)
    for act in (None, "gelu"):
        want = oracle(x, w, b, dy, act == "gelu")
        y, dx, dw, db = run(x, w, b, dy, act)
        assert (dw is None) == (not affine[0]) and (db is None) == (not affine[1])
        for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
            if got is not None:
                near(got, want[name], name)


@gpu
@pytest.mark.parametrize("rows,cols", [(700, 256), (40, 5000), (3, 40000)])
def test_layer_norm_only_the_gradients_that_are_wanted(rows, cols):
    x, w, b, dy = make(rows, cols, torch.float32, torch.float32)
    full = run(x, w, b, dy, "gelu")
    for wanted in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)):
        leaves = [t.detach().requires_grad_(bool(k)) for t, k in zip((x, w, b), wanted)]
        y = training.layer_norm(*leaves, activation="gelu")
        got = iter(torch.autograd.grad(y, [t for t, k in zip(leaves, wanted) if k], dy))
        want = oracle(x, w, b, dy, True)
        for t, k, name in zip(full[1:], wanted, ("dx", "dw", "db")):
            if k:
                near(next(got), want[name], (wanted, name))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layer_norm_strides(dtype):
    t = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(3)
    big = torch.randn(6, 10, 14, 301, generator=g, device="cuda").to(t)
    w, b = (torch.randn(600, generator=g, device="cuda") for _ in range(2))
    spread = torch.randn(300, 2, generator=g, device="cuda")[:, 1]  # a weight with gaps
    views = [big[..., 1:], big[..., :300], big[:, :, ::2, :257], big[:, 3], big[:, :, 4, 7:], big.transpose(0, 1), big.transpose(1, 2)[..., 5:],
             big.transpose(2, 3), big[:1, :1, :1], big[0, 0, 0], big[2:3, :, :, 3:], big[0, 0, :1].expand(9, 301), big[:, :, :, ::2]]
    for v in views:
        n = v.shape[-1]
        for wv in (w[:n], spread[:n] if n <= 300 else w[:n]):
            ref = oracle(v.reshape(-1, n), wv, b[:n], v.flip(0).reshape(-1, n), True)
            y, dx, dw, db = run(v, wv, b[:n], v.flip(0), "gelu")
            assert y.shape == dx.shape == v.shape and y.is_contiguous()
            for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
                near(got, ref[name], (name, tuple(v.shape), v.stride()))
    # gradients that arrive as views: broadcast from one number, transposed, one row for all
    x = big[0, 0].detach().requires_grad_(True)
    n = x.shape[-1]
    for dy in (torch.ones((), dtype=t, device="cuda").expand(14, n), big[1, :, :, 0][0].new_ones(n, 14).t(), big[1, 1, 1:2].expand(14, n)):
        y = training.layer_norm(x, w[:n], b[:n])
        (dx,) = torch.autograd.grad(y, x, dy)
        near(dx, oracle(x.detach(), w[:n], b[:n], dy)["dx"])


@gpu
def test_layer_norm_of_other_views():
    """Windows that overlap in memory, and views that torch marks as negated without touching the memory."""
    g = torch.Generator(device="cuda").manual_seed(4)
    line = torch.randn(400, generator=g, device="cuda")
    w, b = (torch.randn(300, generator=g, device="cuda") for _ in range(2))
    windows = line.unfold(0, 300, 7)
    dy = torch.randn(windows.shape, generator=g, device="cuda")
    want = oracle(windows, w, b, dy, True)
    for name, got in zip(("y", "dx", "dw", "db"), run(windows, w, b, dy, "gelu")):
        near(got, want[name], name)
    x = torch.randn(15, 300, generator=g, device="cuda")
    want = oracle(-x, -w, -b, -dy, True)
    neg = torch._neg_view
    for name, got in zip(("y", "dx", "dw", "db"), run(neg(x), neg(w), neg(b), neg(dy), "gelu")):
        near(got, want[name], name)
    p = torch.nn.Parameter(torch.empty_like(x))
    p.grad = neg(x.clone())
    training.clip_grad_norm_([p], 1.0)
    v = -x.double() / (float(clip_oracle([x], 2)) + 1e-6)
    near(p.grad, (v, v.abs() * 3 * U))


@gpu
def test_layer_norm_guards_what_it_has_saved():
    x, w, b, dy = make(5, 64, torch.float32, torch.float32)
    for act, touched, fails in ((None, 0, True), ("gelu", 1, True), ("gelu", 2, True), (None, 2, False)):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = training.layer_norm(*leaves, activation=act)
        with torch.no_grad():
            leaves[touched].mul_(2)
        if fails:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(y, leaves, dy)
        else:  # the bias is not needed without an activation
            torch.autograd.grad(y, leaves, dy)
    y = training.layer_norm(*leaves)
    torch.autograd.grad(y, leaves, dy)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaves, dy)
    p = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    p.grad = torch.ones(4, device="cuda")
    before = p.grad._version
    training.clip_grad_norm_([p], 1.0)
    assert p.grad._version == before + 1


@gpu
def test_operators_from_several_threads():
    from concurrent.futures import ThreadPoolExecutor

    x, w, b, dy = make(300, 700, torch.float32, torch.float32)
    want = run(x, w, b, dy, "gelu")

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            out = []
            for _ in range(10):
                (p,) = holders([x.clone()])
                out.append((run(x, w, b, dy, "gelu"), training.clip_grad_norm_([p], 1.0, error_if_nonfinite=k % 2 == 0), p.grad))
            torch.cuda.current_stream().synchronize()
            return out

    torch.cuda.synchronize()
    with ThreadPoolExecutor(4) as pool:
        results = [r for rs in pool.map(work, range(4)) for r in rs]
    for got, norm, grad in results:
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and torch.equal(norm, results[0][1])
        assert (grad - results[0][2]).abs().max() <= 4 * U * grad.abs().max()  # the factor from the norm in f64 or in f32


@gpu
def test_layer_norm_of_one_row_of_many_columns():
    """More columns than one launch has work-items for at 16 columns to a workgroup of the join."""
    n = 2 ** 27 + 5
    x = torch.randn(2, n, device="cuda")
    dy = torch.randn(2, n, device="cuda")
    w = torch.ones(n, device="cuda")
    y, dx, dw, db = run(x, w, torch.zeros_like(w), dy, None)
    assert torch.equal(db, dy[0] + dy[1])
    mean = torch.stack([r.double().mean() for r in x])
    inv = torch.stack([(r.double().var(unbiased=False) + EPS).rsqrt() for r in x])
    depth = n / 4096 + 64  # a chunk's chain is short, the join's has the chunks of a lane
    for cols in (slice(0, 1000), slice(2 ** 26, 2 ** 26 + 1000), slice(n - 1000, n)):
        h = (x[:, cols].double() - mean[:, None]) * inv[:, None]
        eh = (h.abs() + 1) * (depth + 8) * U
        near(y[:, cols], (h, eh))
        terms = h * dy[:, cols].double()
        near(dw[cols], (terms.sum(0), (eh * dy[:, cols].double().abs()).sum(0) + 4 * U * terms.abs().sum(0)))


@gpu
@pytest.mark.parametrize("cols", [5, 256, 1000, 20000, 70000])
def test_layer_norm_of_no_rows(cols):
    w = torch.ones(cols, device="cuda", requires_grad=True)
    b = torch.ones(cols, device="cuda", requires_grad=True)
    x = torch.empty(4, 0, cols, device="cuda", requires_grad=True)
    y = training.layer_norm(x, w, b, activation="gelu")
    assert y.shape == x.shape
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert dx.shape == x.shape and not dw.any() and not db.any()


@gpu
@pytest.mark.parametrize("cols", [3, 64, 256, 777, 4096, 20000, 70000])
def test_layer_norm_rows_of_extremes(cols):
    """Rows that are constant, far from zero, huge, tiny, infinite or NaN: each by the definition, and none reaches its neighbours."""
    x, w, b, dy = make(11, cols, torch.float32, torch.float32)
    x[0] = 0
    x[1] = 3.25
    x[2] += 3e4
    x[3] *= 1e15
    x[4] *= 1e-20
    x[6, 0] = math.inf
    x[7, cols // 2] = -math.inf
    x[8, -1] = math.nan
    bad = [6, 7, 8]
    good = [i for i in range(11) if i not in bad]
    for act in (None, "gelu"):
        y, dx, dw, db = run(x, w, b, dy, act)
        want = oracle(x[good], w, b, dy[good], act == "gelu")
        near(y[good], want["y"])
        near(dx[good], want["dx"])
        assert y[bad].isnan().all() and dx[bad].isnan().all()
        assert dw.isnan().all()  # every column has a row without statistics
    # eps decides where nothing varies
    y = training.layer_norm(x[:2], None, None, eps=1.0)
    assert not y.any()


@gpu
def test_gelu_at_its_ends():
    """z chosen by the bias: the normal distribution's tails to the last bits, infinities and NaN as the formula has them."""
    z = torch.tensor([-40.0, -15, -13, -9, -6, -5, -3, -1, -1e-3, -1e-30, 0, 1e-30, 1e-3, 1, 3, 6, 9, 40, 1e30, -1e30, math.inf, -math.inf,
                      math.nan], device="cuda")
    n = z.numel()
    x = torch.zeros(2, n, device="cuda")  # nothing varies: z is the bias
    b = z.clone().requires_grad_(True)
    y = training.layer_norm(x, None, b, activation="gelu")
    (db,) = torch.autograd.grad(y, b, torch.tensor([[1.0], [0.0]], device="cuda").expand(2, n))
    z64 = z.double()
    cdf = 0.5 * torch.erfc(-z64 / math.sqrt(2))
    want = z64 * cdf
    slope = cdf + z64 * torch.exp(-0.5 * z64 * z64) / math.sqrt(2 * math.pi)
    finite = z.isfinite() & (z.abs() < 1e3)
    # 5e-7 on the distribution's tail, 2 u z^2 on exp(-z^2 / 2); results below 2^-126 may vanish
    rel = 1e-6 + 4 * U * z64 * z64
    assert bool(((y[0].double() - want).abs() <= want.abs() * rel + 2.0 ** -125)[finite].all())
    near_zero = (slope.abs() * 1e-6 + (cdf + (z64 * torch.exp(-0.5 * z64 * z64)).abs()) * rel + 2.0 ** -125)
    assert bool(((db.double() - slope).abs() <= near_zero)[finite].all())
    assert y[0, -5] == 1e30 and y[0, -4] == 0 and y[0, -3] == math.inf and y[0, -2].isnan() and y[0, -1].isnan()
    assert db[-5] == 1 and db[-4] == 0 and db[-3:].isnan().all()


@gpu
@pytest.mark.parametrize("rows,cols", [(3, 17), (40, 256), (2, 5000)])
def test_layer_norm_gradient_against_differences(rows, cols):
    x, w, b, dy = make(rows, cols, torch.float32, torch.float32, seed=5)
    g = torch.Generator(device="cuda").manual_seed(9)
    step = 2.0 ** -7
    for act in (None, "gelu"):
        want = oracle(x, w, b, dy, act == "gelu")
        _, *grads = run(x, w, b, dy, act)
        for i, name in enumerate(("dx", "dw", "db")):
            args = [x, w, b]
            v = torch.randn(args[i].shape, generator=g, device="cuda")
            ends, bounds, ends64 = [], [], []
            for s in (step, -step):
                moved = list(args)
                moved[i] = args[i] + s * v
                o = oracle(*moved, None, act == "gelu")["y"]
                ends.append((training.layer_norm(*moved, activation=act).double() * dy.double()).sum())
                ends64.append((o[0] * dy.double()).sum())
                bounds.append(((1.01 * o[1] + rounding(o[0], torch.float32)) * dy.double().abs()).sum())
            along = lambda t: (t.double() * v.double()).sum()
            slope64 = along(want[name][0])
            # what the difference misses of the slope is seen in 64 bits; the rest is the kernels' rounding
            missed = ((ends64[0] - ends64[1]) / (2 * step) - slope64).abs() + slope64.abs() * 1e-6
            allowed = missed + sum(bounds) / (2 * step) + along((1.01 * want[name][1] + rounding(want[name][0], torch.float32)) * v.sign())
            assert abs((ends[0] - ends[1]) / (2 * step) - along(grads[i])) <= allowed, (name, act)


@gpu
@pytest.mark.parametrize("dtype,rows,cols", [("bf16", 2 ** 20 + 3, 2056), ("f32", 33, 66_000_000)])
def test_layer_norm_beyond_32_bit_offsets(dtype, rows, cols):
    t = TYPES[dtype]
    assert rows * cols > 2 ** 31
    x = torch.empty(rows, cols, dtype=t, device="cuda")
    for i in range(0, rows, max(1, 2 ** 28 // cols)):
        x[i:i + max(1, 2 ** 28 // cols)].normal_()
    w, b = (torch.randn(cols, device="cuda") for _ in range(2))
    w.requires_grad_(True)
    x.requires_grad_(True)
    y = training.layer_norm(x, w, b)
    last = slice(rows - 2, rows)
    want = oracle(x.detach()[last], w.detach(), b, x.detach()[last])
    near(y.detach()[last], want["y"])
    dx, dw = torch.autograd.grad(y, (x, w), x.detach())
    del y
    near(dx[last], want["dx"])
    # one column's gradient, over every row: chains of rows / 4 additions
    h = torch.cat([(c.double() - c.double().mean(-1, keepdim=True))[:, :1] / (c.double().var(-1, keepdim=True, unbiased=False) + EPS).sqrt()
                   for c in x.detach().split(max(1, 2 ** 27 // cols))])
    terms = x.detach()[:, :1].double() * h
    assert (dw[0].double() - terms.sum()).abs() <= (rows / 4 + cols / 16 + 64) * U * terms.abs().sum()


@gpu
def test_layer_norm_repeats_its_bits_and_keeps_to_its_rows():
    for rows, cols, t in ((1000, 256, torch.float32), (77, 1023, torch.float16), (9, 40000, torch.bfloat16)):
        x, w, b, dy = make(rows, cols, t, torch.float32)
        leaves = [v.requires_grad_(True) for v in (x, w, b)]
        y = training.layer_norm(*leaves, activation="gelu")
        first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(y, leaves, dy, retain_graph=True)))
        # the same rows among others: y and dx do not depend on the batch
        part = run(x.detach()[3:8], w.detach(), b.detach(), dy[3:8], "gelu")
        assert torch.equal(part[0], y.detach()[3:8]) and torch.equal(part[1], first[0][3:8])


def shape(rows, cols, dtype=capi.F32, params=capi.F32, act=capi.ACT_NONE):
    return capi.LayerNormShape(rows, cols, cols, cols, dtype, params, act, EPS)


@gpu
@pytest.mark.parametrize("rows,cols", [(3, 5), (13, 256), (7, 1001), (2, 30001), (2, 70001)])
def test_c_entries_write_nothing_but_their_outputs(rows, cols):
    L = capi.lib()
    for code, t in ((capi.F32, torch.float32), (capi.BF16, torch.bfloat16)):
        x, w, b, dy = make(rows, cols, t, torch.float32)
        s = shape(rows, cols, code, capi.F32, capi.ACT_GELU)
        room = 64
        hold = lambda n, k: torch.full((n + 2 * room,), 7.0, dtype=k, device="cuda")
        y, dx = hold(rows * cols, t), hold(rows * cols, t)
        dw, db, stats = hold(cols, torch.float32), hold(cols, torch.float32), hold(2 * rows, torch.float32)
        at = lambda v: v.data_ptr() + room * v.element_size()
        st = torch.cuda.current_stream().cuda_stream
        nf, nb = L.rbl_layer_norm_workspace(C.byref(s), 0), L.rbl_layer_norm_workspace(C.byref(s), 1)
        space = torch.full((max(nf, nb) + 256,), 9, dtype=torch.uint8, device="cuda")
        capi._check(L.rbl_layer_norm_forward(0, C.byref(s), x.data_ptr(), w.data_ptr(), b.data_ptr(), at(y), at(stats), space.data_ptr(), nf, st))
        assert bool((space[nf:] == 9).all())
        capi._check(L.rbl_layer_norm_backward(0, C.byref(s), dy.data_ptr(), x.data_ptr(), w.data_ptr(), b.data_ptr(), at(stats), at(dx), at(dw),
                                              at(db), space.data_ptr(), nb, st))
        assert bool((space[max(nf, nb):] == 9).all())
        want = oracle(x, w, b, dy, True)
        want["stats"] = (torch.stack([want["mean"][0], want["r"][0]], 1).reshape(-1), torch.stack([want["mean"][1], want["r"][1]], 1).reshape(-1))
        for name, v in (("y", y), ("dx", dx), ("dw", dw), ("db", db), ("stats", stats)):
            assert bool((v[:room] == 7).all()) and bool((v[-room:] == 7).all()), name
            near(v[room:-room], want[name], name)


@gpu
def test_operators_on_two_streams_at_once():
    """Two streams at the same work, nothing shared: results as on one."""
    x, w, b, dy = make(3000, 512, torch.float32, torch.float32)
    want = run(x, w, b, dy, "gelu")
    params = [torch.nn.Parameter(torch.empty_like(x)) for _ in range(3)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for k in range(12):
        with torch.cuda.stream(streams[k % 2]):
            g = [x * (i + 1) for i in range(3)]
            for p, v in zip(params, g):
                p.grad = v
            norm = training.clip_grad_norm_(params, 2.0)
            got.append((run(x, w, b, dy, "gelu"), norm, g))
    torch.cuda.synchronize()
    for result, norm, g in got:
        assert all(torch.equal(p, q) for p, q in zip(result, want))
        assert torch.equal(norm, got[0][1]) and all(torch.equal(p, q) for p, q in zip(g, got[0][2]))


@gpu
def test_a_captured_step_replays():
    """Forward, backward and clipping in one graph; between replays other work runs and other graphs replay."""
    graphs = []
    for k in range(2):
        x, w, b, dy = make(700, 1000, torch.float32, torch.float32, seed=k)
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                for t in leaves:
                    t.grad = None
                training.layer_norm(*leaves, activation="gelu").backward(dy)
                training.clip_grad_norm_(leaves, 1.0)
        torch.cuda.current_stream().wait_stream(side)
        for t in leaves:
            t.grad = None
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = training.layer_norm(*leaves, activation="gelu")
            y.backward(dy)
            norm = training.clip_grad_norm_(leaves, 1.0)
        graphs.append((graph, leaves, dy, y, norm))
    for turn in range(4):
        for k, (graph, leaves, dy, y, norm) in enumerate(graphs):
            with torch.no_grad():
                leaves[0].normal_(generator=torch.Generator(device="cuda").manual_seed(turn * 2 + k))
            graph.replay()
            eager = [t.detach().clone().requires_grad_(True) for t in leaves]
            ye = training.layer_norm(*eager, activation="gelu")
            ye.backward(dy)
            ne = training.clip_grad_norm_(eager, 1.0)
            torch.cuda.synchronize()
            assert torch.equal(y, ye) and torch.equal(norm, ne)
            assert all(torch.equal(p.grad, q.grad) for p, q in zip(leaves, eager))


@gpu
def test_capture_with_a_live_eager_graph_is_refused():
    x, w, b, dy = make(8, 64, torch.float32, torch.float32)
    w.requires_grad_(True)
    alive = training.layer_norm(x, w, b)
    out = {}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        try:
            training.layer_norm(x, w, b)
        except ValueError as ex:
            out["said"] = str(ex)
        with torch.no_grad():
            out["y"] = training.layer_norm(x, w, b)
        p = torch.nn.Parameter(torch.zeros(4, device="cuda"))
        p.grad = torch.zeros(4, device="cuda")
        try:
            training.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
        except ValueError as ex:
            out["clip"] = str(ex)
    assert "outside this capture" in out["said"] and "a capture cannot do" in out["clip"]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out["y"], alive)


@gpu
def test_second_derivative_is_refused():
    x, w, b, dy = make(4, 32, torch.float32, torch.float32)
    x.requires_grad_(True)
    y = training.layer_norm(x, w, b)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        torch.autograd.grad(y, x, dy, create_graph=True)


@gpu
def test_what_is_saved_may_be_computed_again_or_kept_elsewhere():
    """Hooks on the saved tensors: recomputation runs the forward pass, with gradients, inside the backward pass."""
    torch.manual_seed(3)
    net = torch.nn.Sequential(training.LayerNorm(48, activation="gelu"), torch.nn.Softsign(), training.LayerNorm(48)).cuda()
    query = torch.randn(33, 48, device="cuda")

    def grads(run):
        return torch.autograd.grad(run().square().sum(), list(net.parameters()))

    want = grads(lambda: net(query))
    again = grads(lambda: checkpoint(net, query, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    with torch.autograd.graph.save_on_cpu():
        kept = grads(lambda: net(query))
    assert all(torch.equal(a, b) for a, b in zip(kept, want))


@gpu
def test_what_a_hook_gives_back_may_lie_otherwise():
    """Saved tensors come back with other strides than they had: windows that were kept on the CPU, a weight and a bias with gaps,
    rows and columns exchanged in memory."""
    g = torch.Generator(device="cuda").manual_seed(11)
    line = torch.randn(400, generator=g, device="cuda")
    w, b = (torch.randn(300, generator=g, device="cuda") for _ in range(2))
    windows = line.unfold(0, 300, 1)
    dy = torch.randn(windows.shape, generator=g, device="cuda")
    plain = run(windows, w, b, dy, "gelu")
    with torch.autograd.graph.save_on_cpu():
        kept = run(windows, w, b, dy, "gelu")
    assert all(torch.equal(p, q) for p, q in zip(kept, plain))

    def spread(t):
        if t.dim() == 2:
            return t.t().contiguous().t()
        return torch.stack([t, torch.full_like(t, math.nan)], 1)[:, 0]

    x = windows.contiguous()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread):
        strided = run(x, w, b, dy, "gelu")
    assert all(torch.equal(p, q) for p, q in zip(strided, plain))
    ones = torch.ones_like(w)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: ones[:1].expand(300) if t.dim() == 1 else t):
        repeated = run(x, ones, ones, dy, "gelu")
    assert all(torch.equal(p, q) for p, q in zip(repeated, run(x, ones, ones, dy, "gelu")))


@gpu
@pytest.mark.parametrize("which", [0, 1, 2])
def test_what_a_hook_gives_back_has_to_be_what_was_saved(which):
    x, w, b, dy = make(6, 40, torch.float32, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    ways = {"type": lambda t: t.half(), "shape": lambda t: t[..., :39], "one dimension more": lambda t: t[None], "device": lambda t: t.cpu(),
            "layout": lambda t: t.to_sparse()}
    for name, way in ways.items():
        seen = []  # saved in the order x, weight, bias: pack gets each once

        def pack(t):
            seen.append(t)
            return len(seen) - 1, t

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda k: way(k[1].detach()) if k[0] == which else k[1]):
            y = training.layer_norm(*leaves, activation="gelu")
        assert len(seen) == 3
        with pytest.raises(RuntimeError, match="a hook of the saved tensors has returned " + ("x", "weight", "bias")[which]):
            torch.autograd.grad(y, leaves, dy)


@gpu
def test_the_node_itself_called_with_a_gradient():
    """y.grad_fn(dy) passes torch's engine and its checks by."""
    x, w, b, dy = make(6, 40, torch.float32, torch.float32)
    want = run(x, w, b, dy, "gelu")[1:]
    y = training.layer_norm(*[t.requires_grad_(True) for t in (x, w, b)], activation="gelu")
    with torch.no_grad():
        assert all(torch.equal(p, q) for p, q in zip(y.grad_fn(dy), want))
        for bad in (dy.half(), dy[:5], dy[:, :39], dy[0], dy.cpu(), dy.to_sparse()):
            with pytest.raises(RuntimeError, match="gradient of the result must be a dense"):
                y.grad_fn(bad)
        for bad in ((), (dy, dy)):
            with pytest.raises(TypeError, match="expected 1 arguments"):
                y.grad_fn(*bad)


# ---------------------------------------------------------------------------------------------------- gradient norm, clipping
def clip_oracle(tensors, p):
    """The norm in 64 bits (of what the tensors hold now)."""
    flat = torch.cat([t.double().reshape(-1) for t in tensors])
    return flat.abs().amax() if p == math.inf else flat.abs().sum() if p == 1 else flat.square().sum().sqrt()


def holders(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty_like(g))
        p.grad = g
        out.append(p)
    return out


CLIP_SETS = {
    "one value": [(1, "f32")], "one odd": [(4097, "bf16")], "small": [(n, "f32") for n in (6912, 256, 256, 256, 65536, 256, 256, 256, 1536, 6)],
    "types": [(1000, "f32"), (1001, "f16"), (999, "bf16"), (0, "f32"), (3, "f16"), (250_001, "f32")],
    "many": [(1 + 37 * i % 5000, ("f32", "bf16", "f16")[i % 3]) for i in range(700)], "large": [(9_000_001, "f32"), (7_000_003, "bf16")],
    "tiny": [(1, "bf16"), (3, "f16"), (2, "f32"), (7, "bf16"), (9, "f16"), (2048, "bf16"), (2049, "bf16"), (1024, "f32"), (1027, "f32"), (8, "f16")],
    "pairs": [(1024, "f32"), (2048, "f16")] * 48, "one more": [(1024, "f32"), (2048, "bf16")] * 48 + [(1, "f32")],
    "384 KB": [(98304, "f32")], "384 KB and one": [(98305, "f32")],
    "scattered": [(0, "f32")] * 140 + [(5, "f32")] + [(0, "bf16")] * 3 + [(70, "bf16")] * 129}


@gpu
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("name", list(CLIP_SETS))
def test_clipping_against_64_bits(name, p):
    g = torch.Generator(device="cuda").manual_seed(1)
    room = 3  # odd distances: the tensors' starts have no alignment but their elements'
    held, grads = [], []
    for n, t in CLIP_SETS[name]:
        buf = torch.full((n + 2 * room,), 5.0, dtype=TYPES[t], device="cuda")
        buf[room:room + n].normal_(generator=g)
        held.append(buf)
        grads.append(buf[room:room + n])
    before = [v.clone() for v in grads]
    want = clip_oracle(before, p)
    norm = training.grad_norm(grads, p)
    assert norm.shape == () and norm.dtype == torch.float32
    # sums in f64: the rounding to f32 is all that shows
    assert abs(norm.double() - want) <= want * U * 1.001
    assert all(torch.equal(x, y) for x, y in zip(before, grads))
    params = holders(grads)
    same = training.clip_grad_norm_(params, float(want) * 2, p)  # not reached: not a bit changes
    assert torch.equal(same, norm) and all(torch.equal(x, y) for x, y in zip(before, grads))
    bound = float(want) * 0.37
    assert torch.equal(training.clip_grad_norm_(params, bound, p, error_if_nonfinite=(name == "small")), norm)
    factor = bound / (float(want) + 1e-6)
    for x, y, buf in zip(before, grads, held):
        # the factor rounded to f32 (error_if_nonfinite: computed from the norm rounded to f32), the product to f32, the result to its type
        v = x.double() * factor
        near(y, (v, v.abs() * 3 * U), name)
        assert bool((buf[:room] == 5).all()) and bool((buf[buf.numel() - room:] == 5).all())


@gpu
def test_clipping_needs_no_scale():
    """Values whose squares have no place in f32 on either side."""
    for scale in (1e-30, 1e30):
        v = torch.randn(5000, device="cuda") * scale
        want = float(clip_oracle([v], 2))
        assert abs(float(training.grad_norm([v])) - want) <= want * U * 1.001
    (p,) = holders([torch.randn(5000, device="cuda") * 1e30])
    training.clip_grad_norm_([p], 1.0)
    assert abs(float(training.grad_norm([p.grad])) - 1) < 1e-5
    training.clip_grad_norm_([p], 0.0)
    assert not p.grad.any()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_clipping_by_a_factor_below_f32(dtype):
    """Gradients near the type's end under a small bound: the factor is below f32's normal numbers, its products are not."""
    g = torch.Generator(device="cuda").manual_seed(6)
    for n in (3, 700, 300_001):
        for bound in (1.0, 1e-3, 1e-9):
            for p, check in ((2.0, False), (math.inf, False), (math.inf, True)):
                v = ((torch.rand(n, generator=g, device="cuda") - 0.5) * 2 * 3e38).to(TYPES[dtype])
                before = v.clone()
                want = float(clip_oracle([before], p))
                norm = training.clip_grad_norm_(holders([v]), bound, p, error_if_nonfinite=check)
                assert norm == torch.tensor(want, dtype=torch.float64).float()
                w = before.double() * (bound / (want + 1e-6))
                near(v, (w, w.abs() * 3 * U), (n, bound, p, check))


@gpu
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_clipping_of_what_is_not_finite(p):
    """As the formula: an infinite norm gives the factor 0 (and inf * 0 = NaN), a NaN reaches everything."""
    for bad in (math.inf, -math.inf, math.nan):
        for at in (0, 777, 39_999):
            grads = [torch.randn(40_000, device="cuda"), torch.randn(300, device="cuda").bfloat16()]
            grads[0][at] = bad
            before = [v.clone() for v in grads]
            params = holders(grads)
            with pytest.raises(RuntimeError, match="not clipped"):
                training.clip_grad_norm_(params, 1.0, p, error_if_nonfinite=True)
            assert all(torch.equal(x.nan_to_num(9), y.nan_to_num(9)) for x, y in zip(before, grads))
            norm = training.clip_grad_norm_(params, 1.0, p)
            if math.isnan(bad):
                assert norm.isnan() and all(v.isnan().all() for v in grads)
            else:
                assert norm == math.inf and not grads[1].any() and grads[0][at].isnan() and grads[0].isnan().sum() == 1


@gpu
def test_clipping_of_other_layouts():
    big = torch.randn(40, 30, device="cuda")
    ways = {"transposed": big.clone().t(), "gaps": big.clone()[:, :7], "steps": big.clone()[::3, ::2], "dense 4d": torch.randn(3, 4, 5, 6, device="cuda").permute(2, 0, 3, 1)}
    for name, v in ways.items():
        before = v.clone()
        p = torch.nn.Parameter(torch.empty_like(before))
        p.grad = v
        want = clip_oracle([before], 2)
        assert abs(training.grad_norm([v]).double() - want) <= want * U * 1.001, name
        training.clip_grad_norm_([p], 0.5)
        w = before.double() * (0.5 / (float(want) + 1e-6))
        near(v.contiguous(), (w.contiguous(), (w.abs() * 3 * U).contiguous()), name)
    one = torch.randn(12, device="cuda")
    for pair in ([one, one], [one[:8], one[4:]], [one.view(3, 4)[:, :2], one.view(3, 4)[:, 1:]], [one[:1].expand(5)]):
        with pytest.raises(ValueError, match="memory"):
            training.clip_grad_norm_(holders(pair), 1.0)
    want = clip_oracle([one, one], 2)
    assert abs(training.grad_norm([one, one]).double() - want) <= want * U * 1.001  # only read


@gpu
def test_clipping_without_gradients():
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    q = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    assert training.clip_grad_norm_([p], 1.0) == 0
    q.grad = torch.full((3,), 2.0, device="cuda")
    assert float(training.clip_grad_norm_([p, q], 1.0)) == pytest.approx(math.sqrt(12), rel=2e-7)
    assert p.grad is None
    (e,) = holders([torch.empty(0, device="cuda")])
    assert float(training.clip_grad_norm_([e], 1.0)) == 0 and float(training.clip_grad_norm_(p, 1.0)) == 0
    assert float(training.grad_norm([torch.empty(0, 4, device="cuda")])) == 0


@gpu
def test_clipping_marks_what_it_has_written():
    """Versions grow once where gradients are scaled (in place, or copied for their gaps), and not where they are not."""
    for value in (1.0, math.nan):
        grads = [torch.full((5,), value, device="cuda"), torch.full((4, 6), value, device="cuda")[:, :3], torch.empty(0, device="cuda")]
        params = holders(grads)
        before = [g._version for g in grads]
        if math.isnan(value):
            with pytest.raises(RuntimeError, match="not clipped"):
                training.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
            assert [g._version for g in grads] == before
        for check in (False, True):
            if not (check and math.isnan(value)):
                training.clip_grad_norm_(params, 1.0, error_if_nonfinite=check)
                before = [before[0] + 1, before[1] + 1, before[2]]
                assert [g._version for g in grads] == before


@gpu
@pytest.mark.parametrize("check", [False, True])
def test_clipping_of_gradients_that_share_a_buffer(check):
    """Blocks and steps of one matrix, as a fused layer's gradient that is split by columns: each is scaled, and nothing beside them."""
    g = torch.Generator(device="cuda").manual_seed(2)
    for dtype in TYPES.values():
        whole = torch.randn(50, 41, generator=g, device="cuda").to(dtype)
        before = whole.clone()
        parts = lambda m: [m[:, :7], m[:, 7:20], m[:30, 20:30:2], m[:, 21:30:2], m[30:45, 20:29:2], m[3, 30:40]]
        want = clip_oracle(parts(before), 2)
        norm = training.clip_grad_norm_(holders(parts(whole)), 0.5, error_if_nonfinite=check)
        assert abs(norm.double() - want) <= want * U * 1.001
        touched = torch.zeros(50, 41, dtype=torch.bool, device="cuda")
        for part in parts(touched):
            part.fill_(True)
        assert torch.equal(whole[~touched], before[~touched])
        v = before.double() * (0.5 / (float(want) + 1e-6))
        near(whole[touched], (v[touched], v[touched].abs() * 3 * U))


# ---------------------------------------------------------------------------------------------------- as they are used
def plain_step(net, q, v, bound):
    """Net2's training step in 64 bits from elementary operations (torch's autograd): loss, norm, clipped gradients."""
    x = q.double()
    params = {k: p.detach().double().requires_grad_(True) for k, p in net.state_dict().items()}
    for i in (0, 4):
        x = x @ params[f"body.{i}.weight"].t() + params[f"body.{i}.bias"]
        x = (x - x.mean(-1, keepdim=True)) / (x.var(-1, keepdim=True, unbiased=False) + 1e-5).sqrt()
        x = x * params[f"body.{i + 1}.weight"] + params[f"body.{i + 1}.bias"]
        x = 0.5 * x * torch.erfc(-x / math.sqrt(2))
    e = (v.double() - (x @ params["output.weight"].t() + params["output.bias"])).abs()
    loss = torch.where(e > 1, e * 2 - 1, e * e).mean(-1).mean()
    grads = dict(zip(params, torch.autograd.grad(loss, list(params.values()))))
    norm = torch.sqrt(sum(g.square().sum() for g in grads.values()))
    c = 1.0 if bound is None else min(1.0, bound / (float(norm) + 1e-6))
    return loss, norm, {k: g * c for k, g in grads.items()}


@gpu
@pytest.mark.parametrize("batch", [512, 1, 77])
@pytest.mark.parametrize("bound", [None, 1e-3, 1e3])
def test_a_training_step_of_the_value_net(batch, bound):
    """Net2(native=True) through train_step: loss, norm and clipped gradients as in 64 bits.  The matrix products are torch's, in
    f32; a relative error of 2-norms: the longest chain (two layers of 256 terms, forward and back, sums over the batch) holds
    fewer than 4 (256 + 512) roundings of u each, times the condition of the layer norms (their slopes stay below 4 here)."""
    torch.manual_seed(0)
    net = Net2(num_faces=6, num_dice=1, n_hidden=256, use_layer_norm=True, n_layers=2, native=True).cuda()
    with torch.no_grad():
        net.output.weight *= 50  # predictions of the targets' size
    q = torch.rand(batch, 27, device="cuda")
    v = torch.randn(batch, 6, device="cuda")
    loss64, norm64, grads64 = plain_step(net, q, v, bound)
    opt = torch.optim.SGD(net.parameters(), lr=0.5)
    before = {k: p.detach().clone() for k, p in net.named_parameters()}
    loss, norm = training.train_step(net, opt, q, v, bound)
    bar = 4 * 4 * (256 + 512) * U
    assert abs(loss.double() - loss64) <= bar * loss64 and abs(norm.double() - norm64) <= bar * norm64
    whole = torch.sqrt(sum(g.square().sum() for g in grads64.values()))
    for k, p in net.named_parameters():
        assert (p.grad.double() - grads64[k]).norm() <= bar * whole, k
        assert torch.equal(p.detach(), before[k] - 0.5 * p.grad) or (p.detach() - (before[k] - 0.5 * p.grad)).abs().max() <= 1e-6
    # the trained net goes on as any other: the scripted form and the plain class hold the same values
    plain = Net2(num_faces=6, num_dice=1, n_hidden=256, use_layer_norm=True, n_layers=2).cuda()
    plain.load_state_dict(net.state_dict())
    for other in (plain, torch.jit.script(net), torch.jit.trace(net, q[:1])):
        assert (net(q) - other(q)).abs().max() <= 1e-4


@gpu
def test_layer_norm_module_trains_in_half_precision():
    torch.manual_seed(1)
    for t in (torch.float16, torch.bfloat16):
        m = training.LayerNorm(300, activation="gelu").cuda()
        with torch.no_grad():
            m.weight.normal_(1, 0.2)
            m.bias.normal_(0, 0.2)
        x = torch.randn(7, 5, 300, device="cuda").to(t).requires_grad_(True)
        dy = torch.randn(7, 5, 300, device="cuda").to(t)
        y = m(x)
        y.backward(dy)
        want = oracle(x.detach().reshape(35, 300), m.weight.detach(), m.bias.detach(), dy.reshape(35, 300), True)
        for name, got in (("y", y.detach()), ("dx", x.grad), ("dw", m.weight.grad), ("db", m.bias.grad)):
            near(got, want[name], name)
        h = training.LayerNorm(300, dtype=t, device="cuda", bias=False)
        assert h(x.detach()).dtype == t and "bias=False" in repr(h)


# ---------------------------------------------------------------------------------------------------- refusals (no GPU needed)
def test_layer_norm_refuses():
    x = torch.zeros(4, 8)
    for bad, word in (((x.double(),), "float32, float16"), ((x.long(),), "float32, float16"), ((torch.zeros(()),), "dimension"),
                      ((torch.zeros(3, 0),), "empty"), ((x, torch.ones(7)), "shape"), ((x, torch.ones(1, 8)), "shape"),
                      ((x, torch.ones(8), torch.ones(9)), "shape"), ((x, torch.ones(8).half()), "float32 or of x's type"),
                      ((x.half(), torch.ones(8).bfloat16()), "float32 or of x's type"),
                      ((x.half(), torch.ones(8).half(), torch.ones(8)), "one type"), ((x,), "no CPU path"),
                      ((x.to_sparse(),), "dense")):
        with pytest.raises(ValueError, match=word):
            training.layer_norm(*bad)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        training.layer_norm(torch.autograd.forward_ad.make_dual(x, torch.ones(4, 8)))
    with pytest.raises(ValueError, match="gelu"):
        training.layer_norm(x, activation="tanh")
    with pytest.raises(ValueError, match="gelu"):
        training.LayerNorm(8, activation="relu")
    for size in ((4, 8), 0, ()):
        with pytest.raises(ValueError, match="normalized_shape"):
            training.LayerNorm(size)
    with pytest.raises(ValueError, match="no CPU path"):
        training.LayerNorm(8)(x)
    with pytest.raises(ValueError, match="constant"):
        torch.jit.trace(training.layer_norm, x)
    with pytest.raises(ValueError, match="use_layer_norm"):
        Net2(num_faces=4, num_dice=1, native=True)


def test_clipping_refuses():
    a = torch.nn.Parameter(torch.zeros(4))
    a.grad = torch.ones(4)
    for call, word in ((lambda: training.grad_norm([a.grad]), "no CPU path"), (lambda: training.clip_grad_norm_([a], 1.0), "no CPU path"),
                       (lambda: training.grad_norm([a.grad], 3.0), "norm_type"), (lambda: training.clip_grad_norm_(a, 1.0, 0.0), "norm_type"),
                       (lambda: training.clip_grad_norm_([a], -1.0), "max_norm"), (lambda: training.clip_grad_norm_([a], math.nan), "max_norm"),
                       (lambda: training.grad_norm([a.grad.double()]), "float32, float16"), (lambda: training.grad_norm([a.grad.to_sparse()]), "sparse"),
                       (lambda: training.grad_norm([a.grad, a.grad.to("meta")]), "one device")):
        with pytest.raises(ValueError, match=word):
            call()
    with pytest.raises(ValueError, match="no gradient of its own"):
        training.grad_norm([a])
    for call in (lambda: training.grad_norm([a.grad, None]), lambda: training.clip_grad_norm_([a, 3.0], 1.0)):
        with pytest.raises(TypeError, match="expected tensors"):
            call()
    b = torch.nn.Parameter(torch.zeros(4))
    b.grad = a.grad
    with pytest.raises(ValueError, match="share memory"):
        training.clip_grad_norm_([a, b], 1.0)
    assert training.clip_grad_norm_([], 1.0) == 0 and training.grad_norm([]) == 0


def test_a_refused_clipping_leaves_no_mark():
    """A version that grew though nothing was written would fail the backward pass of whoever has saved the gradient."""
    one = torch.ones(12)
    for grads, call, word in (([one[:4], one[2:6]], {}, "share memory"), ([one[:4]], {}, "no CPU path"),
                              ([one[:4], one[4:].double()], {}, "float32, float16"), ([one[:4], one[4:].to("meta")], {}, "one device"),
                              ([one[:4], one[4:5].expand(3)], {}, "repeats its memory"), ([one[:4]], {"norm_type": 3.0}, "norm_type"),
                              ([one[:4]], {"error_if_nonfinite": True}, "no CPU path")):
        params = []
        for g in grads:
            p = torch.nn.Parameter(torch.empty_like(g))
            p.grad = g
            params.append(p)
        before = [g._version for g in grads]
        with pytest.raises(ValueError, match=word):
            training.clip_grad_norm_(params, 1.0, **call)
        assert [g._version for g in grads] == before, word


def test_memory_that_was_given_back_is_refused():
    """A weight whose storage has been resized to nothing has the address 0, which stands for no weight in the C entries."""
    x, w, b = torch.zeros(4, 8), torch.ones(8), torch.ones(16)[8:]
    for i in range(3):
        args = [t.clone() if k != 2 else torch.ones(16)[8:] for k, t in enumerate((x, w, b))]
        args[i].untyped_storage().resize_(0)
        with pytest.raises(ValueError, match="no memory"):
            training.layer_norm(*args)
        args[i].untyped_storage().resize_(4)  # less than it needs
        with pytest.raises(ValueError, match="no memory"):
            training.layer_norm(*args)
    p = torch.nn.Parameter(torch.zeros(8))
    p.grad = torch.ones(8)
    p.grad.untyped_storage().resize_(0)
    for call in (lambda: training.clip_grad_norm_([p], 1.0), lambda: training.grad_norm([p.grad])):
        with pytest.raises(ValueError, match="no memory"):
            call()
    with pytest.raises(ValueError, match="must be dense"):
        training.layer_norm(x, w.to_sparse())


class Wrapped(torch.Tensor):
    """A tensor that holds another and has no memory of its own."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.size(), dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, f, types, args=(), kwargs=None):
        raise AssertionError(f)


def test_tensors_without_memory_of_their_own_are_refused():
    x, w = torch.zeros(4, 8), torch.ones(8)
    for args in ((x, Wrapped(w)), (x, w, Wrapped(w)), (Wrapped(x), w)):
        with pytest.raises(ValueError, match="no memory"):
            training.layer_norm(*args)
    with pytest.raises(ValueError, match="no memory"):
        training.grad_norm([w, Wrapped(w)])
    with torch.no_grad(), pytest.raises(ValueError, match="no memory"):
        torch.func.vmap(training.layer_norm)(x)


@gpu
def test_memory_that_was_given_back_is_refused_backward():
    x, w, b, dy = make(6, 40, torch.float32, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    for i, name in enumerate(("x", "weight", "bias")):
        y = training.layer_norm(*leaves, activation="gelu")
        kept = leaves[i].detach().clone()
        leaves[i].untyped_storage().resize_(0)
        with pytest.raises(RuntimeError, match="has returned " + name):
            torch.autograd.grad(y, leaves, dy)
        leaves[i].untyped_storage().resize_(kept.numel() * 4)
        with torch.no_grad():
            leaves[i].data.copy_(kept)
    y = training.layer_norm(*leaves, activation="gelu")
    lost = dy.clone()
    lost.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="gradient of the result"):
        torch.autograd.grad(y, leaves, lost)


def clip_says(a, b):
    """What a clipping of two gradients on the CPU is refused for."""
    params = []
    for g in (a, b):
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype))
        p.grad = g
        params.append(p)
    with pytest.raises(ValueError) as said:
        training.clip_grad_norm_(params, 1.0)
    return "memory" if "share memory" in str(said.value) else "fine" if "no CPU path" in str(said.value) else str(said.value)


def test_gradients_of_one_buffer_are_told_apart():
    b = torch.arange(240.0)
    m, t = b.view(12, 20), b.view(3, 8, 10)
    fine = [(m[:, :3], m[:, 3:]), (m[:, 3:], m[:, :3]), (m[:, ::2], m[:, 1::2]), (b[:231].view(11, 21)[:, 4::2], b[:231].view(11, 21)[:, 5::2]), (m[::2, :4], m[::3, 4:]), (m[:5, :7], m[2:, 7:]), (m[:, :5], m[2, 5:]),
            (m.t()[:5], m.t()[5:]), (t[:, :2], t[:, 2:]), (t[:, :, :3], t[:, 1, 3:]), (t[:, 0, :3], t[:, 0, 3:]), (t[:, 1:, :9], t[1, :, 9]),
            (m[:, :10].reshape(12, 5, 2)[..., 0], m[:, 10:]), (m.view(-1)[::2].view(12, 10), m[:, 1::2]), (m[:, 0], m[:, 1]), (m[3:4, :2], m[3:4, 2:]),
            (m[:, :2].view(torch.bfloat16), m[:, 2:]), (b[0], b[1:])]
    for i, (p, q) in enumerate(fine):
        assert clip_says(p, q) == "fine", i
    shared = [(m[:, :4], m[:, 3:]), (m[:, ::2], m[:, 2::2]), (m[::2, :4], m[::3, 3:]), (m[:5, :7], m[4:, 6:]), (m[:, :5], m[2, 4:]), (m, m), (m, m.t()),
              (m[:, :6], m.t()[5:]), (t[:, :3], t[:, 2:]), (t[:, 0, :3], t[:, :, 2:]), (m[:, :2].view(torch.bfloat16)[:, 3:], m[:, 1:]),
              (m[:, 0], m[5]), (b[:1], b[:1])]
    for i, (p, q) in enumerate(shared):
        assert clip_says(p, q) == "memory", i


def test_gradients_of_one_buffer_by_chance():
    """Strided views at random: none that share an element pass; blocks of one grid, with the same steps, pass if they share none."""
    import random

    rng = random.Random(7)
    b = torch.arange(2000.0)
    for _ in range(1500):
        views = []
        for _ in range(2):
            dims = rng.randrange(1, 4)
            size, stride = [rng.randrange(1, 6) for _ in range(dims)], [rng.randrange(1, 40) for _ in range(dims)]
            views.append(b.as_strided(size, stride, rng.randrange(0, 80)))
        share = bool(set(views[0].reshape(-1).tolist()) & set(views[1].reshape(-1).tolist()))
        if share:
            assert clip_says(*views) == "memory", [(v.shape, v.stride(), v.storage_offset()) for v in views]
    grid = b[:1680].view(5, 7, 6, 8)
    for same in (True, False):  # steps of different lengths in one dimension may be refused
        passed = shared = 0
        for _ in range(4000):
            step = [rng.choice((1, 1, 2, 3)) for _ in grid.shape]
            views = []
            for _ in range(2):
                at = []
                for n, k in zip(grid.shape, step):
                    lo = rng.randrange(n)
                    at.append(slice(lo, rng.randrange(lo, n) + 1, k if same else rng.choice((1, 1, 2, 3))))
                views.append(grid[tuple(at)])
            share = bool(set(views[0].reshape(-1).tolist()) & set(views[1].reshape(-1).tolist()))
            said = clip_says(*views)
            assert said == ("memory" if share else "fine") or not (share or same), [(v.shape, v.stride(), v.storage_offset()) for v in views]
            passed, shared = passed + (said == "fine"), shared + share
        assert passed >= 300 and shared >= 100  # both sides are met often


def test_c_entries_refuse():
    """Every refusal of the C ABI comes before the device is touched: it needs none."""
    L = capi.lib()
    one = C.c_void_p(16)  # an address that nothing may read

    def fwd(s, x=one, y=one, space=None, n=0, device=0):
        return L.rbl_layer_norm_forward(device, s and C.byref(s), x, None, None, y, None, space, n, None)

    def bwd(s, dy=one, x=one, stats=one, space=one, n=1 << 40):
        return L.rbl_layer_norm_backward(0, s and C.byref(s), dy, x, None, None, stats, one, one, one, space, n, None)

    def said(status, word):
        assert status != 0 and word in L.rbl_last_error().decode(), L.rbl_last_error()

    for call in (fwd, bwd):
        said(call(None), "shape is null")
        said(call(shape(-1, 8)), "rows")
        said(call(shape(4, 0)), "cols")
        said(call(shape(4, 2 ** 30 + 1)), "cols")
        said(call(shape(2 ** 45, 2 ** 20)), "too large")
        said(call(shape(4, 8, dtype=3)), "dtype")
        said(call(shape(4, 8, dtype=capi.F16, params=capi.BF16)), "param_dtype")
        said(call(shape(4, 8, act=2)), "activation")
        said(call(capi.LayerNormShape(4, 8, -8, 8, 0, 0, 0, EPS)), "strides")
        said(call(shape(4, 8), x=None), "null")
    said(fwd(shape(4, 8), y=None), "null")
    said(bwd(shape(4, 8), dy=None), "null")
    said(bwd(shape(4, 8), stats=None), "null")
    assert L.rbl_layer_norm_workspace(None, 0) == -1 and L.rbl_layer_norm_workspace(C.byref(shape(3, -1)), 1) == -1
    for s in (shape(4, 8), shape(2, 100_000), shape(4096, 256)):
        for backward, call in ((0, fwd), (1, bwd)):
            need = L.rbl_layer_norm_workspace(C.byref(s), backward)
            assert need >= 0
            if need > 0:
                said(call(s, space=one, n=need - 1), "workspace")
                said(call(s, space=None, n=need), "workspace")

    s = shape(4, 20_000)  # one that needs no workspace forward and one backward
    for call, word in ((lambda: fwd(s, x=C.c_void_p(18)), "x, y, dy and dx"), (lambda: fwd(s, y=C.c_void_p(17)), "x, y, dy and dx"),
                       (lambda: bwd(s, dy=C.c_void_p(18)), "x, y, dy and dx"), (lambda: bwd(s, stats=C.c_void_p(20)), "stats"),
                       (lambda: bwd(s, space=C.c_void_p(24)), "workspace must be aligned")):
        said(call(), word)

    def clip(grads, n=None, norm=capi.NORM_2, bound=1.0, out=one, space=one, size=1 << 40, which=L.rbl_grad_clip):
        a = (capi.Grad * max(1, len(grads)))(*[capi.Grad(*g) for g in grads])
        n = len(grads) if n is None else n
        if which == L.rbl_grad_scale:
            return which(0, a, n, bound, out, None)
        if which == L.rbl_grad_norm:
            return which(0, a, n, norm, out, space, size, None)
        return which(0, a, n, norm, bound, out, space, size, None)

    for which in (L.rbl_grad_clip, L.rbl_grad_norm, L.rbl_grad_scale):
        said(clip([], n=-1, which=which), "negative")
        said(clip([(16, -1, 0)], which=which), "numel")
        said(clip([(16, 2 ** 59, 0), (16, 2 ** 59, 0), (16, 2, 0)], which=which), "numel")
        said(clip([(None, 4, 0)], which=which), "null")
        said(clip([(16, 4, 5)], which=which), "dtype")
        said(clip([(16, 4, 0)], out=None, which=which), "norm_dev")
    for which in (L.rbl_grad_clip, L.rbl_grad_norm):
        said(clip([(16, 4, 0)], norm=4, which=which), "norm must be")
        said(clip([(16, 4, 0)], size=7, which=which), "workspace")
        said(clip([(16, 4, 0)], space=None, which=which), "workspace")
        said(clip([(16, 4, 0)], space=C.c_void_p(20), which=which), "aligned")
        said(clip([(18, 4, 0)], which=which), "aligned")
    for which in (L.rbl_grad_clip, L.rbl_grad_scale):
        said(clip([(16, 4, 0)], bound=-1.0, which=which), "max_norm")
        said(clip([(16, 4, 0)], bound=math.nan, which=which), "max_norm")
    said(L.rbl_grad_norm(0, None, 2, capi.NORM_2, one, one, 100, None), "null")
    assert L.rbl_grad_workspace(None, 0) == 0 and L.rbl_grad_workspace(None, 1) == -1
    if capi.device_count() == 0:
        said(fwd(shape(4, 8), n=1 << 40, space=one), "HIP error")
        said(fwd(shape(4, 8), n=1 << 40, space=one, device=-1), "negative")


def test_train_kernels_have_neither_scratch_nor_flat_loads(tmp_path):
    """Every pointer of these kernels is a global one and every array lives in registers; and no packed f32 instruction is left."""
    import os
    import subprocess

    hipcc = "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rebel_amd", "csrc")
    srcs = ["layer_norm_f32.hip", "layer_norm_f16.hip", "layer_norm_bf16.hip", "grad_norm_kernel.hip"]
    runs = [subprocess.Popen([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-I../../include", "-Wno-unused-result", "-Xclang",
                              "-target-feature", "-Xclang", "-packed-fp32-ops", "-S", "--cuda-device-only", src, "-o", str(tmp_path / src)],
                             cwd=csrc, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for src in srcs]
    for src, r in zip(srcs, runs):
        said, _ = r.communicate(timeout=900)
        assert r.returncode == 0, said[-3000:]
        text = (tmp_path / src).read_text()
        for word in ("flat_load", "flat_store", "scratch_load", "scratch_store", "v_pk_fma_f32", "v_pk_mul_f32", "v_pk_add_f32"):
            assert word not in text, (src, word)
        assert ".private_segment_fixed_size: 0" in text

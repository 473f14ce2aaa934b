"""Every variant of the training kernels against the definitions in 64 bits: which of them a call takes depends on its sizes, its type
and which gradients are wanted.  The rules are restated here (and pinned to the library by the workspaces it asks for), so that a
variant that no case reaches is a failure."""
import ctypes as C
import math

import pytest
import torch

from rebel_amd import capi, training
from tests.test_training_ops import EPS, TYPES, U, clip_oracle, holders, make, near, oracle, run

gpu = pytest.mark.gpu
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CODE = {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}
CUS, STREAM_BYTES = 256, 512 << 20


def ceil(a, b):
    return -(-a // b)


# ---------------------------------------------------------------------------------------------------- layer norm: the rules
def even_grid(need, resident):
    return ceil(need, ceil(need, resident))


def forward_variant(rows, cols, dtype):
    """(threads to a row, 16 elements to a thread once or twice, no thread past the row's end, past the caches)"""
    if cols < 16 // SIZE[dtype]:
        return "one element at a time"
    for threads in (4, 8, 16, 32, 64, 128, 256, 512, 1024):
        if cols <= 16 * threads:
            break
    times = 1 if cols <= 16 * threads else 2
    if cols > 16 * threads * times:
        return "chunks"
    return threads, times, cols == 16 * threads * times, threads >= 16 and rows * cols * SIZE[dtype] >= STREAM_BYTES


class Backward:
    """What the backward pass of a shape does: threads to a row (0: chunks of a row), workgroups, rows that one thread adds up."""

    def __init__(self, rows, cols, dtype):
        self.few = rows <= 512 and rows * cols <= 1 << 21
        self.rows, self.cols, self.chunks, self.times = rows, cols, 0, 1
        self.vector = 16 // SIZE[dtype] if cols >= 16 // SIZE[dtype] else 1
        self.width = ceil(cols, 4) * 4
        if cols <= 16384:
            self.threads = 4 if cols <= 32 else 8
            while self.threads < 512 and self.threads * 8 < cols:
                self.threads *= 2
            if cols > 8192:
                self.threads = 1024
            self.times = 2 if cols > 4096 else 1
            self.group = 256 if self.threads <= 64 else self.threads
            need = ceil(rows * self.threads, self.group)
            per_cu = 512 // self.group
            if SIZE[dtype] == 2 and cols <= 4096:
                per_cu = (512 * self.threads * 8 + self.group * cols // 2) // (self.group * cols)
            self.groups = need if self.few or need == 0 else even_grid(need, CUS * min(max(per_cu, 1), 16))
        else:
            self.threads, self.group = 0, 256
            self.chunks = ceil(cols, 1024 * self.vector)
            most = ceil(2 * CUS, self.chunks)
            self.groups = rows if self.few or rows < most else most

    def workspace(self):
        row_sums = 0 if self.threads else self.rows * self.chunks * 8
        return ceil(row_sums, 16) * 16 + (0 if self.few else self.groups * 2 * self.width * 4)

    def variant(self, dtype, wanted):
        """wanted: 'all', 'x' or 'parameters'"""
        sums = "none" if wanted == "x" else "few" if self.few else "partial"
        if not self.threads:
            return "chunks", sums, wanted
        if self.vector == 1:
            return "one element at a time", sums
        even = self.cols == 8 * self.threads * self.times
        stream = sums == "partial" and self.threads >= 16 and self.rows * self.cols * SIZE[dtype] >= STREAM_BYTES
        return self.threads, self.times, even, sums, stream

    def join(self):  # columns to a workgroup where the partial sums are joined
        return None if self.few else 16 if 2 * self.width < 64 * CUS // 2 else 64

    def depth(self):
        """The longest chain of additions behind an element of the parameters' gradients."""
        if self.few:  # four lanes across, the others down the rows, then the wavefronts
            group = self.group if self.threads else 256
            return ceil(self.rows, group // 4) + 4 + group // 64
        if not self.threads:
            mine = ceil(self.rows, self.groups)
        else:
            mine = ceil(self.rows, self.groups * (self.group // self.threads)) + (4 + 4 if self.threads <= 64 else 0)
        lanes = self.join() // 4
        return mine + ceil(self.groups, 1024 // lanes) + 6 + 16


WIDTHS = [3, 20, 32, 50, 64, 100, 128, 200, 256, 400, 512, 700, 1024, 1500, 2048, 2500, 4096, 5000, 8192, 9001, 16384, 20001, 32768, 33000]
STREAMED = [w for w in WIDTHS if 64 < w <= 32768]


def many(cols):  # rows: three rounds of workgroups, and one row more
    return 1300 * max(1, 2048 // cols) + 1


def streamed(cols, dtype):
    return ceil(STREAM_BYTES, cols * SIZE[dtype]) + 1


def cases():
    """(rows, cols, dtype, wanted) of the tests below; all of them with and without GELU."""
    for dtype in TYPES:
        for cols in WIDTHS:
            for wanted in ("all", "x", "parameters"):
                yield 37, cols, dtype, wanted
                yield many(cols), cols, dtype, wanted
        for cols in STREAMED:
            yield streamed(cols, dtype), cols, dtype, "all"


def test_the_rules_are_the_librarys():
    L = capi.lib()
    for dtype in TYPES:
        for cols in sorted({max(1, w + d) for w in WIDTHS + [8, 16, 4097, 8193, 16385, 65537, 200003] for d in (-1, 0, 1)}):
            for rows in (0, 1, 2, 37, 511, 512, 513, 600, 1301, 5000, 100_003, 2_000_001):
                s = capi.LayerNormShape(rows, cols, cols, cols, CODE[dtype], capi.F32, capi.ACT_NONE, EPS)
                assert L.rbl_layer_norm_workspace(C.byref(s), 1) == Backward(rows, cols, dtype).workspace(), (rows, cols, dtype)
                chunks = forward_variant(rows, cols, dtype) == "chunks"
                assert L.rbl_layer_norm_workspace(C.byref(s), 0) == (rows * ceil(cols, 4096 * 4 // SIZE[dtype]) * 8 if chunks else 0)


def test_every_variant_of_layer_norm_has_a_case():
    reached, reachable = set(), set()
    for rows, cols, dtype, wanted in cases():
        plan = Backward(rows, cols, dtype)
        reached |= {(dtype, "forward", forward_variant(rows, cols, dtype)), (dtype, "backward", plan.variant(dtype, wanted))}
        if wanted != "x":
            reached.add((dtype, "join", plan.join()))
    for dtype in TYPES:
        for cols in [*range(1, 300), *(2 ** k + d for k in range(8, 18) for d in (-1, 0, 1)), 100_000]:
            for rows in (1, 37, 600, 20_000, streamed(cols, dtype)):
                plan = Backward(rows, cols, dtype)
                reachable.add((dtype, "forward", forward_variant(rows, cols, dtype)))
                reachable |= {(dtype, "backward", plan.variant(dtype, wanted)) for wanted in ("all", "x", "parameters")}
                reachable.add((dtype, "join", plan.join()))
    assert not reachable - reached, sorted(map(str, reachable - reached))


def compare(x, w, b, dy, gelu, got, depth):
    """got: (y, dx, dw, db), those that are there, against the definition, in blocks of rows; the parameters' gradients with the chain of
    additions that the plan gives (the shared oracle's own is that of the fewest partial sums)."""
    total = {k: [0, 0] for k in ("dw", "db")}
    rows, cols = x.shape
    for at in range(0, rows, max(1, (1 << 25) // cols)):
        part = slice(at, at + max(1, (1 << 25) // cols))
        want = oracle(x[part], w, b, dy[part], gelu)
        for name, v in (("y", got[0]), ("dx", got[1])):
            if v is not None:
                near(v[part], want[name], (name, at))
        n = x[part].shape[0]
        for name in total:
            total[name][0] = total[name][0] + want[name][0]
            total[name][1] = total[name][1] + want[name][1]
        # sum |g h| and sum |g|, of which the oracle's bound has n / 4 + 32 roundings
        x64 = x[part].double()
        h = (x64 - x64.mean(-1, keepdim=True)) / torch.sqrt(x64.var(-1, keepdim=True, unbiased=False) + EPS)
        g = dy[part].double().abs()
        if gelu:
            z = h * w.double() + b.double()
            g = (g * (0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))).abs()
        for name, s in (("dw", (g * h.abs()).sum(0)), ("db", g.sum(0))):
            total[name][1] = total[name][1] + (depth - (n / 4 + 32)) * U * s
        del x64, h, g, want
    for name, v in (("dw", got[2]), ("db", got[3])):
        if v is not None:
            near(v, total[name], name)


@gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("rows", ["few", "many"])
def test_layer_norm_variants(rows, cols, dtype):
    rows = 37 if rows == "few" else many(cols)
    depth = Backward(rows, cols, dtype).depth()
    for gelu, params in ((g, t) for g in (False, True) for t in {torch.float32, TYPES[dtype]}):
        act = "gelu" if gelu else None
        x, w, b, dy = make(rows, cols, TYPES[dtype], params)
        full = run(x, w, b, dy, act)
        compare(x, w, b, dy, gelu, full, depth)
        for wanted in ((1, 0, 0), (0, 1, 1)):
            leaves = [t.detach().requires_grad_(bool(k)) for t, k in zip((x, w, b), wanted)]
            y = training.layer_norm(*leaves, activation=act)
            grads = iter(torch.autograd.grad(y, [t for t, k in zip(leaves, wanted) if k], dy))
            compare(x, w, b, dy, gelu, (y.detach(), *[next(grads) if k else None for k in wanted]), depth)


@gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols", STREAMED)
def test_layer_norm_variants_past_the_caches(cols, dtype):
    rows = streamed(cols, dtype)
    for gelu in (False, True):
        x, w, b, dy = make(rows, cols, TYPES[dtype], torch.float32)
        compare(x, w, b, dy, gelu, run(x, w, b, dy, "gelu" if gelu else None), Backward(rows, cols, dtype).depth())
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------------------------------- gradient norm, clipping
def chunks_of(grads):
    """How many chunks the library cuts a set into: one f64 for each, and one more."""
    a = (capi.Grad * len(grads))(*[capi.Grad(16, n, CODE[t]) for n, t in grads])
    return capi.lib().rbl_grad_workspace(a, len(grads)) // 8 - 1


def mixed(count, size):
    return [(size(i), ("f32", "bf16", "f16")[i % 3]) for i in range(count)]


MB = 1 << 20
# name: (tensors, chunks).  Up to 320 chunks travel in the arguments of one launch; up to 4096 sums are added up by every workgroup of the
# scaling, more by a launch of their own; chunks grow from 8 KB to 128 KB, stay there, and grow again from 1 GB on.
SETS = {"320 chunks": (mixed(320, lambda i: 1 + i), 320), "321 chunks": (mixed(321, lambda i: 1 + i), 321),
        "4096 chunks": (mixed(4096, lambda i: 1 + i % 50), 4096), "4097 chunks": (mixed(4097, lambda i: 1 + i % 50), 4097),
        "5000 tensors": (mixed(5000, lambda i: 1 + 7 * i % 2500), None), "100 MB": (mixed(3, lambda i: 12 * MB + 5 * i + 1), None),
        "200 MB": (mixed(4, lambda i: 20 * MB + 3 * i + 1), None), "600 MB": (mixed(5, lambda i: 48 * MB + i), None),
        "1200 MB": (mixed(7, lambda i: 72 * MB + 3 * i), None)}


def test_every_way_of_clipping_has_a_set():
    for name, (grads, chunks) in SETS.items():
        assert chunks in (None, chunks_of(grads)), name
    of = {name: chunks_of(grads) for name, (grads, _) in SETS.items()}
    size = {name: sum(n * SIZE[t] for n, t in grads) for name, (grads, _) in SETS.items()}
    assert of["5000 tensors"] > 4096 and of["600 MB"] > 4096 and of["1200 MB"] > 4096
    # bytes to a chunk, by what the last chunks of a few large tensors leave over
    chunk = {name: next(1 << k for k in range(13, 40) if sum(ceil(n * SIZE[t], 1 << k) for n, t in SETS[name][0]) == of[name])
             for name in ("100 MB", "200 MB", "600 MB", "1200 MB")}
    assert chunk == {"100 MB": 64 << 10, "200 MB": 128 << 10, "600 MB": 128 << 10, "1200 MB": 256 << 10}, (chunk, size)


def values(name):
    g = torch.Generator(device="cuda").manual_seed(len(name))
    return [torch.randn(n, generator=g, device="cuda").to(TYPES[t]) for n, t in SETS[name][0]]


@gpu
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("name", list(SETS))
def test_clipping_of_many_chunks(name, p):
    grads = values(name)
    want = float(clip_oracle(grads, p))
    norm = training.grad_norm(grads, p)
    assert abs(float(norm) - want) <= want * U * 1.001
    before = [v.clone() for v in grads]
    assert torch.equal(training.clip_grad_norm_(holders(grads), 2 * want, p), norm)
    assert all(torch.equal(x, y) for x, y in zip(before, grads))
    bound = 0.37 * want
    for check in (False, True):
        held = [v.clone() for v in grads]
        assert torch.equal(training.clip_grad_norm_(holders(held), bound, p, error_if_nonfinite=check), norm)
        # as one vector of each type: the factor's rounding, the product's and (check) the norm's
        for t in TYPES.values():
            v = [x.reshape(-1) for x in before if x.dtype == t]
            got = [x.reshape(-1) for x in held if x.dtype == t]
            if v:
                w = torch.cat(v).double() * (bound / (want + 1e-6))
                near(torch.cat(got), (w, w.abs() * 3 * U), (name, check))


@gpu
@pytest.mark.parametrize("name", ["320 chunks", "4096 chunks", "4097 chunks", "5000 tensors"])
def test_clipping_keeps_to_its_workspace(name):
    """The C entries with a workspace of exactly the bytes they ask for, between guards."""
    L = capi.lib()
    for norm, p in ((capi.NORM_1, 1.0), (capi.NORM_2, 2.0), (capi.NORM_INF, math.inf)):
        grads = values(name)
        want = float(clip_oracle(grads, p))
        a = (capi.Grad * len(grads))(*[capi.Grad(v.data_ptr(), v.numel(), CODE[t]) for v, (_, t) in zip(grads, SETS[name][0])])
        need = L.rbl_grad_workspace(a, len(grads))
        space = torch.full((need + 1024,), 9, dtype=torch.uint8, device="cuda")
        out = torch.full((3,), 7.0, device="cuda")
        at, st = space.data_ptr() + 512, torch.cuda.current_stream().cuda_stream
        for call in (lambda: L.rbl_grad_norm(0, a, len(grads), norm, out.data_ptr() + 4, at, need, st),
                     lambda: L.rbl_grad_clip(0, a, len(grads), norm, 0.25 * want, out.data_ptr() + 4, at, need, st)):
            out[1] = 0
            capi._check(call())
            assert abs(float(out[1]) - want) <= want * U * 1.001 and out[0] == 7 and out[2] == 7
            assert bool((space[:512] == 9).all()) and bool((space[512 + need:] == 9).all())
        # half a step of the type at every element (bf16's the coarsest; half of f16's subnormal step), as one vector
        clipped = float(clip_oracle(grads, p))
        assert abs(clipped - 0.25 * want) <= 0.25 * want * (2 ** -8 + 3 * U) + 1e-6 + sum(n for n, _ in SETS[name][0]) * 2 ** -25

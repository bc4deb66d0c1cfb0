"""The layer operators for fields cut into regions, against their definition in 64 bits.

Bounds, per output, from the arithmetic alone.  With T = sum |terms| of the exact sum and K its length:
  * fp32 accumulation in any order, also one that truncates: at most K 2^-23 T (one step of 2^-23 per addition);
    Sums of fp32 results are cut into runs of 512 terms at most, which are added with rounding: (512 + K / 512) 2^-23 T;
  * rounding to the output type: half a step, eps/2 |y| (2^-11 fp16, 2^-8 bf16, 2^-24 fp32), and at least half of fp16's
    smallest step, 2^-25;
  * 8-bit layers: products of 8-bit values are exact in fp32; each block's scale is one rounded product (2^-24) and each
    block's term one more rounded operation: (K + 2 blocks + 2) 2^-23 T.
Quantised values and scales are compared bit for bit with the definition in IEEE fp32.
"""
import itertools

import numpy as np
import pytest

from sphericalrf_b200 import abi

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f16": (abi.TYPE_F16, torch.float16), "bf16": (abi.TYPE_BF16, torch.bfloat16), "f32": (abi.TYPE_F32, torch.float32)}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
POISON = -77.0


@pytest.fixture(scope="module")
def r(built_lib):
    from sphericalrf_b200.testbed import Renderer
    cfg = abi.default_config()
    cfg.grid_size, cfg.log2_hashmap_size = 32, 14
    ren = Renderer(cfg, 0)
    yield ren
    ren.close()


def up(n, to):
    return -(-n // to) * to


def table(rows, cols, dtype, to, fill=float("nan"), lead=()):
    """A buffer with padded rows and a view of its `cols` columns; everything holds `fill`."""
    buf = torch.full((*lead, rows, up(cols, to)), fill, dtype=torch.float32, device="cuda").to(dtype)
    return buf, buf[..., :cols]


class Case:
    """Samples of ragged groups with `front` rows before the first and `back` behind the last, NaN everywhere unused."""

    def __init__(self, sizes, n_in, n_out, kind, seed, front=0, back=0):
        self.sizes, self.n_in, self.n_out, self.kind = list(sizes), n_in, n_out, kind
        self.type_id, self.dtype = TYPES[kind]
        starts = front + np.concatenate([[0], np.cumsum(self.sizes)])
        self.spans = [(int(a), int(b)) for a, b in zip(starts[:-1], starts[1:])]
        self.used = (int(starts[0]), int(starts[-1]))
        self.n_rows = int(starts[-1]) + back
        self.offsets = torch.from_numpy(starts.astype(np.int64)).cuda()
        gen = torch.Generator(device="cuda").manual_seed(seed)
        fill = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        self.xb, self.x = table(self.n_rows, n_in, self.dtype, 8)
        self.wb, self.w = table(n_out, n_in, self.dtype, 8, lead=(len(self.sizes),))
        self.dyb, self.dy = table(self.n_rows, n_out, self.dtype, 8)
        a, b = self.used
        self.x[a:b] = fill(b - a, n_in).relu().to(self.dtype)
        self.w[:] = (fill(len(self.sizes), n_out, n_in) / max(1.0, n_in ** 0.5)).to(self.dtype)
        self.dy[a:b] = (fill(b - a, n_out) / 8).to(self.dtype)

    def layer(self, out_id, relu=False, **kw):
        base = dict(ld_x=self.xb.stride(0), ld_w=self.wb.stride(1), ld_y=self.dyb.stride(0), group_stride=self.wb.stride(0),
                    activation=abi.ACT_RELU if relu else abi.ACT_NONE)
        base.update(kw)
        return abi.make_grouped(len(self.sizes), self.n_rows, self.n_in, self.n_out, self.type_id, out_id, **base)


def fp32_length(terms):
    """The K of the bound for a sum of `terms` products with an fp32 result."""
    return min(terms, 512) + terms // 512 + 1


def check_rows(got, exact, terms, length, used, where, buf, cols):
    """Rows of `used` within the bound; every other element of the buffer still POISON."""
    a, b = used
    g = got[a:b].double()
    dt = got.dtype
    bound = HALF_STEP[dt] * exact.abs() + TINY[dt] + (1 + HALF_STEP[dt]) * length * 2.0 ** -23 * terms
    bad = ~((g - exact).abs() <= bound)
    assert not bad.any(), f"{where}: {int(bad.sum())} of {bad.numel()} off, first {bad.nonzero()[0].tolist()}, worst {float(((g - exact).abs() / bound).nan_to_num(1e9).max()):.3g} bounds"
    rest = buf.clone()
    rest[a:b, :cols] = POISON
    assert bool((rest == POISON).all()), f"{where}: wrote outside its rows"


def run_layer(r, c, out, relu=False, stream=None):
    out_id, dt = TYPES[out]
    yb, y = table(c.n_rows, c.n_out, dt, 8, POISON)
    r.grouped_matmul_device(c.layer(out_id, relu), c.offsets, c.x, c.w, y, stream)
    torch.cuda.synchronize()
    exact = torch.zeros(c.used[1] - c.used[0], c.n_out, dtype=torch.float64, device="cuda")
    terms = torch.zeros_like(exact)
    for g, (a, b) in enumerate(c.spans):
        x, w = c.x[a:b].double(), c.w[g].double()
        exact[a - c.used[0]:b - c.used[0]] = x @ w.t()
        terms[a - c.used[0]:b - c.used[0]] = x.abs() @ w.abs().t()
    if relu:
        exact = exact.clamp_min(0)
    check_rows(y, exact, terms, fp32_length(c.n_in) if out == "f32" else c.n_in, c.used, "layer", yb, c.n_out)
    return y


def run_input_grad(r, c, out, gate=False):
    out_id, dt = TYPES[out]
    dxb, dx = table(c.n_rows, c.n_in, dt, 8, POISON)
    r.grouped_input_grad_device(c.layer(out_id), c.offsets, c.dy, c.w, c.x if gate else None, dx)
    torch.cuda.synchronize()
    exact = torch.zeros(c.used[1] - c.used[0], c.n_in, dtype=torch.float64, device="cuda")
    terms = torch.zeros_like(exact)
    for g, (a, b) in enumerate(c.spans):
        dy, w = c.dy[a:b].double(), c.w[g].double()
        exact[a - c.used[0]:b - c.used[0]] = dy @ w
        terms[a - c.used[0]:b - c.used[0]] = dy.abs() @ w.abs()
    if gate:
        exact = torch.where(c.x[c.used[0]:c.used[1]].double() > 0, exact, 0.0)
    check_rows(dx, exact, terms, fp32_length(c.n_out) if out == "f32" else c.n_out, c.used, "input grad", dxb, c.n_in)


def run_weight_grad(r, c, out):
    out_id, dt = TYPES[out]
    dwb, dw = table(c.n_out, c.n_in, dt, 8, POISON, lead=(len(c.sizes),))
    p = c.layer(out_id)
    space = torch.empty(r.grouped_weight_grad_workspace(p), dtype=torch.uint8, device="cuda")
    r.grouped_weight_grad_device(p, c.offsets, c.dy, c.x, dw, space)
    torch.cuda.synchronize()
    assert bool((dwb[..., c.n_in:] == POISON).all()), "weight grad wrote its padding"
    for g, (a, b) in enumerate(c.spans):
        dy, x = c.dy[a:b].double(), c.x[a:b].double()
        exact, terms = dy.t() @ x, dy.abs().t() @ x.abs()
        bound = HALF_STEP[dt] * exact.abs() + TINY[dt] + (1 + HALF_STEP[dt]) * (fp32_length(b - a) + 300) * 2.0 ** -23 * terms   # + joins of at most 2 x 148 partial sums
        if a == b:
            bound = torch.zeros_like(bound)
        bad = ~((dw[g].double() - exact).abs() <= bound)
        assert not bad.any(), f"group {g} of {b - a}: {int(bad.sum())} of {bad.numel()} off, first {bad.nonzero()[0].tolist()}"


SHAPES = [
    # sizes, n_in, n_out, front, back
    ([1], 16, 16, 0, 0),
    ([128], 64, 64, 0, 0),
    ([129, 127, 0, 1], 64, 64, 0, 5),
    ([0, 0, 3, 0], 32, 64, 7, 3),
    ([300, 17, 64], 33, 65, 1, 2),
    ([5, 250], 1, 1, 0, 0),
    ([200, 56], 100, 31, 0, 130),
    ([700, 1, 511, 130], 257, 300, 3, 0),
    ([40] * 40 + [0] * 30 + [1] * 35, 48, 80, 0, 1),
    ([1000, 2000], 520, 392, 0, 40),
    ([4096], 128, 1030, 0, 0),
    ([20000, 3], 16, 129, 0, 0),
    ([260, 900, 64, 2500], 512, 768, 0, 0),
    ([20000, 3, 0, 18001], 136, 600, 2, 9),
    ([9000, 30000], 700, 264, 0, 0),
    ([700, 90, 0, 1500, 64, 333, 1, 2000], 1100, 600, 0, 11),
    ([30] * 160 + [0] * 3 + [500, 7], 40, 72, 5, 0),
    ([30000], 420, 170, 0, 0),
]


@pytest.mark.parametrize("kind,out,relu", [("f16", "f16", True), ("bf16", "bf16", False), ("f16", "f32", False), ("bf16", "f32", True)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_layer(r, shape, kind, out, relu):
    sizes, n_in, n_out, front, back = SHAPES[shape]
    run_layer(r, Case(sizes, n_in, n_out, kind, shape, front, back), out, relu)


@pytest.mark.parametrize("kind,out,gate", [("f16", "f16", True), ("bf16", "bf16", False), ("bf16", "bf16", True), ("f16", "f32", True)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_input_grad(r, shape, kind, out, gate):
    sizes, n_in, n_out, front, back = SHAPES[shape]
    run_input_grad(r, Case(sizes, n_in, n_out, kind, 50 + shape, front, back), out, gate)


@pytest.mark.parametrize("kind,out", [("f16", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_weight_grad(r, shape, kind, out):
    sizes, n_in, n_out, front, back = SHAPES[shape]
    run_weight_grad(r, Case(sizes, n_in, n_out, kind, 90 + shape, front, back), out)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_long_sums_keep_fp32(r, kind):
    """fp32 results of long sums, in the 2-norm.  An instruction adds 16 products to its accumulator and loses at most one
    step of 2^-23 of it, half a step on average: 32 instructions of a run of 512 lose 32 2^-24 of the run's size, and the
    runs' sizes and errors both add in squares, whatever their number."""
    c = Case([700, 0, 9000], 4096, 1536, kind, 77)
    y = torch.zeros(c.n_rows, c.n_out, device="cuda")
    dx = torch.zeros(c.n_rows, c.n_in, device="cuda")
    dw = torch.zeros(3, c.n_out, c.n_in, device="cuda")
    r.grouped_matmul_device(c.layer(abi.TYPE_F32), c.offsets, c.x, c.w, y)
    r.grouped_input_grad_device(c.layer(abi.TYPE_F32), c.offsets, c.dy, c.w, None, dx)
    p = c.layer(abi.TYPE_F32)
    space = torch.empty(r.grouped_weight_grad_workspace(p), dtype=torch.uint8, device="cuda")
    r.grouped_weight_grad_device(p, c.offsets, c.dy, c.x, dw, space)
    torch.cuda.synchronize()
    for g, (a, b) in enumerate(c.spans):
        if a == b:
            continue
        x, w, dy = c.x[a:b].double(), c.w[g].double(), c.dy[a:b].double()
        for got, exact in ((y[a:b], x @ w.t()), (dx[a:b], dy @ w), (dw[g], dy.t() @ x)):
            assert float((got.double() - exact).norm()) <= 32 * 2.0 ** -24 * float(exact.norm())


def test_nan_of_one_group_stays_there(r):
    c = Case([100, 37, 90], 64, 64, "bf16", 3)
    a, b = c.spans[1]
    c.x[a:b] = float("inf")
    c.dy[a:b] = float("nan")
    for fn in (lambda: run_group_finite(r, c),):
        fn()


def run_group_finite(r, c):
    y = torch.zeros(c.n_rows, c.n_out, dtype=c.dtype, device="cuda")
    dx = torch.zeros(c.n_rows, c.n_in, dtype=c.dtype, device="cuda")
    dw = torch.zeros(len(c.sizes), c.n_out, c.n_in, device="cuda")
    r.grouped_matmul_device(c.layer(c.type_id), c.offsets, c.x, c.w, y)
    r.grouped_input_grad_device(c.layer(c.type_id), c.offsets, c.dy, c.w, c.x, dx)
    p = c.layer(abi.TYPE_F32)
    space = torch.empty(r.grouped_weight_grad_workspace(p), dtype=torch.uint8, device="cuda")
    r.grouped_weight_grad_device(p, c.offsets, c.dy, c.x, dw, space)
    torch.cuda.synchronize()
    a, b = c.spans[1]
    for v in (y, dx):
        assert bool(v[:a].isfinite().all()) and bool(v[b:].isfinite().all()) and not bool(v[a:b].isfinite().all())
    assert bool(dw[0].isfinite().all()) and bool(dw[2].isfinite().all()) and bool(dw[1].isnan().all())


def test_relu_keeps_nan_and_gate_shuts_on_nan(r):
    c = Case([4], 16, 16, "f16", 5)
    c.x[1, 3] = float("nan")
    y = torch.zeros(4, 16, dtype=torch.float16, device="cuda")
    r.grouped_matmul_device(c.layer(abi.TYPE_F16, relu=True), c.offsets, c.x, c.w, y)
    gate = c.x.clone()
    gate[:] = torch.tensor([float("nan"), 0.0, -0.0, 6e-8, -1.0, float("inf"), -float("inf"), 1.0] * 2, device="cuda").half()
    dx = torch.full((4, 16), POISON, dtype=torch.float16, device="cuda")
    r.grouped_input_grad_device(c.layer(abi.TYPE_F16, ld_x=16), c.offsets, c.dy, c.w, gate, dx)
    torch.cuda.synchronize()
    assert bool(y[1].isnan().all()) and bool(y[[0, 2, 3]].isfinite().all())
    open_ = torch.tensor([0, 0, 0, 1, 0, 1, 0, 1] * 2, device="cuda").bool()
    assert bool((dx[:, ~open_] == 0).all())
    exact = (c.dy.double() @ c.w[0].double())[:, open_]
    assert float((dx[:, open_].double() - exact).abs().max()) <= 2.0 ** -11 * float(exact.abs().max()) + 2.0 ** -24 + 16 * 2.0 ** -23 * 16


def test_one_group_without_offsets(r):
    c = Case([300], 64, 48, "f16", 8)
    c.offsets = None
    run_layer(r, c, "f16")
    run_input_grad(r, c, "f16", True)
    run_weight_grad(r, c, "f32")


def test_no_rows(r):
    """n_rows = 0: nothing to write but the weight gradients, which are zero."""
    p = abi.make_grouped(3, 0, 64, 64, abi.TYPE_F16, abi.TYPE_F32)
    off = torch.zeros(4, dtype=torch.int64, device="cuda")
    none = torch.zeros(0, dtype=torch.float16, device="cuda")
    w = torch.zeros(3, 64, 64, dtype=torch.float16, device="cuda")
    dw = torch.full((3, 64, 64), POISON, device="cuda")
    r.grouped_matmul_device(p, off, none, w, none)
    r.grouped_input_grad_device(p, off, none, w, None, none)
    space = torch.empty(r.grouped_weight_grad_workspace(p), dtype=torch.uint8, device="cuda")
    r.grouped_weight_grad_device(p, off, none, none, dw, space)
    torch.cuda.synchronize()
    assert bool((dw == 0).all())


@pytest.mark.parametrize("offsets", [[0, 50, 40, 100], [0, 50, 90, 101], [5, 2, 2, 2], [2 ** 63, 2 ** 63 + 1, 7, 9], [0, 2 ** 40, 2 ** 41, 2 ** 42]])
def test_bad_offsets_are_reported(r, offsets):
    """Offsets that run backwards or out of the buffers: no access outside them, an error at the next check."""
    c = Case([30, 30, 40], 64, 64, "f16", 9)
    c.offsets = torch.from_numpy(np.array(offsets, np.uint64).view(np.int64)).cuda()
    guard = 64
    y = torch.full((guard + c.n_rows + guard, 64), POISON, dtype=torch.float16, device="cuda")
    dw = torch.full((5, 64, 64), POISON, device="cuda")
    for call in range(3):
        if call == 0:
            r.grouped_matmul_device(c.layer(abi.TYPE_F16), c.offsets, c.x, c.w, y[guard:])
        elif call == 1:
            r.grouped_input_grad_device(c.layer(abi.TYPE_F16), c.offsets, c.dy, c.w, None, y[guard:])
        else:
            p = c.layer(abi.TYPE_F32)
            space = torch.empty(r.grouped_weight_grad_workspace(p), dtype=torch.uint8, device="cuda")
            r.grouped_weight_grad_device(p, c.offsets, c.dy, c.x, dw[1:], space)
        with pytest.raises(abi.SrfError, match="offsets") as e:
            r.check_errors()
        assert e.value.status == abi.ERR_ARG
    c8 = Case8([30, 30, 40], 64, 64, 9)
    p = abi.make_grouped(3, c8.base.n_rows, 64, 64, abi.TYPE_E4M3, abi.TYPE_F16)
    r.grouped_matmul_fp8_device(p, c.offsets, c8.x, c8.xs, c8.w, c8.ws, y[guard:])
    with pytest.raises(abi.SrfError, match="offsets"):
        r.check_errors()
    r.check_errors()
    assert bool((y[:guard] == POISON).all()) and bool((y[-guard:] == POISON).all())
    assert bool((dw[0] == POISON).all()) and bool((dw[4] == POISON).all())


@pytest.mark.parametrize("sizes,n_in,n_out", [([5000, 0, 321, 70000], 72, 200), ([3000, 900, 0, 2500, 4000], 1024, 1032)])
def test_weight_grad_is_the_same_every_time(r, sizes, n_in, n_out):
    c = Case(sizes, n_in, n_out, "bf16", 11)
    p = c.layer(abi.TYPE_F32, ld_w=n_in, group_stride=0)
    got = []
    for k in range(3):
        space = torch.full((r.grouped_weight_grad_workspace(p),), 255 - k, dtype=torch.uint8, device="cuda")
        dw = torch.full((len(sizes), n_out, n_in), POISON, device="cuda")
        r.grouped_weight_grad_device(p, c.offsets, c.dy, c.x, dw, space)
        torch.cuda.synchronize()
        got.append(dw)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_small_workspace_is_refused(r):
    c = Case([100], 64, 64, "f16", 12)
    p = c.layer(abi.TYPE_F32)
    space = torch.empty(r.grouped_weight_grad_workspace(p) - 1, dtype=torch.uint8, device="cuda")
    with pytest.raises(abi.SrfError) as e:
        r.grouped_weight_grad_device(p, c.offsets, c.dy, c.x, torch.zeros(1, 64, 64, device="cuda"), space)
    assert e.value.status == abi.ERR_CAPACITY


def test_rows_behind_two_to_the_31_bytes_and_elements(r):
    """The used samples lie behind 2^32 elements of the buffer."""
    far = (1 << 26) + 77
    sizes, n_in, n_out = [0, 150, 131], 72, 64
    n_rows = far + sum(sizes) + 5
    assert far * n_in > 1 << 32
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.empty(n_rows, n_in, dtype=torch.float16, device="cuda")
    y = torch.empty(n_rows, n_out, dtype=torch.float16, device="cuda")
    x[far:] = torch.randn(n_rows - far, n_in, generator=gen, device="cuda").half()
    y[far:] = POISON
    y[far - 8:far] = POISON
    w = (torch.randn(3, n_out, n_in, generator=gen, device="cuda") / 8).half()
    off = torch.tensor([far, far, far + 150, far + 281], device="cuda")
    r.grouped_matmul_device(abi.make_grouped(3, n_rows, n_in, n_out, abi.TYPE_F16), off, x, w, y)
    torch.cuda.synchronize()
    assert bool((y[far - 8:far] == POISON).all()) and bool((y[far + 281:] == POISON).all())
    for g, a, b in ((1, far, far + 150), (2, far + 150, far + 281)):
        exact, terms = x[a:b].double() @ w[g].double().t(), x[a:b].double().abs() @ w[g].double().abs().t()
        assert bool(((y[a:b].double() - exact).abs() <= 2.0 ** -11 * exact.abs() + 2.0 ** -25 + 1.001 * n_in * 2.0 ** -23 * terms).all())


EXTREMES = [
    ([k % 4 for k in range(4096)], 24, 16, 0, 1),          # the most groups
    ([3], 16, 65536, 0, 0),                                # the widest layers
    ([2, 1], 65536, 24, 0, 0),
    ([5, 0, 2], 264, 520, 3, 200000),                      # a capacity far above what is used
    ([1] * 148 * 3, 128, 256, 0, 0),                       # one sample a group
]


@pytest.mark.parametrize("case", range(len(EXTREMES)))
def test_extremes(r, case):
    sizes, n_in, n_out, front, back = EXTREMES[case]
    c = Case(sizes, n_in, n_out, "f16", 300 + case, front, back)
    run_layer(r, c, "f16", True)
    run_layer(r, c, "f32")
    run_input_grad(r, c, "f16", True)
    run_weight_grad(r, c, "f32")
    run_layer_fp8(r, Case8(sizes, n_in, n_out, 310 + case, front, back), "bf16", False)


def test_calls_see_each_other(r):
    """Calls set themselves up while the one in front still runs: a long chain without waits, torch's own kernels in
    between, has the bits of the same chain with a wait after every step."""
    n, off = 5000, torch.tensor([0, 1200, 1200, 5000], device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(6)
    w = (torch.randn(3, 64, 64, generator=gen, device="cuda") / 6).half()
    start = torch.randn(n, 64, generator=gen, device="cuda").half()
    fwd = abi.make_grouped(3, n, 64, 64, abi.TYPE_F16, activation=abi.ACT_RELU)
    bwd, bww = abi.make_grouped(3, n, 64, 64, abi.TYPE_F16), abi.make_grouped(3, n, 64, 64, abi.TYPE_F16, abi.TYPE_F32)
    space = torch.empty(r.grouped_weight_grad_workspace(bww), dtype=torch.uint8, device="cuda")

    def chain(wait):
        a, b, d = start.clone(), torch.zeros_like(start), torch.zeros_like(start)
        dw, total = torch.zeros(3, 64, 64, device="cuda"), torch.zeros(3, 64, 64, device="cuda")
        q, qs = torch.zeros(n, 64, dtype=torch.uint8, device="cuda"), torch.zeros(1, n, device="cuda")
        for i in range(30):
            r.grouped_matmul_device(fwd, off, a, w, b)
            wait()
            r.grouped_input_grad_device(bwd, off, b, w, b.clone() if i % 3 == 0 else None, d)
            wait()
            r.grouped_weight_grad_device(bww, off, d, b, dw, space)
            wait()
            r.quantize_rows_device(abi.TYPE_F16, n, 64, d, 64, q, 64, qs)
            wait()
            total += dw
            a.copy_(d).mul_(0.5).add_(q.view(torch.float8_e4m3fn).half(), alpha=0.001).clamp_(-4, 4)
            wait()
        torch.cuda.synchronize()
        return a, total, q, qs

    for got, want in zip(chain(lambda: None), chain(torch.cuda.synchronize)):
        assert torch.equal(got, want)


# ---- 8 bits ----

def e4m3_reference(v32, scale):
    """IEEE fp32 quotient, then the nearest e4m3 value (bits)."""
    q = np.clip(v32 / scale, -448.0, 448.0).astype(np.float32)
    q[~np.isfinite(v32)] = np.nan
    bits = torch.from_numpy(q).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    bits[~np.isfinite(v32)] = 0x7F
    return bits


def scale_reference(block):
    top = np.max(np.abs(np.where(np.isfinite(block), block, 0)))
    return np.float32(1) if top == 0 else np.maximum(np.float32(top) / np.float32(448), np.float32(2.0 ** -126))


def values(rows, cols, dtype, seed, lead=()):
    gen = torch.Generator().manual_seed(seed)
    v = torch.randn(*lead, rows, cols, generator=gen) * torch.exp2(3 * torch.randn(*lead, rows, 1, generator=gen))
    v = v.to(dtype)
    flat = v.view(-1, cols)
    flat[0] = 0                                            # a block of zeros
    if rows > 3:
        flat[1, 0], flat[2, cols - 1] = float("nan"), float("inf")
        flat[3] = flat[3] * 0 + torch.finfo(dtype).tiny    # the smallest normal value
        flat[3, 0] = torch.finfo(dtype).smallest_normal / 2
    if rows > 5:
        flat[4] = torch.finfo(dtype).max
        flat[5] = -float("inf")
    return v


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,cols,used", [(1, 1, None), (1, 128, None), (37, 129, None), (70, 100, 33), (9, 1000, 9), (130, 2048, 0), (40, 256, 99), (133, 512, None)])
def test_quantize_rows(r, rows, cols, used, kind):
    type_id, dt = TYPES[kind]
    v = values(rows, cols, dt, rows + cols)
    vb, dev = table(rows, cols, dt, 8)
    dev[:] = v.cuda()
    q = torch.full((rows, up(cols, 16)), 0x55, dtype=torch.uint8, device="cuda")
    nb = up(cols, 128) // 128
    scales = torch.full((nb, rows), POISON, device="cuda")
    count = None if used is None else torch.tensor([used], dtype=torch.int64, device="cuda")
    r.quantize_rows_device(type_id, rows, cols, dev, vb.stride(0), q, q.stride(0), scales, n_rows_used=count)
    torch.cuda.synchronize()
    n = rows if used is None else min(used, rows)
    f = v.float().numpy()
    want_q, want_s = np.full(q.shape, 0x55, np.uint8), np.full((nb, rows), POISON, np.float32)
    for i, j in itertools.product(range(n), range(nb)):
        block = f[i, 128 * j:128 * j + 128]
        want_s[j, i] = scale_reference(block)
        want_q[i, 128 * j:min(cols, 128 * j + 128)] = e4m3_reference(block, want_s[j, i])
    assert np.array_equal(scales.cpu().numpy(), want_s)
    assert np.array_equal(q.cpu().numpy(), want_q)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("mats,rows,cols", [(1, 1, 1), (1, 128, 128), (3, 130, 300), (2, 64, 16), (2, 257, 100)])
def test_quantize_weights(r, mats, rows, cols, kind):
    type_id, dt = TYPES[kind]
    v = values(rows, cols, dt, rows + cols, lead=(mats,))
    vb, dev = table(rows, cols, dt, 16, lead=(mats,))
    dev[:] = v.cuda()
    q = torch.full((mats, rows, up(cols, 16)), 0x55, dtype=torch.uint8, device="cuda")
    nr, nc = up(rows, 128) // 128, up(cols, 128) // 128
    scales = torch.full((mats, nr, nc), POISON, device="cuda")
    r.quantize_weights_device(type_id, mats, rows, cols, dev, vb.stride(1), q, q.stride(1), scales)
    torch.cuda.synchronize()
    f = v.float().numpy()
    want_q, want_s = np.full(q.shape, 0x55, np.uint8), np.zeros((mats, nr, nc), np.float32)
    for m, i, j in itertools.product(range(mats), range(nr), range(nc)):
        block = f[m, 128 * i:128 * i + 128, 128 * j:128 * j + 128]
        want_s[m, i, j] = scale_reference(block)
        want_q[m, 128 * i:128 * i + 128, 128 * j:min(cols, 128 * j + 128)] = e4m3_reference(block, want_s[m, i, j])
    assert np.array_equal(scales.cpu().numpy(), want_s)
    assert np.array_equal(q.cpu().numpy(), want_q)


class Case8:
    """A Case in 8 bits: random e4m3 values and random positive scales, NaN in unused places."""

    def __init__(self, sizes, n_in, n_out, seed, front=0, back=0):
        base = Case(sizes, n_in, n_out, "f16", seed, front, back)
        self.base, self.n_in, self.n_out = base, n_in, n_out
        kb, nb = up(n_in, 128) // 128, up(n_out, 128) // 128
        gen = torch.Generator(device="cuda").manual_seed(seed + 1)
        scale = lambda *s: torch.exp2(4 * torch.rand(*s, generator=gen, device="cuda") - 4)  # noqa: E731
        self.xb, self.x = table(base.n_rows, n_in, torch.float8_e4m3fn, 16)
        self.wb, self.w = table(n_out, n_in, torch.float8_e4m3fn, 16, lead=(len(base.sizes),))
        a, b = base.used
        self.x[a:b] = (base.x[a:b].float() * 8 - 2).to(torch.float8_e4m3fn)
        self.w[:] = (base.w.float() * 8).to(torch.float8_e4m3fn)
        self.xs = torch.full((kb, base.n_rows), float("nan"), device="cuda")
        self.xs[:, a:b] = scale(kb, b - a)
        self.ws = scale(len(base.sizes), nb, kb)

    def exact(self):
        c = self.base
        out = torch.zeros(c.used[1] - c.used[0], self.n_out, dtype=torch.float64, device="cuda")
        terms = torch.zeros_like(out)
        for g, (a, b) in enumerate(c.spans):
            x = self.x[a:b].double() * self.xs[:, a:b].t().double().repeat_interleave(128, 1)[:, :self.n_in]
            w = self.w[g].double() * self.ws[g].double().repeat_interleave(128, 0)[:self.n_out].repeat_interleave(128, 1)[:, :self.n_in]
            out[a - c.used[0]:b - c.used[0]] = x @ w.t()
            terms[a - c.used[0]:b - c.used[0]] = x.abs() @ w.abs().t()
        return out, terms


@pytest.mark.parametrize("out,relu", [("f16", True), ("bf16", False), ("f32", False)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_layer_fp8(r, shape, out, relu):
    sizes, n_in, n_out, front, back = SHAPES[shape]
    run_layer_fp8(r, Case8(sizes, n_in, n_out, 200 + shape, front, back), out, relu)


def run_layer_fp8(r, c, out, relu):
    n_in, n_out = c.n_in, c.n_out
    out_id, dt = TYPES[out]
    yb, y = table(c.base.n_rows, n_out, dt, 8, POISON)
    p = abi.make_grouped(len(c.base.sizes), c.base.n_rows, n_in, n_out, abi.TYPE_E4M3, out_id, abi.ACT_RELU if relu else abi.ACT_NONE,
                         c.xb.stride(0), c.wb.stride(1), yb.stride(0), c.wb.stride(0))
    r.grouped_matmul_fp8_device(p, c.base.offsets, c.x, c.xs, c.w, c.ws, y)
    torch.cuda.synchronize()
    exact, terms = c.exact()
    if relu:
        exact = exact.clamp_min(0)
    check_rows(y, exact, terms, n_in + 2 * (up(n_in, 128) // 128) + 2, c.base.used, "fp8 layer", yb, n_out)


# ---- together ----

class Chain:
    """Three layers of regional networks, forward and backward, as a training step runs them: 32 -> 64 -> 64 -> 16."""
    WIDTHS = [32, 64, 64, 16]

    def __init__(self, r, counts, seed=0):
        self.r, n = r, int(sum(counts))
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.counts = torch.tensor(counts, dtype=torch.int32, device="cuda")
        self.offsets = torch.zeros(len(counts) + 1, dtype=torch.int64, device="cuda")
        half = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")  # noqa: E731
        w = self.WIDTHS
        self.h = [half(n, k) for k in w]
        self.h[0][:] = torch.randn(n, w[0], generator=gen, device="cuda").half()
        self.w = [(torch.randn(len(counts), o, i, generator=gen, device="cuda") / i ** 0.5).half() for i, o in zip(w[:-1], w[1:])]
        self.d = [half(n, k) for k in w]
        self.d[3][:] = torch.randn(n, w[3], generator=gen, device="cuda").half() / 4
        self.dw = [torch.zeros(len(counts), o, i, device="cuda") for i, o in zip(w[:-1], w[1:])]
        self.fwd = [abi.make_grouped(len(counts), n, i, o, abi.TYPE_F16, activation=abi.ACT_RELU if k < 2 else abi.ACT_NONE) for k, (i, o) in enumerate(zip(w[:-1], w[1:]))]
        self.bwd = [abi.make_grouped(len(counts), n, i, o, abi.TYPE_F16) for i, o in zip(w[:-1], w[1:])]
        self.bww = [abi.make_grouped(len(counts), n, i, o, abi.TYPE_F16, abi.TYPE_F32) for i, o in zip(w[:-1], w[1:])]
        self.space = torch.empty(max(r.grouped_weight_grad_workspace(p) for p in self.bww), dtype=torch.uint8, device="cuda")
        r._ck(r.lib.srf_sample_offsets(r.ctx, self.counts.data_ptr(), len(counts), self.offsets.data_ptr(), None))   # per-region counts -> offsets

    def step(self, stream=None):
        for k in range(3):
            self.r.grouped_matmul_device(self.fwd[k], self.offsets, self.h[k], self.w[k], self.h[k + 1], stream)
        for k in (2, 1, 0):
            self.r.grouped_weight_grad_device(self.bww[k], self.offsets, self.d[k + 1], self.h[k], self.dw[k], self.space, stream)
            self.r.grouped_input_grad_device(self.bwd[k], self.offsets, self.d[k + 1], self.w[k], self.h[k] if k else None, self.d[k], stream)

    def clear(self):
        for t in self.h[1:] + self.d[:3] + self.dw:
            t.zero_()

    def results(self):
        torch.cuda.synchronize()
        return [t.clone() for t in self.h[1:] + self.d[:3] + self.dw]


def test_training_step_of_regional_networks(r):
    """A run of the calls: the gradients against torch's autograd in 64 bits, and against differences of the loss."""
    counts = [700, 0, 1, 333, 2048]
    c = Chain(r, counts, 5)
    c.step()
    c.results()
    assert c.offsets.tolist() == [0] + np.cumsum(counts).tolist()
    w64 = [w.double().requires_grad_() for w in c.w]
    x64 = c.h[0].double().requires_grad_()

    # A ReLU whose argument is nearer to zero than its rounding may open in one computation and not in the other: a share p of
    # such units moves the gradient by sqrt(p) of its norm, far more than any rounding.  The network is linear between those
    # borders, so the 64-bit chain takes the piece that the kernels were on, and its gradients are the exact ones there.
    open_ = [(c.h[k] > 0).double() for k in (1, 2)]

    def loss(ws, x):
        out, total = [], 0.0
        for g in range(len(counts)):
            h = x[c.offsets[g]:c.offsets[g + 1]]
            for k in range(3):
                h = h @ ws[k][g].t()
                h = h * open_[k][c.offsets[g]:c.offsets[g + 1]] if k < 2 else h
            total = total + (h * c.d[3][c.offsets[g]:c.offsets[g + 1]].double()).sum()
            out.append(h)
        return total, torch.cat(out)

    total, out = loss(w64, x64)
    total.backward()
    # The kernels round activations and gradients to fp16 between layers, 2^-11 of each value at most; over three layers
    # forward and three back that is a few 2^-11 of the tensors' norms: 2-norms within 2^-7 (sixteen half steps).
    def near(a, b, what):
        b = b.detach()
        assert float((a.double() - b).norm()) <= 2.0 ** -7 * float(b.norm()), what
    near(c.h[3], out, "output")
    near(c.d[0], x64.grad, "input gradient")
    for k in range(3):
        near(c.dw[k], w64[k].grad, f"weight gradient {k}")
        assert bool((c.dw[k][1] == 0).all())
    # differences of the 64-bit loss along a random direction of the weights
    gen = torch.Generator(device="cuda").manual_seed(1)
    dirs = [torch.randn(w.shape, generator=gen, device="cuda").double() for w in c.w]
    eps = 1e-6
    with torch.no_grad():
        hi, _ = loss([w + eps * d for w, d in zip(w64, dirs)], x64)
        lo, _ = loss([w - eps * d for w, d in zip(w64, dirs)], x64)
    slope = sum(float((g.double() * d).sum()) for g, d in zip(c.dw, dirs))
    size = sum(float(g.double().norm() * d.norm()) for g, d in zip(c.dw, dirs))
    assert abs(slope - float(hi - lo) / (2 * eps)) <= 2.0 ** -7 * size


def test_graphs_and_streams(r):
    """Captured and replayed, two chains with workspaces of their own on two streams at once: the same bits as eager."""
    chains = [Chain(r, [500, 20, 0, 4000], 1), Chain(r, [31, 3000, 129, 1], 2)]
    want = []
    for c in chains:
        c.step()
        want.append(c.results())
    graphs, streams = [], [torch.cuda.Stream() for _ in chains]
    for c, s in zip(chains, streams):
        c.clear()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.step(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
        assert all(bool((t == 0).all()) for t in c.results())     # capture runs nothing
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    for c, w in zip(chains, want):
        assert all(torch.equal(a, b) for a, b in zip(c.results(), w))
    # new counts in the captured buffers: the replay reads them on the device
    chains[0].counts[:] = torch.tensor([1, 4000, 500, 19], dtype=torch.int32, device="cuda")
    r._ck(r.lib.srf_sample_offsets(r.ctx, chains[0].counts.data_ptr(), 4, chains[0].offsets.data_ptr(), None))
    torch.cuda.synchronize()
    chains[0].clear()
    torch.cuda.synchronize()
    graphs[0].replay()
    again = chains[0].results()
    chains[0].clear()
    chains[0].step()
    assert all(torch.equal(a, b) for a, b in zip(again, chains[0].results()))
    assert not torch.equal(again[0], want[0][0])


def test_rendering_chain_in_8_bits(r):
    """Weights and samples to 8 bits, the layer, its samples to 8 bits again, the next layer."""
    counts, widths = [300, 0, 77, 900], [256, 384, 128]
    n = sum(counts)
    gen = torch.Generator(device="cuda").manual_seed(3)
    off = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)])).cuda()
    h = torch.randn(n + 20, widths[0], generator=gen, device="cuda").to(torch.bfloat16)
    exact = h[:n].double()
    for k, (i, o) in enumerate(zip(widths[:-1], widths[1:])):
        w = (torch.randn(4, o, i, generator=gen, device="cuda") / i ** 0.5).to(torch.bfloat16)
        w8, ws = torch.zeros(4, o, i, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(4, -(-o // 128), -(-i // 128), device="cuda")
        x8, xs = torch.zeros(n + 20, i, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(-(-i // 128), n + 20, device="cuda")
        y = torch.zeros(n + 20, o, dtype=torch.bfloat16, device="cuda")
        r.quantize_weights_device(abi.TYPE_BF16, 4, o, i, w, i, w8, i, ws)
        r.quantize_rows_device(abi.TYPE_BF16, n + 20, i, h, i, x8, i, xs, n_rows_used=off[4:])
        r.grouped_matmul_fp8_device(abi.make_grouped(4, n + 20, i, o, abi.TYPE_E4M3, abi.TYPE_BF16, abi.ACT_RELU), off, x8, xs, w8, ws, y)
        exact = torch.cat([exact[off[g]:off[g + 1]] @ w[g].double().t() for g in range(4)]).relu()
        h = y
    torch.cuda.synchronize()
    # each 8-bit rounding is at most 2^-4 of a value, of random sign: four of them, root mean square 2^-4 / sqrt(3) each
    assert float((h[:n].double() - exact).norm()) <= 4 * 2.0 ** -4 / 3 ** 0.5 * float(exact.norm())
    assert bool((h[n:] == 0).all())
    r.check_errors()


def test_other_current_device_and_wide_limits(r):
    """Refusals reach the caller as the library's errors."""
    c = Case([10], 64, 64, "f16", 1)
    for bad in (dict(n_groups=4097), dict(n_in=0), dict(activation=abi.ACT_LOGISTIC), dict(out_type=abi.TYPE_BF16)):
        p = c.layer(abi.TYPE_F16)
        for k, v in bad.items():
            setattr(p, k, v)
        with pytest.raises(abi.SrfError) as e:
            r.grouped_matmul_device(p, c.offsets, c.x, c.w, torch.zeros(10, 64, dtype=torch.float16, device="cuda"))
        assert e.value.status == abi.ERR_ARG

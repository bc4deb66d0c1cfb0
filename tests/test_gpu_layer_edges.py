"""Edges of the layer operators beside those of test_gpu_layers.py, whose bounds and cases these tests use."""
import ctypes as C

import numpy as np
import pytest

from sphericalrf_b200 import abi
from helpers import make_renderer, small_scene
from test_gpu_layers import POISON, TYPES, Case, Case8, Chain, check_rows, e4m3_reference, r, scale_reference, table, up  # noqa: F401  (r is the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def exponents(shape, low, high, seed):
    """Scales of random mantissa between 2^low and 2^high."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.exp2(low + (high - low) * torch.rand(*shape, generator=gen, device="cuda", dtype=torch.float64)).float()


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("scales", ["small", "smaller", "subnormal", "large", "mixed", "zero"])
@pytest.mark.parametrize("sizes,n_in,n_out", [([129, 127, 0, 1], 64, 64), ([300, 17, 64], 300, 500), ([9000, 30000], 700, 264)])
def test_scales_whose_product_is_no_normal_number(r, sizes, n_in, n_out, scales, out):  # noqa: F811
    """Two scales may be far from 1 where the results are ordinary numbers.  Their product may not be rounded to fewer bits,
    vanish or become infinite on the way.  The bound is the one of every 8-bit layer: a block's sum meets two roundings, be
    it by the product of the scales or by one after the other."""
    c = Case8(sizes, n_in, n_out, 400, 2, 3)
    a, b = c.base.used
    big_x = (c.base.x[a:b].float() * 100).clamp(max=448).to(torch.float8_e4m3fn)
    big_w = (c.base.w.float().abs() * n_in ** 0.5 * 100).clamp(max=448).to(torch.float8_e4m3fn)
    xs, ws = c.xs[:, a:b].shape, c.ws.shape
    if scales == "large":
        # sums of at most 128 x 2^-8 x 2^-9 against a product of 2^128 to 2^132
        c.x[a:b] = (2.0 ** -8 * (c.base.x[a:b].float() > 0.5).float()).to(torch.float8_e4m3fn)
        c.w[:] = (2.0 ** -9 * c.base.w.float().sign()).to(torch.float8_e4m3fn)
        c.xs[:, a:b], c.ws = exponents(xs, 116, 118, 1), exponents(ws, 12, 14, 2)
    elif scales == "zero":
        # a block of zeros whose scales' product is infinite: its term is 0
        c.x[a:b, :128] = 0
        c.xs[0, a:b], c.ws[:, :, 0] = 2.0 ** 118, 2.0 ** 118
    else:
        c.x[a:b], c.w[:] = big_x, big_w
        low_x, low_w = {"small": (-126, -14), "smaller": (-82, -62), "subnormal": (-145, 8), "mixed": (-126, -14)}[scales]
        c.xs[:, a:b], c.ws = exponents(xs, low_x, low_x + 4, 1), exponents(ws, low_w, low_w + 4, 2)
        if scales == "mixed":
            c.xs[:, a:b:2] = exponents(c.xs[:, a:b:2].shape, -4, 0, 3)
    out_id, dt = TYPES[out]
    yb, y = table(c.base.n_rows, n_out, dt, 8, POISON)
    p = abi.make_grouped(len(sizes), c.base.n_rows, n_in, n_out, abi.TYPE_E4M3, out_id, abi.ACT_NONE, c.xb.stride(0), c.wb.stride(1), yb.stride(0), c.wb.stride(0))
    r.grouped_matmul_fp8_device(p, c.base.offsets, c.x, c.xs, c.w, c.ws, y)
    torch.cuda.synchronize()
    exact, terms = c.exact()
    assert bool((exact.abs() < 2.0 ** 127).all())
    blocks = up(n_in, 128) // 128
    check_rows(y, exact, terms, n_in + 2 * blocks + 2, c.base.used, scales, yb, n_out)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_scales_that_are_not_finite_stay_in_their_rows(r, bad):  # noqa: F811
    c = Case8([100], 256, 96, 401)
    c.x[:] = 1.0
    c.w[:] = 1.0
    c.xs[1, 40] = bad
    y = torch.full((100, 96), POISON, device="cuda")
    r.grouped_matmul_fp8_device(abi.make_grouped(1, 100, 256, 96, abi.TYPE_E4M3, abi.TYPE_F32), None, c.x, c.xs, c.w, c.ws, y)
    torch.cuda.synchronize()
    assert not bool(y[40].isfinite().any())
    rest = torch.arange(100, device="cuda") != 40
    exact, terms = c.exact()
    assert bool(((y.double() - exact).abs() <= 1.001 * 262 * 2.0 ** -23 * terms)[rest].all())


def test_frames_do_not_fail_for_a_layer_call(built_lib):
    """Bad offsets of a layer call are the layer's error: frames in between render, srf_check_errors reports them once."""
    sc = small_scene()
    ren = make_renderer(sc)
    post = abi.default_post()
    want = ren.render(sc["view"], post)
    c = Case([30, 30, 40], 64, 64, "f16", 9)
    y = torch.zeros(c.n_rows, 64, dtype=torch.float16, device="cuda")
    ren.grouped_matmul_device(c.layer(abi.TYPE_F16), torch.tensor([0, 50, 40, 100], device="cuda"), c.x, c.w, y)
    torch.cuda.synchronize()
    assert (ren.render(sc["view"], post) == want).all()
    frame = ren.render_frame(sc["view"], post, want_stats=True)
    assert frame["stats"]["error_flags"] == 0
    ren.dump_samples(sc["view"], 0, 10, 1 << 20)
    with pytest.raises(abi.SrfError, match="offsets") as e:
        ren.check_errors()
    assert e.value.status == abi.ERR_ARG
    ren.check_errors()
    ren.close()


def test_calls_without_a_stream_run_on_the_current_one(r):  # noqa: F811
    """Behind torch's work on a stream of its own, and captured with it."""
    c = Chain(r, [500, 20, 0, 4000], 1)
    c.step()
    want = c.results()
    c.clear()
    torch.cuda.synchronize()
    s, x = torch.cuda.Stream(), c.h[0].clone()
    c.h[0].zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)          # the samples arrive late
        c.h[0].copy_(x)
        c.step()
        got = [t.clone() for t in c.h[1:] + c.d[:3] + c.dw]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    c.clear()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.step()
    assert all(bool((t == 0).all()) for t in c.results())
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(c.results(), want))


@pytest.fixture
def cudart(r):  # noqa: F811
    """The CUDA runtime that torch and the library share."""
    lib = C.CDLL("libcudart.so.12")
    lib.cudaStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    lib.cudaStreamSynchronize.argtypes = [C.c_void_p]
    lib.cudaStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    assert lib.cudaGetLastError() == 0
    yield lib
    lib.cudaGetLastError()


def test_an_older_error_of_the_thread_is_not_the_calls(r, cudart):  # noqa: F811
    """A launch that succeeds takes an older error off the thread; a call without samples launches nothing."""
    none, w = torch.zeros(0, dtype=torch.float16, device="cuda"), torch.zeros(1, 64, 64, dtype=torch.float16, device="cuda")
    layer, stream = abi.make_grouped(1, 0, 64, 64), torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    try:
        assert cudart.cudaSetDevice(4096) != 0                 # the host program's own mistake
        left = cudart.cudaPeekAtLastError()
        assert left != 0
        r.grouped_matmul_device(layer, None, none, w, none, stream)
        r.grouped_input_grad_device(layer, None, none, w, None, none, stream)
        r.quantize_rows_device(abi.TYPE_F16, 0, 64, none, 64, none, 64, none, stream=stream)
        assert cudart.cudaPeekAtLastError() == left            # still there for the host program to see
    finally:
        cudart.cudaGetLastError()


def test_a_failed_launch_leaves_no_error_behind(r, cudart):  # noqa: F811
    """A launch into a capture that a synchronisation has broken is refused by the runtime."""
    c = Case([300], 64, 48, "f16", 8)
    y = torch.full((300, 48), POISON, dtype=torch.float16, device="cuda")
    layer, s, graph = c.layer(abi.TYPE_F16), torch.cuda.Stream(), C.c_void_p()
    torch.cuda.synchronize()
    try:
        assert cudart.cudaStreamBeginCapture(s.cuda_stream, 0) == 0
        assert cudart.cudaStreamSynchronize(s.cuda_stream) != 0
        cudart.cudaGetLastError()
        with pytest.raises(abi.SrfError, match="did not launch: ") as e:
            r.grouped_matmul_device(layer, c.offsets, c.x, c.w, y, s.cuda_stream)
        assert e.value.status == abi.ERR_CUDA
        assert cudart.cudaPeekAtLastError() == 0
    finally:
        cudart.cudaStreamEndCapture(s.cuda_stream, C.byref(graph))       # reports the broken capture
        cudart.cudaGetLastError()
    r.grouped_matmul_device(layer, c.offsets, c.x, c.w, y)
    torch.cuda.synchronize()
    assert not bool((y == POISON).any())


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(64, 512), (37, 200)])
@pytest.mark.parametrize("what", ["plain", "tiny", "nan"])
def test_quantised_zeros_keep_their_sign(r, what, rows, cols, kind):  # noqa: F811
    """Whichever way a block's quotients are taken: all values ordinary, a tiny scale, a NaN beside them."""
    type_id, dt = TYPES[kind]
    gen = torch.Generator().manual_seed(rows)
    v = torch.randn(rows, cols, generator=gen)
    v[torch.rand(rows, cols, generator=gen) < 0.3] = -0.0
    v[torch.rand(rows, cols, generator=gen) < 0.3] = 0.0
    v[0, :128] = -0.0                                     # a block of negative zeros
    v = (v * (2.0 ** -110 if what == "tiny" and kind == "bf16" else 1.0)).to(dt)
    if what == "nan":
        v[::5, 3] = float("nan")
    dev = v.cuda()
    for per in (1, 128):
        q = torch.full((rows, up(cols, 16)), 0x55, dtype=torch.uint8, device="cuda")
        nb, nr = up(cols, 128) // 128, up(rows, 128) // 128
        if per == 1:
            scales = torch.zeros(nb, rows, device="cuda")
            r.quantize_rows_device(type_id, rows, cols, dev, cols, q, q.stride(0), scales)
        else:
            scales = torch.zeros(1, nr, nb, device="cuda")
            r.quantize_weights_device(type_id, 1, rows, cols, dev, cols, q, q.stride(0), scales)
        torch.cuda.synchronize()
        f, want = v.float().numpy(), np.full(q.shape, 0x55, np.uint8)
        for i in range(0, rows, per):
            for j in range(0, cols, 128):
                block = f[i:i + per, j:min(cols, j + 128)]
                want[i:i + per, j:min(cols, j + 128)] = e4m3_reference(block, scale_reference(block))
        assert np.array_equal(q.cpu().numpy(), want), f"rows {per}"


def test_8_bit_calls_see_each_other(r):  # noqa: F811
    """Samples and weights to 8 bits and the layer on them, over and over in the same buffers: without waits the bits of the
    same chain with a wait after every step.  Scales change by powers of two from turn to turn."""
    n, k, off = 3000, 256, torch.tensor([0, 1200, 1200, 3000], device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(8)
    start = torch.randn(n, k, generator=gen, device="cuda").half()
    w0 = (torch.randn(3, k, k, generator=gen, device="cuda") / 16).half()
    layer = abi.make_grouped(3, n, k, k, abi.TYPE_E4M3, abi.TYPE_F16)

    def chain(wait):
        h, w, y = start.clone(), w0.clone(), torch.zeros(n, k, dtype=torch.float16, device="cuda")
        q, qs = torch.zeros(n, k, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(k // 128, n, device="cuda")
        w8, ws = torch.zeros(3, k, k, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(3, k // 128, k // 128, device="cuda")
        seen = []
        for i in range(30):
            r.quantize_weights_device(abi.TYPE_F16, 3, k, k, w, k, w8, k, ws)
            wait()
            r.quantize_rows_device(abi.TYPE_F16, n, k, h, k, q, k, qs)
            wait()
            r.grouped_matmul_fp8_device(layer, off, q, qs, w8, ws, y)
            wait()
            seen.append(y.clone())
            h.copy_(y).clamp_(-8, 8).add_(start, alpha=2.0 ** (i % 5 - 2))
            w.copy_(w0).mul_(2.0 ** (i % 3))
            wait()
        torch.cuda.synchronize()
        return seen + [q.view(torch.uint8), qs, w8.view(torch.uint8), ws]

    for got, want in zip(chain(lambda: None), chain(torch.cuda.synchronize)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("sizes,n_in,n_out,relu", [
    ([130, 0, 37], 65536, 40, True), ([3], 16500, 1, False), ([300, 60], 9001, 300, True), ([20000, 3, 20001], 8200, 300, False)])
def test_deep_sums_are_rounded_once(r, sizes, n_in, n_out, relu):  # noqa: F811
    """fp16 results of long sums of one sign, where an accumulator that truncates falls short of the sum by as much as the
    rounding itself (4.3e-4 at 65536 products).  Sums are cut into runs of 512 like those of fp32 results: half a step of
    fp16 and (512 + runs) 2^-23 of the sum, at most 7.7e-5."""
    c = Case(sizes, n_in, n_out, "f16", 500)
    c.x[:], c.w[:] = c.x.abs(), c.w.abs()
    y = torch.full((c.n_rows, up(n_out, 8)), POISON, dtype=torch.float16, device="cuda")
    r.grouped_matmul_device(c.layer(abi.TYPE_F16, relu), c.offsets, c.x, c.w, y)
    # the same sums as an input gradient: samples of width n_out in the place of dx, gated by their own sign
    gate = torch.randn(c.n_rows, up(n_out, 8), device="cuda").half()
    wt = torch.zeros(len(sizes), n_in, up(n_out, 8), dtype=torch.float16, device="cuda")
    wt[:, :, :n_out] = c.w.transpose(1, 2)
    dx = torch.full_like(y, POISON)
    p = abi.make_grouped(len(sizes), c.n_rows, n_out, n_in, abi.TYPE_F16, ld_x=up(n_out, 8), ld_w=up(n_out, 8), ld_y=c.xb.stride(0))
    r.grouped_input_grad_device(p, c.offsets, c.x, wt, gate if relu else None, dx)
    torch.cuda.synchronize()
    for g, (a, b) in enumerate(c.spans):
        exact = c.x[a:b].double() @ c.w[g].double().t()
        bound = exact * (2.0 ** -11 + 1.001 * (512 + n_in // 512 + 1) * 2.0 ** -23)
        assert bool(((y[a:b, :n_out].double() - exact).abs() <= bound).all()), "layer"
        shut = ~(gate[a:b, :n_out] > 0) if relu else torch.zeros_like(exact, dtype=torch.bool)
        assert bool((dx[a:b, :n_out][shut] == 0).all())
        assert bool((((dx[a:b, :n_out].double() - exact).abs() <= bound) | shut).all()), "input gradient"
    assert bool((y[:, n_out:] == POISON).all()) and bool((dx[:, n_out:] == POISON).all())


def test_weight_grad_of_a_million_samples(r):  # noqa: F811
    """More tiles than workers, so that a worker owns whole sums of 2048 runs.  In the 2-norm: the runs' own error (half a step
    an instruction of 16, 32 2^-24 of a run's size) and that of adding them one by one, half a step each of a sum that grows
    with the square root of their number: sqrt(sum of k / m for k = 1 .. m) = sqrt(m / 2) half steps."""
    n, n_in, n_out, runs = 1 << 20, 2048, 4864, 2048
    gen = torch.Generator(device="cuda").manual_seed(10)
    x, dy = torch.empty(n, n_in, dtype=torch.bfloat16, device="cuda"), torch.empty(n, n_out, dtype=torch.bfloat16, device="cuda")
    for t in (x, dy):
        for i in range(0, n, 1 << 16):
            t[i:i + (1 << 16)] = torch.randn(1 << 16, t.shape[1], generator=gen, device="cuda").bfloat16()
    p = abi.make_grouped(1, n, n_in, n_out, abi.TYPE_BF16, abi.TYPE_F32)
    space = torch.empty(r.grouped_weight_grad_workspace(p), dtype=torch.uint8, device="cuda")
    dw = torch.full((1, n_out, n_in), POISON, device="cuda")
    r.grouped_weight_grad_device(p, None, dy, x, dw, space)
    torch.cuda.synchronize()
    for cols in (slice(0, 64), slice(2500, 2564), slice(n_out - 64, n_out)):
        exact = torch.zeros(64, n_in, dtype=torch.float64, device="cuda")
        for i in range(0, n, 1 << 16):
            exact += dy[i:i + (1 << 16), cols].double().t() @ x[i:i + (1 << 16)].double()
        assert float((dw[0, cols].double() - exact).norm()) <= (32 + (runs / 2) ** 0.5) * 2.0 ** -24 * float(exact.norm())


def test_8_bit_chains_captured_on_two_streams(r):  # noqa: F811
    """Quantisation and two 8-bit layers, captured once and replayed on two streams at a time, on new samples: eager bits."""
    def make(seed, counts):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        n, k = sum(counts), 256
        s = dict(n=n, k=k, off=torch.from_numpy(np.concatenate([[0], np.cumsum(counts)])).cuda(), groups=len(counts))
        s["h"] = torch.randn(n, k, generator=gen, device="cuda").bfloat16()
        s["w"] = (torch.randn(len(counts), k, k, generator=gen, device="cuda") / 16).bfloat16()
        s["q"], s["qs"] = torch.zeros(n, k, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(2, n, device="cuda")
        s["w8"], s["ws"] = torch.zeros(len(counts), k, k, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(len(counts), 2, 2, device="cuda")
        s["y"] = torch.zeros(2, n, k, dtype=torch.bfloat16, device="cuda")
        return s

    def step(s):
        layer = abi.make_grouped(s["groups"], s["n"], s["k"], s["k"], abi.TYPE_E4M3, abi.TYPE_BF16, abi.ACT_RELU)
        r.quantize_weights_device(abi.TYPE_BF16, s["groups"], s["k"], s["k"], s["w"], s["k"], s["w8"], s["k"], s["ws"])
        for x, y in ((s["h"], s["y"][0]), (s["y"][0], s["y"][1])):
            r.quantize_rows_device(abi.TYPE_BF16, s["n"], s["k"], x, s["k"], s["q"], s["k"], s["qs"], n_rows_used=s["off"][-1:])
            r.grouped_matmul_fp8_device(layer, s["off"], s["q"], s["qs"], s["w8"], s["ws"], y)

    chains, graphs = [make(1, [700, 0, 33, 5000]), make(2, [1, 128, 2000])], []
    for s in chains:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(s)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in chains]
    for turn in range(3):
        for s in chains:
            s["h"].mul_(0.5 + turn).neg_()
            s["y"].zero_()
        torch.cuda.synchronize()
        for _ in range(2):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        got = [s["y"].clone() for s in chains]
        for s, y in zip(chains, got):
            s["y"].zero_()
            step(s)
            torch.cuda.synchronize()
            assert torch.equal(s["y"], y) and bool((y != 0).any())
    r.check_errors()

"""Refusals of the layer operators (srf_grouped_matmul and its neighbours): the checks are plain host C++, compiled here
with a small driver, so no GPU and no real memory is needed.  The addresses are numbers that nothing reads."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

from sphericalrf_b200 import abi

ROOT = Path(__file__).resolve().parent.parent

DRIVER = r'''
#include <cstring>
#include "sphericalrf_b200/csrc/srf_layer_args.h"
using namespace srf;
static int say(const std::string& s, char* out) { strncpy(out, s.c_str(), 255); out[255] = 0; return s.empty(); }
#define P const void*
#define O const uint64_t*
#define F const float*
extern "C" {
size_t size_of(int what) {
    const size_t v[] = {sizeof(srf_grouped_t), offsetof(srf_grouped_t, n_rows), offsetof(srf_grouped_t, out_type), offsetof(srf_grouped_t, ld_x),
                        offsetof(srf_grouped_t, ld_y), offsetof(srf_grouped_t, group_stride)};
    return v[what];
}
int matmul(const srf_grouped_t* g, O o, P x, P w, P y, char* out) { srf_grouped_t p; return say(refuse_matmul(g, o, x, w, y, &p), out); }
int input_grad(const srf_grouped_t* g, O o, P dy, P w, P gate, P dx, char* out) { srf_grouped_t p; return say(refuse_input_grad(g, o, dy, w, gate, dx, &p), out); }
int weight_grad(const srf_grouped_t* g, O o, P dy, P x, P dw, P sp, size_t n, char* out) { srf_grouped_t p; return say(refuse_weight_grad(g, o, dy, x, dw, sp, n, &p), out); }
int fp8(const srf_grouped_t* g, O o, P x, F xs, P w, F ws, P y, char* out) { srf_grouped_t p; return say(refuse_matmul_fp8(g, o, x, xs, w, ws, y, &p), out); }
int rows(int t, uint64_t n, O u, uint32_t c, P in, uint64_t li, P q, uint64_t lo, F s, char* out) { return say(refuse_quantize_rows(t, n, u, c, in, &li, q, &lo, s), out); }
int weights(int t, uint32_t m, uint32_t n, uint32_t c, P in, uint64_t li, P q, uint64_t lo, F s, char* out) { return say(refuse_quantize_weights(t, m, n, c, in, &li, q, &lo, s), out); }
}
'''

MB = 1 << 20
X, W, Y, G8, OFF, SX, SW, SP = (0x7f0000000000 + i * 1024 * MB for i in range(8))   # 1 GB apart


@pytest.fixture(scope="module")
def drv(tmp_path_factory):
    d = tmp_path_factory.mktemp("args")
    (d / "drv.cpp").write_text(DRIVER)
    cxx = "/usr/bin/g++" if Path("/usr/bin/g++").exists() else "g++"
    r = subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", str(ROOT), str(d / "drv.cpp"), "-o", str(d / "drv.so")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = C.CDLL(str(d / "drv.so"))
    lib.size_of.restype = C.c_size_t
    v, u64, u32 = C.c_void_p, C.c_uint64, C.c_uint32
    g = C.POINTER(abi.Grouped)
    for name, types in dict(matmul=[g, v, v, v, v], input_grad=[g, v, v, v, v, v], weight_grad=[g, v, v, v, v, v, C.c_size_t],
                            fp8=[g, v, v, v, v, v, v], rows=[C.c_int, u64, v, u32, v, u64, v, u64, v],
                            weights=[C.c_int, u32, u32, u32, v, u64, v, u64, v]).items():
        getattr(lib, name).argtypes = types + [C.c_char_p]
    return lib


def ask(fn, *args):
    """The refusal's text; "" when the call may go on."""
    out = C.create_string_buffer(256)
    ok = fn(*args, out)
    assert bool(ok) == (out.value == b"")
    return out.value.decode()


def layer(**kw):
    base = dict(n_groups=4, n_rows=1000, n_in=64, n_out=32)
    fields = {k: kw.pop(k) for k in list(kw) if k in ("struct_size", "reserved")}
    base.update(kw)
    g = abi.make_grouped(**base)
    for k, v in fields.items():
        setattr(g, k, v)
    return g


def test_struct_layout(drv):
    got = [drv.size_of(i) for i in range(6)]
    f = abi.Grouped
    assert got == [C.sizeof(f), f.n_rows.offset, f.out_type.offset, f.ld_x.offset, f.ld_y.offset, f.group_stride.offset]


def test_good_calls_pass(drv):
    assert ask(drv.matmul, layer(), OFF, X, W, Y) == ""
    assert ask(drv.matmul, layer(n_groups=1), None, X, W, Y) == ""
    assert ask(drv.matmul, layer(n_rows=0), OFF, None, W, None) == ""
    assert ask(drv.matmul, layer(n_in=63, ld_x=64, ld_w=64, n_out=33, ld_y=40, out_type=abi.TYPE_F32, activation=abi.ACT_RELU), OFF, X, W, Y) == ""
    assert ask(drv.input_grad, layer(), OFF, Y, W, None, X) == ""
    assert ask(drv.input_grad, layer(), OFF, Y, W, G8, X) == ""
    assert ask(drv.weight_grad, layer(out_type=abi.TYPE_F32), OFF, Y, X, W, SP, 1 << 20) == ""
    assert ask(drv.fp8, layer(type=abi.TYPE_E4M3, out_type=abi.TYPE_BF16), OFF, X, SX, W, SW, Y) == ""
    assert ask(drv.rows, abi.TYPE_F16, 7, None, 64, X, 0, Y, 0, SX) == ""
    assert ask(drv.rows, abi.TYPE_BF16, 0, None, 64, None, 0, None, 0, None) == ""
    assert ask(drv.weights, abi.TYPE_BF16, 3, 100, 61, X, 64, Y, 64, SX) == ""


@pytest.mark.parametrize("kw,word", [
    (dict(struct_size=8), "struct_size"), (dict(reserved=1), "reserved"), (dict(n_groups=0), "n_groups"), (dict(n_groups=4097), "n_groups"),
    (dict(n_rows=1 << 31), "n_rows"), (dict(n_in=0), "n_in"), (dict(n_out=65537), "n_out"), (dict(type=abi.TYPE_F32), "type"),
    (dict(type=abi.TYPE_E4M3), "type"), (dict(type=abi.TYPE_F16, out_type=abi.TYPE_BF16), "out_type"), (dict(activation=abi.ACT_LOGISTIC), "activation"),
    (dict(ld_x=56), "d_x"), (dict(n_in=60), "16 bytes"), (dict(ld_w=68), "16 bytes"), (dict(n_out=33), "16 bytes"), (dict(ld_x=1 << 40), "strides"),
    (dict(group_stride=32 * 64 - 8), "overlap"), (dict(group_stride=32 * 64 + 4), "16 bytes"), (dict(ld_y=1 << 34), "2^40"),
])
def test_bad_descriptions(drv, kw, word):
    assert word in ask(drv.matmul, layer(**kw), OFF, X, W, Y)


@pytest.mark.parametrize("args,word", [
    ((None, X, W, Y), "d_offsets"), ((OFF + 4, X, W, Y), "d_offsets"), ((OFF, None, W, Y), "d_x"), ((OFF, X, None, Y), "d_w"), ((OFF, X, W, None), "d_y"),
    ((OFF, X + 8, W, Y), "aligned"), ((OFF, X, W + 2, Y), "aligned"), ((OFF, X, W, Y + 4), "aligned"),
    ((OFF, X, W, X), "overlaps d_x"), ((OFF, X, W, W + 16), "overlaps d_w"), ((OFF, X, W, X + 1000 * 128 - 16), "overlaps d_x"),
    ((Y + 800, X, W, Y), "overlaps d_offsets"),
])
def test_bad_arrays(drv, args, word):
    assert word in ask(drv.matmul, layer(), *args)


def test_neighbours_in_one_allocation_do_not_overlap(drv):
    assert ask(drv.matmul, layer(), OFF, X, W, X + 1000 * 128) == ""


def test_gradient_refusals(drv):
    assert "activation" in ask(drv.input_grad, layer(activation=abi.ACT_RELU), OFF, Y, W, None, X)
    assert "overlaps d_gate" in ask(drv.input_grad, layer(), OFF, Y, W, X, X)
    assert "d_gate" in ask(drv.input_grad, layer(), OFF, Y, W, G8 + 2, X)
    f32 = dict(out_type=abi.TYPE_F32)
    assert "2^26" in ask(drv.weight_grad, layer(n_rows=(1 << 26) + 1, **f32), OFF, Y, X, W, SP, 1 << 20)
    assert "too large" in ask(drv.weight_grad, layer(n_rows=1 << 22, n_in=65536, n_out=65536, **f32), OFF, Y, X, W, SP, 1 << 20)
    assert "d_workspace is NULL" in ask(drv.weight_grad, layer(**f32), OFF, Y, X, W, None, 0)
    assert "overlaps d_workspace" in ask(drv.weight_grad, layer(**f32), OFF, Y, X, W, W, 1 << 20)
    assert "d_workspace overlaps d_x" in ask(drv.weight_grad, layer(**f32), OFF, Y, X, W, X, 1 << 20)
    assert "aligned" in ask(drv.weight_grad, layer(**f32), OFF, Y, X, W, SP + 8, 1 << 20)


def test_fp8_refusals(drv):
    good = dict(type=abi.TYPE_E4M3, out_type=abi.TYPE_F16)
    assert "type must be SRF_TYPE_E4M3" in ask(drv.fp8, layer(), OFF, X, SX, W, SW, Y)
    assert "out_type" in ask(drv.fp8, layer(type=abi.TYPE_E4M3, out_type=abi.TYPE_E4M3), OFF, X, SX, W, SW, Y)
    assert "d_x_scales is NULL" in ask(drv.fp8, layer(**good), OFF, X, None, W, SW, Y)
    assert "d_w_scales" in ask(drv.fp8, layer(**good), OFF, X, SX, W, SW + 2, Y)
    assert "16 bytes" in ask(drv.fp8, layer(**good, n_in=72), OFF, X, SX, W, SW, Y)
    assert "overlaps d_x_scales" in ask(drv.fp8, layer(**good), OFF, X, Y + 64, W, SW, Y)


def test_quantize_refusals(drv):
    assert "type" in ask(drv.rows, abi.TYPE_F32, 7, None, 64, X, 0, Y, 0, SX)
    assert "n_cols" in ask(drv.rows, abi.TYPE_F16, 7, None, 0, X, 0, Y, 0, SX)
    assert "16 bytes" in ask(drv.rows, abi.TYPE_F16, 7, None, 65, X, 72, Y, 72, SX)
    assert "d_scales is NULL" in ask(drv.rows, abi.TYPE_F16, 7, None, 64, X, 0, Y, 0, None)
    assert "d_scales overlaps d_in" in ask(drv.rows, abi.TYPE_F16, 7, None, 64, X, 0, Y, 0, X + 64)
    assert "d_out overlaps d_in" in ask(drv.rows, abi.TYPE_F16, 7, None, 64, X, 0, X, 0, SX)
    assert "d_n_rows_used" in ask(drv.rows, abi.TYPE_F16, 7, OFF + 4, 64, X, 0, Y, 0, SX)
    assert "n_matrices" in ask(drv.weights, abi.TYPE_F16, 0, 7, 64, X, 0, Y, 0, SX)
    assert "n_rows" in ask(drv.weights, abi.TYPE_F16, 1, 0, 64, X, 0, Y, 0, SX)
    assert "less than its width" in ask(drv.weights, abi.TYPE_F16, 1, 7, 64, X, 32, Y, 0, SX)

"""The Python wrappers of the layer operators, above a library that only records its calls: no GPU is needed."""
import pytest

from sphericalrf_b200 import abi
from sphericalrf_b200.testbed import Renderer

torch = pytest.importorskip("torch")


class RecordingLib:
    """Stands in for the library: every call succeeds and leaves its arguments."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return abi.OK
        return call


@pytest.fixture
def rec():
    ren = Renderer(abi.default_config(), device=-1, lib=RecordingLib())      # torch's number of host memory, where the tensors lie
    ren.lib.calls.clear()
    return ren


def tensors():
    f = dict(dtype=torch.float16)
    return dict(off=torch.tensor([0, 4, 9]), x=torch.zeros(9, 64, **f), y=torch.zeros(9, 32, **f), w=torch.zeros(2, 32, 64, **f),
                gate=torch.zeros(9, 64, **f), dw=torch.zeros(2, 32, 64), space=torch.zeros(64, dtype=torch.uint8),
                x8=torch.zeros(9, 64, dtype=torch.uint8), w8=torch.zeros(2, 32, 64, dtype=torch.float8_e4m3fn), xs=torch.zeros(1, 9),
                ws=torch.zeros(2, 1, 1), used=torch.tensor([9]))


def calls(ren, change=None, **kw):
    """Every wrapper of a layer operator once, with tensors of the right sizes but for those of `change`."""
    off, x, y, w, gate, dw, space, x8, w8, xs, ws, used = {**tensors(), **(change or {})}.values()
    layer, grad = abi.make_grouped(2, 9, 64, 32), abi.make_grouped(2, 9, 64, 32, out_type=abi.TYPE_F32)
    layer8 = abi.make_grouped(2, 9, 64, 32, abi.TYPE_E4M3, abi.TYPE_F16)
    return [
        lambda: ren.grouped_matmul_device(layer, off, x, w, y, **kw),
        lambda: ren.grouped_input_grad_device(layer, off, y, w, gate, x, **kw),
        lambda: ren.grouped_weight_grad_device(grad, off, y, x, dw, space, **kw),
        lambda: ren.grouped_matmul_fp8_device(layer8, off, x8, xs, w8, ws, y, **kw),
        lambda: ren.quantize_rows_device(abi.TYPE_F16, 9, 64, x, 64, x8, 64, xs, n_rows_used=used, **kw),
        lambda: ren.quantize_weights_device(abi.TYPE_F16, 2, 32, 64, w, 64, w8, 64, ws, **kw),
    ]


def test_calls_run_on_the_current_stream(rec, monkeypatch):
    """Without a stream of their own, calls are ordered with torch's work on the tensors."""
    asked = []
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: asked.append(device) or 4321)
    for call in calls(rec):
        call()
    assert [args[-1] for _, args in rec.lib.calls] == [4321] * 6 and asked == [-1] * 6


@pytest.mark.parametrize("stream", [0, 77])
def test_a_given_stream_is_used(rec, stream):
    for call in calls(rec, stream=stream):
        call()
    assert [args[-1] for _, args in rec.lib.calls] == [stream] * 6


# which of the six calls take a tensor
USERS = dict(off=(0, 1, 2, 3), x=(0, 1, 2, 4), y=(0, 1, 2, 3), w=(0, 1, 5), gate=(1,), dw=(2,), space=(2,), x8=(3, 4), w8=(3, 5), xs=(3, 4), ws=(3, 5), used=(4,))


def refused(ren, change, name, word):
    for k, call in enumerate(calls(ren, change, stream=0)):
        before = len(ren.lib.calls)
        if k in USERS[name]:
            with pytest.raises(abi.SrfError, match=word) as e:
                call()
            assert e.value.status == abi.ERR_ARG and len(ren.lib.calls) == before
        else:
            call()
            assert len(ren.lib.calls) == before + 1


@pytest.mark.parametrize("name", [n for n in USERS if n != "space"])
def test_another_type_is_refused(rec, name):
    t = tensors()[name]
    refused(rec, {name: t.to(torch.int32)}, name, "is of type torch.int32")


@pytest.mark.parametrize("name", [n for n in USERS if n != "space"])
def test_less_memory_is_refused(rec, name):
    """One value less than the call needs; a view of a tensor that goes on behind it is not that; a repeated row is."""
    t = tensors()[name]
    refused(rec, {name: t.flatten()[:-1].clone()}, name, "has memory for")
    if t.numel() > 1 and t.dtype is not torch.float8_e4m3fn:
        refused(rec, {name: t.flatten()[:1].clone().expand(t.numel())}, name, "has memory for")
    more = torch.zeros(t.numel() + 8, dtype=torch.uint8).to(t.dtype)
    for call in calls(rec, {name: more[4:4 + t.numel()]}, stream=0):
        call()


@pytest.mark.parametrize("name", list(USERS))
def test_another_device_is_refused(name):
    ren = Renderer(abi.default_config(), device=0, lib=RecordingLib())
    other = {k: SimpleTensor(v) for k, v in tensors().items()}
    other[name] = tensors()[name]
    refused(ren, other, name, "is on cpu")


class SimpleTensor:
    """A tensor of host memory that says it is on device 0."""

    def __init__(self, t):
        self.t = t

    def __getattr__(self, what):
        return getattr(self.t, what)

    def get_device(self):
        return 0


def test_padded_rows_and_nothing_are_taken(rec):
    """Rows with gaps whose last one ends with its values; no gate, no offsets, no rows."""
    wide = torch.zeros(9, 72, dtype=torch.float16)
    layer = abi.make_grouped(1, 9, 64, 32, ld_x=72)
    w, y = torch.zeros(32, 64, dtype=torch.float16), torch.zeros(9, 32, dtype=torch.float16)
    rec.grouped_matmul_device(layer, None, wide[:, :64], w, y, stream=0)
    rec.grouped_input_grad_device(layer, None, y, w, None, wide.flatten()[:8 * 72 + 64].clone(), stream=0)
    none = torch.zeros(0, dtype=torch.float16)
    rec.grouped_matmul_device(abi.make_grouped(3, 0, 64, 64, out_type=abi.TYPE_F32), torch.zeros(4, dtype=torch.int64), none, torch.zeros(3, 64, 64, dtype=torch.float16), none, stream=0)
    assert len(rec.lib.calls) == 3
    with pytest.raises(abi.SrfError, match="x has memory for 639"):
        rec.grouped_matmul_device(layer, None, torch.zeros(639, dtype=torch.float16), w, y, stream=0)


@pytest.mark.parametrize("name", ["x", "y", "w", "gate", "dw", "x8", "w8", "ws"])
def test_transposed_views_are_refused(rec, name):
    t = tensors()[name]
    wide = torch.zeros(4, 4, t.numel(), dtype=torch.uint8).to(t.dtype)       # memory enough for every stride
    refused(rec, {name: wide[:, :, :t.numel() // 2].transpose(1, 2)}, name, "values of a row")

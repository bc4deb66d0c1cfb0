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


def calls(ren, **kw):
    """Every wrapper of a layer operator once, with tensors of the right sizes."""
    f = dict(dtype=torch.float16)
    off = torch.tensor([0, 4, 9])
    x, y, w, gate = torch.zeros(9, 64, **f), torch.zeros(9, 32, **f), torch.zeros(2, 32, 64, **f), torch.zeros(9, 64, **f)
    dw, space = torch.zeros(2, 32, 64), torch.zeros(64, dtype=torch.uint8)
    x8, w8, xs, ws = torch.zeros(9, 64, dtype=torch.uint8), torch.zeros(2, 32, 64, dtype=torch.uint8), torch.zeros(1, 9), torch.zeros(2, 1, 1)
    layer, grad = abi.make_grouped(2, 9, 64, 32), abi.make_grouped(2, 9, 64, 32, out_type=abi.TYPE_F32)
    layer8 = abi.make_grouped(2, 9, 64, 32, abi.TYPE_E4M3, abi.TYPE_F16)
    return [
        lambda: ren.grouped_matmul_device(layer, off, x, w, y, **kw),
        lambda: ren.grouped_input_grad_device(layer, off, y, w, gate, x, **kw),
        lambda: ren.grouped_weight_grad_device(grad, off, y, x, dw, space, **kw),
        lambda: ren.grouped_matmul_fp8_device(layer8, off, x8, xs, w8, ws, y, **kw),
        lambda: ren.quantize_rows_device(abi.TYPE_F16, 9, 64, x, 64, x8, 64, xs, n_rows_used=off[2:], **kw),
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

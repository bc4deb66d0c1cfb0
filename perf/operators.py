"""The library's layer operators for fields that are cut into regions, as cases to measure.

A scene too large for one network is cut into regions with a network each; the samples of a frame or of a training batch
are sorted by region, and a layer is then one matrix product per region over that region's samples.  The operators:

  product    y[r] = act(W[g] x[r]) for every sample r of group g, 16-bit values, fp32 sums
  grads      the gradients of the same layer: dx[r] = W[g]^T dy[r] (zero where the ReLU before the layer was shut) and
             dW[g] = sum over r of dy[r] x[r]^T, in fp32
  product8   the same layer on 8-bit (e4m3) samples and weights: one scale per sample and 128 inputs, one scale per
             128 x 128 block of a matrix
  quantize   16-bit samples or weights to such 8-bit values and scales

`own` is set from outside: false computes the plain form in elementary torch operations, true makes the library's calls.
"""
import functools
import math

import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126


def listed():
    return [
        # The last unfinished rays of a frame: a handful of samples for each of a few small networks.  Latency alone.
        dict(name="product_small", op="product", type="f16", out="f16", groups=8, rows=24, slack=8, n_in=64, n_out=64, relu=True, spread="even"),
        # A frame's samples through the first layer of 64 regional networks of the renderer's own widths (32 -> 64).
        dict(name="product_narrow", op="product", type="f16", out="f16", groups=64, rows=1048613, slack=4096, n_in=32, n_out=64, relu=True, spread="skewed"),
        # Few samples, many wide networks: the weights are what has to be read.
        dict(name="product_stream", op="product", type="bf16", out="bf16", groups=64, rows=160, slack=0, n_in=2048, n_out=1408, relu=False, spread="even"),
        # A training batch through a wide layer, an odd width out: the tensor cores' case.
        dict(name="product_wide", op="product", type="bf16", out="bf16", groups=16, rows=32801, slack=100, n_in=2048, n_out=2043, relu=True, spread="skewed"),
        # The gradients of a hidden layer for a small batch.
        dict(name="grads_small", op="grads", type="f16", out="f16", groups=4, rows=100, slack=28, n_in=64, n_out=64, relu=True, spread="skewed"),
        # The gradients of a hidden layer of the renderer's width over a full training batch (2^18 samples).
        dict(name="grads_narrow", op="grads", type="f16", out="f16", groups=16, rows=262144, slack=0, n_in=64, n_out=64, relu=True, spread="skewed"),
        # The gradients of a wide layer.
        dict(name="grads_wide", op="grads", type="bf16", out="bf16", groups=8, rows=16389, slack=64, n_in=2048, n_out=2048, relu=False, spread="skewed"),
        # One sample through one 8-bit layer.
        dict(name="product8_one", op="product8", out="f16", groups=1, rows=1, slack=0, n_in=1024, n_out=1024, relu=True, spread="even"),
        # Few samples for many 8-bit networks.
        dict(name="product8_few", op="product8", out="bf16", groups=32, rows=131, slack=5, n_in=2048, n_out=2048, relu=False, spread="even"),
        # A frame's batch through wide 8-bit layers.
        dict(name="product8_wide", op="product8", out="bf16", groups=8, rows=32773, slack=0, n_in=4096, n_out=2048, relu=True, spread="skewed"),
        # Weights to 8 bits after a training step.
        dict(name="quantize_weights", op="quantize", type="bf16", block=128, groups=8, rows=1024, slack=0, n_in=1000),
        # A frame's batch of activations to 8 bits.
        dict(name="quantize_rows", op="quantize", type="f16", block=1, groups=1, rows=65539, slack=61, n_in=2048),
    ]


def draw(rng):
    def log_int(low, high):
        return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    def width(low, high):
        n = log_int(low, high)
        return n if rng.random() < 0.4 else min(high, -(-n // 16) * 16)

    op = rng.choice(["product", "product", "grads", "product8", "quantize"])
    if op == "quantize":
        block = rng.choice([1, 1, 128])
        n_in, groups = width(16, 4096), 1 if block == 1 else log_int(1, 16)
        rows = log_int(1, max(1, min(131072, 134217728 // (n_in * groups))))
        return dict(op=op, type=rng.choice(["f16", "bf16"]), block=block, groups=groups, rows=rows, slack=rng.choice([0, rows // 10]) if block == 1 else 0, n_in=n_in)
    n_in, n_out = width(16, 4096), width(16, 4096)
    groups = log_int(1, max(1, min(128, 2 ** 27 // (n_in * n_out))))
    rows = log_int(1, max(1, min(1048576, int((1.3e11 if op == "grads" else 2.7e11) / (2 * n_in * n_out)), 2 ** 27 // (n_in + n_out))))
    if op == "grads":
        rows = min(rows, 2 ** 25 // (n_in + n_out))
    case = dict(op=op, groups=groups, rows=rows, slack=rng.choice([0, rows // 16, 7]), n_in=n_in, n_out=n_out, relu=rng.random() < 0.5, spread=rng.choice(["even", "skewed"]))
    if op == "product8":
        case["out"] = rng.choice(["f16", "bf16"])
    else:
        case["type"] = rng.choice(["f16", "bf16"])
        case["out"] = case["type"] if op == "grads" else rng.choice([case["type"], case["type"], "f32"])
    return case


def _empty_groups(case):
    """Groups without samples: an eighth of them where the spread is skewed, and those for which no sample is left."""
    empty = case["groups"] // 8 if case["spread"] == "skewed" else 0
    return max(empty, case["groups"] - case["rows"])


def _sizes(case, seed):
    """Samples per group: numpy int64[groups]."""
    r = np.random.RandomState(seed % (2 ** 31))
    busy = case["groups"] - _empty_groups(case)
    if case["spread"] == "even":
        n = np.full(busy, case["rows"] // busy)
        n[: case["rows"] % busy] += 1
    else:
        share = 0.1 + r.random_sample(busy) ** 2
        n = 1 + np.floor((case["rows"] - busy) * share / share.sum()).astype(np.int64)
        n[0] += case["rows"] - n.sum()
    sizes = np.zeros(case["groups"], np.int64)
    sizes[r.permutation(case["groups"])[:busy]] = n
    return sizes


def _up(n, to):
    return -(-n // to) * to


def _pad(t, to):
    """`t` with its rows `to`-aligned: a view of a buffer whose row stride is a multiple of `to` values."""
    cols = t.shape[-1]
    if cols % to == 0:
        return t.contiguous()
    buf = torch.zeros(*t.shape[:-1], _up(cols, to), dtype=t.dtype, device=t.device)
    buf[..., :cols] = t
    return buf[..., :cols]


def _blocks(t, rows, cols):
    """[..., R, C] -> [..., ceil(R / rows), rows, ceil(C / cols), cols], zeros behind the end."""
    r, c = t.shape[-2:]
    t = torch.nn.functional.pad(t, (0, _up(c, cols) - c, 0, _up(r, rows) - r))
    return t.reshape(*t.shape[:-2], _up(r, rows) // rows, rows, _up(c, cols) // cols, cols)


def _quantize(v, rows):
    """fp32 [G, R, C] -> e4m3 values [G, R, C] and fp32 scales [G, ceil(R / rows), ceil(C / 128)]."""
    b = _blocks(v, rows, 128)
    top = b.abs().amax(dim=(-3, -1), keepdim=True)
    scale = torch.where(top > 0, (top / E4M3_MAX).clamp_min(SCALE_MIN), torch.ones_like(top))
    q = (b / scale).clamp(-E4M3_MAX, E4M3_MAX)
    q = q.reshape(v.shape[0], b.shape[1] * rows, -1)[:, : v.shape[1], : v.shape[2]].to(torch.float8_e4m3fn)
    return q, scale[:, :, 0, :, 0]


@functools.lru_cache(None)
def _renderer():
    """One context, as a program keeps it."""
    from sphericalrf_b200 import abi
    from sphericalrf_b200.testbed import Renderer
    cfg = abi.default_config()
    cfg.grid_size, cfg.log2_hashmap_size = 32, 14
    return Renderer(cfg, torch.cuda.current_device())


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    s = dict(case)
    rows, n_in = case["rows"], case["n_in"]
    if case["op"] == "quantize":
        # activations spread over several binades from sample to sample
        v = normal(case["groups"], rows + case["slack"], n_in)
        v *= torch.exp2(4 * normal(case["groups"], rows + case["slack"], 1).clamp(-2.5, 2.5))
        s["v"] = _pad((v if case["block"] == 1 else v * 0.02).to(TYPES[case["type"]]), 16)
        if own:
            from sphericalrf_b200 import abi
            s["renderer"], s["type_id"] = _renderer(), getattr(abi, "TYPE_" + case["type"].upper())
            s["q"] = torch.zeros(case["groups"], rows + case["slack"], _up(n_in, 16), dtype=torch.float8_e4m3fn, device=dev)
            nb = _up(n_in, 128) // 128
            s["scale"] = torch.zeros((nb, rows + case["slack"]) if case["block"] == 1 else (case["groups"], _up(rows, 128) // 128, nb), device=dev)
            s["count"] = torch.tensor([rows], dtype=torch.int64, device=dev)
        return s
    n_out, groups, cap = case["n_out"], case["groups"], rows + case["slack"]
    sizes = _sizes(case, seed)
    starts = np.concatenate([[0], np.cumsum(sizes)])
    s["offsets"] = torch.from_numpy(starts).to(dev)
    # where the plain form puts sample r: its group, and its place in the group
    gid = np.repeat(np.arange(groups), sizes)
    s["gid"], s["place"] = torch.from_numpy(gid).to(dev), torch.from_numpy(np.arange(rows) - starts[gid]).to(dev)
    s["longest"] = int(sizes.max())
    x, w = normal(cap, n_in).relu_(), normal(groups, n_out, n_in) / math.sqrt(n_in)
    if case["op"] == "product8":
        q, scale = _quantize(x[None], 1)
        s["x"], s["x_scale"] = _pad(q[0], 16), scale[0].t().contiguous()  # scales [ceil(n_in / 128), samples]
        q, s["w_scale"] = _quantize(w, 128)
        s["w"], s["w_scale"] = _pad(q, 16), s["w_scale"].contiguous()
    else:
        s["x"], s["w"] = _pad(x.to(TYPES[case["type"]]), 8), _pad(w.to(TYPES[case["type"]]), 8)
    if case["op"] == "grads":
        s["dy"] = _pad((normal(cap, n_out) / 16).to(TYPES[case["type"]]), 8)
    if own:
        from sphericalrf_b200 import abi
        s["renderer"] = r = _renderer()
        type_id = lambda t: getattr(abi, "TYPE_" + t.upper())  # noqa: E731
        ld = dict(ld_x=s["x"].stride(0), ld_w=s["w"].stride(1), ld_y=_up(n_out, 8), group_stride=s["w"].stride(0))
        if case["op"] == "grads":
            s["grad_x"] = abi.make_grouped(groups, cap, n_in, n_out, type_id(case["type"]), type_id(case["out"]), **ld)
            s["grad_w"] = abi.make_grouped(groups, cap, n_in, n_out, type_id(case["type"]), abi.TYPE_F32, ld_x=ld["ld_x"], ld_y=ld["ld_y"], ld_w=_up(n_in, 8))
            s["dx"] = torch.zeros(cap, _up(n_in, 8), dtype=TYPES[case["out"]], device=dev)
            s["dw"] = torch.zeros(groups, n_out, _up(n_in, 8), device=dev)
            s["space"] = torch.empty(r.grouped_weight_grad_workspace(s["grad_w"]), dtype=torch.uint8, device=dev)
        else:
            act = abi.ACT_RELU if case["relu"] else abi.ACT_NONE
            kind = abi.TYPE_E4M3 if case["op"] == "product8" else type_id(case["type"])
            s["layer"] = abi.make_grouped(groups, cap, n_in, n_out, kind, type_id(case["out"]), activation=act, **ld)
            s["y"] = torch.zeros(cap, _up(n_out, 8), dtype=TYPES[case["out"]], device=dev)
    return s


def _run_own(s):
    r, rows = s["renderer"], s["rows"]
    if s["op"] == "product":
        r.grouped_matmul_device(s["layer"], s["offsets"], s["x"], s["w"], s["y"])
        return s["y"][:rows, : s["n_out"]]
    if s["op"] == "grads":
        r.grouped_input_grad_device(s["grad_x"], s["offsets"], s["dy"], s["w"], s["x"] if s["relu"] else None, s["dx"])
        r.grouped_weight_grad_device(s["grad_w"], s["offsets"], s["dy"], s["x"], s["dw"], s["space"])
        return {"dx": s["dx"][:rows, : s["n_in"]], "dw": s["dw"][:, :, : s["n_in"]]}
    if s["op"] == "product8":
        r.grouped_matmul_fp8_device(s["layer"], s["offsets"], s["x"], s["x_scale"], s["w"], s["w_scale"], s["y"])
        return s["y"][:rows, : s["n_out"]]
    v = s["v"]
    if s["block"] == 1:
        r.quantize_rows_device(s["type_id"], v.shape[1], s["n_in"], v[0], v.stride(1), s["q"], s["q"].stride(1), s["scale"], n_rows_used=s["count"])
        return {"q": s["q"][0, :rows, : s["n_in"]], "scale": s["scale"][:, :rows]}
    r.quantize_weights_device(s["type_id"], s["groups"], rows, s["n_in"], v, v.stride(1), s["q"], s["q"].stride(1), s["scale"])
    return {"q": s["q"][:, :, : s["n_in"]], "scale": s["scale"]}


def _grouped(s, v):
    """Samples [rows, C] -> one padded batch [groups, longest, C]."""
    out = torch.zeros(s["groups"], s["longest"], v.shape[1], device=v.device)
    out[s["gid"], s["place"]] = v
    return out


def _spread_scale(scale, rows, cols):
    """Weight scales [G, R / 128, C / 128] -> [G, R, C]."""
    return scale.repeat_interleave(128, 1)[:, :rows].repeat_interleave(128, 2)[:, :, :cols]


def run(state):
    if own:
        return _run_own(state)
    s, rows = state, state["rows"]
    if s["op"] == "quantize":
        v = s["v"][:, :rows].float()
        q, scale = _quantize(v, s["block"])
        if s["block"] == 1:
            return {"q": q[0], "scale": scale[0].t()}
        return {"q": q, "scale": scale}
    if s["op"] == "grads":
        dy, x, w = s["dy"][:rows].float(), s["x"][:rows].float(), s["w"].float()
        dyg = _grouped(s, dy)
        dx = torch.matmul(dyg, w)[s["gid"], s["place"]]
        if s["relu"]:
            dx = torch.where(x > 0, dx, torch.zeros_like(dx))
        dw = torch.matmul(dyg.transpose(1, 2), _grouped(s, x))
        return {"dx": dx.to(TYPES[s["out"]]), "dw": dw}
    x, w = s["x"][:rows].float(), s["w"].float()
    if s["op"] == "product8":
        x = x * s["x_scale"][:, :rows].t().repeat_interleave(128, 1)[:, : s["n_in"]]
        w = w * _spread_scale(s["w_scale"], s["n_out"], s["n_in"])
    y = torch.matmul(_grouped(s, x), w.transpose(1, 2))[s["gid"], s["place"]]
    if s["relu"]:
        y = y.clamp_min(0)
    return y.to(TYPES[s["out"]])


def work(case):
    rows, n_in = case["rows"], case["n_in"]
    if case["op"] == "quantize":
        n = case["groups"] * rows * n_in
        scales = case["groups"] * _up(n_in, 128) // 128 * (rows if case["block"] == 1 else _up(rows, 128) // 128)
        return {"bytes": 3 * n + 4 * scales, "flops": 3 * n}
    n_out, busy = case["n_out"], case["groups"] - _empty_groups(case)
    width_out = 4 if case["out"] == "f32" else 2
    if case["op"] == "product":
        return {"bytes": 2 * rows * n_in + 2 * busy * n_in * n_out + width_out * rows * n_out, "flops": 2 * rows * n_in * n_out}
    if case["op"] == "grads":
        return {"bytes": 2 * rows * (2 * n_in + n_out) + 2 * busy * n_in * n_out + 4 * case["groups"] * n_in * n_out, "flops": 4 * rows * n_in * n_out}
    scales = 4 * (rows * _up(n_in, 128) // 128 + busy * (_up(n_in, 128) // 128) * (_up(n_out, 128) // 128))
    return {"bytes": rows * n_in + busy * n_in * n_out + scales + 2 * rows * n_out, "flops": 2 * rows * n_in * n_out}


def _round_e4m3(v):
    """float64 -> the nearest e4m3 value, ties to the even one: three fraction bits, the smallest exponent -6."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact(case, seed):
    s = prepare(case, seed)
    rows, n_in = case["rows"], case["n_in"]
    if case["op"] == "quantize":
        v, per, nb = s["v"][:, :rows].double(), case["block"], _up(n_in, 128) // 128
        q = torch.empty_like(v)
        scale = v.new_ones(case["groups"], -(-rows // per), nb)
        for j in range(nb):
            part = v[:, :, 128 * j : 128 * j + 128]
            top = part.abs().amax(2)
            if per > 1:
                top = torch.stack([t.amax(1) for t in top.split(per, 1)], 1)
            scale[:, :, j] = torch.where(top > 0, (top / E4M3_MAX).clamp_min(SCALE_MIN), scale[:, :, j])
            q[:, :, 128 * j : 128 * j + 128] = _round_e4m3(part / scale[:, :, j].repeat_interleave(per, 1)[:, :rows, None])
        if per == 1:
            return {"q": q[0], "scale": scale[0].t()}
        return {"q": q, "scale": scale}
    first = s["offsets"].tolist()
    n_out = case["n_out"]
    y = torch.zeros(rows, n_in if case["op"] == "grads" else n_out, dtype=torch.float64, device=s["x"].device)
    dw = y.new_zeros(case["groups"], n_out, n_in) if case["op"] == "grads" else None
    for g in range(case["groups"]):
        a, b = first[g], first[g + 1]
        if a == b:
            continue
        x, w = s["x"][a:b].double(), s["w"][g].double()
        if case["op"] == "grads":
            dy = s["dy"][a:b].double()
            y[a:b] = dy @ w
            if case["relu"]:
                y[a:b] *= (x > 0).double()
            dw[g] = dy.t() @ x
            continue
        if case["op"] == "product8":
            for j in range(s["x_scale"].shape[0]):
                x[:, 128 * j : 128 * j + 128] *= s["x_scale"][j, a:b, None].double()
                w[:, 128 * j : 128 * j + 128] *= s["w_scale"][g, :, j].double().repeat_interleave(128)[:n_out, None]
        y[a:b] = x @ w.t()
        if case["relu"]:
            y[a:b] = torch.where(y[a:b] > 0, y[a:b], 0.0)
    return {"dx": y, "dw": dw} if case["op"] == "grads" else y

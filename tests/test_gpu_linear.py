"""The fused linear layer against its formula in 64 bits: types, activations, odd sizes, strides, streams, graphs."""

from __future__ import annotations

from pathlib import Path
import subprocess
import sys

import pytest
import torch

import helion_b200 as hb
from helion_b200 import _lib
from helion_b200.fused_linear import _ARGS
from linear_reference import GATED
from linear_reference import check

pytestmark = pytest.mark.gpu
DEV = "cuda"
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh", *GATED)


def make(m, n, k, dtype=torch.bfloat16, activation="none", bias=None, residual=False, out=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + m + 3 * n + 7 * k)

    def normal(*shape, dt, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dt)

    rows = 2 * n if activation in GATED else n
    out = out or dtype
    return dict(
        x=normal(m, k, dt=dtype), weight=normal(rows, k, dt=dtype, std=k**-0.5),
        bias=None if bias is None else normal(rows, dt=bias, std=0.5),
        residual=normal(m, n, dt=out) if residual else None, activation=activation,
    ), out


def call(a, out):
    return hb.linear(a["x"], a["weight"], a["bias"], activation=a["activation"], residual=a["residual"], out_dtype=out)


def status_ok():
    torch.cuda.synchronize()
    return _lib.load().hb200_device_status(1) == 0


# one row, a decode batch, tile edges, several tiles, both sides of every size at which another form takes over
SIZES = [
    (1, 1, 8), (1, 128, 4096), (1, 1000, 136), (2, 3, 16), (7, 5001, 72), (15, 130, 1032), (16, 64, 64), (17, 257, 520),
    (33, 127, 24), (64, 128, 2048), (65, 200, 264), (129, 96, 1032), (200, 640, 2048), (256, 256, 128), (257, 129, 136),
    (300, 1000, 1064), (513, 264, 72), (1003, 499, 520), (5, 8, 16384), (128, 8, 8192), (383, 512, 512), (640, 2048, 256),
]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("activation", ["none", "silu_and_mul"])
def test_sizes(m, n, k, activation):
    a, out = make(m, n, k, activation=activation, residual=True)
    y = call(a, out)
    assert status_ok()
    check(y, **a)


# sizes at which each form of the CTA-pair kernel runs on 148 SMs: tiles 256, 192 and 128 columns wide, K whole or split
# over two or four pairs, tiles in one wave and in several
FORMS = [(2048, 4096, 128), (640, 4096, 2040), (256, 9000, 512), (512, 4096, 4088), (768, 1536, 4096), (256, 4096, 4096),
         (640, 1024, 4096), (512, 1024, 4088), (512, 512, 4096), (300, 520, 3584), (70, 8200, 1032),
         (266, 7136, 72), (283, 14280, 72), (132, 9488, 72), (281, 10408, 72), (6315, 536, 72), (4303, 264, 3192),
         (5185, 208, 1928), (5127, 136, 1528), (4858, 128, 9952), (2061, 200, 4840), (2161, 136, 3704)]


@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("activation", ["none", "silu_and_mul"])
@pytest.mark.parametrize("m,n,k", FORMS)
def test_pair_forms(m, n, k, activation, dtype, out):
    if activation in GATED:
        n //= 2
    a, out = make(m, n, k, dtype, activation, dtype, True, out)
    y = call(a, out)
    assert status_ok()
    check(y, **a)
    assert torch.equal(call(a, out), y)  # partial sums are added in a fixed order
    # one column fewer than fits any vector or box
    weight, bias = a["weight"], a["bias"]
    if activation in GATED:
        keep = torch.cat([torch.arange(n - 1), n + torch.arange(n - 1)]).to(DEV)
        weight, bias = weight[keep], bias[keep]
    else:
        weight, bias = weight[:-1], bias[:-1]
    b = dict(a, weight=weight, bias=bias, residual=a["residual"][:, :-1])
    check(call(b, out), **b)


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(3, 77, 128), (70, 264, 640), (700, 520, 264), (266, 7136, 72)])
def test_activations_and_types(m, n, k, dtype, activation):
    for bias, residual, out in ((None, False, dtype), (dtype, True, dtype), (torch.float32, True, torch.float32)):
        a, out = make(m, n, k, dtype, activation, bias, residual, out)
        y = call(a, out)
        assert y.dtype is out and status_ok()
        check(y, **a)


@pytest.mark.parametrize("activation", ["gelu_tanh", "silu_and_mul"])
@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("m,n,k", [(9, 333, 72), (90, 131, 200), (433, 387, 328), (1537, 641, 1032), (283, 7139, 72)])
def test_odd_widths_in_every_output_type(m, n, k, dtype, out, activation):
    a, out = make(m, n, k, dtype, activation, torch.float32, True, out)
    y = call(a, out)
    assert status_ok()
    check(y, **a)
    wide = torch.full((m, n + 3), float("nan"), dtype=out, device=DEV)
    wide[:, 2 : 2 + n] = a["residual"]
    assert torch.equal(call({**a, "residual": wide[:, 2 : 2 + n]}, out), y)


@pytest.mark.parametrize("m,n", [(1, 136), (40, 136), (600, 136), (266, 7136)])
def test_strides_and_shapes(m, n):
    a, out = make(m, n, 256, bias=torch.bfloat16, residual=True)
    want = call(a, out)
    wide = torch.full((m, 256 + 72), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 8:264] = a["x"]
    assert torch.equal(call({**a, "x": wide[:, 8:264]}, out), want)  # a slice with a pitch, read in place
    wide[:, 3:259] = a["x"]
    assert torch.equal(call({**a, "x": wide[:, 3:259]}, out), want)  # rows off the 16-byte grid
    assert torch.equal(call({**a, "x": a["x"].t().contiguous().t()}, out), want)
    assert torch.equal(call({**a, "weight": a["weight"].t().contiguous().t()}, out), want)
    tall = torch.full((n + 1, 264), float("nan"), dtype=torch.bfloat16, device=DEV)
    tall[1:, :256] = a["weight"]
    assert torch.equal(call({**a, "weight": tall[1:, :256]}, out), want)
    res = torch.full((m, n + 14), float("nan"), dtype=torch.bfloat16, device=DEV)
    res[:, 5 : n + 5] = a["residual"]
    assert torch.equal(call({**a, "residual": res[:, 5 : n + 5]}, out), want)
    assert torch.equal(call({**a, "residual": a["residual"].t().contiguous().t()}, out), want)
    assert torch.equal(call({**a, "bias": torch.stack([a["bias"], a["bias"]], 1)[:, 1]}, out), want)
    one = a["residual"][:1].expand(m, -1)  # one residual row for all
    check(call({**a, "residual": one}, out), **{**a, "residual": one})
    same = a["x"][:1].expand(m, -1)  # one row of x for all
    check(call({**a, "x": same}, out), **{**a, "x": same})
    if m % 2 == 0:
        y = hb.linear(a["x"].view(2, m // 2, 256), a["weight"], a["bias"], residual=a["residual"].view(2, m // 2, n))
        assert torch.equal(y.view(m, n), want)
    assert torch.equal(hb.linear(a["x"][0], a["weight"]), hb.linear(a["x"][:1], a["weight"])[0])
    assert status_ok()


def test_empty():
    w = torch.zeros(24, 64, dtype=torch.float16, device=DEV)
    assert hb.linear(torch.zeros(0, 64, dtype=torch.float16, device=DEV), w).shape == (0, 24)
    assert hb.linear(torch.zeros(5, 0, 64, dtype=torch.float16, device=DEV), w, activation="silu_and_mul").shape == (5, 0, 12)
    assert hb.linear(torch.zeros(3, 64, dtype=torch.float16, device=DEV), w[:0]).shape == (3, 0)


@pytest.mark.parametrize("m,n", [(2, 300), (500, 300), (300, 7136)])
def test_infinities_and_nan_stay_in_their_rows_and_columns(m, n):
    a, out = make(m, n, 264)
    clean = call(a, out)
    a["x"][1, 5] = float("nan")
    a["weight"][7, 100] = float("inf")
    y = call(a, out)
    assert torch.isnan(y[1]).all()
    rows = torch.arange(m, device=DEV) != 1
    cols = torch.arange(n, device=DEV) != 7
    assert torch.equal(y[rows][:, cols], clean[rows][:, cols])
    assert not torch.isfinite(y[:, 7]).any()
    relu = call({**a, "activation": "relu"}, out)
    assert torch.isnan(relu[1]).all()


def test_rows_past_the_edges_are_not_written_and_calls_repeat():
    lib = _lib.load()
    for m, n, k in ((3, 100, 64), (270, 300, 72), (500, 300, 72), (500, 257, 72), (500, 304, 72), (270, 7500, 72),
                    (270, 7497, 72), (270, 7504, 72), (2061, 203, 4840)):
        a, _ = make(m, n, k)
        ldo = n + 20 if n % 8 else n + 24  # (row pitches on and off the 16-byte grid)
        out = torch.full((m + 2, ldo), 7.0, dtype=torch.bfloat16, device=DEV)
        for _ in range(2):
            rc = lib.hb200_linear(_ARGS.pack(a["x"].data_ptr(), a["weight"].data_ptr(), 0, 0, out[1:].data_ptr(), m, n, k, k, k, 0,
                                             ldo, 0, 0, 1, 0, 0, 0), torch.cuda.current_stream().cuda_stream)
            assert rc == 0 and status_ok()
            assert torch.equal(out[1 : m + 1, :n], call(a, torch.bfloat16))
            assert (out[0] == 7).all() and (out[-1] == 7).all() and (out[:, n:] == 7).all()
        # the residual may be the output itself
        res = torch.randn(m, ldo, device=DEV).to(torch.bfloat16)
        want = hb.linear(a["x"], a["weight"], residual=res[:, :n])
        rc = lib.hb200_linear(_ARGS.pack(a["x"].data_ptr(), a["weight"].data_ptr(), 0, res.data_ptr(), res.data_ptr(), m, n, k, k, k,
                                         ldo, ldo, 0, 0, 1, 0, 0, 0), torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and status_ok() and torch.equal(res[:, :n], want)


def test_streams_and_graphs_are_independent():
    cases = [make(m, 520, 1024, activation="gelu", residual=True, seed=s) for s, m in enumerate((1, 24, 90, 700))]
    cases += [make(2061, 200, 4840, residual=True), make(266, 7136, 264, activation="silu_and_mul")]
    want = [call(a, out) for a, out in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, (a, out) in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(call(a, out))
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for y, w in zip(got, want))
    graphs = []
    for a, out in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call(a, out)
        graphs.append((graph, y))
    for a, _ in cases:
        a["x"].mul_(2)  # a replay reads the inputs as they are then
    want = [call(a, out) for a, out in cases]
    torch.cuda.synchronize()
    for s, (graph, _) in zip(streams, graphs):  # replayed at the same time: they share nothing
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for (_, y), w in zip(graphs, want)) and status_ok()


def test_operands_written_by_the_kernel_in_front():
    """Launches overlap the tail of the kernel in front of them: x, weight, bias and residual that it wrote are seen
    whole, by this operator and by the package's other overlapping kernel behind it, eagerly and from a graph."""
    g = torch.Generator(device=DEV).manual_seed(11)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(torch.bfloat16)

    x, seed_w = normal(512, 512), normal(512, 512, std=512**-0.5)
    a8 = (torch.randn(16, 512, generator=g, device=DEV) * 0.05).to(torch.float8_e4m3fn)
    b8 = [(torch.randn(1024, 512, generator=g, device=DEV) * 0.05).to(torch.float8_e4m3fn) for _ in range(2)]
    one = torch.ones(1, device=DEV)
    buf, weight8 = torch.empty_like(x), torch.empty_like(b8[0])
    tall = normal(7136, 512, std=512**-0.5)
    tall_now = torch.empty_like(tall)
    c = torch.empty(16, 1024, dtype=torch.bfloat16, device=DEV)

    def chain(sync):
        out = []
        wait = torch.cuda.synchronize if sync else (lambda: None)
        w, r = seed_w, x
        for step in range(12):
            m = (512, 3, 96, 40)[step % 4]
            y = hb.linear(x, w, residual=r, activation="gelu_tanh")  # [512, 512]
            wait()
            z = hb.linear(y[:m], y, y[0], residual=r[:m])  # what was just written as x, weight and bias
            wait()
            buf.copy_(y)
            wait()
            u = hb.linear(z, buf, activation="silu_and_mul")  # the weight copied a moment ago
            wait()
            weight8.copy_(b8[step % 2])
            wait()
            v = hb.linear(x[:2], buf)
            wait()
            hb.scaled_mm(c, a8, weight8.t(), one, one)  # its weight was written before the linear call in front of it
            wait()
            torch.mul(tall, float(step), out=tall_now)
            wait()
            p = hb.linear(y[:300], tall_now)
            wait()
            out += [y, z, u, v, c.clone(), p]
            wait()
            w, r = (y * 0.05).to(torch.bfloat16), y
        return out

    want = chain(True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(chain(False), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(False)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and status_ok()


FIRST_CALL = """
import sys; sys.path.insert(0, {root!r})
import torch
import helion_b200 as hb
torch.manual_seed(0)
cases = []
for m, n, k in ((1, 256, 512), (100, 8192, 1024), (512, 1024, 4096), (2048, 2048, 512), (2064, 200, 4840)):
    x = torch.randn(m, k, device="cuda").to(torch.bfloat16)
    cases.append((x, (torch.randn(n, k, device="cuda") / k**0.5).to(torch.bfloat16)))
logits = torch.randn(20000, 64, device="cuda")
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    ys = [hb.linear(x, w, activation="silu") for x, w in cases]
    few, many = hb.route_experts(logits[:50], 4), hb.route_experts(logits, 4)
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(y, hb.linear(x, w, activation="silu")) for y, (x, w) in zip(ys, cases))
for got, want in ((few, hb.route_experts(logits[:50], 4)), (many, hb.route_experts(logits, 4))):
    assert all(torch.equal(a, b) for a, b in zip(got, want))
print("captured")
"""


def test_first_call_of_a_process_may_be_captured():
    code = FIRST_CALL.format(root=str(Path(__file__).resolve().parent.parent))
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_registered_operator_and_inference_only():
    a, out = make(9, 64, 128, bias=torch.bfloat16)
    want = call(a, out)
    assert torch.equal(torch.ops.helion_b200.linear(a["x"], a["weight"], a["bias"], None, "none", out), want)
    torch.library.opcheck(torch.ops.helion_b200.linear, (a["x"], a["weight"], a["bias"], None, "none", out),
                          test_utils=("test_schema", "test_faketensor"))
    w = torch.nn.Parameter(a["weight"])
    with torch.no_grad():
        assert torch.equal(hb.linear(a["x"], w, a["bias"]), want)
    with pytest.raises(RuntimeError):
        hb.linear(a["x"], w, a["bias"]).float().sum().backward()


def test_function_transforms():
    """Inside torch.func transforms tensors have no address of their own: the call goes through the registered operator."""
    a, out = make(6, 64, 128, residual=True)
    want = call(a, out)
    one_row = torch.vmap(lambda x, r: hb.linear(x, a["weight"], residual=r))(a["x"], a["residual"])
    assert torch.equal(one_row, torch.stack([hb.linear(x, a["weight"], residual=r) for x, r in zip(a["x"], a["residual"])]))
    kept = torch.func.functionalize(lambda r: hb.linear(a["x"], a["weight"], residual=r))(a["residual"])
    assert torch.equal(kept, want)
    bias = torch.randn(16, device=DEV)
    logits = torch.randn(5, 16, device=DEV)
    for got, plain in zip(torch.func.functionalize(lambda b: hb.route_experts(logits, 3, bias=b))(bias),
                          hb.route_experts(logits, 3, bias=bias)):
        assert torch.equal(got, plain)


def test_outputs_under_inference_mode():
    a, out = make(3, 40, 64)
    with torch.inference_mode():
        y = call(a, out)
        weights, experts = hb.route_experts(torch.randn(3, 16, device=DEV), 2)
    assert y.is_inference() and weights.is_inference() and experts.is_inference()
    assert y.device == a["x"].device and torch.equal(y, call(a, out))


@pytest.mark.parametrize("m,n,k", [(1, 64, 28672), (7, 19000, 4104), (70, 256, 8200), (130, 200, 4096), (200, 1024, 16384),
                                   (256, 19200, 2048), (520, 2304, 4616), (1100, 4999, 1032)])
@pytest.mark.parametrize("activation", ["none", "silu_and_mul"])
def test_long_sums_in_fp32_outputs_do_not_drift(m, n, k, activation):
    """Products of one sign: every truncated addition errs towards zero, so a sum over all of K in one chain would be
    off by up to K / 16 steps of 2^-24, more than the bound for chains of at most 640 elements allows from K = 4096 on."""
    a, _ = make(m, n, k, activation=activation)
    a["x"], a["weight"] = a["x"].abs() + 0.125, a["weight"].abs()
    y = call(a, torch.float32)
    check(y, **a)
    assert torch.equal(y, call(a, torch.float32)) and status_ok()

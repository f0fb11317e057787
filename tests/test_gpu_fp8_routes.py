"""Which kernels the e4m3 operators launch, and each of those kernels against 64 bits.

The kernels are chosen by shape, alignment and the number of SMs; here the shapes are derived from the SM count and the
kernels that ran are read from a trace of the device, so that a changed rule cannot leave a kernel untested unseen.
Tolerances are those of test_gpu_fp8.py, which counts the roundings.
"""

from __future__ import annotations

import pathlib
import re
import subprocess
import sys

import pytest
import torch
from torch.autograd import DeviceType
from torch.profiler import ProfilerActivity, profile

from oracle import fp8_oracle as F8
from test_gpu_fp8 import BF16, FP8, U, _check_norm, _close, _gen, _operands, _pitched, _placed, _rows, _scratch, _untouched

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from lczero_triton_b200 import build, ops as module

    build.build()
    with profile(activities=[ProfilerActivity.CUDA], acc_events=True):  # the first trace of a process sets itself up
        torch.zeros(1, device="cuda")
        torch.cuda.synchronize()
    return module


@pytest.fixture(autouse=True)
def _no_device_timeouts():
    yield
    from lczero_triton_b200 import _lib

    status, detail = _lib.device_status()
    assert status == 0, f"a kernel's bounded wait ran out: {detail}"


def _kernels(call) -> list[str]:
    """The library's kernels that a call launches, in order, without their argument lists."""
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA], acc_events=True) as trace:
        call()
        torch.cuda.synchronize()
    events = sorted((e for e in trace.events() if e.device_type == DeviceType.CUDA), key=lambda e: e.time_range.start)
    names = (re.search(r"lc0b200::(?:\(anonymous namespace\)::)?([a-z0-9_]+(?:<[^>]*>)?)", e.name) for e in events)
    return [name.group(1) for name in names if name]


# ------------------------------------------------------------------ the product, kernel by kernel
#
# The rule: the 256 x 256 pair tile where it gives three fifths of the SMs a CTA, else the 128 x 128 tile where that does;
# both for more than 64 rows.  Then 64-, 32- and 16-token tiles, the widest of which there are two fifths of the SMs.

ROUTES = {"few16": "gemm_fp8_few_kernel<16, false>", "few32": "gemm_fp8_few_kernel<32, false>",
          "few64": "gemm_fp8_few_kernel<64, false>", "few64 of many rows": "gemm_fp8_few_kernel<64, false>",
          "tile128": "gemm_fp8_kernel<128, 1, {}>", "tile128, several a CTA": "gemm_fp8_kernel<128, 1, {}>",
          "pair": "gemm_fp8_kernel<256, 2, {}>", "pair, several a pair": "gemm_fp8_kernel<256, 2, {}>"}
ACTIVATION = {"none": 0, "mish": 1, "relu": 2, "swish": 3}


def _shape(route: str, ragged: int) -> tuple[int, int]:
    """Rows and columns that take the route, with `ragged` columns (at most 128; of the pair tile 256) in the last tile."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    enough, some = sms * 3 // 5, sms * 2 // 5
    if route == "few16":
        return 3, 256 + ragged
    if route == "few32":
        return 48, 128 * (-(-some // 2) - 1) + ragged  # two token tiles a weight tile
    if route == "few64":
        return 61, 128 * (some - 1) + ragged
    if route == "few64 of many rows":
        return 100, 128 * (-(-some // 2) - 1) + ragged
    if route == "tile128":
        return 1000, 128 * (-(-enough // 8) - 1) + ragged  # eight tiles of rows, four of the pair's
    if route == "tile128, several a CTA":
        return 1000, 128 * (sms // 8) + ragged  # more tiles than SMs, and still too few for pairs
    if route == "pair":
        return 3000, 256 * (-(-enough // 24) - 1) + ragged  # twelve pair tiles of rows, two CTAs each
    return 3000, 256 * (sms // 24) + ragged


def _product(ops, route: str, out, a, a_scale, w, w_scale, **more) -> None:
    ran = _kernels(lambda: ops.gemm_fp8(out, a, a_scale, w, w_scale, **more))
    assert ran == [ROUTES[route].format(ACTIVATION[more.get("activation", "none")])]


@pytest.mark.parametrize("activation", ["none", "mish", "relu", "swish"])
@pytest.mark.parametrize("route", ROUTES)
def test_product_activations(ops, route, activation) -> None:
    for ragged, k in ((72, 384), (127, 300)):
        m, n = _shape(route, ragged)
        a, a_scale, w, w_scale = _operands(80, m, n, k)
        up = -(-k // 16) * 16
        a, w = _placed(a, up), _placed(w, up)
        bias = (4 * torch.randn(n, generator=_gen(81))).to(BF16).cuda()
        want, size = F8.gemm(a, a_scale, w, w_scale, bias, activation)
        for dtype in (BF16, torch.float32):
            out = _pitched(m, n, dtype, n + (-n % 8))
            _product(ops, route, out, a, a_scale, w, w_scale, bias=bias, activation=activation)
            _close(out, want, size, k, activation)
            _untouched(out)


@pytest.mark.parametrize("activation", ["mish", "relu", "swish"])
@pytest.mark.parametrize("route", ROUTES)
def test_product_activation_range(ops, route, activation) -> None:
    """Neighbouring columns that are all small, all large or infinite: codes of zero, so that the sum is the bias."""
    (m, n), k = _shape(route, 104), 128
    a, w = (torch.zeros((rows, k), device="cuda").to(FP8) for rows in (m, n))
    a_scale, w_scale = torch.ones((1, m), device="cuda"), torch.ones((-(-n // 128), 1), device="cuda")
    bias = torch.linspace(-60.0, 60.0, n).to(BF16)
    bias[-8:] = torch.tensor([1e4, 1e10, 1e19, 1e30, 3e38, 1e5, 80.0, float("inf")]).to(BF16)
    bias = bias.cuda()
    want = F8.activate(bias.double(), activation)[:-1]
    for dtype in (BF16, torch.float32):
        out = torch.empty((m, n), dtype=dtype, device="cuda")
        _product(ops, route, out, a, a_scale, w, w_scale, bias=bias, activation=activation)
        assert bool((out[:, -1] == float("inf")).all())
        error = (out[:, :-1].double() - want).abs()
        allowed = want.abs() * ((2.0 ** -8 if dtype is BF16 else U) + 1e-5)
        assert bool((error <= allowed).all()), float((error - allowed).max())


@pytest.mark.parametrize("route", ROUTES)
def test_product_nan_stays_in_its_row_and_column(ops, route) -> None:
    (m, n), k = _shape(route, 100), 640
    a, a_scale, w, w_scale = _operands(82, m, n, k)
    clean, out = torch.empty((m, n), device="cuda"), torch.empty((m, n), device="cuda")
    ops.gemm_fp8(clean, a, a_scale, w, w_scale)
    column = n - 2
    a.view(torch.uint8)[1, 300] = 0x7F
    a_scale[4, m - 1] = float("inf")
    w.view(torch.uint8)[column, 5] = 0xFF
    _product(ops, route, out, a, a_scale, w, w_scale)
    assert bool(torch.isnan(out[1]).all()) and bool(torch.isnan(out[:, column]).all())
    assert not bool(torch.isfinite(out[m - 1]).any())
    rows = [i for i in range(m) if i not in (1, m - 1)]
    columns = [j for j in range(n) if j != column]
    assert torch.equal(out[rows][:, columns], clean[rows][:, columns])


@pytest.mark.parametrize("activation", ["mish", "relu", "swish"])
@pytest.mark.parametrize("route", ROUTES)
def test_product_nan_passes_the_activation(ops, route, activation) -> None:
    (m, n), k = _shape(route, 64), 256
    a, a_scale, w, w_scale = _operands(83, m, n, k)
    for dtype in (BF16, torch.float32):
        clean, out = torch.empty((m, n), dtype=dtype, device="cuda"), torch.empty((m, n), dtype=dtype, device="cuda")
        ops.gemm_fp8(clean, a, a_scale, w, w_scale, activation=activation)
        kept = a.view(torch.uint8)[1, 7].clone()
        a.view(torch.uint8)[1, 7] = 0x7F
        _product(ops, route, out, a, a_scale, w, w_scale, activation=activation)
        a.view(torch.uint8)[1, 7] = kept
        assert bool(torch.isnan(out[1]).all())
        assert torch.equal(out[0], clean[0]) and torch.equal(out[2:], clean[2:])


@pytest.mark.parametrize("k", [1, 16, 31, 100, 128, 129, 300, 1152])
@pytest.mark.parametrize("route", ROUTES)
def test_product_inner(ops, route, k) -> None:
    m, n = _shape(route, 40)
    a, a_scale, w, w_scale = _operands(84 + k, m, n, k)
    want, size = F8.gemm(a, a_scale, w, w_scale)
    up = -(-k // 16) * 16
    for pitch, offset in ((up, 0), (up + 48, 16)):
        for dtype in (BF16, torch.float32):
            out = _pitched(m, n, dtype)
            _product(ops, route, out, _placed(a, pitch, offset), a_scale, _placed(w, pitch, offset), w_scale)
            _close(out, want, size, k)
            _untouched(out)


@pytest.mark.parametrize("route, ragged", [(route, ragged) for route in ROUTES
                                           for ragged in (1, 8, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 192, 255, 256)
                                           if ragged <= 128 or route.startswith("pair")])
def test_product_columns(ops, route, ragged) -> None:
    (m, n), k = _shape(route, ragged), 256
    a, a_scale, w, w_scale = _operands(85, m, n, k)
    bias = torch.randn(n, generator=_gen(86)).to(BF16).cuda()
    want, size = F8.gemm(a, a_scale, w, w_scale, bias)
    for dtype, pitch in ((BF16, n), (BF16, -(-n // 8) * 8 + 8), (torch.float32, n + 1)):
        out = _pitched(m, n, dtype, pitch)
        _product(ops, route, out, a, a_scale, w, w_scale, bias=bias)
        _close(out, want, size, k)
        _untouched(out)


@pytest.mark.parametrize("route", ROUTES)
def test_product_scales(ops, route) -> None:
    """Scales far from one, whose products with codes would overflow, in rows and columns of a larger batch's arrays."""
    (m, n), k = _shape(route, 56), 512
    a, a_scale, w, w_scale = _operands(87, m, n, k)
    wide = _pitched(4, m, torch.float32, m + 37, 5)
    wide.copy_(a_scale * 2.0 ** 126)
    w_wide = _pitched(-(-n // 128), 4, torch.float32, 7, 3)
    w_wide.copy_(w_scale * 2.0 ** -126)
    want, size = F8.gemm(a, wide, w, w_wide)
    out = torch.full((m, 2 * n), 7.0, device="cuda")
    _product(ops, route, out[:, n:], a, wide, w, w_wide)
    _close(out[:, n:], want, size, k)
    assert bool((out[:, :n] == 7).all())


@pytest.mark.parametrize("route", ROUTES)
def test_layer_over_every_kernel(ops, route) -> None:
    """The layer is its two parts, whichever kernel multiplies: the same bits."""
    for k, activation in ((384, "none"), (1000, "mish"), (200, "swish")):
        m, n = _shape(route, 88)
        x = _rows(88, m, k)
        _, _, w, w_scale = _operands(89, 1, n, k)
        w = _placed(w, -(-k // 16) * 16)
        bias = torch.randn(n, generator=_gen(90)).to(BF16).cuda()
        q, scale = _pitched(m, k, FP8, -(-k // 16) * 16), torch.empty((-(-k // 128), m), device="cuda")
        ops.quantize_fp8(q, scale, x)
        kernel = ROUTES[route].format(ACTIVATION[activation])
        want_run = ["gemm_fp8_few_kernel<16, true>"] if m <= 16 else ["quantize_fp8_rows_kernel", kernel]
        for dtype in (BF16, torch.float32):
            want, out = torch.empty((m, n), dtype=dtype, device="cuda"), _pitched(m, n, dtype)
            ops.gemm_fp8(want, q, scale, w, w_scale, bias=bias, activation=activation)
            scratch = _scratch(m, k)
            assert _kernels(lambda: ops.linear_fp8(out, x, w, w_scale, bias, *scratch, activation=activation)) == want_run
            assert torch.equal(out, want)
            _untouched(out)


@pytest.mark.parametrize("route", ROUTES)
def test_products_at_once_and_replayed(ops, route) -> None:
    """Two streams of products and layers with scratch of their own, then a captured run on new inputs: the bits of a call alone."""
    (m, n), k = _shape(route, 24), 640
    _, _, w, w_scale = _operands(91, 1, n, k)
    bias = torch.randn(n, generator=_gen(92)).to(BF16).cuda()
    inputs = [_rows(93 + i, m, k) for i in range(2)]
    states = [{"x": x.clone(), "q": torch.empty((m, k), dtype=FP8, device="cuda"), "s": torch.empty((5, m), device="cuda"),
               "out": torch.empty((m, n), dtype=BF16, device="cuda"), "layer": torch.empty((m, n), dtype=BF16, device="cuda"),
               "scratch": _scratch(m, k)} for x in inputs]

    def run(s) -> None:
        ops.quantize_fp8(s["q"], s["s"], s["x"])
        ops.gemm_fp8(s["out"], s["q"], s["s"], w, w_scale, bias=bias, activation="mish")
        ops.linear_fp8(s["layer"], s["x"], w, w_scale, bias, *s["scratch"], activation="mish")

    want = []
    for s in states:
        run(s)
        want.append(s["out"].clone())
        assert torch.equal(s["layer"], s["out"])
        s["out"].zero_()
        s["layer"].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for stream, s in zip(streams, states):
            with torch.cuda.stream(stream):
                run(s)
    torch.cuda.synchronize()
    for s, expected in zip(states, want):
        assert torch.equal(s["out"], expected) and torch.equal(s["layer"], expected)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(states[0])
    for which in (1, 0, 1):
        states[0]["x"].copy_(inputs[which])
        graph.replay()
        assert torch.equal(states[0]["out"], want[which]) and torch.equal(states[0]["layer"], want[which])


FIRST_CALLS = """
import torch
from lczero_triton_b200 import ops
bf16, fp8 = torch.bfloat16, torch.float8_e4m3fn
calls, results = [], []
for m, n, k in ((4, 256, 512), (61, 7496, 256), (1000, 1352, 256), (3000, 840, 256), (40, 100, 257)):
    x = torch.randn((m, k), device="cuda").to(bf16)
    w, gamma = torch.randn((n, k), device="cuda").to(bf16), torch.ones(k, dtype=bf16, device="cuda")
    q, s = torch.empty((m, k), dtype=fp8, device="cuda"), torch.empty((-(-k // 128), m), device="cuda")
    wq, ws = torch.empty((n, k), dtype=fp8, device="cuda"), torch.empty((-(-n // 128), -(-k // 128)), device="cuda")
    outs = [torch.empty((m, n), dtype=bf16, device="cuda") for _ in range(2)]
    scratch = torch.empty(m * -(-k // 16) * 16, dtype=fp8, device="cuda"), torch.empty(m * -(-k // 128), device="cuda")
    def call(x=x, w=w, gamma=gamma, q=q, s=s, wq=wq, ws=ws, outs=outs, scratch=scratch):
        ops.quantize_fp8(wq, ws, w, block_rows=128)
        ops.rms_norm(None, x, gamma, q_out=q, q_scale=s)
        ops.gemm_fp8(outs[0], q, s, wq, ws, activation="mish")
        ops.linear_fp8(outs[1], x, wq, ws, None, *scratch)
    calls.append(call)
    results += outs
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    for call in calls:
        call()
graph.replay()
kept = [r.clone() for r in results]
for r in results:
    r.zero_()
for call in calls:
    call()
assert all(torch.equal(r, k) for r, k in zip(results, kept))
print("captured first")
"""


def test_first_calls_of_a_process_may_be_captured(ops) -> None:
    """Nothing that a first call sets up (attributes, addresses, tensor maps) is forbidden while a stream is captured."""
    root = pathlib.Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured first" in done.stdout, done.stderr[-2000:]


# ------------------------------------------------------------------ launches that the binding counts

@pytest.mark.parametrize("m, k, extra, offset, w_extra", [
    (1, 256, 0, 0, 0), (16, 256, 0, 0, 0), (1, 256, 3, 0, 0),  # one launch; the pitch of a single row says nothing
    (16, 256, 3, 0, 0), (4, 256, 0, 1, 0), (4, 260, 4, 0, 12),  # rows that are not whole aligned words
    (16, 256, 0, 0, 5), (17, 256, 0, 0, 0)])
def test_linear_counts_its_launches(ops, m, k, extra, offset, w_extra) -> None:
    from lczero_triton_b200 import _lib

    n = 96
    x = _pitched(m, k, BF16, k + extra, offset)
    x.copy_(_rows(70, m, k))
    _, _, w, w_scale = _operands(71, 1, n, k)
    w, out, scratch = _placed(w, k + w_extra), torch.empty((m, n), dtype=BF16, device="cuda"), _scratch(m, k)
    ops.linear_fp8(out, x, w, w_scale, None, *scratch)
    before = _lib.launch_count()
    launched = _kernels(lambda: ops.linear_fp8(out, x, w, w_scale, None, *scratch))
    assert _lib.launch_count() - before == len(launched), launched


# ------------------------------------------------------------------ the CUDA-core product

@pytest.mark.parametrize("n", [64 * 65535, 64 * 65535 + 1, 64 * 70000 + 130])
def test_cuda_core_product_of_many_columns(ops, n) -> None:
    """More tiles of 64 columns than a grid has in y."""
    m, k = 3, 5
    a = torch.randint(-8, 9, (m, k), generator=_gen(72)).float().to(FP8).cuda()
    w = torch.randint(-8, 9, (n, k), generator=torch.Generator("cuda").manual_seed(73), device="cuda").float().to(FP8)
    a_scale = torch.tensor([[1.0, 0.5, 2.0]], device="cuda")
    w_scale = torch.exp2(torch.randint(-3, 4, (-(-n // 128), 1), generator=torch.Generator("cuda").manual_seed(74), device="cuda").float())
    out = _pitched(m, n, torch.float32)
    assert _kernels(lambda: ops.gemm_fp8(out, a, a_scale, w, w_scale)) == [f"gemm_fp8_simt_kernel<{str(n > 64 * 65535).lower()}>"]
    # Small whole numbers times powers of two: every step is exact.
    want = (a.float() @ w.float().t()) * a_scale.t() * w_scale.repeat_interleave(128)[:n]
    assert torch.equal(out, want)


# ------------------------------------------------------------------ RMS norm

@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("width", [64, 256, 1024, 1111, 4096, 9001, 17000])
@pytest.mark.parametrize("of_x, of_gamma, epsilon", [(-62, 0, 0.0), (-62, -40, 0.0), (-62, 60, 0.0), (-75, 0, 2.0 ** -126)])
def test_rms_norm_at_its_lower_limit(ops, rows, width, of_x, of_gamma, epsilon) -> None:
    """mean(v^2) + epsilon from 2^-126 on.  Squares below fp32's normal range are off by 2^-150 at the most, so the mean is:
    one rounding relative to 2^-126, half of one in the result.  The tolerance has it to spare (16 additions are counted for
    the trees, which have 13 at the most)."""
    x, skip = _rows(75, rows, width) * 2.0 ** of_x, _rows(76, rows, width) * 2.0 ** of_x
    gamma = ((1 + 0.2 * torch.randn(width, generator=_gen(77))) * 2.0 ** of_gamma).to(BF16).cuda()
    v = x.double() + skip.double()
    assert bool((v.square().mean(dim=1) + epsilon >= 2.0 ** -126).all())
    least = (v * gamma.double()).abs()
    assert bool(((least == 0) | (least >= 2.0 ** -126)).all())
    out, q = torch.empty((rows, width), dtype=BF16, device="cuda"), torch.empty((rows, width), dtype=FP8, device="cuda")
    scale = torch.empty((-(-width // 128), rows), device="cuda")
    ops.rms_norm(out, x, gamma, epsilon=epsilon, skip=skip, q_out=q, q_scale=scale)
    _check_norm(x, skip, gamma, epsilon, out, None, q, scale)


@pytest.mark.parametrize("width", [64, 1111, 2048, 20000])
def test_rms_norm_whose_squares_vanish(ops, width) -> None:
    """Below the limit, as documented: infinities without an epsilon, and with one the formula's tiny values."""
    x, gamma = torch.full((2, width), 2.0 ** -76, dtype=BF16, device="cuda"), torch.ones(width, dtype=BF16, device="cuda")
    out = torch.empty_like(x)
    ops.rms_norm(out, x, gamma, epsilon=0.0)
    assert bool((out == float("inf")).all())
    ops.rms_norm(out, x, gamma, epsilon=1e-6)
    _check_norm(x, None, gamma, 1e-6, out, None, None, None)


# One warp a row up to 2048 channels where there are more rows than SMs; a CTA a row for wider ones.
WORD_TIERS = [(96, "1, 16"), (256, "1, 32"), (264, "2, 32"), (512, "2, 32"), (520, "4, 32"), (1024, "4, 32"), (1032, "6, 32"), (1160, "6, 32"),
              (1408, "6, 32"), (1536, "6, 32"), (1544, "8, 32"), (1920, "8, 32"), (2048, "8, 32"), (2056, "2, 256"), (4096, "2, 256"),
              (4104, "4, 256"), (8192, "4, 256"), (8200, "8, 256"), (16384, "8, 256")]


@pytest.mark.parametrize("parts", ["out", "skip+out", "skip+residual+out", "q", "skip+residual+q", "skip+residual+out+q"])
@pytest.mark.parametrize("width, tier", WORD_TIERS)
def test_rms_norm_of_many_rows(ops, width, tier, parts) -> None:
    rows = torch.cuda.get_device_properties(0).multi_processor_count + 6
    parts = parts.split("+")
    def view(dtype):
        return _pitched(rows, width, dtype, width + 24, 8)
    x, gamma = view(BF16), (1 + 0.2 * torch.randn(width, generator=_gen(96))).to(BF16).cuda()
    x.copy_(_rows(97, rows, width))
    skip = view(BF16) if "skip" in parts else None
    if skip is not None:
        skip.copy_(_rows(98, rows, width))
    residual, out = view(BF16) if "residual" in parts else None, view(BF16) if "out" in parts else None
    q = view(FP8) if "q" in parts else None
    scale = _pitched(-(-width // 128), rows, torch.float32, rows + 3, 1) if "q" in parts else None
    ran = _kernels(lambda: ops.rms_norm(out, x, gamma, epsilon=1e-5, skip=skip, residual_out=residual, q_out=q, q_scale=scale))
    assert ran == [f"rms_norm_kernel<{tier}, {str(skip is not None).lower()}, {str(q is not None).lower()}>"]
    _check_norm(x, skip, gamma, 1e-5, out, residual, q, scale)
    for t in (x, skip, residual, out, q, scale):
        if t is not None:
            _untouched(t)


@pytest.mark.parametrize("width, tier", WORD_TIERS)
def test_rms_norm_of_many_rows_in_place(ops, width, tier) -> None:
    """The new residual over the old one, the result over the input; then the same with the two exchanged."""
    rows = torch.cuda.get_device_properties(0).multi_processor_count + 1
    gamma = (1 + 0.2 * torch.randn(width, generator=_gen(99))).to(BF16).cuda()
    for swapped in (False, True):
        x, skip = _rows(100, rows, width), _rows(101, rows, width)
        x_in, skip_in = x.clone(), skip.clone()
        out, residual = (skip, x) if swapped else (x, skip)
        q, scale = torch.empty((rows, width), dtype=FP8, device="cuda"), torch.empty((-(-width // 128), rows), device="cuda")
        ran = _kernels(lambda: ops.rms_norm(out, x, gamma, skip=skip, residual_out=residual, q_out=q, q_scale=scale))
        assert ran == [f"rms_norm_kernel<{tier}, true, true>"]
        _check_norm(x_in, skip_in, gamma, 1e-6, out, residual, q, scale)


# ------------------------------------------------------------------ refused calls

def test_refused_calls_write_nothing(ops) -> None:
    """What the refusals of the wrappers and of the library leave behind: every tensor as it was, byte for byte."""
    from lczero_triton_b200._lib import Lc0B200Error

    a, a_scale, w, w_scale = _operands(110, 8, 64, 256)
    x, out, gamma = _rows(111, 8, 256), _rows(112, 8, 64), torch.ones(256, dtype=BF16, device="cuda")
    q, scale = torch.zeros((8, 256), device="cuda").to(FP8), torch.full((2, 8), 3.0, device="cuda")
    scratch = [t.view(torch.uint8).fill_(0x5A) for t in _scratch(8, 256)]
    scratch = [scratch[0].view(FP8), scratch[1].view(torch.float32)]
    everything = [a, a_scale, w, w_scale, x, out, gamma, q, scale, *scratch]
    before = [t.contiguous().view(torch.uint8).clone() for t in everything]
    torch.cuda.synchronize()
    for call in [
            lambda: ops.gemm_fp8(out[:7], a, a_scale, w, w_scale),
            lambda: ops.gemm_fp8(out, a, a_scale[:1], w, w_scale),
            lambda: ops.gemm_fp8(out, a, a_scale, w[:, :255], w_scale),
            lambda: ops.gemm_fp8(out, a, a_scale, w, w_scale, bias=gamma),
            lambda: ops.gemm_fp8(out, x, a_scale, w, w_scale),
            lambda: ops.gemm_fp8(out, a, a_scale, w, w_scale, activation="tanh"),
            lambda: ops.gemm_fp8(out, a[:1].expand(8, 256), a_scale, w, w_scale),
            lambda: ops.linear_fp8(out, x, w, w_scale, None, scratch[0][:8 * 255], scratch[1]),
            lambda: ops.linear_fp8(out, x, w, w_scale, None, scratch[0], scratch[1][:15]),
            lambda: ops.linear_fp8(out, x, w, w_scale, None, scratch[0][1:], scratch[1]),
            lambda: ops.linear_fp8(out, x, w, w_scale, None, *scratch, activation="tanh"),
            lambda: ops.linear_fp8(out, a, w, w_scale, None, *scratch),
            lambda: ops.rms_norm(x, x, gamma[:255]),
            lambda: ops.rms_norm(x, x, gamma, residual_out=x),
            lambda: ops.rms_norm(None, x, gamma),
            lambda: ops.rms_norm(x, x, gamma, q_out=q),
            lambda: ops.rms_norm(x, x, gamma, epsilon=-1.0),
            lambda: ops.rms_norm(x, x, gamma, q_out=q, q_scale=scale.t()),
            lambda: ops.rms_norm(x, x[:1].expand(8, 256), gamma),
            lambda: ops.quantize_fp8(q, scale.t().contiguous(), x),
            lambda: ops.quantize_fp8(q, scale, x, block_rows=64),
            lambda: ops.quantize_fp8(q, scale, x[:1].expand(8, 256)),
            lambda: ops.quantize_fp8(q[:, :128], scale, x),
    ]:
        def refused(call=call) -> None:
            with pytest.raises((ValueError, KeyError, Lc0B200Error)):
                call()
        assert _kernels(refused) == []
    for t, kept in zip(everything, before):
        assert torch.equal(t.contiguous().view(torch.uint8), kept)

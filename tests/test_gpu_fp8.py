"""GPU parity of the e4m3 operators (quantisers, RMS norm, block-scaled product, dense layer) against 64-bit forms.

Tolerances count roundings.  u = 2^-24 is half a step of fp32, 2^-8 of bf16, 2^-4 of e4m3 (relative to the value; 2^-10
absolute below e4m3's normal range).
* Quantiser: codes and scales are a handful of IEEE operations and are compared bit for bit.
* RMS norm: v = x + skip is one fp32 rounding; the sum of squares of a width w is off by at most (w / 32 + 16) u
  relative (at most w / 32 terms in a row per lane, then trees), half of that after the root; division, root and the two
  products add four more.
* Product: every term of a 128-block enters an fp32 sum (at most 128 additions, each off by one step 2 u of the
  running magnitude at the most), then one product and one addition per block, one for the bias and one for the product
  of the two scales: at most (256 + 4 * blocks + 8) u times sum |a| |w| s, and the result's own rounding.  The
  activations have a slope of at most 1.1 and their fast exponentials and divisions are good to 1e-5 relative.
"""

from __future__ import annotations

import pytest
import torch

from oracle import fp8_oracle as F8

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from lczero_triton_b200 import build, ops as module

    build.build()
    return module


def _gen(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def _rows(seed: int, rows: int, width: int) -> torch.Tensor:
    gen = _gen(seed)
    return (torch.randn((rows, width), generator=gen) * torch.exp(torch.randn(width, generator=gen))).to(BF16).cuda()


def _pitched(rows: int, width: int, dtype, pitch: int | None = None, offset: int = 0, fill: int = 0x5A) -> torch.Tensor:
    """A [rows, width] view with a pitch and a start offset (elements) into a buffer filled with a byte."""
    size = torch.empty(0, dtype=dtype).element_size()
    pitch = width if pitch is None else pitch
    raw = torch.full(((offset + rows * pitch) * size + 64,), fill, dtype=torch.uint8, device="cuda")
    return raw.view(dtype)[offset:offset + rows * pitch].view(rows, pitch)[:, :width]


def _untouched(view: torch.Tensor, fill: int = 0x5A) -> None:
    """Every byte of the view's buffer outside the view still holds the fill."""
    size = view.element_size()
    raw = torch.empty(0, dtype=torch.uint8, device="cuda").set_(view.untyped_storage())
    kept = torch.ones(raw.numel(), dtype=torch.bool, device="cuda")
    inside = kept.as_strided((view.shape[0], view.shape[1] * size), (view.stride(0) * size, 1), view.storage_offset() * size)
    inside.fill_(False)
    assert bool((raw[kept] == fill).all()), "bytes outside the result were written"


def _bytes(t: torch.Tensor) -> torch.Tensor:
    return t.contiguous().view(torch.uint8)


def _same_codes(got: torch.Tensor, want: torch.Tensor) -> None:
    value = got.double().cpu()
    want = want.cpu()
    assert torch.equal(torch.isnan(value), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(value), torch.nan_to_num(want))


def _same_floats(got: torch.Tensor, want: torch.Tensor) -> None:
    got, want = got.cpu(), want.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0))


# ------------------------------------------------------------------ quantiser

QUANTIZE_SHAPES = [(1, 1), (1, 128), (3, 127), (17, 129), (64, 1024), (5, 1000), (130, 257), (33, 1536), (2, 8200),
                   (1025, 640), (16, 512), (15, 520)]


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows, width", QUANTIZE_SHAPES)
@pytest.mark.parametrize("layout", ["aligned", "pitched", "odd"])
def test_quantize(ops, rows, width, block_rows, layout) -> None:
    x = _rows(1, rows, width)
    up = -(-width // 16) * 16
    pitch_in, pitch_out, offset = {"aligned": (up, up, 0), "pitched": (up + 24, up + 40, 8), "odd": (width + 3, width + 5, 1)}[layout]
    source = _pitched(rows, width, BF16, pitch_in, offset)
    source.copy_(x)
    out = _pitched(rows, width, FP8, pitch_out, offset)
    want, want_scale = F8.quantize(x.cpu(), block_rows)
    scale = _pitched(*want_scale.shape, torch.float32, want_scale.shape[1] + 3, 1)
    ops.quantize_fp8(out, scale, source, block_rows=block_rows)
    _same_codes(out, want)
    _same_floats(scale, want_scale)
    _untouched(out)
    _untouched(scale)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_special_values(ops, block_rows) -> None:
    """Zeros of both signs, blocks below and at the threshold, the largest bf16, infinities and NaN, one block each."""
    x = _rows(2, 130, 128 * 10 + 5)
    tiny = 2.0 ** -117
    x[:, 0:128] = 0.0
    x[::2, 0:128] = -0.0
    x[:, 128:256] = x[:, 128:256].clamp(-1, 1) * (tiny * 0.99)
    x[:, 256:384] = 0.0
    x[0, 256], x[129, 300] = tiny, -tiny
    x[:, 384:512] = 2.0 ** -133  # subnormal
    x[:, 512:640] *= 2.0 ** 100
    x[7, 520] = torch.finfo(BF16).max
    x[9, 700] = float("inf")
    x[11, 800] = float("-inf")
    x[128, 900] = float("nan")
    x[12, 1284] = float("nan")  # in the short last block
    out = torch.empty(x.shape, dtype=FP8, device="cuda")
    want, want_scale = F8.quantize(x.cpu(), block_rows)
    scale = torch.empty_like(want_scale, device="cuda")
    ops.quantize_fp8(out, scale, x, block_rows=block_rows)
    _same_codes(out, want)
    _same_floats(scale, want_scale)
    values = F8.dequantize_rows(out, scale) if block_rows == 1 else F8.dequantize_tiles(out, scale)
    assert torch.isnan(values[9, 640:768]).all() and torch.isnan(values[11, 768:896]).all()  # nothing non-finite hides
    assert torch.isnan(values[128, 896:1024]).all()


def test_quantize_no_rows(ops) -> None:
    ops.quantize_fp8(torch.empty((0, 64), dtype=FP8, device="cuda"), torch.empty((1, 0), device="cuda"),
                     torch.empty((0, 64), dtype=BF16, device="cuda"))
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows, width", [(40000, 130), (100, 70000), (9000000, 8)])
def test_quantize_long_and_wide(ops, rows, width) -> None:
    x = torch.randn((rows, width), device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(BF16)
    for block_rows in (1, 128):
        out = torch.empty((rows, width), dtype=FP8, device="cuda")
        want, want_scale = F8.quantize(x, block_rows)
        scale = torch.empty_like(want_scale)
        ops.quantize_fp8(out, scale, x, block_rows=block_rows)
        assert torch.equal(out.double(), want)
        assert torch.equal(scale, want_scale)


@pytest.mark.parametrize("rows, width", [(9000000, 7), (50000, 333)])
def test_quantize_long_odd_tiles(ops, rows, width) -> None:
    """More row tiles than a grid has in y: a CTA takes several, whole ones and the last short one."""
    x = torch.randn((rows, width), device="cuda", generator=torch.Generator("cuda").manual_seed(4)).to(BF16)
    want, want_scale = F8.quantize(x, 128)
    out, scale = torch.empty((rows, width), dtype=FP8, device="cuda"), torch.empty_like(want_scale)
    ops.quantize_fp8(out, scale, x, block_rows=128)
    assert torch.equal(out.double(), want)
    assert torch.equal(scale, want_scale)


# ------------------------------------------------------------------ RMS norm

def _check_norm(x, skip, gamma, epsilon, out, residual, q, scale) -> None:
    width = x.shape[1]
    want = F8.rms_norm(x, gamma, epsilon, skip)
    relative = ((width / 32 + 16) / 2 + 6) * U
    if residual is not None:
        assert torch.equal(_bytes(residual), _bytes((x.float() + skip.float()).to(BF16)))
    if out is not None:
        error = (out.double() - want).abs()
        assert bool((error <= want.abs() * (2.0 ** -8 + 2 * relative) + 2.0 ** -134).all()), float((error / want.abs()).max())
    if q is not None:
        _, want_scale = F8.quantize(want)
        spread = scale.double().t().repeat_interleave(128, dim=1)[:, :width]
        assert bool(((scale.double() - want_scale.double()).abs() <= want_scale.double() * (relative + 4 * U)).all())
        error = (q.double() * spread - want).abs()
        allowed = want.abs() * (2.0 ** -4 + 4 * relative) + spread * 2.0 ** -10 * (1 + 8 * U)
        assert bool((error <= allowed).all()), float((error / allowed).max())


NORM_SHAPES = [(1, 64), (15, 128), (16, 96), (17, 120), (1000, 32), (200, 136), (1, 1), (3, 8), (33, 31), (7, 128), (5, 130), (3, 1000), (64, 1024), (9, 1111), (5, 1536), (3, 2048), (4, 2056),
               (1, 4096), (3, 4100), (2, 8192), (2, 16384), (2, 16392), (1, 40000)]


@pytest.mark.parametrize("rows, width", NORM_SHAPES)
@pytest.mark.parametrize("parts", ["out", "skip+out", "skip+residual+out", "q", "skip+residual+q", "skip+residual+out+q"])
def test_rms_norm(ops, rows, width, parts) -> None:
    parts = parts.split("+")
    x, gamma = _rows(4, rows, width), (1 + 0.2 * torch.randn(width, generator=_gen(5))).to(BF16).cuda()
    skip = _rows(6, rows, width) if "skip" in parts else None
    residual = _pitched(rows, width, BF16) if "residual" in parts else None
    out = _pitched(rows, width, BF16) if "out" in parts else None
    q = _pitched(rows, width, FP8) if "q" in parts else None
    scale = _pitched(-(-width // 128), rows, torch.float32) if "q" in parts else None
    assert ops.rms_norm(out, x, gamma, epsilon=1e-5, skip=skip, residual_out=residual, q_out=q, q_scale=scale) is out
    _check_norm(x, skip, gamma, 1e-5, out, residual, q, scale)
    for t in (residual, out, q, scale):
        if t is not None:
            _untouched(t)


@pytest.mark.parametrize("rows, width", [(2367, 61), (2369, 300), (4739, 255), (9471, 257), (9473, 512), (5001, 7)])
def test_rms_norm_many_narrow_rows(ops, rows, width) -> None:
    """Several rows to a CTA, the last one not full, in and out of place."""
    x, skip = _rows(17, rows, width), _rows(18, rows, width)
    gamma = torch.randn(width + 1, generator=_gen(19)).to(BF16).cuda()[1:]
    x_in, skip_in = x.clone(), skip.clone()
    out, q = _pitched(rows, width, BF16, width + 3, 1), _pitched(rows, width, FP8, width + 1)
    scale = _pitched(-(-width // 128), rows, torch.float32)
    ops.rms_norm(out, x, gamma, skip=skip, q_out=q, q_scale=scale)
    _check_norm(x, skip, gamma, 1e-6, out, None, q, scale)
    for t in (out, q, scale):
        _untouched(t)
    ops.rms_norm(x, x, gamma, skip=skip, residual_out=skip)
    _check_norm(x_in, skip_in, gamma, 1e-6, x, skip, None, None)


@pytest.mark.parametrize("width", [96, 256, 1023, 2048, 3000, 17000])
@pytest.mark.parametrize("offset, extra", [(0, 16), (8, 8), (1, 0), (2, 3)])
def test_rms_norm_pitches(ops, width, offset, extra) -> None:
    rows, up = 5, -(-width // 16) * 16
    pitch = up + extra
    def view(dtype):
        return _pitched(rows, width, dtype, pitch, offset)
    x, skip = view(BF16), view(BF16)
    x.copy_(_rows(7, rows, width)); skip.copy_(_rows(8, rows, width))
    gamma = torch.randn(width + 1, generator=_gen(9)).to(BF16).cuda()[1:]  # any alignment
    out, residual, q = view(BF16), view(BF16), view(FP8)
    scale = _pitched(-(-width // 128), rows, torch.float32, rows + 2, 1)
    ops.rms_norm(out, x, gamma, epsilon=1e-6, skip=skip, residual_out=residual, q_out=q, q_scale=scale)
    _check_norm(x, skip, gamma, 1e-6, out, residual, q, scale)
    for t in (out, residual, q, scale):
        _untouched(t)


@pytest.mark.parametrize("width", [64, 1000, 1111, 4096, 20000])
def test_rms_norm_in_place(ops, width) -> None:
    """The new residual over the old one, the result over the input: as a decoder layer calls it."""
    x, skip, gamma = _rows(10, 6, width), _rows(11, 6, width), torch.ones(width, dtype=BF16, device="cuda")
    x_in, skip_in = x.clone(), skip.clone()
    ops.rms_norm(x, x, gamma, skip=skip, residual_out=skip)
    _check_norm(x_in, skip_in, gamma, 1e-6, x, skip, None, None)


@pytest.mark.parametrize("width", [256, 1111, 4096])
def test_rms_norm_special_rows(ops, width) -> None:
    """A row of zeros, one with a NaN, one with an infinity, one whose squares overflow; neighbours unharmed."""
    x = _rows(12, 6, width)
    x[0] = 0.0
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    x[3] = 1e30
    gamma = torch.ones(width, dtype=BF16, device="cuda")
    out, q = torch.empty_like(x), torch.empty(x.shape, dtype=FP8, device="cuda")
    scale = torch.empty((-(-width // 128), 6), device="cuda")
    ops.rms_norm(out, x, gamma, epsilon=1e-6, q_out=q, q_scale=scale)
    assert bool((out[0] == 0).all()) and bool((scale[:, 0] == 1).all())
    assert bool(torch.isnan(out[1]).all()) and bool(torch.isnan(scale[:, 1]).all())
    assert bool(torch.isnan(out[2, 5])) and bool((out[2, 6:] == 0).all())
    assert bool((out[3] == 0).all())
    _check_norm(x[4:], None, gamma, 1e-6, out[4:], None, q[4:], scale[:, 4:])
    ops.rms_norm(out, x, gamma, epsilon=0.0)
    assert bool(torch.isnan(out[0]).all())  # 0 / 0


@pytest.mark.parametrize("width", [64, 256, 1024, 1111, 4096, 9001, 17000])
@pytest.mark.parametrize("of_x, of_gamma, epsilon", [(-50, -40, 0.0), (-60, 0, 1e-6), (-60, -70, 1e-6), (50, 60, 0.0), (60, -100, 1e-6)])
def test_rms_norm_far_from_one(ops, width, of_x, of_gamma, epsilon) -> None:
    """Rows and gammas of small and large powers of two (their products are fp32 numbers), blocks that count as zeros, rows
    whose sum of squares is past fp32."""
    rows = 200
    x, skip = _rows(13, rows, width) * 2.0 ** of_x, _rows(14, rows, width) * 2.0 ** of_x
    gamma = ((1 + 0.2 * torch.randn(width, generator=_gen(15))) * 2.0 ** of_gamma).to(BF16).cuda()
    for n in (3, rows):
        out, q = torch.empty((n, width), dtype=BF16, device="cuda"), torch.empty((n, width), dtype=FP8, device="cuda")
        scale = torch.empty((-(-width // 128), n), device="cuda")
        ops.rms_norm(out, x[:n], gamma, epsilon=epsilon, skip=skip[:n], q_out=q, q_scale=scale)
        squares = (x[:n].double() + skip[:n].double()).square().sum(dim=1)
        fits, lost = squares < 0.99 * 2.0 ** 128, squares > 1.01 * 2.0 ** 128
        assert of_x >= 60 or bool(fits.all())
        _check_norm(x[:n][fits], skip[:n][fits], gamma, epsilon, out[fits], None, q[fits], scale[:, fits])
        assert bool((out[lost] == 0).all()) and bool((q[lost].float() == 0).all()) and bool((scale[:, lost] == 1).all())


@pytest.mark.parametrize("width", [64, 1024, 1111, 20000])
def test_rms_norm_of_a_row_added_to_itself(ops, width) -> None:
    x, gamma = _rows(16, 5, width), torch.ones(width, dtype=BF16, device="cuda")
    before, residual = x.clone(), torch.empty_like(x)
    ops.rms_norm(x, x, gamma, skip=x, residual_out=residual)
    _check_norm(before, before, gamma, 1e-6, x, residual, None, None)


# ------------------------------------------------------------------ product

def _operands(seed: int, m: int, n: int, k: int):
    a, a_scale = F8.quantize(_rows(seed, m, k))
    w, w_scale = F8.quantize(torch.randn((n, k), generator=_gen(seed + 1)).cuda() * k ** -0.5, 128)
    return a.float().to(FP8), a_scale, w.float().to(FP8), w_scale


def _placed(t: torch.Tensor, pitch: int, offset: int = 0) -> torch.Tensor:
    view = _pitched(*t.shape, t.dtype, pitch, offset, fill=0x7E)  # 0x7E = 448: padding that is read would show
    view.view(torch.uint8).copy_(t.view(torch.uint8))
    return view


def _close(got, want, size, k: int, activation: str = "none") -> None:
    summed = (256 + 4 * -(-k // 128) + 8) * U * size
    rounding = 2.0 ** -8 if got.dtype == BF16 else U
    fast = 1e-5 if activation in ("mish", "swish") else 0.0
    allowed = 1.1 * summed + (rounding + fast) * want.abs() + 1e-30
    error = (got.double() - want).abs()
    assert bool(torch.isfinite(got.double()).all())
    assert bool((error <= allowed).all()), float((error / allowed).max())


M_SIZES = [1, 2, 7, 15, 16, 17, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300, 513]
N_SIZES = [1, 8, 16, 63, 64, 100, 127, 128, 129, 256, 257, 500]
K_SIZES = [1, 16, 31, 100, 127, 128, 129, 256, 300, 1000, 1152]


@pytest.mark.parametrize("m", M_SIZES)
@pytest.mark.parametrize("n, k", [(128, 256), (200, 1000), (257, 129), (512, 1024)])
def test_gemm_rows(ops, m, n, k) -> None:
    a, a_scale, w, w_scale = _operands(20 + m, m, n, k)
    up = -(-k // 16) * 16
    a, w = _placed(a, up), _placed(w, up)
    bias = torch.randn(n, generator=_gen(21)).to(BF16).cuda()
    want, size = F8.gemm(a, a_scale, w, w_scale, bias)
    for dtype in (BF16, torch.float32):
        out = _pitched(m, n, dtype)
        ops.gemm_fp8(out, a, a_scale, w, w_scale, bias=bias)
        _close(out, want, size, k)
        _untouched(out)


@pytest.mark.parametrize("m", [3, 64, 200])
@pytest.mark.parametrize("n", N_SIZES)
def test_gemm_columns(ops, m, n) -> None:
    k = 384
    a, a_scale, w, w_scale = _operands(22 + n, m, n, k)
    want, size = F8.gemm(a, a_scale, w, w_scale)
    for dtype, pitch in ((BF16, n), (BF16, -(-n // 8) * 8 + 8), (torch.float32, n + 1)):
        out = _pitched(m, n, dtype, pitch)
        ops.gemm_fp8(out, a, a_scale, w, w_scale)
        _close(out, want, size, k)
        _untouched(out)


@pytest.mark.parametrize("m", [5, 64, 150])
@pytest.mark.parametrize("k", K_SIZES)
def test_gemm_inner(ops, m, k) -> None:
    n = 136
    a, a_scale, w, w_scale = _operands(23 + k, m, n, k)
    want, size = F8.gemm(a, a_scale, w, w_scale)
    up = -(-k // 16) * 16
    for pitch, offset in ((up, 0), (up + 48, 16), (k, 0), (k + 5, 3)):  # the last two may be for the CUDA cores
        out = _pitched(m, n, torch.float32)
        ops.gemm_fp8(out, _placed(a, pitch, offset), a_scale, _placed(w, pitch, offset), w_scale)
        _close(out, want, size, k)
        _untouched(out)


@pytest.mark.parametrize("activation", ["none", "mish", "relu", "swish"])
@pytest.mark.parametrize("m, n, k", [(4, 300, 256), (64, 128, 640), (200, 320, 256), (700, 512, 384)])
def test_gemm_activations(ops, activation, m, n, k) -> None:
    a, a_scale, w, w_scale = _operands(24, m, n, k)
    bias = (4 * torch.randn(n, generator=_gen(25))).to(BF16).cuda()
    want, size = F8.gemm(a, a_scale, w, w_scale, bias, activation)
    for dtype in (BF16, torch.float32):
        out = torch.empty((m, n), dtype=dtype, device="cuda")
        ops.gemm_fp8(out, a, a_scale, w, w_scale, bias=bias, activation=activation)
        _close(out, want, size, k, activation)


# Few rows, the CUDA-core form (an odd pitch) and pair tiles; every other kernel is in test_gpu_fp8_routes.py.
@pytest.mark.parametrize("activation", ["mish", "relu", "swish"])
@pytest.mark.parametrize("m, pitch", [(3, 128), (70, 128), (70, 129), (4000, 128), (6000, 128)])
def test_gemm_activation_range(ops, activation, m, pitch) -> None:
    """Neighbouring columns that are all small, all large or infinite: codes of zero, so that the sum is the bias."""
    n, k = 520, 128
    a, w = (_placed(torch.zeros((rows, k), device="cuda").to(FP8), pitch) for rows in (m, n))
    a_scale, w_scale = torch.ones((1, m), device="cuda"), torch.ones((5, 1), device="cuda")
    bias = torch.linspace(-60.0, 60.0, n).to(BF16)
    bias[-8:] = torch.tensor([1e4, 1e10, 1e19, 1e30, 3e38, 1e5, 80.0, float("inf")]).to(BF16)
    bias = bias.cuda()
    want = F8.activate(bias.double(), activation)
    want[-1] = float("inf")
    for dtype in (BF16, torch.float32):
        out = torch.empty((m, n), dtype=dtype, device="cuda")
        ops.gemm_fp8(out, a, a_scale, w, w_scale, bias=bias, activation=activation)
        assert bool((out[:, -1] == float("inf")).all())
        error = (out[:, :-1].double() - want[:-1]).abs()
        allowed = want[:-1].abs() * ((2.0 ** -8 if dtype is BF16 else U) + 1e-5)
        assert bool((error <= allowed).all()), float((error - allowed).max())


@pytest.mark.parametrize("activation", ["mish", "relu", "swish"])
@pytest.mark.parametrize("m, n", [(4000, 520), (6000, 1000)])
def test_gemm_activations_of_large_tiles(ops, activation, m, n) -> None:
    test_gemm_activations(ops, activation, m, n, 384)


# Large enough for every tile shape and several tiles per CTA.
@pytest.mark.parametrize("m, n, k", [(1, 4096, 4096), (8, 8192, 2048), (16, 1024, 8192), (48, 1536, 1024), (64, 24576, 256),
                                     (96, 4096, 1024), (777, 1858, 1000), (2048, 1024, 1024), (4096, 1536, 512),
                                     (5000, 4096, 1024), (40000, 1024, 256), (20011, 1000, 384)])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_gemm_large(ops, m, n, k, dtype) -> None:
    a, a_scale, w, w_scale = _operands(26, m, n, k)
    up = -(-k // 16) * 16
    a, w = _placed(a, up), _placed(w, up)
    bias = torch.randn(n, generator=_gen(27)).to(BF16).cuda()
    want, size = F8.gemm(a, a_scale, w, w_scale, bias)
    out = _pitched(m, n, dtype)
    ops.gemm_fp8(out, a, a_scale, w, w_scale, bias=bias)
    _close(out, want, size, k)
    _untouched(out)
    again = torch.empty_like(out)
    ops.gemm_fp8(again, a, a_scale, w, w_scale, bias=bias)
    assert torch.equal(again, out)


# Several tiles per CTA pair whose finishing and first block run into one another: one block or two, ragged last columns.
@pytest.mark.parametrize("activation", ["none", "mish", "swish"])
@pytest.mark.parametrize("m, n, k", [(40000, 264, 128), (40000, 300, 100), (30011, 1000, 129), (70000, 40, 64), (20001, 1858, 256)])
def test_gemm_many_tiles(ops, m, n, k, activation) -> None:
    a, a_scale, w, w_scale = _operands(37, m, n, k)
    up = -(-k // 16) * 16
    a, w = _placed(a, up), _placed(w, up)
    bias = torch.randn(n, generator=_gen(38)).to(BF16).cuda()
    want, size = F8.gemm(a, a_scale, w, w_scale, bias, activation)
    for dtype in (BF16, torch.float32):
        out = _pitched(m, n, dtype, n + (-n % 8))
        ops.gemm_fp8(out, a, a_scale, w, w_scale, bias=bias, activation=activation)
        _close(out, want, size, k, activation)
        _untouched(out)


@pytest.mark.parametrize("m", [3, 64, 130, 600])
def test_gemm_nan_stays_in_its_row_and_column(ops, m) -> None:
    n, k = 260, 640
    a, a_scale, w, w_scale = _operands(28, m, n, k)
    clean = torch.empty((m, n), device="cuda")
    ops.gemm_fp8(clean, a, a_scale, w, w_scale)
    a.view(torch.uint8)[1, 300] = 0x7F
    a_scale[4, m - 1] = float("inf")
    w.view(torch.uint8)[258, 5] = 0xFF
    out = torch.empty((m, n), device="cuda")
    ops.gemm_fp8(out, a, a_scale, w, w_scale)
    assert bool(torch.isnan(out[1]).all()) and bool(torch.isnan(out[:, 258]).all())
    assert not bool(torch.isfinite(out[m - 1]).any())
    rows = [i for i in range(m) if i not in (1, m - 1)]
    columns = [j for j in range(n) if j != 258]
    assert torch.equal(out[rows][:, columns], clean[rows][:, columns])


@pytest.mark.parametrize("activation", ["mish", "relu", "swish"])
@pytest.mark.parametrize("m, pitch", [(3, 256), (3, 257), (70, 256), (300, 256)])
def test_gemm_nan_passes_the_activation(ops, activation, m, pitch) -> None:
    n, k = 130, 256
    a, a_scale, w, w_scale = _operands(33, m, n, k)
    clean, out = torch.empty((m, n), device="cuda"), torch.empty((m, n), device="cuda")
    ops.gemm_fp8(clean, _placed(a, pitch), a_scale, w, w_scale, activation=activation)
    a.view(torch.uint8)[1, 7] = 0x7F
    ops.gemm_fp8(out, _placed(a, pitch), a_scale, w, w_scale, activation=activation)
    assert bool(torch.isnan(out[1]).all())
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2:], clean[2:])


def test_gemm_scales_of_slices(ops) -> None:
    """Rows of a larger batch: codes, scales and results are views with the batch's pitches."""
    m, n, k = 500, 192, 512
    a, a_scale, w, w_scale = _operands(29, m, n, k)
    whole = torch.empty((m, n), device="cuda")
    ops.gemm_fp8(whole, a, a_scale, w, w_scale)
    for first, last in ((0, 1), (3, 20), (100, 333), (499, 500)):
        out = torch.full((m, 2 * n), 7.0, device="cuda")
        ops.gemm_fp8(out[first:last, n:], a[first:last], a_scale[:, first:last], w, w_scale)
        want, size = F8.gemm(a[first:last], a_scale[:, first:last], w, w_scale)
        _close(out[first:last, n:], want, size, k)
        assert bool((out[:, :n] == 7).all()) and bool((out[last:] == 7).all()) and bool((out[:first] == 7).all())


def test_gemm_extreme_scales(ops) -> None:
    """Scales far from one: their product is formed in fp32 and applied to each block's sum."""
    m, n, k = 40, 130, 256
    a, a_scale, w, w_scale = _operands(30, m, n, k)
    a_scale *= 2.0 ** 60
    w_scale *= 2.0 ** -62
    want, size = F8.gemm(a, a_scale, w, w_scale)
    for rows in (40, 5):
        out = torch.empty((rows, n), device="cuda")
        ops.gemm_fp8(out, a[:rows], a_scale[:, :rows], w, w_scale)
        _close(out, want[:rows], size[:rows], k)


@pytest.mark.parametrize("m, pitch", [(5, 256), (5, 257), (200, 257)])
def test_gemm_scales_that_only_fit_together(ops, m, pitch) -> None:
    """Scale times code overflows, the product of the two scales does not."""
    n, k = 130, 256
    a, a_scale, w, w_scale = _operands(34, m, n, k)
    a_scale *= 2.0 ** 126
    w_scale *= 2.0 ** -126
    want, size = F8.gemm(a, a_scale, w, w_scale)
    out = torch.empty((m, n), device="cuda")
    ops.gemm_fp8(out, _placed(a, pitch), a_scale, _placed(w, pitch), w_scale)
    _close(out, want, size, k)


@pytest.mark.parametrize("m, n", [(3, 300), (200, 300)])
def test_offsets_past_32_bits(ops, m, n) -> None:
    """Rows and scales a long way apart: every operand's last row begins past element 2^31."""
    k, far = 384, (2 ** 31 // (m - 1) // 64 + 1) * 64
    def apart(rows, columns, dtype, pitch):
        return torch.empty((rows - 1) * pitch + columns, dtype=dtype, device="cuda").as_strided((rows, columns), (pitch, 1))
    x = apart(m, k, BF16, far)
    x.copy_(_rows(35, m, k))
    q, scale = apart(m, k, FP8, far), apart(3, m, torch.float32, 2 ** 30 + 4)
    ops.quantize_fp8(q, scale, x)
    codes, want_scale = F8.quantize(x)
    _same_codes(q, codes)
    _same_floats(scale, want_scale)
    w = torch.randn((n, k), generator=_gen(36)).to(BF16).cuda()
    w_q, w_scale = torch.empty((n, k), dtype=FP8, device="cuda"), torch.empty((-(-n // 128), 3), device="cuda")
    ops.quantize_fp8(w_q, w_scale, w, block_rows=128)
    want, size = F8.gemm(q, scale, w_q, w_scale)
    out = apart(m, n, BF16, far)
    ops.gemm_fp8(out, q, scale, w_q, w_scale)
    _close(out, want, size, k)
    out.zero_()
    ops.linear_fp8(out, x, w_q, w_scale, None, *_scratch(m, k))
    _close(out, want, size, k)
    gamma = torch.ones(k, dtype=BF16, device="cuda")
    norm = apart(m, k, BF16, far)
    ops.rms_norm(norm, x, gamma, epsilon=1e-6, q_out=q, q_scale=scale)
    _check_norm(x, None, gamma, 1e-6, norm, None, q, scale)


def test_no_rows(ops) -> None:
    a, a_scale, w, w_scale = _operands(31, 4, 64, 128)
    ops.gemm_fp8(torch.empty((0, 64), dtype=BF16, device="cuda"), a[:0], a_scale[:, :0], w, w_scale)
    ops.linear_fp8(torch.empty((0, 64), dtype=BF16, device="cuda"), torch.empty((0, 128), dtype=BF16, device="cuda"), w,
                   w_scale, None, torch.empty(16, dtype=FP8, device="cuda"), torch.empty(4, device="cuda"))
    ops.rms_norm(torch.empty((0, 64), dtype=BF16, device="cuda"), torch.empty((0, 64), dtype=BF16, device="cuda"),
                 torch.ones(64, dtype=BF16, device="cuda"))
    torch.cuda.synchronize()


# ------------------------------------------------------------------ the layer, and all of them together

def _scratch(m: int, k: int):
    return (torch.empty(m * -(-k // 16) * 16, dtype=FP8, device="cuda"), torch.empty(m * -(-k // 128), device="cuda"))


@pytest.mark.parametrize("m, n, k", [(1, 256, 512), (3, 100, 130), (64, 384, 1000), (333, 512, 1024), (8, 64, 33)])
def test_linear(ops, m, n, k) -> None:
    """The layer is its two parts: the same bits."""
    x = _pitched(m, k, BF16, k + 5, 1)
    x.copy_(_rows(40, m, k))
    _, _, w, w_scale = _operands(41, 1, n, k)
    w = _placed(w, -(-k // 16) * 16)
    bias = torch.randn(n, generator=_gen(42)).to(BF16).cuda()
    q, scale = _pitched(m, k, FP8, -(-k // 16) * 16), torch.empty((-(-k // 128), m), device="cuda")
    ops.quantize_fp8(q, scale, x)
    for dtype in (BF16, torch.float32):
        want, out = torch.empty((m, n), dtype=dtype, device="cuda"), _pitched(m, n, dtype, n + 3)
        ops.gemm_fp8(want, q, scale, w, w_scale, bias=bias, activation="mish")
        ops.linear_fp8(out, x, w, w_scale, bias, *_scratch(m, k), activation="mish")
        assert torch.equal(out, want)
        _untouched(out)


@pytest.mark.parametrize("m", [1, 2, 7, 8, 15, 16, 17])
@pytest.mark.parametrize("n, k, extra", [(256, 512, 0), (1000, 1000, 8), (129, 136, 24), (4096, 2048, 0), (40, 8, 0)])
def test_linear_few_rows(ops, m, n, k, extra) -> None:
    """Up to 16 rows run as one launch: still the bits of its two parts, also where blocks are zeros, tiny or not finite."""
    x = _pitched(m, k, BF16, k + extra, 8 if extra else 0)
    x.copy_(_rows(43, m, k))
    x[0, : min(k, 128)] = 0.0
    if m > 2:
        x[1] *= 2.0 ** -125
        x[2, k // 2] = float("nan")
    if m > 7:
        x[5, k - 1] = float("-inf")
        x[6, :4] = torch.finfo(BF16).max
    _, _, w, w_scale = _operands(44, 1, n, k)
    w = _placed(w, -(-k // 16) * 16)
    bias = torch.randn(n, generator=_gen(45)).to(BF16).cuda()
    q, scale = _pitched(m, k, FP8, -(-k // 16) * 16), torch.empty((-(-k // 128), m), device="cuda")
    ops.quantize_fp8(q, scale, x)
    for dtype, activation in ((BF16, "none"), (torch.float32, "mish")):
        want, out = torch.empty((m, n), dtype=dtype, device="cuda"), _pitched(m, n, dtype, n + 3)
        ops.gemm_fp8(want, q, scale, w, w_scale, bias=bias, activation=activation)
        ops.linear_fp8(out, x, w, w_scale, bias, *_scratch(m, k), activation=activation)
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(out, nan=0.0), torch.nan_to_num(want, nan=0.0))
        _untouched(out)


def _block(ops, s) -> None:
    """A feed-forward block as a decoder runs it: norm of the residual straight to codes, two products, next norm."""
    ops.rms_norm(None, s["x"], s["gamma1"], skip=s["residual"], residual_out=s["residual1"], q_out=s["q"], q_scale=s["q_scale"])
    ops.gemm_fp8(s["hidden"], s["q"], s["q_scale"], s["w1"], s["w1_scale"], bias=s["b1"], activation="mish")
    ops.linear_fp8(s["branch"], s["hidden"], s["w2"], s["w2_scale"], s["b2"], *s["scratch"])
    ops.rms_norm(s["out"], s["branch"], s["gamma2"], skip=s["residual1"], residual_out=s["residual2"])


def _block_state(ops, m: int, d: int, f: int) -> dict:
    s = {"x": _rows(50, m, d), "residual": _rows(51, m, d)}
    for name, width in (("gamma1", d), ("gamma2", d), ("b1", f), ("b2", d)):
        s[name] = (1 + 0.1 * torch.randn(width, generator=_gen(len(name) + width))).to(BF16).cuda()
    for name, n, k in (("w1", f, d), ("w2", d, f)):
        w = (torch.randn((n, k), generator=_gen(n)) * k ** -0.5).to(BF16).cuda()
        s[name], s[f"{name}_scale"] = torch.empty((n, k), dtype=FP8, device="cuda"), torch.empty((-(-n // 128), -(-k // 128)), device="cuda")
        ops.quantize_fp8(s[name], s[f"{name}_scale"], w, block_rows=128)
    for name, width in (("residual1", d), ("residual2", d), ("branch", d), ("out", d), ("hidden", f)):
        s[name] = torch.empty((m, width), dtype=BF16, device="cuda")
    s["q"], s["q_scale"] = torch.empty((m, d), dtype=FP8, device="cuda"), torch.empty((-(-d // 128), m), device="cuda")
    s["scratch"] = _scratch(m, f)
    return s


RESULTS = ("residual1", "q_scale", "hidden", "branch", "residual2", "out")


@pytest.mark.parametrize("m, d, f", [(1, 256, 512), (17, 1024, 1536), (640, 768, 1024)])
def test_feed_forward_block(ops, m, d, f) -> None:
    """Each stage held to its 64-bit form on what the stage before stored."""
    s = _block_state(ops, m, d, f)
    _block(ops, s)
    _check_norm(s["x"], s["residual"], s["gamma1"], 1e-6, None, s["residual1"], s["q"], s["q_scale"])
    want, size = F8.gemm(s["q"], s["q_scale"], s["w1"], s["w1_scale"], s["b1"], "mish")
    _close(s["hidden"], want, size, d, "mish")
    codes, scale = F8.quantize(s["hidden"])
    want, size = F8.gemm(codes, scale, s["w2"], s["w2_scale"], s["b2"])
    _close(s["branch"], want, size, f)
    _check_norm(s["branch"], s["residual1"], s["gamma2"], 1e-6, s["out"], s["residual2"], None, None)


@pytest.mark.parametrize("m", [2, 300])
def test_feed_forward_block_captured_and_on_another_stream(ops, m) -> None:
    s = _block_state(ops, m, 512, 640)
    _block(ops, s)
    want = {name: s[name].clone() for name in RESULTS}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for name in RESULTS:
            s[name].zero_()
        _block(ops, s)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(s[name], want[name]) for name in RESULTS)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _block(ops, s)
    other = _rows(52, m, 512)
    first = s["x"].clone()
    for _ in range(3):  # replays see new inputs and repeat old results
        s["x"].copy_(other)
        graph.replay()
        assert not torch.equal(s["out"], want["out"])
        s["x"].copy_(first)
        graph.replay()
        assert all(torch.equal(s[name], want[name]) for name in RESULTS)


def test_two_calls_at_once(ops) -> None:
    """Two blocks on two streams with workspaces of their own, interleaved."""
    states = [_block_state(ops, m, 512, 1024) for m in (40, 40)]
    _block(ops, states[0])
    want = {name: states[0][name].clone() for name in RESULTS}
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for stream, s in zip(streams, states):
            with torch.cuda.stream(stream):
                _block(ops, s)
    torch.cuda.synchronize()
    for s in states:
        assert all(torch.equal(s[name], want[name]) for name in RESULTS)


def test_wrapper_refusals(ops) -> None:
    a, a_scale, w, w_scale = _operands(60, 8, 64, 256)
    out = torch.empty((8, 64), dtype=BF16, device="cuda")
    x = torch.empty((8, 256), dtype=BF16, device="cuda")
    for call, text in [
            (lambda: ops.gemm_fp8(out[:7], a, a_scale, w, w_scale), "shape"),
            (lambda: ops.gemm_fp8(out.half(), a, a_scale, w, w_scale), "bfloat16 or float32"),
            (lambda: ops.gemm_fp8(out, a, a_scale.t().contiguous(), w, w_scale), "a_scale"),
            (lambda: ops.gemm_fp8(out, a, a_scale, w[:, :255], w_scale), "w must"),
            (lambda: ops.gemm_fp8(out, a, a_scale, w, w_scale.half()), "w_scale"),
            (lambda: ops.gemm_fp8(out, a, a_scale, w, w_scale, bias=torch.zeros(63, dtype=BF16, device="cuda")), "bias"),
            (lambda: ops.gemm_fp8(torch.empty((64, 8), dtype=BF16, device="cuda").t(), a, a_scale, w, w_scale), "contiguous rows"),
            (lambda: ops.gemm_fp8(out, x, a_scale, w, w_scale), "float8"),
            (lambda: ops.linear_fp8(out, x, w, w_scale, None, torch.empty(8 * 255, dtype=FP8, device="cuda"), torch.empty(16, device="cuda")), "scratch_q"),
            (lambda: ops.linear_fp8(out, x, w, w_scale, None, torch.empty(8 * 256, dtype=FP8, device="cuda"), torch.empty(15, device="cuda")), "scratch_scale"),
            (lambda: ops.rms_norm(x, x, torch.ones(255, dtype=BF16, device="cuda")), "gammas"),
            (lambda: ops.quantize_fp8(a, torch.empty((8, 2), device="cuda"), x), "scale"),
    ]:
        with pytest.raises(ValueError, match=text):
            call()
    from lczero_triton_b200._lib import Lc0B200Error
    with pytest.raises(Lc0B200Error, match="null pointer"):
        ops.rms_norm(x, x, torch.ones(256, dtype=BF16, device="cuda"), residual_out=torch.empty_like(x))
    with pytest.raises(Lc0B200Error, match="null pointer"):
        ops.rms_norm(None, x, torch.ones(256, dtype=BF16, device="cuda"))
    with pytest.raises(Lc0B200Error, match="bad shape"):
        ops.rms_norm(x, x[:1].expand(8, 256), torch.ones(256, dtype=BF16, device="cuda"))  # rows that all lie on one another
    with pytest.raises(KeyError):
        ops.gemm_fp8(out, a, a_scale, w, w_scale, activation="tanh")
    before = out.clone()
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.int16), before.view(torch.int16))

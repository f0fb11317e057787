"""Which kernels the e4m3 operators launch, and each of those kernels against 64 bits.

The kernels are chosen by shape, alignment and the number of SMs; here the shapes are derived from the SM count and the
kernels that ran are read from a trace of the device, so that a changed rule cannot leave a kernel untested unseen.
Tolerances are those of test_gpu_fp8.py, which counts the roundings.
"""

from __future__ import annotations

import re

import pytest
import torch
from torch.autograd import DeviceType
from torch.profiler import ProfilerActivity, profile

from test_gpu_fp8 import BF16, FP8, _check_norm, _gen, _operands, _pitched, _placed, _rows, _scratch

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

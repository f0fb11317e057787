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

from test_gpu_fp8 import BF16, FP8, _gen, _operands, _pitched, _placed, _rows, _scratch

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

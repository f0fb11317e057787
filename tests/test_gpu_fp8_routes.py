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

"""CPU checks of the e4m3 entry points: what they refuse, with which status, before they touch a device; and the oracle's
rounding against torch's own conversion."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lczero_triton_b200 import _lib, build, ops
from oracle import fp8_oracle as F8

OK, NULL, SHAPE, UNSUPPORTED, MISALIGNED = 0, 1, 2, 3, 4
P = 4096  # a pointer that is never dereferenced: validation fails first, or there are no rows


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def _call(fn, defaults: dict, **changes) -> int:
    return fn(*{**defaults, **changes}.values())


QUANTIZE = dict(out=P, scale=P, x=P, rows=4, width=256, block_rows=1, ld_in=256, ld_out=256, ld_scale=4, stream=None)


@pytest.mark.parametrize("changes, status", [
    (dict(rows=0), OK),
    (dict(out=None), NULL), (dict(scale=None), NULL), (dict(x=None), NULL),
    (dict(rows=-1), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(width=0), SHAPE), (dict(width=(1 << 30) + 1), SHAPE),
    (dict(block_rows=64), UNSUPPORTED), (dict(block_rows=0), UNSUPPORTED),
    (dict(ld_in=255), SHAPE), (dict(ld_out=255), SHAPE), (dict(ld_scale=3), SHAPE),
    (dict(block_rows=128, ld_scale=1), SHAPE),
    (dict(x=P + 1), MISALIGNED), (dict(scale=P + 2), MISALIGNED),
])
def test_quantize_refusals(lib, changes, status) -> None:
    assert _call(lib.lc0b200_quantize_fp8, QUANTIZE, **changes) == status


RMS = dict(out=P, residual=P, q=P, scale=P, x=P, skip=P, gamma=P, rows=4, width=256, epsilon=1e-6, ld_in=256, ld_skip=256,
           ld_out=256, ld_residual=256, ld_q=256, ld_scale=4, stream=None)


@pytest.mark.parametrize("changes, status", [
    (dict(rows=0), OK), (dict(rows=0, out=None, ld_out=0), OK), (dict(rows=0, q=None, scale=None, ld_q=0, ld_scale=0), OK),
    (dict(rows=0, residual=None, skip=None, ld_skip=0, ld_residual=0), OK),
    (dict(out=None, q=None, scale=None), NULL), (dict(q=None), NULL), (dict(scale=None), NULL), (dict(x=None), NULL),
    (dict(gamma=None), NULL), (dict(skip=None), NULL),
    (dict(rows=-1), SHAPE), (dict(width=0), SHAPE), (dict(epsilon=-1e-6), SHAPE), (dict(epsilon=float("nan")), SHAPE),
    (dict(ld_in=255), SHAPE), (dict(ld_skip=255), SHAPE), (dict(ld_out=255), SHAPE), (dict(ld_residual=255), SHAPE),
    (dict(ld_q=255), SHAPE), (dict(ld_scale=3), SHAPE),
    (dict(x=P + 1), MISALIGNED), (dict(skip=P + 1), MISALIGNED), (dict(out=P + 1), MISALIGNED),
    (dict(residual=P + 1), MISALIGNED), (dict(gamma=P + 1), MISALIGNED), (dict(scale=P + 1), MISALIGNED),
])
def test_rms_norm_refusals(lib, changes, status) -> None:
    assert _call(lib.lc0b200_rms_norm, RMS, **changes) == status


GEMM = dict(out=P, a=P, a_scale=P, w=P, w_scale=P, bias=P, m=4, n=32, k=256, lda=256, ld_a_scale=4, ldw=256, ld_w_scale=2,
            ldc=32, out_kind=_lib.OUT_BF16, activation=0, stream=None)


@pytest.mark.parametrize("changes, status", [
    (dict(m=0), OK), (dict(m=0, bias=None), OK),
    (dict(out=None), NULL), (dict(a=None), NULL), (dict(a_scale=None), NULL), (dict(w=None), NULL), (dict(w_scale=None), NULL),
    (dict(m=-1), SHAPE), (dict(m=1 << 31), SHAPE), (dict(n=0), SHAPE), (dict(k=0), SHAPE), (dict(k=(1 << 30) + 1), SHAPE),
    (dict(lda=255), SHAPE), (dict(ldw=255), SHAPE), (dict(ldc=31), SHAPE), (dict(ld_a_scale=3), SHAPE),
    (dict(ld_w_scale=1), SHAPE), (dict(k=257, lda=272, ldw=272), SHAPE),
    (dict(out_kind=_lib.OUT_S32), UNSUPPORTED), (dict(out_kind=-1), UNSUPPORTED), (dict(activation=4), UNSUPPORTED),
    (dict(out=P + 1), MISALIGNED), (dict(out=P + 2, out_kind=_lib.OUT_F32), MISALIGNED), (dict(bias=P + 1), MISALIGNED),
    (dict(a_scale=P + 2), MISALIGNED), (dict(w_scale=P + 2), MISALIGNED),
])
def test_gemm_refusals(lib, changes, status) -> None:
    assert _call(lib.lc0b200_gemm_fp8, GEMM, **changes) == status


LINEAR = dict(out=P, a=P, w=P, w_scale=P, bias=P, scratch_q=P, scratch_scale=P, m=4, n=32, k=256, lda=256, ldw=256,
              ld_w_scale=2, ldc=32, out_kind=_lib.OUT_BF16, activation=0, stream=None)


@pytest.mark.parametrize("changes, status", [
    (dict(m=0), OK),
    (dict(out=None), NULL), (dict(a=None), NULL), (dict(w=None), NULL), (dict(w_scale=None), NULL),
    (dict(scratch_q=None), NULL), (dict(scratch_scale=None), NULL),
    (dict(m=-1), SHAPE), (dict(n=0), SHAPE), (dict(k=0), SHAPE), (dict(lda=255), SHAPE), (dict(ldc=31), SHAPE),
    (dict(scratch_q=P + 8), MISALIGNED), (dict(scratch_scale=P + 8), MISALIGNED), (dict(a=P + 1), MISALIGNED),
    (dict(out_kind=_lib.OUT_S32), UNSUPPORTED), (dict(activation=-1), UNSUPPORTED),
])
def test_linear_refusals(lib, changes, status) -> None:
    assert _call(lib.lc0b200_linear_fp8, LINEAR, **changes) == status


def test_wrappers_refuse_cpu_tensors() -> None:
    x = torch.zeros((4, 256), dtype=torch.bfloat16)
    q = torch.zeros((4, 256), dtype=torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="CUDA"):
        ops.quantize_fp8(q, torch.zeros((2, 4)), x)
    with pytest.raises(ValueError, match="block_rows"):
        ops.quantize_fp8(q, torch.zeros((2, 4)), x, block_rows=32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rms_norm(x.clone(), x, torch.ones(256, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA"):
        ops.gemm_fp8(x, q, torch.zeros((2, 4)), q, torch.zeros((1, 2)))
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear_fp8(x, x, q, torch.zeros((1, 2)), None, q, torch.zeros(8))


def test_oracle_rounds_like_the_type() -> None:
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    finite = every[torch.isfinite(every)].double().unique()
    middles = (finite[1:] + finite[:-1]) / 2
    x = torch.cat([finite, middles, torch.nextafter(middles.float(), torch.tensor(1e9)).double(),
                   torch.nextafter(middles.float(), torch.tensor(-1e9)).double(),
                   torch.randn(10000, dtype=torch.float64, generator=torch.Generator().manual_seed(1)) * 60]).clamp(-448, 448)
    assert torch.equal(F8.round_e4m3(x.float()), x.float().to(torch.float8_e4m3fn).double())
    assert F8.round_e4m3(torch.tensor([1e9, -1e9])).tolist() == [448.0, -448.0]
    assert torch.isnan(F8.round_e4m3(torch.tensor([float("nan")]))).all()

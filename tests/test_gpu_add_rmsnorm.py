"""add_rmsnorm against its definition in 64 bits: rows of every length around the units, wavefronts and workgroups, every
type, codes and scales per row and per block, rows without alignment, rows that are zero or not finite."""
from __future__ import annotations

import pytest
import torch

from forge_amd import _lib
from forge_amd import ops_decoder as ops
from forge_amd import ops_gemm
from forge_amd.errors import ConfigError
from tests._decoder_ref import HALF_ULP, norm_ref
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-5


def _data(m, k, dt, rdt, seed=0):
    g = gen(seed + 31 * m + k)
    x = (torch.randn(m, k, generator=g) * 3).to(dt)
    r = None if rdt is None else (torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-6, 7, (m, 1), generator=g).float())).to(rdt)
    return x, r, (1 + 0.2 * torch.randn(k, generator=g)).to(dt)


def _check(x, r, w, got, quant, block=128):
    y, h = norm_ref(x, r, w, EPS)
    assert torch.equal(got.residual.cpu(), h)  # one rounding of an exact sum in fp64, or of fp32's: the same but for ties
    k = x.shape[1]
    if quant is None:
        u, tiny = HALF_ULP[x.dtype]
        assert got.y.dtype == x.dtype and got.scale is None
        # fp32 arithmetic in front of the rounding: a sum of k squares, a square root, two quotients, two products
        assert bool(((got.y.cpu().double() - y).abs() <= (u + 2.0 ** -20) * y.abs() + tiny).all())
        return
    top = 127.0 if quant == "int8" else 448.0
    width = block if quant == "fp8_block" else k
    nb = -(-k // width)
    amax = torch.nn.functional.pad(y, (0, nb * width - k)).view(-1, nb, width).abs().amax(-1)
    s = torch.where(amax > 0, amax / top, torch.ones_like(amax))
    scale = got.scale.cpu().double().reshape(-1, nb)
    assert bool(((scale - s).abs() <= 2.0 ** -20 * s).all())
    ratio = y / scale.repeat_interleave(width, 1)[:, :k]
    if quant == "int8":
        assert got.y.dtype == torch.int8
        assert bool(((got.y.cpu().double() - ratio).abs() <= 0.5 + 127 * 2.0 ** -19).all())
    else:  # three bits below the first: half a step is 2^-4 of the value, 2^-10 below 2^-6
        assert got.y.dtype == torch.float8_e4m3fn
        assert bool(((got.y.cpu().float().double() - ratio).abs() <= ratio.abs() * (2.0 ** -4 + 2.0 ** -18) + 2.0 ** -10).all())


TYPES = [(BF, BF), (BF, FP), (BF, None), (HF, HF), (HF, FP), (FP, FP), (FP, None)]
QUANTS = [None, "int8", "fp8", "fp8_block"]
# one column; under, at and past a unit, a wavefront of units, a workgroup; units per thread 1, 2, 4; the longest row
SHAPES = [(1, 1), (3, 7), (2, 8), (5, 9), (4, 511), (4, 512), (3, 520), (1, 4096), (2, 5001), (3, 8200), (1, 32768), (600, 1000)]


@pytest.mark.parametrize("quant", QUANTS)
@pytest.mark.parametrize("dt,rdt", TYPES)
def test_against_the_definition(dt, rdt, quant):
    for m, k in SHAPES:
        x, r, w = _data(m, k, dt, rdt)
        got = ops.add_rmsnorm(x.to(DEV), w.to(DEV), None if r is None else r.to(DEV), eps=EPS, quant=quant)
        _check(x, r, w, got, quant)


@pytest.mark.parametrize("block", [8, 16, 64, 256, 512])
def test_blocks(block):
    for m, k in ((3, 1000), (700, 640)):
        x, r, w = _data(m, k, BF, BF)
        got = ops.add_rmsnorm(x.to(DEV), w.to(DEV), r.to(DEV), eps=EPS, quant="fp8_block", block=block)
        assert got.scale.shape == (m, -(-k // block))
        _check(x, r, w, got, "fp8_block", block)


@pytest.mark.parametrize("quant", QUANTS)
def test_strides_offsets_and_weights(quant):
    """Rows at odd elements, of a wider tensor, an expanded residual, weights of another type or none."""
    x, r, w = _data(5, 777, BF, FP)
    wide_x, wide_r = torch.zeros(5, 801, dtype=BF, device=DEV), torch.zeros(5, 790, device=DEV)
    wide_x[:, 3:780], wide_r[:, 1:778] = x.to(DEV), r.to(DEV)
    got = ops.add_rmsnorm(wide_x[:, 3:780], w.float().to(DEV), wide_r[:, 1:778], eps=EPS, quant=quant)
    _check(x, r, w.float(), got, quant)
    one = r[:1].expand(5, 777)
    _check(x, one, None, ops.add_rmsnorm(x.to(DEV), None, one.to(DEV), eps=EPS, quant=quant), quant)
    x3 = x.to(DEV).view(5, 1, 777)
    got = ops.add_rmsnorm(x3, w.to(DEV), r.to(DEV).view(5, 1, 777), eps=EPS, quant=quant)
    assert got.y.shape == got.residual.shape == x3.shape
    flat = ops.add_rmsnorm(x.to(DEV), w.to(DEV), r.to(DEV), eps=EPS, quant=quant)
    assert torch.equal(got.y.view(torch.uint8).flatten(), flat.y.view(torch.uint8).flatten())


def test_in_place():
    x, r, w = _data(9, 1234, HF, HF)
    rd = r.to(DEV)
    got = ops.add_rmsnorm(x.to(DEV), w.to(DEV), rd, eps=EPS, residual_out=rd)
    assert got.residual is rd
    _check(x, r, w, got, None)


def test_rows_of_zeros_and_rows_that_are_not_finite():
    x, r, w = _data(6, 512, BF, BF)
    r.zero_()
    x[0] = 0.0
    x[1, 5] = float("nan")
    x[2, 9] = float("inf")
    x[3] = torch.finfo(BF).max / 4  # the squares overflow: the norm is that of an infinite row
    for quant in QUANTS:
        got = ops.add_rmsnorm(x.to(DEV), w.to(DEV), r.to(DEV), eps=EPS, quant=quant)
        y = got.y.cpu().float()
        assert bool((y[0] == 0).all())
        if quant is None or quant.startswith("fp8"):
            assert bool(y[1].isnan().all()) and bool(y[2, 9].isnan()) and bool((y[2, 10:] == 0).all())
        if quant is not None:
            s = got.scale.cpu().reshape(6, -1)
            assert bool((s[:3] == 1).all()) and bool((s[3] == 1).all())
        assert bool((y[3] == 0).all())
        _check(x[4:], r[4:], w, type(got)(got.y[4:], None if got.scale is None else got.scale[4:], got.residual[4:]), quant)


def test_codes_feed_the_linears():
    """The codes and scales are those that the linears take, block scales in the order of columns that they read."""
    x, r, w = _data(33, 512, BF, BF)
    g = gen(5)
    wq, sw = ops_gemm.quantize_weight_fp8((torch.randn(256, 512, generator=g) * 0.05).to(DEV), "block2d")
    norm = ops.add_rmsnorm(x.to(DEV), w.to(DEV), r.to(DEV), eps=EPS)
    fused = ops.add_rmsnorm(x.to(DEV), w.to(DEV), r.to(DEV), eps=EPS, quant="fp8_block")
    y = ops_gemm.fp8_linear(fused.y, wq, sw, x_scale=fused.scale).float()
    # quantising the normed values after their rounding to bf16 moves codes by at most a step
    ref = ops_gemm.fp8_linear(norm.y, wq, sw).float()
    assert (y - ref).norm() <= 2.0 ** -4 * ref.norm()
    i8 = ops.add_rmsnorm(x.to(DEV), w.to(DEV), r.to(DEV), eps=EPS, quant="int8")
    w8, s8 = ops_gemm.quantize_weight_int8((torch.randn(256, 512, generator=g) * 0.05).to(DEV))
    acc = i8.y.cpu().long() @ w8.cpu().long().t()
    exact = acc.double() * i8.scale.cpu().double().view(-1, 1) * s8.cpu().double().view(1, -1)
    y = ops_gemm.int8_gemm(i8.y, i8.scale, w8, s8, out_dtype=FP).cpu().double()
    assert bool(((y - exact).abs() <= 2.0 ** -22 * exact.abs()).all())


def test_no_rows():
    got = ops.add_rmsnorm(torch.empty(0, 64, dtype=BF, device=DEV), None, torch.empty(0, 64, dtype=BF, device=DEV), quant="int8")
    assert got.y.shape == (0, 64) and got.scale.shape == (0,) and got.residual.shape == (0, 64)


def test_refusals():
    x, w = torch.zeros(2, 64, dtype=BF, device=DEV), torch.ones(64, dtype=BF, device=DEV)
    for bad in (dict(quant="fp4"), dict(quant="fp8_block", block=100), dict(residual=x[:1]), dict(residual=x.half()),
                dict(residual_out=x), dict(residual=x, residual_out=x.float()), dict(residual=x, residual_out=x.t().contiguous().t()),
                dict(weight=w[:5]), dict(weight=w.int()), dict(x=x.int()), dict(weight=w.cpu())):
        with pytest.raises(ConfigError):
            ops.add_rmsnorm(**{"x": x, "weight": w, **bad})
    with pytest.raises(ops_gemm.HardwareUnsupported):
        ops.add_rmsnorm(x.cpu(), w.cpu())
    with pytest.raises(Exception, match="32768"):
        ops.add_rmsnorm(torch.zeros(1, 32769, dtype=BF, device=DEV), None)


@pytest.mark.parametrize("quant", QUANTS)
@pytest.mark.parametrize("dt,rdt", [(BF, BF), (BF, FP), (BF, None), (FP, FP), (FP, None)])
def test_products_with_the_weight_past_the_type(dt, rdt, quant):
    """h w passes fp32's range where h / rms * w does not: in some rows, in a few columns of a row, in the last odd unit."""
    for m, k in ((4, 64), (3, 1000), (5, 5001), (2, 20000), (600, 1030)):
        x, r, w = _data(m, k, dt, rdt)
        w = w.float()
        w[k // 2], w[k - 1] = 2e23, -1e24
        x[1] = (x[1].float() * 1e15).to(dt)  # the squares' sum stays below 2^127
        x[0, k - 1] = 3.0
        got = ops.add_rmsnorm(x.to(DEV), w.to(DEV), None if r is None else r.to(DEV), eps=EPS, quant=quant)
        _check(x, r, w, got, quant)


def test_squares_past_the_type_behind_a_large_weight():
    """The norm of such a row is infinite, as that of any row whose squares overflow, and its finite values are zeros."""
    x, w = torch.full((2, 520), 3e38, dtype=BF, device=DEV), torch.full((520,), 2.0, dtype=BF, device=DEV)
    for quant in QUANTS:
        got = ops.add_rmsnorm(x, w, quant=quant)
        assert bool((got.y.float() == 0).all()) and (got.scale is None or bool((got.scale == 1).all()))


def test_products_past_the_type_in_place():
    x, _, w = _data(3, 777, BF, None)
    w = w.float()
    w[5] = 1e24
    x[2] *= 1e15
    y = x.to(DEV)
    status = _lib.lib().fg_add_rmsnorm(y.data_ptr(), 777, _lib.BF16, None, 0, None, 0, 0, w.to(DEV).data_ptr(), _lib.F32, EPS,
                                       y.data_ptr(), 777, _lib.BF16, None, 0, 0, 0, 3, 777, _lib.stream_of(y))
    assert status == _lib.OK
    _check(x, None, w, ops.NormOutput(y, None, x), None)


def test_one_row_in_the_place_of_its_input():
    """Codes too, whatever the strides: the row is read before any of it is written."""
    x, _, w = _data(1, 5001, BF, None)
    wd = w.to(DEV)
    for ydt in (_lib.BF16, _lib.I8, _lib.E4M3):
        y, s = x.to(DEV), torch.zeros(1, device=DEV)
        status = _lib.lib().fg_add_rmsnorm(y.data_ptr(), 6000, _lib.BF16, None, 0, None, 0, 0, wd.data_ptr(), _lib.BF16, EPS, y.data_ptr(),
                                           7000, ydt, s.data_ptr(), 1, 0, 0, 1, 5001, _lib.stream_of(y))
        assert status == _lib.OK
        raw = y.view(torch.int8 if ydt == _lib.I8 else torch.float8_e4m3fn)[:, :5001] if ydt != _lib.BF16 else y
        _check(x, None, w, ops.NormOutput(raw, None if ydt == _lib.BF16 else s, x), {_lib.I8: "int8", _lib.E4M3: "fp8"}.get(ydt))

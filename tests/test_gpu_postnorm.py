"""postnorm_add_rmsnorm against its definition in 64 bits: rows of every length around the units, wavefronts and workgroups, every
type, gates by column and by row, codes and scales, places and strides, rows that are zero or not finite."""
from __future__ import annotations

import pytest
import torch

from forge_amd import ops_decoder as ops
from forge_amd import ops_gemm
from forge_amd.errors import ConfigError
from tests._decoder_ref import HALF_ULP
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-5
QUANTS = [None, "int8", "fp8", "fp8_block"]
# a norm in fp32: a sum of k squares adds 8 a unit, four units, six steps of a wavefront and sixteen wavefronts, of which a square
# root keeps half; it, two quotients and up to five products more: 35 roundings of 2^-24
REL = 35 * 2.0 ** -24


def _data(m, k, dt, rdt, gate=None, seed=0):
    g = gen(seed + 17 * m + k)
    x = (torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-6, 7, (m, 1), generator=g).float())).to(dt)
    r = (torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-6, 7, (m, 1), generator=g).float())).to(rdt)
    pw, w = ((1 + 0.2 * torch.randn(k, generator=g)).to(dt) for _ in range(2))
    gt = None if gate is None else torch.randn(*((m, k) if gate == "rows" else (k,)), generator=g).to(dt)
    return x, pw, r, w, gt


def _run(x, pw, r, w, gate, **kw):
    pw, r, w, gate = (None if t is None else t.to(DEV) for t in (pw, r, w, gate))
    return ops.postnorm_add_rmsnorm(x.to(DEV), pw, r, w, gate=gate, eps=EPS, **kw)


def _check(x, pw, r, w, gate, got, quant, scale=1.0, block=128, post_eps=EPS):
    xd = x.double()
    b = xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + post_eps) * scale
    b = b if pw is None else b * pw.double()
    b = b if gate is None else b * gate.double()
    h = got.residual.cpu().double()
    u, tiny = HALF_ULP[r.dtype]
    exact = r.double() + b
    # what is added is off by REL, the fp32 sum by a rounding, the type's by another
    assert got.residual.dtype == r.dtype
    assert bool(((h - exact).abs() <= REL * b.abs() + (u + 2.0 ** -23) * exact.abs() + tiny).all())
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)  # of the residual as it is kept
    y = y if w is None else y * w.double()
    k = x.shape[1]
    if quant is None:
        u, tiny = HALF_ULP[x.dtype]
        assert got.y.dtype == x.dtype and got.scale is None
        assert bool(((got.y.cpu().double() - y).abs() <= (u + REL) * y.abs() + tiny).all())
        return
    top, width = 127.0 if quant == "int8" else 448.0, block if quant == "fp8_block" else k
    nb = -(-k // width)
    amax = torch.nn.functional.pad(y, (0, nb * width - k)).view(-1, nb, width).abs().amax(-1)
    s = torch.where(amax > 0, amax / top, torch.ones_like(amax))
    got_s = got.scale.cpu().double().reshape(-1, nb)
    assert bool(((got_s - s).abs() <= 2 * REL * s).all())
    ratio = y / got_s.repeat_interleave(width, 1)[:, :k]
    if quant == "int8":
        assert got.y.dtype == torch.int8
        assert bool(((got.y.cpu().double() - ratio).abs() <= 0.5 + 127 * 2 * REL).all())
    else:
        assert got.y.dtype == torch.float8_e4m3fn
        assert bool(((got.y.cpu().float().double() - ratio).abs() <= ratio.abs() * (2.0 ** -4 + 4 * REL) + 2.0 ** -10).all())


SHAPES = [(1, 1), (3, 7), (2, 8), (5, 9), (4, 511), (4, 512), (3, 520), (1, 4096), (2, 5001), (3, 8200), (1, 32768), (600, 1000),
          (601, 7), (515, 256), (520, 1028), (530, 2049), (514, 4096), (513, 4097)]  # many rows: their squares by strides up to 4096


@pytest.mark.parametrize("quant", QUANTS)
@pytest.mark.parametrize("dt,rdt", [(BF, BF), (BF, FP), (HF, HF), (HF, FP), (FP, FP)])
def test_against_the_definition(dt, rdt, quant):
    for i, (m, k) in enumerate(SHAPES):
        gate, scale = (None, "columns", "rows")[i % 3], (1.0, 0.37)[i % 2]
        x, pw, r, w, gt = _data(m, k, dt, rdt, gate)
        _check(x, pw, r, w, gt, _run(x, pw, r, w, gt, residual_scale=scale, quant=quant), quant, scale)


@pytest.mark.parametrize("block", [8, 64, 512])
def test_blocks_and_another_epsilon(block):
    for m, k in ((3, 1000), (700, 640), (700, 2500)):
        x, pw, r, w, gt = _data(m, k, BF, BF, "rows")
        got = _run(x, pw, r, w, gt, quant="fp8_block", block=block, post_eps=0.1)
        assert got.scale.shape == (m, -(-k // block))
        _check(x, pw, r, w, gt, got, "fp8_block", block=block, post_eps=0.1)


@pytest.mark.parametrize("quant", QUANTS)
def test_strides_offsets_and_missing_factors(quant):
    """Rows at odd elements of wider tensors, an expanded gate and residual, factors of other types or none."""
    x, pw, r, w, gt = _data(5, 777, BF, FP, "rows")
    wide_x, wide_g = torch.zeros(5, 801, dtype=BF, device=DEV), torch.zeros(5, 790, dtype=HF, device=DEV)
    wide_x[:, 3:780], wide_g[:, 1:778] = x.to(DEV), gt.to(DEV)
    got = ops.postnorm_add_rmsnorm(wide_x[:, 3:780], pw.float().to(DEV), r.to(DEV), w.half().to(DEV), gate=wide_g[:, 1:778], eps=EPS,
                                   quant=quant)
    _check(x, pw.float(), r, w.half(), gt.half(), got, quant)
    one, row = r[:1].expand(5, 777), gt[:1].expand(5, 777)
    got = ops.postnorm_add_rmsnorm(x.to(DEV), None, one.to(DEV), None, gate=row.to(DEV), eps=EPS, quant=quant)
    _check(x, None, one, None, row, got, quant)
    got = ops.postnorm_add_rmsnorm(x.to(DEV), None, r.to(DEV), None, gate=gt[0].to(DEV).expand(5, 777), eps=EPS, quant=quant)
    _check(x, None, r, None, row, got, quant)
    x3 = x.to(DEV).view(5, 1, 777)
    got = ops.postnorm_add_rmsnorm(x3, pw.to(DEV), r.to(DEV).view(5, 1, 777), w.to(DEV), gate=gt.to(DEV).view(5, 1, 777), eps=EPS,
                                   quant=quant)
    assert got.y.shape == got.residual.shape == x3.shape
    flat = _run(x, pw, r, w, gt, quant=quant)
    assert torch.equal(got.y.view(torch.uint8).flatten(), flat.y.view(torch.uint8).flatten())


def test_in_place():
    x, pw, r, w, gt = _data(9, 1234, HF, HF, "columns")
    rd = r.to(DEV)
    got = ops.postnorm_add_rmsnorm(x.to(DEV), pw.to(DEV), rd, w.to(DEV), gate=gt.to(DEV), eps=EPS, residual_out=rd)
    assert got.residual is rd
    _check(x, pw, r, w, gt, got, None)


def test_rows_of_zeros_and_rows_that_are_not_finite():
    x, pw, r, w, _ = _data(6, 512, BF, BF)
    x[0] = 0.0
    x[1, 5] = float("nan")
    x[2, 9] = float("inf")
    x[3] = torch.finfo(BF).max / 4  # the squares overflow: the block's part is zero
    for quant in QUANTS:
        got = _run(x, pw, r, w, None, quant=quant)
        assert torch.equal(got.residual[0].cpu(), r[0]) and torch.equal(got.residual[3].cpu(), r[3])
        assert bool(got.residual[1].isnan().all()) and bool(got.residual[2, 9].isnan())
        for i in (0, 3, 4, 5):  # nothing of one row shows in another
            part = ops.NormOutput(got.y[i:i + 1], None if got.scale is None else got.scale[i:i + 1], got.residual[i:i + 1])
            _check(torch.zeros_like(x[i:i + 1]) if i == 3 else x[i:i + 1], pw, r[i:i + 1], w, None, part, quant)


@pytest.mark.parametrize("quant", QUANTS)
def test_products_with_the_weight_past_the_type(quant):
    for m, k in ((4, 64), (5, 5001), (600, 1030)):
        x, pw, r, w, gt = _data(m, k, BF, FP, "rows")
        w = w.float()
        w[k // 2], w[k - 1] = 2e23, -1e24
        r[1] = r[1] * 1e15  # the squares' sum stays below 2^127
        _check(x, pw, r, w, gt, _run(x, pw, r, w, gt, quant=quant), quant)


def test_zeros_of_a_row_without_epsilon_past_its_end():
    """1 / rms is infinite or large: the columns that a unit has past the row's end do not show in the row's second norm."""
    x, r = torch.zeros(2, 13, dtype=BF), torch.ones(2, 13, dtype=BF)
    x[1, 0] = 1e-18
    got = ops.postnorm_add_rmsnorm(x.to(DEV), None, r.to(DEV), None, eps=0.0)
    assert bool(got.y[0].isnan().all())  # zero by zero, as the formula has it
    _check(x[1:], None, r[1:], None, None, ops.NormOutput(got.y[1:], None, got.residual[1:]), None, post_eps=0.0)


def test_no_rows():
    e = torch.empty(0, 64, dtype=BF, device=DEV)
    got = ops.postnorm_add_rmsnorm(e, None, e, None, quant="int8")
    assert got.y.shape == (0, 64) and got.scale.shape == (0,) and got.residual.shape == (0, 64)


def test_refusals():
    x, w = torch.zeros(2, 64, dtype=BF, device=DEV), torch.ones(64, dtype=BF, device=DEV)
    for bad in (dict(quant="fp4"), dict(quant="fp8_block", block=100), dict(residual=x[:1]), dict(residual=x.half()),
                dict(residual_out=x.float()), dict(residual_out=x.t().contiguous().t()), dict(weight=w[:5]), dict(weight=w.int()),
                dict(post_weight=w[:5]), dict(gate=w[:5]), dict(gate=x[:1]), dict(gate=x.int()), dict(gate=w.cpu()), dict(x=x.int()),
                dict(post_weight=w.cpu())):
        with pytest.raises(ConfigError):
            ops.postnorm_add_rmsnorm(**{"x": x, "post_weight": w, "residual": x.clone(), "weight": w, **bad})
    with pytest.raises(ops_gemm.HardwareUnsupported):
        ops.postnorm_add_rmsnorm(x.cpu(), None, x.cpu(), None)
    with pytest.raises(Exception, match="gate"):
        ops.postnorm_add_rmsnorm(x, None, x, None, gate=x, residual_out=x)
    long = torch.zeros(1, 32769, dtype=BF, device=DEV)
    with pytest.raises(Exception, match="32768"):
        ops.postnorm_add_rmsnorm(long, None, long, None)


@pytest.mark.parametrize("m,k", [(600, 1024), (600, 1000), (520, 4096)])
def test_many_rows_as_the_steps_one_by_one(m, k):
    """Up to 4096 columns the squares are added up in the order of torch's own sum: the same quotients, and the residual to the bit."""
    x, pw, r, w, gt = (None if t is None else t.to(DEV) for t in _data(m, k, BF, BF, "columns"))
    xf = x.float()
    b = xf / torch.sqrt((xf * xf).mean(-1, keepdim=True) + EPS) * pw.float() * 0.5 * gt.float()
    got = ops.postnorm_add_rmsnorm(x, pw, r, w, gate=gt, residual_scale=0.5, eps=EPS)
    # fp32 sums that differ in their last place in some rows would show in one of 2^13 residuals or so
    assert int((got.residual != (r.float() + b).to(BF)).sum()) <= m * k // 2 ** 13

"""Microscaled 4-bit operators on the GPU against the float64 oracle."""
import numpy as np
import pytest
import torch

from oracle import fp4 as F4
from thor_int8_gemm_b200 import ops

pytestmark = pytest.mark.gpu
KINDS = ("mxfp4", "nvfp4")
DEV = "cuda:0"


def rand_bf16(rng, s, d, spread=2.0):
    v = rng.standard_normal((s, d)) * np.exp(spread * rng.standard_normal((s, 1)))
    return torch.from_numpy(v).to(torch.bfloat16)


def check_operand(got, x, kind):
    """(q, sf, q_scale) against the oracle's quantisation of the bf16 tensor x, every byte."""
    q, sf, qs = got
    code, byte, rs = F4.quant(x.double().numpy(), kind)
    S, D = x.shape
    g = q.cpu().numpy()
    gcode = np.stack([g & 15, g >> 4], 2).reshape(S, D).astype(np.int64)
    dead = np.zeros((S, D), bool)
    if kind == "nvfp4":
        assert np.array_equal(qs.cpu().numpy().astype(np.float64), rs, equal_nan=True)
        dead |= np.isnan(rs)[:, None]
    else:
        assert qs is None
        dead |= np.repeat(byte == 255, 32, 1)[:, :D]
    # a zero may carry either sign; what stands under a NaN scale is not looked at
    same = (gcode == code) | (((gcode | code) & 7) == 0) | dead
    assert same.all(), np.argwhere(~same)[:5]
    assert sf.numel() == ops.fp4_scale_bytes(S, D, kind)
    # rows of the tiles, blocks filled up to a multiple of four with zeros
    words = F4.tile_scales(byte).reshape(-(-S // 128), -1, 32, 4, 4).transpose(0, 3, 2, 1, 4).reshape(-(-S // 128) * 128, -1)[:S]
    got_words = sf.cpu().numpy().reshape(-(-S // 128), -1, 32, 4, 4).transpose(0, 3, 2, 1, 4).reshape(-(-S // 128) * 128, -1)[:S]
    ok = np.ones(S, bool) if rs is None else ~np.isnan(rs)
    assert np.array_equal(got_words[ok], words[ok])
    assert np.array_equal(ops.fp4_scale_rows(sf, S, D, kind).cpu().numpy()[ok], byte[ok])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("s,d", [(1, 8), (1, 16), (3, 24), (5, 40), (129, 128), (33, 264), (64, 1288), (300, 2048),
                                 (2, 8192), (7, 8200), (5, 12288), (3, 49152), (2100, 1024), (2500, 3072)])
def test_quant_rows(kind, s, d):
    rng = np.random.default_rng(s * 100003 + d)
    x = rand_bf16(rng, s, d)
    check_operand(ops.quant_rows_fp4(x.to(DEV), kind), x, kind)


@pytest.mark.parametrize("kind", KINDS)
def test_quant_every_border_and_extreme(kind):
    """Rows whose values sit on and beside every border, all-zero rows and blocks, subnormals, the
    largest finite bf16, NaN and infinities."""
    grid = torch.arange(-255, 256, dtype=torch.float64).to(torch.bfloat16)
    rows = [torch.cat([grid, grid[:1]])]
    rows += [(rows[0].double() * 2.0 ** e).to(torch.bfloat16) for e in (-133, -120, -60, 7, 119)]
    for m in range(128, 256):   # a block maximum of every significand
        r = (torch.arange(512, dtype=torch.float64) % 16 - 8).to(torch.bfloat16)
        r[0::16] = m / 16.0
        rows.append(r)
    z = torch.zeros(512, dtype=torch.bfloat16)
    rows.append(z)
    half = rows[0].clone()
    half[:48] = 0
    rows.append(half)
    big = rows[0].clone()
    big[5] = torch.finfo(torch.bfloat16).max
    rows.append(big)
    for v in (float("nan"), float("inf"), -float("inf")):
        r = rows[0].clone()
        r[100] = v
        rows.append(r)
    x = torch.stack(rows)
    got = ops.quant_rows_fp4(x.to(DEV), kind)
    check_operand(got, x, kind)
    code, byte, rs = F4.quant(x.double().numpy(), kind)
    val = F4.value(code, byte, rs, kind)
    out = ops.dequant_rows_fp4(*got, kind, out_dtype=torch.float32).cpu().numpy()
    ref = val.astype(np.float32)
    assert np.array_equal(out, ref, equal_nan=True)


@pytest.mark.parametrize("kind", KINDS)
def test_quant_strided_rows_and_other_bytes_untouched(kind):
    rng = np.random.default_rng(3)
    big = rand_bf16(rng, 9, 200).to(DEV)
    x = big[1:8, 8:8 + 136]
    check_operand(ops.quant_rows_fp4(x, kind), x.cpu(), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_dequant_types(kind, dtype):
    rng = np.random.default_rng(11)
    x = rand_bf16(rng, 37, 168, spread=0.5)
    code, byte, rs = F4.quant(x.double().numpy(), kind)
    ref = torch.from_numpy(F4.value(code, byte, rs, kind)).to(dtype)
    out = ops.dequant_rows_fp4(*ops.quant_rows_fp4(x.to(DEV), kind), kind, out_dtype=dtype).cpu()
    assert torch.equal(out, ref)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("s,d,form", [(1, 64, "batch"), (10, 264, "index"), (64, 1024, "batch"), (35, 2048, "w"),
                                      (20, 1288, "w"), (6, 8192, "index"), (4, 9216, "batch"), (3, 20488, "w"),
                                      (2500, 1024, "index"), (2200, 3072, "batch"), (2051, 2048, "w"),
                                      (2300, 4096, "index")])
def test_rms_mod_quant_equals_quant_of_h(kind, s, d, form):
    rng = np.random.default_rng(d + s)
    x = rand_bf16(rng, s, d, 0.5).to(DEV)
    n_mod = 3 if form == "index" else 1 if s % 2 else 2
    shift, scale = (rand_bf16(rng, n_mod, d, 0.2).to(DEV) for _ in range(2))
    kw = dict(eps=1e-6)
    if form == "index":
        kw["mod_index"] = torch.from_numpy(rng.integers(0, n_mod, s).astype(np.int32)).to(DEV)
    if form == "w":
        kw["w"] = rand_bf16(rng, 1, d, 0.1).view(-1).to(DEV)
        kw["scale_is_multiplier"] = True
    h = ops.rms_mod_quant(x, shift, scale, kind="int8", return_h=True, **kw)[2]
    got = ops.rms_mod_quant_fp4(x, shift, scale, kind=kind, **kw)
    check_operand(got, h.cpu(), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,f", [(1, 8), (3, 136), (77, 2568), (20, 12288), (2, 24576), (130, 1024)])
def test_swiglu_quant_equals_quant_of_act(kind, m, f):
    rng = np.random.default_rng(m + f)
    y = rand_bf16(rng, m, 2 * f, 0.3).to(DEV)
    act = ops.swiglu_quant_fc1(y, kind="int8", return_act=True)[2]
    check_operand(ops.swiglu_quant_fp4_fc1(y, kind), act.cpu(), kind)


# ---------------------------------------------------------------- products
def operand(rng, rows, k, kind, scale=1.0):
    """Random quantised matrix: the GPU buffers and the float64 values."""
    x = (rand_bf16(rng, rows, k, 0.5).double() * scale).to(torch.bfloat16)
    got = ops.quant_rows_fp4(x.to(DEV), kind)
    return got, F4.value(*F4.quant(x.double().numpy(), kind), kind)


def tolerance(xv, wv, k, ref, dtype):
    """fp32 accumulation of K products in K / 64 steps: each addition is off by at most one unit in
    the last place (2^-23, whatever the hardware's rounding) of the sum of magnitudes, each K = 64 product
    sum likewise; then the epilogue's two multiplications and addition (2^-24 each) and half a unit
    of the output type."""
    mag = np.abs(xv) @ np.abs(wv).T
    steps = -(-k // 64)
    return mag * 2.0 ** -23 * (2 * steps + 2) + np.abs(ref) * (torch.finfo(dtype).eps / 2 + 2.0 ** -22)


SHAPES = [(1, 64, 64), (1, 1, 8), (3, 7, 24), (128, 64, 256), (5, 130, 520), (64, 192, 1024), (130, 257, 2104),
          (256, 512, 768), (333, 1000, 264), (300, 5, 520), (300, 9, 264),
          (2100, 1003, 136), (1, 1024, 4096), (300, 300, 4104), (700, 2304, 640)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm(kind, m, n, k):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    (xq, xsf, xs), xv = operand(rng, m, k, kind)
    (wq, wsf, ws), wv = operand(rng, n, k, kind, 0.02)
    dtype = (torch.bfloat16, torch.float16, torch.float32)[(m + n + k) // 8 % 3]
    bias = torch.from_numpy(rng.standard_normal(n) * 0.1).to(dtype) if n % 2 == 0 else None
    ref = xv @ wv.T + (bias.double().numpy() if bias is not None else 0)
    out = ops.gemm_fp4(xq, wq, xsf, wsf, xs, ws, None if bias is None else bias.to(DEV), kind=kind, out_dtype=dtype)
    err = np.abs(out.cpu().double().numpy() - ref)
    tol = tolerance(xv, wv, k, ref, dtype)
    assert (err <= tol).all(), (err / tol).max()
    assert ops.device_status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k,form", [(1, 64, 256, "one"), (12, 136, 520, "batch"), (257, 512, 1032, "batch"),
                                        (130, 264, 2104, "index"), (600, 2304, 640, "inplace"),
                                        (2600, 1032, 512, "index"), (2048, 2304, 1288, "inplace")])
def test_gated(kind, m, n, k, form):
    """res + gate * (product + bias), rounded once: two more float32 roundings than the plain product (each
    2^-24 of the gated term or the sum) before the output's half unit."""
    rng = np.random.default_rng(m + n + k)
    (xq, xsf, xs), xv = operand(rng, m, k, kind)
    (wq, wsf, ws), wv = operand(rng, n, k, kind, 0.02)
    bias = rand_bf16(rng, 1, n, 0.1).view(-1) if form != "one" else None
    res = rand_bf16(rng, m, n, 0.1)
    n_gate = {"one": 1, "batch": 3 if m % 3 == 0 else 1, "index": 5, "inplace": 2}[form]
    gate = rand_bf16(rng, n_gate, n, 0.1)
    idx = rng.integers(0, n_gate, m).astype(np.int32) if form == "index" else np.arange(m) // (m // n_gate)
    y = xv @ wv.T + (bias.double().numpy() if bias is not None else 0)
    g = gate.double().numpy()[idx]
    ref = res.double().numpy() + g * y
    res_d = res.to(DEV)
    kw = dict(gate_index=torch.from_numpy(idx).to(DEV)) if form == "index" else {}
    out = ops.gemm_fp4_gated(xq, wq, xsf, wsf, xs, ws, None if bias is None else bias.to(DEV), res_d, gate.to(DEV),
                             kind=kind, out=res_d if form == "inplace" else None, **kw)
    assert (out is res_d) == (form == "inplace")
    err = np.abs(out.cpu().double().numpy() - ref)
    steps = -(-k // 64)
    acc = np.abs(xv) @ np.abs(wv).T * 2.0 ** -23 * (2 * steps + 2) + np.abs(y) * 2.0 ** -22
    tol = np.abs(g) * acc + np.abs(ref) * (2.0 ** -8 + 2.0 ** -23)
    assert (err <= tol).all(), (err / tol).max()
    assert ops.device_status() == 0

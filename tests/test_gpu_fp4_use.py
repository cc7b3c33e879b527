"""The microscaled 4-bit operators as they are used: together, in a DiT block, under torch.compile, on other
streams and in CUDA graphs; empty and far-off sizes; NaN, infinities and unwritten padding."""
import numpy as np
import pytest
import torch

from oracle import fp4 as F4
from thor_int8_gemm_b200 import dit, ops

pytestmark = pytest.mark.gpu
KINDS = ("mxfp4", "nvfp4")
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert ops.device_status() == 0


def randn(g, *s, scale=1.0):
    return (torch.randn(*s, generator=g, device=DEV) * scale).to(torch.bfloat16)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def product(x, w, bias=None, kind="nvfp4", **kw):
    return ops.gemm_fp4(x[0], w[0], x[1], w[1], x[2], w[2], bias, kind=kind, **kw)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,T,hidden,heads,ffn", [(2, 64, 256, 2, 520), (1, 300, 384, 3, 1024), (2, 1100, 512, 4, 1024)])
def test_dit_block(kind, B, T, hidden, heads, ffn):
    """The block is its operators in a row; its fused gate is the product's own epilogue; and it stays
    near the block whose linears are exact on the dequantised operands."""
    M = B * T
    g = gen(5)
    x, cond = randn(g, M, hidden), randn(g, B, 6 * hidden, scale=0.1)
    blk = dit.DiTBlock(hidden, heads, ffn, kind=kind, device=DEV, seed=7)
    fused = dit.DiTBlock(hidden, heads, ffn, kind=kind, device=DEV, seed=7, fused_gate=True)
    sh1, sc1, g1, sh2, sc2, g2 = blk.modulation(cond)
    h1 = ops.rms_mod_quant_fp4(x, sh1, sc1, rows_per_mod=T, eps=blk.eps, kind=kind)
    qkv = blk.qkv(*h1)
    exact = ops.dequant_rows_fp4(*h1, kind, out_dtype=torch.float32).double() @ ops.dequant_rows_fp4(
        blk.qkv.w, blk.qkv.w_sf, blk.qkv.ws, kind, out_dtype=torch.float32).double().t() + blk.qkv.bias.double()
    # float32 accumulation stays far below the bf16 rounding of the result
    assert ((qkv.double() - exact).abs() <= exact.abs() * 2.0 ** -8 + exact.abs().max() * 2.0 ** -16).all()
    a = ops.quant_rows_fp4(blk.attention(qkv, B), kind)
    y1 = blk.gated(x, g1, blk.proj(*a), B)
    h2 = ops.rms_mod_quant_fp4(y1, sh2, sc2, rows_per_mod=T, eps=blk.eps, kind=kind)
    a2 = ops.swiglu_quant_fp4_fc1(blk.fc1(*h2), kind)
    y2 = blk.gated(y1, g2, blk.fc2(*a2), B)
    assert torch.equal(blk(x, cond, B), y2)
    z1 = ops.gemm_fp4_gated(a[0], blk.proj.w, a[1], blk.proj.w_sf, a[2], blk.proj.ws, blk.proj.bias, x, g1,
                            rows_per_gate=T, kind=kind)
    h2 = ops.rms_mod_quant_fp4(z1, sh2, sc2, rows_per_mod=T, eps=blk.eps, kind=kind)
    a2 = ops.swiglu_quant_fp4_fc1(blk.fc1(*h2), kind)
    z2 = ops.gemm_fp4_gated(a2[0], blk.fc2.w, a2[1], blk.fc2.w_sf, a2[2], blk.fc2.ws, blk.fc2.bias, z1, g2,
                            rows_per_gate=T, kind=kind)
    assert torch.equal(fused(x, cond, B), z2)


@pytest.mark.parametrize("kind", KINDS)
def test_compiled_ops_match_eager(kind):
    from thor_int8_gemm_b200 import torch_ops  # noqa: F401
    t = torch.ops.t8g
    g = gen(3)
    M, D, F = 300, 520, 1032
    x, shift, scale, res, gate = randn(g, M, D), randn(g, 1, D), randn(g, 1, D), randn(g, M, D), randn(g, 1, D)
    w1, w2 = (ops.quant_rows_fp4(randn(g, *s, scale=0.02), kind) for s in ((2 * F, D), (D, F)))
    none = torch.empty(0, device=DEV)

    def mlp(x, shift, scale, a, a_sf, a_s, b, b_sf, b_s, res, gate):
        q, sf, s = t.rms_mod_quant_fp4(x, shift, scale, None, None, x.shape[0], False, 1e-6, kind)
        q, sf, s = t.swiglu_quant_fp4(t.gemm_fp4(q, a, sf, a_sf, s, a_s, None, kind, torch.bfloat16), kind)
        return t.gemm_fp4_gated(q, b, sf, b_sf, s, b_s, None, res, gate, x.shape[0], kind)

    args = (x, shift, scale, w1[0], w1[1], none if w1[2] is None else w1[2], w2[0], w2[1],
            none if w2[2] is None else w2[2], res, gate)
    h = ops.rms_mod_quant_fp4(x, shift, scale, rows_per_mod=M, eps=1e-6, kind=kind)
    a = ops.swiglu_quant_fp4_fc1(product(h, w1, kind=kind), kind)
    want = ops.gemm_fp4_gated(a[0], w2[0], a[1], w2[1], a[2], w2[2], None, res, gate, rows_per_gate=M, kind=kind)
    assert torch.equal(torch.compile(mlp, backend="aot_eager", fullgraph=True)(*args), want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(5, 200, 1032), (700, 520, 2056)])
def test_graph_replay_and_streams(kind, m, n, k):
    """Two captured graphs of the same calls replayed in turn and together with a third stream: each
    gives what the eager calls give for its inputs; nothing is shared between calls."""
    g = gen(9)
    w = ops.quant_rows_fp4(randn(g, n, k, scale=0.02), kind)
    bias = randn(g, n)
    xs = [randn(g, m, k) for _ in range(3)]
    eager = [product(ops.quant_rows_fp4(x, kind), w, bias, kind) for x in xs]
    torch.cuda.synchronize()
    graphs, ins, outs = [], [], []
    for _ in range(2):
        buf = torch.zeros_like(xs[0])
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = product(ops.quant_rows_fp4(buf, kind), w, bias, kind)
        graphs.append(gr), ins.append(buf), outs.append(out)
    for turn in range(3):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ins[0].copy_(xs[turn])
            graphs[0].replay()
        ins[1].copy_(xs[(turn + 1) % 3])
        graphs[1].replay()
        third = torch.cuda.Stream()
        third.wait_stream(torch.cuda.current_stream())
        q = ops.quant_rows_fp4(xs[2], kind, stream=third)
        direct = product(q, w, bias, kind, stream=third)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager[turn])
        assert torch.equal(outs[1], eager[(turn + 1) % 3]) and torch.equal(direct, eager[2])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [3, 200, 1500])
def test_nan_and_infinity_stay_in_their_rows(kind, m):
    g = gen(m)
    x = randn(g, m, 776)
    bad = sorted({0, m // 2, m - 1})
    for i, v in zip(bad, (float("nan"), float("inf"), -float("inf"))):
        x[i, 100 * i % 776] = v
    w = ops.quant_rows_fp4(randn(g, 264, 776, scale=0.02), kind)
    out = product(ops.quant_rows_fp4(x, kind), w, kind=kind)
    clean = x.clone()
    clean[bad] = 0
    ref = product(ops.quant_rows_fp4(clean, kind), w, kind=kind)
    keep = torch.ones(m, dtype=torch.bool, device=DEV)
    keep[bad] = False
    assert out[bad].isnan().all() and torch.equal(out[keep], ref[keep])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(1, 130, 264), (77, 200, 520), (130, 300, 1032), (2050, 1100, 776)])
def test_padding_is_not_read_into_results(kind, m, n, k):
    """NaN scales in the tiles' unused rows, ones in the bytes between a row of codes and the next, and
    output columns past N: none of them matters or changes."""
    g = gen(m + n)
    x, w = randn(g, m, k), randn(g, n, k, scale=0.02)
    xq, wq = ops.quant_rows_fp4(x, kind), ops.quant_rows_fp4(w, kind)
    want = product(xq, wq, kind=kind)

    def soiled(op, rows):
        q, sf, s = op
        blocks = -(-k // ops.FP4_BLOCK[kind])
        tiles = torch.full((-(-rows // 128), -(-blocks // 4), 32, 4, 4), 255, dtype=torch.uint8, device=DEV)
        src = sf.view(tiles.shape)
        r = torch.arange(tiles.shape[0] * 128, device=DEV).view(-1, 4, 32)
        live = (r < rows).permute(0, 2, 1)[:, None, :, :, None].expand_as(tiles)
        tiles = torch.where(live, src, tiles).contiguous().view(-1)
        wide = torch.full((rows, k // 2 + 48 - k // 2 % 16), 0x77, dtype=torch.uint8, device=DEV)
        wide[:, :k // 2] = q
        return wide[:, :k // 2], tiles, s

    pad = -(-n // 8) * 8 + 16
    buf = torch.full((m, pad), 7.0, dtype=torch.bfloat16, device=DEV)
    product(soiled(xq, m), soiled(wq, n), kind=kind, out=buf[:, :n])
    assert torch.equal(buf[:, :n], want)
    assert (buf[:, n:] == 7).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(4921, 4112, 8), (4921, 4112, 520), (2305, 9232, 264)])
def test_tiles_without_work_for_some_warps(kind, m, n, k):
    """Persistent tiles where some epilogue warps have no rows or no columns and run ahead of the others: the
    result does not depend on which warp is first."""
    g = gen(m + n)
    x, w = ops.quant_rows_fp4(randn(g, m, k), kind), ops.quant_rows_fp4(randn(g, n, k, scale=0.02), kind)
    res, gate = randn(g, m, n), randn(g, 3, n)
    val = lambda o: ops.dequant_rows_fp4(*o, kind, out_dtype=torch.float32).double()  # noqa: E731
    y = val(x) @ val(w).t()
    rows = -(-m // 3)
    want = res.double() + gate.double()[torch.arange(m, device=DEV) // rows] * y
    first = None
    for _ in range(8):
        got = ops.gemm_fp4_gated(x[0], w[0], x[1], w[1], x[2], w[2], None, res, gate, rows_per_gate=rows, kind=kind)
        # half a bf16 unit, and float32 accumulation far below 2^-14 of these operands' sums
        assert ((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -14 * y.abs().max()).all()
        out = product(x, w, kind=kind)
        assert ((out.double() - y).abs() <= y.abs() * 2.0 ** -8 + 2.0 ** -14 * y.abs().max()).all()
        first = first or (got, out)
        assert torch.equal(got, first[0]) and torch.equal(out, first[1])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", (520, 552, 576, 640, 648, 680, 744, 768))
def test_gated_last_columns(kind, n):
    """The gated form where the columns end in each 32 of a tile's row slice, in a padded residual updated in place:
    the same values, and what lies past the columns and rows stays."""
    m, k = 333, 264
    g = gen(n)
    x, w = ops.quant_rows_fp4(randn(g, m, k), kind), ops.quant_rows_fp4(randn(g, n, k, scale=0.02), kind)
    big, gate = randn(g, m + 3, n + 8), randn(g, 5, n)
    keep, res = big.clone(), big[:m, :n]
    idx = torch.randint(0, 5, (m,), generator=g, device=DEV, dtype=torch.int32)
    val = lambda o: ops.dequant_rows_fp4(*o, kind, out_dtype=torch.float32).double()  # noqa: E731
    y = val(x) @ val(w).t()
    want = res.double() + gate.double()[idx.long()] * y
    ops.gemm_fp4_gated(x[0], w[0], x[1], w[1], x[2], w[2], None, res, gate, gate_index=idx, kind=kind, out=res)
    # half a bf16 unit, and float32 accumulation far below 2^-14 of these operands' sums
    assert ((res.double() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -14 * (gate.abs().max() * y.abs().max())).all()
    assert torch.equal(big[m:], keep[m:]) and torch.equal(big[:, n:], keep[:, n:])


@pytest.mark.parametrize("kind", KINDS)
def test_scales_and_repeats(kind):
    """Row and weight scales in their forms (a row, one for all, none), an operand without a row scale,
    and the same bits from the same call, with K split over a cluster and not."""
    g = gen(1)
    for m, n, k in ((1, 264, 4096), (100, 264, 2056), (600, 1032, 1032)):
        x, w = ops.quant_rows_fp4(randn(g, m, k), kind), ops.quant_rows_fp4(randn(g, n, k, scale=0.02), kind)
        xs = torch.rand(m, generator=g, device=DEV) + 0.5
        ws = torch.rand(n, generator=g, device=DEV) + 0.5
        one = torch.tensor([0.75], device=DEV)
        base = ops.gemm_fp4(x[0], w[0], x[1], w[1], kind=kind, out_dtype=torch.float32)
        call = lambda a, b: ops.gemm_fp4(x[0], w[0], x[1], w[1], a, b, kind=kind, out_dtype=torch.float32)  # noqa: E731
        assert torch.equal(call(xs, None), base * xs[:, None])
        assert torch.equal(call(None, ws), base * ws)
        assert torch.equal(call(xs, one), (base * xs[:, None]) * 0.75)
        assert torch.equal(call(xs, ws), (base * xs[:, None]) * ws)
        assert torch.equal(base, ops.gemm_fp4(x[0], w[0], x[1], w[1], kind=kind, out_dtype=torch.float32))


@pytest.mark.parametrize("kind", KINDS)
def test_empty(kind):
    e = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    q = ops.quant_rows_fp4(e, kind)
    assert q[0].shape == (0, 32) and q[1].numel() == 0
    assert ops.dequant_rows_fp4(*q, kind).shape == (0, 64)
    w = ops.quant_rows_fp4(torch.ones(16, 64, dtype=torch.bfloat16, device=DEV), kind)
    assert product(q, w, kind=kind).shape == (0, 16)
    assert product(w, q, kind=kind).shape == (16, 0)
    assert ops.swiglu_quant_fp4_fc1(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV), kind)[0].shape == (0, 16)
    m = torch.ones(1, 64, dtype=torch.bfloat16, device=DEV)
    assert ops.rms_mod_quant_fp4(e, m, m, rows_per_mod=1, kind=kind)[0].shape == (0, 32)


def test_wrapper_refusals():
    x = torch.ones(4, 64, dtype=torch.bfloat16, device=DEV)
    q, sf, s = ops.quant_rows_fp4(x, "nvfp4")
    with pytest.raises(ValueError, match="multiple of 8"):
        ops.quant_rows_fp4(x[:, :60], "nvfp4")
    with pytest.raises(ValueError, match="unit stride"):
        ops.quant_rows_fp4(x.t(), "nvfp4")
    with pytest.raises(TypeError):
        ops.quant_rows_fp4(x.float(), "nvfp4")
    with pytest.raises(ValueError, match="at least"):
        ops.gemm_fp4(q, q, sf[:256], sf, s, s)
    with pytest.raises(ValueError, match="M elements"):
        ops.gemm_fp4(q, q, sf, sf, s[:2], s)
    with pytest.raises(ValueError, match="1 or N"):
        ops.gemm_fp4(q, q, sf, sf, s, s[:2])
    with pytest.raises(ValueError, match="has K="):
        ops.gemm_fp4(q, q[:, :28], sf, sf, s, s)
    with pytest.raises(ValueError, match="bias"):
        ops.gemm_fp4(q, q, sf, sf, s, s, x[0, :3].contiguous())
    with pytest.raises(ValueError, match="out has shape"):
        ops.gemm_fp4(q, q, sf, sf, s, s, out=x)
    with pytest.raises(ValueError, match="multiple of 8"):
        ops.dequant_rows_fp4(q[:, :30], sf, s, "nvfp4")
    with pytest.raises(ValueError, match="past the"):
        ops.rms_mod_quant_fp4(x, x[:1], x[:1], rows_per_mod=2, kind="nvfp4")
    with pytest.raises(ValueError, match="same shape"):
        ops.swiglu_quant_fp4(x, x[:, :56], "nvfp4")
    w8 = ops.quant_rows_fp4(torch.ones(8, 64, dtype=torch.bfloat16, device=DEV), "nvfp4")
    res, gate = torch.ones(4, 8, dtype=torch.bfloat16, device=DEV), torch.ones(2, 8, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="past the 2 gate rows"):
        ops.gemm_fp4_gated(q, w8[0], sf, w8[1], s, w8[2], None, res, gate, rows_per_gate=1)
    with pytest.raises(ValueError, match="res has shape"):
        ops.gemm_fp4_gated(q, w8[0], sf, w8[1], s, w8[2], None, res[:2], gate, rows_per_gate=2)


@pytest.mark.parametrize("kind", KINDS)
def test_general_path_equals_compiled_one(kind, monkeypatch):
    """What the compiled call path launches, the general one launches too, bit for bit (another stream
    object, a row map, a wide rows-per-batch count take it anyway)."""
    class Declines:
        def __getattr__(self, name):
            return lambda *a: False

    g = gen(4)
    m, d, n = 70, 520, 264
    x, y = randn(g, m, d), randn(g, m, 2 * d)
    shift, scale = randn(g, 1, d), randn(g, 1, d)
    w = ops.quant_rows_fp4(randn(g, n, d, scale=0.02), kind)
    bias, res, gate = randn(g, n), randn(g, m, n), randn(g, 1, n)

    def calls(rows):
        q = ops.quant_rows_fp4(x, kind)
        out = [*q, *ops.rms_mod_quant_fp4(x, shift, scale, rows_per_mod=rows, kind=kind),
               *ops.swiglu_quant_fp4_fc1(y, kind), product(q, w, bias, kind), ops.dequant_rows_fp4(*q, kind),
               ops.gemm_fp4_gated(q[0], w[0], q[1], w[1], q[2], w[2], bias, res, gate, rows_per_gate=rows, kind=kind)]
        # scale tiles hold unwritten rows: compare row by row
        out[1], out[4], out[7] = (ops.fp4_scale_rows(t, m, d, kind) for t in (out[1], out[4], out[7]))
        return [t for t in out if t is not None]

    fast = calls(m)
    wide = calls((1 << 32) + 1)
    monkeypatch.setattr(ops, "_fp4_module", Declines())
    general = calls(m)
    for a, b, c in zip(fast, wide, general):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("kind", KINDS)
def test_offsets_past_2_31(kind):
    """Inputs and outputs of more than 2^31 elements: the last rows equal those of a call of their own."""
    g = gen(2)
    D, tail = 12288, 256
    S = (1 << 31) // D // 128 * 128 + 1024
    x = torch.empty(S, D, dtype=torch.bfloat16, device=DEV)
    x[-tail:] = randn(g, tail, D)
    x[:tail] = randn(g, tail, D)
    x[tail:-tail] = 1
    big, small = ops.quant_rows_fp4(x, kind), ops.quant_rows_fp4(x[-tail:].clone(), kind)
    assert torch.equal(big[0][-tail:], small[0])
    assert torch.equal(ops.fp4_scale_rows(big[1], S, D, kind)[-tail:], ops.fp4_scale_rows(small[1], tail, D, kind))
    del x
    val = ops.dequant_rows_fp4(*big, kind)
    assert torch.equal(val[-tail:], ops.dequant_rows_fp4(*small, kind))
    del val
    w = ops.quant_rows_fp4(randn(g, 16384, D, scale=0.02), kind)
    out = product(big, w, kind=kind)
    assert out.numel() > 1 << 31
    assert torch.equal(out[-tail:], product(small, w, kind=kind))

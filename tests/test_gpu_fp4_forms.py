"""Forms of the 4-bit operators in which tiles, scales and special values meet, bytes that are not theirs, and repeated calls."""
import pytest
import torch

from test_gpu_fp4 import check_operand
from thor_int8_gemm_b200 import _lib, ops

pytestmark = pytest.mark.gpu
KINDS = ("mxfp4", "nvfp4")
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert ops.device_status() == 0


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *s, scale=1.0):
    return (torch.randn(*s, generator=g, device=DEV) * scale).to(torch.bfloat16)


# ---------------------------------------------------------------- the same inputs, and the definition in 64 bits
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("op,m,n,k", [("swiglu", 77, 640, 2568), ("swiglu", 420, 64, 1552), ("norm", 300, 520, 1288),
                                      ("norm", 2100, 264, 1024), ("quant", 130, 200, 776)])
def test_repeats_whatever_ran_between(kind, op, m, n, k):
    """A quantiser and the product behind it give the same bits for the same inputs, whatever other inputs, and
    whatever freed memory their outputs land in, came between."""
    g = gen(m + k)
    w = ops.quant_rows_fp4(randn(g, n, k, scale=0.02), kind)
    shift, scale, res, gate = randn(g, 1, k, scale=0.1), randn(g, 1, k, scale=0.1), randn(g, m, n), randn(g, 1, n)
    inputs = [randn(g, m, 2 * k if op == "swiglu" else k) for _ in range(2)]

    def run(x):
        if op == "swiglu":
            a = ops.swiglu_quant_fp4_fc1(x, kind)
        elif op == "norm":
            a = ops.rms_mod_quant_fp4(x, shift, scale, rows_per_mod=m, kind=kind)
        else:
            a = ops.quant_rows_fp4(x, kind)
        return ops.gemm_fp4_gated(a[0], w[0], a[1], w[1], a[2], w[2], None, res, gate, rows_per_gate=m, kind=kind)

    first = [run(x) for x in inputs]
    for turn in range(12):
        soiled = [torch.full((size,), 37 * turn % 256, dtype=torch.uint8, device=DEV) for size in (512, 4096, 40000, 400000)]
        del soiled
        for x, want in zip(inputs, first):
            assert torch.equal(run(x), want)


@pytest.mark.parametrize("kind", KINDS)
def test_swiglu_codes_against_64_bits(kind):
    """The codes are those of act, and act is the float64 value rounded to bf16 but for what its float32
    evaluation adds: five roundings (exp, 1 + e, the division, g * s, the product with up) of 2^-24 each, below 2^-21, beside
    half a bf16 unit.  So a code that differs from the float64 value's belongs to an act that near the border between two
    bf16 values."""
    y = randn(gen(13), 300, 2 * 2568)
    act = ops.swiglu_quant_fc1(y, "int8", return_act=True)[2]
    check_operand(ops.swiglu_quant_fp4_fc1(y, kind), act.cpu(), kind)
    g, u = y.double().chunk(2, 1)
    exact = g / (1 + torch.exp(-g)) * u
    half_unit = torch.exp2(torch.floor(torch.log2(exact.abs().clamp(min=2.0 ** -126))) - 8)
    assert ((act.double() - exact).abs() <= half_unit + exact.abs() * 2.0 ** -21).all()


def value(op, kind):
    return ops.dequant_rows_fp4(*op, kind, out_dtype=torch.float32).double()


# ---------------------------------------------------------------- products of many tiles
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k,form", [(4921, 4112, 520, "rows"), (2305, 9229, 264, "one"), (4921, 4112, 8, "none")])
def test_many_tiles_in_every_output_type(kind, dtype, m, n, k, form):
    """340 and 370 output tiles over at most 74 CTA pairs: both accumulators and the columns that they share, a tile's first
    scales copied early (K of more than 256) and not, with row and weight scales, one weight scale, and the operands' own.

    Tolerance: K / 64 accumulation steps as in test_gpu_fp4.tolerance (a unit of the sum of magnitudes for each addition and
    each K = 64 sum), three float32 roundings of the scaled sum and of the sum with the bias (2^-24 each, below
    2^-22 of the larger), half a unit of the output type (half its smallest number where it is subnormal)."""
    g = gen(m + n + k)
    x, w = ops.quant_rows_fp4(randn(g, m, k), kind), ops.quant_rows_fp4(randn(g, n, k, scale=0.02), kind)
    xs, ws = x[2], w[2]
    xv, wv = value((x[0], x[1], None), kind), value((w[0], w[1], None), kind)
    if form != "none":
        xs = (torch.rand(m, generator=g, device=DEV) + 0.5) * (1 if xs is None else xs)
        ws = torch.rand(n if form == "rows" else 1, generator=g, device=DEV) + 0.5
        if w[2] is not None:   # nvfp4: near the scales that the weight was quantised with
            ws = ws * (w[2] if form == "rows" else w[2].median())
    bias = randn(g, n, scale=0.1).to(dtype)
    scale = 1.0
    if xs is not None:
        scale = scale * xs.double()[:, None]
    if ws is not None:
        scale = scale * ws.double()
    y = xv @ wv.t() * scale
    want = y + bias.double()
    fi = torch.finfo(dtype)
    tol = (xv.abs() @ wv.abs().t() * scale) * (2.0 ** -23 * (2 * -(-k // 64) + 2)) + torch.maximum(y.abs(), want.abs()) * 2.0 ** -22
    tol += want.abs() * (fi.eps / 2) + fi.tiny * fi.eps / 2
    first = None
    for _ in range(4):
        out = ops.gemm_fp4(x[0], w[0], x[1], w[1], xs, ws, bias, kind=kind, out_dtype=dtype)
        assert ((out.double() - want).abs() <= tol).all()
        first = out if first is None else first
        assert torch.equal(out, first)


# ---------------------------------------------------------------- rows without elements
def test_rows_without_elements_have_the_scale_of_zeros():
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    for call in (lambda s: lib.t8g_quant_rows_fp4(None, 0, None, 0, None, s, 300, 0, _lib.QUANT_NVFP4, stream),
                 lambda s: lib.t8g_rms_mod_quant_fp4(None, 0, None, None, None, 0, None, 300, 0, 1e-6, None, 0, None, s, 300, 0,
                                                     _lib.QUANT_NVFP4, stream),
                 lambda s: lib.t8g_swiglu_quant_fp4(None, None, 0, None, 0, None, s, 300, 0, _lib.QUANT_NVFP4, stream)):
        scale = torch.full((301,), 7.0, device=DEV)
        assert call(scale.data_ptr()) == 0
        assert (scale[:300] == 2.0 ** -100).all() and scale[300] == 7
    e = torch.empty(5, 0, dtype=torch.bfloat16, device=DEV)
    zeros = ops.quant_rows_fp4(torch.zeros(5, 16, dtype=torch.bfloat16, device=DEV), "nvfp4")[2]
    m = torch.empty(1, 0, dtype=torch.bfloat16, device=DEV)
    for q, sf, s in (ops.quant_rows_fp4(e, "nvfp4"), ops.swiglu_quant_fp4_fc1(e, "nvfp4"), ops.swiglu_quant_fp4(e, e, "nvfp4"),
                     ops.rms_mod_quant_fp4(e, m, m, rows_per_mod=5, kind="nvfp4")):
        assert q.shape == (5, 0) and sf.numel() == 0 and torch.equal(s, zeros)
        assert ops.dequant_rows_fp4(q, sf, s, "nvfp4").shape == (5, 0)
    assert ops.quant_rows_fp4(e, "mxfp4")[2] is None


# ---------------------------------------------------------------- special values behind a norm and a SwiGLU
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("s,d", [(60, 1536), (2060, 1536), (2100, 1024), (2052, 4096), (33, 264), (7, 8200)])
def test_norm_of_special_values(kind, s, d):
    """NaN and infinities in x and in the modulation, and h that is finite in float32 but past bf16's largest number (3.3895e38
    times a normalised 1, plus 1e36), in rows of the register kernel (2048 rows and more of 256 n) and of the others:
    the same operand as quantising the stored h."""
    g = gen(d + s)
    x, shift, scale = randn(g, s, d), randn(g, 4, d), randn(g, 4, d)
    idx = torch.randint(0, 2, (s,), generator=g, device=DEV, dtype=torch.int32)
    top = torch.finfo(torch.bfloat16).max
    x[1, 3], x[2, d - 1], x[s - 1, d // 2] = float("nan"), float("inf"), -float("inf")
    x[3] = 0
    x[4] = 1.0
    scale[2], shift[2] = top, 1e36
    idx[4] = 2
    scale[3, 5], shift[3, d - 9] = float("inf"), float("nan")
    idx[5] = idx[s - 2] = 3
    x[6] = torch.randn(d, generator=g, device=DEV).bfloat16() * 1e-38   # subnormal h under a multiplier of 1e-3
    kw = dict(mod_index=idx, scale_is_multiplier=True, eps=1e-6)
    h = ops.rms_mod_quant(x, shift, scale, kind="int8", return_h=True, **kw)[2]
    assert h[4].isinf().all() and h[[1, 2]].isnan().any(1).all()
    check_operand(ops.rms_mod_quant_fp4(x, shift, scale, kind=kind, **kw), h.cpu(), kind)
    w = randn(g, d)
    w[d - 2] = float("nan")
    kw["w"] = w
    h = ops.rms_mod_quant(x, shift, scale, kind="int8", return_h=True, **kw)[2]
    check_operand(ops.rms_mod_quant_fp4(x, shift, scale, kind=kind, **kw), h.cpu(), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,f", [(40, 136), (77, 2568), (900, 1536), (9, 24576)])
def test_swiglu_of_special_values(kind, m, f):
    """NaN and infinities in gate and up (-inf * 0 is NaN), act past bf16's largest number and act among its
    subnormals: the same operand as quantising the stored act."""
    y = randn(gen(m + f), m, 2 * f)
    y[1, 2], y[2, f + 1] = float("nan"), float("nan")
    y[3, f - 1], y[4, 0] = float("inf"), -float("inf")
    y[5, 2 * f - 1], y[m - 1, f + 5] = float("inf"), -float("inf")
    y[6, 7], y[6, f + 7] = 3e38, 3e38
    y[7, :f] = -88.0
    y[8, f:] = y[8, f:] * 1e-38
    act = ops.swiglu_quant_fc1(y, "int8", return_act=True)[2]
    check_operand(ops.swiglu_quant_fp4_fc1(y, kind), act.cpu(), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("s,form", [(2048, "batch"), (2304, "index"), (2049, "w")])
def test_norm_of_many_rows_of_1536(kind, s, form):
    g = gen(s)
    d, n_mod = 1536, 3 if s % 3 == 0 else 1
    x, shift, scale = randn(g, s, d), randn(g, n_mod, d), randn(g, n_mod, d)
    kw = {}
    if form == "index":
        kw["mod_index"] = torch.randint(0, n_mod, (s,), generator=g, device=DEV, dtype=torch.int32)
    if form == "w":
        kw["w"] = randn(g, d)
    h = ops.rms_mod_quant(x, shift, scale, kind="int8", return_h=True, **kw)[2]
    check_operand(ops.rms_mod_quant_fp4(x, shift, scale, kind=kind, **kw), h.cpu(), kind)


# ---------------------------------------------------------------- bytes that are not the call's
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("op,s,d", [("quant", 9, 136), ("quant", 129, 264), ("quant", 2500, 1024), ("norm", 35, 1288),
                                    ("norm", 2049, 1024), ("norm", 2100, 1536), ("swiglu", 77, 2568), ("swiglu", 161, 40)])
def test_other_bytes_stay(kind, op, s, d):
    """Through the C entry, into buffers that hold something: the bytes between a row's codes and the next row, the block scales
    of rows past the last (up to a multiple of 128) and what lies behind the buffers are left; the rest is the call's,
    whatever the pitch."""
    g = gen(s + d)
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    code = ops.FP4_CODE[kind]
    pitch, n_sf = -(-d // 32) * 16 + 48, ops.fp4_scale_bytes(s, d, kind)
    q = torch.full((s + 1, pitch), 0xA5, dtype=torch.uint8, device=DEV)
    sf = torch.full((n_sf + 512,), 0xA5, dtype=torch.uint8, device=DEV)
    qs = torch.full((s + 1,), 7.0, device=DEV)
    scale = qs.data_ptr() if kind == "nvfp4" else None
    to = (q.data_ptr(), pitch, sf.data_ptr(), scale, s, d, code, stream)
    big = randn(g, s, 2 * d + 24)
    if op == "quant":
        rc = lib.t8g_quant_rows_fp4(big.data_ptr(), big.stride(0), *to)
        want = ops.quant_rows_fp4(big[:, :d], kind)
    elif op == "norm":
        mod = randn(g, 2, d + 8)
        rc = lib.t8g_rms_mod_quant_fp4(big.data_ptr(), big.stride(0), None, mod[0].data_ptr(), mod[1].data_ptr(), d + 8, None, s, 0,
                                       1e-6, *to)
        want = ops.rms_mod_quant_fp4(big[:, :d], mod[:1, :d], mod[1:, :d], rows_per_mod=s, eps=1e-6, kind=kind)
    else:
        rc = lib.t8g_swiglu_quant_fp4(big.data_ptr(), big.data_ptr() + 2 * (d + 8), big.stride(0), *to)
        want = ops.swiglu_quant_fp4(big[:, :d], big[:, d + 8:2 * d + 8], kind)
    assert rc == 0, lib.t8g_last_error()
    assert torch.equal(q[:s, :d // 2], want[0])
    assert (q[:s, d // 2:] == 0xA5).all() and (q[s] == 0xA5).all() and (sf[n_sf:] == 0xA5).all()
    rows = sf[:n_sf].view(-(-s // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-s // 128) * 128, -1)
    assert (rows[s:] == 0xA5).all()
    blocks = -(-d // ops.FP4_BLOCK[kind])
    assert torch.equal(rows[:s, :blocks], ops.fp4_scale_rows(want[1], s, d, kind)) and (rows[:s, blocks:] == 0).all()
    if kind == "nvfp4":
        assert torch.equal(qs[:s], want[2]) and qs[s] == 7
    else:
        assert (qs == 7).all()


# ---------------------------------------------------------------- refusals
def test_no_modulation_row_is_refused():
    x, none = torch.ones(4, 64, dtype=torch.bfloat16, device=DEV), torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="split evenly over 0"):
        ops.rms_mod_quant_fp4(x, none, none)
    with pytest.raises(ValueError, match="past the 0"):
        ops.rms_mod_quant_fp4(x, none, none, rows_per_mod=4)
    with pytest.raises(_lib.T8GError, match="shift is null"):
        ops.rms_mod_quant_fp4(x, none, none, mod_index=torch.zeros(4, dtype=torch.int32, device=DEV))
    assert ops.rms_mod_quant_fp4(none, none, none)[0].shape == (0, 32)


# ---------------------------------------------------------------- the given stream
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", ["stream", "handle", "default"])
def test_outputs_belong_to_the_given_stream(kind, form):
    """A call on a given stream while the current one is far behind: a block that the current stream's work freed but has yet to
    write is not taken for its outputs, whichever call it is."""
    g = gen(21)
    m, n, k = 300, 264, 520
    x, y, one = randn(g, m, k), randn(g, m, 2 * k), randn(g, 1, k)
    w = ops.quant_rows_fp4(randn(g, n, k, scale=0.02), kind)
    res, gate, index = randn(g, m, n), randn(g, 1, n), torch.zeros(m, dtype=torch.int32, device=DEV)

    def calls(stream):
        q = ops.quant_rows_fp4(x, kind, stream=stream)
        h = ops.rms_mod_quant_fp4(x, one, one, rows_per_mod=m, kind=kind, stream=stream)
        hw = ops.rms_mod_quant_fp4(x, one, one, w=one[0], kind=kind, stream=stream)
        a = ops.swiglu_quant_fp4_fc1(y, kind, stream=stream)
        b = ops.swiglu_quant_fp4(y[:, :k], y[:, k:], kind, stream=stream)
        out = [ops.dequant_rows_fp4(*op, kind, stream=stream) for op in (q, h, hw, a, b)]
        out.append(ops.gemm_fp4(q[0], w[0], q[1], w[1], q[2], w[2], kind=kind, stream=stream))
        out += [ops.gemm_fp4_gated(q[0], w[0], q[1], w[1], q[2], w[2], None, res, gate, kind=kind, stream=stream, **kw)
                for kw in (dict(rows_per_gate=m), dict(gate_index=index))]
        return out

    want = calls(None)
    torch.cuda.synchronize()
    current = torch.cuda.Stream()
    side = torch.cuda.default_stream() if form == "default" else torch.cuda.Stream()
    given = {"stream": side, "handle": side.cuda_stream, "default": 0}[form]
    calls(given)
    torch.cuda.synchronize()
    with torch.cuda.stream(current):
        # every size of the outputs, freed while their writing still waits behind a sleep of the current stream
        sizes = [t.numel() * t.element_size() for t in want] + [m * k // 2, m * 272, m * 4, ops.fp4_scale_bytes(m, k, kind)]
        blocks = [torch.empty(size, dtype=torch.uint8, device=DEV) for size in sizes for _ in range(4)]
        torch.cuda._sleep(200_000_000)   # about 0.1 s
        for t in blocks:
            t.fill_(0xFF)
        del blocks, t
        late = torch.cuda.Event()
        late.record()
        got = calls(given)
    side.synchronize()
    assert not late.query()   # the calls ran while the current stream slept
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)

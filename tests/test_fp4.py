"""Microscaled 4-bit operators, what needs no GPU: the oracle, the layout, refusals, custom-op shapes."""
import ctypes
import sys

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from oracle import fp4 as F4
from thor_int8_gemm_b200 import _lib, dit, ops

KINDS = ("mxfp4", "nvfp4")
P = ctypes.c_void_p(4096)


def test_oracle_rounds_to_nearest_even_code():
    for i in range(7):
        mid = (F4.POINTS[i] + F4.POINTS[i + 1]) / 2
        code = F4._e2m1(np.array([mid, np.nextafter(mid, 0), np.nextafter(mid, 9)]))
        assert list(code) == [i if i % 2 == 0 else i + 1, i, i + 1]
    assert F4._e2m1(np.array([5.0, 6.0, 7.9])).tolist() == [6, 7, 7]
    bytes_ = F4._e4m3(F4.e4m3_value(np.arange(127)))
    assert np.array_equal(bytes_, np.arange(127))


@pytest.mark.parametrize("kind", KINDS)
def test_oracle_error_is_within_half_a_step(kind):
    """Every value is within half the distance of its neighbours' codes, or above 6 scales, where it
    saturates (mxfp4: up to 8; nvfp4: up to 6 * (1 + 2^-4) by the scale's rounding, more where the scale
    is subnormal, which these rows avoid)."""
    rng = np.random.default_rng(0)
    v = torch.from_numpy(rng.standard_normal((40, 160))).to(torch.bfloat16).double().numpy()
    code, byte, rs = F4.quant(v, kind)
    val = F4.value(code, byte, rs, kind)
    scale = F4.e8m0_value(byte) if kind == "mxfp4" else F4.e4m3_value(byte) * rs[:, None]
    wide = np.repeat(scale, F4.BLOCK[kind], 1)[:, :160]
    a = np.abs(v) / wide
    half = np.where(a < 2, 0.25, np.where(a < 4, 0.5, 1.0))
    top = 2.0 if kind == "mxfp4" else 6 / 16
    assert (np.abs(v - val) / wide <= np.where(a > 6, top, half) + 1e-12).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("s,d", [(1, 8), (128, 64), (129, 1288), (300, 3080)])
def test_scale_bytes_and_rows(kind, s, d):
    n = ops.fp4_scale_bytes(s, d, kind)
    assert n == _lib.load().t8g_fp4_scale_bytes(s, d, ops.FP4_CODE[kind])
    byte = np.random.default_rng(1).integers(0, 255, (s, -(-d // F4.BLOCK[kind])))
    tiled = F4.tile_scales(byte)
    assert tiled.size == n
    assert np.array_equal(ops.fp4_scale_rows(torch.from_numpy(tiled), s, d, kind).numpy(), byte)
    # byte of row r, block b of a 128 x 4 tile
    r, b = s - 1, byte.shape[1] - 1
    at = (r // 128 * -(-byte.shape[1] // 4) + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4
    assert tiled[at] == byte[r, b]


@pytest.mark.parametrize("kind", KINDS)
def test_scale_rows_of_nothing(kind):
    assert ops.fp4_scale_rows(torch.zeros(0, dtype=torch.uint8), 0, 64, kind).shape == (0, 64 // F4.BLOCK[kind])
    assert ops.fp4_scale_rows(torch.zeros(0, dtype=torch.uint8), 5, 0, kind).shape == (5, 0)


def test_scale_bytes_refuses():
    lib = _lib.load()
    assert lib.t8g_fp4_scale_bytes(-1, 64, 2) == -1 and lib.t8g_fp4_scale_bytes(1, 64, 0) == -1
    with pytest.raises(ValueError):
        ops.fp4_scale_bytes(-1, 64, "mxfp4")
    with pytest.raises(ValueError):
        ops.fp4_scale_bytes(1, 64, "int8")


def refused(rc, needle):
    msg = _lib.load().t8g_last_error().decode()
    assert rc in (_lib.T8G_ERR_INVALID_ARGUMENT, _lib.T8G_ERR_UNSUPPORTED) and needle in msg, (rc, msg)


@pytest.mark.parametrize("kw,needle", [
    (dict(D=12), "multiple of 8"), (dict(D=-8), "negative"), (dict(S=-1), "negative"), (dict(kind=1), "not a 4-bit"),
    (dict(D=49160), "exceeds"), (dict(S=1 << 40), "too many"), (dict(x=None), "x is null"),
    (dict(x=ctypes.c_void_p(4104)), "16-byte"), (dict(ld_x=64), "row stride"), (dict(ld_x=132), "row stride"),
    (dict(q=None), "null"), (dict(sf=None), "null"), (dict(q=ctypes.c_void_p(4104)), "16-byte"),
    (dict(sf=ctypes.c_void_p(4104)), "16-byte"), (dict(ld_q=48), "row stride"), (dict(ld_q=72), "row stride"),
    (dict(kind=3, scale=None), "q_scale is null"), (dict(kind=3, scale=ctypes.c_void_p(4098)), "4-byte"),
])
def test_quant_refuses(kw, needle):
    a = dict(x=P, ld_x=128, q=P, ld_q=64, sf=P, scale=P, S=4, D=128, kind=2)
    a.update(kw)
    refused(_lib.load().t8g_quant_rows_fp4(a["x"], a["ld_x"], a["q"], a["ld_q"], a["sf"], a["scale"], a["S"], a["D"],
                                           a["kind"], None), needle)


def test_other_rows_refuse():
    lib = _lib.load()
    rms = lambda **k: lib.t8g_rms_mod_quant_fp4(  # noqa: E731
        P, 128, k.get("w"), k.get("shift", P), k.get("scale", P), k.get("ld_mod", 128), k.get("index"), k.get("rpm", 4), 0,
        1e-6, P, 64, P, P, 4, 128, k.get("kind", 3), None)
    refused(rms(shift=None), "shift is null")
    refused(rms(scale=ctypes.c_void_p(8)), "scale must be")
    refused(rms(ld_mod=120), "row stride")
    refused(rms(rpm=0), "rows_per_mod")
    refused(rms(w=ctypes.c_void_p(8)), "w must be")
    refused(rms(index=ctypes.c_void_p(2)), "mod_index")
    refused(rms(kind=0), "not a 4-bit")
    refused(lib.t8g_swiglu_quant_fp4(P, P, 24584, P, 12304, P, P, 4, 24584, 3, None), "exceeds")
    refused(lib.t8g_swiglu_quant_fp4(P, ctypes.c_void_p(8), 128, P, 64, P, P, 4, 128, 3, None), "up must be")
    refused(lib.t8g_dequant_rows_fp4(P, 64, P, None, P, 5, 128, 4, 128, 3, None), "out_dtype")
    refused(lib.t8g_dequant_rows_fp4(P, 64, P, None, ctypes.c_void_p(8), 0, 128, 4, 128, 3, None), "16-byte")
    refused(lib.t8g_dequant_rows_fp4(P, 64, P, None, P, 0, 132, 4, 128, 3, None), "row stride")
    # nothing to do: no pointer is looked at
    assert lib.t8g_quant_rows_fp4(None, 0, None, 0, None, None, 0, 128, 2, None) == 0
    assert lib.t8g_swiglu_quant_fp4(None, None, 0, None, 0, None, None, 3, 0, 3, None) == 0


@pytest.mark.parametrize("kw,needle", [
    (dict(K=0), "bad sizes"), (dict(K=12), "bad sizes"), (dict(M=-1), "bad sizes"), (dict(N=1 << 31), "below"),
    (dict(kind=0), "not a 4-bit"), (dict(dt=3), "out_dtype"), (dict(out=None), "out is null"), (dict(x=None), "null"),
    (dict(x_sf=None), "null"), (dict(w_sf=ctypes.c_void_p(8)), "16-byte"), (dict(ld_x=120), "row stride"),
    (dict(ld_w=48), "row stride"), (dict(ws_n=2), "neither 1 nor N"), (dict(bias_n=3), "neither 0 nor N"),
    (dict(bias_n=128, bias=None), "bias"), (dict(ld_out=120), "smaller"), (dict(ld_out=132), "multiple of 16"),
    (dict(out=ctypes.c_void_p(8)), "16-byte"), (dict(xs=ctypes.c_void_p(2)), "4-byte"),
])
def test_gemm_refuses(kw, needle):
    a = dict(x=P, x_sf=P, xs=P, w=P, w_sf=P, ws=P, ws_n=128, bias=P, bias_n=0, out=P, dt=0, M=16, N=128, K=256, ld_x=128,
             ld_w=128, ld_out=128, kind=3)
    a.update(kw)
    refused(_lib.load().t8g_gemm_fp4(a["x"], a["x_sf"], a["xs"], a["w"], a["w_sf"], a["ws"], a["ws_n"], a["bias"],
                                     a["bias_n"], a["out"], a["dt"], a["M"], a["N"], a["K"], a["ld_x"], a["ld_w"],
                                     a["ld_out"], a["kind"], None), needle)


@pytest.mark.parametrize("kw,needle", [
    (dict(N=124, ld_out=128), "multiple of 8"), (dict(res=None), "null"), (dict(gate=None), "null"),
    (dict(rpg=0), "rows_per_gate"), (dict(ld_res=120), "strides"), (dict(ld_gate=132), "strides"),
    (dict(res=ctypes.c_void_p(4096 + 64)), "overlaps"), (dict(res=P, ld_res=136), "ld_out != ld_res"),
])
def test_gated_refuses(kw, needle):
    far = ctypes.c_void_p(1 << 30)
    a = dict(res=far, ld_res=128, gate=far, ld_gate=128, index=None, rpg=16, out=P, N=128, ld_out=128)
    a.update(kw)
    refused(_lib.load().t8g_gemm_fp4_gated(P, P, P, P, P, P, 1, None, 0, a["res"], a["ld_res"], a["gate"], a["ld_gate"],
                                           a["index"], a["rpg"], a["out"], 16, a["N"], 256, 128, 128, a["ld_out"], 3, None),
            needle)


def test_cpu_tensors_and_kinds_are_refused():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.quant_rows_fp4(x, "mxfp4")
    with pytest.raises(ValueError, match="4-bit"):
        ops.quant_rows_fp4(x, "int8")
    q = torch.zeros(4, 32, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.dequant_rows_fp4(q, torch.zeros(512, dtype=torch.uint8), None, "mxfp4")
    with pytest.raises(ValueError, match="CUDA"):
        ops.gemm_fp4(q, q, q.view(-1), q.view(-1), kind="mxfp4")
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.gemm_fp4(None, q, q.view(-1), q.view(-1), kind="mxfp4")
    with pytest.raises(TypeError, match="out_dtype"):
        ops.gemm_fp4(q, q, q.view(-1), q.view(-1), kind="mxfp4", out_dtype=torch.float64)
    with pytest.raises(ValueError, match="no 4-bit form"):
        dit.DiTBlock(64, 2, 64, kind="nvfp4", fused_mlp=True)


def test_compiled_call_path_declines():
    """Host tensors, objects that are no tensors, wrong types and shapes are left to the general path,
    without an exception left behind; a wrong number of arguments is an error."""
    F = ops._fp4_fast()
    q, sf, x = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), torch.zeros(4, 64)
    out = torch.zeros(4, 4, dtype=torch.bfloat16)
    assert F.gemm(q, q, sf, sf, None, None, None, out, torch.bfloat16, 0, 8, 2, None) is False
    assert F.gemm(q, None, 3, sf, None, None, None, out, torch.bfloat16, 0, 8, 2, None) is False
    assert F.gemm(q, q, sf, sf, None, None, None, out, torch.bfloat16, "0", 8, 2, None) is False
    assert F.gated(q, q, sf, sf, None, None, None, out, out, out, 4, 2, 0) is False
    assert F.dequant(q, sf, None, x, 2, 2, None) is False
    assert F.quant_rows(x, q, sf, None, 2, None) is False
    assert F.quant_rows("x", q, sf, None, 2, None) is False
    assert F.swiglu_fc1(x, q, sf, None, 2, None) is False
    assert F.rms_mod_quant(x, x, x, 4, 0, 1e-6, q, sf, None, 2, None) is False
    assert F.rms_mod_quant(x, x, x, 4, 0, "eps", q, sf, None, 2, None) is False
    for f in (F.gemm, F.gated, F.dequant, F.quant_rows, F.swiglu_fc1, F.rms_mod_quant, F.setup):
        with pytest.raises(TypeError):
            f(q)


def test_missing_call_path_leaves_the_general_one(monkeypatch):
    """Without the compiled call path (not built, or for another Python) the wrappers go on to the general path, which
    refuses host tensors here and launches on a GPU."""
    name = f"{ops.__package__}._t8g_fp4"
    monkeypatch.setattr(ops, "_fp4_module", None)
    monkeypatch.delattr(sys.modules[ops.__package__], "_t8g_fp4", raising=False)
    monkeypatch.setitem(sys.modules, name, None)   # the import statement raises ImportError
    x, q, sf = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    for call in (lambda: ops.quant_rows_fp4(x, "mxfp4"), lambda: ops.swiglu_quant_fp4_fc1(x, "nvfp4"),
                 lambda: ops.rms_mod_quant_fp4(x, x[:1], x[:1], rows_per_mod=4),
                 lambda: ops.dequant_rows_fp4(q, sf, None, "mxfp4"), lambda: ops.gemm_fp4(q, q, sf, sf, kind="mxfp4"),
                 lambda: ops.gemm_fp4_gated(q, q, sf, sf, None, None, None, x[:, :4], x[:1, :4], rows_per_gate=4)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("kind", KINDS)
def test_custom_ops_trace(kind):
    from thor_int8_gemm_b200 import torch_ops  # noqa: F401
    t = torch.ops.t8g

    def mlp(x, shift, scale, w1, w1_sf, w1_s, w2, w2_sf, w2_s, res, gate):
        q, sf, s = t.rms_mod_quant_fp4(x, shift, scale, None, None, x.shape[0], False, 1e-6, kind)
        y = t.gemm_fp4(q, w1, sf, w1_sf, s, w1_s, None, kind, torch.bfloat16)
        q, sf, s = t.swiglu_quant_fp4(y, kind)
        return t.gemm_fp4_gated(q, w2, sf, w2_sf, s, w2_s, None, res, gate, x.shape[0], kind)

    with FakeTensorMode():
        e = lambda *s, d=torch.bfloat16: torch.empty(s, dtype=d, device="cuda")  # noqa: E731
        u8, f32 = torch.uint8, torch.float32
        sb = lambda r, k: ops.fp4_scale_bytes(r, k, kind)  # noqa: E731
        args = (e(300, 520), e(1, 520), e(1, 520), e(1040, 260, d=u8), e(sb(1040, 520), d=u8), e(1040, d=f32),
                e(520, 260, d=u8), e(sb(520, 520), d=u8), e(520, d=f32), e(300, 520), e(1, 520))
        q, sf, s = t.quant_rows_fp4(args[0], kind)
        assert q.shape == (300, 260) and q.stride() == (272, 1) and sf.shape == (sb(300, 520),)
        assert s.shape == (300 if kind == "nvfp4" else 0,)
        out = t.gemm_fp4(q, args[3], sf, args[4], s, args[5], None, kind, torch.float32)
        assert out.shape == (300, 1040) and out.dtype == f32
        with pytest.raises(Exception):
            t.quant_rows_fp4(e(3, 12), kind)
    gm = make_fx(mlp, tracing_mode="fake")(*args)
    targets = [str(n.target) for n in gm.graph.nodes if n.op == "call_function"]
    for name in ("rms_mod_quant_fp4", "gemm_fp4", "swiglu_quant_fp4", "gemm_fp4_gated"):
        assert f"t8g.{name}.default" in targets

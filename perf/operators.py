"""The microscaled 4-bit operators: what is timed, in plain torch and through the framework.

Two formats of e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign) with a scale per block of a row:

    mxfp4   blocks of 32, scale a power of two (e8m0): 2^(floor(log2(max |x|)) - 2)
    nvfp4   blocks of 16, scale e4m3, and one float32 power of two 2^r per row, r the least with
            max |row| <= 6 * 448 * 2^r and r >= -100: block scale = e4m3(max |block| / (6 * 2^r))

An operand is (q, sf, q_scale): q holds two codes a byte (the even column in the low half), rows at a
pitch that is a multiple of 16 bytes; sf the block scales in tiles of 128 rows x 4 blocks, row r and
block b of a tile at byte (r % 32) * 16 + (r // 32) * 4 + b; q_scale [rows] float32 or None (mxfp4).

`op` is one of
    quant   quantise rows of bf16, and the values that the codes stand for
    linear  the product of two quantised matrices with a bias
    gated   that product as a gated residual: res + gate[batch element] * (x w^T + bias)
    norm    RMSNorm + modulation + quantisation, and the linear layer behind it (attention's input)
    swiglu  silu(gate) * up + quantisation, and the gated projection behind it (the end of an MLP)
"""
import importlib.util
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_EPS = 1e-6
_BLOCK = {"mxfp4": 32, "nvfp4": 16}
_OUT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    case = lambda name, op, kind, m, n, k, out="bf16", batch=1: dict(  # noqa: E731
        name=name, op=op, kind=kind, M=m, N=n, K=k, out=out, batch=batch)
    return [
        # one token's activations before a projection: latency
        case("quant_token", "quant", "nvfp4", 1, 0, 4096),
        # the activations of a 32768-token sample, hidden size of the DiT sweep
        case("quant_32768x3072", "quant", "mxfp4", 32768, 0, 3072),
        # a single token through a fused q/k/v projection: the weights are what is read
        case("linear_token_nv", "linear", "nvfp4", 1, 9216, 3072),
        # text tokens through a small projection, sizes that fill no tile, float32 out
        case("linear_ragged_f32", "linear", "mxfp4", 333, 1000, 2104, "f32"),
        # q/k/v projection of an image's tokens
        case("linear_8192_nv", "linear", "nvfp4", 8192, 9216, 3072),
        # the first MLP product of the 32768-token sample: the largest product of the sweep's block
        case("linear_32768_mx", "linear", "mxfp4", 32768, 24576, 3072),
        # a short sequence's output projection
        case("gated_64_mx", "gated", "mxfp4", 64, 1536, 4096, batch=2),
        # the second MLP product of the 32768-token sample, two batch elements
        case("gated_32768_nv", "gated", "nvfp4", 32768, 3072, 12288, batch=2),
        # a few hundred tokens of an odd hidden size, the last block of a row cut off
        case("norm_ragged_mx", "norm", "mxfp4", 1000, 520, 1288, batch=5),
        # the attention half's input: norm, modulation, q/k/v
        case("norm_8192_nv", "norm", "nvfp4", 8192, 9216, 3072, batch=2),
        # a short odd sequence's MLP end
        case("swiglu_ragged_nv", "swiglu", "nvfp4", 77, 640, 2568),
        # the MLP end of a 16384-token sample
        case("swiglu_16384_mx", "swiglu", "mxfp4", 16384, 3072, 12288, batch=2),
    ]


def draw(rng):
    op = rng.choice(("quant", "linear", "linear", "gated", "norm", "swiglu"))
    kind = rng.choice(("mxfp4", "nvfp4"))
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    m = log(1, 32768)
    n, k = log(64, 16384), 8 * log(16, 1536)
    if op in ("gated", "swiglu"):
        n -= n % 8
    m = min(m, 32768 * 24576 * 3072 // (n * k))  # no product beyond the largest listed one
    out = rng.choice(("bf16", "bf16", "f16", "f32")) if op == "linear" else "bf16"
    batch = rng.choice((1, 2, 3)) if op in ("gated", "norm", "swiglu") else 1
    return dict(op=op, kind=kind, M=-(-m // batch) * batch, N=0 if op == "quant" else n, K=k, out=out, batch=batch)


# ---------------------------------------------------------------- the formats in plain torch
def _two_to(e):
    """2^e in float32, exactly, for whole e from -127 to 127 (2^-127 is a subnormal number)."""
    return torch.where(e > -127, (e.int() + 127) << 23, torch.full_like(e.int(), 1 << 22)).view(torch.float32)


def _blocks(v, kind):
    b = _BLOCK[kind]
    return torch.nn.functional.pad(v, (0, -v.shape[1] % b)).view(v.shape[0], -1, b)


def _codes(v, kind):
    """bf16 values held in float32 [S, D] -> codes [S, D] (0..15), block scales as bytes and as values
    [S, blocks], row scale or None."""
    x = _blocks(v, kind)
    top = x.abs().amax(2)
    if kind == "mxfp4":
        rs = None
        scale_byte = (torch.frexp(top).exponent + (127 - 3)).clamp(0, 254)
        scale_byte = torch.where(top > 0, scale_byte, torch.zeros_like(scale_byte)).to(torch.uint8)
        scale = _two_to(scale_byte.int() - 127)
        y = x / scale[:, :, None]
    else:
        amax = top.amax(1)
        m, e = torch.frexp(amax)  # amax = m 2^e, 0.5 <= m < 1; 2688 = 0.65625 * 2^12
        r = torch.where(m <= 0.65625, e - 12, e - 11)
        r = torch.where(amax > 0, r, torch.full_like(r, -100)).clamp(min=-100)
        rs = _two_to(r)
        t = x / rs[:, None, None]
        f8 = (top / rs[:, None] / 6).to(torch.float8_e4m3fn)
        scale_byte, scale = f8.view(torch.uint8), f8.float()
        y = torch.where(scale[:, :, None] > 0, t / scale[:, :, None].clamp(min=2.0**-9), torch.zeros_like(t))
    a = y.abs().clamp(max=6)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | (y < 0).to(torch.uint8) << 3
    return code.view(v.shape[0], -1)[:, :v.shape[1]], scale_byte, scale, rs


def _values(code, scale, rs, kind):
    mag = (code & 7).float()
    a = torch.where(mag < 4, mag / 2, torch.where(mag < 6, mag - 2, 2 * mag - 8))
    a = torch.where(code > 7, -a, a)
    v = (_blocks(a, kind) * scale[:, :, None]).view(code.shape[0], -1)[:, :code.shape[1]]
    return v if rs is None else v * rs[:, None]


def _operand(v, kind):
    """bf16 values -> (q, sf, q_scale) as described above, K beside them."""
    code, scale_byte, _, rs = _codes(v.float(), kind)
    s, d = code.shape
    q = torch.zeros(s, -(-d // 32) * 16, dtype=torch.uint8, device=v.device)
    q[:, :d // 2] = code[:, 0::2] | code[:, 1::2] << 4
    p = torch.nn.functional.pad(scale_byte, (0, -scale_byte.shape[1] % 4, 0, -s % 128))
    sf = p.view(-1, 4, 32, p.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)
    return q[:, :d // 2], sf, rs, kind


def _unpack(operand):
    """(codes [S, D], block scale bytes [S, blocks], row scale) of an operand."""
    q, sf, rs, kind = operand
    s, d = q.shape[0], 2 * q.shape[1]
    code = torch.stack([q & 15, q >> 4], dim=2).view(s, d)
    nb = -(-d // _BLOCK[kind])
    byte = sf.view(-(-s // 128), -(-nb // 4), 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-s // 128) * 128, -1)
    return code, byte[:s, :nb], rs


def _decode(operand):
    code, byte, rs = _unpack(operand)
    if operand[3] == "mxfp4":
        scale = _two_to(byte.int() - 127)
    else:
        scale = byte.contiguous().view(torch.float8_e4m3fn).float()
    return _values(code, scale, rs, operand[3])


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    m, n, k, b = case["M"], case["N"], case["K"], case["batch"]
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    # activations: channels and tokens of different size, as behind a norm or an attention
    act = lambda r, c: (rand(r, c) * torch.exp(0.5 * rand(1, c)) * torch.exp(0.3 * rand(r, 1))).bfloat16()  # noqa: E731
    s = dict(case)
    if case["op"] == "quant":
        s["x"] = act(m, k)
        return s
    s["w"] = _operand((rand(n, k) * 0.02).bfloat16(), case["kind"])
    s["bias"] = (rand(n) * 0.1).to(_OUT[case["out"]])
    if case["op"] in ("linear", "gated"):
        s["x"] = _operand(act(m, k), case["kind"])
    if case["op"] in ("gated", "swiglu"):
        s["res"] = rand(m, n).bfloat16()
        s["gate"] = (0.5 * rand(b, n)).bfloat16()
    if case["op"] == "norm":
        s["x"] = act(m, k)
        s["shift"], s["scale"] = (0.1 * rand(b, k)).bfloat16(), (0.1 * rand(b, k)).bfloat16()
    if case["op"] == "swiglu":
        s["y"] = rand(m, 2 * k).bfloat16()  # the first product's output: gate and up halves
    return s


# ---------------------------------------------------------------- the operators
def _ops():
    if _ROOT not in sys.path:
        sys.path.insert(0, _ROOT)
    import __graft_entry__

    __graft_entry__.load_package()
    from thor_int8_gemm_b200 import ops

    return ops


def _rows_of(t, m):
    return t.repeat_interleave(m // t.shape[0], 0)


def _norm(s, dtype):
    x = s["x"].to(dtype)
    h = x * torch.rsqrt(x.square().mean(1, keepdim=True) + _EPS)
    mult = _rows_of((1 + s["scale"].float()).bfloat16().to(dtype), s["M"])
    return (h * mult + _rows_of(s["shift"].to(dtype), s["M"])).bfloat16()


def _swiglu(s, dtype):
    gate, up = s["y"][:, :s["K"]].to(dtype), s["y"][:, s["K"]:].to(dtype)
    return (gate / (1 + torch.exp(-gate)) * up).bfloat16()


def _product(s, x):
    y = x @ _decode(s["w"]).t() + s["bias"].float()
    if "res" in s:
        y = s["res"].float() + _rows_of(s["gate"].float(), s["M"]) * y
    return y.to(_OUT[s["out"]])


def run(s):
    op, kind = s["op"], s["kind"]
    if own:
        ops = _ops()
        if op == "quant":
            return ops.dequant_rows_fp4(*ops.quant_rows_fp4(s["x"], kind), kind)
        if op == "norm":
            x, x_sf, xs = ops.rms_mod_quant_fp4(s["x"], s["shift"], s["scale"], rows_per_mod=s["M"] // s["batch"],
                                                eps=_EPS, kind=kind)
        elif op == "swiglu":
            x, x_sf, xs = ops.swiglu_quant_fp4_fc1(s["y"], kind)
        else:
            x, x_sf, xs, _ = s["x"]
        w, w_sf, ws, _ = s["w"]
        if "res" in s:
            return ops.gemm_fp4_gated(x, w, x_sf, w_sf, xs, ws, s["bias"], s["res"], s["gate"],
                                      rows_per_gate=s["M"] // s["batch"], kind=kind)
        return ops.gemm_fp4(x, w, x_sf, w_sf, xs, ws, s["bias"], kind=kind, out_dtype=_OUT[s["out"]])
    if op == "quant":
        code, _, scale, rs = _codes(s["x"].float(), kind)
        return _values(code, scale, rs, kind).bfloat16()
    if op in ("linear", "gated"):
        return _product(s, _decode(s["x"]))
    h = _norm(s, torch.float32) if op == "norm" else _swiglu(s, torch.float32)
    code, _, scale, rs = _codes(h.float(), kind)
    return _product(s, _values(code, scale, rs, kind))


def work(case):
    m, n, k, kind = case["M"], case["N"], case["K"], case["kind"]
    operand = lambda rows: rows * (k / 2 + -(-k // _BLOCK[kind]) + (4 if kind == "nvfp4" else 0))  # noqa: E731
    if case["op"] == "quant":
        return {"bytes": 4.0 * m * k, "flops": 4.0 * m * k}
    out = 4 if case["out"] == "f32" else 2
    read = {"linear": operand(m), "gated": operand(m), "norm": 2.0 * m * k + 4.0 * case["batch"] * k, "swiglu": 4.0 * m * k}
    gated = 2.0 * (m + case["batch"]) * n if case["op"] in ("gated", "swiglu") else 0.0
    return {"bytes": read[case["op"]] + operand(n) + out * n + gated + float(out) * m * n, "flops": 2.0 * m * n * k}


# ---------------------------------------------------------------- the definition in 64 bits
def _power(e):
    """2^e in float64, exactly, for whole e from -1022 to 1023."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


_POINTS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_values(v, kind):
    """float64 [S, D] -> what its quantisation stands for, by comparison with the borders between values."""
    s, d = v.shape
    x = _blocks(v, kind)
    top = x.abs().amax(2)
    below = lambda t: torch.frexp(t).exponent - 1  # noqa: E731  floor(log2 t), t > 0
    if kind == "mxfp4":
        scale = _power((below(top.clamp(min=2.0**-140)) - 2).clamp(min=-127))
    else:
        amax = top.amax(1).clamp(min=2.0**-140)
        r = below(amax / 2688)
        r = (r + (amax > 2688 * _power(r)).int()).clamp(min=-100)
        rs = _power(r)
        want = top / (6 * rs[:, None])
        unit = _power(below(want.clamp(min=2.0**-20)).clamp(min=-6) - 3)
        scale = torch.round(want / unit) * unit * rs[:, None]
    a = x.abs() / torch.where(scale > 0, scale, torch.full_like(scale, 2.0**400))[:, :, None]
    point = torch.zeros_like(a)
    for i in range(7):  # a value midway between two goes to the one with the even code
        border = (_POINTS[i] + _POINTS[i + 1]) / 2
        point = torch.where(a > border if i % 2 == 0 else a >= border, _POINTS[i + 1], point)
    return (torch.sign(x) * point * scale[:, :, None]).view(s, -1)[:, :d]


def _exact_operand(operand):
    code, byte, rs = _unpack(operand)
    table = torch.tensor(_POINTS + tuple(-p for p in _POINTS), dtype=torch.float64, device=code.device)
    byte = byte.to(torch.float64)
    if operand[3] == "mxfp4":
        scale = _power(byte - 127)
    else:
        e, f = torch.floor(byte / 8), byte % 8
        scale = torch.where(e > 0, (1 + f / 8) * _power(e - 7), f * 2.0**-9) * rs.double()[:, None]
    wide = scale.repeat_interleave(_BLOCK[operand[3]], 1)[:, :code.shape[1]]
    return table[code.long()] * wide


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quant":
        return _exact_values(s["x"].double(), case["kind"])
    if case["op"] in ("linear", "gated"):
        x = _exact_operand(s["x"])
    else:
        h = _norm(s, torch.float64) if case["op"] == "norm" else _swiglu(s, torch.float64)
        x = _exact_values(h.double(), case["kind"])
    y = x @ _exact_operand(s["w"]).t() + s["bias"].double()
    if "res" in s:
        y = s["res"].double() + _rows_of(s["gate"].double(), s["M"]) * y
    return y

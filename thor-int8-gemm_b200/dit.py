"""A DiT block whose linear layers and norm/quant ops run on this library's kernels.

Shapes follow the synthetic DiT the workload describes (hidden 3072, 24 heads of 128,
SwiGLU FFN 12288, adaLN modulation from a [B, 6*hidden] conditioning vector); weights are
random-init N(0, 0.02) and quantised per output channel.  The data flow is the
reference's fused block (src/ck_fused_patch.py:152-172) with per-token quantisation:

    h1  = rms_norm(x) * (1 + scale_msa) + shift_msa     -> int8/fp8 + per-token scale
    qkv = h1 @ Wqkv^T (fused dequant GEMM)               -> SDPA (torch, outside the hot path)
    o   = quant(attn) @ Wproj^T;  x += gate_msa * o       (gated residual: stock torch, or
                                                          the GEMM's epilogue, fused_gate)
    h2  = rms_norm(x) * (1 + scale_mlp) + shift_mlp     -> int8/fp8 + per-token scale
    y   = h2 @ Wfc1^T  [M, 2F];  a = quant(silu(y[:, :F]) * y[:, F:]) (read in place)
    z   = a @ Wfc2^T;  x += gate_mlp * z

kind is "int8", "fp8_e4m3", or a microscaled 4-bit format ("mxfp4", "nvfp4": weights and
activations both in it), for which the same operators have their _fp4 forms.

Tokens are laid out batch-major ([B*T, hidden]); `tokens_per_batch` maps every token to
its batch element's modulation row.  Multi-GPU runs shard the token dimension (see
`shard.py`): weights and conditioning are replicated and no collective is needed.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import ops


class QuantLinear:
    """A linear layer with a per-output-channel quantised weight [N, K]."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, kind: str = "int8"):
        if weight.dtype != torch.bfloat16:
            weight = weight.to(torch.bfloat16)
        self.kind = kind
        self.w, self.ws = ops.quant_rows(weight.contiguous(), kind)
        self.bias = None if bias is None else bias.to(torch.bfloat16).contiguous()
        self.out_features, self.in_features = weight.shape

    def __call__(self, xq: torch.Tensor, xs: torch.Tensor, out: torch.Tensor | None = None, stream=None):
        return ops.gemm_dequant(xq, self.w, xs, self.ws, self.bias, out=out, stream=stream)

    def gated(self, operand, res, gate, rows_per_gate: int, out: torch.Tensor | None = None):
        """res + gate * linear(operand), the gated residual in the GEMM's epilogue."""
        xq, xs = operand
        return ops.gemm_gated(xq, self.w, xs, self.ws, self.bias, res, gate, rows_per_gate=rows_per_gate, out=out)


class Fp4Linear:
    """A linear layer with a microscaled 4-bit weight [N, K]; takes a 4-bit activation (q, sf, q_scale)."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, kind: str = "nvfp4"):
        self.kind = kind
        self.w, self.w_sf, self.ws = ops.quant_rows_fp4(weight.to(torch.bfloat16).contiguous(), kind)
        self.bias = None if bias is None else bias.to(torch.bfloat16).contiguous()
        self.out_features, self.in_features = weight.shape

    def __call__(self, x: torch.Tensor, x_sf: torch.Tensor, x_scale: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, stream=None):
        return ops.gemm_fp4(x, self.w, x_sf, self.w_sf, x_scale, self.ws, self.bias, kind=self.kind, out=out,
                            stream=stream)

    def gated(self, operand, res, gate, rows_per_gate: int, out: torch.Tensor | None = None):
        """res + gate * linear(operand), the gated residual in the product's epilogue."""
        x, x_sf, x_scale = operand
        return ops.gemm_fp4_gated(x, self.w, x_sf, self.w_sf, x_scale, self.ws, self.bias, res, gate,
                                  rows_per_gate=rows_per_gate, kind=self.kind, out=out)


class DiTBlock:
    """Synthetic DiT block (see module docstring)."""

    def __init__(self, hidden: int = 3072, heads: int = 24, ffn: int = 12288, kind: str = "int8",
                 device=None, seed: int = 0, eps: float = 1e-6, fused_mlp: bool = False,
                 fused_gate: bool = False):
        if hidden % heads:
            raise ValueError("hidden must be a multiple of heads")
        self.fp4 = kind in ops.FP4_CODE
        if self.fp4 and fused_mlp:
            raise ValueError("fused_mlp (SwiGLU in fc1's epilogue) has no 4-bit form")
        self.hidden, self.heads, self.ffn, self.kind, self.eps = hidden, heads, ffn, kind, eps
        device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def w(n, k):
            return (torch.randn(n, k, generator=g, device=device) * 0.02).to(torch.bfloat16)

        def b(n):
            return (torch.randn(n, generator=g, device=device) * 0.01).to(torch.bfloat16)

        linear = Fp4Linear if self.fp4 else QuantLinear
        self.qkv = linear(w(3 * hidden, hidden), b(3 * hidden), kind)
        self.proj = linear(w(hidden, hidden), b(hidden), kind)
        self.fc1 = linear(w(2 * ffn, hidden), b(2 * ffn), kind)
        self.fc2 = linear(w(hidden, ffn), b(hidden), kind)
        # fused_mlp: fc1 with the SwiGLU in its epilogue (gate / up rows interleaved once), which
        # also reports each row's max |act| so that act is quantised as a plain stream
        self.fused_mlp = fused_mlp
        # fused_gate: proj and fc2 apply the gated residual in their epilogue (gemm_gated, or
        # gemm_fp4_gated, which rounds once where the other keeps torch's three bf16 roundings)
        self.fused_gate = fused_gate
        if fused_mlp:
            il = ops.interleave_gate_up
            self.fc1_il = (il(self.fc1.w), il(self.fc1.ws), il(self.fc1.bias))

    def modulation(self, cond: torch.Tensor):
        """Split the conditioning [B, 6*hidden] into shift/scale/gate for attention and MLP."""
        return [c.contiguous() for c in cond.to(torch.bfloat16).chunk(6, dim=-1)]

    def norm_quant(self, x, shift, scale, tokens_per_batch):
        if self.fp4:
            return ops.rms_mod_quant_fp4(x, shift, scale, rows_per_mod=tokens_per_batch, eps=self.eps, kind=self.kind)
        return ops.rms_mod_quant(x, shift, scale, rows_per_mod=tokens_per_batch, eps=self.eps, kind=self.kind)

    def attention(self, qkv: torch.Tensor, batch: int) -> torch.Tensor:
        M = qkv.shape[0]
        T = M // batch
        hd = self.hidden // self.heads
        q, k, v = qkv.view(batch, T, 3, self.heads, hd).permute(2, 0, 3, 1, 4)
        o = F.scaled_dot_product_attention(q, k, v)
        return o.transpose(1, 2).reshape(M, self.hidden)

    @staticmethod
    def gated(x, gate, y, batch):
        """x + gate[b] * y per batch element (the stock gated residual)."""
        M, H = x.shape
        return (x.view(batch, M // batch, H) + gate.view(batch, 1, H) * y.view(batch, M // batch, H)).view(M, H)

    def linears_and_norms(self, x, cond, batch, attn_fn=None):
        """The block with a pluggable attention (default: torch SDPA); returns the new x."""
        T = x.shape[0] // batch
        shift_msa, scale_msa, gate_msa, shift_mlp, scale_mlp, gate_mlp = self.modulation(cond)
        # a quantised activation is the tuple that its linear layer takes: (q, scale) or (q, sf, scale)
        qkv = self.qkv(*self.norm_quant(x, shift_msa, scale_msa, T))
        attn = (attn_fn or self.attention)(qkv, batch)
        # the quantiser takes row-strided input; only a non-unit inner stride needs a copy
        quant = ops.quant_rows_fp4 if self.fp4 else ops.quant_rows
        a = quant(attn if attn.stride(-1) == 1 else attn.contiguous(), self.kind)
        if self.fused_gate:
            x = self.proj.gated(a, x, gate_msa, T)
        else:
            x = self.gated(x, gate_msa, self.proj(*a), batch)
        h2 = self.norm_quant(x, shift_mlp, scale_mlp, T)
        if self.fused_mlp:
            w_il, ws_il, b_il = self.fc1_il
            a = ops.gemm_swiglu_quant(h2[0], w_il, h2[1], ws_il, b_il, kind=self.kind)[:2]
        elif self.fp4:
            a = ops.swiglu_quant_fp4_fc1(self.fc1(*h2), self.kind)
        else:
            a = ops.swiglu_quant_fc1(self.fc1(*h2), kind=self.kind)
        if self.fused_gate:
            # x is this block's own tensor here: update it in place
            return self.fc2.gated(a, x, gate_mlp, T, out=x)
        return self.gated(x, gate_mlp, self.fc2(*a), batch)

    def __call__(self, x: torch.Tensor, cond: torch.Tensor, batch: int) -> torch.Tensor:
        return self.linears_and_norms(x, cond, batch)

    def linear_ops(self, M: int) -> float:
        """Integer/float ops of the four GEMMs for M tokens (2*M*N*K each)."""
        h, f = self.hidden, self.ffn
        return 2.0 * M * (3 * h * h + h * h + 2 * f * h + h * f)

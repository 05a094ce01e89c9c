"""The dense shared expert of a sparse layer, beside the routed path.

Every sparse layer of the model adds a shared expert that all rows pass through:
``hidden + routed_moe + shared_mlp`` (python/reference/glmrt_reference/glm_moe_dsa_layer_ref.py:157-206),
with ``shared_mlp = expert_forward(normalized, shared weights)`` (moe_ref.py:17-21): the same
gate / up / SwiGLU / down arithmetic as a routed expert, but dense -- float32 math on the stored
weights, no activation quantisation -- and run by the coordinator, not by the expert workers
(``docs/balanced-path.md:53-66`` times it as "shared MLP" next to routing and dispatch).

It is three dense products over all rows.  With weights kept in float32 or bf16 they go to the
library GEMM (cuBLAS through ``torch.matmul``; float32 accumulation) with the SwiGLU between them;
with weights in 8-bit floating point (a scale for each block of 128) they run on this library's own
kernels (``fp8.py``).  The result enters the routed layer's combine as the shared delta (``MoeLayer.forward_residual``), where
``out = bf16(residual + bf16(shared + routed))`` is formed in one pass
(native/cuda/kernels/residual.cu:36-62).  Nothing here touches the routed experts' kernels.
"""
from __future__ import annotations

import torch

from . import fp8
from .block_norm import block_norm


class DenseSharedExpert:
    """Shared-expert weights resident on the current device: gate/up ``[I, H]``, down ``[H, I]``.

    ``dtype``: ``torch.float32`` reproduces the reference's float32 arithmetic exactly as stated
    (weights up-cast once at load, TF32 off); ``torch.bfloat16`` keeps the weights as stored and
    lets the GEMMs accumulate in float32 (outputs of the first two GEMMs are rounded to bf16);
    ``torch.float8_e4m3fn`` quantises the weights once at load (128 x 128 blocks) and the rows in each
    call (``fp8.gated_mlp``), a quarter of the float32 form's bytes.
    """

    def __init__(self, gate_proj: torch.Tensor, up_proj: torch.Tensor, down_proj: torch.Tensor,
                 dtype: torch.dtype = torch.float32):
        assert gate_proj.shape == up_proj.shape and down_proj.shape == gate_proj.shape[::-1]
        dev = torch.device("cuda", torch.cuda.current_device())
        self.dtype = dtype
        self.inter = gate_proj.shape[0]
        if dtype == fp8.E4M3:
            self.gate, self.up, self.down = (fp8.quantize_weight(w.to(dev)) for w in (gate_proj, up_proj, down_proj))
            return
        self.gate_up = torch.cat([gate_proj, up_proj], dim=0).to(dev, dtype).contiguous()   # [2I, H]: one GEMM for both
        self.down = down_proj.to(dev, dtype).contiguous()

    def delta(self, normalized_bf16: torch.Tensor) -> torch.Tensor:
        """bf16 ``expert_forward(normalized)`` rows: what the layer adds as ``shared_mlp``."""
        assert normalized_bf16.dtype == torch.bfloat16 and normalized_bf16.is_cuda
        if self.dtype == fp8.E4M3:
            return fp8.gated_mlp(normalized_bf16, *self.gate, *self.up, *self.down)
        prev = torch.backends.cuda.matmul.allow_tf32
        torch.backends.cuda.matmul.allow_tf32 = False
        try:
            x = normalized_bf16.to(self.dtype)
            gu = (x @ self.gate_up.T).float()
            g, u = gu[:, :self.inter], gu[:, self.inter:]
            act = torch.nn.functional.silu(g) * u
            y = act.to(self.dtype) @ self.down.T
        finally:
            torch.backends.cuda.matmul.allow_tf32 = prev
        return y.to(torch.bfloat16)


def sparse_layer_forward(routed_layer, shared: DenseSharedExpert, residual_bf16: torch.Tensor,
                         normalized_bf16: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``residual + routed_moe(normalized) + shared_mlp(normalized)`` with the two additions folded into
    the routed layer's combine (glm_moe_dsa_layer_ref.py:190-198)."""
    return routed_layer.forward_residual(normalized_bf16, residual_bf16, shared.delta(normalized_bf16), out)


class SparseBlock:
    """A whole sparse layer after its attention: ``forward(residual, attention_delta)`` adds the delta to the
    residual stream and normalises it (``block_norm``), runs the shared expert and the routed experts on the
    normalised rows, and returns the new residual stream (glm_moe_dsa_layer_ref.py:157-206).

    Batches of at most ``few_rows`` rows (default: as many as it takes, 16) go through ``MoeLayer.forward_few`` (bf16
    activations in the experts), larger ones through ``forward_residual`` (NVFP4 activations); 0 keeps all on the latter.
    The default is for accuracy: of the layer 6144 / 2048 with 256 experts the former is the faster one up to 4 rows (1 row
    48 against 57 us, 4 rows 130 / 134), even at 5 and slower above (8 rows 240 / 212, 16 rows 445 / 340).
    """

    def __init__(self, routed_layer, shared: DenseSharedExpert, norm_weight: torch.Tensor, eps: float = 1e-5,
                 few_rows: int | None = None):
        self.routed, self.shared, self.eps = routed_layer, shared, eps
        self.norm_weight = norm_weight.to(routed_layer.device).contiguous()
        self.few_rows = routed_layer.FEW_MAX_ROWS if few_rows is None else few_rows
        if not 0 <= self.few_rows <= routed_layer.FEW_MAX_ROWS:
            raise ValueError(f"few_rows must be 0..{routed_layer.FEW_MAX_ROWS}")

    def forward(self, residual_bf16: torch.Tensor, attention_delta_bf16: torch.Tensor | None = None) -> torch.Tensor:
        residual, rows = block_norm(residual_bf16, attention_delta_bf16, norm_weight=self.norm_weight, eps=self.eps)
        if rows.shape[0] == 0:
            return residual
        shared = self.shared.delta(rows)
        if rows.shape[0] <= self.few_rows:
            return self.routed.forward_few(rows, residual_bf16=residual, shared_delta_bf16=shared)
        return self.routed.forward_residual(rows, residual, shared)

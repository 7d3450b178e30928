"""MI355X-native (gfx950) Cheby-RKV hot path of OrthoSSM.

Fused softsign -> Clenshaw -> per-head damping -> tanh -> per-head EMA scan,
with dynamic lambda, EMA carry across chunks, bf16 I/O, the fused TTT
coefficient gradient, the backward and the full online-TTT path,
implemented as hand-written HIP kernels behind the C ABI of
``include/osm.h`` (library ``orthossm_amd/_lib/libosm.so``); the engine's
call sites in ``orthossm_amd.engine``.

For layers that learn at test time with a matrix-valued state: the gated delta
rule (chunked forward and backward, one-token step), layer norm and gradient
clipping, and ``GatedDeltaLayer``, which runs them together.
"""
from .ops import cheby_ema, cheby_ema_backward, cheby_ema_forward, cheby_ema_ttt
from .sdpc_kernel import apply_cheby_rkv_core, apply_cheby_rkv_v10
from .engine import ChebyContextPath, ChebyState
from .delta import gated_delta, gated_delta_backward, gated_delta_forward, gated_delta_step
from .norm import layer_norm, layer_norm_backward, layer_norm_forward
from .grad_clip import clip_grad_norm, grad_norm
from .delta_layer import GatedDeltaLayer

__all__ = ["cheby_ema", "cheby_ema_forward", "cheby_ema_backward", "cheby_ema_ttt", "apply_cheby_rkv_v10",
           "apply_cheby_rkv_core", "ChebyContextPath", "ChebyState", "gated_delta", "gated_delta_forward",
           "gated_delta_backward", "gated_delta_step", "layer_norm", "layer_norm_forward", "layer_norm_backward",
           "clip_grad_norm", "grad_norm", "GatedDeltaLayer"]

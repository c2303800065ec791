"""``mamba_ssm.ops.triton.layer_norm`` import path (the names that mixer_seq_simple.py:24 and mamba_simplemotif.py:26 import), served
by the gfx950 HIP kernels. Despite the module path, nothing here is Triton."""
from motif_mamba_amd.layer_norm import RMSNorm, layer_norm_fn, rms_norm_fn

__all__ = ["RMSNorm", "layer_norm_fn", "rms_norm_fn"]

"""motif_mamba_amd -- MI355X (gfx950) selective-scan hot path of Motif-Mamba.

Public API (drop-in for the reference's):
  selective_scan_fn, SelectiveScanFn   (mamba_ssm/ops/selective_scan_interface.py:24-61, 237-259)
  SelectiveScanPQFn                    (selective_scan_interface.py:93-150, forward; with z too)
  selective_state_update               (upstream mamba_ssm.ops.triton.selective_state_update)
  causal_conv1d_fn, causal_conv1d_update (package causal-conv1d, mamba_simplemotif.py:16-19)
  mamba_inner_fn, MambaInnerFn         (selective_scan_interface.py:454-656)

Layers whose state decays by one scalar per head and step (no counterpart in the reference):
  linear_attention_fn, linear_attention_update, group_norm_fn, and LinearAttentionBlock, which runs them together

Layers whose state is corrected under each key as well (no counterpart in the reference):
  delta_rule_fn, delta_rule_update, and GatedDeltaBlock, which runs them with the norms and the conv

The norm at a layer's entry:
  layer_norm_fn, rms_norm_fn, RMSNorm  (un-vendored mamba_ssm.ops.triton.layer_norm, mixer_seq_simple.py:24)
"""
from .selective_scan import SelectiveScanFn, SelectiveScanPQFn, selective_scan_fn
from .causal_conv1d import causal_conv1d_fn, causal_conv1d_update
from .state_update import selective_state_update
from .mamba_inner import MambaInnerFn, mamba_inner_fn
from .linear_attention import LinearAttentionFn, linear_attention_fn, linear_attention_update
from .group_norm import GroupNormFn, group_norm_fn
from .linear_block import LinearAttentionBlock
from .delta_rule import DeltaRuleFn, delta_rule_fn, delta_rule_update
from .layer_norm import LayerNormFn, RMSNorm, layer_norm_fn, rms_norm_fn
from .delta_block import GatedDeltaBlock

__all__ = ["SelectiveScanFn", "SelectiveScanPQFn", "selective_scan_fn", "selective_state_update",
           "causal_conv1d_fn", "causal_conv1d_update", "MambaInnerFn", "mamba_inner_fn",
           "LinearAttentionFn", "linear_attention_fn", "linear_attention_update", "GroupNormFn", "group_norm_fn",
           "LinearAttentionBlock", "DeltaRuleFn", "delta_rule_fn", "delta_rule_update", "LayerNormFn", "layer_norm_fn",
           "rms_norm_fn", "RMSNorm", "GatedDeltaBlock"]

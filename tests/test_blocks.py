"""CPU checks of the layers that run this package's operators together: what they are built with, no kernel is launched."""
import pytest
import torch


@pytest.mark.parametrize("default", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("block", ["GatedDeltaBlock", "LinearAttentionBlock"])
def test_the_cached_state_is_float32(block, default):
    """Single tokens take and give a float32 state, which a model built under another default dtype has too."""
    import motif_mamba_amd
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        m = getattr(motif_mamba_amd, block)(32, nheads=2, headdim=16, d_state=8, dtype=default)
        conv, state = m.allocate_inference_cache(3)
    finally:
        torch.set_default_dtype(before)
    assert state.dtype == torch.float32 and state.shape == (3, 2, 8, 16) and not state.any()
    assert conv.dtype == default and not conv.any()

"""Buffers of the modules around the latent cache under casts of the model that holds them (CPU)."""
import pytest
import torch

FREQ = (1.0 / 10000.0 ** (torch.arange(32, dtype=torch.float64) / 32)).float()


@pytest.mark.parametrize("cast", ["bfloat16", "half", "double"])
def test_frequencies_keep_their_32_bits(cast):
    from dsa_triton_ascend_b200 import LatentCacheAppend, RotaryEmbedding
    m = torch.nn.ModuleList([RotaryEmbedding(FREQ), LatentCacheAppend(FREQ, norm_weight=torch.rand(512)),
                             LatentCacheAppend(FREQ), torch.nn.Linear(2, 2)])
    weight = m[1].norm_weight.clone()
    getattr(m, cast)()
    for part in m[:3]:
        assert part.inv_freq.dtype == torch.float32 and torch.equal(part.inv_freq, FREQ)
    assert torch.equal(m[1].norm_weight, weight) and m[2].norm_weight is None
    assert m[3].weight.dtype != torch.float32
    m.float()
    assert torch.equal(m[0].inv_freq, FREQ) and torch.equal(m[1].norm_weight, weight)


def test_weights_in_the_latents_type_follow_a_cast():
    from dsa_triton_ascend_b200 import LatentCacheAppend
    m = LatentCacheAppend(FREQ, norm_weight=torch.rand(512).bfloat16())
    assert m.half().norm_weight.dtype == torch.float16 and m.inv_freq.dtype == torch.float32


def test_buffers_follow_the_device():
    from dsa_triton_ascend_b200 import RotaryEmbedding
    m = RotaryEmbedding(FREQ).to(device="meta", dtype=torch.bfloat16)
    assert m.inv_freq.is_meta and m.inv_freq.dtype == torch.float32
    assert "inv_freq" in dict(m.named_buffers()) and not m.state_dict()

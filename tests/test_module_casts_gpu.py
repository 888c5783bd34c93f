"""Modules that were cast with their model compute what they were made for."""
import pytest
import torch

from tests.latent_ref import inv_freq, paged

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_rotary_after_a_cast(dtype):
    from dsa_triton_ascend_b200 import RotaryEmbedding, rotary_embedding
    x = torch.randn(2, 5, 3, 64, device="cuda").to(DT[dtype])
    pos = torch.randint(0, 100000, (2, 5), device="cuda")
    m = torch.nn.Sequential(RotaryEmbedding(inv_freq(device="cpu"))).to(device="cuda", dtype=DT[dtype])
    assert torch.equal(m[0](x, pos), rotary_embedding(x, pos, inv_freq()))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("norm", ["io", "fp32", "other"])
def test_append_after_a_cast(dtype, norm):
    from dsa_triton_ascend_b200 import LatentCacheAppend, latent_cache_append
    dt = DT[dtype]
    table, blocks = paged(torch.Generator(device="cuda").manual_seed(2), [20], 16)
    x, r = torch.randn(1, 3, 1, 512, device="cuda").to(dt), torch.randn(1, 3, 1, 64, device="cuda").to(dt)
    a, b = ([torch.zeros(blocks, 16, 1, w, device="cuda", dtype=dt) for w in (512, 64)] for _ in range(2))
    w = (1 + 0.1 * torch.randn(512)).to({"io": dt, "fp32": torch.float32, "other": DT["fp16" if dtype == "bf16" else "bf16"]}[norm])
    m = torch.nn.Sequential(LatentCacheAppend(inv_freq(device="cpu"), norm_weight=w)).to(dt).cuda()
    m[0](x, r, *a, block_table=table, actual_seq_lengths_kv=[20])
    w = w if norm == "fp32" else w.to(dt)
    latent_cache_append(x, r, *b, inv_freq(), block_table=table, actual_seq_lengths_kv=[20], norm_weight=w.cuda())
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and int(a[0].count_nonzero()) > 1400

"""rotary_embedding on inputs without elements that claim any strides."""
import pytest
import torch

from tests.latent_ref import inv_freq

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(0, 3, 64), (4, 0, 64)])
def test_nothing_to_rotate_with_strides_of_zero(shape):
    """Such a tensor counts as contiguous whatever its strides are."""
    from dsa_triton_ascend_b200 import rotary_embedding, rotary_embedding_grad
    x = torch.ones((), device="cuda").expand(shape)
    pos = torch.zeros(shape[0], dtype=torch.int32, device="cuda")
    for f in (rotary_embedding, rotary_embedding_grad):
        y = f(x, pos, inv_freq(), layout="TND")
        assert y.shape == shape and y.stride(-1) == 1

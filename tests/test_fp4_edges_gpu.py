"""fp4_ds_mla attention where it can go wrong: queries whose parts differ in size by
many orders of magnitude, against 64 bits."""

import pytest
import torch

from tests import fp4_ref as R
from tests.test_fp4_gpu import MANY, SCALE, check_sparse, ints, make_pool, randn, sparse_case, status_clean
from vllm_fp8kv import fp4_ds_mla as F

pytestmark = pytest.mark.gpu


def both(q, pool, idx, want, scale):
    """The call by itself and, from 33 heads on, enough copies of it for the kernel of
    many heads."""
    check_sparse(q, pool, idx, want, scale)
    if q.shape[1] > 32:
        T = 80
        assert F.fp4_kernel_name(q.shape[1], 1, T, idx.shape[2]) == MANY


@pytest.mark.parametrize("H", [16, 128])
@pytest.mark.parametrize("latent,rope", [(-100, 0), (-100, 20), (-60, 60), (-126, -20), (-30, 90)])
def test_tiny_latent_part_beside_a_rope(H, latent, rope):
    """The latents' power of two must not carry the rope's products out of fp32's
    range: q latents of 2^latent, q ropes of 2^rope, cached ropes of up to 2^36,
    a scale that makes the scores ordinary."""
    pool = R.quantize(randn(201, 300, 512), (randn(202, 300, 64).double() * 2.0 ** 36).to(torch.bfloat16))
    q, idx = sparse_case(203, 5, H, 200, 300, mask=0.1)
    q = torch.cat([q[..., :512].double() * 2.0 ** latent, q[..., 512:].double() * 2.0 ** rope], 2).to(torch.bfloat16)
    q[1, 0] = randn(204, 576)  # an ordinary head among them: its scores are next to 0
    scale = SCALE * 2.0 ** (-36 - rope)
    both(q, pool, idx, R.attend(q, pool, idx, scale), scale)
    status_clean()


@pytest.mark.parametrize("H", [16, 128])
@pytest.mark.parametrize("latent", [-120, -40, -14, 12, 100])
def test_latents_decide_beside_cached_ropes_of_zero(H, latent):
    """Latents far smaller than q's rope keep their bits where the cached ropes are
    zero: the score is theirs alone."""
    pool = R.quantize(randn(205, 300, 512), torch.zeros(300, 64, dtype=torch.bfloat16, device="cuda"))
    q, idx = sparse_case(206, 5, H, 200, 300, mask=0.1)
    q = torch.cat([q[..., :512].double() * 2.0 ** latent, q[..., 512:].double()], 2).to(torch.bfloat16)
    scale = SCALE * 2.0 ** -latent
    both(q, pool, idx, R.attend(q, pool, idx, scale), scale)
    status_clean()

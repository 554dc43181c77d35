"""fp4_ds_mla attention where it can go wrong: queries whose parts differ in size by
many orders of magnitude, and calls that take long, against 64 bits."""

import pytest
import torch

from tests import fp4_ref as R
from tests.test_fp4_gpu import MANY, SCALE, check_sparse, dense_slots, ints, make_pool, randn, sparse_case, status_clean
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


@pytest.mark.parametrize("H", [16, 128])
def test_calls_longer_than_the_wait_limit(H):
    """A wait gives up after less than 0.4 s; a call may take longer without one that
    does.  One token's q and one page table serve all rows (stride 0, the same 64
    pages again and again), so that the call is long and its inputs small."""
    page, times, own = 64, 64, 64
    pool = make_pool(210, page * own)
    table = torch.randperm(own, device="cuda").to(torch.int32).repeat(times).view(1, -1)
    n = page * own * times  # 262144 positions, each row of the pool `times` times
    T = 8192 if H == 128 else 20000
    q = randn(211, 1, H, 576).expand(T, H, 576)
    req = torch.zeros(T, dtype=torch.int32, device="cuda")
    lens = torch.full((T,), n, dtype=torch.int32, device="cuda")
    lens[1::7] = n - 1000
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    out, lse = F.fp4_ds_mla_decode(q, pool, req, table, lens, SCALE, block_size=page, return_lse=True)
    b.record()
    status_clean()
    assert a.elapsed_time(b) > 450  # ms: else this shows nothing
    slots = dense_slots(table, req[:2], lens[:2], page)
    want = R.attend(q[:2], pool, slots, SCALE)
    for t in (0, T // 2 // 7 * 7, (T - 2) // 7 * 7):
        R.check((out[t:t + 1], lse[t:t + 1]), [w[:1] for w in want])
        R.check((out[t + 1:t + 2], lse[t + 1:t + 2]), [w[1:] for w in want])


@pytest.mark.parametrize("H", [1, 16, 40, 128])
@pytest.mark.parametrize("T", [3, 64, 150, 400])
def test_dense_short_contexts(H, T):
    """Contexts of one or two chunks, by themselves and beside a longer one: fewer
    chunks a worker than pieces of a cut unit have."""
    pool = make_pool(220, 3200)
    table = torch.randperm(50, device="cuda")[:40].to(torch.int32).view(4, 10)
    q = randn(221, T, H, 576)
    req = (torch.arange(T, device="cuda") % 4).to(torch.int32)
    rows = torch.arange(T, device="cuda")
    for most, long in ((64, 64), (130, 130), (64, 600)):
        lens = ints(222 + most, most + 1, (T,)).to(torch.int32)
        lens[T // 2] = long
        got = F.fp4_ds_mla_decode(q, pool, req, table, lens, SCALE, return_lse=True)
        R.check(got, R.attend(q, pool, dense_slots(table[req.long()], rows, lens, 64), SCALE))
        tight = table[:, :(most + 63) // 64].contiguous()  # (the longest row the table holds is short, too)
        if long == most:
            again = F.fp4_ds_mla_decode(q, pool, req, tight, lens, SCALE, return_lse=True)
            R.check(again, R.attend(q, pool, dense_slots(table[req.long()], rows, lens, 64), SCALE))
    status_clean()

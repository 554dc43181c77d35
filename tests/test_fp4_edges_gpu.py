"""fp4_ds_mla attention where it can go wrong: queries whose parts differ in size by
many orders of magnitude, special values, lengths around the borders of a chunk in both
kernels, and calls that take long, against 64 bits."""

import pytest
import torch

from tests import fp4_ref as R
from tests.test_fp4_gpu import MANY, SCALE, check_sparse, dense_slots, ints, make_pool, randn, sparse_case, status_clean
from vllm_fp8kv import fp4_ds_mla as F

pytestmark = pytest.mark.gpu

FEW = "decode_fp4_kernel"


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


def copies(kernel, q, topk, times=400):
    """How many copies of q's rows a call needs to go to `kernel`."""
    T, H, _ = q.shape
    for r in range(1, times):
        if F.fp4_kernel_name(H, 1, T * r, topk) == kernel:
            return r
    raise AssertionError(f"no call of {H} heads and top-{topk} goes to {kernel}")


@pytest.mark.parametrize("H", [1, 16, 17, 32, 33, 48, 64, 65, 128, 130])
@pytest.mark.parametrize("topk", [1, 63, 64, 65, 127, 128, 129, 192, 193, 500])
def test_every_length_in_every_kernel(H, topk):
    """Around the borders of a chunk of either kernel: all head counts in the kernel
    of few heads, those above 32 in the other one too, where it is chosen at all."""
    pool = make_pool(230, 900)
    q, idx = sparse_case(231 + topk, 3, H, topk, 900, mask=0.2)
    idx[1, :, -1] = -1
    idx[2, :, 0] = -1
    want = R.attend(q, pool, idx, SCALE)
    for kernel in (FEW, MANY) if H >= 64 or (H > 32 and topk > 64) else (FEW,):
        r = copies(kernel, q, topk)
        out, lse = F.fp4_ds_mla_sparse_decode(q.repeat(r, 1, 1), pool, idx.repeat(r, 1, 1), SCALE, return_lse=True)
        for i in {0, r // 2, r - 1}:
            R.check((out[3 * i:3 * i + 3], lse[3 * i:3 * i + 3]), want)
    status_clean()


@pytest.mark.parametrize("kernel,H", [("few", 16), ("few", 40), ("many", 64), ("many", 128)])
@pytest.mark.parametrize("topk", [100, 700])
def test_special_values_in_attended_rows(kernel, H, topk):
    """NaN scales, NaN ropes and infinite scores show in the rows (and heads) that
    attend to them and in no other; an entry whose score is -inf weighs nothing."""
    kernel = FEW if kernel == "few" else MANY
    pool = make_pool(240, 800)
    q, _ = sparse_case(241, 6, H, topk, 800)
    q[..., 512] = q[..., 512].abs() + 0.5
    pool[790, 256 + 31] = 0x7F                                     # the last group of the latents
    pool[791, 288:290] = torch.tensor([0xC0, 0x7F], device="cuda")  # rope: NaN
    pool[792, 288:290] = torch.tensor([0x80, 0x7F], device="cuda")  # +inf
    pool[793, 288:290] = torch.tensor([0x80, 0xFF], device="cuda")  # -inf
    idx = ints(242, 780, (6, 1, topk)).to(torch.int32)
    for t, at in ((1, 790), (2, 791), (3, 792), (4, 793)):
        idx[t, 0, topk - 7 * t] = at
    masked = idx.clone()
    masked[4, 0, topk - 28] = -1
    r = copies(kernel, q, topk)
    out, lse = F.fp4_ds_mla_sparse_decode(q.repeat(r, 1, 1), pool, idx.repeat(r, 1, 1), SCALE, return_lse=True)
    clean = [0, 4, 5]
    want = [w[clean] for w in R.attend(q, pool, torch.where(masked >= 790, -1, masked), SCALE)]
    for i in {0, r // 2, r - 1}:
        o, l = out[6 * i:6 * i + 6], lse[6 * i:6 * i + 6]
        assert o[1:4].isnan().all() and l[1:4].isnan().all()
        R.check((o[clean], l[clean]), want)
    nothing = torch.full_like(idx[:1], 793)  # scores of -inf alone: as nothing to attend
    rows = q[5:].repeat(6 * r, 1, 1)
    out, lse = F.fp4_ds_mla_sparse_decode(rows, pool, nothing.repeat(6 * r, 1, 1), SCALE, return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    status_clean()

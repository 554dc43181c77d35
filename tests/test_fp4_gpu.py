"""fp4_ds_mla on the GPU: writer, read-back and attention against 64-bit references."""

import pytest
import torch

from tests import fp4_ref as R
from vllm_fp8kv import _native as N
from vllm_fp8kv import fp4_ds_mla as F
from vllm_fp8kv.cache_writer import concat_and_cache_mla

pytestmark = pytest.mark.gpu

SCALE = 192 ** -0.5
MANY = "decode_fp4_tc_kernel"


def randn(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def make_pool(seed, slots):
    return R.quantize(randn(seed, slots, 512), randn(seed + 1, slots, 64))


def ints(seed, hi, shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(0, hi, shape, generator=g, device="cuda")


def status_clean():
    torch.cuda.synchronize()
    assert N.device_status() == 0


# ------------------------------------------------------------------ writer
def write(kv_c, k_pe, slots, num_slots):
    pool = torch.full((num_slots, 416), 0xA5, dtype=torch.uint8, device="cuda")
    F.concat_and_cache_fp4_ds_mla(kv_c, k_pe, pool, slots)
    return pool


@pytest.mark.parametrize("n", [1, 7, 8, 9, 1000, 5003])
def test_writer_bytes(n):
    kv_c, k_pe = randn(n, n, 512), randn(n + 1, n, 64)
    slots = torch.randperm(2 * n + 3, device="cuda")[:n]
    slots[::5] = -1
    if n > 2:
        slots[2] = 2 * n + 3  # behind the pool: skipped
    pool = write(kv_c, k_pe, slots, 2 * n + 3)
    want = torch.full_like(pool, 0xA5)
    kept = (slots >= 0) & (slots < 2 * n + 3)
    want[slots[kept]] = R.quantize(kv_c, k_pe)[kept]
    assert torch.equal(pool, want)  # other rows are left as they were


def test_writer_bytes_over_the_whole_range():
    """Every power of two a bf16 has, groups from all zeros to overflow."""
    e = torch.arange(-133, 128, device="cuda").double()
    g = randn(3, 261 * 32, 16).double() * (2.0 ** e).repeat_interleave(32)[:, None]
    g = g.clamp(-3.3e38, 3.3e38).to(torch.bfloat16)
    g[::9] = 0.0
    g[1::9, 3] = -0.0
    kv_c = g.view(-1, 512)
    k_pe = randn(4, kv_c.shape[0], 64)
    slots = torch.arange(len(kv_c), device="cuda")
    assert torch.equal(write(kv_c, k_pe, slots, len(kv_c)), R.quantize(kv_c, k_pe))


def test_writer_borders_of_codes_and_scales():
    """Values exactly on a rounding border of their code, amaxes exactly on one of
    their scale."""
    scales = torch.arange(1, 127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], dtype=torch.float64, device="cuda")
    g = torch.cat([scales[:, None] * ties, -scales[:, None] * ties], 1)     # amax = 6 * scale
    mid = 6 * (scales[1:] + scales[:-1]) / 2
    h = torch.zeros(len(mid), 16, dtype=torch.float64, device="cuda")
    h[:, 0], h[:, 1], h[:, 2] = mid, -mid / 2, mid / 8
    g = torch.cat([g, h])
    g = torch.cat([g, torch.zeros(-len(g) % 32, 16, dtype=torch.float64, device="cuda")])
    kv_c = g.to(torch.bfloat16)
    assert torch.equal(kv_c[:len(scales)].double(), g[:len(scales)])  # the borders are bf16 values
    kv_c = kv_c.view(-1, 512)
    k_pe = randn(5, kv_c.shape[0], 64)
    slots = torch.arange(len(kv_c), device="cuda")
    assert torch.equal(write(kv_c, k_pe, slots, len(kv_c)), R.quantize(kv_c, k_pe))


def test_writer_special_values():
    kv_c, k_pe = randn(6, 4, 512), randn(7, 4, 64)
    kv_c[0, 5], kv_c[0, 20], kv_c[1, 500] = float("nan"), float("inf"), float("-inf")
    kv_c[2, 33], kv_c[2, 34] = float("inf"), float("nan")
    k_pe[3, 0], k_pe[3, 1] = float("nan"), float("inf")
    slots = torch.arange(4, device="cuda")
    pool, want = write(kv_c, k_pe, slots, 4), R.quantize(kv_c, k_pe)
    assert torch.equal(pool[:, 256:], want[:, 256:])
    codes = want[:, 256:288] != 127  # the codes of a NaN group say nothing
    same = (pool[:, :256] == want[:, :256]).view(4, 32, 8).all(2)
    assert same[codes].all()
    back = F.dequant_fp4_ds_mla_rows(pool, slots).double()
    assert back[0, :16].isnan().all() and back[2, 32:48].isnan().all()
    assert back[0, 20] == 2688 and back[1, 500] == -2688


def test_writer_strides_alignment_and_dtype_route():
    base = randn(8, 50, 1300)
    slots = torch.arange(50, device="cuda")
    for at in (0, 1, 8):  # 2-byte aligned views take the scalar loads
        kv_c, k_pe = base[:, at:at + 512], base[:, 600 + at:664 + at]
        pool = torch.zeros(5, 10, 416, dtype=torch.uint8, device="cuda")
        concat_and_cache_mla(kv_c, k_pe, pool, slots, "fp4_ds_mla")
        assert torch.equal(pool.view(-1, 416), R.quantize(kv_c.contiguous(), k_pe))
    pool = torch.zeros(4, 416, dtype=torch.uint8, device="cuda")
    F.concat_and_cache_fp4_ds_mla(base[:0, :512], base[:0, :64], pool, slots[:0])
    assert not pool.any()


# ------------------------------------------------------------------ read-back
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("n", [0, 1, 31, 4097])
def test_rows(n, dtype):
    pool = make_pool(10, 700)
    slots = ints(11, 720, (n,)).to(dtype) - 10  # some in front of the pool, some behind
    got = F.dequant_fp4_ds_mla_rows(pool, slots)
    ok = (slots >= 0) & (slots < 700)
    want = R.values(pool)[slots.clamp(0, 699).long()] * ok[:, None]
    assert torch.equal(got.double(), want)


def test_every_code_and_scale_reads_back():
    pool = make_pool(12, 256)
    pool[:, :256] = torch.arange(256, device="cuda")[None, :]
    pool[:, 256:288] = torch.arange(256, device="cuda")[:, None]
    got = F.dequant_fp4_ds_mla_rows(pool, torch.arange(256, device="cuda"))
    want = R.values(pool)
    assert torch.equal(got.double().nan_to_num(1e9), want.nan_to_num(1e9))


def test_rows_into_a_strided_output():
    pool = make_pool(13, 64)
    big = torch.full((33, 592), 7.0, dtype=torch.bfloat16, device="cuda")
    F.dequant_fp4_ds_mla_rows(pool, torch.arange(32, device="cuda"), out=big[:32, 8:584])
    assert torch.equal(big[:32, 8:584].double(), R.values(pool)[:32])
    assert (big[:, :8] == 7).all() and (big[:, 584:] == 7).all() and (big[32] == 7).all()


def gather_want(pool, table, lens, starts, page):
    rows = []
    for b, n in enumerate(lens):
        p = torch.arange(n, device="cuda") + starts[b]
        ok = p // page < table.shape[1]
        pg = table[b].long()[(p // page).clamp(max=table.shape[1] - 1)]
        s = pg * page + p % page
        ok &= (s >= 0) & (s < len(pool))
        rows.append(R.values(pool)[s.clamp(0, len(pool) - 1)] * ok[:, None])
    return torch.cat(rows) if rows else torch.zeros(0, 576, dtype=torch.float64, device="cuda")


@pytest.mark.parametrize("page", [1, 16, 64, 100])
@pytest.mark.parametrize("lens", [[1], [0, 0, 5, 0, 64, 65, 0], [130, 1, 0, 257], [0, 0]])
def test_gather(lens, page):
    pool = make_pool(20, 1000)
    B = len(lens)
    table = (ints(21, 1100 // page, (B, 300 // page + 1)) - 3 // page).to(torch.int32)  # some pages outside
    starts = ints(22, 90, (B,)).to(torch.int32)
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    got = F.gather_fp4_ds_mla(pool, table, cu, sum(lens), block_size=page, seq_starts=starts)
    assert torch.equal(got.double(), gather_want(pool, table, lens, starts.tolist(), page))


@pytest.mark.parametrize("B", [31, 32, 33, 1025, 2500])
def test_gather_many_sequences(B):
    pool = make_pool(23, 512)
    lens = [(7 * b) % 5 for b in range(B)]
    table = ints(24, 32, (B, 1)).to(torch.int32)
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    got = F.gather_fp4_ds_mla(pool, table, cu, sum(lens), block_size=16)
    req = torch.arange(B, device="cuda").repeat_interleave(torch.tensor(lens, device="cuda"))
    pos = torch.arange(sum(lens), device="cuda") - cu.long()[req]
    assert torch.equal(got.double(), R.values(pool)[table[req, 0].long() * 16 + pos])


def test_gather_leaves_the_other_rows():
    pool = make_pool(25, 64)
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    out = torch.full((20, 576), 3.0, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([2, 5, 9], dtype=torch.int32, device="cuda")
    F.gather_fp4_ds_mla(pool, table, cu, 20, out=out)
    want = R.values(pool)
    assert torch.equal(out[2:5].double(), want[:3]) and torch.equal(out[5:9].double(), want[:4])
    assert (out[:2] == 3).all() and (out[9:] == 3).all()
    F.gather_fp4_ds_mla(pool, table[:0], cu[:1], 20, out=out)  # no sequences
    assert (out[9:] == 3).all()


# ------------------------------------------------------------------ attention
def sparse_case(seed, T, H, topk, slots, G=1, mask=0.0):
    idx = ints(seed, slots, (T, G, topk)).to(torch.int32)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 5)
    idx[torch.rand(T, G, topk, generator=g, device="cuda") < mask] = -1
    return randn(seed + 2, T, H, 576), idx


def check_sparse(q, pool, idx, want, scale=SCALE):
    """The call by itself and, where that does not take the kernel of many heads,
    its rows repeated until it does."""
    (T, H), (G, topk) = q.shape[:2], idx.shape[1:]
    R.check(F.fp4_ds_mla_sparse_decode(q, pool, idx, scale, return_lse=True), want)
    if F.fp4_kernel_name(H, G, T, topk) == MANY:
        return
    for reps in (16, 64, 256):
        if F.fp4_kernel_name(H, G, T * reps, topk) == MANY:
            out, lse = F.fp4_ds_mla_sparse_decode(q.repeat(reps, 1, 1), pool, idx.repeat(reps, 1, 1), scale,
                                                  return_lse=True)
            for i in range(0, reps, 5):
                R.check((out[i * T:i * T + T], lse[i * T:i * T + T]), want)
            return


@pytest.mark.parametrize("H", [1, 3, 8, 16, 17, 24, 32, 40, 64, 65, 96, 128, 130, 256])
@pytest.mark.parametrize("topk", [1, 63, 64, 65, 500])
def test_sparse_heads_and_lengths(H, topk):
    pool = make_pool(30, 900)
    q, idx = sparse_case(31 + topk, 3, H, topk, 900, mask=0.2)
    want = R.attend(q, pool, idx, SCALE)
    R.check(F.fp4_ds_mla_sparse_decode(q, pool, idx[:, 0], SCALE, return_lse=True), want)
    check_sparse(q, pool, idx, want)
    status_clean()


@pytest.mark.parametrize("H,T,topk", [(16, 1, 4096), (16, 300, 130), (128, 1, 4096), (128, 90, 200), (64, 40, 333),
                                      (48, 5, 2048), (128, 75, 1024)])
def test_sparse_division_of_work(H, T, topk):
    """One unit over many SMs, many units per SM, units cut at odd places."""
    pool = make_pool(32, 5000)
    q, idx = sparse_case(33, T, H, topk, 5000, mask=0.05)
    got = F.fp4_ds_mla_sparse_decode(q, pool, idx, SCALE, return_lse=True)
    R.check(got, R.attend(q, pool, idx, SCALE))
    status_clean()


@pytest.mark.parametrize("H,G", [(16, 2), (32, 2), (128, 2), (256, 2), (192, 3)])
def test_sparse_groups(H, G):
    pool = make_pool(34, 400)
    q, idx = sparse_case(35, 4, H, 150, 400, G=G, mask=0.3)
    check_sparse(q, pool, idx, R.attend(q, pool, idx, SCALE, G))


@pytest.mark.parametrize("H", [16, 128])
def test_sparse_masks(H):
    """Rows without a live entry, live entries only at the ends, indices outside
    the pool, and masked slots whose rows hold NaN."""
    pool = make_pool(36, 300)
    pool[0, 256:288] = 0x7F   # NaN scales in the row a masked group may fetch
    pool[0, 288:416] = 0xFF   # and a NaN rope
    q, idx = sparse_case(37, 8, H, 333, 299)
    idx += 1                   # never row 0
    idx[0] = -1
    idx[1, :, 1:] = -1
    idx[2, :, :-1] = -1
    idx[3, :, ::2] = 300
    idx[4, :, 64:128] = 2 ** 31 - 1
    idx[5, :, :256] = -(2 ** 31)
    idx[6, :, 3::4] = -1
    idx = torch.where(idx == 300, 100000, idx)
    check_sparse(q, pool, idx, R.attend(q, pool, idx, SCALE))


@pytest.mark.parametrize("H", [16, 128])
def test_nothing_to_attend(H):
    q = randn(38, 3, H, 576)
    pool = make_pool(39, 64)
    for p, idx in ((pool, torch.zeros(3, 0, dtype=torch.int32, device="cuda")),
                   (pool[:0], torch.zeros(3, 100, dtype=torch.int32, device="cuda"))):
        out, lse = F.fp4_ds_mla_sparse_decode(q, p, idx, SCALE, return_lse=True)
        assert (out == 0).all() and torch.isneginf(lse).all()
    table = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    req = torch.arange(3, dtype=torch.int32, device="cuda")
    for lens in ([0, 0, 0], [5, -3, 1]):  # an empty table holds no position
        out, lse = F.fp4_ds_mla_decode(q, pool, req, table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                       SCALE, return_lse=True)
        assert (out == 0).all() and torch.isneginf(lse).all()
    out = F.fp4_ds_mla_sparse_decode(q[:0], pool, idx[:0], SCALE)
    assert out.shape == (0, H, 512)
    status_clean()


@pytest.mark.parametrize("H", [16, 128])
def test_scores_of_any_size(H):
    """Rising maxima chunk after chunk, and per-head q sizes from 1e-30 to 1e30
    of which each head's own power of two takes account."""
    pool = make_pool(40, 2000)
    q = randn(41, 2, H, 576)
    ramp = torch.linspace(0.05, 4.0, 2000, device="cuda")[:, None]
    pool = R.quantize((randn(42, 2000, 512).float() * ramp).to(torch.bfloat16), randn(43, 2000, 64))
    idx = torch.arange(2000, dtype=torch.int32, device="cuda").expand(2, 1, 2000)
    check_sparse(q, pool, idx, R.attend(q, pool, idx, SCALE))
    size = 10.0 ** torch.linspace(-30, 30, H, device="cuda")
    q2 = (q.float() * size[:, None]).to(torch.bfloat16)
    # heads one at a time, each with the scale that makes its scores ordinary
    if H > 32:  # enough rows for the kernel of many heads
        q2, idx = q2.repeat(8, 1, 1), idx.repeat(8, 1, 1)
        assert F.fp4_kernel_name(H, 1, 16, 2000) == MANY
    for h in range(0, H, max(1, H // 8)):
        sc = SCALE / float(size[h])
        got = F.fp4_ds_mla_sparse_decode(q2, pool, idx, sc, return_lse=True)
        want = R.attend(q2[:, h:h + 1], pool, idx, sc)
        R.check((got[0][:, h:h + 1], got[1][:, h:h + 1]), want)


@pytest.mark.parametrize("H", [16, 128])
@pytest.mark.parametrize("size", [30.0, 1e-3])
def test_peaked_and_flat_rows(H, size):
    """Scores of hundreds, where one entry takes nearly all the weight and the others'
    lies below what P can hold, and scores that are nearly the same."""
    pool = make_pool(48, 900)
    q, idx = sparse_case(49, 9, H, 700, 900, mask=0.1)
    q = q * size
    check_sparse(q, pool, idx, R.attend(q, pool, idx, SCALE))


@pytest.mark.parametrize("H", [16, 128])
@pytest.mark.parametrize("scale", [-0.07, 0.0, -0.0])
def test_softmax_scale_of_any_sign(H, scale):
    """A negative scale turns the order of the scores round; with 0 all live
    entries weigh the same.  Masked entries stay out either way."""
    pool = make_pool(46, 500)
    q, idx = sparse_case(47, 3, H, 321, 500, mask=0.3)
    idx[1] = -1
    check_sparse(q, pool, idx, R.attend(q, pool, idx, scale), scale)


@pytest.mark.parametrize("H", [16, 128])
def test_nan_in_an_attended_row_shows(H):
    pool = make_pool(44, 200)
    pool[17, 256] = 0x7F
    q, _ = sparse_case(45, 2, H, 100, 200)
    idx = torch.arange(100, dtype=torch.int32, device="cuda").repeat(2, 1)
    idx[1, 17] = 150
    out, lse = F.fp4_ds_mla_sparse_decode(q, pool, idx, SCALE, return_lse=True)
    assert out[0].isnan().all() and lse[0].isnan().all()
    want = R.attend(q[1:], pool, idx[1:, None], SCALE)
    R.check((out[1:], lse[1:]), want)
    if H > 32:
        assert F.fp4_kernel_name(H, 1, 128, 100) == MANY
        out, lse = F.fp4_ds_mla_sparse_decode(q.repeat(64, 1, 1), pool, idx.repeat(64, 1), SCALE, return_lse=True)
        assert out[::2].isnan().all() and lse[::2].isnan().all()
        R.check((out[1:2], lse[1:2]), want)
        R.check((out[127:], lse[127:]), want)


def paged_slots(table, req, tok, page, max_blocks):
    blk = tok.long() // page
    ok = (tok >= 0) & (blk < max_blocks)
    s = table.long()[req.long()[:, None, None], blk.clamp(0, max_blocks - 1)] * page + tok.long() % page
    return torch.where(ok, s, -1)


@pytest.mark.parametrize("H", [16, 128])
@pytest.mark.parametrize("page", [1, 16, 64, 100])
def test_paged(H, page):
    pool = make_pool(50, 1600)
    blocks = 400 // page
    table = (ints(51, 1700 // page, (4, blocks + 2))).to(torch.int32)[:, :blocks]  # rows strided; some pages outside
    req = torch.tensor([3, 0, 0, 2, 1], dtype=torch.int32, device="cuda")
    q = randn(52, 5, H, 576)
    tok = (ints(53, 430, (5, 1, 170)) - 5).to(torch.int32)  # some negative, some behind the table
    want = R.attend(q, pool, paged_slots(table, req, tok, page, blocks), SCALE)
    for reps in (1, 24) if H > 32 else (1,):
        out, lse = F.fp4_ds_mla_sparse_decode_paged(q.repeat(reps, 1, 1), pool, req.repeat(reps), table,
                                                    tok.repeat(reps, 1, 1), SCALE, block_size=page, return_lse=True)
        for i in range(0, reps, 6):
            R.check((out[5 * i:5 * i + 5], lse[5 * i:5 * i + 5]), want)
    assert H <= 32 or F.fp4_kernel_name(H, 1, 5 * 24, 170) == MANY


@pytest.mark.parametrize("H", [16, 128])
def test_padding_tokens(H):
    """Tokens with a negative request attend to nothing, whatever their other
    inputs hold, and leave the others' results alone."""
    pool = make_pool(54, 640)
    table = ints(55, 10, (3, 6)).to(torch.int32)
    T = 80  # (both kernels at 128 heads: sparse calls of 80 and of 4 tokens)
    req = (torch.arange(T, device="cuda") % 4 - 1).to(torch.int32)
    q = randn(56, T, H, 576)
    tok = ints(57, 384, (T, 1, 200)).to(torch.int32)
    lens = ints(58, 384, (T,)).to(torch.int32)
    at = table.clone()[req.long().clamp(0)]  # a row a token
    rows = torch.arange(T, device="cuda")
    masked = torch.where((req < 0)[:, None, None], -1, paged_slots(at, rows, tok, 64, 6))
    want = R.attend(q, pool, masked, SCALE)
    for n in (T, 4):
        got = F.fp4_ds_mla_sparse_decode_paged(q[:n], pool, req[:n], table, tok[:n], SCALE, return_lse=True)
        R.check(got, [w[:n] for w in want])
    got = F.fp4_ds_mla_decode(q, pool, req, table, lens, SCALE, return_lse=True)
    live = torch.where(req < 0, 0, lens)
    R.check(got, R.attend(q, pool, dense_slots(at, rows, live, 64), SCALE))
    status_clean()


def dense_slots(table, req, lens, page):
    most = max(1, int(lens.max()))
    pos = torch.arange(most, device="cuda")
    tok = torch.where(pos[None, :] < lens[:, None], pos[None, :], -1)[:, None, :]
    return paged_slots(table, req, tok, page, table.shape[1])


@pytest.mark.parametrize("H", [1, 16, 40, 64, 128, 200])
@pytest.mark.parametrize("page", [1, 16, 64, 100, 128])
def test_dense(H, page):
    pool = make_pool(60, 3000)
    blocks = 700 // page
    table = torch.stack([torch.randperm(3000 // page, device="cuda")[:blocks] for _ in range(6)]).to(torch.int32)
    lens = torch.tensor([0, 1, 64, 65, 699, 300, 299], dtype=torch.int32, device="cuda").clamp(max=blocks * page)
    req = torch.tensor([0, 1, 2, 3, 4, 5, 5], dtype=torch.int32, device="cuda")
    q = randn(61, 7, H, 576)
    got = F.fp4_ds_mla_decode(q, pool, req, table, lens, SCALE, block_size=page, return_lse=True)
    R.check(got, R.attend(q, pool, dense_slots(table, req, lens, page), SCALE))
    status_clean()


@pytest.mark.parametrize("H", [16, 128])
def test_dense_long_and_lopsided(H):
    """One context much longer than the others, and more tokens than threads."""
    pool = make_pool(62, 20000)
    table = torch.arange(312, dtype=torch.int32, device="cuda").repeat(2, 1)
    q = randn(63, 2, H, 576)
    for lens in ([19968, 3], [1, 19967]):
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        req = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        got = F.fp4_ds_mla_decode(q, pool, req, table, ln, SCALE, return_lse=True)
        R.check(got, R.attend(q, pool, dense_slots(table, req, ln, 64), SCALE))
    T = 1200
    q = randn(64, T, 16, 576)
    ln = ((torch.arange(T, device="cuda") * 37) % 150).to(torch.int32)
    req = torch.zeros(T, dtype=torch.int32, device="cuda")
    got = F.fp4_ds_mla_decode(q, pool, req, table, ln, SCALE, return_lse=True)
    R.check(got, R.attend(q, pool, dense_slots(table, req, ln, 64), SCALE))


@pytest.mark.parametrize("H", [16, 128])
def test_dense_lengths_beyond_the_table_and_pages_outside(H):
    pool = make_pool(65, 640)
    table = torch.tensor([[0, 9, 10], [1, -1, 2]], dtype=torch.int32, device="cuda")  # 10 and -1: outside
    lens = torch.tensor([2 ** 31 - 1, 150], dtype=torch.int32, device="cuda")
    req = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    q = randn(66, 2, H, 576)
    got = F.fp4_ds_mla_decode(q, pool, req, table, lens, SCALE, return_lse=True)
    R.check(got, R.attend(q, pool, dense_slots(table, req, lens.clamp(max=192), 64), SCALE))


@pytest.mark.parametrize("H", [16, 128])
def test_offsets_past_32_bits(H):
    slots = 10_500_000  # 4.4 GB of rows
    pool = torch.zeros(slots, 416, dtype=torch.uint8, device="cuda")
    tail = make_pool(67, 2000)
    pool[-2000:] = tail
    q = randn(68, 2, H, 576)
    idx = (slots - 1 - ints(69, 2000, (2, 1, 300))).to(torch.int32)
    check_sparse(q, pool, idx, R.attend(q, tail, idx.long() - (slots - 2000), SCALE))
    back = F.dequant_fp4_ds_mla_rows(pool, idx[0, 0])
    assert torch.equal(back.double(), R.values(pool[idx[0, 0].long()]))
    kv_c, k_pe = randn(70, 3, 512), randn(71, 3, 64)
    F.concat_and_cache_fp4_ds_mla(kv_c, k_pe, pool, torch.tensor([slots - 1, 5_200_000, slots - 7], device="cuda"))
    assert torch.equal(pool[[slots - 1, 5_200_000, slots - 7]], R.quantize(kv_c, k_pe))


@pytest.mark.parametrize("H,T", [(16, 4), (128, 4), (128, 80)])
def test_q_layouts_and_workspace(H, T):
    pool = make_pool(72, 500)
    q, idx = sparse_case(73, T, H, 200, 500)
    want = F.fp4_ds_mla_sparse_decode(q, pool, idx, SCALE, return_lse=True)
    ws = torch.full((F.fp4_workspace_bytes(T, H) + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    views = [q.transpose(0, 1).contiguous().transpose(0, 1),                       # head-major
             torch.cat([q, q], 2)[:, :, :576],                                     # padded rows
             torch.cat([q[..., :3], q], 2)[:, :, 3:]]                              # misaligned rows
    for v in views:
        got = F.fp4_ds_mla_sparse_decode(v, pool, idx, SCALE, return_lse=True, workspace=ws)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = q[:1].clone().as_strided((1, H, 576), (H * 576 + 4, 576, 1))  # a single token's stride is not used
    assert odd.stride(0) % 8 == 4
    assert torch.equal(F.fp4_ds_mla_sparse_decode(odd, pool, idx[:1], SCALE),
                       F.fp4_ds_mla_sparse_decode(q[:1], pool, idx[:1], SCALE))
    wide = torch.cat([idx, idx], 2)[:, :, :200]
    assert torch.equal(F.fp4_ds_mla_sparse_decode(q, pool, wide, SCALE), want[0])


@pytest.mark.parametrize("H", [16, 128])
def test_repeats_bit_for_bit_and_on_a_side_stream(H):
    pool = make_pool(74, 4000)
    q, idx = sparse_case(75, 20, H, 1111, 4000, mask=0.1)
    want = F.fp4_ds_mla_sparse_decode(q, pool, idx, SCALE, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    with torch.cuda.stream(side):
        for _ in range(3):
            outs.append(F.fp4_ds_mla_sparse_decode(q, pool, idx, SCALE, return_lse=True))
    here = F.fp4_ds_mla_sparse_decode(q, pool, idx, SCALE, return_lse=True)  # at the same time
    torch.cuda.current_stream().wait_stream(side)
    for o, l in outs + [here]:
        assert torch.equal(o, want[0]) and torch.equal(l, want[1])


@pytest.mark.parametrize("H", [16, 128])
def test_graph_serves_new_lengths_and_tokens(H):
    """A captured step (write, dense attention) replays with new tokens, slots and
    lengths in its input tensors."""
    pool = make_pool(76, 64 * 20)
    table = torch.arange(20, dtype=torch.int32, device="cuda").view(2, 10)
    req = torch.arange(2, dtype=torch.int32, device="cuda")
    kv_c, k_pe, q = randn(77, 2, 512), randn(78, 2, 64), randn(79, 2, H, 576)
    slots = torch.zeros(2, dtype=torch.int64, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")

    def step():
        F.concat_and_cache_fp4_ds_mla(kv_c, k_pe, pool, slots)
        return F.fp4_ds_mla_decode(q, pool, req, table, lens, SCALE, return_lse=True)

    keep = pool.clone()
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    pool.copy_(keep)
    for i, ln in enumerate(([1, 640], [65, 0], [300, 301])):
        lens.copy_(torch.tensor(ln, dtype=torch.int32))
        slots.copy_(torch.tensor([max(ln[0] - 1, 0), 640 + max(ln[1] - 1, 0)]))
        kv_c.copy_(randn(80 + i, 2, 512))
        keep[slots] = R.quantize(kv_c, k_pe)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool, keep)
        R.check(got, R.attend(q, pool, dense_slots(table, req, lens, 64), SCALE))


@pytest.mark.parametrize("H", [16, 128])
def test_two_graphs_share_a_workspace(H):
    """Nothing in the workspace outlives a call: graphs of different sizes replay in
    turn over one."""
    pool = make_pool(95, 3000)
    cases = [sparse_case(96, 9, H, 1500, 3000, mask=0.1), sparse_case(97, 31, H, 700, 3000, mask=0.1)]
    ws = torch.full((F.fp4_workspace_bytes(31, H),), 0xFF, dtype=torch.uint8, device="cuda")
    want = [F.fp4_ds_mla_sparse_decode(q, pool, idx, SCALE, return_lse=True) for q, idx in cases]
    graphs, outs = [], []
    for q, idx in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(F.fp4_ds_mla_sparse_decode(q, pool, idx, SCALE, return_lse=True, workspace=ws))
        graphs.append(g)
    for i in (0, 1, 1, 0, 1, 0):
        outs[i][0].zero_()
        graphs[i].replay()
        assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1])


@pytest.mark.parametrize("H", [16, 128])
def test_calls_in_a_row_see_each_other(H):
    """Launched without a pause, so that each kernel is on the SMs before the one in
    front of it is done: rows that are written anew between reads of them."""
    n, times = 256, 40
    pool = make_pool(90, 640)
    slots = torch.randperm(640, device="cuda")[:n]
    idx = slots.to(torch.int32).view(1, n).repeat(40, 1)
    q = randn(92, 40, H, 576)
    kv_c, k_pe = randn(93, times, n, 512), randn(94, times, n, 64)
    torch.cuda.synchronize()
    got = []
    for i in range(times):
        F.concat_and_cache_fp4_ds_mla(kv_c[i], k_pe[i], pool, slots)
        got.append((F.dequant_fp4_ds_mla_rows(pool, slots), F.fp4_ds_mla_sparse_decode(q, pool, idx, SCALE)))
    for i in range(times):
        rows = R.quantize(kv_c[i], k_pe[i])
        assert torch.equal(got[i][0].double(), R.values(rows)), i
        fresh = F.fp4_ds_mla_sparse_decode(q, rows, torch.arange(n, dtype=torch.int32, device="cuda").repeat(40, 1),
                                           SCALE)
        assert torch.equal(got[i][1], fresh), i


def test_a_request_from_prompt_to_answer():
    """Together, as a server runs them: a prompt is written in two chunks, its
    cached part read back for prefill attention, then tokens are decoded, all
    over one pool, dense and by top-k of every position alike."""
    H, page, reqs = 16, 64, 3
    pool = torch.zeros(30 * page, 416, dtype=torch.uint8, device="cuda")
    mirror = pool.clone()
    table = torch.randperm(30, device="cuda")[:reqs * 8].view(reqs, 8).to(torch.int32)
    lens = [0] * reqs

    def append(seed, counts):
        n = sum(counts)
        kv_c, k_pe = randn(seed, n, 512), randn(seed + 1, n, 64)
        pos = torch.cat([torch.arange(lens[b], lens[b] + c) for b, c in enumerate(counts)]).cuda()
        req = torch.arange(reqs).repeat_interleave(torch.tensor(counts)).cuda()
        slots = table[req, pos // page].long() * page + pos % page
        F.concat_and_cache_fp4_ds_mla(kv_c, k_pe, pool.view(30, page, 416), slots)
        mirror[slots] = R.quantize(kv_c, k_pe)
        for b, c in enumerate(counts):
            lens[b] += c

    append(90, [100, 1, 64])
    append(92, [37, 200, 0])
    assert torch.equal(pool, mirror)
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    ctx = F.gather_fp4_ds_mla(pool, table, cu, sum(lens), block_size=page)
    assert torch.equal(ctx.double(), gather_want(mirror, table, lens, [0] * reqs, page))
    req = torch.arange(reqs, dtype=torch.int32, device="cuda")
    for step in range(3):
        append(94 + 2 * step, [1, 1, 1])
        q = randn(120 + step, reqs, H, 576)
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        want = R.attend(q, mirror, dense_slots(table, req, ln, page), SCALE)
        dense = F.fp4_ds_mla_decode(q, pool, req, table, ln, SCALE, block_size=page, return_lse=True)
        R.check(dense, want)
        tok = torch.arange(max(lens), device="cuda").repeat(reqs, 1)
        tok = torch.where(tok < ln[:, None], tok, -1).to(torch.int32)
        R.check(F.fp4_ds_mla_sparse_decode_paged(q, pool, req, table, tok, SCALE, block_size=page, return_lse=True), want)
    status_clean()

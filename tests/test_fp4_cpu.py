"""Refusals of the fp4_ds_mla entry points, and the writer's reference itself: no GPU needed."""

import re

import pytest
import torch

from tests import fp4_ref as R
from tests.conftest import REPO
from vllm_fp8kv import _native as N
from vllm_fp8kv import fp4_ds_mla as F
from vllm_fp8kv.cache_writer import concat_and_cache_mla


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def pool(n=64):
    return torch.zeros(n, 416, dtype=torch.uint8)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("call", [
    lambda: F.concat_and_cache_fp4_ds_mla(torch.zeros(2, 512), bf(2, 64), pool(), torch.arange(2)),
    lambda: F.concat_and_cache_fp4_ds_mla(bf(2, 512), bf(2, 63), pool(), torch.arange(2)),
    lambda: F.concat_and_cache_fp4_ds_mla(bf(2, 512), bf(2, 64), pool(), torch.arange(3)),
    lambda: F.concat_and_cache_fp4_ds_mla(bf(2, 512), bf(2, 64), torch.zeros(64, 656, dtype=torch.uint8), torch.arange(2)),
    lambda: F.concat_and_cache_fp4_ds_mla(bf(2, 512), bf(2, 64), pool().to(torch.int8), torch.arange(2)),
    lambda: F.dequant_fp4_ds_mla_rows(pool().t().contiguous().t(), torch.arange(2)),
    lambda: F.dequant_fp4_ds_mla_rows(pool(), torch.arange(2).float()),
    lambda: F.gather_fp4_ds_mla(pool(), i32(2, 3), i32(2), 4),
    lambda: F.gather_fp4_ds_mla(pool(), i32(2, 3).long(), i32(3), 4),
    lambda: F.gather_fp4_ds_mla(pool(), i32(2, 3), i32(3), 4, seq_starts=i32(3)),
    lambda: F.gather_fp4_ds_mla(pool(), i32(2, 3), i32(3), 4, block_size=0),
    lambda: F.fp4_ds_mla_sparse_decode(torch.zeros(1, 16, 576), pool(), i32(1, 8), 0.1),
    lambda: F.fp4_ds_mla_sparse_decode(bf(1, 16, 576).half(), pool(), i32(1, 8), 0.1),
    lambda: F.fp4_ds_mla_sparse_decode(bf(1, 16, 512), pool(), i32(1, 8), 0.1),
    lambda: F.fp4_ds_mla_sparse_decode(bf(1, 16, 576), pool(), i32(1, 3, 8), 0.1),
    lambda: F.fp4_ds_mla_sparse_decode(bf(1, 16, 576), pool(), i32(2, 8), 0.1),
    lambda: F.fp4_ds_mla_sparse_decode(bf(1, 16, 576), pool(), i32(1, 8).long(), 0.1),
    lambda: F.fp4_ds_mla_sparse_decode_paged(bf(1, 16, 576), pool(), i32(2), i32(1, 1), i32(1, 8), 0.1),
    lambda: F.fp4_ds_mla_sparse_decode_paged(bf(1, 16, 576), pool(), i32(1), i32(1), i32(1, 8), 0.1),
    lambda: F.fp4_ds_mla_decode(bf(1, 16, 576), pool(), i32(1), i32(1, 1), i32(2), 0.1),
    lambda: F.fp4_ds_mla_decode(bf(1, 16, 576), pool(), i32(1), i32(1, 1), i32(1).long(), 0.1),
    lambda: F.fp4_ds_mla_decode(bf(1, 16, 576), pool(), i32(1), i32(1, 1), i32(1), 0.1, block_size=0),
])
def test_refusals(call):
    with pytest.raises(AssertionError):
        call()


@pytest.mark.parametrize("call", [
    lambda: F.concat_and_cache_fp4_ds_mla(bf(2, 512), bf(2, 64), pool(), torch.arange(2)),
    lambda: F.dequant_fp4_ds_mla_rows(pool(), torch.arange(2)),
    lambda: F.gather_fp4_ds_mla(pool(), i32(2, 3), i32(3), 4),
    lambda: F.fp4_ds_mla_sparse_decode(bf(1, 16, 576), pool(), i32(1, 8), 0.1),
    lambda: F.fp4_ds_mla_decode(bf(1, 16, 576), pool(), i32(1), i32(1, 1), i32(1), 0.1),
])
def test_cpu_tensors_fail_loudly(call):
    with pytest.raises(N.Fp8MlaError, match="no CPU path"):
        call()


def test_the_writer_route_refuses_other_formats():
    with pytest.raises(NotImplementedError):
        concat_and_cache_mla(bf(1, 512), bf(1, 64), pool(), torch.arange(1), "fp4_other")


def c_decode(**over):
    args = dict(q=256, T=1, H=16, q_st=16 * 576, q_sh=576, kv=256, num_slots=64, idx=256, G=1, topk=32, idx_st=32,
                idx_sg=32, sm=0.1, out=256, out_st=16 * 512, out_sh=512, lse=None, lse_st=16, ws=None, ws_bytes=0,
                stream=None)
    args.update(over)
    return N.lib().fp8mla_fp4_sparse_decode(*args.values())


@pytest.mark.parametrize("over,needle", [
    (dict(T=-1), b"bad sizes"),
    (dict(G=3), b"not divisible"),
    (dict(num_slots=1 << 31), b"bad sizes"),
    (dict(topk=(1 << 30) + 1), b"too large"),
    (dict(q=None), b"null pointer"),
    (dict(idx=None), b"null pointer"),
    (dict(q=264), b"q must be 16-byte aligned"),
    (dict(q_sh=577), b"q must be 16-byte aligned"),
    (dict(out_st=8193), b"out must be 16-byte aligned"),
    (dict(kv=272), b"kv cache must be 32-byte aligned"),
])
def test_c_refusals(over, needle):
    assert c_decode(**over) == N.ERR_INVALID_ARGUMENT
    assert needle in N.lib().fp8mla_last_error()


def test_c_table_refusals():
    L = N.lib()

    def dense(block_size=64, max_blocks=4, stride=4, req=256, table=256, lens=256):
        return L.fp8mla_fp4_decode(256, 1, 16, 16 * 576, 576, 256, 64, req, table, stride, max_blocks, block_size,
                                   lens, 0.1, 256, 16 * 512, 512, None, 16, None, 0, None)

    for kw, needle in ((dict(block_size=0), b"bad block table"), (dict(stride=3), b"bad block table"),
                       (dict(max_blocks=1 << 30, stride=1 << 30), b"positions"),
                       (dict(max_blocks=1 << 58, stride=1 << 58), b"positions"), (dict(req=None), b"required"),
                       (dict(table=None), b"required"), (dict(lens=None), b"context_lens")):
        assert dense(**kw) == N.ERR_INVALID_ARGUMENT
        assert needle in L.fp8mla_last_error(), (kw, L.fp8mla_last_error())
    assert L.fp8mla_fp4_gather(256, 64, 256, 1, 2, 64, 256, 1, None, 4, 256, 576, None) == N.ERR_INVALID_ARGUMENT
    assert L.fp8mla_fp4_gather(256, 64, 256, 1 << 58, 1 << 58, 64, 256, 1, None, 4, 256, 576,
                               None) == N.ERR_INVALID_ARGUMENT
    assert L.fp8mla_fp4_gather(256, 64, 256, 2, 2, 64, 256, 1, None, 4, 256, 575, None) == N.ERR_INVALID_ARGUMENT
    assert L.fp8mla_fp4_write(256, 511, 256, 64, 256, 1, 256, 64, None) == N.ERR_INVALID_ARGUMENT
    assert L.fp8mla_fp4_write(256, 512, 256, 64, None, 1, 256, 64, None) == N.ERR_INVALID_ARGUMENT
    assert L.fp8mla_fp4_write(256, 512, 256, 64, 256, 1, 264, 64, None) == N.ERR_INVALID_ARGUMENT
    assert L.fp8mla_fp4_dequant_rows(256, 64, 256, 1, 264, 576, None) == N.ERR_INVALID_ARGUMENT
    assert c_decode(T=0) == N.OK and L.fp8mla_fp4_write(None, 512, None, 64, None, 0, None, 0, None) == N.OK


def test_workspace_and_names():
    assert F.fp4_workspace_bytes(0, 16) == 0
    assert F.fp4_workspace_bytes(1, 16) > 0 and F.fp4_workspace_bytes(1, 16) % 16 == 0
    assert F.fp4_workspace_bytes(3, 16, 1, 64) == 0            # whole rows: nothing to join
    for T, topk in ((1, 2048), (5, 100), (300, 777)):
        assert F.fp4_workspace_bytes(T, 16, 1, topk) <= F.fp4_workspace_bytes(T, 16)
    # the kernel of many heads: from 33 heads a group, and enough work to fill its tiles
    one, pair = "decode_fp4_kernel", "decode_fp4_tc_kernel"
    assert F.fp4_kernel_name(16) == F.fp4_kernel_name(32) == F.fp4_kernel_name(128, 4, 64, 2048) == one
    assert F.fp4_kernel_name(33) == F.fp4_kernel_name(128) == pair
    assert F.fp4_kernel_name(128, 1, 1, 2048) == one and F.fp4_kernel_name(128, 1, 64, 2048) == pair
    assert F.fp4_kernel_name(64, 1, 4, 2048) == one and F.fp4_kernel_name(40, 1, 64, 2048) == pair


def test_header_constants_match_python_module():
    text = open(f"{REPO}/include/fp8mla.h").read()
    for name, val in [("ROW_BYTES", F.ROW_BYTES), ("GROUP", F.GROUP), ("SCALE_OFF", F.SCALE_OFF),
                      ("ROPE_OFF", F.ROPE_OFF)]:
        m = re.search(rf"#define FP8MLA_FP4_{name} (\d+)", text)
        assert m and int(m.group(1)) == val, name


def test_reference_round_trips_and_rounds_to_even():
    """The reference of the GPU tests: representable groups come back as they
    were, borders go to the even code."""
    lv = torch.tensor(R.LEVELS + [-v for v in R.LEVELS], dtype=torch.float64)
    rows = R.quantize((lv * 0.5).repeat(32).view(1, 512).to(torch.bfloat16), bf(1, 64))
    back = R.values(rows)[0, :512]
    assert torch.equal(back, (lv * 0.5).repeat(32))
    g = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -5, 0, 0, 0, 0, 0, 0], dtype=torch.float64)
    back = R.values(R.quantize(g.repeat(32).view(1, 512).to(torch.bfloat16), bf(1, 64)))[0, :16]
    assert back.tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -0.0, -4, 0, 0, 0, 0, 0, 0]


def test_short_rows_of_few_heads_go_to_the_kernel_of_few_heads():
    """Units of one or two chunks need no more than one SM each: nothing there is for
    128-row tiles to gain at up to 32 heads."""
    for H in (1, 8, 16, 17, 32):
        for T in (1, 2, 7, 37, 64, 74, 75, 148, 256):
            for topk in (0, 1, 63, 64, 65, 100, 127, 128):
                assert F.fp4_kernel_name(H, 1, T, topk) == "decode_fp4_kernel", (H, T, topk)
                if topk <= 64:
                    assert F.fp4_workspace_bytes(T, H, 1, topk) == 0
    assert F.fp4_kernel_name(128, 1, 148, 64) == "decode_fp4_tc_kernel"

// abi_fp4.cu -- the C entry points of the 4-bit cache (include/fp8mla.h):
// argument checks, the division of work, workspace layout and dispatch.
#include "common.cuh"
#include "decode_fp4.h"
#include "wait_limit.h"

using namespace fp8mla;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int64_t kMaxTopk = 1LL << 30, kMaxT = 1LL << 24, kMaxH = 1 << 16;

// How a call's units are dealt out (decode_fp4.h).
struct Plan {
  int rows, workers, hb_per_group, chunk, min_per;
  int64_t per;  // 0: from the lengths, on the device
  bool cuts;    // some unit may be cut
  bool tc;      // the paired tensor-core kernel
  double us;    // expected time (lengths known)
};
// Expected time, us, of a call whose workers take `per` chunks each of units of n
// chunks; `cut`: units are cut, so there are partial results, a merge, and more
// changes of unit than need be, unless n is a multiple of `per`.  Fitted to 560 calls of
// either kernel; on 1755 shapes (8 to 128 heads, 1 to 256 tokens, top-1 to top-4096:
// profiles/fp4_cost_model.txt) it is off by 5% in the 16-head kernel and by 18% in the
// paired one, mostly above it, and choosing by it costs 0.3% on average against the
// best choice for each call, at worst 24% (top-512, 1 token, 8 heads: 15.0 us whole, 12.1
// cut).  For instance, 16-head kernel / paired kernel / chosen, measured:
//   tokens   top-64, 16 heads    top-64, 128 heads    top-2048, 40        top-2048, 64        top-2048, 128
//   1        7.3 / 10.9 / 7.3    7.2 / 12.7 / 7.2     18.4 / 17.7 / 18.4  18.9 / 19.3 / 18.9  19.3 / 20.1 / 19.3
//   8        7.3 / 11.4 / 7.3    7.9 / 13.0 / 7.9     23.7 / 26.1 / 23.7  25.5 / 29.2 / 25.5  34.1 / 34.1 / 34.1
//   32       7.7 / 11.8 / 7.7    13.7 / 13.4 / 13.7   42.9 / 48.5 / 42.9  45.7 / 51.0 / 45.7  88 / 52.1 / 52.1
//   148      8.5 / 19.9 / 8.5    46 / 23.0 / 23.0     133 / 100 / 100     176 / 102 / 102     346 / 104 / 104
double cost(bool tc, int64_t per, int64_t n, bool cut) {
  const double units = per > n ? (double)per / (double)n : 1.0;
  if (tc) return 2.8 + 2.46 * (double)per + 8.6 * units + (!cut ? 0 : n % per == 0 ? 11.4 : 24.6);
  return 1.6 + 1.21 * (double)per + 4.6 * units + (!cut ? 0 : n % per == 0 ? 6.3 : 9.6);
}

// topk < 0: whole contexts, of at most max_len positions
Plan plan_with(bool tc, int64_t T, int64_t H, int64_t G, int64_t topk, int64_t max_len) {
  Plan p;
  const int64_t hpg = H / G;
  p.tc = tc;
  p.rows = p.tc ? kFp4TcRows : 16;
  p.workers = p.tc ? device_sm_count() / 2 : device_sm_count();
  p.hb_per_group = (int)((hpg + p.rows - 1) / p.rows);
  p.chunk = p.tc ? kFp4TcChunk : kFp4Chunk;
  const int64_t chunk = p.chunk, units = T * G * p.hb_per_group;
  const int64_t len = topk < 0 ? max_len : topk;
  const int64_t n = len > chunk ? (len + chunk - 1) / chunk : 1;  // chunks of a unit (at most)
  p.min_per = p.tc ? 1 : (int)(n < kFp4MinPer ? n : kFp4MinPer);
  const int64_t total = units * n;
  if (total < p.workers) p.workers = (int)total;
  if (topk < 0) {
    p.per = 0;
    p.cuts = n > 1;
    p.us = 0;
    return p;
  }
  p.per = (total + p.workers - 1) / p.workers;
  if (p.per < p.min_per) p.per = p.min_per;
  // whole units, or equal runs whose borders cut units
  const int64_t whole = (p.per + n - 1) / n * n;
  p.us = cost(tc, whole, n, false);
  p.cuts = whole != p.per && 1.02 * cost(tc, p.per, n, true) < p.us;  // (near ties: no partials)
  if (p.cuts)
    p.us = cost(tc, p.per, n, true);
  else
    p.per = whole;
  p.workers = (int)((total + p.per - 1) / p.per);
  return p;
}
// Which kernel: the one that should be done first.  Lengths that only the device
// knows are taken for long ones: there the paired kernel is ahead from 33 heads on
// (with 17 to 32 it wastes three quarters of its tile).
Plan plan_of(int64_t T, int64_t H, int64_t G, int64_t topk, int64_t max_len) {
  const Plan one = plan_with(false, T, H, G, topk, max_len), pair = plan_with(true, T, H, G, topk, max_len);
  return (topk < 0 ? H / G > 32 : pair.us < one.us) ? pair : one;
}
int64_t info_bytes(const Plan& p) { return (int64_t)p.workers * 4 * 8; }
int64_t part_bytes(const Plan& p) { return (int64_t)2 * p.workers * p.rows * FP8MLA_NOPE * 4; }
int64_t workspace_of(const Plan& p) {
  return p.cuts ? part_bytes(p) + (int64_t)2 * p.workers * p.rows * 8 + info_bytes(p) : 0;
}

int check_table(const int32_t* req_id, const int32_t* block_table, int64_t bt_stride, int64_t max_blocks,
                int64_t block_size, int64_t T) {
  if (block_size <= 0 || block_size > (1 << 20) || max_blocks < 0 || bt_stride < max_blocks)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "bad block table: block_size=%lld max_blocks=%lld stride=%lld",
                     (long long)block_size, (long long)max_blocks, (long long)bt_stride);
  if (max_blocks > INT32_MAX / block_size)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT,
                     "a block-table row of %lld pages of %lld covers more than 2^31 - 1 positions", (long long)max_blocks,
                     (long long)block_size);
  if (T > 0 && (req_id == nullptr || (max_blocks > 0 && block_table == nullptr)))
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "req_id and block_table are required");
  return FP8MLA_OK;
}

int attend(const uint16_t* q, int64_t T, int64_t H, int64_t q_st, int64_t q_sh, const uint8_t* kv,
           int64_t num_slots, const int32_t* idx, int64_t G, int64_t topk, int64_t idx_st, int64_t idx_sg,
           const int32_t* lens, const int32_t* req_id, const int32_t* block_table, int64_t bt_stride,
           int64_t max_blocks, int64_t block_size, float sm_scale, uint16_t* out, int64_t out_st, int64_t out_sh,
           float* lse, int64_t lse_st, void* workspace, int64_t workspace_bytes, void* stream) {
  if (T < 0 || H <= 0 || G <= 0 || topk < 0 || num_slots < 0 || num_slots >= (1LL << 31))
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "bad sizes T=%lld H=%lld G=%lld topk=%lld num_slots=%lld",
                     (long long)T, (long long)H, (long long)G, (long long)topk, (long long)num_slots);
  if (H % G != 0)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "h_q=%lld not divisible by kv_groups=%lld", (long long)H,
                     (long long)G);
  if (topk > kMaxTopk || T > kMaxT || H > kMaxH)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "topk, T or H too large");
  if (T == 0) return FP8MLA_OK;
  if (q == nullptr || out == nullptr || (num_slots > 0 && kv == nullptr) || (lens == nullptr && topk > 0 && idx == nullptr))
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "null pointer");
  if (!aligned16(q) || q_st % 8 || q_sh % 8)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "q must be 16-byte aligned with row strides multiple of 16 bytes");
  if (!aligned16(out) || out_st % 8 || out_sh % 8)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "out must be 16-byte aligned with strides multiple of 8 elements");
  if ((reinterpret_cast<uintptr_t>(kv) & 31u) != 0)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "kv cache must be 32-byte aligned");
  if (int rc = require_sm100()) return rc;

  const int64_t hpg = H / G;
  const Plan p = plan_of(T, H, G, lens != nullptr ? -1 : topk, max_blocks * block_size);
  if (p.cuts && (workspace == nullptr || workspace_bytes < workspace_of(p) ||
                 (reinterpret_cast<uintptr_t>(workspace) & 31u) != 0))
    return set_error(FP8MLA_ERR_WORKSPACE, "needs %lld bytes of 32-B aligned workspace, got %lld",
                     (long long)workspace_of(p), (long long)workspace_bytes);
  Fp4DecodeArgs a{};
  a.q = q;
  a.q_st = q_st;
  a.q_sh = q_sh;
  a.kv = kv;
  a.num_slots = num_slots;
  a.lens = lens;
  a.idx = idx;
  a.idx_st = idx_st;
  a.idx_sg = idx_sg;
  a.T = (int)T;
  a.H = (int)H;
  a.G = (int)G;
  a.topk = (int)topk;
  a.hpg = (int)hpg;
  a.rows = p.rows;
  a.hb_per_group = p.hb_per_group;
  a.workers = p.workers;
  a.per = p.per;
  a.min_per = p.min_per;
  a.scale_log2 = sm_scale * kLog2e;
  a.out = out;
  a.out_st = out_st;
  a.out_sh = out_sh;
  a.lse = lse;
  a.lse_st = lse_st;
  a.req_id = req_id;
  // the kernels tell paged calls by the table: an empty one is never read, but
  // its pointer may be null
  a.block_table = req_id != nullptr && block_table == nullptr ? req_id : block_table;
  a.bt_stride = bt_stride;
  a.max_blocks = max_blocks;
  a.block_size = (int)block_size;
  a.block_shift = -1;
  for (int k = 0; k < 31; ++k)
    if (block_table != nullptr && (int64_t)1 << k == block_size) a.block_shift = k;
  a.max_len = max_blocks * block_size;
  a.wait_looks = handoff_wait_iters() / (kMaxWaitIters / kMaxWaitLooks);
  if (p.cuts) {
    char* ws = static_cast<char*>(workspace);
    a.ws_o = reinterpret_cast<float*>(ws);
    a.ws_info = reinterpret_cast<int64_t*>(ws + part_bytes(p));
    a.ws_ml = reinterpret_cast<float2*>(ws + part_bytes(p) + info_bytes(p));
  }

  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return p.tc ? launch_decode_fp4_tc(a, p.cuts, st) : launch_decode_fp4(a, p.cuts, st);
}

}  // namespace

extern "C" {

int fp8mla_fp4_write(const uint16_t* kv_c, int64_t kv_c_stride, const uint16_t* k_pe, int64_t k_pe_stride,
                     const int64_t* slot_mapping, int64_t N, uint8_t* cache, int64_t num_slots, void* stream) {
  clear_error();
  if (N < 0 || num_slots < 0 || kv_c_stride < FP8MLA_NOPE || k_pe_stride < FP8MLA_ROPE)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "bad writer sizes/strides");
  if (N == 0) return FP8MLA_OK;
  if (kv_c == nullptr || k_pe == nullptr || slot_mapping == nullptr || (num_slots > 0 && cache == nullptr))
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "null pointer");
  if (!aligned16(cache)) return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "cache must be 16-byte aligned");
  if (int rc = require_sm100()) return rc;
  return launch_fp4_write(kv_c, kv_c_stride, k_pe, k_pe_stride, slot_mapping, N, cache, num_slots,
                          static_cast<cudaStream_t>(stream));
}

int fp8mla_fp4_dequant_rows(const uint8_t* kv, int64_t num_slots, const int64_t* slots, int64_t n, uint16_t* out,
                            int64_t out_stride, void* stream) {
  clear_error();
  if (n < 0 || num_slots < 0 || out_stride < kDqk)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "bad row-dequant arguments");
  if (n == 0) return FP8MLA_OK;
  if ((num_slots > 0 && kv == nullptr) || slots == nullptr || out == nullptr)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "null pointer");
  if (!aligned16(kv) || !aligned16(out) || out_stride % 8 != 0)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "row dequant needs 16-byte aligned rows");
  if (int rc = require_sm100()) return rc;
  return launch_fp4_rows(kv, num_slots, slots, n, out, out_stride, static_cast<cudaStream_t>(stream));
}

int fp8mla_fp4_gather(const uint8_t* kv, int64_t num_slots, const int32_t* block_table, int64_t bt_stride,
                      int64_t max_blocks, int64_t block_size, const int32_t* cu_seq_lens, int64_t B,
                      const int32_t* seq_starts, int64_t n, uint16_t* out, int64_t out_stride, void* stream) {
  clear_error();
  if (n < 0 || num_slots < 0 || B < 0 || B > INT32_MAX || out_stride < kDqk || block_size <= 0 ||
      block_size > (1 << 20) || max_blocks < 0 || max_blocks > INT32_MAX || bt_stride < max_blocks)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "bad gather sizes or strides");
  if (n == 0 || B == 0) return FP8MLA_OK;
  if ((num_slots > 0 && kv == nullptr) || cu_seq_lens == nullptr || out == nullptr ||
      (max_blocks > 0 && block_table == nullptr))
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "null pointer");
  if (!aligned16(kv) || !aligned16(out) || out_stride % 8 != 0)
    return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "gather needs 16-byte aligned rows");
  if (int rc = require_sm100()) return rc;
  return launch_fp4_gather(kv, num_slots, block_table, bt_stride, max_blocks, (int)block_size, cu_seq_lens, (int)B,
                           seq_starts, n, out, out_stride, static_cast<cudaStream_t>(stream));
}

int64_t fp8mla_fp4_workspace_bytes(int64_t T, int64_t H, int64_t G, int64_t topk) {
  if (T <= 0 || T > kMaxT || H <= 0 || H > kMaxH || G <= 0 || H % G != 0 || topk < -1 || topk > kMaxTopk) return 0;
  return workspace_of(plan_of(T, H, G, topk, INT32_MAX));
}

const char* fp8mla_fp4_kernel_name(int64_t T, int64_t H, int64_t G, int64_t topk) {
  if (T <= 0 || T > kMaxT || H <= 0 || H > kMaxH || G <= 0 || H % G != 0 || topk < -1 || topk > kMaxTopk) return "";
  return plan_of(T, H, G, topk, INT32_MAX).tc ? "decode_fp4_tc_kernel" : "decode_fp4_kernel";
}

int fp8mla_fp4_sparse_decode(const uint16_t* q, int64_t T, int64_t H, int64_t q_stride_t, int64_t q_stride_h,
                             const uint8_t* kv, int64_t num_slots, const int32_t* indices, int64_t G, int64_t topk,
                             int64_t idx_stride_t, int64_t idx_stride_g, float sm_scale, uint16_t* out,
                             int64_t out_stride_t, int64_t out_stride_h, float* lse, int64_t lse_stride_t,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  return attend(q, T, H, q_stride_t, q_stride_h, kv, num_slots, indices, G, topk, idx_stride_t, idx_stride_g,
                nullptr, nullptr, nullptr, 0, 0, 0, sm_scale, out, out_stride_t, out_stride_h, lse, lse_stride_t,
                workspace, workspace_bytes, stream);
}

int fp8mla_fp4_sparse_decode_paged(const uint16_t* q, int64_t T, int64_t H, int64_t q_stride_t, int64_t q_stride_h,
                                   const uint8_t* kv, int64_t num_slots, const int32_t* req_id,
                                   const int32_t* block_table, int64_t bt_stride, int64_t max_blocks,
                                   int64_t block_size, const int32_t* token_idx, int64_t G, int64_t topk,
                                   int64_t ti_stride_t, int64_t ti_stride_g, float sm_scale, uint16_t* out,
                                   int64_t out_stride_t, int64_t out_stride_h, float* lse, int64_t lse_stride_t,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_table(req_id, block_table, bt_stride, max_blocks, block_size, T)) return rc;
  return attend(q, T, H, q_stride_t, q_stride_h, kv, num_slots, token_idx, G, topk, ti_stride_t, ti_stride_g,
                nullptr, req_id, block_table, bt_stride, max_blocks, block_size, sm_scale, out, out_stride_t,
                out_stride_h, lse, lse_stride_t, workspace, workspace_bytes, stream);
}

int fp8mla_fp4_decode(const uint16_t* q, int64_t T, int64_t H, int64_t q_stride_t, int64_t q_stride_h,
                      const uint8_t* kv, int64_t num_slots, const int32_t* req_id, const int32_t* block_table,
                      int64_t bt_stride, int64_t max_blocks, int64_t block_size, const int32_t* context_lens,
                      float sm_scale, uint16_t* out, int64_t out_stride_t, int64_t out_stride_h, float* lse,
                      int64_t lse_stride_t, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_table(req_id, block_table, bt_stride, max_blocks, block_size, T)) return rc;
  if (T > 0 && context_lens == nullptr) return set_error(FP8MLA_ERR_INVALID_ARGUMENT, "context_lens is required");
  return attend(q, T, H, q_stride_t, q_stride_h, kv, num_slots, nullptr, 1, 0, 0, 0, context_lens, req_id,
                block_table, bt_stride, max_blocks, block_size, sm_scale, out, out_stride_t, out_stride_h, lse,
                lse_stride_t, workspace, workspace_bytes, stream);
}

}  // extern "C"

// decode_fp4.h -- internal arguments of the fp4_ds_mla attention kernels, their
// division of work, and the launchers of the cache kernels.
//
// Work is a list of units (query token, kv group, head block), token-major,
// each of ceil(entries / chunk) chunks (at least one, so an empty row is
// written too).  The chunks of all units, in order, are dealt to the workers
// (an SM or an SM pair) in equal consecutive runs of `per` chunks: the loads
// are balanced to one chunk whatever the lengths, and only the units that a
// run's border cuts leave partial results, at most two per worker.  A worker
// whose first chunk lies inside a unit writes that unit's piece to its slot
// 2w; a piece that starts a unit and does not finish it goes to slot 2w + 1.
// The merge kernel joins a cut unit's pieces in order, so results do not
// depend on timing.
#pragma once
#include <atomic>

#include "common.cuh"
#include "decode.h"

namespace fp8mla {

struct Fp4DecodeArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint8_t* kv;
  int64_t num_slots;
  const int32_t* idx;    // top-k entries (null for an empty list; lens == null)
  int64_t idx_st, idx_sg;
  const int32_t* lens;   // set: the entries of token t are positions 0 .. lens[t]-1
  int T, H, G, topk;
  int hpg;               // heads per kv group
  int rows;              // heads per unit
  int hb_per_group;      // ceil(hpg / rows)
  float scale_log2;      // sm_scale * log2(e)
  uint16_t* out;
  int64_t out_st, out_sh;
  float* lse;
  int64_t lse_st;
  const int32_t* req_id; // block table set: idx holds request-local positions
  const int32_t* block_table;
  int64_t bt_stride, max_blocks;
  int block_size;
  int block_shift;       // log2(block_size) when it is a power of two, else -1
  int64_t max_len;       // max_blocks * block_size (lens set)
  int64_t per;           // chunks per worker; 0 = from the lengths, on the device
  int min_per;           // ... but at least this many, or a mean unit's
  int workers;
  float* ws_o;           // [2 * workers][rows][512] unnormalised partials
  float2* ws_ml;         // [2 * workers][rows] (reference max in log2 units, sum)
  int64_t* ws_info;      // [workers][4]: unit, first chunk in it, its chunks, per
  uint32_t wait_looks;   // limit of decode_fp4_kernel's hand-off waits
};

// Raises a kernel's dynamic shared memory limit, once per device.
struct SmemLimit {
  std::atomic<uint64_t> done{0};  // bit per device
  template <typename Kern>
  int raise(Kern kern, size_t bytes) {
    int dev = 0;
    if (int rc = check_cuda(cudaGetDevice(&dev), "current device")) return rc;
    if (dev < 64 && ((done.load(std::memory_order_acquire) >> dev) & 1u)) return FP8MLA_OK;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
    return check_cuda(e, "shared memory attribute");
  }
};

// One worker per SM, 16 heads per unit (decode_fp4.cu).  `cuts`: some unit may
// be cut, so the merge follows.
int launch_decode_fp4(const Fp4DecodeArgs& a, bool cuts, cudaStream_t st);
// One worker per SM pair, up to 128 heads per unit (decode_fp4_tc.cu).
int launch_decode_fp4_tc(const Fp4DecodeArgs& a, bool cuts, cudaStream_t st);
int read_device_status_fp4_tc(unsigned int* status, bool reset, cudaStream_t st);
constexpr int kFp4TcRows = 128;
constexpr int kFp4TcChunk = 128;
int launch_merge_fp4(const Fp4DecodeArgs& a, float bias, cudaStream_t st);
constexpr int kFp4Chunk = 64;   // entries per chunk
constexpr int kFp4MinPer = 3;   // chunks of a piece of a cut unit: three groups of warps take one each
int read_device_status_fp4(unsigned int* status, bool reset, cudaStream_t st);
// launch_wait_timeout_selftest for the wait loop of these kernels.
int launch_wait_timeout_selftest_fp4(uint32_t looks, uint64_t* elapsed_ns, cudaStream_t st);

int launch_fp4_write(const uint16_t* kv_c, int64_t kv_c_stride, const uint16_t* k_pe, int64_t k_pe_stride,
                     const int64_t* slot_mapping, int64_t N, uint8_t* cache, int64_t num_slots,
                     cudaStream_t st);
int launch_fp4_rows(const uint8_t* kv, int64_t num_slots, const int64_t* slots, int64_t n, uint16_t* out,
                    int64_t out_stride, cudaStream_t st);
int launch_fp4_gather(const uint8_t* kv, int64_t num_slots, const int32_t* block_table, int64_t bt_stride,
                      int64_t max_blocks, int block_size, const int32_t* cu, int B, const int32_t* starts,
                      int64_t n, uint16_t* out, int64_t out_stride, cudaStream_t st);

}  // namespace fp8mla

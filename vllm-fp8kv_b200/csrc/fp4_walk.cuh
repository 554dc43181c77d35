// fp4_walk.cuh -- device side of the division of work (decode_fp4.h): where a
// worker starts, its walk over chunks, and the pipelined way from an entry to
// its slot.
#pragma once
#include "common.cuh"
#include "decode_fp4.h"
#include "tc_ptx.cuh"

namespace fp8mla {
namespace fp4 {

// Entries one unit of token t attends over.
__device__ __forceinline__ int entries_of(const Fp4DecodeArgs& a, int64_t t) {
  if (a.lens == nullptr) return a.topk;
  const int64_t n = a.lens[t];
  return (int)(n < 0 ? 0 : n > a.max_len ? a.max_len : n);
}
template <int kChunk>
__device__ __forceinline__ int chunks_of(int entries) {
  return entries > kChunk ? (entries - 1) / kChunk + 1 : 1;  // (entries go up to 2^31 - 1)
}

// u / d: nearly always in 32 bits.
__device__ __forceinline__ int64_t quotient(int64_t u, int d) {
  return (u >> 32) == 0 ? (int64_t)((uint32_t)u / (uint32_t)d) : u / d;
}

struct Share {  // in shared memory: one worker's share of the chunk list
  int64_t total;       // chunks of the call
  int64_t per;         // chunks per worker
  int64_t start_unit;  // the worker's first unit, its first chunk of it
  int start_chunk;
  int64_t scan[32];
};

// Fills `s` for `worker`: from the sizes, or (lengths on the device) from two
// passes over the lengths.  All threads of the block call it.
template <int kChunk, int kThreads>
__device__ void divide(const Fp4DecodeArgs& a, Share& s, int worker) {
  const int per_tok = a.G * a.hb_per_group;
  if (a.lens == nullptr) {
    if (threadIdx.x == 0) {
      const int64_t n = chunks_of<kChunk>(a.topk), at = (int64_t)worker * a.per;
      s.total = (int64_t)a.T * per_tok * n;
      s.per = a.per;
      s.start_unit = quotient(at, n);
      s.start_chunk = (int)(at - s.start_unit * n);
    }
    __syncthreads();
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t sum = 0;
  for (int t = threadIdx.x; t < a.T; t += kThreads) sum += chunks_of<kChunk>(entries_of(a, t));
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (lane == 0) s.scan[warp] = sum;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < kThreads / 32; ++w) total += s.scan[w];
  total *= per_tok;
  int64_t per = quotient(total + a.workers - 1, a.workers);
  // pieces of a cut unit have min_per chunks at least, but units that are shorter on
  // average are not lined up behind one another for that while SMs stand idle
  if (per < a.min_per) {
    const int64_t mean = quotient(total, a.T * per_tok);
    const int64_t least = mean < a.min_per ? mean : a.min_per;
    if (per < least) per = least;
  }
  const int64_t at = (int64_t)worker * per;
  int64_t before = 0;  // chunks of the tokens in front of this pass
  for (int t0 = 0; t0 < a.T; t0 += kThreads) {
    const int t = t0 + threadIdx.x;
    const int n = t < a.T ? chunks_of<kChunk>(entries_of(a, t)) : 0;
    const int64_t mine = (int64_t)n * per_tok;
    int64_t inc = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += v;
    }
    __syncthreads();  // the sums of the pass before have been read
    if (lane == 31) s.scan[warp] = inc;
    __syncthreads();
    int64_t base = before;
    for (int w = 0; w < warp; ++w) base += s.scan[w];
    const int64_t hi = base + inc, lo = hi - mine;
    if (t < a.T && at >= lo && at < hi) {
      const int64_t u = quotient(at - lo, n);
      s.start_unit = (int64_t)t * per_tok + u;
      s.start_chunk = (int)(at - lo - u * n);
    }
    for (int w = 0; w < kThreads / 32; ++w) before += s.scan[w];
  }
  if (threadIdx.x == 0) {
    s.total = total;
    s.per = per;
  }
  __syncthreads();
}

// A worker's place in the chunk list.
template <int kChunk>
struct Walk {
  int64_t left;   // chunks of this worker from the current one on (none: <= 0)
  int64_t unit;   // t * (G * hb_per_group) + group * hb_per_group + head block
  int64_t t;
  int grp, hb;
  int c, n;       // chunk within the unit, chunks of the unit
  int entries;
  __device__ __forceinline__ void open(const Fp4DecodeArgs& a, int64_t u) {
    const int per_tok = a.G * a.hb_per_group;
    unit = u;
    t = quotient(u, per_tok);
    const int r = (int)(u - t * per_tok);
    grp = r / a.hb_per_group;
    hb = r - grp * a.hb_per_group;
    c = 0;
    entries = entries_of(a, t);
    n = chunks_of<kChunk>(entries);
  }
  __device__ __forceinline__ Walk(const Fp4DecodeArgs& a, const Share& s, int worker) {
    const int64_t at = (int64_t)worker * s.per;
    left = s.total - at < s.per ? s.total - at : s.per;
    if (left > 0) {
      open(a, s.start_unit);
      c = s.start_chunk;
    }
  }
  // chunks of this worker in the current unit, from the current chunk on
  __device__ __forceinline__ int here() const { return (int)(left < n - c ? left : n - c); }
  __device__ __forceinline__ void next_unit(const Fp4DecodeArgs& a, int done) {
    left -= done;
    if (left > 0) open(a, unit + 1);
  }
};

// What the merge has to know of a worker's first unit (one thread calls it).
template <int kChunk>
__device__ __forceinline__ void note_start(const Fp4DecodeArgs& a, const Share& s, int worker) {
  if (a.ws_info == nullptr) return;
  int64_t* info = a.ws_info + 4 * (int64_t)worker;
  info[1] = 0;
  if ((int64_t)worker * s.per < s.total) {
    info[0] = s.start_unit;
    info[1] = s.start_chunk;
    info[2] = chunks_of<kChunk>(entries_of(a, s.start_unit / (a.G * a.hb_per_group)));
  }
  info[3] = s.per;
}

__device__ __forceinline__ int32_t block_of(const Fp4DecodeArgs& a, int32_t v) {
  return a.block_shift >= 0 ? (v >> a.block_shift) : v / a.block_size;
}
// Block-table word of an entry (0 without a table), and the entry's slot given
// that word; -1: masked, behind the table, or outside the pool.
__device__ __forceinline__ int32_t table_word(const Fp4DecodeArgs& a, int32_t req, int32_t v) {
  if (a.block_table == nullptr || v < 0) return 0;
  if (req < 0) return -1;  // a padding token
  const int32_t blk = block_of(a, v);
  return blk < a.max_blocks ? a.block_table[(int64_t)req * a.bt_stride + blk] : -1;
}
__device__ __forceinline__ int32_t slot_of(const Fp4DecodeArgs& a, int32_t v, int32_t page) {
  int64_t s = v;
  if (a.block_table != nullptr) {
    if (v < 0 || page < 0) return -1;
    const int32_t blk = block_of(a, v);
    s = (int64_t)page * a.block_size + (v - blk * a.block_size);
  }
  return s >= 0 && s < a.num_slots ? (int32_t)s : -1;
}

// The slots of rows row, row + 32, .. (kRows of them) of every `kStride`-th chunk
// of a worker's run: entries are read three steps ahead of their use and block-table
// words two, so that a step waits for what is left of one latency.
template <int kChunk, int kStride, int kRows>
struct Slots {
  Walk<kChunk> ahead;
  int row;
  int32_t req = 0;
  const int32_t* idx_row = nullptr;
  int32_t v[3][kRows], rq[3], pg[2][kRows];  // of the current step and the next ones
  __device__ __forceinline__ void at_unit(const Fp4DecodeArgs& a) {
    if (ahead.left <= 0) return;
    if (a.block_table != nullptr) req = a.req_id[ahead.t];
    if (a.lens == nullptr) idx_row = a.idx + ahead.t * a.idx_st + ahead.grp * a.idx_sg;
  }
  __device__ __forceinline__ void step(const Fp4DecodeArgs& a) {
    if (--ahead.left > 0 && ++ahead.c == ahead.n) {
      ahead.open(a, ahead.unit + 1);
      at_unit(a);
    }
  }
  __device__ __forceinline__ void fetch(const Fp4DecodeArgs& a, int32_t (&e)[kRows]) const {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int pos = ahead.c * kChunk + row + 32 * i;
      e[i] = ahead.left <= 0 || pos >= ahead.entries ? -1 : a.lens == nullptr ? idx_row[pos] : pos;
    }
  }
  __device__ __forceinline__ void words(const Fp4DecodeArgs& a, int32_t r, const int32_t (&e)[kRows],
                                        int32_t (&p)[kRows]) const {
#pragma unroll
    for (int i = 0; i < kRows; ++i) p[i] = table_word(a, r, e[i]);
  }
  // of chunks first, first + kStride, ... of the run
  __device__ __forceinline__ Slots(const Fp4DecodeArgs& a, const Share& s, int worker, int row_, int first)
      : ahead(a, s, worker), row(row_) {
    at_unit(a);
    if (first) step(a);  // (0 or 1)
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      v[0][i] = v[1][i] = v[2][i] = -1;
      pg[0][i] = pg[1][i] = 0;
    }
    rq[0] = rq[1] = rq[2] = 0;
  }
  // The first kN steps, in one pass: two latencies.  (In next() the loads of a step
  // are waited for when its registers move up, which is one latency a call.)
  template <int kN>
  __device__ __forceinline__ void start(const Fp4DecodeArgs& a, int32_t (&slot)[kN][kRows]) {
    int32_t e[kN][kRows], p[kN][kRows], r[kN];
#pragma unroll
    for (int x = 0; x < kN; ++x) {
      fetch(a, e[x]);
      r[x] = req;
#pragma unroll
      for (int k = 0; k < kStride; ++k) step(a);
    }
#pragma unroll
    for (int x = 0; x < kN; ++x) words(a, r[x], e[x], p[x]);
#pragma unroll
    for (int x = 0; x < kN; ++x)
#pragma unroll
      for (int i = 0; i < kRows; ++i) slot[x][i] = slot_of(a, e[x][i], p[x][i]);
  }
  // The next step; the first call after start() fills the pipeline.
  __device__ __forceinline__ void next(const Fp4DecodeArgs& a, int32_t (&slot)[kRows], bool fill) {
#pragma unroll 1
    for (int k = fill ? 0 : 3; k < 4; ++k) shift(a, slot);
  }
  __device__ __forceinline__ void shift(const Fp4DecodeArgs& a, int32_t (&slot)[kRows]) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      slot[i] = slot_of(a, v[0][i], pg[0][i]);
      v[0][i] = v[1][i];
      v[1][i] = v[2][i];
      pg[0][i] = pg[1][i];
    }
    rq[1] = rq[2];
    fetch(a, v[2]);
    rq[2] = req;
    words(a, rq[1], v[1], pg[1]);
#pragma unroll
    for (int k = 0; k < kStride; ++k) step(a);
  }
};

// Bounded wait of a whole warp: every lane looks (so every lane has acquired the
// phase) and the vote gives all of them one verdict.  A phase that is complete
// costs 18 cycles; one lane looking for the others and passing the verdict on
// costs 190.  `limit` counts looks, rounded up to kUnroll.  kUnroll: the compiler's
// choice would be 8 KB of code for every wait.
template <int kUnroll>
__device__ __forceinline__ bool wait(uint64_t& b, uint32_t parity, uint32_t where,
                                     uint32_t limit = kMaxWaitLooks) {
  const uint32_t at = smem_u32(&b);
#pragma unroll 1
  for (uint32_t it = 0; it < limit; it += kUnroll)
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (__all_sync(0xFFFFFFFFu, tc::mbar_try_wait(at, parity))) return true;
  if ((threadIdx.x & 31) == 0) atomicOr(&tc::g_device_status, tc::kStatusWaitTimeout | (where << 8));
  return false;
}

__device__ __forceinline__ void bulk_g2s(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

}  // namespace fp4
}  // namespace fp8mla

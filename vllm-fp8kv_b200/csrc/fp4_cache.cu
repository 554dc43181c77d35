// fp4_cache.cu -- the fp4_ds_mla cache around the attention: the writer, the
// row read-back and the read-back of whole sequences.  All three move bytes:
// 1152 in and 416 out per written token, 416 in and 1152 out per token read,
// and run at 0.90 to 0.92 of a plain copy's rate (6.5 TB/s).  One warp owns one row
// and one lane one scale group (16 values: 8 code bytes, one scale byte), so no
// value crosses a lane and every access of a warp is one contiguous run.  What
// held them at two thirds of that were instructions (conversions by way of fp32,
// 64-bit divisions by every lane) and too few resident warps.
#include "fp4.cuh"
#include "decode.h"
#include "decode_fp4.h"

namespace fp8mla {
namespace {
using namespace fp8mla::fp4;

// The kernels may start before the one in front of them is done (pdl_wait), so no
// pointer is __restrict__: loads that the compiler takes for reads of constant
// memory may be moved in front of the wait, or be served from before it.
constexpr int kBlock = 256;
constexpr int kWarps = kBlock / 32;

// ------------------------------------------------------------------ writer
// Per group: scale = e4m3(clamp(amax / 6, 2^-9, 448)), code = e2m1(x / scale),
// both round to nearest even, the code saturating at 6.  A group that holds a
// NaN gets a NaN scale and reads back as NaN.
//
// x / scale without a division per value: q = x * (1 / scale) is within 2^-22
// (relative) of the quotient.  A rounding border t of e2m1 has at most 3
// significant bits and t * scale at most 7, x has 8: the quotient is either t
// exactly or at least 2^-8 (relative) away from it.  Rounding q to 12
// significant bits (half an ulp: 2^-12) moves it onto t in the first case and
// not across it in the second, so the conversion decides as the exact quotient
// would.
__device__ __forceinline__ float snap12(float q) {
  return __uint_as_float((__float_as_uint(q) + 0x800u) & 0xFFFFF000u);
}
// 2 values -> 2 codes, x0 in the low nibble
__device__ __forceinline__ uint32_t f32x2_to_e2m1x2(float x0, float x1) {
  uint32_t r;
  asm("{\n .reg .b8 b;\n cvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n cvt.u32.u8 %0, b;\n}\n"
      : "=r"(r)
      : "f"(x1), "f"(x0));
  return r;
}

template <bool kVec>
__device__ __forceinline__ void load16(uint32_t (&w)[8], const uint16_t* src) {
  if (kVec) {
    const uint4 a = reinterpret_cast<const uint4*>(src)[0];
    const uint4 b = reinterpret_cast<const uint4*>(src)[1];
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = (uint32_t)src[2 * j] | ((uint32_t)src[2 * j + 1] << 16);
  }
}
template <bool kVec>
__device__ __forceinline__ uint4 load8(const uint16_t* r) {
  if (kVec) return *reinterpret_cast<const uint4*>(r);
  return make_uint4((uint32_t)r[0] | ((uint32_t)r[1] << 16), (uint32_t)r[2] | ((uint32_t)r[3] << 16),
                    (uint32_t)r[4] | ((uint32_t)r[5] << 16), (uint32_t)r[6] | ((uint32_t)r[7] << 16));
}

// kVec: rows of both inputs 16-byte aligned.  A row a warp with all of an SM's warps
// resident: 17.3 us for 65536 rows, 6.0 TB/s (with the next row prefetched and half
// the warps 19.0).
template <bool kVec>
__global__ void __launch_bounds__(kBlock, kVec ? 8 : 4) fp4_write_kernel(
    const uint16_t* kv_c, int64_t kv_c_stride, const uint16_t* k_pe,
    int64_t k_pe_stride, const int64_t* slot_mapping, int64_t N,
    uint8_t* cache, int64_t num_slots) {
  if (threadIdx.x == 0) pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warps_total = (int64_t)gridDim.x * kWarps;
  for (int64_t tok = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32; tok < N; tok += warps_total) {
    const int64_t slot = slot_mapping[tok];
    uint32_t in[8];  // 16 latent values
    load16<kVec>(in, kv_c + tok * kv_c_stride + lane * 16);
    uint4 rope = make_uint4(0, 0, 0, 0);
    if (lane < 8) rope = load8<kVec>(k_pe + tok * k_pe_stride + lane * 8);
    if (slot >= 0 && slot < num_slots) {  // else a padding token
      // amax on the bf16 bits: magnitudes order as integers, NaN above inf
      uint32_t m2 = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m2 = __vmaxu2(m2, in[j] & 0x7FFF7FFFu);
      const uint32_t m = max(m2 & 0xFFFFu, m2 >> 16);
      const bool nan = m > 0x7F80u;
      const float want = fminf(fmaxf(__fdiv_rn(__uint_as_float(m << 16), 6.0f), 0.001953125f), 448.0f);
      uint16_t sb;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(sb) : "f"(0.0f), "f"(want));
      const uint32_t s2 = e4m3x2_to_f16(sb);
      const float inv = __frcp_rn(__half2float(__ushort_as_half((unsigned short)(s2 & 0xFFFFu))));
      uint32_t q[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        q[h] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w = in[4 * h + j];
          q[h] |= f32x2_to_e2m1x2(snap12(bf16_lo(w) * inv), snap12(bf16_hi(w) * inv)) << (8 * j);
        }
      }
      uint8_t* row = cache + slot * (int64_t)kFp4RowBytes;
      reinterpret_cast<uint2*>(row)[lane] = make_uint2(q[0], q[1]);
      row[kFp4ScaleOff + lane] = nan ? (uint8_t)0x7F : (uint8_t)sb;
      if (lane < 8) reinterpret_cast<uint4*>(row + kFp4RopeOff)[lane] = rope;
    }
  }
}

// ------------------------------------------------------------------ read-back
struct RowIn {
  uint2 codes;
  uint32_t scale;
  uint4 rope;
};
__device__ __forceinline__ void row_load(RowIn& in, const uint8_t* kv, int64_t slot, int lane) {
  if (slot >= 0) {
    const uint8_t* row = kv + slot * (int64_t)kFp4RowBytes;
    in.codes = reinterpret_cast<const uint2*>(row)[lane];
    in.scale = row[kFp4ScaleOff + lane];
    in.rope = lane < 8 ? reinterpret_cast<const uint4*>(row + kFp4RopeOff)[lane] : make_uint4(0, 0, 0, 0);
  } else {
    in.codes = make_uint2(0, 0);
    in.scale = 0;
    in.rope = make_uint4(0, 0, 0, 0);
  }
}
// Rows that start at 32-byte sectors are stored a sector a lane.
__device__ __forceinline__ bool whole_sectors(const uint16_t* out, int64_t out_stride) {
  return out_stride % 16 == 0 && (reinterpret_cast<uintptr_t>(out) & 31) == 0;
}
__device__ __forceinline__ void row_store(const RowIn& in, uint16_t* dst, int lane, bool sectors) {
  const uint32_t s = bf16_scale(in.scale);
  uint32_t a[4], b[4];
  e2m1x8_to_f16(in.codes.x, a);
  e2m1x8_to_f16(in.codes.y, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = scaled_bf16x2(a[i], s);
    b[i] = scaled_bf16x2(b[i], s);
  }
  uint16_t* o = dst + 16 * lane;
  if (sectors) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(o), "r"(a[0]), "r"(a[1]),
                 "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "r"(b[2]), "r"(b[3])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(o)[0] = make_uint4(a[0], a[1], a[2], a[3]);
    reinterpret_cast<uint4*>(o)[1] = make_uint4(b[0], b[1], b[2], b[3]);
  }
  if (lane < 8) reinterpret_cast<uint4*>(dst + kNope)[lane] = in.rope;
}

// A row a warp: 32 registers, so all of an SM's warps are resident, each with one
// row in flight (17.3 us for 65536 rows; 20.8 with two rows a step, 22.1 with four).
__global__ void __launch_bounds__(kBlock, 8) fp4_rows_kernel(const uint8_t* kv, int64_t num_slots,
                                                          const int64_t* slots, int64_t n,
                                                          uint16_t* out, int64_t out_stride) {
  if (threadIdx.x == 0) pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const bool sectors = whole_sectors(out, out_stride);
  for (int64_t r = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32; r < n; r += (int64_t)gridDim.x * kWarps) {
    const int64_t s = slots[r];
    RowIn in;
    row_load(in, kv, s < num_slots ? s : -1, lane);
    row_store(in, out + r * out_stride, lane, sectors);
  }
}

// Sequence b with cu[b] <= r < cu[b + 1] (-1 if there is none): a warp looks at
// 32 evenly spaced entries at a time, so 1024 sequences take two rounds.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int B, int64_t r, int lane) {
  int lo = 0, n = B;  // the answer, if any, is in [lo, lo + n)
  if (r < cu[0] || r >= cu[B]) return -1;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lo + lane * step;
    const bool le = lane * step < n && cu[at] <= r;
    const int k = __popc(__ballot_sync(0xFFFFFFFFu, le)) - 1;  // the last probe at or below r
    const int left = n - k * step;
    lo += k * step;
    n = left < step ? left : step;
  }
  return lo;
}

// A warp reads kRun consecutive rows: it looks for the first one's sequence, lane
// i finds row i's slot, and the rows are in flight together.  196608 rows: 51.2 us,
// 6.0 TB/s (runs of 8 in two halves the same, but 1.0 us more for few rows).
constexpr int kRun = 4;

__global__ void __launch_bounds__(kBlock) fp4_gather_kernel(
    const uint8_t* kv, int64_t num_slots, const int32_t* block_table,
    int64_t bt_stride, int64_t max_blocks, int block_size, const int32_t* cu, int B,
    const int32_t* starts, int64_t n, uint16_t* out, int64_t out_stride) {
  if (threadIdx.x == 0) pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const bool sectors = whole_sectors(out, out_stride);
  const int64_t step = (int64_t)gridDim.x * kWarps * kRun;
  const int64_t max_pos = max_blocks * block_size;
  const int first = cu[0], last = cu[B];
  for (int64_t r0 = ((int64_t)blockIdx.x * kWarps + threadIdx.x / 32) * kRun; r0 < n && r0 < last; r0 += step) {
    if (r0 + kRun <= first) continue;
    int b = sequence_of(cu, B, r0 < first ? first : r0, lane);  // (first < last, so there is one)
    const int64_t r = r0 + lane;
    int64_t slot = -2;  // not a row of any sequence
    if (lane < kRun && r >= first && r < n && r < last) {
      while (r >= cu[b + 1]) ++b;
      slot = -1;
      const int64_t p = r - cu[b] + (starts != nullptr ? starts[b] : 0);
      if (p >= 0 && p < max_pos) {  // (below 2^32: a row of the sequence plus its start)
        const int64_t blk = (uint32_t)p / (uint32_t)block_size;
        const int64_t s = (int64_t)block_table[b * bt_stride + blk] * block_size + (p - blk * block_size);
        if (s >= 0 && s < num_slots) slot = s;
      }
    }
    RowIn in[kRun];
    int64_t s[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      s[i] = __shfl_sync(0xFFFFFFFFu, slot, i);
      row_load(in[i], kv, s[i], lane);
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (s[i] >= -1) row_store(in[i], out + (r0 + i) * out_stride, lane, sectors);
  }
}

// at most `waves` blocks per SM; the kernels stride over the rest
int grid_of(int64_t blocks, int waves) {
  const int64_t cap = (int64_t)device_sm_count() * waves;
  return (int)(blocks < cap ? blocks : cap);
}

}  // namespace

int launch_fp4_write(const uint16_t* kv_c, int64_t kv_c_stride, const uint16_t* k_pe, int64_t k_pe_stride,
                     const int64_t* slot_mapping, int64_t N, uint8_t* cache, int64_t num_slots,
                     cudaStream_t st) {
  const int grid = grid_of((N + kWarps - 1) / kWarps, 16);
  const bool vec = kv_c_stride % 8 == 0 && k_pe_stride % 8 == 0 &&
                   ((reinterpret_cast<uintptr_t>(kv_c) | reinterpret_cast<uintptr_t>(k_pe)) & 15) == 0;
  return check_cuda(launch_pdl(vec ? fp4_write_kernel<true> : fp4_write_kernel<false>, dim3(grid), dim3(kBlock), 0, st, kv_c, kv_c_stride, k_pe,
                               k_pe_stride, slot_mapping, N, cache, num_slots),
                    "fp4_write_kernel launch");
}

int launch_fp4_rows(const uint8_t* kv, int64_t num_slots, const int64_t* slots, int64_t n, uint16_t* out,
                    int64_t out_stride, cudaStream_t st) {
  const int grid = grid_of((n + kWarps - 1) / kWarps, 16);
  return check_cuda(launch_pdl(fp4_rows_kernel, dim3(grid), dim3(kBlock), 0, st, kv, num_slots, slots, n, out,
                               out_stride),
                    "fp4_rows_kernel launch");
}

int launch_fp4_gather(const uint8_t* kv, int64_t num_slots, const int32_t* block_table, int64_t bt_stride,
                      int64_t max_blocks, int block_size, const int32_t* cu, int B, const int32_t* starts,
                      int64_t n, uint16_t* out, int64_t out_stride, cudaStream_t st) {
  const int grid = grid_of((n + kWarps * kRun - 1) / (kWarps * kRun), 16);
  return check_cuda(launch_pdl(fp4_gather_kernel, dim3(grid), dim3(kBlock), 0, st, kv, num_slots, block_table,
                               bt_stride, max_blocks, block_size, cu, B, starts, n, out, out_stride),
                    "fp4_gather_kernel launch");
}

}  // namespace fp8mla

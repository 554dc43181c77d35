// fp4_cache.cu -- the fp4_ds_mla cache around the attention: the writer, the
// row read-back and the read-back of whole sequences.  All three move bytes:
// 1152 in and 416 out per written token, 416 in and 1152 out per token read.
// One warp owns one row and one lane one scale group (16 values: 8 code bytes,
// one scale byte), so no value crosses a lane and every access of a warp is
// one contiguous run.
#include "fp4.cuh"
#include "decode.h"
#include "decode_fp4.h"

namespace fp8mla {
namespace {
using namespace fp8mla::fp4;

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

struct WriterIn {
  int64_t slot;
  uint32_t w[8];  // 16 bf16 latent values
  uint4 rope;     // lanes 0..7: 8 bf16 rope values
};
__device__ __forceinline__ void load16(uint32_t (&w)[8], const uint16_t* src, bool vec) {
  if (vec) {
    const uint4 a = reinterpret_cast<const uint4*>(src)[0];
    const uint4 b = reinterpret_cast<const uint4*>(src)[1];
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = (uint32_t)src[2 * j] | ((uint32_t)src[2 * j + 1] << 16);
  }
}
__device__ __forceinline__ uint4 load8(const uint16_t* r, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(r);
  return make_uint4((uint32_t)r[0] | ((uint32_t)r[1] << 16), (uint32_t)r[2] | ((uint32_t)r[3] << 16),
                    (uint32_t)r[4] | ((uint32_t)r[5] << 16), (uint32_t)r[6] | ((uint32_t)r[7] << 16));
}

__global__ void __launch_bounds__(kBlock) fp4_write_kernel(
    const uint16_t* __restrict__ kv_c, int64_t kv_c_stride, const uint16_t* __restrict__ k_pe,
    int64_t k_pe_stride, const int64_t* __restrict__ slot_mapping, int64_t N,
    uint8_t* __restrict__ cache, int64_t num_slots) {
  if (threadIdx.x == 0) pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warps_total = (int64_t)gridDim.x * kWarps;
  const bool vec_c = (kv_c_stride % 8) == 0 && (reinterpret_cast<uintptr_t>(kv_c) & 15) == 0;
  const bool vec_pe = (k_pe_stride % 8) == 0 && (reinterpret_cast<uintptr_t>(k_pe) & 15) == 0;
  auto load = [&](WriterIn& in, int64_t tok) {
    in.slot = slot_mapping[tok];
    load16(in.w, kv_c + tok * kv_c_stride + lane * 16, vec_c);
    in.rope = lane < 8 ? load8(k_pe + tok * k_pe_stride + lane * 8, vec_pe) : make_uint4(0, 0, 0, 0);
  };
  int64_t tok = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  WriterIn cur, nxt;
  if (tok < N) load(cur, tok);
  for (; tok < N; tok += warps_total) {
    if (tok + warps_total < N) load(nxt, tok + warps_total);
    const int64_t slot = cur.slot;
    if (slot >= 0 && slot < num_slots) {  // else a padding token
      // amax on the bf16 bits: magnitudes order as integers, NaN above inf
      uint32_t m2 = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m2 = __vmaxu2(m2, cur.w[j] & 0x7FFF7FFFu);
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
          const uint32_t w = cur.w[4 * h + j];
          q[h] |= f32x2_to_e2m1x2(snap12(bf16_lo(w) * inv), snap12(bf16_hi(w) * inv)) << (8 * j);
        }
      }
      uint8_t* row = cache + slot * (int64_t)kFp4RowBytes;
      reinterpret_cast<uint2*>(row)[lane] = make_uint2(q[0], q[1]);
      row[kFp4ScaleOff + lane] = nan ? (uint8_t)0x7F : (uint8_t)sb;
      if (lane < 8) reinterpret_cast<uint4*>(row + kFp4RopeOff)[lane] = cur.rope;
    }
    cur = nxt;
  }
}

// ------------------------------------------------------------------ read-back
struct RowIn {
  uint2 codes;
  uint32_t scale;
  uint4 rope;
};
__device__ __forceinline__ void row_load(RowIn& in, const uint8_t* __restrict__ kv, int64_t slot, int lane) {
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
__device__ __forceinline__ void row_store(const RowIn& in, uint16_t* __restrict__ dst, int lane) {
  uint32_t s = e4m3x2_to_f16(in.scale * 0x0101u);
  uint32_t a[4], b[4];
  e2m1x8_to_f16(in.codes.x, a);
  e2m1x8_to_f16(in.codes.y, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = f16x2_to_bf16x2(mul_f16x2(a[i], s));
    b[i] = f16x2_to_bf16x2(mul_f16x2(b[i], s));
  }
  uint4* o = reinterpret_cast<uint4*>(dst + 16 * lane);
  o[0] = make_uint4(a[0], a[1], a[2], a[3]);
  o[1] = make_uint4(b[0], b[1], b[2], b[3]);
  if (lane < 8) reinterpret_cast<uint4*>(dst + kNope)[lane] = in.rope;
}

constexpr int kRowsPerStep = 4;  // rows of a warp in flight together

__global__ void __launch_bounds__(kBlock) fp4_rows_kernel(const uint8_t* __restrict__ kv, int64_t num_slots,
                                                          const int64_t* __restrict__ slots, int64_t n,
                                                          uint16_t* __restrict__ out, int64_t out_stride) {
  if (threadIdx.x == 0) pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * kWarps * kRowsPerStep;
  for (int64_t r0 = ((int64_t)blockIdx.x * kWarps + threadIdx.x / 32) * kRowsPerStep; r0 < n; r0 += step) {
    RowIn in[kRowsPerStep];
#pragma unroll
    for (int i = 0; i < kRowsPerStep; ++i) {
      int64_t s = r0 + i < n ? slots[r0 + i] : -1;
      if (s >= num_slots) s = -1;
      row_load(in[i], kv, s, lane);
    }
#pragma unroll
    for (int i = 0; i < kRowsPerStep; ++i)
      if (r0 + i < n) row_store(in[i], out + (r0 + i) * out_stride, lane);
  }
}

// Sequence b with cu[b] <= r < cu[b + 1] (-1 if there is none): a warp looks at
// 32 evenly spaced entries at a time, so 1024 sequences take two rounds.
__device__ __forceinline__ int sequence_of(const int32_t* __restrict__ cu, int B, int64_t r, int lane) {
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

__global__ void __launch_bounds__(kBlock) fp4_gather_kernel(
    const uint8_t* __restrict__ kv, int64_t num_slots, const int32_t* __restrict__ block_table,
    int64_t bt_stride, int64_t max_blocks, int block_size, const int32_t* __restrict__ cu, int B,
    const int32_t* __restrict__ starts, int64_t n, uint16_t* __restrict__ out, int64_t out_stride) {
  if (threadIdx.x == 0) pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * kWarps * kRowsPerStep;
  for (int64_t r0 = ((int64_t)blockIdx.x * kWarps + threadIdx.x / 32) * kRowsPerStep; r0 < n; r0 += step) {
    int b = sequence_of(cu, B, r0, lane);
    if (b < 0 && r0 >= cu[0]) continue;  // behind the last sequence
    int64_t slot[kRowsPerStep];
    bool mine[kRowsPerStep];
#pragma unroll
    for (int i = 0; i < kRowsPerStep; ++i) {
      const int64_t r = r0 + i;
      if (b < 0 && r < n) b = sequence_of(cu, B, r, lane);  // in front of the first sequence
      while (b >= 0 && r >= cu[b + 1]) b = b + 1 < B ? b + 1 : -1;
      mine[i] = b >= 0 && r < n;
      slot[i] = -1;
      if (mine[i]) {
        const int64_t p = r - cu[b] + (starts != nullptr ? starts[b] : 0);
        const int64_t blk = p / block_size;
        if (p >= 0 && blk < max_blocks) {
          const int64_t s = (int64_t)block_table[b * bt_stride + blk] * block_size + (p - blk * block_size);
          if (s >= 0 && s < num_slots) slot[i] = s;
        }
      }
    }
    RowIn in[kRowsPerStep];
#pragma unroll
    for (int i = 0; i < kRowsPerStep; ++i) row_load(in[i], kv, slot[i], lane);
#pragma unroll
    for (int i = 0; i < kRowsPerStep; ++i)
      if (mine[i]) row_store(in[i], out + (r0 + i) * out_stride, lane);
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
  return check_cuda(launch_pdl(fp4_write_kernel, dim3(grid), dim3(kBlock), 0, st, kv_c, kv_c_stride, k_pe,
                               k_pe_stride, slot_mapping, N, cache, num_slots),
                    "fp4_write_kernel launch");
}

int launch_fp4_rows(const uint8_t* kv, int64_t num_slots, const int64_t* slots, int64_t n, uint16_t* out,
                    int64_t out_stride, cudaStream_t st) {
  const int grid = grid_of((n + kWarps * kRowsPerStep - 1) / (kWarps * kRowsPerStep), 16);
  return check_cuda(launch_pdl(fp4_rows_kernel, dim3(grid), dim3(kBlock), 0, st, kv, num_slots, slots, n, out,
                               out_stride),
                    "fp4_rows_kernel launch");
}

int launch_fp4_gather(const uint8_t* kv, int64_t num_slots, const int32_t* block_table, int64_t bt_stride,
                      int64_t max_blocks, int block_size, const int32_t* cu, int B, const int32_t* starts,
                      int64_t n, uint16_t* out, int64_t out_stride, cudaStream_t st) {
  const int grid = grid_of((n + kWarps * kRowsPerStep - 1) / (kWarps * kRowsPerStep), 16);
  return check_cuda(launch_pdl(fp4_gather_kernel, dim3(grid), dim3(kBlock), 0, st, kv, num_slots, block_table,
                               bt_stride, max_blocks, block_size, cu, B, starts, n, out, out_stride),
                    "fp4_gather_kernel launch");
}

}  // namespace fp8mla

// decode_fp4.cu -- attention over fp4_ds_mla rows, 16 query heads per unit.
//
//   S = scale q . [latent | rope],  P = softmax(S),  O = P . latent
//
// A persistent CTA per SM walks its run of 64-entry chunks (decode_fp4.h).
// The 416-byte rows stay 4-bit in shared memory; both products unpack them in
// registers, straight into mma.sync fragments.  Shared memory sees 416 bytes of a row
// written and twice read, and 1152 of q (18 KB for every 16 entries).
//   * latents are exact in fp16 (fp4.cuh), so the latent products are fp16
//     MMAs: q is scaled per head by a power of two (q_power), to a largest value in
//     [2^8, 2^9) where the softmax scale is of ordinary size, and converted (exact
//     down to 2^-25 of that value, below it an error under 2^-33 of it), and P keeps
//     11 bits where bf16 keeps 8;
//   * the rope (bf16 as stored) and q's rope (times the same power of two)
//     go through bf16 MMAs into the same accumulators.
//
// Warp roles (512 threads):
//   warps 0-11  three groups of four.  A group takes every third chunk of a
//               unit's piece on its own, with its own maximum, sum and O, so the
//               three stand at different phases and fill each other's waits.
//               Warp w of a group computes S of entries [16w, +16), then, behind
//               the group's barrier, O of dims [128w, +128).  q (16 heads x 576,
//               as A fragments) is read from shared memory, once per 16 entries.
//               At the end of a piece the groups' results are joined.
//   warps 12-15 producers: entries -> slots -> TMA copies of 16 rows each
// The registers move from the producers to the others (setmaxnreg).  (No call that is
// not inlined may stand in this kernel: it would hold all of it to 128 registers,
// and spilling them made it three times slower.)
//
// Measured, us: 256 x 16 heads x top-2048 88.7 (two units on each of 128 SMs, 39% of
// a plain copy's rate); 64 x 16 heads over up to 16384 positions 85.6; 4 x 16 heads x
// top-256 10.7.  A chunk takes 2650 cycles of an SM, in which its MMAs take 1090, the
// conversions 1020 and the issue slots of its 86 instructions a row 1440: no pipe
// is full, and there are no registers for a fourth group.  Steps on the way:
// 150 with warps that did S and warps that did O, 126 with warps that do both, 92 in
// three groups, 88 with the producers' entries pipelined.
#include "decode_fp4.h"
#include "fp4.cuh"
#include "fp4_walk.cuh"
#include "tc_cluster.cuh"
#include "tc_ptx.cuh"
#include "tma_map.h"

namespace fp8mla {
namespace {
using namespace fp8mla::fp4;
using namespace fp8mla::tc;

constexpr int kBH = 16;           // heads per unit
constexpr int kBN = kFp4Chunk;    // entries per chunk
constexpr int kStages = 6;
constexpr int kStageBytes = kBN * kFp4RowBytes;  // 26624
constexpr int kGroups = kFp4MinPer, kGWarps = 4, kPWarps = 4;
constexpr int kCWarps = kGroups * kGWarps;
constexpr int kThreads = 32 * (kCWarps + kPWarps);
constexpr int kCRegs = 152, kPRegs = 56;  // launched with 128 each
static_assert(kCWarps * kCRegs + kPWarps * kPRegs <= (kCWarps + kPWarps) * 128, "register split");
constexpr int kQSteps = kDqk / 16;        // 36: 32 of the latents, 4 of the rope
constexpr float kRescale = 8.0f;  // the reference maximum lags by at most 2^8 ...
constexpr float kBias = 6.0f;     // ... and P is stored times 2^6: below 2^14 in
                                  // fp16, above its smallest value from 2^-30 on

struct Smem {
  uint8_t raw[kStages][kStageBytes];   // 128-B aligned TMA destinations
  uint32_t q[kQSteps][32][4];             // q as A fragments
  float join[kGWarps][16][32][4];         // a group's O on its way to the next group
  uint32_t p[kGroups][2][kBN / 16][32][4];  // P as A fragments of the O product
  float smax[kGroups][2][kGWarps][kBH];
  float lpart[kGroups][kGWarps][kBH];     // a piece's sums
  float gm[kGroups][kBH], gl[kGroups][kBH];
  float qscale[kBH];                      // score = qscale * accumulator (log2 units)
  uint32_t live[kStages][2];              // 16 bits per producer warp
  uint64_t raw_full[kStages], raw_empty[kStages];
  Share share;
};
static_assert(offsetof(Smem, q) % 16 == 0 && offsetof(Smem, live) % 8 == 0 && offsetof(Smem, raw_full) % 8 == 0, "alignment");
static_assert(sizeof(Smem) + 128 <= 227 * 1024, "shared memory budget");

template <int kRegs>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kRegs));
}
// Barriers: all compute warps (id 1), one group (id 2 + group), and the same
// with an "any of us" vote.
__device__ __forceinline__ void compute_sync() {
  asm volatile("bar.sync 1, %0;\n" ::"n"(32 * kCWarps) : "memory");
}
__device__ __forceinline__ void group_sync(int grp) {
  asm volatile("bar.sync %0, %1;\n" ::"r"(2 + grp), "n"(32 * kGWarps) : "memory");
}
__device__ __forceinline__ bool group_any(int grp, bool mine) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.or.pred q, %2, %3, p;\n"
      " selp.b32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"((uint32_t)mine), "r"(2 + grp), "n"(32 * kGWarps)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The chunk row that column n of an 8-column tile stands for, n even: n / 2,
// n odd: 4 + (n / 2 + 1) % 4.  It is both the S product's B column and the O
// product's k index, so P needs no shuffle between them; the rows of a column
// pair differ by an odd number (S loads of two rows meet no bank twice: a row
// is 104 words) and the rows of the even, or odd, columns are all different
// modulo 4 (neither do the O loads of four rows).
__device__ __forceinline__ int row_even(int pair) { return pair; }
__device__ __forceinline__ int row_odd(int pair) { return 4 + ((pair + 1) & 3); }

// Place in the ring of stages: the stage, and the parity of its current round.
struct Ring {
  int st = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void ahead(int n) {  // 0 <= n <= kStages
    st += n;
    if (st >= kStages) {
      st -= kStages;
      ph ^= 1;
    }
  }
};

// A wait between producers and compute warps.  A limit of 0 looks (a test's) stands for
// one that does not suspend the warp.
__device__ __forceinline__ bool hand_off(const Fp4DecodeArgs& a, uint64_t& b, uint32_t parity, uint32_t where) {
  if (a.wait_looks != 0) return wait<4>(b, parity, where, a.wait_looks);
  if (__all_sync(0xFFFFFFFFu, mbar_test_wait(smem_u32(&b), parity))) return true;
  if ((threadIdx.x & 31) == 0) atomicOr(&g_device_status, kStatusWaitTimeout | (where << 8));
  return false;
}

// ------------------------------------------------------------------ producers
// Warp pw owns rows [16 pw, +16) of every chunk: lanes 0-15 those of the even
// chunks of the worker's run, lanes 16-31 of the odd ones.  A run of consecutive
// slots (the pages of a whole context) is one bulk copy, other rows go four at
// a time through gather4; masked rows are not read (a group with some fetches
// row 0 for them) and their bits stay clear.
__device__ void produce(const Fp4DecodeArgs& a, Smem& s, const CUtensorMap* tm, int pw, int lane) {
  Slots<kBN, 2, 1> slots(a, s.share, blockIdx.x, 16 * pw + (lane & 15), lane >> 4);
  const int64_t chunks = Walk<kBN>(a, s.share, blockIdx.x).left;
  bool ok = true;
  int64_t armed = 0;
  Ring ring;
  int32_t early[2][1];
  slots.start(a, early);
#pragma unroll 1
  for (int64_t g = 0; g < chunks && ok; g += 2) {
    int32_t at[1];
    if (g >= 4)
      slots.next(a, at, g == 4);
    else
      at[0] = early[g >> 1][0];
    const int32_t slot = at[0];
    const uint32_t live2 = __ballot_sync(0xFFFFFFFFu, slot >= 0);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (g + half >= chunks) break;
      const int st = ring.st;
      if (g + half >= kStages) ok = hand_off(a, s.raw_empty[st], ring.ph ^ 1, 20);
      if (!ok) break;
      const uint32_t live = (live2 >> (16 * half)) & 0xFFFFu;
      const int n = __popc(live);
      const int32_t s0 = __shfl_sync(0xFFFFFFFFu, slot, 16 * half);
      const bool run = (live & (live + 1)) == 0 &&
                       __all_sync(0xFFFFFFFFu, (lane >> 4) != half || slot < 0 || slot == s0 + (lane & 15));
      const uint32_t bar = smem_u32(&s.raw_full[st]);
      const uint32_t dst = smem_u32(&s.raw[st][16 * pw * kFp4RowBytes]);
      // groups of four rows with a live one
      const uint32_t grp = (live & 0xFu ? 1u : 0u) | (live & 0xF0u ? 2u : 0u) | (live & 0xF00u ? 4u : 0u) |
                           (live & 0xF000u ? 8u : 0u);
      if (lane == 0) {
        reinterpret_cast<uint16_t*>(s.live[st])[pw] = (uint16_t)live;
        mbar_arrive_expect_tx(bar, run ? (uint32_t)(n * kFp4RowBytes) : (uint32_t)(__popc(grp) * 4 * kFp4RowBytes));
      }
      __syncwarp();
      if (run) {
        if (lane == 0 && n > 0) bulk_g2s(dst, a.kv + (int64_t)s0 * kFp4RowBytes, (uint32_t)(n * kFp4RowBytes), bar);
      } else {
        const int32_t r = slot >= 0 ? slot : 0;
        const int src = 16 * half + ((4 * lane) & 15);
        const int32_t r0 = __shfl_sync(0xFFFFFFFFu, r, src);
        const int32_t r1 = __shfl_sync(0xFFFFFFFFu, r, src + 1);
        const int32_t r2 = __shfl_sync(0xFFFFFFFFu, r, src + 2);
        const int32_t r3 = __shfl_sync(0xFFFFFFFFu, r, src + 3);
        if (lane < 4 && ((grp >> lane) & 1u)) tma_gather4(dst + lane * 4 * kFp4RowBytes, tm, 0, r0, r1, r2, r3, bar);
      }
      ++armed;
      ring.ahead(1);
    }
  }
  // the stages armed last have landed before the warp returns, even after a
  // failed wait
  for (int64_t x = armed > kStages ? armed - kStages : 0; x < armed; ++x)
    (void)wait<4>(s.raw_full[x % kStages], (uint32_t)(x / kStages) & 1, 26);
}

// ------------------------------------------------------------------ compute
// After a failed wait a warp goes on to the end, for the barriers that it shares with
// others, on whatever its stages hold, and releases no stage any more: a stage is
// armed anew only when all that it was armed with before has landed, so that the
// producers' last waits name their last copies.
//
// Fragment coordinates: lane = 4 gq + q4.  Thread q4 of a quad owns latent
// dims [128 q4, +128) of a row and rope dims [16 q4, +16); it walks its four
// 32-dim pieces in the order i ^ (q4 >> 1) and its two rope halves in the order
// h ^ (q4 & 1), so that 8 lanes' 16-byte loads cover all banks.  q's fragments
// follow the same order: k-step 8 i + 2 j (+ 1) of piece i holds dims 8 j, .. + 3
// (+ 4, .. + 7) of it, k-step 32 + 2 h (+ 1) the same of rope half h.

// q of the unit -> fragments in shared memory.  A half-warp owns a head, lane
// j of it dims [32 j, +32) and rope dims [4 j, +4).
__device__ void load_q(const Fp4DecodeArgs& a, Smem& s, const Walk<kBN>& x, int cw, int lane) {
  if (cw >= kBH / 2) return;
  const int row = 2 * cw + (lane >> 4), j16 = lane & 15;
  const bool hv = row < min(kBH, a.hpg - x.hb * kBH);
  const uint16_t* src = a.q + x.t * a.q_st + (int64_t)(x.grp * a.hpg + x.hb * kBH + (hv ? row : 0)) * a.q_sh;
  const uint4 z4 = make_uint4(0, 0, 0, 0);
  uint4 v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = hv ? reinterpret_cast<const uint4*>(src + 32 * j16)[j] : z4;
  const uint2 rp = hv ? *reinterpret_cast<const uint2*>(src + kNope + 4 * j16) : make_uint2(0, 0);
  uint32_t mx = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    mx = __vmaxu2(mx, __vmaxu2(__vmaxu2(v[j].x & 0x7FFF7FFFu, v[j].y & 0x7FFF7FFFu),
                               __vmaxu2(v[j].z & 0x7FFF7FFFu, v[j].w & 0x7FFF7FFFu)));
  const uint32_t mxr = __vmaxu2(rp.x & 0x7FFF7FFFu, rp.y & 0x7FFF7FFFu);
  // largest magnitudes (as bits) of the head's latent part and of its rope
  uint32_t m = max(mx & 0xFFFFu, mx >> 16), mr = max(mxr & 0xFFFFu, mxr >> 16);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    mr = max(mr, __shfl_xor_sync(0xFFFFFFFFu, mr, o));
  }
  const int k = q_power((int)m, (int)mr, a.scale_log2);
  const float up = __uint_as_float((uint32_t)(127 + k) << 23);
  if (j16 == 0) s.qscale[row] = a.scale_log2 * __uint_as_float((uint32_t)(127 - k) << 23);
  const int r = row >> 3, gq = row & 7;
  {
    const int q4 = j16 >> 2, i = (j16 & 3) ^ (q4 >> 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t* f0 = s.q[8 * i + 2 * j][4 * gq + q4];
      uint32_t* f1 = s.q[8 * i + 2 * j + 1][4 * gq + q4];
      f0[r] = pack_f16x2(bf16_lo(v[j].x) * up, bf16_hi(v[j].x) * up);
      f0[2 + r] = pack_f16x2(bf16_lo(v[j].y) * up, bf16_hi(v[j].y) * up);
      f1[r] = pack_f16x2(bf16_lo(v[j].z) * up, bf16_hi(v[j].z) * up);
      f1[2 + r] = pack_f16x2(bf16_lo(v[j].w) * up, bf16_hi(v[j].w) * up);
    }
  }
  {
    // rope dims 4 j16 .. + 3: quad thread j16 / 4, 8-dim half (j16 / 2) % 2, k-step j16 % 2 of it
    const int q4 = j16 >> 2, h = ((j16 >> 1) & 1) ^ (q4 & 1);
    uint32_t* f = s.q[32 + 2 * h + (j16 & 1)][4 * gq + q4];
    f[r] = pack_bf16x2(bf16_lo(rp.x) * up, bf16_hi(rp.x) * up);
    f[2 + r] = pack_bf16x2(bf16_lo(rp.y) * up, bf16_hi(rp.y) * up);
  }
}

// Accumulators of 16 entries (two tiles of 8, their rows 8 apart): row is this
// lane's column gq of the first.
__device__ __forceinline__ void score_tiles(const uint32_t (*q)[32][4], const uint8_t* row, int lane,
                                            float (&x)[2][4]) {
  const int q4 = lane & 3;
  float c0[2][4], c1[2][4];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) c0[t][i] = c1[t][i] = 0.f;
  uint32_t sc[2][2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint2 v = *reinterpret_cast<const uint2*>(row + t * 8 * kFp4RowBytes + kFp4ScaleOff + 8 * q4);
    const uint32_t sel = (q4 >> 1) ? 0x1032u : 0x3210u;
    sc[t][0] = __byte_perm(v.x, 0, sel);
    sc[t][1] = __byte_perm(v.y, 0, sel);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 w[2];
    uint32_t s_lo[2], s_hi[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      w[t] = *reinterpret_cast<const uint4*>(row + t * 8 * kFp4RowBytes + 64 * q4 + 16 * (i ^ (q4 >> 1)));
      const uint32_t s2 = e4m3x2_to_f16((i & 1) ? sc[t][i >> 1] >> 16 : sc[t][i >> 1]);
      s_lo[t] = __byte_perm(s2, 0, 0x1010);
      s_hi[t] = __byte_perm(s2, 0, 0x3232);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 a0 = *reinterpret_cast<const uint4*>(q[8 * i + 2 * j][lane]);
      const uint4 a1 = *reinterpret_cast<const uint4*>(q[8 * i + 2 * j + 1][lane]);
      const uint32_t f0[4] = {a0.x, a0.y, a0.z, a0.w}, f1[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        uint32_t h[4];
        e2m1x8_to_f16(j == 0 ? w[t].x : j == 1 ? w[t].y : j == 2 ? w[t].z : w[t].w, h);
        const uint32_t sj = j < 2 ? s_lo[t] : s_hi[t];
        mma_f16(c0[t], f0, mul_f16x2(h[0], sj), mul_f16x2(h[1], sj));
        mma_f16(c1[t], f1, mul_f16x2(h[2], sj), mul_f16x2(h[3], sj));
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 a0 = *reinterpret_cast<const uint4*>(q[32 + 2 * h][lane]);
    const uint4 a1 = *reinterpret_cast<const uint4*>(q[33 + 2 * h][lane]);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint4 w = *reinterpret_cast<const uint4*>(row + t * 8 * kFp4RowBytes + kFp4RopeOff + 32 * q4 +
                                                      16 * (h ^ (q4 & 1)));
      mma_bf16_16816(c0[t], a0.x, a0.y, a0.z, a0.w, w.x, w.y);
      mma_bf16_16816(c1[t], a1.x, a1.y, a1.z, a1.w, w.z, w.w);
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[t][i] = c0[t][i] + c1[t][i];
}

// O += P V of one chunk over this warp's 128 dims.  A thread owns 16 of them (one scale
// group): code_at, scale_at name it within a row.
__device__ __forceinline__ void output_step(const uint8_t* raw, const uint32_t (*p)[32][4], uint64_t live, int lane,
                                            int code_at, int scale_at, int ra, int rb, float (&acc)[16][4]) {
#pragma unroll
  for (int kk = 0; kk < kBN / 16; ++kk) {
    const uint4 pv = *reinterpret_cast<const uint4*>(p[kk][lane]);
    const uint32_t pa[4] = {pv.x, pv.y, pv.z, pv.w};
    const uint8_t* r0 = raw + (16 * kk + ra) * kFp4RowBytes;
    const uint8_t* r1 = raw + (16 * kk + rb) * kFp4RowBytes;
    const uint2 w0 = *reinterpret_cast<const uint2*>(r0 + code_at);
    const uint2 w1 = *reinterpret_cast<const uint2*>(r1 + code_at);
    const uint2 w2 = *reinterpret_cast<const uint2*>(r0 + 8 * kFp4RowBytes + code_at);
    const uint2 w3 = *reinterpret_cast<const uint2*>(r1 + 8 * kFp4RowBytes + code_at);
    uint32_t b0 = r0[scale_at], b1 = r1[scale_at];
    uint32_t b2 = r0[8 * kFp4RowBytes + scale_at], b3 = r1[8 * kFp4RowBytes + scale_at];
    if (live != ~0ull) {  // P is 0 there, but a NaN scale would still spread
      const uint32_t lv = (uint32_t)(live >> (16 * kk));
      b0 = (lv >> ra) & 1u ? b0 : 0u;
      b1 = (lv >> rb) & 1u ? b1 : 0u;
      b2 = (lv >> (ra + 8)) & 1u ? b2 : 0u;
      b3 = (lv >> (rb + 8)) & 1u ? b3 : 0u;
    }
    const uint32_t s01 = e4m3x2_to_f16(b0 | (b1 << 8)), s23 = e4m3x2_to_f16(b2 | (b3 << 8));
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 8 of the thread's dims
      const uint32_t c0 = h ? w0.y : w0.x, c1 = h ? w1.y : w1.x, c2 = h ? w2.y : w2.x, c3 = h ? w3.y : w3.x;
      // nibble pairs (row of the even k index low, of the odd one high): even
      // dims, then odd dims
      uint32_t e01[4], e23[4];
      e2m1x8_to_f16((c0 & 0x0F0F0F0Fu) | ((c1 << 4) & 0xF0F0F0F0u), e01);
      e2m1x8_to_f16((c2 & 0x0F0F0F0Fu) | ((c3 << 4) & 0xF0F0F0F0u), e23);
#pragma unroll
      for (int b = 0; b < 4; ++b)
        mma_f16(acc[8 * h + 2 * b], pa, mul_f16x2(e01[b], s01), mul_f16x2(e23[b], s23));
      e2m1x8_to_f16(((c0 >> 4) & 0x0F0F0F0Fu) | (c1 & 0xF0F0F0F0u), e01);
      e2m1x8_to_f16(((c2 >> 4) & 0x0F0F0F0Fu) | (c3 & 0xF0F0F0F0u), e23);
#pragma unroll
      for (int b = 0; b < 4; ++b)
        mma_f16(acc[8 * h + 2 * b + 1], pa, mul_f16x2(e01[b], s01), mul_f16x2(e23[b], s23));
    }
  }
}

__device__ void compute(const Fp4DecodeArgs& a, Smem& s, int cw, int lane) {
  const int gq = lane >> 2, q4 = lane & 3;
  const int grp = cw / kGWarps, gw = cw % kGWarps;
  Walk<kBN> w(a, s.share, blockIdx.x);
  int pb = 0;
  Ring piece_at;  // stage of the piece's first chunk
  bool ok = true;
  const int ra = row_even(q4), rb = row_odd(q4);  // rows of k indices 2 q4, 2 q4 + 1
  const uint32_t tile_at = (16 * gw + ((gq & 1) ? row_odd(gq >> 1) : row_even(gq >> 1))) * kFp4RowBytes;
  const int code_at = 64 * gw + 8 * gq, scale_at = kFp4ScaleOff + 8 * gw + gq;
  while (w.left > 0) {
    const int nch = w.here();
    load_q(a, s, w, cw, lane);
    compute_sync();
    float acc[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const float qs[2] = {s.qscale[gq], s.qscale[gq + 8]};
    Ring ring = piece_at;
    ring.ahead(grp);
    for (int c = grp; c < nch; c += kGroups) {
      if (ok) ok = hand_off(a, s.raw_full[ring.st], ring.ph, 21);
      const uint64_t live = *reinterpret_cast<const uint64_t*>(s.live[ring.st]);
      const uint8_t* raw = s.raw[ring.st];
      float x[2][4];
      score_tiles(s.q, raw + tile_at, lane, x);
      // scores in log2 units, masked ones -inf, and this warp's maxima
      const uint32_t lv = (uint32_t)(live >> (16 * gw));
      bool grown = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mt = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          x[t][2 * r] = (lv >> (8 * t + ra)) & 1u ? x[t][2 * r] * qs[r] : -INFINITY;
          x[t][2 * r + 1] = (lv >> (8 * t + rb)) & 1u ? x[t][2 * r + 1] * qs[r] : -INFINITY;
          mt = fmaxf(mt, fmaxf(x[t][2 * r], x[t][2 * r + 1]));
        }
        mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, 1));
        mt = fmaxf(mt, __shfl_xor_sync(0xFFFFFFFFu, mt, 2));
        if (q4 == 0) s.smax[grp][pb][gw][gq + 8 * r] = mt;
        grown |= mt > m[r] + kRescale;
      }
      // P against the reference maximum so far
      float p[2][4];
      auto exps = [&]() {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float sub = m[r] == -INFINITY ? 0.f : m[r] - kBias;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            p[t][2 * r] = ex2_approx(x[t][2 * r] - sub);
            p[t][2 * r + 1] = ex2_approx(x[t][2 * r + 1] - sub);
          }
        }
        *reinterpret_cast<uint4*>(s.p[grp][pb][gw][lane]) =
            make_uint4(pack_f16x2(p[0][0], p[0][1]), pack_f16x2(p[0][2], p[0][3]), pack_f16x2(p[1][0], p[1][1]),
                       pack_f16x2(p[1][2], p[1][3]));
      };
      exps();
      // The group's barrier: P is in place.  Where a maximum has outgrown the
      // reference (the first chunk, seldom later) all take the chunk's maximum.
      if (group_any(grp, grown)) {
        float al[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float tm = m[r];
#pragma unroll
          for (int i = 0; i < kGWarps; ++i) tm = fmaxf(tm, s.smax[grp][pb][i][gq + 8 * r]);
          al[r] = m[r] == -INFINITY ? 0.f : ex2_approx(m[r] - tm);
          m[r] = tm;
          l[r] *= al[r];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          acc[i][0] *= al[0];
          acc[i][1] *= al[0];
          acc[i][2] *= al[1];
          acc[i][3] *= al[1];
        }
        exps();
        group_sync(grp);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        l[0] += p[t][0] + p[t][1];
        l[1] += p[t][2] + p[t][3];
      }
      output_step(raw, s.p[grp][pb], live, lane, code_at, scale_at, ra, rb, acc);
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(smem_u32(&s.raw_empty[ring.st]));
      ring.ahead(kGroups);
      pb ^= 1;
    }
    piece_at.ahead(nch % kStages);
    if ((nch / kStages) & 1) piece_at.ph ^= 1;

    // ---- join the groups: maxima and sums, then O from the last group to the first
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 1);
      l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 2);
      if (q4 == 0) s.lpart[grp][gw][gq + 8 * r] = l[r];
      if (gw == 0 && q4 == 0) s.gm[grp][gq + 8 * r] = m[r];
    }
    compute_sync();
    float mm[2], lt[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int h = gq + 8 * r;
      mm[r] = fmaxf(fmaxf(s.gm[0][h], s.gm[1][h]), s.gm[2][h]);
      const float ref = mm[r] == -INFINITY ? 0.f : mm[r];
      lt[r] = 0.f;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        float li = 0.f;
#pragma unroll
        for (int k = 0; k < kGWarps; ++k) li += s.lpart[i][k][h];
        lt[r] += li == 0.f ? 0.f : li * ex2_approx(s.gm[i][h] - ref);
      }
      const float f = m[r] == -INFINITY ? 0.f : ex2_approx(m[r] - ref);
      if (m[r] != -INFINITY || l[r] != 0.f) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          acc[i][2 * r] *= f;
          acc[i][2 * r + 1] *= f;
        }
      }
    }
#pragma unroll
    for (int g = kGroups - 1; g >= 0; --g) {
      if (grp == g) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float4* at = reinterpret_cast<float4*>(s.join[gw][i][lane]);
          if (g < kGroups - 1) {
            const float4 o = *at;
            acc[i][0] += o.x;
            acc[i][1] += o.y;
            acc[i][2] += o.z;
            acc[i][3] += o.w;
          }
          if (g > 0) *at = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
        }
      }
      if (g > 0) compute_sync();
    }
    // ---- the piece: a whole unit goes to the output, a cut one to its slot
    if (grp == 0) {
      const bool whole = w.c == 0 && nch == w.n;
      const int h0 = w.grp * a.hpg + w.hb * kBH;
      const int nh = min(kBH, a.hpg - w.hb * kBH);
      const int64_t slot = 2 * (int64_t)blockIdx.x + (w.c == 0 ? 1 : 0);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = gq + 8 * r;
        if (row >= nh) continue;
        // column 2 q4 + j of the 16 tiles: the 16 dims of thread gq = 2 q4 + j
        const int d = 128 * gw + 32 * q4;
        if (whole) {
          const float inv = lt[r] > 0.f ? 1.f / lt[r] : (lt[r] == 0.f ? 0.f : lt[r]);
          uint4* o = reinterpret_cast<uint4*>(a.out + w.t * a.out_st + (int64_t)(h0 + row) * a.out_sh + d);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[i] = pack_bf16x2(acc[8 * (j & 1) + 2 * i][2 * r + (j >> 1)] * inv,
                                 acc[8 * (j & 1) + 2 * i + 1][2 * r + (j >> 1)] * inv);
            o[j] = make_uint4(v[0], v[1], v[2], v[3]);
          }
          if (a.lse != nullptr && gw == 0 && q4 == 0)
            a.lse[w.t * a.lse_st + h0 + row] = lt[r] == 0.f ? -INFINITY : (mm[r] - kBias) * kLn2 + logf(lt[r]);
        } else {
          float4* o = reinterpret_cast<float4*>(a.ws_o + (slot * kBH + row) * kNope + d);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              o[4 * j + i] = make_float4(acc[4 * i][2 * r + j], acc[4 * i + 1][2 * r + j], acc[4 * i + 2][2 * r + j],
                                         acc[4 * i + 3][2 * r + j]);
          if (gw == 0 && q4 == 0) a.ws_ml[slot * kBH + row] = make_float2(mm[r], lt[r]);
        }
      }
    }
    w.next_unit(a, nch);
  }
}

__global__ void __launch_bounds__(kThreads, 1)
    decode_fp4_kernel(const Fp4DecodeArgs a, const __grid_constant__ CUtensorMap tm) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  Smem& s = *reinterpret_cast<Smem*>(smem_raw + (((raw_base + 127u) & ~127u) - raw_base));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&s.raw_full[i]), kPWarps);
      mbar_init(smem_u32(&s.raw_empty[i]), kGWarps);
    }
    mbar_init_fence();
  }
  __syncthreads();
  if (threadIdx.x == 0) pdl_launch_dependents();
  pdl_wait();  // the previous kernel of the stream has completed: global memory from here on
  divide<kBN, kThreads>(a, s.share, blockIdx.x);
  if (threadIdx.x == 0) note_start<kBN>(a, s.share, blockIdx.x);
  if (warp < kCWarps) {
    regs_inc<kCRegs>();
    compute(a, s, warp, lane);
  } else {
    regs_dec<kPRegs>();
    produce(a, s, &tm, warp - kCWarps, lane);
  }
}

// ------------------------------------------------------------------ merge
// Joins the pieces of a cut unit for one head: out = sum 2^(m_i - m) O_i /
// sum 2^(m_i - m) l_i.  A unit's first border is the one in front of a worker
// that starts in it at most `per` chunks behind its start.
//   kSplit 1  block (w - 1, head) joins the unit that worker w's border is the first
//             to cut, if it is; most units have two or three pieces
//   kSplit 4  block (unit, head), for calls of few units, which many workers share
//             (74 or 148 pieces of one long context): each of four groups of 128
//             threads takes every fourth piece, eight loads in flight
//             (131071 positions, 128 heads, whole call: 64 instead of 78 us)
// A block's time is a chain of loads (the border, the pieces' sums, their O); the
// first O's are fetched with the sums: 61.5 instead of 64.4 us there.
template <int kSplit>
__global__ void __launch_bounds__(128 * kSplit) merge_fp4_kernel(const Fp4DecodeArgs a, float bias) {
  __shared__ int border;
  __shared__ __align__(16) float part[kSplit][128][4];
  if (threadIdx.x == 0) {
    pdl_launch_dependents();
    border = 0;
  }
  pdl_wait();
  int w = blockIdx.x + 1;
  if (kSplit > 1) {
    __syncthreads();
    for (int i = threadIdx.x + 1; i < a.workers; i += 128 * kSplit) {
      const int64_t* info = a.ws_info + 4 * (int64_t)i;
      if (info[1] > 0 && info[1] <= info[3] && info[0] == blockIdx.x) border = i;
    }
    __syncthreads();
    w = border;
    if (w == 0) return;
  }
  const int64_t* info = a.ws_info + 4 * (int64_t)w;
  const int64_t c = info[1], per = info[3];
  if (c == 0 || c > per) return;  // no cut here, or an earlier border cuts the unit too
  const int64_t unit = info[0], n = info[2];
  const int pieces = 1 + (int)((n - c + per - 1) / per);
  const int per_tok = a.G * a.hb_per_group;
  const int64_t t = unit / per_tok;
  const int rest = (int)(unit - t * per_tok), grp = rest / a.hb_per_group, hb = rest - grp * a.hb_per_group;
  const int row = blockIdx.y;
  if (row >= min(a.rows, a.hpg - hb * a.rows)) return;
  // workspace row of piece i
  auto at = [&](int i) -> int64_t { return (i == 0 ? 2 * (int64_t)w - 1 : 2 * (int64_t)(w - 1 + i)) * a.rows + row; };
  const int lane = threadIdx.x & 31, g4 = threadIdx.x >> 7, d4 = threadIdx.x & 127;
  // the first pieces' O are on their way while the sums are joined
  constexpr int kEarly = 4;
  float4 early[kEarly];
#pragma unroll
  for (int k = 0; k < kEarly; ++k) {
    const int i = g4 + k * kSplit;
    early[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < pieces) early[k] = reinterpret_cast<const float4*>(a.ws_o + at(i) * kNope)[d4];
  }
  // every warp: the maximum, then the sum
  float m = -INFINITY, l = 0.f;
  for (int i = lane; i < pieces; i += 32) m = fmaxf(m, a.ws_ml[at(i)].x);
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  const float ref = m == -INFINITY ? 0.f : m;
  for (int i = lane; i < pieces; i += 32) {
    const float2 ml = a.ws_ml[at(i)];
    l += exp2f(ml.x - ref) * ml.y;
  }
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](int i, const float4& o) {
    const float f = exp2f(a.ws_ml[at(i)].x - ref);
    acc.x += f * o.x;
    acc.y += f * o.y;
    acc.z += f * o.z;
    acc.w += f * o.w;
  };
#pragma unroll
  for (int k = 0; k < kEarly; ++k)
    if (g4 + k * kSplit < pieces) add(g4 + k * kSplit, early[k]);
#pragma unroll 8
  for (int i = g4 + kEarly * kSplit; i < pieces; i += kSplit)
    add(i, reinterpret_cast<const float4*>(a.ws_o + at(i) * kNope)[d4]);
  if (kSplit > 1) {
    *reinterpret_cast<float4*>(part[g4][d4]) = acc;
    __syncthreads();
    if (g4 != 0) return;
#pragma unroll
    for (int g = 1; g < kSplit; ++g) {
      const float4 o = *reinterpret_cast<const float4*>(part[g][d4]);
      acc.x += o.x;
      acc.y += o.y;
      acc.z += o.z;
      acc.w += o.w;
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const int64_t h = (int64_t)grp * a.hpg + hb * a.rows + row;
  reinterpret_cast<uint2*>(a.out + t * a.out_st + h * a.out_sh)[d4] =
      make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  if (a.lse != nullptr && d4 == 0)
    a.lse[t * a.lse_st + h] = l == 0.f ? -INFINITY : (m - bias) * kLn2 + logf(l);
}

// Self-test of the error path of fp4::wait: as wait_timeout_selftest_kernel, the same
// code (63) in this file's status word.
__device__ unsigned long long g_selftest_ns = 0;
__global__ void __launch_bounds__(32) wait_timeout_selftest_fp4_kernel(uint32_t looks) {
  __shared__ uint64_t bar;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bar), 1);
    mbar_init_fence();
  }
  __syncwarp();
  unsigned long long t0, t1;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  (void)wait<1>(bar, 0, 63, looks);
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1));
  if (threadIdx.x == 0) g_selftest_ns = t1 - t0;
}

}  // namespace

int launch_wait_timeout_selftest_fp4(uint32_t looks, uint64_t* elapsed_ns, cudaStream_t st) {
  wait_timeout_selftest_fp4_kernel<<<1, 32, 0, st>>>(looks);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  unsigned long long ns = 0;
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&ns, g_selftest_ns, sizeof(ns));
  *elapsed_ns = ns;
  return check_cuda(e, "wait timeout self-test");
}

int launch_merge_fp4(const Fp4DecodeArgs& a, float bias, cudaStream_t st) {
  if (a.workers < 2) return FP8MLA_OK;
  const int64_t units = (int64_t)a.T * a.G * a.hb_per_group;
  const cudaError_t e =
      units * 8 <= a.workers
          ? launch_pdl(merge_fp4_kernel<4>, dim3((unsigned)units, (unsigned)a.rows), dim3(512), 0, st, a, bias)
          : launch_pdl(merge_fp4_kernel<1>, dim3((unsigned)(a.workers - 1), (unsigned)a.rows), dim3(128), 0, st, a,
                       bias);
  return check_cuda(e, "merge_fp4_kernel launch");
}

int launch_decode_fp4(const Fp4DecodeArgs& a, bool cuts, cudaStream_t st) {
  CUtensorMap tm{};
  if (a.num_slots > 0)
    if (int rc = encode_fp4_row_map(&tm, a.kv, a.num_slots)) return rc;
  const size_t smem = sizeof(Smem) + 128;
  static SmemLimit limit;
  if (int rc = limit.raise(decode_fp4_kernel, smem)) return rc;
  if (int rc = check_cuda(launch_pdl(decode_fp4_kernel, dim3((unsigned)a.workers), dim3(kThreads), smem, st, a, tm),
                          "decode_fp4_kernel launch"))
    return rc;
  return cuts ? launch_merge_fp4(a, kBias, st) : FP8MLA_OK;
}

int read_device_status_fp4(unsigned int* status, bool reset, cudaStream_t st) {
  unsigned int v = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, tc::g_device_status, sizeof(v), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && reset && v != 0) {
    const unsigned int zero = 0;
    e = cudaMemcpyToSymbolAsync(tc::g_device_status, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  *status = v;
  return check_cuda(e, "device status read");
}

}  // namespace fp8mla

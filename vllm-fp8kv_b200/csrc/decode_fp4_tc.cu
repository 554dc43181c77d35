// decode_fp4_tc.cu -- attention over fp4_ds_mla rows for many heads: up to 128
// query heads per unit on a pair of SMs (a 2-CTA cluster) that share
// cta_group::2 tcgen05 MMAs.
//
//   S = scale q . [latent | rope],  P = softmax(S),  O = P . latent
//
// The pair splits the heads: CTA c owns heads [64c, +64) and its tensor memory
// holds their S and O.  A tile is 128 entries and an MMA spans both SMs:
//   S    M=128 heads, N=128 entries, K=576 (36 k-steps); CTA c supplies the rows
//        of its "own" entries [64c, +64)
//   O    M=128 heads, N=256 dims (two MMAs for the 512), K=128 entries; CTA c
//        supplies dims [128c, +128) of each MMA (latent tiles c and c + 2, its
//        "half") of all 128 entries
// A tile's 52 MMAs take 2200 cycles; 64-entry tiles would need 88 MMAs for the same
// entries.  K (own rows, 72 KB) and V (halves, 64 KB) are single in shared memory,
// in fp16; the 4-bit rows never lie there, they go from memory to registers a tile
// ahead.  Each buffer drains in parts: K in two groups of blocks, refilled for the
// next tile while the other group and the O product of the tile before are still
// running; V while the next tile's S runs.
//
// Measured, us: 64 x 128 heads x top-2048, paged: 54.6 (16 tiles a pair); its
// products take 22.5 at the rate of a large matrix product, its rows' bytes 8.3.
// A tile takes 4400 cycles.  What bounds it is the traffic of shared memory, about 3000
// cycles of it: K and V written (136 KB), read by the MMAs (192 KB), P, and the rows'
// way through the L1; S runs at half its rate beside the unpacking.  About 11 us go by
// before the first S (cold code, and a chain of three memory latencies: entries,
// block table, rows) and 5 behind the last P; a change of unit costs 9 (q, O).
// Steps on the way: 182 (64-entry tiles of mma.sync: 181), 112 one call per role, 79 waits
// that vote, 67 rows by way of registers, 65 the scout, 62 waits not unrolled and rows
// prefetched into L2, 56 rows read sector by sector.
//
// The latents are exact in fp16 (fp4.cuh), so the 32 latent k-steps of S and the
// O product are fp16 MMAs: q is converted, scaled per head by a power of two where
// it needs that (load_q), and P keeps 11 bits where bf16 keeps 8.  The
// rope's four k-steps are bf16 MMAs (q's rope times the same power of two) into
// the same accumulator.
//
// Units are dealt to the pairs in equal runs of tiles (decode_fp4.h).  Every role
// walks the run on its own; only q, the softmax state and O change at unit
// borders, and the next unit's q is in place before the last unit's O is stored.
//
// Accumulator layout of an M=128 pair MMA (measured): per CTA, lanes [0,64) hold
// its 64 rows x columns [0, N/2), lanes [64,128) the same rows x [N/2, N).  So
// softmax thread L owns head L & 63 and entries [64 (L >> 6), +64) of a tile.
//
// Tensor memory (512 columns, both CTAs):
//   [  0,256)  O, dims [0,256) MMA in [0,128), dims [256,512) MMA in [128,256)
//   [256,320)  S
//   [320,512)  q dims [0,384), the A operand of 24 k-steps (lanes L and L^64
//              hold the same head)
// Shared memory (217 KB):
//   q    dims [384,512) fp16, rope bf16: 3 x 64-dim swizzled blocks of 64 rows  24 KB
//   k    own 64 entries x 576 dims, 9 blocks of 64 rows                         72 KB
//   v    128 entries x this CTA's half, 4 blocks of 128 rows                    64 KB
//   p    P of 64 heads x 128 entries, 2 blocks                                  16 KB
//   stage  half of q's latents on their way in                                  33 KB
//
// Warp roles (512 threads per CTA; warp w runs on SM sub-partition w % 4):
//   warps 0-3         softmax, q, and the stores of O
//   warp 4            tensor memory allocation; the even CTA's issues every MMA of
//                     the pair
//   warps 5, 6, 7, 9  K: own rows [16i, +16) of every tile, loaded into registers
//                     a tile ahead -> K blocks
//   warps 10, 11, 13, 14
//                     V: the half of entries [32i, +32) of every tile, likewise
//   warp 15           scout: entries -> slots and live bits of all 128 entries
//   warps 8, 12       idle: sub-partition 0 runs the issuing warp and one softmax
//                     warp alone
// Barriers that gate the issuing thread live in the even CTA and count arrivals
// of both CTAs; the completion of pair MMAs reaches both CTAs through a multicast
// commit.  Every wait is bounded, and a role stops after a failed one.  No load uses
// cluster multicast; there are no copies that could outlive the CTA.
#include "decode_fp4.h"
#include "fp4.cuh"
#include "fp4_walk.cuh"
#include "tc_cluster.cuh"
#include "tc_ptx.cuh"

namespace fp8mla {
namespace {
using namespace fp8mla::fp4;
using namespace fp8mla::tc;

constexpr int kN = kFp4TcChunk;            // 128 entries per tile
constexpr int kOwn = kN / 2;
constexpr int kQBlockBytes = 64 * 128;
constexpr int kKBlockBytes = kOwn * 128;   // 8 KB: 64 own rows of a 64-dim block
constexpr int kVBlockBytes = kN * 128;     // 16 KB
constexpr int kPBlockBytes = 64 * 128;     // 64 heads x 64 entries
constexpr int kScoutRing = 4;               // tiles of slots
constexpr int kSoftmaxWarps = 4, kKWarps = 4, kVWarps = 4;
constexpr int kMmaWarp = 4;
constexpr int kThreads = 16 * 32;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 0, kColS = 256, kColQ = 320;
constexpr float kRescale = 8.0f;  // the reference maximum lags by at most 2^8 ...
constexpr float kBias = 6.0f;     // ... and P is stored times 2^6: below 2^14 in
                                  // fp16, above its smallest value from 2^-30 on

constexpr uint32_t idesc(int n, bool bf16, bool b_mn_major) {
  return bf16 ? idesc_bf16(128, n, b_mn_major)
              : idesc_bf16(128, n, b_mn_major) & ~((1u << 7) | (1u << 10));
}
constexpr uint32_t kIdescLatent = idesc(kN, false, false);
constexpr uint32_t kIdescRope = idesc(kN, true, false);
constexpr uint32_t kIdescPV = idesc(256, false, true);

struct Smem {
  uint8_t q[3 * kQBlockBytes];  // 1024-aligned (offset 0)
  uint8_t k[9 * kKBlockBytes];
  uint8_t v[4 * kVBlockBytes];
  uint8_t p[2 * kPBlockBytes];
  uint8_t stage[64][528];       // half a latent of every head (rows 4 banks apart)
  float half_max[2][128];       // a tile's maxima per thread, by tile parity
  float lsum[128];              // a finished piece: its sums per thread,
  int done_t, done_head, done_heads, done_row;  // token, first head, heads, first row of partials (< 0: none)
  uint32_t qmax[128];           // largest latent magnitudes per thread
  int qk[64], qagain[2];        // powers of two of the heads; any not 0 among 32
  int32_t slot[kScoutRing][kN];   // a tile's slots, and its live bits
  uint32_t vmask[kScoutRing][4];
  int piece_tiles[2];           // tiles of a piece, by its parity (softmax -> MMA)
  uint64_t kfull[2], kempty[2];  // K blocks [0,4) and [4,9); kfull: even CTA
  uint64_t vfull, pfull, sempty, qready, oempty;  // even CTA, both CTAs arrive
  uint64_t sfull, pvdone, ofull, drain;           // commits
  uint64_t slots_full[kScoutRing], slots_empty[kScoutRing];
  uint64_t meet;                // the softmax warps of this CTA
  Share share;
  uint32_t tmem_base;
};
static_assert(offsetof(Smem, k) % 1024 == 0 && offsetof(Smem, v) % 1024 == 0 && offsetof(Smem, p) % 1024 == 0,
              "swizzle atoms need 1024-B alignment");
static_assert(offsetof(Smem, kfull) % 8 == 0 && offsetof(Smem, stage) % 16 == 0, "");
static_assert(sizeof(Smem) + 1024 <= 227 * 1024, "shared memory budget");

__device__ __forceinline__ uint32_t swz(uint32_t r, uint32_t c) { return r * 128u + ((c ^ (r & 7u)) << 4); }

struct Ctx {
  const Fp4DecodeArgs* a;
  Smem* s;
  int worker;
  uint32_t rank, tmem;
  int64_t tiles;  // of this worker
};
__device__ __forceinline__ uint32_t bar(uint64_t& b) { return smem_u32(&b); }

// ------------------------------------------------------------------ MMA issuer (even CTA)
// The whole warp walks the issuing code, and each MMA and commit elects the lane
// that issues it (always the same one): control and addresses are then uniform
// over the warp and the operands stay in uniform registers, where the MMAs need
// them.  Measured on one pair alone, cycles per S / O MMA: 32.5 / 64.7 so, 54 / 65
// under `if (lane == 0)`.  The election stands in front of every instruction,
// which also keeps the warp converged: with one election for the whole role the
// lane parts from the others at the first commit, while the code goes on in
// registers that they share.
__device__ __forceinline__ void pair_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n elect.sync _|e, 0xFFFFFFFF;\n setp.ne.b32 p, %4, 0;\n"
      " @e tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void pair_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n elect.sync _|e, 0xFFFFFFFF;\n setp.ne.b32 p, %4, 0;\n"
      " @e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t& b) {
  asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xFFFFFFFF;\n"
      " @e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}\n" ::"r"(
          bar(b)),
      "h"((uint16_t)3)
      : "memory");
}
// The role is two short loops of four MMAs a turn, entered once a tile: code that
// is met again only a tile later is fetched anew each time.
__device__ void mma_role(const Ctx& c) {
  Smem& s = *c.s;
  const uint32_t tQ = c.tmem + kColQ, tS = c.tmem + kColS, tO = c.tmem + kColO;
  const uint64_t qdesc = sdesc_sw128(smem_u32(s.q), 16, 1024);
  const uint64_t kdesc = sdesc_sw128(smem_u32(s.k), 16, 1024);
  const uint64_t pdesc = sdesc_sw128(smem_u32(s.p), 16, 1024);
  const uint64_t vdesc = sdesc_sw128(smem_u32(s.v), kVBlockBytes, 1024);
  const uint32_t tiles = (uint32_t)c.tiles;
  uint32_t p = 0;      // pieces opened
  int left = 0;        // tiles of the open piece whose S is still to come
  bool first = false;  // the next O begins its piece
  auto ts_blocks = [&](int from, int to) {
#pragma unroll 1
    for (int b = from; b < to; ++b) {
      const uint64_t bd = kdesc + (uint64_t)((b * kKBlockBytes) >> 4);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        pair_ts(tS, tQ + 32 * b + 8 * i, bd + (uint64_t)(2 * i), kIdescLatent, (b | i) ? 1u : 0u);
    }
  };
  // S goes one tile ahead of O within a piece; a new piece, whose q may be long in
  // coming, waits until the O's of the one before are on their way
  uint32_t js = 0, jo = 0;  // next S, next O
  while (jo < tiles) {
    if (js < tiles && (js == jo || (js == jo + 1 && left > 0))) {
      if (left == 0) {
        if (!wait<1>(s.qready, p & 1, 35)) return;
        left = s.piece_tiles[p & 1];
        ++p;
        first = true;
      }
      if (js > 0 && !wait<1>(s.sempty, (js - 1) & 1, 34)) return;
      if (!wait<1>(s.kfull[0], js & 1, 37)) return;
      tc_fence_after();
      // K blocks 0-5: q in tensor memory
      ts_blocks(0, 4);
      commit(s.kempty[0]);
      if (!wait<1>(s.kfull[1], js & 1, 39)) return;
      tc_fence_after();
      ts_blocks(4, 6);
      // blocks 6, 7 (latents) and 8 (rope): q in shared memory
#pragma unroll 1
      for (int b = 0; b < 3; ++b) {
        const uint64_t ad = qdesc + (uint64_t)((b * kQBlockBytes) >> 4);
        const uint64_t bd = kdesc + (uint64_t)(((6 + b) * kKBlockBytes) >> 4);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          pair_ss(tS, ad + (uint64_t)(2 * i), bd + (uint64_t)(2 * i), b < 2 ? kIdescLatent : kIdescRope, 1u);
      }
      commit(s.kempty[1]);
      commit(s.sfull);
      ++js;
      --left;
    } else {
      if (first && p > 1 && !wait<1>(s.oempty, p & 1, 45)) return;  // of piece p - 2
      if (!wait<1>(s.pfull, jo & 1, 36)) return;
      if (!wait<1>(s.vfull, jo & 1, 38)) return;
      tc_fence_after();
      const uint32_t acc = first ? 0u : 1u;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {  // dims half h: entries [0,64) and [64,128)
        const uint64_t bd = vdesc + (uint64_t)((h * 2 * kVBlockBytes) >> 4);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          pair_ss(tO + 128 * h, pdesc + (uint64_t)(((i >> 2) * kPBlockBytes + (i & 3) * 32) >> 4),
                  bd + (uint64_t)((i * 16 * 128) >> 4), kIdescPV, i > 0 ? 1u : acc);
      }
      commit(s.pvdone);  // P and V may be written again
      ++jo;
      if (left == 0 && jo == js) commit(s.ofull);
      first = false;
    }
  }
}

// One warp of each CTA, when the last MMA has been issued: the even CTA's issuing warp,
// and in the odd CTA, where nobody issues, a softmax warp that has seen the last O (a
// warp that came here at the start would have to wait for as long as the call takes).
// Every arrival that is still on its way to one of
// this CTA's barriers is seen in before the CTA may exit (one that finds its
// target gone is an illegal access; the closing cluster barrier alone does not
// hold it back).  The drain commit arrives once every MMA is done.  Of the last
// tile, the multicast arrivals of the other commits and the odd CTA's release of
// S need not have been waited for by anyone; their earlier phases have been, so
// the parity names the right one.  (Every other arrival gates a wait, and oempty
// is not signalled for the last unit.)
__device__ void settle(const Ctx& c) {
  Smem& s = *c.s;
  if (c.rank == 0) commit(s.drain);
  if (!wait<1>(s.drain, 0, 46) || c.tiles == 0) return;
  const uint32_t par = (uint32_t)(c.tiles - 1) & 1;
  (void)(wait<1>(s.kempty[0], par, 48) && wait<1>(s.kempty[1], par, 48) &&
         wait<1>(s.pvdone, par, 48) &&
         (c.rank != 0 || wait<1>(s.sempty, par, 48)));
}

// ------------------------------------------------------------------ scout
// Entries -> slots for all 128 entries of a tile, up to four tiles ahead.
__device__ void scout(const Ctx& c, int lane) {
  const Fp4DecodeArgs& a = *c.a;
  Smem& s = *c.s;
  Slots<kN, 1, 4> slots(a, s.share, c.worker, lane, 0);
  int32_t early[2][4];
  slots.start(a, early);
  const int tiles = (int)c.tiles;
#pragma unroll 1
  for (int j = 0; j < tiles; ++j) {
    int32_t slot[4];
    if (j >= 2) {
      slots.next(a, slot, j == 2);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        slot[i] = early[0][i];
        early[0][i] = early[1][i];
      }
    }
    const int r = j % kScoutRing;
    if (j >= kScoutRing && !wait<1>(s.slots_empty[r], (uint32_t)(j / kScoutRing + 1) & 1, 40)) break;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s.slot[r][32 * i + lane] = slot[i];
      const uint32_t live = __ballot_sync(0xFFFFFFFFu, slot[i] >= 0);
      if (lane == 0) s.vmask[r][i] = live;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(s.slots_full[r]));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int32_t sl = c.rank == 0 ? slot[i] : slot[2 + i];
      if (sl >= 0) {
        const uint8_t* row = a.kv + (int64_t)sl * kFp4RowBytes;
#pragma unroll
        for (int x = 0; x < 4; ++x)
          asm volatile("prefetch.global.L2 [%0];\n" ::"l"(row + (x < 3 ? 128 * x : kFp4RowBytes - 1)));
      }
    }
  }
}

// ------------------------------------------------------------------ K and V
// Four lanes read a row of 8 (lane / 4), lane q of them the 32 code bytes of one
// 64-dim block: whole sectors, and one or two cache lines a row.  Stored in the same
// order, the four lanes' chunks would lie in the same banks of their four blocks; so
// lane q takes the block's two halves in the order i ^ (q & 1), and the words of each
// in the order s ^ (q & 2).  With the swizzle of the row, eight lanes then touch every
// bank once.
__device__ __forceinline__ void load32(uint4 (&w)[2], const uint8_t* at) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
               : "=r"(w[0].x), "=r"(w[0].y), "=r"(w[0].z), "=r"(w[0].w), "=r"(w[1].x), "=r"(w[1].y), "=r"(w[1].z),
                 "=r"(w[1].w)
               : "l"(at));
}
struct Codes {
  uint4 w[2];    // halves of the block
  uint32_t sc;   // its four scales
  __device__ __forceinline__ void load(const uint8_t* row, int at) {
    load32(w, row + at);
    sc = *reinterpret_cast<const uint32_t*>(row + kFp4ScaleOff + at / 8);
  }
  __device__ __forceinline__ void zero() {
    w[0] = w[1] = make_uint4(0, 0, 0, 0);
    sc = 0;
  }
  // to the block's row at `block`, row r of it
  __device__ __forceinline__ void store(uint32_t block, uint32_t r, int q) const;
};

// 32 codes and their two scales -> four 16-byte chunks of fp16 at `at` (the
// shared address of the first, swizzled: the others differ from it in bits 4 and
// 5).  Not inlined: one copy serves every use.
__device__ __noinline__ void unpack32(uint4 w, uint32_t scales, uint32_t at) {
  const uint32_t s2 = e4m3x2_to_f16(scales);
  const uint32_t sl = __byte_perm(s2, 0, 0x1010), sh = __byte_perm(s2, 0, 0x3232);
  const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h[4];
    e2m1x8_to_f16(word[i], h);
    const uint32_t sc = i < 2 ? sl : sh;
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(at ^ (16u * i)), "r"(mul_f16x2(h[0], sc)),
                 "r"(mul_f16x2(h[1], sc)), "r"(mul_f16x2(h[2], sc)), "r"(mul_f16x2(h[3], sc))
                 : "memory");
  }
}

__device__ __forceinline__ uint4 select(bool p, const uint4& x, const uint4& y) {
  return make_uint4(p ? x.x : y.x, p ? x.y : y.y, p ? x.z : y.z, p ? x.w : y.w);
}
__device__ __forceinline__ void Codes::store(uint32_t block, uint32_t r, int q) const {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t half = i ^ (q & 1);
    const bool turn = q & 2;
    const uint4 v = select(half, w[1], w[0]);
    // bytes 0 and 1: the scales of the words stored first and last
    const uint32_t s2 = __byte_perm(sc, 0, (half ? 0x32u : 0x10u) ^ (turn ? 0x11u : 0u));
    unpack32(select(turn, make_uint4(v.z, v.w, v.x, v.y), v), s2, (block + swz(r, 4 * half)) ^ (turn ? 32u : 0u));
  }
}

// K warp kw: own rows [16 kw, +16) of every tile, loaded into registers one tile
// ahead.
__device__ void k_role(const Ctx& c, int kw, int lane) {
  const Fp4DecodeArgs& a = *c.a;
  Smem& s = *c.s;
  const int r8 = lane >> 2, q = lane & 3;
  Codes w[2][2];  // [8 rows][group of blocks]
  uint4 rope[2][2];
  auto load = [&](uint32_t j) -> bool {
    const uint32_t r = j % kScoutRing;
    if (!wait<1>(s.slots_full[r], (j / kScoutRing) & 1, 41)) return false;
    const int32_t* at = s.slot[r] + kOwn * (int)c.rank + 16 * kw + r8;
    const int32_t slot[2] = {at[0], at[8]};
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(s.slots_empty[r]));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int32_t sl = slot[h];
      if (sl >= 0) {  // a masked row keeps what the registers hold: its score is replaced
        const uint8_t* row = a.kv + (int64_t)sl * kFp4RowBytes;
        w[h][0].load(row, 32 * q);
        w[h][1].load(row, 128 + 32 * q);
        load32(rope[h], row + kFp4RopeOff + 32 * q);
      }
    }
    return true;
  };
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[h][0].zero();
    w[h][1].zero();
    rope[h][0] = rope[h][1] = make_uint4(0, 0, 0, 0);
  }
  const uint32_t tiles = (uint32_t)c.tiles;
  bool ok = tiles > 0 && load(0);
  for (uint32_t j = 0; j < tiles && ok; ++j) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {  // blocks [0,4): latent tiles 0, 1; blocks [4,9): 2, 3 and the rope
      if (ok && j > 0) ok = wait<1>(s.kempty[g], (j - 1) & 1, 43);
      if (!ok) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t r = 16 * kw + 8 * h + r8;
        w[h][g].store(smem_u32(s.k + (4 * g + q) * kKBlockBytes), r, q);
        if (g == 1) {
          *reinterpret_cast<uint4*>(s.k + 8 * kKBlockBytes + swz(r, 2 * q)) = rope[h][0];
          *reinterpret_cast<uint4*>(s.k + 8 * kKBlockBytes + swz(r, 2 * q + 1)) = rope[h][1];
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(bar(s.kfull[g]), 0);
    }
    if (ok && j + 1 < tiles) ok = load(j + 1);  // behind the fences, so that none waits for loads
  }
}

// V warp vw: entries [32 vw, +32) of every tile, the CTA's half.
__device__ void v_role(const Ctx& c, int vw, int lane) {
  const Fp4DecodeArgs& a = *c.a;
  Smem& s = *c.s;
  const int r8 = lane >> 2, q = lane & 3;
  // latent tiles rank and rank + 2, two 64-dim blocks of each
  const int bytes = 64 * ((int)c.rank + 2 * (q >> 1)) + 32 * (q & 1);
  Codes w[4];
  auto load = [&](uint32_t j) -> bool {
    const uint32_t r = j % kScoutRing;
    if (!wait<1>(s.slots_full[r], (j / kScoutRing) & 1, 42)) return false;
    const int32_t* at = s.slot[r] + 32 * vw + r8;
    const int32_t slot[4] = {at[0], at[8], at[16], at[24]};
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(s.slots_empty[r]));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t sl = slot[i];
      if (sl >= 0) {
        const uint8_t* row = a.kv + (int64_t)sl * kFp4RowBytes;
        w[i].load(row, bytes);
      } else {  // zeros: P is 0 there, and nothing else may be
        w[i].zero();
      }
    }
    return true;
  };
  const uint32_t tiles = (uint32_t)c.tiles;
  bool ok = tiles > 0 && load(0);
  for (uint32_t j = 0; j < tiles && ok; ++j) {
    if (j > 0 && !wait<1>(s.pvdone, (j - 1) & 1, 44)) break;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i].store(smem_u32(s.v + q * kVBlockBytes), 32 * vw + 8 * i + r8, q);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive_cluster(bar(s.vfull), 0);
    if (j + 1 < tiles) ok = load(j + 1);  // behind the fence, so that it waits for no load
  }
}

// ------------------------------------------------------------------ softmax
// The four softmax warps of a CTA meet, with a bounded wait (a warp that gave up
// elsewhere never comes).
struct Meet {
  uint32_t n = 0;
  __device__ __forceinline__ bool operator()(Smem& s, int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(s.meet));
    return wait<1>(s.meet, n++ & 1, 47);
  }
};

// q of the unit (nh heads from q0 on): dims [0,384) -> tensor memory (lanes L and L^64 both hold head
// L & 63), the rest -> swizzled shared memory (thread hh writes chunks [4 hh, +4)
// of each block); padding rows are zero.  `scale` turns the head's accumulators
// into scores in log2 units.
// A thread needs its head's whole row, and 32 rows read 16 bytes at a time are 32
// lines an instruction; so a warp reads 512 bytes of one row an instruction, and
// the rows change hands in shared memory.  The copies are asynchronous:
// through registers, four rows at a time, each four waited for the ones before.
// Returns the scale, -1 after a failed wait.
__device__ __forceinline__ float load_q(Smem& s, const uint16_t* q0, int64_t q_sh, int nh, float scale_log2,
                                     uint32_t tmem, Meet meet) {
  const int L = threadIdx.x, m = L & 63, hh = L >> 6, lane = L & 31, warp = L >> 5;
  const uint4 z4 = make_uint4(0, 0, 0, 0);
  auto mag = [](const uint4& v) {
    return __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
  };
  const uint32_t trow = tmem + ((uint32_t)(warp * 32) << 16);
  // First as it is, which is exact enough where the head's largest latent magnitude
  // lies in [2^-2, 2^15] (an fp16 subnormal's error is below 2^-23 of it then).
  // Else again times 2^k (q_power).
  int k = 0;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    // the sign of the softmax scale goes with q, so that scores scale by a positive factor
    const float up = copysignf(__uint_as_float((uint32_t)(127 + k) << 23), scale_log2);
    auto f16 = [&](const uint4& v) {
      auto one = [&](uint32_t u) { return pack_f16x2(bf16_lo(u) * up, bf16_hi(u) * up); };
      return make_uint4(one(v.x), one(v.y), one(v.z), one(v.w));
    };
    uint32_t mx = 0;
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {  // latent dims [256 half, +256)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = 16 * warp + i;
        cp_async16(smem_u32(s.stage[r] + 16 * lane), q0 + (r < nh ? r : 0) * q_sh + 256 * half + 8 * lane, r < nh ? 16 : 0);  // zeros past nh
      }
      if (half == 1) {  // the rope, four rows an instruction
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * warp + 4 * i + (lane >> 3);
          const uint4 x = r < nh ? reinterpret_cast<const uint4*>(q0 + r * q_sh + kNope)[lane & 7] : z4;
          const float ur = pass == 0 ? up : copysignf(__uint_as_float((uint32_t)(127 + s.qk[r]) << 23), scale_log2);
          auto one = [&](uint32_t u) { return pack_bf16x2(bf16_lo(u) * ur, bf16_hi(u) * ur); };
          *reinterpret_cast<uint4*>(s.q + 2 * kQBlockBytes + swz(r, lane & 7)) =
              make_uint4(one(x.x), one(x.y), one(x.z), one(x.w));
        }
      }
      asm volatile("cp.async.wait_all;\n" ::: "memory");
      if (!meet(s, lane)) return -1.f;
      const uint4* row = reinterpret_cast<const uint4*>(s.stage[m]);
#pragma unroll 1
      for (int c0 = 0; c0 < (half == 0 ? 128 : 64); c0 += 32) {  // to tensor memory
        uint32_t o[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint4 x = row[c0 / 4 + i];
          mx = __vmaxu2(mx, mag(x));
          const uint4 v = f16(x);
          o[4 * i] = v.x;
          o[4 * i + 1] = v.y;
          o[4 * i + 2] = v.z;
          o[4 * i + 3] = v.w;
        }
        tmem_st32(trow + kColQ + 128 * half + c0, o);
      }
      if (half == 1) {  // dims [384,512) to shared memory
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint4 x = row[16 + 8 * (i >> 2) + 4 * hh + (i & 3)];
          mx = __vmaxu2(mx, mag(x));
          *reinterpret_cast<uint4*>(s.q + (i >> 2) * kQBlockBytes + swz(m, 4 * hh + (i & 3))) = f16(x);
        }
      }
      s.qmax[L] = max(mx & 0xFFFFu, mx >> 16);
      if (!meet(s, lane)) return -1.f;  // the stage has been read (and the maxima are in place)
    }
    tmem_wait_st();
    if (pass == 1) break;
    const int bm = (int)max(s.qmax[L], s.qmax[L ^ 64]);
    const bool again = bm != 0 && bm < 0x7F80 && (bm < 0x3E80 || bm > 0x4700);
    if (again) {
      uint32_t mr = 0;
      for (int i = 0; i < 8; ++i) mr = __vmaxu2(mr, mag(reinterpret_cast<const uint4*>(q0 + m * q_sh + kNope)[i]));
      const int br = (int)max(mr & 0xFFFFu, mr >> 16);
      k = q_power(bm, br, scale_log2);
    }
    if (hh == 0) s.qk[m] = k;
    const bool any = __any_sync(0xFFFFFFFFu, again);
    if (hh == 0 && lane == 0) s.qagain[warp] = any ? 1 : 0;
    if (!meet(s, lane)) return -1.f;
    if (s.qagain[0] == 0 && s.qagain[1] == 0) break;
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncwarp();
  const float scale = fabsf(scale_log2) * __uint_as_float((uint32_t)(127 - k) << 23);
  return scale == 0.f ? 1.1754944e-38f : scale;  // a masked score is an infinity times the scale
}
constexpr uint32_t kLoadMeets = 1;  // meetings of load_q, 5 or 9: only their parity counts

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// two fp32 operations in one instruction, each rounded as on its own
__device__ __forceinline__ float2 fma2(float2 v, float m, float a) {
  const float2 m2 = make_float2(m, m), a2 = make_float2(a, a);
  asm("fma.rn.f32x2 %0, %0, %1, %2;\n"
      : "+l"(reinterpret_cast<uint64_t&>(v))
      : "l"(reinterpret_cast<const uint64_t&>(m2)), "l"(reinterpret_cast<const uint64_t&>(a2)));
  return v;
}
__device__ __forceinline__ float2 add2(float2 v, float2 w) {
  asm("add.rn.f32x2 %0, %0, %1;\n"
      : "+l"(reinterpret_cast<uint64_t&>(v))
      : "l"(reinterpret_cast<const uint64_t&>(w)));
  return v;
}

// A whole sector of the thread's own row.
__device__ __forceinline__ void store32(void* dst, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

__device__ void softmax_role(const Ctx& c, int warp, int lane) {
  const Fp4DecodeArgs& a = *c.a;
  Smem& s = *c.s;
  const int L = threadIdx.x, m = L & 63, hh = L >> 6;
  const uint32_t trow = c.tmem + ((uint32_t)(warp * 32) << 16);
  Walk<kN> w(a, s.share, c.worker);
  bool ok = true;
  uint32_t j = 0, piece = 0;
  float scale = 0.f, m_ref = 0.f;
  Meet meet;
  const bool sectors = ((reinterpret_cast<uintptr_t>(a.out) | (a.out_st * 2) | (a.out_sh * 2)) & 31) == 0;
  // a turn: q of a piece, O of the piece before, the tiles of the piece
  while (w.left > 0 || piece > 0) {
    if (w.left > 0) {
      const int h0 = 64 * (int)c.rank, head0 = w.hb * a.rows + h0;  // of its group
      const int nh = max(0, min(64, min(a.rows - h0, a.hpg - head0)));
      scale = load_q(s, a.q + w.t * a.q_st + (int64_t)(w.grp * a.hpg + (nh > 0 ? head0 : 0)) * a.q_sh, a.q_sh, nh,
                     a.scale_log2, c.tmem, meet);
      if (scale < 0.f) break;
      meet.n += kLoadMeets;
      // (the piece two before this one, whose place it takes, is past its last S)
      if (L == 0) s.piece_tiles[piece & 1] = w.here();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(bar(s.qready), 0);
    }
    if (piece > 0) {
      if (!wait<1>(s.ofull, (piece - 1) & 1, 32)) break;
      tc_fence_after();
      const int t = s.done_t, head = s.done_head + m, prow = s.done_row + m;
      const bool hv = m < s.done_heads, whole = s.done_row < 0;
      const float lt = s.lsum[L] + s.lsum[L ^ 64];
      const float inv = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);
      if (hv && hh == 0) {
        if (whole) {
          if (a.lse != nullptr)
            a.lse[t * a.lse_st + head] = lt == 0.f ? -INFINITY : (m_ref - kBias) * kLn2 + logf(lt);
        } else {
          a.ws_ml[prow] = make_float2(m_ref, lt);
        }
      }
#pragma unroll 1
      for (int c0 = 0; c0 < 256; c0 += 32) {
        uint32_t o[32];
        tmem_ld32(trow + kColO + c0, o);
        tmem_wait_ld();
        const int d = 256 * (c0 >> 7) + 128 * hh + (c0 & 127);
        if (hv && whole) {
          uint16_t* dst = a.out + t * a.out_st + (int64_t)head * a.out_sh + d;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t v[8];
#pragma unroll
            for (int x = 0; x < 8; ++x)
              v[x] = pack_bf16x2(__uint_as_float(o[16 * e + 2 * x]) * inv, __uint_as_float(o[16 * e + 2 * x + 1]) * inv);
            if (sectors) {
              store32(dst + 16 * e, v);
            } else {
              reinterpret_cast<uint4*>(dst)[2 * e] = make_uint4(v[0], v[1], v[2], v[3]);
              reinterpret_cast<uint4*>(dst)[2 * e + 1] = make_uint4(v[4], v[5], v[6], v[7]);
            }
          }
        } else if (hv) {
          float* dst = a.ws_o + (int64_t)prow * kNope + d;
#pragma unroll
          for (int e = 0; e < 4; ++e) store32(dst + 8 * e, reinterpret_cast<uint32_t(&)[8]>(o[8 * e]));
        }
      }
      tc_fence_before();
      __syncwarp();
      // the next unit's O may begin (nobody waits behind the last one: see settle)
      if (lane == 0 && w.left > 0) mbar_arrive_cluster(bar(s.oempty), 0);
    }
    if (w.left <= 0) break;
    const int n = w.here();
    float l = 0.f;
    m_ref = -INFINITY;
    for (int i = 0; i < n; ++i, ++j) {
      const uint32_t par = j & 1;
      ok = wait<1>(s.sfull, par, 31);
      const uint32_t r = j % kScoutRing;
      if (ok) ok = wait<1>(s.slots_full[r], (j / kScoutRing) & 1, 30);
      if (!ok) break;
      const uint32_t live0 = s.vmask[r][2 * hh], live1 = s.vmask[r][2 * hh + 1];
      tc_fence_after();
      uint32_t sv[64];
      tmem_ld32(trow + kColS, reinterpret_cast<uint32_t(&)[32]>(sv[0]));
      tmem_ld32(trow + kColS + 32, reinterpret_cast<uint32_t(&)[32]>(sv[32]));
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive_cluster(bar(s.sempty), 0);  // S may be written again
        mbar_arrive(bar(s.slots_empty[r]));
      }
      if ((live0 & live1) != 0xFFFFFFFFu) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          if (!((live0 >> e) & 1u)) sv[e] = 0xFF800000u;  // -inf (the scale is positive)
          if (!((live1 >> e) & 1u)) sv[32 + e] = 0xFF800000u;
        }
      }
      float pm = __uint_as_float(sv[0]);
#pragma unroll
      for (int e = 1; e < 63; e += 2) pm = max3(pm, __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
      pm = fmaxf(pm, __uint_as_float(sv[63])) * scale;
      s.half_max[par][L] = pm;
      ok = meet(s, lane);
      if (!ok) break;
      const float tmax = fmaxf(pm, s.half_max[par][L ^ 64]);
      float alpha = 1.f;
      if (tmax > m_ref + kRescale || (m_ref == -INFINITY && tmax > -INFINITY)) {
        alpha = m_ref == -INFINITY ? 1.f : ex2_approx(m_ref - tmax);
        m_ref = tmax;
        l *= alpha;
      }
      const float sub = m_ref == -INFINITY ? 0.f : m_ref - kBias;
      // P, in registers until O of the tile before has read its P
      uint32_t pk[32];
      float2 l2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float2 x = fma2(make_float2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), scale, -sub);
        const float2 p2 = make_float2(ex2_approx(x.x), ex2_approx(x.y));
        l2 = add2(l2, p2);
        pk[e] = pack_f16x2(p2.x, p2.y);
      }
      l += l2.x + l2.y;
      if (j > 0) ok = wait<1>(s.pvdone, (j - 1) & 1, 33);
      if (!ok) break;
      if (__any_sync(0xFFFFFFFFu, alpha != 1.f) && i > 0) {
        tc_fence_after();
#pragma unroll 1
        for (int c0 = 0; c0 < 256; c0 += 32) {
          uint32_t o[32];
          tmem_ld32(trow + kColO + c0, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st32(trow + kColO + c0, o);
        }
        tmem_wait_st();
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        *reinterpret_cast<uint4*>(s.p + hh * kPBlockBytes + swz(m, e)) =
            make_uint4(pk[4 * e], pk[4 * e + 1], pk[4 * e + 2], pk[4 * e + 3]);
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(bar(s.pfull), 0);
    }
    if (!ok) break;
    // the piece's sums and place, for the stores of its O
    s.lsum[L] = l;
    if (L == 0) {
      const int h0 = 64 * (int)c.rank;  // of the unit
      s.done_t = (int)w.t;
      s.done_head = w.grp * a.hpg + w.hb * a.rows + h0;
      s.done_heads = min(a.rows - h0, a.hpg - w.hb * a.rows - h0);
      s.done_row = w.c == 0 && n == w.n ? -a.rows : (2 * c.worker + (w.c == 0 ? 1 : 0)) * a.rows + h0;
    }
    if (!meet(s, lane)) break;
    w.next_unit(a, n);
    ++piece;
  }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    decode_fp4_tc_kernel(const __grid_constant__ Fp4DecodeArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  Smem& s = *reinterpret_cast<Smem*>(smem_raw + (((raw_base + 1023u) & ~1023u) - raw_base));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Ctx c;
  c.a = &a;
  c.s = &s;
  c.worker = blockIdx.x >> 1;
  c.rank = cluster_rank();  // == blockIdx.x & 1

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(s.kfull[i]), 2 * kKWarps);
      mbar_init(bar(s.kempty[i]), 1);
    }
    for (int i = 0; i < kScoutRing; ++i) {
      mbar_init(bar(s.slots_full[i]), 1);
      mbar_init(bar(s.slots_empty[i]), kKWarps + kVWarps + kSoftmaxWarps);
    }
    mbar_init(bar(s.vfull), 2 * kVWarps);
    mbar_init(bar(s.pfull), 2 * kSoftmaxWarps);
    mbar_init(bar(s.sempty), 2 * kSoftmaxWarps);
    mbar_init(bar(s.qready), 2 * kSoftmaxWarps);
    mbar_init(bar(s.oempty), 2 * kSoftmaxWarps);
    mbar_init(bar(s.sfull), 1);
    mbar_init(bar(s.pvdone), 1);
    mbar_init(bar(s.ofull), 1);
    mbar_init(bar(s.drain), 1);
    mbar_init(bar(s.meet), kSoftmaxWarps);
    mbar_init_fence();
  }
  if (warp == kMmaWarp) {
    tmem_alloc_pair(smem_u32(&s.tmem_base), kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // barriers of both CTAs initialised, tensor memory allocated
  tc_fence_after();
  if (threadIdx.x == 0) pdl_launch_dependents();
  pdl_wait();  // the previous kernel of the stream has completed: global memory from here on
  c.tmem = s.tmem_base;
  divide<kN, kThreads>(a, s.share, c.worker);
  if (threadIdx.x == 0 && c.rank == 0) note_start<kN>(a, s.share, c.worker);
  c.tiles = max((int64_t)0, Walk<kN>(a, s.share, c.worker).left);

  // one call per role: the loops of all roles together have to stay in the SM's
  // instruction cache (with each role inlined twice, and the unpacking and the
  // softmax unrolled in full, warps waited for instructions most of the time:
  // 182 instead of 112 us at 64 x 128 heads x top-2048)
  if (warp < kSoftmaxWarps) {
    softmax_role(c, warp, lane);
  } else if (warp == kMmaWarp) {
    if (c.rank == 0) mma_role(c);
  } else if (warp < 8 || warp == 9) {
    k_role(c, warp < 8 ? warp - 5 : 3, lane);
  } else if (warp == 15) {
    scout(c, lane);
  } else if (warp != 8 && warp != 12) {
    v_role(c, warp < 12 ? warp - 10 : warp - 11, lane);
  }

  if (warp == (c.rank == 0 ? kMmaWarp : 0)) settle(c);

  // both CTAs: no MMA of the pair may still run, no arrival may still target the
  // other CTA, before tensor memory is freed and the CTAs exit
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc_pair(c.tmem, kTmemCols);
  }
}

}  // namespace

int launch_decode_fp4_tc(const Fp4DecodeArgs& a, bool cuts, cudaStream_t st) {
  const size_t smem = sizeof(Smem) + 1024;  // + alignment slack
  static SmemLimit limit;
  if (int rc = limit.raise(decode_fp4_tc_kernel, smem)) return rc;
  if (int rc = check_cuda(launch_pdl(decode_fp4_tc_kernel, dim3((unsigned)(2 * a.workers)), dim3(kThreads), smem, st,
                                     a),
                          "decode_fp4_tc_kernel launch"))
    return rc;
  return cuts ? launch_merge_fp4(a, kBias, st) : FP8MLA_OK;
}

int read_device_status_fp4_tc(unsigned int* status, bool reset, cudaStream_t st) {
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

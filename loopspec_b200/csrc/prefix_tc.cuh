// Shared-prefix attention on the 5th-generation tensor cores, for many query
// rows a kv head (the formulas and types are in prefix_attn.cuh; the terms of
// an fp32 q are tiles beside each other in shared memory, those of P columns
// beside each other in tensor memory, and the products add up).
//
// A unit is (MT row tiles of 128, kv head, key range). Either the rows are
// query heads of any requests and the keys a range of the prefix (they are the
// same for all; the result is a part to be joined), or, where requests bring
// whole tiles of rows (prompts), the rows are one request's and the keys a
// range of the prefix followed by the request's own positions; with one range
// that is the whole result, which is normalised and stored.
// One CTA a unit:
//   2 or 3 producer warps gather K and V rows, a tile of 128 keys each in turn,
//     through the block table with 16-byte cp.async into a ring of
//     128-byte-swizzled tiles;
//   one warp issues S = Q K^T and O += P V (tcgen05.mma, M = 128): K is the
//     K-major operand as gathered, V the MN-major one, so neither is moved
//     again; S and O live in tensor memory;
//   8 MT softmax warps: two threads a row, 64 of the tile's 128 scores each
//     (with one thread a row two warps an SM quarter could not cover each
//     other's latencies: 3200-3500 cycles a pair of tiles). They agree on the
//     row's maximum through shared memory and write P over S in the operand's
//     type (the A operand of the second product comes from tensor memory). O
//     is rescaled only when a row's maximum has grown by more than 2^8 since
//     its reference was set: until then the old reference stays, weights reach
//     2^8, and nothing else changes, as the reference cancels in o / l. With terms
//     of an fp32 q they also add up the tiles' products themselves.
// With MT = 2 the tensor cores work on one row tile while the softmax warps
// work on the other; with MT = 1 on the next key tile (two score buffers).
//
// Bound: for prompts the softmax warps' issue slots (58 % used, the
// exponentials' unit 60 %, with the waits on tensor memory between) beside the
// tensor cores: 4 prompts of up to 700 tokens behind 8192 positions, 32 heads of
// 128, 293-326 us by the clock under load, 1.0-0.9 PFLOP/s, six tenths of a library
// product's rate; 8 of up to 509 behind 16384, 32 heads of 64, 648 us, 0.65 PFLOP/s,
// as half as many dimensions come with each exponential. fp32 q: 4 prompts of up to
// 400 behind 4096, 16 heads of 128, 165 us (bf16 cache, three terms), 134 (f16, two).
// For decode batches the gathering of K
// and V: 64 requests behind 32768 positions 61 us with their own positions and
// the joining pass, 203 MB, 3.3 TB/s.
//
// A row must not see what later tokens of its request hold: their scores leave
// by selection, but a weight of 0 times a NaN or infinity in V is NaN. So the
// producers look at the V rows that only some of a unit's rows see (at most as
// many as the unit has tokens), copy zeros for one that is not finite, and
// note it; the rows that do see it add its term at the end.
#pragma once

#include "prefix_attn.cuh"

namespace ls {

constexpr int kTcKeys = 128;          // keys of a tile
constexpr int kTcRows = 128;          // rows of a tile

template <int HD, int TERMS, int MT>
struct TcLayout {
  static_assert(TERMS == 1 || MT == 1, "the terms of q and P take the second row tile's room");
  static constexpr int kTile = kTcKeys * HD * 2;           // bytes of a K, V or Q tile
  static constexpr int kProducer = 8 * MT;                 // first producer warp
  static constexpr int kStages = HD == 64 ? 8 : TERMS == 3 ? 4 : TERMS * MT == 2 ? 5 : 6;
  // A producer waits for a stage by the parity of its turn, which is only right
  // while the turn before that one is over. Copy i waits for copy i - ST to be
  // used; its warp has seen copy i - P - ST used, and copies are used in order
  // but for neighbours (K of a tile before V of the one ahead), so copy
  // i - 2 ST is over for certain if ST >= P + 2.
  static constexpr int kProducers = kStages >= 5 ? 3 : 2;
  static_assert(kStages >= kProducers + 2, "a stage's turns would be mistaken for one another");
  static constexpr int kMma = kProducer + kProducers;      // the issuing warp
  // The tensor cores' sums lose their lower bits towards zero with every addition,
  // so the error of one sum over a unit's keys grows with their number: with fp32
  // queries 2.0e-5 of the output behind 8192 positions, 3.9e-5 behind 16384. With
  // terms of an fp32 q each key tile's product is therefore a sum of its own, and
  // the softmax warps add them up in registers, rounding to nearest: 7e-7 to 9e-7 at
  // any length. (With 16-bit q the rounding of P is a hundred times that.)
  static constexpr bool kOwnSums = TERMS > 1;
  static constexpr bool kShareRegs = MT == 2 || kOwnSums;
  static constexpr int kSoftWarps = 8 * MT;
  // a whole number of warpgroups where registers are handed over
  static constexpr int kThreads = kShareRegs ? 32 * (kSoftWarps + 4) : 32 * (kMma + 1);
  static_assert(kThreads >= 32 * (kMma + 1), "a warp for each role");
  // The softmax warps draw on what the last four warps give back. With MT = 2 a
  // thread is launched with 96 registers: 640 x 96 = 512 x 104 + 128 x 64; with
  // sums of their own with 168: 384 x 168 = 256 x 200 + 128 x 104 (with 56 left to
  // the two or three producers they hold up the rest: 1600 tokens behind 4096, fp32
  // on bf16, heads of 128: 196 us, 165 with 104, 172 without handing over).
  static constexpr int kSoftRegs = MT == 2 ? 104 : 200, kRestRegs = MT == 2 ? 64 : 104;
  static constexpr int kLaunchRegs = kShareRegs ? (32 * kSoftWarps * kSoftRegs + 128 * kRestRegs) / kThreads : 0;
  static constexpr int kMaxBuffers = MT == 1 ? 2 : 1;      // see the softmax warps
  static constexpr int kBars = 2 * kStages + 2 + 2 + 2 + 2 + 1 + 1;
  static constexpr int kQTiles = MT * TERMS;
  static constexpr int kRowScales = TERMS == 2 ? kTcRows : 0;   // see kScaledRows
  static constexpr int kSmem = kQTiles * kTile + kStages * kTile + (kMaxBuffers * MT * 2 * kTcRows + kRowScales) * 4 + kBars * 8 +
                               8 * 4 + 16;
  // Eighths of the exponentials on the FMA units. The softmax is bound by issue
  // slots: with heads of 128 the tensor cores take longer and none is best
  // (0, 1, 2, 3 eighths: 289, 296, 308, 326 us for 2100 tokens behind 8192
  // positions), with heads of 64 one (740, 648, 672, 672 us for 3050 behind 16384;
  // with one it also depends on how the compiler orders the loop: 645 to 760 us).
  static constexpr int kPoly = TERMS == 1 && HD == 64 ? 1 : 0;
  // tensor memory columns: two buffers of scores, each with room for P's terms (64 each) over them, then O
  static constexpr uint32_t kScores = 0, kBuffer = TERMS == 3 ? 192 : 128, kOut = 2 * kBuffer;
  static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");
};

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// The issuing warp runs its loop as one: every lane computes the same operands,
// which keeps them in uniform registers, and only the instruction itself is
// predicated on the elected lane. (With the loop inside `if (lane == 0)` each
// product cost ~70 cycles to issue, twice what N = 64 needs to execute.)
// Matrix descriptors are passed by their low words; `hi` is the same for all.
__device__ __forceinline__ void tc_mma_ss(uint32_t leader, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %0, 0;\n\t"
      "mov.b64 a, {%2, %4};\n\tmov.b64 b, {%3, %4};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], a, b, %5, p;\n\t}" ::"r"(leader),
      "r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem], A packed two 16-bit values a column.
__device__ __forceinline__ void tc_mma_ts(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t hi,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %0, 0;\n\t"
      "mov.b64 b, {%3, %4};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], b, %5, p;\n\t}" ::"r"(leader),
      "r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tc_commit_if(uint32_t leader, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}" ::"r"(leader),
      "r"(bar)
      : "memory");
}

__device__ __forceinline__ uint32_t elect_one() {
  uint32_t leader;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(leader));
  return leader;
}

// Low word of a 128-byte-swizzled operand's descriptor. K-major: rows of 128
// bytes, 8-row groups 1024 bytes apart (`mn_bytes` unused). MN-major: 64
// elements of MN a row, 8 rows of K a group, the next 64 of MN `mn_bytes` away.
__device__ __forceinline__ uint32_t umma_lo(uint32_t smem_addr, uint32_t mn_bytes) {
  return ((smem_addr >> 4) & 0x3FFF) | ((mn_bytes >> 4) << 16);
}
// High word: group stride 1024, descriptor version 1, 128-byte swizzle.
constexpr uint32_t kUmmaHi = (1024u >> 4) | (1u << 14) | (2u << 29);

template <typename C>
__host__ __device__ constexpr uint32_t tc_idesc(int M, int N, bool b_mn_major) {
  const uint32_t type = std::is_same<C, __half>::value ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// 32 lanes x 32 consecutive columns a warp.
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// Wait for this thread's loads into r. The registers pass through the wait, so
// that no arithmetic on them is moved ahead of it.
template <int N>
__device__ __forceinline__ void tmem_ld_done(uint32_t (&r)[N]) {
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i])::"memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Packed pairs of fp32 (one instruction for two).
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ float2 unpair(uint64_t a) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(a));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// As max2_nan, of three.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x of a pair on the FMA units, for 16-bit weights: x = n + f with n = round(x)
// (added to 1.5 * 2^23 it sits in the low mantissa bits), |f| <= 1/2, 2^f by the
// cubic that minimises the largest relative error there (Remez exchange: 7.5e-5,
// a fiftieth of bf16's half unit, a seventh of f16's), times 2^n put together
// from its exponent bits: 0 from n = -127 on down, so a masked score weighs
// nothing. NaN is not passed on: a row with a NaN score has a NaN reference, whose
// other exponentials are NaN, and a reference of +inf makes the row's sum NaN.
__device__ __forceinline__ uint64_t exp2_poly(uint64_t x) {
  constexpr float kMagic = 12582912.f;
  const float2 v = unpair(x);
  x = pair(fmaxf(v.x, -127.f), fmaxf(v.y, -127.f));
  const uint64_t t = add2(x, pair(kMagic, kMagic));
  const uint64_t f = fma2(add2(t, pair(-kMagic, -kMagic)), pair(-1.f, -1.f), x);
  uint64_t y = fma2(f, pair(0.055171669f, 0.055171669f), pair(0.24261112f, 0.24261112f));
  y = fma2(y, f, pair(0.69326099f, 0.69326099f));
  y = fma2(y, f, pair(0.99992807f, 0.99992807f));
  const float2 n = unpair(t);
  return mul2(y, pair(__uint_as_float((__float_as_uint(n.x) << 23) + 0x3f800000u),
                      __uint_as_float((__float_as_uint(n.y) << 23) + 0x3f800000u)));
}

// Polls of one wait before it gives up: a poll that finds nothing suspends for
// microseconds, the longest wait of a sound run is a few hundred.
constexpr uint32_t kTcWaitLimit = 1u << 20;

// Wait unless an earlier wait timed out. A warp whose wait times out does not
// leave its loop: it waits no more and goes on over what is there, so that no
// lane and no warp is missing from a collective or a barrier of the others; the
// status word tells. (A vote on the outcome would cost 31 cycles a wait, a
// barrier that is ready 13.)
__device__ __forceinline__ void wait_on(bool& ok, uint32_t bar, uint32_t parity, int* err, int code) {
  if (ok && !mbar_try_wait(bar, parity)) {
    uint32_t i = 0;
    while (i < kTcWaitLimit && !mbar_try_wait(bar, parity)) ++i;
    ok = i < kTcWaitLimit;
    if (!ok) atomicCAS(err, kDevOk, code);
  }
}

// Arrive on `bar` once this thread's cp.async copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}


__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void cp_async16_to(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// Columns first .. first + HD / 2 of a row by the formula in fp32, by one thread.
template <int HD, typename Q, typename C>
__device__ __noinline__ void redo_row(PoolView<C> pools, KeyRanges keys, const Q* q, float scale_log2, Q* dst, int first) {
  const int all = keys_in(keys);
  float m = -INFINITY;
  for (int i = 0; i < all; ++i) m = max2_nan(m, score_of<HD>(pools, slot_of(pools, keys, i), q, scale_log2));
  const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 1
  for (int d0 = first; d0 < first + HD / 2; d0 += 8) {   // a few at a time: an array by itself would be in memory
    float l = 0.f, acc[8] = {};
    for (int i = 0; i < all && m == m; ++i) {
      const long slot = slot_of(pools, keys, i);
      const float w = exp2_fast(score_of<HD>(pools, slot, q, scale_log2) - base);
      l += w;
      if (slot < 0) continue;
#pragma unroll
      for (int d = 0; d < 8; ++d) acc[d] += w * (float)pools.v[slot * pools.stride + d0 + d];
    }
#pragma unroll
    for (int d = 0; d < 8; ++d) dst[d0 + d] = (Q)(m == m ? acc[d] / l : m);
  }
}

// Whether 8 packed 16-bit values hold a NaN or infinity (exponent bits all set).
template <typename C>
__device__ __forceinline__ bool not_finite8(const uint4& v) {
  constexpr uint32_t kExp = std::is_same<C, __half>::value ? 0x7C00u : 0x7F80u;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & kExp) == kExp || ((w[i] >> 16) & kExp) == kExp;
  return bad;
}

// grid: 1-D over (row tile fastest, kv head, part, request if `own`): CTAs that run together read the same keys.
template <int HD, typename Q, typename C, int TERMS, int MT>
__global__ void __launch_bounds__(TcLayout<HD, TERMS, MT>::kThreads, 1) prefix_tc_kernel(PrefixAttnArgs a) {
  using L = TcLayout<HD, TERMS, MT>;
  constexpr int ST = L::kStages;
  constexpr int CH = HD / 8;                       // 16-byte chunks of a row
  constexpr uint32_t kBlock = kTcRows * 128;       // bytes of 64 columns of a tile
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* s_q = smem;
  unsigned char* s_ring = smem + L::kQTiles * L::kTile;
  float* s_max = reinterpret_cast<float*>(s_ring + ST * L::kTile);   // [kMaxBuffers][MT][half][row]
  float* s_scale = s_max + L::kMaxBuffers * MT * 2 * kTcRows;        // [kRowScales]
  const uint32_t bars = smem_u32(s_scale + L::kRowScales);
  uint32_t* s_bad = reinterpret_cast<uint32_t*>(s_scale + L::kRowScales) + 2 * L::kBars;   // [8] bits
  uint32_t* s_tmem = s_bad + 8;
  const uint32_t full0 = bars, empty0 = full0 + 8 * ST, s_full = empty0 + 8 * ST, p_full = s_full + 16,
                 pv_done = p_full + 16, o_done = pv_done + 16, q_full = o_done + 16, noted = q_full + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the first kernel of a call: launched early, it waits for what came before,
  // and only then lets the next one start
  pdl_wait();
  pdl_launch_dependents();

  // the unit: its rows, and its keys as prefix positions [ka0, ka1) and own positions [kb0, kb1)
  const int G = a.nh / a.nkv;
  unsigned u = blockIdx.x;
  const int tile = (int)(u % (unsigned)a.prefix_tiles);
  u /= (unsigned)a.prefix_tiles;
  const int g = (int)(u % (unsigned)a.nkv);
  u /= (unsigned)a.nkv;
  const unsigned n_parts = max(1, a.prefix_parts);
  const int part = (int)(u % n_parts), req = (int)(u / n_parts);
  int start = 0, n_new = a.n_tokens, len = 0;
  if (a.own && !request_range(a, req, start, n_new, len)) return;
  const int rows = n_new * G;                      // rows of the kv head
  const int row0 = tile * (MT * kTcRows);
  if (row0 >= rows) return;
  const int seen0 = len - n_new + 1;               // own positions the request's first new token sees
  // A part is a run of key tiles: of the prefix's, followed by the request's own if `own`.
  const int j0 = part * (a.prefix_chunk / kTcKeys), j1 = j0 + a.prefix_chunk / kTcKeys;
  const int n_shared = (a.prefix_len + kTcKeys - 1) / kTcKeys;
  const int ka0 = min(a.prefix_len, j0 * kTcKeys), ka1 = min(a.prefix_len, j1 * kTcKeys);
  const int last_row = min(rows, row0 + MT * kTcRows) - 1;
  const int see_first = seen0 + div_by(row0, G, a.g_magic);          // own positions every row sees, and some row sees
  const int kb0 = max(0, j0 - n_shared) * kTcKeys;
  const int kb1 = a.own ? min(max(0, j1 - n_shared) * kTcKeys, min(len, seen0 + div_by(last_row, G, a.g_magic))) : 0;
  const int na = (ka1 - ka0 + kTcKeys - 1) / kTcKeys;
  const int n = na + (max(0, kb1 - kb0) + kTcKeys - 1) / kTcKeys;    // key tiles
  const int* own_table = a.block_table + req * a.table_stride;

  // softmax warps of a row tile's half with rows of their own; the others have nothing to do
  auto live_warps = [&](int t) { return max(0, min(4, (rows - row0 - t * kTcRows + 31) / 32)); };
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(full0 + 8 * s, 32);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(s_full + 8 * b, 1);
      // with MT = 2 a buffer belongs to a row tile; one without rows is never used
      mbar_init(p_full + 8 * b, max(1, 2 * live_warps(MT == 2 ? b : 0)));
      mbar_init(pv_done + 8 * b, 1);
      mbar_init(o_done + 8 * b, 1);
    }
    mbar_init(q_full, 8 * MT);
    mbar_init(noted, L::kProducers);
    for (int i = 0; i < 8; ++i) s_bad[i] = 0;
    fence_barrier_init();
  }
  if (warp == L::kMma) {
    tmem_alloc(smem_u32(s_tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const int tiles_here = MT == 2 && live_warps(1) > 0 ? 2 : 1;   // row tiles with rows

  if (warp < L::kProducer) {
    // ---------------------------------------------------------------- softmax
    if (L::kShareRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kSoftRegs));
    const int t = MT == 2 ? warp >> 3 : 0, half = (warp >> 2) & 1, quarter = warp & 3;
    // the row tile's queries, swizzled; rows past the last are zeros
    {
      unsigned char* dst = s_q + t * L::kTile;
      const Q* q = static_cast<const Q*>(a.q);
      Raw8<Q> v[CH / 2];                             // all of them on their way at once
#pragma unroll
      for (int k = 0; k < CH / 2; ++k) {
        const int i = (threadIdx.x & 255) + 256 * k, r = i / CH, c = i % CH, rr = row0 + t * kTcRows + r;
        v[k] = Raw8<Q>();
        if (rr < rows) {
          const int tok = div_by(rr, G, a.g_magic), h = g * G + rr - tok * G;
          v[k].load(q + (long)(start + tok) * a.q_stride + (long)h * HD + c * 8);
        }
      }
#pragma unroll
      for (int k = 0; k < CH / 2; ++k) {
        const int i = (threadIdx.x & 255) + 256 * k, r = i / CH, c = i % CH;
        unsigned char* to = dst + (c >> 3) * kBlock + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        if constexpr (TERMS == 1) {                  // q is of the cache's type: as it is
          *reinterpret_cast<uint4*>(to) = v[k].v[0];
        } else {
          float f[8];
          v[k].get(f);
          if constexpr (kScaledRows<TERMS, C>) {
            float most = 0.f;
#pragma unroll
            for (int x = 0; x < 8; ++x) most = fmaxf(most, fabsf(f[x]));
#pragma unroll
            for (int x = 1; x < CH; x <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));   // CH lanes a row
            const int shift = row_shift(most);
            const float up = power2(shift);
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] *= up;
            if (c == 0) s_scale[r] = a.scale_log2 * power2(-shift);
          }
          uint32_t term[4][TERMS];
#pragma unroll
          for (int x = 0; x < 4; ++x) split2<TERMS, C>(f[2 * x], f[2 * x + 1], term[x]);
#pragma unroll
          for (int x = 0; x < TERMS; ++x)
            *reinterpret_cast<uint4*>(to + x * L::kTile) = make_uint4(term[0][x], term[1][x], term[2][x], term[3][x]);
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      if constexpr (kScaledRows<TERMS, C>) asm volatile("bar.sync 9, 256;" ::: "memory");   // the row tile's scales are there
    }
    const int r = quarter * 32 + lane, rr = row0 + t * kTcRows + r;
    if (quarter < live_warps(t)) {
      const int pair_bar = 1 + t * 4 + quarter;      // the two warps of 32 rows
      const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
      const uint32_t out = lanes + L::kOut + t * 128 + half * (HD / 2);
      // own positions this row sees, within the unit's
      const int row_tok = div_by(rr, G, a.g_magic);
      const int see = rr < rows ? min(kb1, seen0 + row_tok) : kb1;
      const int see_least = __reduce_min_sync(0xffffffffu, see);
      const float scale_log2 = kScaledRows<TERMS, C> ? s_scale[r] : a.scale_log2;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      float own_sum[L::kOwnSums ? HD / 2 : 1] = {};
      auto add_product = [&](float keep) {           // ... and all of it brought to the new one
        uint32_t v[HD / 2];
#pragma unroll
        for (int c = 0; c < HD / 2; c += 32) tmem_ld_x32(out + c, v + c);
        tmem_ld_done(v);
#pragma unroll
        for (int i = 0; i < (L::kOwnSums ? HD / 2 : 0); ++i) own_sum[i] = (own_sum[i] + __uint_as_float(v[i])) * keep;
      };
      for (int j = 0; j < n; ++j) {
        const int b = MT == 1 ? j & 1 : t;
        const uint32_t ph = (MT == 1 ? j >> 1 : j) & 1;
        // keys of this tile that the row sees, counted from this thread's first
        int left = (j < na ? ka1 - ka0 - j * kTcKeys : see - kb0 - (j - na) * kTcKeys) - half * 64;
        const bool cut = j < na ? j == na - 1 : see_least - kb0 - (j - na) * kTcKeys < kTcKeys;
        wait_on(ok, s_full + 8 * b, ph, a.status, kDevTimeoutAcc);
        tc_fence_after();
        const uint32_t sc = lanes + L::kScores + b * L::kBuffer;
        uint32_t s[64];
        tmem_ld_x32(sc + half * 64, s);
        tmem_ld_x32(sc + half * 64 + 32, s + 32);
        tmem_ld_done(s);
        if (cut) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i >= left) s[i] = 0xff800000u;     // -inf
        }
        float mx[4] = {m, m, m, m};
#pragma unroll
        for (int i = 0; i < 64; i += 2)
          mx[(i >> 1) & 3] = max3_nan(mx[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        float top = max2_nan(max2_nan(mx[0], mx[1]), max2_nan(mx[2], mx[3]));
        // The other half's maximum. The barrier also tells that both have read
        // their scores, which P is written over. One buffer does for MT = 2: the
        // next tile's scores come only after both have finished this one.
        float* row_max = s_max + ((MT == 1 ? j & 1 : t) * 2) * kTcRows + r;
        row_max[half * kTcRows] = top;
        tc_fence_before();
        asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
        tc_fence_after();
        top = max2_nan(top, row_max[(half ^ 1) * kTcRows]);
        // m and top are raw scores; their distance counts after the scale. A NaN
        // score makes the reference NaN, and with it the whole row
        const bool move = m == -INFINITY ? top != -INFINITY : !((top - m) * scale_log2 <= kGrow);
        float keep = 1.f;
        if (__any_sync(0xffffffffu, move)) {
          keep = move && m > -INFINITY ? exp2_fast((m - top) * scale_log2) : 1.f;
          if (move) m = top;
          // inf - inf: the row is NaN, whichever way its weights are computed
          l = m == INFINITY ? NAN : l * keep;
          if (!L::kOwnSums && j > 0) {
            wait_on(ok, pv_done + 8 * t, (j - 1) & 1, a.status, kDevTimeoutAcc);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 2; c += 16) {
              uint32_t v[16];
              tmem_ld_x16(out + c, v);
              tmem_ld_done(v);
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * keep);
              tmem_st_x16(out + c, v);
            }
          }
        }
        const float base = (m == -INFINITY ? 0.f : m * scale_log2) - weight_bias(C());
        // Of eight pairs kPoly go to the FMA units, the others to the special
        // function units, which do 4 of these a cycle and SM quarter
        const uint64_t scale = pair(scale_log2, scale_log2), minus = pair(-base, -base);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int i0 = 0; i0 < 32; i0 += 16) {
          uint32_t p[TERMS][16];
#pragma unroll
          for (int i = i0; i < i0 + 16; ++i) {
            const uint64_t x = fma2(pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale, minus);
            uint64_t w;
            if ((i * L::kPoly) % 8 < L::kPoly) {
              w = exp2_poly(x);
            } else {
              const float2 v = unpair(x);
              w = pair(exp2_fast(v.x), exp2_fast(v.y));
            }
            sum[i & 1] = add2(sum[i & 1], w);
            const float2 v = unpair(w);
            uint32_t term[TERMS];
            split2<TERMS, C>(v.x, v.y, term);
#pragma unroll
            for (int x = 0; x < TERMS; ++x) p[x][i - i0] = term[x];
          }
#pragma unroll
          for (int x = 0; x < TERMS; ++x) tmem_st_x16(sc + x * 64 + half * 32 + i0, p[x]);
        }
        const float2 total = unpair(add2(sum[0], sum[1]));
        l += total.x + total.y;
        if constexpr (L::kOwnSums) {
          if (j > 0) {                               // the product of the tile before this one, by the old reference
            wait_on(ok, pv_done + 8 * t, (j - 1) & 1, a.status, kDevTimeoutAcc);
            tc_fence_after();
            add_product(keep);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * b);
      }
      // join the two halves' sums; a wait that timed out leaves zeros
      if (n > 0) wait_on(ok, o_done + 8 * t, 0, a.status, kDevTimeoutAcc);
      if (a.own) wait_on(ok, noted, 0, a.status, kDevTimeoutAcc);
      const bool have = n > 0 && ok;
      tc_fence_after();
      if constexpr (L::kOwnSums) {                   // the sum takes the last product's place
        add_product(1.f);
#pragma unroll
        for (int c = 0; c < HD / 2; c += 16) tmem_st_x16(out + c, reinterpret_cast<const uint32_t*>(own_sum + c));
        tmem_st_wait();
      }
      float* row_sum = s_max + ((MT == 1 ? n & 1 : t) * 2) * kTcRows + r;
      row_sum[half * kTcRows] = l;
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
      l = row_sum[0] + row_sum[kTcRows];
      const int tok = start + row_tok, h = g * G + rr - row_tok * G;
      // zeros for a row that sees nothing; one whose scores are all -inf is 0 / 0
      const bool nothing = a.prefix_len == 0 && see <= 0;
      const float inv = !have ? 0.f : !a.direct ? 1.f : nothing ? 0.f : 1.f / l;
      const float base = (m == -INFINITY ? 0.f : m * scale_log2) - weight_bias(C());
      const long at = ((long)part * a.n_tokens + tok) * a.nh + h;
      float zero = 0.f;                              // NaN if some output is not finite
      if (!a.direct && rr < rows && half == 0)
        a.part_ml[at] = have ? make_float2(m * scale_log2, l) : make_float2(-INFINITY, 0.f);
      // Parts leave by a patch of the row tile's queries, which are done with:
      // a warp's rows by CW columns, 16-byte chunks swizzled, so that it stores
      // whole rows of 4 CW bytes (a thread storing its own row by itself
      // touches 32 lines with every instruction: 8000 cycles for the tile).
      constexpr int CW = HD / 4, CPR = CW / 4;
      unsigned char* patch = s_q + t * L::kTile + (half * 4 + quarter) * (32 * CW * 4);
      auto place = [&](int row, int chunk) {
        return reinterpret_cast<float4*>(patch + row * (CW * 4) + ((chunk ^ (CPR == 8 ? row & 7 : (row >> 1) & 3)) << 4));
      };
#pragma unroll 1
      for (int c = 0; c < HD / 2; c += 16) {
        uint32_t v[16];
        tmem_ld_x16(out + c, v);
        tmem_ld_done(v);
        float f[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = have ? __uint_as_float(v[i]) * inv : 0.f;
        const int d = half * (HD / 2) + c;
        if (a.own && have && rr < rows) {            // terms left out of the products
          for (int w = 0; w < 8; ++w)
            for (uint32_t bits = s_bad[w]; bits; bits &= bits - 1) {
              const int pos = see_first + w * 32 + __ffs(bits) - 1;
              if (pos >= see) continue;
              const long slot = ((long)own_table[pos >> a.page_shift] << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
              const C* k = static_cast<const C*>(a.k_pool) + slot * a.slot_stride + (long)g * HD;
              const C* v = static_cast<const C*>(a.v_pool) + slot * a.slot_stride + (long)g * HD + d;
              const float p = weight_of<HD>(static_cast<const Q*>(a.q) + (long)tok * a.q_stride + (long)h * HD, k, base,
                                            a.scale_log2) * inv;
#pragma unroll
              for (int i = 0; i < 16; ++i) f[i] += p * (float)v[i];
            }
        }
        if constexpr (kTermsLose<Q, C>) {
#pragma unroll
          for (int i = 0; i < 16; ++i) zero = fmaf(f[i], 0.f, zero);
        }
        if (a.direct) {
          if (rr < rows) {
            Q* dst = static_cast<Q*>(a.out) + (long)tok * a.out_stride + (long)h * HD + d;
            store8(dst, *reinterpret_cast<float(*)[8]>(f));
            store8(dst + 8, *reinterpret_cast<float(*)[8]>(f + 8));
          }
          continue;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) *place(lane, (c % CW) / 4 + i) = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
        if ((c + 16) % CW) continue;
        __syncwarp();
#pragma unroll
        for (int k = 0; k < CPR; ++k) {
          const int row = k * (32 / CPR) + lane / CPR, chunk = lane % CPR;
          const long to = __shfl_sync(0xffffffffu, at, row);
          if (row0 + t * kTcRows + quarter * 32 + row < rows)
            store4(a.part_o + to * HD + half * (HD / 2) + c + 16 - CW + chunk * 4, *place(row, chunk));
        }
        __syncwarp();
      }
      if constexpr (kTermsLose<Q, C>) {
        if (a.direct && zero != 0.f && have && rr < rows)
          redo_row<HD>(PoolView<C>(a, g, HD), KeyRanges{a.prefix_table, ka0, ka1, own_table, kb0, see},
                       static_cast<const Q*>(a.q) + (long)tok * a.q_stride + (long)h * HD, a.scale_log2,
                       static_cast<Q*>(a.out) + (long)tok * a.out_stride + (long)h * HD, half * (HD / 2));
      }
      tc_fence_before();
    }
  } else if (L::kShareRegs) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kRestRegs));
  }
  if (warp >= L::kProducer && warp < L::kMma) {
    // --------------------------------------------------------------- producer
    constexpr int RPI = 32 / CH;                   // rows copied at a time
    const int c = lane % CH, hi = lane / CH;
    const C* kp = static_cast<const C*>(a.k_pool) + (long)g * HD + c * 8;
    const C* vp = static_cast<const C*>(a.v_pool) + (long)g * HD + c * 8;
    const int mask = (1 << a.page_shift) - 1;
    const uint32_t dst0 = smem_u32(s_ring) + (c >> 3) * kBlock + hi * 128;
    // Copy i (2 j: K of tile j, 2 j + 1: its V) goes to stage i % ST and is the
    // work of warp i % kProducers; the barrier counts each thread's part in when it has
    // landed, so the producers run a ring ahead. Lane l knows the slots of rows
    // l, l + 32, l + 64, l + 96; their blocks are loaded a copy ahead.
    int next[4];
    auto look_up = [&](int i) {
      const int j = i >> 1;
      const bool own = j >= na;
      const int* table = own ? own_table : a.prefix_table;
      const int pos = (own ? kb0 + (j - na) * kTcKeys : ka0 + j * kTcKeys) + lane, end = i >= 2 * n ? 0 : own ? kb1 : ka1;
#pragma unroll
      for (int q = 0; q < 4; ++q) next[q] = pos + 32 * q < end ? table[(pos + 32 * q) >> a.page_shift] : 0;
    };
    const int first = warp - L::kProducer;
    bool ok = true;
    look_up(first);
    for (int i = first; i < 2 * n; i += L::kProducers) {
      const int j = i >> 1, st = i % ST;
      const bool own = j >= na, is_v = i & 1;
      const int pos = (own ? kb0 + (j - na) * kTcKeys : ka0 + j * kTcKeys) + lane, end = own ? kb1 : ka1;
      int slot[4];                                 // -1: filled with zeros
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int at = pos + 32 * q;
        const long sl = ((long)next[q] << a.page_shift) + (at & mask);
        const bool fits = next[q] >= 0 && sl < a.n_slots;
        if (!fits && at < end) atomicCAS(a.status, kDevOk, kDevBadIndex);
        slot[q] = fits && at < end ? (int)sl : -1;
      }
      look_up(i + L::kProducers);
      if (own && is_v) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int at = pos + 32 * q;
          if (slot[q] >= 0 && at >= see_first) {   // a row that only some of the unit's rows see
            const C* row = static_cast<const C*>(a.v_pool) + (long)slot[q] * a.slot_stride + (long)g * HD;
            bool bad = false;
            for (int x = 0; x < HD; x += 8) bad |= not_finite8<C>(*reinterpret_cast<const uint4*>(row + x));
            if (bad) {
              atomicOr(s_bad + ((at - see_first) >> 5), 1u << ((at - see_first) & 31));
              slot[q] = -1;
            }
          }
        }
        __syncwarp();
      }
      if (i >= ST) wait_on(ok, empty0 + 8 * st, (i / ST - 1) & 1, a.status, kDevTimeoutEmpty);
      const uint32_t dst = dst0 + st * L::kTile;
      const C* src = is_v ? vp : kp;
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int x = 0; x < 32 / RPI; ++x) {
          const int row_slot = __shfl_sync(0xffffffffu, slot[q], x * RPI + hi);
          const int r = x * RPI + hi;              // the swizzle goes by the row modulo 8
          cp_async16_to(dst + (32 * q + x * RPI) * 128 + (((c & 7) ^ (r & 7)) << 4),
                        src + (long)max(row_slot, 0) * a.slot_stride, row_slot >= 0);
        }
      cp_async_arrive(full0 + 8 * st);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(noted);
    cp_async_commit();
    cp_async_wait<0>();
  } else if (warp == L::kMma) {
    // ------------------------------------------------------------------- issue
    constexpr uint32_t idesc_s = tc_idesc<C>(kTcRows, kTcKeys, false);
    constexpr uint32_t idesc_o = tc_idesc<C>(kTcRows, HD, true);
    const uint32_t leader = elect_one();
    const uint32_t ring_k = umma_lo(smem_u32(s_ring), 0), ring_v = umma_lo(smem_u32(s_ring), kBlock),
                   q0 = umma_lo(smem_u32(s_q), 0);
    bool ok = n > 0;
    auto wait_full = [&](int i) {
      wait_on(ok, full0 + 8 * (i % ST), (i / ST) & 1, a.status, kDevTimeoutFull);
      fence_proxy_async();                         // copies came by the generic proxy; the products read by the async one
    };
    auto release = [&](int i) {                    // copy i's stage, if another copy will want it
      if (i + ST < 2 * n) tc_commit_if(leader, empty0 + 8 * (i % ST));
    };
    auto scores = [&](int t, int b, int j) {       // S[b] = Q[t] K[j]^T, smallest terms first
      const uint32_t k = ring_k + ((2 * j % ST) * L::kTile >> 4), q = q0 + (t * L::kTile >> 4);
#pragma unroll
      for (int x = TERMS - 1; x >= 0; --x)
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          const uint32_t off = ((i >> 2) * kBlock + (i & 3) * 32) >> 4;
          tc_mma_ss(leader, tmem + L::kScores + b * L::kBuffer, q + (x * L::kTile >> 4) + off, k + off, kUmmaHi, idesc_s,
                    i != 0 || x != TERMS - 1);
        }
      tc_commit_if(leader, s_full + 8 * b);
    };
    auto outputs = [&](int t, int b, int j) {      // O[t] += P[b] V[j]
      const uint32_t v = ring_v + (((2 * j + 1) % ST) * L::kTile >> 4);
#pragma unroll
      for (int x = TERMS - 1; x >= 0; --x)
#pragma unroll
        for (int i = 0; i < kTcKeys / 16; ++i)
          tc_mma_ts(leader, tmem + L::kOut + t * 128, tmem + L::kScores + b * L::kBuffer + x * 64 + i * 8,
                    v + (i * 2048 >> 4), kUmmaHi, idesc_o,
                    i != 0 || x != TERMS - 1 ? 1u : L::kOwnSums ? 0u : (uint32_t)(j != 0));
      // A softmax warp at tile j may wait for product j - 1: it knows of j - 2, so
      // the turn is plain. For the last product, which it could be two turns
      // ahead of, there is a barrier of its own.
      tc_commit_if(leader, pv_done + 8 * t);
      if (j == n - 1) tc_commit_if(leader, o_done + 8 * t);
    };
    if (n > 0) {
      wait_on(ok, q_full, 0, a.status, kDevTimeoutFull);
      wait_full(0);
      tc_fence_after();
      for (int t = 0; t < tiles_here; ++t) scores(t, t, 0);
      release(0);
    }
    for (int j = 0; j < n; ++j) {
      const bool more = j + 1 < n;
      if (more) wait_full(2 * j + 2);
      if (MT == 1 && more) {
        // the buffer's P was consumed by the product issued before this one
        tc_fence_after();
        scores(0, (j + 1) & 1, j + 1);
        release(2 * j + 2);
      }
      wait_full(2 * j + 1);
      for (int t = 0; t < tiles_here; ++t) {
        const int b = MT == 1 ? j & 1 : t;
        wait_on(ok, p_full + 8 * b, (MT == 1 ? j >> 1 : j) & 1, a.status, kDevTimeoutAcc);
        tc_fence_after();
        outputs(t, b, j);
        if (t + 1 == tiles_here) release(2 * j + 1);
        if (MT == 2 && more) {
          scores(t, t, j + 1);
          if (t + 1 == tiles_here) release(2 * j + 2);
        }
      }
    }
    // No product is under way when the tensor memory is given back: the softmax
    // warps have seen the last ones end, unless a wait of theirs timed out.
    bool ended = n > 0;
    for (int t = 0; t < tiles_here; ++t) wait_on(ended, o_done + 8 * t, 0, a.status, kDevTimeoutAcc);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == L::kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace ls

// Shared-prefix attention on the 5th-generation tensor cores: the prefix units
// of a batch with 16-bit queries (the formulas are in prefix_attn.cuh).
//
// A unit is (MT row tiles of 128, kv head, key range); its rows are query
// heads of any requests, since the prefix is the same for all. One CTA a unit:
//   4 producer warps gather the range's K and V rows, 128 keys at a time,
//     through the prefix's block table with 16-byte cp.async into a ring of
//     128-byte-swizzled tiles;
//   one thread issues S = Q K^T and O += P V (tcgen05.mma, M = 128): K is the
//     K-major operand as gathered, V the MN-major one, so neither is moved
//     again; S and O live in tensor memory;
//   4 MT softmax warps own a row a thread: no reduction crosses threads. A
//     thread reads its 128 scores, writes P over them in the operand's type
//     (the A operand of the second product comes from tensor memory) and keeps
//     the running maximum and sum. O is rescaled only when a row's maximum has
//     grown by more than 2^8 since its reference was set: until then the old
//     reference stays, weights reach 2^8, and nothing else changes, as the
//     reference cancels in o / l.
// With MT = 2 the tensor cores work on one row tile while the softmax warps
// work on the other; with MT = 1 on the next key tile (two score buffers).
#pragma once

#include "prefix_attn.cuh"

namespace ls {

constexpr int kTcKeys = 128;          // keys of a tile
constexpr int kTcRows = 128;          // rows of a tile
constexpr float kTcGrow = 8.f;        // log2 growth of a row's maximum that moves its reference

template <int HD, int MT>
struct TcLayout {
  static constexpr int kThreads = MT == 1 ? 384 : 512;
  static constexpr int kProducer = 4 * MT;                 // first producer warp
  static constexpr int kMma = kProducer + 4;               // the issuing warp
  static constexpr int kTile = kTcKeys * HD * 2;           // bytes of a K, V or Q tile
  static constexpr int kStages = HD == 64 ? 8 : MT == 1 ? 6 : 5;
  static constexpr int kBars = 2 * kStages + 2 + 2 + 2 + 1;
  static constexpr int kSmem = MT * kTile + kStages * kTile + 2 * kTcKeys * 4 + kBars * 8 + 16;
  static constexpr int kPoly = 3;                          // eighths of the exponentials on the FMA units
  static constexpr uint32_t kScores = 0, kOut = 256;       // tensor memory columns
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

#define LS_TMEM32(r)                                                                                          \
  r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7], r[8], r[9], r[10], r[11], r[12], r[13], r[14], r[15], r[16], \
      r[17], r[18], r[19], r[20], r[21], r[22], r[23], r[24], r[25], r[26], r[27], r[28], r[29], r[30], r[31]

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

__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
#undef LS_TMEM32

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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x of a pair on the FMA units, for 16-bit weights: x = n + f with n = round(x)
// (added to 1.5 * 2^23 it sits in the low mantissa bits), |f| <= 1/2, 2^f by the
// cubic that minimises the largest relative error there (Remez exchange: 7.5e-5,
// a fiftieth of bf16's half unit, a seventh of f16's), n added to the exponent.
// Below 2^-126 the result stays about 2^-127 instead of 0.
__device__ __forceinline__ uint64_t exp2_poly(uint64_t x) {
  constexpr float kMagic = 12582912.f;
  const float2 v = unpair(x);
  x = pair(fmaxf(v.x, -126.f), fmaxf(v.y, -126.f));
  const uint64_t t = add2(x, pair(kMagic, kMagic));
  const uint64_t f = fma2(add2(t, pair(-kMagic, -kMagic)), pair(-1.f, -1.f), x);
  uint64_t y = fma2(f, pair(0.055171669f, 0.055171669f), pair(0.24261112f, 0.24261112f));
  y = fma2(y, f, pair(0.69326099f, 0.69326099f));
  y = fma2(y, f, pair(0.99992807f, 0.99992807f));
  const float2 n = unpair(t), r = unpair(y);
  return pair(__uint_as_float(__float_as_uint(r.x) + (__float_as_uint(n.x) << 23)),
              __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(n.y) << 23)));
}

// A whole warp's wait: all lanes agree on the outcome, so none leaves the others in a collective.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code));
}

// Arrive on `bar` once this thread's cp.async copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void producers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// grid: 1-D over (row tile fastest, kv head, part): CTAs that run together read the same keys.
template <int HD, typename C, int MT>
__global__ void __launch_bounds__(TcLayout<HD, MT>::kThreads, 1) prefix_tc_kernel(PrefixAttnArgs a) {
  using L = TcLayout<HD, MT>;
  constexpr int ST = L::kStages;
  constexpr int CH = HD / 8;                       // 16-byte chunks of a row
  constexpr uint32_t kBlock = kTcRows * 128;       // bytes of 64 columns of a tile
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* s_q = smem;
  unsigned char* s_ring = smem + MT * L::kTile;
  int* s_slot = reinterpret_cast<int*>(s_ring + ST * L::kTile);      // [2][kTcKeys]
  const uint32_t bars = smem_u32(s_slot + 2 * kTcKeys);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_slot + 2 * kTcKeys + 2 * L::kBars);
  const uint32_t full0 = bars, empty0 = full0 + 8 * ST, s_full = empty0 + 8 * ST, p_full = s_full + 16,
                 pv_done = p_full + 16, q_full = pv_done + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int G = a.nh / a.nkv;
  const int tile = blockIdx.x % a.prefix_tiles;
  const int g = (blockIdx.x / a.prefix_tiles) % a.nkv;
  const int part = blockIdx.x / a.prefix_tiles / a.nkv;
  const int rows = a.n_tokens * G;                 // rows of the kv head
  const int row0 = tile * (MT * kTcRows);
  const int k0 = part * a.prefix_chunk, k1 = min(a.prefix_len, k0 + a.prefix_chunk);
  const int n = (k1 - k0 + kTcKeys - 1) / kTcKeys; // key tiles, at least one

  // softmax warps with rows of their own; the others have nothing to do
  auto live_warps = [&](int t) { return max(0, min(4, (rows - row0 - t * kTcRows + 31) / 32)); };
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(full0 + 8 * s, 128);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(s_full + 8 * b, 1);
      // with MT = 2 a buffer belongs to a row tile; one without rows is never used
      mbar_init(p_full + 8 * b, max(1, live_warps(MT == 2 ? b : 0)));
      mbar_init(pv_done + 8 * b, 1);
    }
    mbar_init(q_full, 4 * MT);
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
  pdl_launch_dependents();

  if (warp < L::kProducer) {
    // ---------------------------------------------------------------- softmax
    if (MT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int t = warp >> 2, quarter = warp & 3;
    // the row tile's queries, swizzled; rows past the last are zeros
    {
      unsigned char* dst = s_q + t * L::kTile;
      const C* q = static_cast<const C*>(a.q);
      for (int i = threadIdx.x & 127; i < kTcRows * CH; i += 128) {
        const int r = i / CH, c = i % CH, rr = row0 + t * kTcRows + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (rr < rows) {
          const int tok = rr / G, h = g * G + rr - tok * G;
          v = *reinterpret_cast<const uint4*>(q + (long)tok * a.q_stride + (long)h * HD + c * 8);
        }
        *reinterpret_cast<uint4*>(dst + (c >> 3) * kBlock + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    const int r = quarter * 32 + lane, rr = row0 + t * kTcRows + r;
    if (quarter < live_warps(t)) {
      const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
      const uint32_t out = lanes + L::kOut + t * 128;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < n && ok; ++j) {
        const int b = MT == 1 ? j & 1 : t;
        const uint32_t ph = (MT == 1 ? j >> 1 : j) & 1;
        ok = warp_wait(s_full + 8 * b, ph, a.status, kDevTimeoutAcc);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sc = lanes + L::kScores + b * 128;
        uint32_t s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_x32(sc + 32 * c, s + 32 * c);
        tmem_ld_wait();
        if (j == n - 1) {                          // keys past the range
          const int left = k1 - k0 - j * kTcKeys;
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i >= left) s[i] = 0xff800000u;     // -inf
        }
        float mx[4] = {m, m, m, m};
#pragma unroll
        for (int i = 0; i < 128; i += 2)
          mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        // m and top are raw scores; their distance counts after the scale
        const bool move = m == -INFINITY ? top != -INFINITY : (top - m) * a.scale_log2 > kTcGrow;
        if (__any_sync(0xffffffffu, move)) {
          const float keep = move && m != -INFINITY ? exp2_fast((m - top) * a.scale_log2) : 1.f;
          if (move) m = top;
          l *= keep;
          if (j > 0) {
            ok = warp_wait(pv_done + 8 * t, (j - 1) & 1, a.status, kDevTimeoutAcc);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint32_t v[32];
              tmem_ld_x32(out + c, v);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * keep);
              tmem_st_x32(out + c, v);
            }
          }
        }
        const float base = (m == -INFINITY ? 0.f : m * a.scale_log2) - weight_bias(C());
        // Of eight pairs kPoly go to the FMA units, the others to the special
        // function units, which do 4 of these a cycle and SM quarter
        const uint64_t scale = pair(a.scale_log2, a.scale_log2), minus = pair(-base, -base);
        uint64_t sum[2] = {0, 0};
        uint32_t p[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) {
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
          p[i] = pack2(v.x, v.y, C());
          if (i == 31) tmem_st_x32(sc, p);
        }
        tmem_st_x32(sc + 32, p + 32);
        const float2 total = unpair(add2(sum[0], sum[1]));
        l += total.x + total.y;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * b);
      }
      if (ok) ok = warp_wait(pv_done + 8 * t, (n - 1) & 1, a.status, kDevTimeoutAcc);
      tc_fence_after();
      long at = 0;
      if (rr < rows) {
        const int tok = rr / G;
        at = ((long)part * a.n_tokens + tok) * a.nh + g * G + rr - tok * G;
        a.part_ml[at] = ok ? make_float2(m * a.scale_log2, l) : make_float2(-INFINITY, 0.f);
      }
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t v[32];
        tmem_ld_x32(out + c, v);
        tmem_ld_wait();
        if (rr < rows) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(a.part_o + at * HD + c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      }
      tc_fence_before();
    }
  } else if (warp < L::kMma) {
    // --------------------------------------------------------------- producer
    if (MT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const int tid = threadIdx.x - 32 * L::kProducer;
    constexpr int RPI = 128 / CH;                  // rows copied at a time by the 4 warps
    const int c = tid % CH, r0 = tid / CH;
    const C* kp = static_cast<const C*>(a.k_pool) + (long)g * HD + c * 8;
    const C* vp = static_cast<const C*>(a.v_pool) + (long)g * HD + c * 8;
    const int mask = (1 << a.page_shift) - 1;
    // the block of key `tid` of tile j: loaded a tile ahead, looked at when its turn comes
    auto block_of = [&](int j) {
      const int pos = k0 + j * kTcKeys + tid;
      return pos < k1 ? a.prefix_table[pos >> a.page_shift] : 0;
    };
    int next = block_of(0);
    bool ok = true;
    // copy i (2 j: K, 2 j + 1: V) goes to stage i % ST; the barrier counts each
    // thread's part in when it has landed, so the producers run a ring ahead
    int issued = 0;
    // after a wait that timed out the warp copies no more but stays in the barriers
    for (int j = 0; j < n; ++j) {
      int* slots = s_slot + (j & 1) * kTcKeys;
      const int pos = k0 + j * kTcKeys + tid;
      const long sl = ((long)next << a.page_shift) + (pos & mask);
      const bool fits = next >= 0 && sl < a.n_slots;
      if (!fits && pos < k1) atomicCAS(a.status, kDevOk, kDevBadIndex);
      slots[tid] = fits && pos < k1 ? (int)sl : -1;   // -1: filled with zeros
      if (j + 1 < n) next = block_of(j + 1);
      producers_sync();
#pragma unroll 1
      for (int kv = 0; kv < 2 && ok; ++kv) {
        const int st = issued % ST;
        if (issued >= ST) ok = warp_wait(empty0 + 8 * st, (issued / ST - 1) & 1, a.status, kDevTimeoutEmpty);
        if (!ok) break;
        unsigned char* dst = s_ring + st * L::kTile + (c >> 3) * kBlock;
        const C* src = kv ? vp : kp;
#pragma unroll
        for (int i = 0; i < kTcKeys / RPI; ++i) {
          const int r = r0 + i * RPI;
          const int slot = slots[r];
          cp_async16(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4), src + (long)max(slot, 0) * a.slot_stride, slot >= 0);
        }
        cp_async_arrive(full0 + 8 * st);
        ++issued;
      }
    }
    cp_async_commit();
    cp_async_wait<0>();
  } else {
    // ------------------------------------------------------------------- issue
    if (MT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == L::kMma) {
      constexpr uint32_t idesc_s = tc_idesc<C>(kTcRows, kTcKeys, false);
      constexpr uint32_t idesc_o = tc_idesc<C>(kTcRows, HD, true);
      const uint32_t leader = elect_one();
      const uint32_t ring_k = umma_lo(smem_u32(s_ring), 0), ring_v = umma_lo(smem_u32(s_ring), kBlock),
                     q0 = umma_lo(smem_u32(s_q), 0);
      auto wait_full = [&](int i) {
        const bool ok = warp_wait(full0 + 8 * (i % ST), (i / ST) & 1, a.status, kDevTimeoutFull);
        fence_proxy_async();                       // copies came by the generic proxy; the products read by the async one
        tc_fence_after();
        return ok;
      };
      auto release = [&](int i) {                  // copy i's stage, if another copy will want it
        if (i + ST < 2 * n) tc_commit_if(leader, empty0 + 8 * (i % ST));
      };
      auto scores = [&](int t, int b, int j) {     // S[b] = Q[t] K[j]^T
        const uint32_t k = ring_k + ((2 * j % ST) * L::kTile >> 4), q = q0 + (t * L::kTile >> 4);
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          const uint32_t off = ((i >> 2) * kBlock + (i & 3) * 32) >> 4;
          tc_mma_ss(leader, tmem + L::kScores + b * 128, q + off, k + off, kUmmaHi, idesc_s, i != 0);
        }
        tc_commit_if(leader, s_full + 8 * b);
      };
      auto outputs = [&](int t, int b, int j) {    // O[t] += P[b] V[j]
        const uint32_t v = ring_v + (((2 * j + 1) % ST) * L::kTile >> 4);
#pragma unroll
        for (int i = 0; i < kTcKeys / 16; ++i)
          tc_mma_ts(leader, tmem + L::kOut + t * 128, tmem + L::kScores + b * 128 + i * 8, v + (i * 2048 >> 4), kUmmaHi,
                    idesc_o, i != 0 ? 1u : (uint32_t)(j != 0));
        tc_commit_if(leader, pv_done + 8 * t);
      };
      bool ok = warp_wait(q_full, 0, a.status, kDevTimeoutFull) && wait_full(0);
      if (ok) {
        for (int t = 0; t < tiles_here; ++t) scores(t, t, 0);
        release(0);
      }
      for (int j = 0; j < n && ok; ++j) {
        const bool more = j + 1 < n;
        if (MT == 1) {
          // the buffer's P was consumed by the product issued before this one
          if (more) {
            if (!(ok = wait_full(2 * j + 2))) break;
            scores(0, (j + 1) & 1, j + 1);
            release(2 * j + 2);
          }
          ok = wait_full(2 * j + 1) && warp_wait(p_full + 8 * (j & 1), (j >> 1) & 1, a.status, kDevTimeoutAcc);
          if (!ok) break;
          tc_fence_after();
          outputs(0, j & 1, j);
          release(2 * j + 1);
        } else {
          if (!(ok = wait_full(2 * j + 1))) break;
          for (int t = 0; t < tiles_here; ++t) {
            if (!(ok = warp_wait(p_full + 8 * t, j & 1, a.status, kDevTimeoutAcc))) break;
            tc_fence_after();
            outputs(t, t, j);
            if (t + 1 == tiles_here) release(2 * j + 1);
            if (more) {
              if (t == 0 && !(ok = wait_full(2 * j + 2))) break;
              scores(t, t, j + 1);
              if (t + 1 == tiles_here) release(2 * j + 2);
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == L::kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace ls

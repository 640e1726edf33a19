// Attention of a batch whose requests share a long prefix, over paged K/V.
//
// Token t of request i (n_i new tokens, len_i own positions including them)
// attends to every prefix position and to its own positions
// 0 .. len_i - n_i + (t - start_i):
//   o_t = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q_t.k_j - max).
// The softmax splits over disjoint key ranges: a range yields (m, l, o) =
// (max, sum of exp(s - m), sum of exp(s - m) v), and ranges join as
//   m = max m_r,  l = sum l_r e^(m_r - m),  o = sum o_r e^(m_r - m).
// So the prefix is one range set whose rows are the query heads of ALL
// requests' tokens (its K/V are read once for the batch instead of once per
// token), each request's own positions are another, and a last pass joins
// them.
//
// This file: the unit kernel. A unit is (row tile of 16, kv head, key range)
// of the prefix or of one request. Four warps split the range's keys, 16 at a
// time, each through its own ring of cp.async stages (no CTA barrier in the
// loop), S = q K^T and O += P V on mma.sync m16n8k16 with fp32 accumulators;
// the G query heads of a kv head and the request's tokens are the rows, so a
// K/V tile is used by all of them. The warps join in shared memory, and the
// unit writes its (m, l, o) in fp32.
//
// Types: bf16 or f16 K/V. q of the cache's type enters the product exactly.
// fp32 q enters as a sum of TERMS values of the cache's type, each the
// rounding of what the ones before leave (bf16: 3 x 8 bits, f16: 2 x 11),
// S = sum of the terms' products, and P likewise, so nothing of fp32's 24 bits
// is lost to the 16-bit operands. With 16-bit q and output P is rounded once
// to the cache's type, as fine as the output's own rounding. An f16 P is
// scaled by 2^7 (and the sum with it), which keeps small weights and low
// terms out of the subnormals. Scores, running max, sums and outputs are fp32.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "qk_norm.cuh"

namespace ls {

struct PrefixAttnArgs {
  const void* q;
  long q_stride;            // elements between tokens
  const void* k_pool;
  const void* v_pool;
  long slot_stride;         // elements between slots
  int n_slots;
  const int* prefix_table;
  int prefix_len;
  const int* block_table;
  long table_stride;
  const int* lens;
  const int* token_start;
  int n_requests, n_tokens, max_new, max_len;
  int page_shift;
  int nh, nkv;
  float scale_log2;         // scale * log2(e): scores in powers of two
  void* out;
  long out_stride;
  // partials: part p of row (t, h): o[(p * T + t) * nh + h][HD], ml[...] = (m, l)
  float* part_o;
  float2* part_ml;
  int prefix_parts, prefix_chunk;    // key ranges of the prefix, positions each
  int suffix_parts, suffix_chunk;
  int prefix_tiles, suffix_tiles;    // row tiles of 16 (prefix: of its own kernel's rows)
  bool prefix_units;                 // the unit kernel also does the prefix
  bool own, direct;                  // tcgen05 kernel: rows of one request and its own positions; whole results
  int* status;
};

constexpr int kUnitThreads = 128;
constexpr int kUnitKeys = 16;      // keys of a warp's stage
constexpr int kUnitWarps = kUnitThreads / 32;
// Stages of a warp's ring and CTAs an SM: 16-bit queries of 128 take 166
// registers a thread, so a third CTA fits beside two when the rings shrink to
// two stages (one copy in flight a warp, 12 warps); fp32 queries hold two or
// three terms of q and leave room for two CTAs with three stages.
template <int HD, int TERMS>
__host__ __device__ constexpr int unit_stages() { return HD == 128 && TERMS == 1 ? 2 : 3; }
template <int HD, int TERMS>
__host__ __device__ constexpr int unit_ctas() { return HD == 128 ? (TERMS == 1 ? 3 : 2) : TERMS == 3 ? 3 : 4; }

template <int HD>
__host__ __device__ constexpr int unit_row_bytes() { return HD * 2 + 16; }   // padded: fragment reads hit distinct banks
template <int HD>
__host__ __device__ constexpr int unit_stage_bytes() { return 2 * kUnitKeys * unit_row_bytes<HD>(); }
template <int HD, int TERMS>
constexpr size_t unit_smem_bytes() { return (size_t)kUnitWarps * unit_stages<HD, TERMS>() * unit_stage_bytes<HD>(); }

// Joining the warps reuses the rings: kUnitWarps x 16 rows of HD floats, padded
// so that the 8 rows a warp stores at once lie in different banks.
template <int HD>
__host__ __device__ constexpr int unit_join_row() { return HD + 8; }
static_assert(unit_smem_bytes<64, 1>() >= sizeof(float) * kUnitWarps * 16 * unit_join_row<64>(), "join buffer");
static_assert(unit_smem_bytes<128, 1>() >= sizeof(float) * kUnitWarps * 16 * unit_join_row<128>(), "join buffer");

// Two fp32 values as a packed pair of the cache's type, lower index in the low half.
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) { return pack_bf16(a, b); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack2(uint32_t u, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}
__device__ __forceinline__ float2 unpack2(uint32_t u, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
// TERMS values of the cache's type that add up to x: each rounds what is left.
template <int TERMS, typename C>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&term)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    term[i] = pack2(a, b, C());
    if (i + 1 < TERMS) {
      const float2 h = unpack2(term[i], C());
      a -= h.x;
      b -= h.y;
    }
  }
}

// log2 of the factor on every weight p (it cancels in o / l).
__device__ __forceinline__ float weight_bias(__nv_bfloat16) { return 0.f; }
__device__ __forceinline__ float weight_bias(__half) { return 7.f; }

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                         __nv_bfloat16) {
  mma_bf16(d, a, b0, b1);
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                         __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_fast(float x) {   // ex2.approx: 2 ulp; exp2(-inf) = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A request's token range and own length; false (and the status word) when they are out of bounds.
__device__ __forceinline__ bool request_range(const PrefixAttnArgs& a, int i, int& start, int& n, int& len) {
  start = a.token_start[i];
  n = a.token_start[i + 1] - start;
  len = a.lens[i];
  if (start < 0 || n < 0 || n > a.max_new || start > a.n_tokens - n || len < 0 || len > a.max_len) {
    atomicCAS(a.status, kDevOk, kDevBadLength);
    return false;
  }
  return true;
}

// Two consecutive values of a query row as fp32.
__device__ __forceinline__ float2 load2(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 load2(const __nv_bfloat16* p) {
  return unpack2(*reinterpret_cast<const uint32_t*>(p), __nv_bfloat16());
}
__device__ __forceinline__ float2 load2(const __half* p) {
  return unpack2(*reinterpret_cast<const uint32_t*>(p), __half());
}

// Whether a warp's 16 V rows in shared memory hold a NaN or infinity (exponent bits all set).
template <int HD, typename C>
__device__ __forceinline__ bool any_not_finite(const unsigned char* vb, int lane) {
  constexpr uint32_t kExp = std::is_same<C, __half>::value ? 0x7C00u : 0x7F80u;
  bool found = false;
  for (int w = lane; w < kUnitKeys * HD / 2; w += 32) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(vb + (w / (HD / 2)) * unit_row_bytes<HD>() + (w % (HD / 2)) * 4);
    found |= (v & kExp) == kExp || ((v >> 16) & kExp) == kExp;
  }
  return __any_sync(0xffffffffu, found);
}

// O += P V over one stage without the tensor cores, each row adding only the positions it sees.
template <int HD, typename C>
__device__ __forceinline__ void add_by_weight(float (&o)[HD / 8][4], const float (&p)[2][4], const unsigned char* vb,
                                           int key, int k1, const int (&see)[2], int lane) {
  const int tig = lane & 3;
#pragma unroll 1
  for (int k = 0; k < kUnitKeys; ++k) {
    const int from = (lane & ~3) | ((k & 7) >> 1);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float even = k < 8 ? p[0][2 * e] : p[1][2 * e], odd = k < 8 ? p[0][2 * e + 1] : p[1][2 * e + 1];
      const float w = __shfl_sync(0xffffffffu, k & 1 ? odd : even, from);
      if (key + k >= k1 || key + k >= see[e]) continue;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        const float2 v = unpack2(
            *reinterpret_cast<const uint32_t*>(vb + k * unit_row_bytes<HD>() + (i * 8 + tig * 2) * 2), C());
        o[i][2 * e] += w * v.x;
        o[i][2 * e + 1] += w * v.y;
      }
    }
  }
}

// grid: 1-D over prefix units (part, row tile, kv head), then suffix units
// (part, row tile, kv head, request).
template <int HD, typename Q, typename C, int TERMS>
__global__ void __launch_bounds__(kUnitThreads, unit_ctas<HD, TERMS>()) prefix_unit_kernel(PrefixAttnArgs a) {
  constexpr int ST = unit_stages<HD, TERMS>();
  constexpr int RB = unit_row_bytes<HD>();
  constexpr int KS = HD / 16;
  constexpr int NT = HD / 8;
  constexpr int CH = HD / 8;                     // 16-byte chunks of a K/V row
  constexpr int LR = 32 / CH;                    // rows a warp copies at a time
  extern __shared__ __align__(16) unsigned char s_ring[];
  __shared__ float s_ml[kUnitWarps][16][2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int G = a.nh / a.nkv;
  const int mask = (1 << a.page_shift) - 1;
  pdl_launch_dependents();
  // A prefix kernel ahead of this one runs on beside it; this grid is not done
  // before that one is, which every way out of it below waits for

  // the unit
  unsigned u = blockIdx.x;
  const unsigned n_prefix = a.prefix_units ? (unsigned)(a.prefix_parts * a.prefix_tiles * a.nkv) : 0;
  const bool suffix = u >= n_prefix;
  if (suffix) u -= n_prefix;
  const unsigned parts = suffix ? a.suffix_parts : a.prefix_parts, tiles = suffix ? a.suffix_tiles : a.prefix_tiles;
  const int part = (int)(u % parts);
  u /= parts;
  const int tile = (int)(u % tiles);
  u /= tiles;
  const int g = (int)(u % (unsigned)a.nkv), req = (int)(u / (unsigned)a.nkv);   // req 0 for the prefix
  const int* table = suffix ? a.block_table + req * a.table_stride : a.prefix_table;
  const int bound = suffix ? a.max_len : a.prefix_len;                          // positions the table covers
  const int chunk = suffix ? a.suffix_chunk : a.prefix_chunk;
  const int k0 = part * chunk;
  const int first = k0 + warp * kUnitKeys, step = kUnitWarps * kUnitKeys;
  // the block of key `key + lane`: loaded a step ahead of its copy, the first
  // ones beside the request's length
  auto block_of = [&](int key) {
    return lane < kUnitKeys && key + lane < bound ? table[(key + lane) >> a.page_shift] : 0;
  };
  int block[ST - 1];
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) block[s] = block_of(first + s * step);
  int ahead = block_of(first + (ST - 1) * step);
  int start = 0, n = a.n_tokens, len = a.prefix_len;
  if (suffix && !request_range(a, req, start, n, len)) return pdl_wait();
  const int rows = n * G;
  if (tile * 16 >= rows) return pdl_wait();
  const int seen0 = suffix ? len - n + 1 : len;                   // positions the first token sees
  const int seen_by_all = seen0 + (suffix ? tile * 16 / G : 0);   // ... every row of the tile
  const int k1 = min(len, k0 + chunk);
  const int slot_part = suffix ? a.prefix_parts + part : part;

  unsigned char* ring = s_ring + (size_t)warp * ST * unit_stage_bytes<HD>();
  const C* kp = static_cast<const C*>(a.k_pool) + (long)g * HD;
  const C* vp = static_cast<const C*>(a.v_pool) + (long)g * HD;
  // stage s <- keys [key, key + 16): rows past the range or with a bad block
  // are filled with zeros, so what the pool holds there never enters a product
  auto issue = [&](int key, int block, int s) {
    unsigned char* dst = ring + s * unit_stage_bytes<HD>();
    int slot = -1;
    if (lane < kUnitKeys && key + lane < k1) {
      const long sl = ((long)block << a.page_shift) + ((key + lane) & mask);
      if (block < 0 || sl >= a.n_slots) atomicCAS(a.status, kDevOk, kDevBadIndex);
      else slot = (int)sl;
    }
#pragma unroll
    for (int i = 0; i < kUnitKeys / LR; ++i) {
      const int r = i * LR + lane / CH, c = lane % CH;
      const int sl = __shfl_sync(0xffffffffu, slot, r);
      const long off = (long)max(sl, 0) * a.slot_stride + c * 8;
      cp_async16(dst + r * RB + c * 16, kp + off, sl >= 0);
      cp_async16(dst + (kUnitKeys + r) * RB + c * 16, vp + off, sl >= 0);
    }
  };

  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

#pragma unroll
  for (int s = 0; s < ST - 1; ++s) {
    if (first + s * step < k1) issue(first + s * step, block[s], s);
    cp_async_commit();
  }

  // this thread's two rows: token, head, and the number of positions it sees
  long row_at[2];                                // t * nh + h, or -1
  int see[2];
  uint32_t qf[TERMS][KS][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = tile * 16 + gid + 8 * e;
    row_at[e] = -1;
    see[e] = 0;
    const Q* src = nullptr;
    if (r < rows) {
      const int j = r / G, t = start + j, h = g * G + (r - j * G);
      row_at[e] = (long)t * a.nh + h;
      see[e] = suffix ? seen0 + j : len;
      src = static_cast<const Q*>(a.q) + (long)t * a.q_stride + (long)h * HD;
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const float2 x = src ? load2(src + ks * 16 + tig * 2 + 8 * f) : make_float2(0.f, 0.f);
        uint32_t term[TERMS];
        split2<TERMS, C>(x.x, x.y, term);
#pragma unroll
        for (int i = 0; i < TERMS; ++i) qf[i][ks][e + 2 * f] = term[i];
      }
    }
  }

  int s = 0;
  for (int key = first; key < k1; key += step) {
    const int next = key + (ST - 1) * step;
    int sn = s + ST - 1;
    if (sn >= ST) sn -= ST;
    if (next < k1) issue(next, ahead, sn);
    cp_async_commit();
    ahead = block_of(next + step);
    cp_async_wait<ST - 1>();
    __syncwarp();
    const unsigned char* kb = ring + s * unit_stage_bytes<HD>();
    const unsigned char* vb = kb + kUnitKeys * RB;
    // chains of products that wait for one another cost ~20 cycles a link:
    // each term (or half of the head) has accumulators of its own
    constexpr int CHAINS = TERMS == 1 ? 2 : TERMS;
    float acc[CHAINS][2][4];
#pragma unroll
    for (int i = 0; i < CHAINS; ++i)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) acc[i][nt][0] = acc[i][nt][1] = acc[i][nt][2] = acc[i][nt][3] = 0.f;
    // K fragments of both key octets: lane l names row l % 8 of matrix l / 8
    const int kr = (lane & 7) + ((lane >> 4) << 3), kc = ((lane >> 3) & 1) * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t kf[4];
      ldmatrix_x4(kf, kb + kr * RB + (ks * 16 + kc) * 2);
#pragma unroll
      for (int i = 0; i < TERMS; ++i) {
        const int ch = TERMS == 1 ? ks & 1 : i;
        mma16816(acc[ch][0], qf[i][ks], kf[0], kf[1], C());
        mma16816(acc[ch][1], qf[i][ks], kf[2], kf[3], C());
      }
    }
    float sc[2][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[nt][e] = acc[CHAINS - 1][nt][e];        // smallest terms first
#pragma unroll
        for (int i = CHAINS - 2; i >= 0; --i) sc[nt][e] += acc[i][nt][e];
      }
    // scores in powers of two; masked ones leave by selection, whatever they hold
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int pos = key + nt * 8 + tig * 2 + (e & 1);
        const bool in = pos < k1 && pos < see[e >> 1];
        sc[nt][e] = in ? sc[nt][e] * a.scale_log2 : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], sc[nt][e]);
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
      const float base = mx[e] == -INFINITY ? 0.f : mx[e];
      const float keep = exp2_fast(m[e] - base);
      m[e] = mx[e];
      mx[e] = base - weight_bias(C());
      l[e] *= keep;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        o[i][2 * e] *= keep;
        o[i][2 * e + 1] *= keep;
      }
    }
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[nt][e] = exp2_fast(sc[nt][e] - mx[e >> 1]);
        l[e >> 1] += sc[nt][e];
      }
    uint32_t pf[TERMS][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t term[TERMS];
      split2<TERMS, C>(sc[e >> 1][2 * (e & 1)], sc[e >> 1][2 * (e & 1) + 1], term);
#pragma unroll
      for (int i = 0; i < TERMS; ++i) pf[i][e] = term[i];
    }
    // A weight of 0 times a NaN or infinity is NaN: where some rows of the tile
    // must not see a position that others see, a value that is not finite is
    // kept out of the product, and added one weight at a time
    if (key + kUnitKeys > seen_by_all && any_not_finite<HD, C>(vb, lane)) {
      add_by_weight<HD, C>(o, sc, vb, key, k1, see, lane);
    } else {
    const int vr = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
    for (int np = 0; np < NT / 2; ++np) {
      uint32_t vf[4];
      ldmatrix_x4_trans(vf, vb + vr * RB + (np * 16 + (lane >> 4) * 8) * 2);
#pragma unroll
      for (int i = 0; i < TERMS; ++i) {
        mma16816(o[2 * np], pf[i], vf[0], vf[1], C());
        mma16816(o[2 * np + 1], pf[i], vf[2], vf[3], C());
      }
    }
    }
    __syncwarp();   // the stage is refilled by the next turn's copy
    if (++s == ST) s = 0;
  }
  cp_async_wait<0>();

  // join the warps
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    if (tig == 0) {
      s_ml[warp][gid + 8 * e][0] = m[e];
      s_ml[warp][gid + 8 * e][1] = l[e];
    }
  }
  __syncthreads();   // also: every warp is done with its ring
  float* s_o = reinterpret_cast<float*>(s_ring);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float2*>(s_o + ((warp * 16 + gid + 8 * e) * unit_join_row<HD>() + i * 8 + tig * 2)) =
          make_float2(o[i][2 * e], o[i][2 * e + 1]);
  __syncthreads();
  constexpr int TPR = kUnitThreads / 16;         // threads of a row
  const int r = threadIdx.x / TPR, c0 = (threadIdx.x % TPR) * (HD / TPR);
  pdl_wait();
  if (tile * 16 + r >= rows) return;
  float mm = -INFINITY;
#pragma unroll
  for (int w = 0; w < kUnitWarps; ++w) mm = fmaxf(mm, s_ml[w][r][0]);
  const float base = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f, wt[kUnitWarps];
#pragma unroll
  for (int w = 0; w < kUnitWarps; ++w) {
    wt[w] = exp2_fast(s_ml[w][r][0] - base);
    ll += s_ml[w][r][1] * wt[w];
  }
  const int rr = tile * 16 + r, j = rr / G;
  const long at = (long)slot_part * a.n_tokens * a.nh + (long)(start + j) * a.nh + g * G + (rr - j * G);
  if (c0 == 0) a.part_ml[at] = make_float2(mm, ll);
#pragma unroll
  for (int c = 0; c < HD / TPR; c += 4) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kUnitWarps; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(s_o + (w * 16 + r) * unit_join_row<HD>() + c0 + c);
      acc.x += v.x * wt[w];
      acc.y += v.y * wt[w];
      acc.z += v.z * wt[w];
      acc.w += v.w * wt[w];
    }
    *reinterpret_cast<float4*>(a.part_o + at * HD + c0 + c) = acc;
  }
}

__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v.x, v.y, __nv_bfloat16()), pack2(v.z, v.w, __nv_bfloat16()));
}
__device__ __forceinline__ void store4(__half* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v.x, v.y, __half()), pack2(v.z, v.w, __half()));
}

constexpr int kJoinThreads = 128;
constexpr int kJoinBatch = 8;

// Join the parts of each row: HD/4 threads a row, 4 columns each. grid: (token,
// heads over kJoinThreads/(HD/4)). Tokens past token_start[R] and those of a
// request that was skipped get zeros, as do rows that see nothing. Bound: the
// latency of two loads (lengths; parts, all at once) after the parts are there.
template <int HD, typename Q>
__global__ void __launch_bounds__(kJoinThreads) prefix_join_kernel(PrefixAttnArgs a) {
  constexpr int TPR = HD / 4;
  const int t = blockIdx.x;
  // whether a valid request holds the token: written by nobody ahead of this kernel
  bool mine = false;
  for (int i = threadIdx.x; i < a.n_requests; i += kJoinThreads) {
    const int start = a.token_start[i], end = a.token_start[i + 1], len = a.lens[i];
    mine |= t >= start && t < end && start >= 0 && end - start <= a.max_new && end <= a.n_tokens && len >= 0 &&
            len <= a.max_len;
  }
  const bool ok = __syncthreads_or(mine);
  pdl_wait();
  const int h = blockIdx.y * (kJoinThreads / TPR) + threadIdx.x / TPR;
  if (h >= a.nh) return;
  const int c = (threadIdx.x % TPR) * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (ok) {
    const int parts = a.prefix_parts + a.suffix_parts;
    const long stride = (long)a.n_tokens * a.nh, row = (long)t * a.nh + h;
    float mm = -INFINITY, ll = 0.f;
    for (int p0 = 0; p0 < parts; p0 += kJoinBatch) {
      float2 ml[kJoinBatch];
      float4 v[kJoinBatch];
#pragma unroll
      for (int p = 0; p < kJoinBatch; ++p) {
        const bool in = p0 + p < parts;
        const long at = (in ? p0 + p : p0) * stride + row;
        ml[p] = __ldcg(a.part_ml + at);
        v[p] = __ldcg(reinterpret_cast<const float4*>(a.part_o + at * HD + c));
        if (!in) ml[p].x = -INFINITY;
      }
      float top = mm;
#pragma unroll
      for (int p = 0; p < kJoinBatch; ++p) top = fmaxf(top, ml[p].x);
      const float base = top == -INFINITY ? 0.f : top;
      const float keep = exp2_fast(mm - base);
      mm = top;
      ll *= keep;
      acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
      for (int p = 0; p < kJoinBatch; ++p) {
        const float w = exp2_fast(ml[p].x - base);
        if (p0 + p >= parts) break;
        ll += ml[p].y * w;
        acc.x += v[p].x * w;
        acc.y += v[p].y * w;
        acc.z += v[p].z * w;
        acc.w += v[p].w * w;
      }
    }
    const float inv = ll == 0.f ? 0.f : 1.f / ll;
    acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  }
  store4(static_cast<Q*>(a.out) + (long)t * a.out_stride + (long)h * HD + c, acc);
}

}  // namespace ls

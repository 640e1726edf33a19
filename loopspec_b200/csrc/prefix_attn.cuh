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
// This file: the stream kernel, for few query rows a kv head, and the joining
// pass. A unit is (row tile, kv head, key range) of the prefix or of one
// request; the G query heads of a kv head and the request's tokens are the
// rows, so a K/V tile is used by all of them. Each warp works by itself through
// its units, 16 keys at a time, as one stream, while the next tiles, of this
// unit or the next one, are on their way into the warp's ring by cp.async (a
// CTA for each unit, with its lookups, loads and joins one after the other,
// took 8500 cycles a unit beside the 1500 a tile).
// The products run on mma.sync m16n8k16, fp32 accumulators, with the keys as
// M: S^T = K q^T (16 keys by 8 rows) and O^T += V^T P^T. A decode step has one
// to eight rows a kv head; as N they cost half the products and registers that
// they cost as M. A row tile is 8 RT rows, whose products share the fragments
// of K and V. A unit's (m, l, o) goes out in
// fp32; O is rescaled only when a row's maximum has grown by more than 2^8 since
// its reference was set (the reference cancels in o / l).
// Bound: the latency of short reads at the lengths of a decode step (a cold read
// of this size ramps up for some 13 us), then HBM. 16 requests of up to 700
// positions behind 2048, 16 heads, fp32 q: 63 MB in 21.4 us with the joining
// pass, 2.9 TB/s; 4 requests behind 333: 6.7 us, call after call in a graph.
//
// Types: bf16 or f16 K/V. q of the cache's type enters the product exactly.
// fp32 q enters as a sum of TERMS values of the cache's type, each the
// rounding of what the ones before leave, S = sum of the terms' products, and P
// likewise: bf16 3 x 8 bits, all that fp32 has; f16 2 x 11 bits, 22 of its 24 (a
// third term would cost a half more products for errors below those of the sums).
// For f16 each row of q is first multiplied by the power of two that brings its
// largest element to [2^14, 2^15), and its scores' scale divided by it, so that q
// may have any size and low terms stay out of the subnormals. With 16-bit q and
// output P is rounded once to the cache's type, as fine as the output's own
// rounding (errors against 64 bits, relative to the outputs' size: bf16 0.0022, 0.0017
// without; f16 0.00027, 0.00021). An f16 P is scaled by 2^7 (and the sum with it),
// which keeps small weights and low terms out of the subnormals. Scores, running
// max, sums and outputs are fp32.
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
  uint32_t g_magic;         // ceil(2^32 / (nh / nkv)), see div_by
  float scale_log2;         // scale * log2(e): scores in powers of two
  void* out;
  long out_stride;
  // partials: part p of row (t, h): o[(p * T + t) * nh + h][HD], ml[...] = (m, l)
  float* part_o;
  float2* part_ml;
  int prefix_parts, prefix_chunk;    // key ranges of the prefix, positions each
  int suffix_parts, suffix_chunk;    // ... of max_len own positions
  int prefix_tiles, suffix_tiles;    // row tiles, of their kernels' rows
  bool prefix_units, suffix_units;   // what a launch of the stream kernel does
  bool behind;                       // it runs beside a kernel of the same call
  bool own, direct;                  // tcgen05 kernel: rows of one request and its own positions; whole results
  int* status;
};

constexpr int kUnitThreads = 128;
constexpr int kUnitKeys = 16;      // keys of a warp's stage
constexpr int kUnitWarps = kUnitThreads / 32;
// CTAs an SM by the registers that q (TERMS x RT) and O (RT) take, and the
// stages of a warp's ring that this leaves shared memory for.
template <int HD, int TERMS, int RT>
__host__ __device__ constexpr int unit_ctas() {
  return HD == 128 ? (TERMS * RT <= 3 ? 3 : 2) : (TERMS * RT <= 4 ? 4 : 3);
}
template <int HD, int TERMS, int RT>
__host__ __device__ constexpr int unit_stages() { return unit_ctas<HD, TERMS, RT>() >= (HD == 128 ? 3 : 4) ? 2 : 3; }

template <int HD>
__host__ __device__ constexpr int unit_row_bytes() { return HD * 2 + 16; }   // padded: fragment reads hit distinct banks
template <int HD>
__host__ __device__ constexpr int unit_stage_bytes() { return 2 * kUnitKeys * unit_row_bytes<HD>(); }
template <int HD, int TERMS, int RT>
constexpr size_t unit_smem_bytes() { return (size_t)kUnitWarps * unit_stages<HD, TERMS, RT>() * unit_stage_bytes<HD>(); }

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

// The transpose of an 8 x 8 tile of 16-bit values, two a lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

// r / G by a multiplication: `magic` is ceil(2^32 / G), the quotient at most one too large for r < 2^31.
__device__ __forceinline__ int div_by(int r, int G, uint32_t magic) {
  if (G == 1) return r;
  const int q = (int)__umulhi((uint32_t)r, magic);
  return q * G > r ? q - 1 : q;
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

// The exponent shift that brings a largest |q| of `most` to [2^14, 2^15): 0 for rows of zeros and those that are not
// finite. What it is for: f16 terms of an fp32 q.
template <int TERMS, typename C>
constexpr bool kScaledRows = TERMS > 1 && std::is_same<C, __half>::value;
__device__ __forceinline__ int row_shift(float most) {
  const int e = (int)(__float_as_uint(most) >> 23);       // biased; most >= 0
  return e == 0xff || most == 0.f ? 0 : min(126, 127 + 14 - e);
}
__device__ __forceinline__ float power2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// Two consecutive values of a query row as fp32.
__device__ __forceinline__ float2 load2(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 load2(const __nv_bfloat16* p) {
  return unpack2(*reinterpret_cast<const uint32_t*>(p), __nv_bfloat16());
}
__device__ __forceinline__ float2 load2(const __half* p) {
  return unpack2(*reinterpret_cast<const uint32_t*>(p), __half());
}

// A maximum that is NaN when an operand is.
__device__ __forceinline__ float max2_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

constexpr float kGrow = 8.f;   // log2 growth of a row's maximum that moves its reference

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

// O^T += V^T P^T over one stage without the tensor cores, each row adding only the positions it sees.
template <int HD, typename C, int RT>
__device__ __forceinline__ void add_by_weight(float (&o)[RT][HD / 16][4], const float (&p)[RT][4],
                                              const unsigned char* vb, int key, int k1, const int (&see)[RT][2],
                                              int lane) {
  const int gid = lane >> 2, tig = lane & 3;
#pragma unroll 1
  for (int k = 0; k < kUnitKeys; ++k) {
    const int from = (k & 7) * 4 + tig;
    const C* row = reinterpret_cast<const C*>(vb + k * unit_row_bytes<HD>());
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float w = __shfl_sync(0xffffffffu, k < 8 ? p[rt][e] : p[rt][2 + e], from);
        if (key + k >= k1 || key + k >= see[rt][e]) continue;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          o[rt][i][e] += w * (float)row[i * 16 + gid];
          o[rt][i][2 + e] += w * (float)row[i * 16 + 8 + gid];
        }
      }
  }
}

// The pools' rows of one kv head.
template <typename C>
struct PoolView {
  const C* k;
  const C* v;
  long stride;
  int n_slots, page_shift;
  __device__ __forceinline__ PoolView(const PrefixAttnArgs& a, int g, int hd)
      : k(static_cast<const C*>(a.k_pool) + (long)g * hd), v(static_cast<const C*>(a.v_pool) + (long)g * hd),
        stride(a.slot_stride), n_slots(a.n_slots), page_shift(a.page_shift) {}
};

// The weight of a key for a row by the formula; `base`: the row's reference in
// powers of two, less the weights' bias.
template <int HD, typename Q, typename C>
__device__ __noinline__ float weight_of(const Q* q, const C* k, float base, float scale_log2) {
  float s = 0.f;
  for (int i = 0; i < HD; ++i) s += (float)q[i] * (float)k[i];
  return exp2_fast(s * scale_log2 - base);
}

// Whether terms of q and P can make NaN of what is infinite: a term of 0, or of the
// other sign than the one before it, times infinity is NaN, and the whole of it
// infinite. An f16 weight is 0 below 2^-32 of the largest even as the only term. So
// rows that come out not finite are computed once more by the formula, where they
// are whole: in the joining pass, or at the end of a unit that is all of its rows.
template <typename Q, typename C>
constexpr bool kTermsLose = !std::is_same<Q, C>::value || std::is_same<C, __half>::value;

// Keys of a unit: positions [p0, p1) of a table, then [p2, p3) of another.
struct KeyRanges {
  const int* table;
  int p0, p1;
  const int* then;
  int p2, p3;
};

// slot of key i of the ranges; -1: a block that is not there, its K and V are zeros
template <typename C>
__device__ __forceinline__ long slot_of(const PoolView<C>& pools, const KeyRanges& keys, int i) {
  const int n = max(0, keys.p1 - keys.p0), pos = i < n ? keys.p0 + i : keys.p2 + i - n;
  const int block = (i < n ? keys.table : keys.then)[pos >> pools.page_shift];
  const long slot = ((long)block << pools.page_shift) + (pos & ((1 << pools.page_shift) - 1));
  return block < 0 || slot >= pools.n_slots ? -1L : slot;
}
__device__ __forceinline__ int keys_in(const KeyRanges& keys) { return max(0, keys.p1 - keys.p0) + max(0, keys.p3 - keys.p2); }

// score in powers of two
template <int HD, typename Q, typename C>
__device__ __forceinline__ float score_of(const PoolView<C>& pools, long slot, const Q* q, float scale_log2) {
  float s = 0.f;
  if (slot >= 0) {
    const C* k = pools.k + slot * pools.stride;
#pragma unroll 4
    for (int d = 0; d < HD; ++d) s += (float)q[d] * (float)k[d];
  }
  return s * scale_log2;
}

// A row's whole result by the formula in fp32, columns c .. c + 3, by the HD / 4
// lanes of its group: each weighs a key, all add its value. Inlined: a kernel with
// a call in it took 0.6 us more with 256 CTAs, 3 with 1024, though none called.
template <int HD, typename Q, typename C>
__device__ __forceinline__ float4 row_by_formula(PoolView<C> pools, KeyRanges keys, const Q* q, float scale_log2, int c,
                                              unsigned group) {
  constexpr int L = HD / 4;
  const int lane = threadIdx.x % L, all = keys_in(keys);
  float m = -INFINITY;
  for (int i = lane; i < all; i += L) m = max2_nan(m, score_of<HD>(pools, slot_of(pools, keys, i), q, scale_log2));
#pragma unroll
  for (int o = 1; o < L; o <<= 1) m = max2_nan(m, __shfl_xor_sync(group, m, o));
  if (m != m) return make_float4(m, m, m, m);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < all; i0 += L) {
    const int slot = i0 + lane < all ? (int)slot_of(pools, keys, i0 + lane) : -1;
    const float w = i0 + lane < all ? exp2_fast(score_of<HD>(pools, slot, q, scale_log2) - base) : 0.f;
    l += w;
#pragma unroll 1
    for (int k = 0; k < L; ++k) {
      const float wk = __shfl_sync(group, w, k, L);
      const int sk = __shfl_sync(group, slot, k, L);
      if (sk < 0) continue;
      const C* v = pools.v + sk * pools.stride + c;
      acc = make_float4(acc.x + wk * (float)v[0], acc.y + wk * (float)v[1], acc.z + wk * (float)v[2], acc.w + wk * (float)v[3]);
    }
  }
#pragma unroll
  for (int o = 1; o < L; o <<= 1) l += __shfl_xor_sync(group, l, o);
  return make_float4(acc.x / l, acc.y / l, acc.z / l, acc.w / l);
}

constexpr int kBatchRequests = 256;    // looked up at a time; 32 x 8 for the search

// Units of a batch of requests: their lengths, and where each one's units begin.
struct UnitMap {
  int first[kBatchRequests + 1];
  int start[kBatchRequests], n[kBatchRequests], len[kBatchRequests];
  int warp_sum[kUnitWarps];
};

// grid: any number of CTAs. Units with work are numbered one after the other --
// the prefix's, then request by request: row tile, key range, kv head fastest --
// and warp w of W takes units w, w + W, ...: a request's length decides how many
// it has, so every CTA sums them up first (up to kBatchRequests at a time).
template <int HD, typename Q, typename C, int TERMS, int RT>
__global__ void __launch_bounds__(kUnitThreads, unit_ctas<HD, TERMS, RT>()) prefix_stream_kernel(PrefixAttnArgs a) {
  constexpr int ST = unit_stages<HD, TERMS, RT>();
  constexpr int ROWS = 8 * RT;                   // rows of a tile
  constexpr int RB = unit_row_bytes<HD>();
  constexpr int KS = HD / 16;
  constexpr int MT = HD / 16;                    // 16-dimension tiles of O^T
  constexpr int CH = HD / 8;                     // 16-byte chunks of a K/V row
  constexpr int LR = 32 / CH;                    // rows a warp copies at a time
  constexpr unsigned kAll = 0xffffffffu;
  extern __shared__ __align__(16) unsigned char s_ring[];
  __shared__ UnitMap s_map;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int G = a.nh / a.nkv;
  const int mask = (1 << a.page_shift) - 1;
  // A call's first kernel is launched early: it waits for what came before, and
  // only then lets the next one start. Behind another kernel of the call its
  // inputs are there; it waits at the end, so that it is not done before that one.
  if (!a.behind) pdl_wait();
  pdl_launch_dependents();
  unsigned char* ring = s_ring + (size_t)warp * ST * unit_stage_bytes<HD>();
  const int W = gridDim.x * kUnitWarps, w = warp * gridDim.x + blockIdx.x;

  for (int req0 = 0; req0 < (a.suffix_units ? a.n_requests : 1); req0 += kBatchRequests) {
    const int n_prefix = a.prefix_units && req0 == 0 ? a.prefix_parts * a.prefix_tiles * a.nkv : 0;
    const int n_req = a.suffix_units ? min(kBatchRequests, a.n_requests - req0) : 0;
    int n_units = n_prefix;
    if (n_req) {
      __syncthreads();                           // the last batch's map is done with
      constexpr int PER = kBatchRequests / kUnitThreads;
      int count[PER], sum = 0;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = threadIdx.x * PER + k;
        count[k] = 0;
        int start, n, len;
        if (i < n_req && request_range(a, req0 + i, start, n, len)) {
          s_map.start[i] = start;
          s_map.n[i] = n;
          s_map.len[i] = len;
          count[k] = (n * G + ROWS - 1) / ROWS * ((len + a.suffix_chunk - 1) / a.suffix_chunk) * a.nkv;
        }
        sum += count[k];
      }
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kAll, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31) s_map.warp_sum[warp] = upto;
      __syncthreads();
      int at = n_prefix + upto - sum;
#pragma unroll
      for (int v = 0; v < kUnitWarps; ++v) {
        if (v < warp) at += s_map.warp_sum[v];
        n_units += s_map.warp_sum[v];
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        s_map.first[threadIdx.x * PER + k] = at;
        at += count[k];
      }
      if (threadIdx.x == kUnitThreads - 1) s_map.first[kBatchRequests] = at;
      __syncthreads();
    }
    struct Unit {
      int req, g, tile, part, start, n, len, k0, k1;   // req -1: the prefix; keys [k0, k1), at least one
    };
    auto unit_of = [&](int u) {
      Unit x;
      int tiles = a.prefix_tiles;
      x.req = -1;
      x.start = 0;
      x.n = a.n_tokens;
      x.len = a.prefix_len;
      int chunk = a.prefix_chunk;
      if (u >= n_prefix) {
        // the last request whose first unit is <= u: one of 32 eights, one of 8
        int i = (__popc(__ballot_sync(kAll, s_map.first[lane * 8] <= u)) - 1) * 8;
        i += __popc(__ballot_sync(kAll, lane < 8 && s_map.first[i + (lane & 7)] <= u)) - 1;
        u -= s_map.first[i];
        x.req = req0 + i;
        x.start = s_map.start[i];
        x.n = s_map.n[i];
        x.len = s_map.len[i];
        chunk = a.suffix_chunk;
        tiles = (x.n * G + ROWS - 1) / ROWS;
      }
      const int v = u / a.nkv;
      x.g = u - v * a.nkv;
      x.part = v / tiles;
      x.tile = v - x.part * tiles;
      x.k0 = x.part * chunk;
      x.k1 = min(x.len, x.k0 + chunk);
      // what some row of the tile sees (a range that nobody sees gives the part of no weight)
      if (x.req >= 0)
        x.k1 = max(x.k0 + 1, min(x.k1, x.len - x.n + 1 + div_by(min(x.n * G, (x.tile + 1) * ROWS) - 1, G, a.g_magic)));
      return x;
    };

    // the next tile to copy: its table, head, key; the blocks of its keys are
    // loaded (`ahead`, a key a lane) when the tile before it is copied
    int p_unit = w;
    const int* p_table = a.prefix_table;
    int p_g = 0, p_key = 0, p_k1 = 0, ahead = 0, to = 0;
    auto look = [&]() { ahead = lane < kUnitKeys && p_key + lane < p_k1 ? p_table[(p_key + lane) >> a.page_shift] : 0; };
    auto open = [&]() {
      p_k1 = 0;
      if (p_unit < n_units) {
        const Unit x = unit_of(p_unit);
        p_unit += W;
        p_g = x.g;
        p_key = x.k0;
        p_k1 = x.k1;
        p_table = x.req >= 0 ? a.block_table + x.req * a.table_stride : a.prefix_table;
        look();
      }
    };
    // copy it into stage `to`: rows past the range or with a bad block are
    // filled with zeros, so what the pool holds there never enters a product
    auto push = [&]() {
      if (p_k1 > 0) {
        unsigned char* dst = ring + to * unit_stage_bytes<HD>();
        int slot = -1;
        if (lane < kUnitKeys && p_key + lane < p_k1) {
          const long sl = ((long)ahead << a.page_shift) + ((p_key + lane) & mask);
          if (ahead < 0 || sl >= a.n_slots) atomicCAS(a.status, kDevOk, kDevBadIndex);
          else slot = (int)sl;
        }
        const int c = lane % CH;
        const char* kp = static_cast<const char*>(a.k_pool) + ((long)p_g * HD + c * 8) * 2;
        const long to_v = static_cast<const char*>(a.v_pool) - static_cast<const char*>(a.k_pool);
        const int row_bytes = (int)(a.slot_stride * 2);
#pragma unroll
        for (int i = 0; i < kUnitKeys / LR; ++i) {
          const int r = i * LR + lane / CH;
          const int sl = __shfl_sync(kAll, slot, r);
          const char* src = kp + (long)max(sl, 0) * row_bytes;
          cp_async16(dst + r * RB + c * 16, src, sl >= 0);
          cp_async16(dst + (kUnitKeys + r) * RB + c * 16, src + to_v, sl >= 0);
        }
        p_key += kUnitKeys;
        if (p_key < p_k1) look();
        else open();
        if (++to == ST) to = 0;
      }
      cp_async_commit();
    };
    open();
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) push();

    int at = 0;                                  // the stage of the next tile to use
    for (int c_unit = w; c_unit < n_units; c_unit += W) {
      const Unit x = unit_of(c_unit);
      const bool suffix = x.req >= 0;
      const int g = x.g, tile = x.tile, part = x.part, start = x.start, n = x.n, len = x.len, k0 = x.k0, k1 = x.k1;
      const int rows = n * G;
      const int seen0 = suffix ? len - n + 1 : len;                   // positions the first token sees
      const int seen_by_all = seen0 + (suffix ? div_by(tile * ROWS, G, a.g_magic) : 0);   // ... every row of the tile

      // q of row gid of each eight as the second operand
      uint32_t qf[TERMS][RT][KS][2];
      float row_scale[RT][2];                    // of the scores of rows 2 tig and 2 tig + 1, where rows have one of their own
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int r = tile * ROWS + rt * 8 + gid;
        const Q* src = nullptr;
        if (r < rows) {
          const int j = div_by(r, G, a.g_magic);
          src = static_cast<const Q*>(a.q) + (long)(start + j) * a.q_stride + (long)(g * G + r - j * G) * HD + tig * 2;
        }
        if constexpr (TERMS == 1) {              // q is of the cache's type: as it is
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              qf[0][rt][ks][x] = src ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8 * x) : 0;
        } else {
          float up = 1.f;
          if constexpr (kScaledRows<TERMS, C>) {
            float most = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const float2 v = src ? load2(src + ks * 16 + 8 * x) : make_float2(0.f, 0.f);
                most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
              }
            most = fmaxf(most, __shfl_xor_sync(kAll, most, 1));
            most = fmaxf(most, __shfl_xor_sync(kAll, most, 2));
            const int shift = row_shift(most);
            up = power2(shift);
#pragma unroll
            for (int e = 0; e < 2; ++e) row_scale[rt][e] = a.scale_log2 * power2(-__shfl_sync(kAll, shift, (tig * 2 + e) * 4));
          }
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float2 v = src ? load2(src + ks * 16 + 8 * x) : make_float2(0.f, 0.f);
              uint32_t term[TERMS];
              split2<TERMS, C>(v.x * up, v.y * up, term);
#pragma unroll
              for (int i = 0; i < TERMS; ++i) qf[i][rt][ks][x] = term[i];
            }
        }
      }
      // the scores and outputs of this thread belong to rows 2 tig and 2 tig + 1
      // of each eight: the number of positions they see
      int see[RT][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = tile * ROWS + rt * 8 + tig * 2 + e;
          see[rt][e] = r >= rows ? 0 : suffix ? seen0 + div_by(r, G, a.g_magic) : len;
        }
      float o[RT][MT][4], m[RT][2], l[RT][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        m[rt][0] = m[rt][1] = -INFINITY;
        l[rt][0] = l[rt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[rt][i][0] = o[rt][i][1] = o[rt][i][2] = o[rt][i][3] = 0.f;
      }

      for (int key = k0; key < k1; key += kUnitKeys) {
        push();
        cp_async_wait<ST - 1>();
        __syncwarp();
        const unsigned char* kb = ring + at * unit_stage_bytes<HD>();
        const unsigned char* vb = kb + kUnitKeys * RB;
        // S^T: chains of products that wait for one another cost ~20 cycles a
        // link, so each term (or half of the head) has accumulators of its own
        constexpr int CHAINS = TERMS == 1 ? 2 : TERMS;
        float acc[CHAINS][RT][4];
#pragma unroll
        for (int i = 0; i < CHAINS; ++i)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) acc[i][rt][0] = acc[i][rt][1] = acc[i][rt][2] = acc[i][rt][3] = 0.f;
        // lane l names row l % 8 of matrix l / 8: (keys, keys + 8) x (dims, dims + 8)
        const unsigned char* kr = kb + ((lane & 7) + ((lane >> 3) & 1) * 8) * RB + (lane >> 4) * 16;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t kf[4];
          ldmatrix_x4(kf, kr + ks * 32);
#pragma unroll
          for (int i = 0; i < TERMS; ++i)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              mma16816(acc[TERMS == 1 ? ks % CHAINS : i][rt], kf, qf[i][rt][ks][0], qf[i][rt][ks][1], C());
        }
        // Scores in powers of two; masked ones leave by selection, whatever they
        // hold. c[0], c[1]: key gid, rows 2 tig and 2 tig + 1; c[2], c[3]: key gid + 8.
        float sc[RT][4], mx[RT][2];
        const bool cut = key + kUnitKeys > min(k1, seen_by_all);
        bool move = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = acc[CHAINS - 1][rt][e];    // smallest terms first
#pragma unroll
            for (int i = CHAINS - 2; i >= 0; --i) v += acc[i][rt][e];
            sc[rt][e] = v * (kScaledRows<TERMS, C> ? row_scale[rt][e & 1] : a.scale_log2);
            if (cut) {
              const int pos = key + gid + (e >> 1) * 8;
              if (pos >= k1 || pos >= see[rt][e & 1]) sc[rt][e] = -INFINITY;
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v = fmaxf(sc[rt][e], sc[rt][2 + e]);
            v = fmaxf(v, __shfl_xor_sync(kAll, v, 4));
            v = fmaxf(v, __shfl_xor_sync(kAll, v, 8));
            v = fmaxf(v, __shfl_xor_sync(kAll, v, 16));
            mx[rt][e] = v;
            move |= m[rt][e] == -INFINITY ? v != -INFINITY : v - m[rt][e] > kGrow;
          }
        }
        if (__any_sync(kAll, move)) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const bool grown = m[rt][e] == -INFINITY || mx[rt][e] - m[rt][e] > kGrow;
              const float keep = grown && m[rt][e] != -INFINITY ? exp2_fast(m[rt][e] - mx[rt][e]) : 1.f;
              if (grown) m[rt][e] = mx[rt][e];
              l[rt][e] *= keep;
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                o[rt][i][e] *= keep;
                o[rt][i][2 + e] *= keep;
              }
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float base = (m[rt][e & 1] == -INFINITY ? 0.f : m[rt][e & 1]) - weight_bias(C());
            sc[rt][e] = exp2_fast(sc[rt][e] - base);
            if (TERMS > 1) l[rt][e & 1] += sc[rt][e];
          }
        // A weight of 0 times a NaN or infinity is NaN: where some rows of the
        // tile must not see a position that others see, a value that is not
        // finite is kept out of the product, and added one weight at a time
        if (key + kUnitKeys > seen_by_all && any_not_finite<HD, C>(vb, lane)) {
          add_by_weight<HD, C, RT>(o, sc, vb, key, k1, see, lane);
          if constexpr (TERMS == 1) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int e = 0; e < 4; ++e) l[rt][e & 1] += sc[rt][e];
          }
        } else {
          uint32_t pf[TERMS][RT][2];             // P^T as the second operand: rows become columns
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              uint32_t term[TERMS];
              split2<TERMS, C>(sc[rt][2 * x], sc[rt][2 * x + 1], term);
              if constexpr (TERMS == 1) {        // the weights that the product gets: the rounding of a large one cancels
                const float2 w = unpack2(term[0], C());
                l[rt][0] += w.x;
                l[rt][1] += w.y;
              }
#pragma unroll
              for (int i = 0; i < TERMS; ++i) pf[i][rt][x] = transpose8x8(term[i]);
            }
          const unsigned char* vr = vb + ((lane & 7) + (lane >> 4) * 8) * RB + ((lane >> 3) & 1) * 16;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            uint32_t vf[4];
            ldmatrix_x4_trans(vf, vr + i * 32);
#pragma unroll
            for (int x = 0; x < TERMS; ++x)
#pragma unroll
              for (int rt = 0; rt < RT; ++rt) mma16816(o[rt][i], vf, pf[x][rt][0], pf[x][rt][1], C());
          }
        }
        __syncwarp();   // the stage is refilled by the next turn's copy
        if (++at == ST) at = 0;
      }

      // the unit's part; the eight lanes of a row store 32 bytes side by side
      const long base = (long)(suffix ? a.prefix_parts + part : part) * a.n_tokens * a.nh;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = l[rt][e];
          sum += __shfl_xor_sync(kAll, sum, 4);
          sum += __shfl_xor_sync(kAll, sum, 8);
          sum += __shfl_xor_sync(kAll, sum, 16);
          const int r = tile * ROWS + rt * 8 + tig * 2 + e;
          if (r >= rows) continue;
          const int j = div_by(r, G, a.g_magic);
          const long row = base + (long)(start + j) * a.nh + g * G + r - j * G;
          if (gid == 0) a.part_ml[row] = make_float2(m[rt][e], sum);
          float* dst = a.part_o + row * HD + gid;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            dst[i * 16] = o[rt][i][e];
            dst[i * 16 + 8] = o[rt][i][2 + e];
          }
        }
    }
    cp_async_wait<0>();
  }
  if (a.behind) pdl_wait();
}

__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v.x, v.y, __nv_bfloat16()), pack2(v.z, v.w, __nv_bfloat16()));
}
__device__ __forceinline__ void store4(__half* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v.x, v.y, __half()), pack2(v.z, v.w, __half()));
}

constexpr int kJoinThreads = 128;
constexpr int kJoinBatch = 4;

// Join the parts of each row: HD/4 threads a group, 4 columns each. With SPLIT
// (more than kJoinBatch parts) the groups of a CTA share one row's parts, else
// each has a row of its own. grid: (token, heads over the rows of a CTA).
// Tokens past token_start[R] and those of a request that was skipped get zeros,
// as do rows that see nothing. Bound: the latency of two loads (lengths; parts,
// all at once) after the parts are there; told that one CTA an SM will do, the
// compiler takes the registers that this needs (48; 40 otherwise: 23.7 us a call
// with 16 requests behind 2048 positions and fp32 queries, 23.3 so).
template <int HD, typename Q, typename C, bool SPLIT>
__global__ void __launch_bounds__(kJoinThreads, 1) prefix_join_kernel(PrefixAttnArgs a) {
  constexpr int TPR = HD / 4, GROUPS = kJoinThreads / TPR;
  __shared__ float4 s_acc[SPLIT ? GROUPS : 1][TPR];
  __shared__ float2 s_ml[GROUPS];
  __shared__ int s_req, s_len, s_seen;   // the token's request, its own positions, and those that the token sees
  const int t = blockIdx.x;
  if (!a.behind) pdl_wait();
  // no early launch of what follows: CTAs of the next call that wait here took
  // the places of this call's last ones (16 requests behind 2048 positions with
  // fp32 queries, call after call: 31.6 us with it, 22.6 without)
  // Whether a valid request holds the token: written by no kernel of the call. This
  // also tells of ranges that are out of bounds where no kernel ran for the requests'
  // own positions (max_new or max_len is 0).
  bool mine = false;
  for (int i = threadIdx.x; i < a.n_requests; i += kJoinThreads) {
    int start, n, len;
    if (request_range(a, i, start, n, len) && t >= start && t - start < n) {
      mine = true;
      s_req = i;
      s_len = len;
      s_seen = len - n + 1 + (t - start);
    }
  }
  const bool ok = __syncthreads_or(mine);
  if (a.behind) pdl_wait();
  const int group = threadIdx.x / TPR, c = (threadIdx.x % TPR) * 4;
  const int h = SPLIT ? blockIdx.y : blockIdx.y * GROUPS + group;
  if (!SPLIT && h >= a.nh) return;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float mm = -INFINITY, ll = 0.f;
  if (ok) {
    // own positions past the length have no parts
    const int parts = a.prefix_parts + (a.suffix_parts ? (s_len + a.suffix_chunk - 1) / a.suffix_chunk : 0);
    const long stride = (long)a.n_tokens * a.nh, row = (long)t * a.nh + h;
    constexpr int STEP = SPLIT ? GROUPS : 1;
    for (int p0 = SPLIT ? group : 0; p0 < parts; p0 += STEP * kJoinBatch) {
      float2 ml[kJoinBatch];
      float4 v[kJoinBatch];
#pragma unroll
      for (int p = 0; p < kJoinBatch; ++p) {
        ml[p] = make_float2(-INFINITY, 0.f);
        v[p] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p0 + p * STEP < parts) {
          const long at = (p0 + p * STEP) * stride + row;
          ml[p] = __ldcg(a.part_ml + at);
          v[p] = __ldcg(reinterpret_cast<const float4*>(a.part_o + at * HD + c));
        }
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
        ll += ml[p].y * w;
        acc.x += v[p].x * w;
        acc.y += v[p].y * w;
        acc.z += v[p].z * w;
        acc.w += v[p].w * w;
      }
    }
  }
  if (SPLIT) {
    s_acc[group][threadIdx.x % TPR] = acc;
    if (c == 0) s_ml[group] = make_float2(mm, ll);
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) mm = fmaxf(mm, s_ml[i].x);
    const float base = mm == -INFINITY ? 0.f : mm;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    ll = 0.f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      const float w = exp2_fast(s_ml[i].x - base);
      const float4 v = s_acc[i][threadIdx.x % TPR];
      ll += s_ml[i].y * w;
      acc.x += v.x * w;
      acc.y += v.y * w;
      acc.z += v.z * w;
      acc.w += v.w * w;
    }
  }
  // zeros for a row that sees nothing; one whose scores are all -inf is 0 / 0
  const bool sees = ok && (a.prefix_len > 0 || s_seen > 0);
  const float inv = sees ? 1.f / ll : 0.f;
  acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  if constexpr (kTermsLose<Q, C>) {                 // a row that is not finite, by the formula
    const unsigned group_lanes = TPR == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
    const float zero = fmaf(acc.x, 0.f, fmaf(acc.y, 0.f, fmaf(acc.z, 0.f, acc.w * 0.f)));
    if (__any_sync(group_lanes, sees && zero != 0.f)) {
      const KeyRanges keys{a.prefix_table, 0, a.prefix_len, a.block_table + s_req * a.table_stride, 0, s_seen};
      acc = row_by_formula<HD>(PoolView<C>(a, h / (a.nh / a.nkv), HD), keys,
                               static_cast<const Q*>(a.q) + (long)t * a.q_stride + (long)h * HD, a.scale_log2, c, group_lanes);
    }
  }
  store4(static_cast<Q*>(a.out) + (long)t * a.out_stride + (long)h * HD + c, acc);
}

// Whole results of the tcgen05 kernel: zeros for the tokens that no valid request
// holds, beside that kernel (as a part of it this would take registers from its
// softmax: 645 -> 710 us for 8 prompts of up to 509 behind 16384). Where every range
// is in bounds they follow one another, and what lies outside is nobody's; else each
// token is looked up, so that one that a valid request holds is left to it.
// grid: any number of CTAs, a token at a time each; 32 registers a thread, so that
// one fits beside a CTA of that kernel.
template <int HD, typename Q>
__global__ void __launch_bounds__(kJoinThreads, 16) prefix_clear_kernel(PrefixAttnArgs a) {
  pdl_launch_dependents();
  bool valid = true;
  for (int i = threadIdx.x; i < a.n_requests; i += kJoinThreads) {
    int start, n, len;
    valid &= request_range(a, i, start, n, len);
  }
  const bool sound = __syncthreads_and(valid);
  // tokens [0, head) and [tail, n_tokens)
  const int head = sound ? a.token_start[0] : 0, tail = sound ? a.token_start[a.n_requests] : 0;
  for (long k = blockIdx.x; k < (long)head + a.n_tokens - tail; k += gridDim.x) {
    const long t = k < head ? k : tail + (k - head);
    if (!sound) {
      bool held = false;
      for (int i = threadIdx.x; i < a.n_requests; i += kJoinThreads) {
        int start, n, len;
        held |= request_range(a, i, start, n, len) && t >= start && t - start < n;
      }
      if (__syncthreads_or(held)) continue;
    }
    Q* dst = static_cast<Q*>(a.out) + t * a.out_stride;
    for (int i = threadIdx.x; i < a.nh * (HD / 4); i += kJoinThreads) store4(dst + i * 4, make_float4(0.f, 0.f, 0.f, 0.f));
  }
  pdl_wait();   // not done before the kernel beside it
}

}  // namespace ls

// Per-head RMS norm of the queries and keys, the position rotation in the
// same pass, and the new K/V rows written to their cache slots.
//
// For each head x of a token's q and k:  y = x * rsqrt(mean(x^2) + eps) * w,
// then for each rotated pair (y1, y2) with angle table entry (c, s)
//   (y1, y2) -> (y1 c - y2 s, y2 c + y1 s),
// pairs being (i, i + rot/2), or (2i, 2i + 1) in the interleaved form; the
// dimensions past `rot` pass unrotated. v is copied. All arithmetic is fp32
// and each output is rounded once, to its own type.
//
// HD/16 lanes own one head, 16 elements each: two 8-element chunks that hold
// whole pairs, so the rotation needs no exchange between lanes and the norm is
// log2(HD/16) shuffles. A warp covers 32*16/HD heads at a time.
//
// Bound: HBM for prompts (each row is read once, q, k and v written once),
// launch latency for decode batches. 8191 tokens of 16 + 32 heads of 128 in f16
// (203 MB): 37.7 us, 5.4 TB/s, four fifths of a plain copy; up to 61 tokens 2.1
// us, call after call in a graph.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace ls {

constexpr int kQkThreads = 128;

struct QkNormArgs {
  const void* qkv;
  long qkv_stride;       // elements
  int n_tokens, nh, nkv;
  const void* q_weight;
  const void* k_weight;
  int weight_type;
  float eps;
  const float* rope;     // [max_positions][2][rot/2]: cosines, then sines
  int max_positions, rot;
  const int* positions;
  const int* slots;      // or null: token t goes to row t
  void* k_pool;
  void* v_pool;
  long slot_stride;      // elements
  int n_slots;
  void* q_out;
  long q_out_stride;     // elements
  int* status;
  int parts;   // warps that share a token
};

__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = ld_f4(p), b = ld_f4(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) {
  unpack8(*reinterpret_cast<const uint4*>(p), f);
}
__device__ __forceinline__ void load8(const __half* p, float (&f)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
  __nv_bfloat162 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(v);
}
__device__ __forceinline__ void store8(__half* p, const float (&f)[8]) {
  __half2 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(v);
}
__device__ __forceinline__ void load8_as(const void* p, int type, int i, float (&f)[8]) {
  if (type == 0) load8(static_cast<const __nv_bfloat16*>(p) + i, f);
  else if (type == 1) load8(static_cast<const __half*>(p) + i, f);
  else load8(static_cast<const float*>(p) + i, f);
}

// 8 consecutive values as loaded: they wait in this form, half the registers of fp32 for 16-bit types.
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const { load8(reinterpret_cast<const T*>(v), f); }
};

// A warp takes one of `parts` parts of a token's heads: U passes of 512/HD heads,
// whose loads are all issued before the first is used.
template <typename T, typename C, int HD, bool INTERLEAVED, int U>
__global__ void __launch_bounds__(kQkThreads) qk_norm_rope_kernel(QkNormArgs a) {
  constexpr int L = HD / 16;                 // lanes of one head
  constexpr int HEADS = 32 / L;              // heads of a pass
  const unsigned unit = blockIdx.x * (kQkThreads / 32) + threadIdx.x / 32;
  const int t = (int)(unit / (unsigned)a.parts), part = (int)(unit % (unsigned)a.parts);
  if (t >= a.n_tokens) return;
  const int lane = threadIdx.x & 31, j = lane % L;
  const int heads = a.nh + 2 * a.nkv;
  pdl_wait();                // launched early: inputs may be on their way
  pdl_launch_dependents();   // what follows waits for this kernel in the same way
  const int pos = a.positions[t];
  const int slot = a.slots ? a.slots[t] : t;
  const T* src = static_cast<const T*>(a.qkv) + (long)t * a.qkv_stride;

  // this lane's chunks (units of 8 elements): the rotated ones hold whole
  // pairs, the rest are neighbours
  int ca, cb;
  bool turn_a, turn_b;
  const int rc = a.rot / 8;                  // rotated chunks, an even number
  if (INTERLEAVED) {
    ca = j;
    cb = j + L;
    turn_a = ca < rc;
    turn_b = cb < rc;
  } else {
    turn_a = turn_b = j < rc / 2;
    ca = turn_a ? j : rc + 2 * (j - rc / 2);
    cb = turn_a ? j + rc / 2 : ca + 1;
  }
  // the heads are on their way while the position is looked up
  const int first = part * (HEADS * U) + lane / L;
  Raw8<T> xs[U], ys[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = min(first + u * HEADS, heads - 1);   // past the last: read it again, store nothing
    xs[u].load(src + (long)h * HD + 8 * ca);
    ys[u].load(src + (long)h * HD + 8 * cb);
  }

  const bool pos_ok = pos >= 0 && pos < a.max_positions;
  const bool slot_ok = pos_ok && slot >= 0 && slot < a.n_slots;
  // a slot of -1 marks padding, whose K/V go nowhere
  if (lane == 0 && (!pos_ok || slot < -1 || slot >= a.n_slots)) atomicCAS(a.status, kDevOk, kDevBadIndex);

  // cosines and sines: 8 pairs (i, i + rot/2), or 4 pairs of each chunk
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cs[i] = 1.f;
    sn[i] = 0.f;
  }
  if (pos_ok) {
    const float* row = a.rope + (long)pos * a.rot;
    const int half = a.rot / 2;
    if (INTERLEAVED) {
      if (turn_a) {
        *reinterpret_cast<float4*>(cs) = ld_f4(row + 4 * ca);
        *reinterpret_cast<float4*>(sn) = ld_f4(row + half + 4 * ca);
      }
      if (turn_b) {
        *reinterpret_cast<float4*>(cs + 4) = ld_f4(row + 4 * cb);
        *reinterpret_cast<float4*>(sn + 4) = ld_f4(row + half + 4 * cb);
      }
    } else if (turn_a) {
      load8(row + 8 * j, cs);
      load8(row + half + 8 * j, sn);
    }
  }

  T* q_row = static_cast<T*>(a.q_out) + (long)t * a.q_out_stride;
  C* k_row = static_cast<C*>(a.k_pool) + (long)(slot_ok ? slot : 0) * a.slot_stride;
  C* v_row = static_cast<C*>(a.v_pool) + (long)(slot_ok ? slot : 0) * a.slot_stride;
  // the whole warp stays in the loop: the norm's shuffles need every lane
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float x[8], y[8];
    xs[u].get(x);
    ys[u].get(y);
    const int h = first + u * HEADS;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i] + y[i] * y[i];
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (h >= heads) continue;
    if (h >= a.nh + a.nkv) {
      if (slot_ok) {
        store8(v_row + (long)(h - a.nh - a.nkv) * HD + 8 * ca, x);
        store8(v_row + (long)(h - a.nh - a.nkv) * HD + 8 * cb, y);
      }
      continue;
    }
    float wx[8], wy[8];
    const void* w = h < a.nh ? a.q_weight : a.k_weight;
    load8_as(w, a.weight_type, 8 * ca, wx);
    load8_as(w, a.weight_type, 8 * cb, wy);
    const float inv = rsqrtf(ss / HD + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = x[i] * inv * wx[i];
      y[i] = y[i] * inv * wy[i];
    }
    // unrotated chunks stay out of the products: 0 * inf would spoil them
    if (INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x1 = x[2 * i], x2 = x[2 * i + 1], y1 = y[2 * i], y2 = y[2 * i + 1];
        if (turn_a) {
          x[2 * i] = x1 * cs[i] - x2 * sn[i];
          x[2 * i + 1] = x2 * cs[i] + x1 * sn[i];
        }
        if (turn_b) {
          y[2 * i] = y1 * cs[4 + i] - y2 * sn[4 + i];
          y[2 * i + 1] = y2 * cs[4 + i] + y1 * sn[4 + i];
        }
      }
    } else if (turn_a) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x1 = x[i], x2 = y[i];
        x[i] = x1 * cs[i] - x2 * sn[i];
        y[i] = x2 * cs[i] + x1 * sn[i];
      }
    }
    if (h < a.nh) {
      store8(q_row + (long)h * HD + 8 * ca, x);
      store8(q_row + (long)h * HD + 8 * cb, y);
    } else if (slot_ok) {
      store8(k_row + (long)(h - a.nh) * HD + 8 * ca, x);
      store8(k_row + (long)(h - a.nh) * HD + 8 * cb, y);
    }
  }
}

}  // namespace ls

// Block tables and slot maps from request lengths, on the GPU.
//
// Request i holds len_i tokens in blocks of `page` slots (its table row) and
// changes by delta_i: it grows (delta_i new tokens) or is cut back (rejected
// drafts, a finished request). With have = ceil(len / page) and
// need = ceil((len + delta) / page) it takes max(0, need - have) blocks and
// gives back max(0, have - need). The free blocks are a stack; what is given
// back is pushed first, in request order and ascending block index, then the
// k-th new block (request order) is popped: entry count + given - 1 - k. New
// token j of request i sits at position len_i + j, in slot
// table[i][pos / page] * page + pos % page.
//
// One launch. Every CTA computes the three running sums over the requests
// (tokens, blocks taken, blocks given back) by itself, a few KB from L2, so no
// CTA waits for another's; then tokens and blocks are spread over the grid,
// each found by a binary search in the sums. A pop that reaches below the
// stack's old top reads the giving request's table entry itself and pushes
// write only above it, so no read of the call meets a write of the call,
// except where lens and the count are updated in place: then the grid is one
// thread-block cluster (at most 8 CTAs) and they are written after a barrier.
// Nothing changes when the call cannot be done as a whole.
//
// Bound: launch and dependent-load latency (a decode step moves a few KB).
// Call after call in a graph: 61 requests 3.7 us, 517 requests with up to eight
// drafts each 5.5 us, 96 prompts of up to 2048 tokens (1.2 MB written) 4.6 us.
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"

namespace ls {

constexpr int kSlotThreads = 512;
constexpr int kSlotMaxCluster = 8;       // portable cluster size
constexpr int kSlotMaxRequests = 16384;  // three int32 sums a request in shared memory: 192 KB

struct SlotArgs {
  const int* lens;
  const int* delta;
  int n_requests;
  int* table;
  long table_stride;
  int table_width;
  int* free_blocks;
  int free_capacity;
  const int* free_count;
  int n_blocks;
  int page_shift;
  int base;
  int max_tokens;
  int* slots;
  int* positions;
  int* requests;
  int* token_start;
  int* lens_out;
  int* free_count_out;
  int* status;
  bool in_place;
};

inline size_t slot_smem_bytes(int n_requests) { return sizeof(int) * 3 * ((size_t)n_requests + 1); }

// Last index i with sums[i] <= k, for sums ascending, sums[0] = 0 and k < sums[n].
__device__ __forceinline__ int owner_of(const int* sums, int n, int k) {
  int lo = 0, hi = n;   // sums[lo] <= k < sums[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= k) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kSlotThreads) build_slots_kernel(SlotArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ int s_sums[];
  const int R = a.n_requests;
  int* s_tok = s_sums;
  int* s_grow = s_sums + (R + 1);
  int* s_back = s_sums + 2 * (R + 1);
  __shared__ long long s_tok_part[kSlotThreads / 32];
  __shared__ int2 s_part[kSlotThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int page = 1 << a.page_shift;
  const long capacity = (long)a.table_width << a.page_shift;
  pdl_wait();                // launched early: inputs may be on their way
  pdl_launch_dependents();   // what follows waits for this kernel in the same way

  // running sums: each thread adds a run of consecutive requests, the block
  // scans the runs (64-bit: lengths may be garbage), the thread lays them out
  const int per = (R + kSlotThreads - 1) / kSlotThreads;
  const int r0 = min(R, tid * per), r1 = min(R, r0 + per);
  long long tok = 0;
  int grow = 0, back = 0;   // table entries, below 2^31 in all
  int bad = 0;
  for (int i = r0; i < r1; ++i) {
    const long len = a.lens[i], now = len + a.delta[i];
    if (len < 0 || len > capacity || now < 0 || now > capacity) {
      bad = 1;
      continue;
    }
    const int have = (int)((len + page - 1) >> a.page_shift), need = (int)((now + page - 1) >> a.page_shift);
    tok += max(0L, now - len);
    grow += max(0, need - have);
    back += max(0, have - need);
  }
  const long count = a.free_count[0];
  long long tok_to = tok;
  int grow_to = grow, back_to = back;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, tok_to, o);
    const int g = __shfl_up_sync(0xffffffffu, grow_to, o), b = __shfl_up_sync(0xffffffffu, back_to, o);
    if (lane >= o) {
      tok_to += t;
      grow_to += g;
      back_to += b;
    }
  }
  if (lane == 31) {
    s_tok_part[warp] = tok_to;
    s_part[warp] = make_int2(grow_to, back_to);
  }
  bad = __syncthreads_or(bad);
  // the warps' totals: each warp scans the 16 of them again
  long long n_tok_all = lane < kSlotThreads / 32 ? s_tok_part[lane] : 0;
  int2 all = lane < kSlotThreads / 32 ? s_part[lane] : make_int2(0, 0);
#pragma unroll
  for (int o = 1; o < kSlotThreads / 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, n_tok_all, o);
    const int g = __shfl_up_sync(0xffffffffu, all.x, o), b = __shfl_up_sync(0xffffffffu, all.y, o);
    if (lane >= o) {
      n_tok_all += t;
      all.x += g;
      all.y += b;
    }
  }
  const int before = max(0, warp - 1);
  const long long tok_before = __shfl_sync(0xffffffffu, n_tok_all, before);
  const int grow_before = __shfl_sync(0xffffffffu, all.x, before), back_before = __shfl_sync(0xffffffffu, all.y, before);
  const long long total_tok = __shfl_sync(0xffffffffu, n_tok_all, kSlotThreads / 32 - 1);
  const long total_grow = __shfl_sync(0xffffffffu, all.x, kSlotThreads / 32 - 1),
             total_back = __shfl_sync(0xffffffffu, all.y, kSlotThreads / 32 - 1);
  tok_to += (warp ? tok_before : 0) - tok;
  grow_to += (warp ? grow_before : 0) - grow;
  back_to += (warp ? back_before : 0) - back;
  int code = kDevOk;
  if (bad || count < 0 || count > a.free_capacity) code = kDevBadLength;
  else if (total_tok > a.max_tokens) code = kDevTooManyTokens;
  else if (total_grow > count + total_back) code = kDevNoBlocks;
  else if (count + total_back - total_grow > a.free_capacity) code = kDevBadLength;

  // unsigned: the loops' counters go past their ends, which may be 2^31 - 1, by up to a step
  const unsigned at = blockIdx.x * kSlotThreads + tid, step = gridDim.x * kSlotThreads;
  const unsigned n_buffer = (unsigned)a.max_tokens, n_req = (unsigned)R;
  if (code != kDevOk) {   // all or nothing
    if (at == 0) atomicCAS(a.status, kDevOk, code);
    for (unsigned k = at; k < n_buffer; k += step) {
      a.slots[k] = -1;
      a.positions[k] = 0;
      a.requests[k] = -1;
    }
    for (unsigned i = at; i <= n_req; i += step) a.token_start[i] = 0;
    if (a.lens_out != a.lens)
      for (unsigned i = at; i < n_req; i += step) a.lens_out[i] = a.lens[i];
    if (a.free_count_out != a.free_count && at == 0) a.free_count_out[0] = (int)count;
    return;
  }

  int t = (int)tok_to, g = grow_to, b = back_to;
  for (int i = r0; i < r1; ++i) {
    const int len = a.lens[i], now = len + a.delta[i];
    const int have = (len + page - 1) >> a.page_shift, need = (now + page - 1) >> a.page_shift;
    s_tok[i] = t;
    s_grow[i] = g;
    s_back[i] = b;
    t += max(0, now - len);
    g += max(0, need - have);
    b += max(0, have - need);
  }
  const int n_tok = (int)total_tok, n_take = (int)total_grow, n_give = (int)total_back;
  if (tid == 0) {
    s_tok[R] = n_tok;
    s_grow[R] = n_take;
    s_back[R] = n_give;
  }
  __syncthreads();

  // the p-th block given back by this call
  auto given = [&](int p) {
    const int i = owner_of(s_back, R, p);
    const int now = a.lens[i] + a.delta[i];
    return a.table[i * a.table_stride + ((now + page - 1) >> a.page_shift) + (p - s_back[i])];
  };
  // the k-th new block of this call
  auto taken = [&](int k) {
    const long p = count + n_give - 1 - k;
    return p < count ? a.free_blocks[p] : given((int)(p - count));
  };

  for (unsigned k = at; k < n_buffer; k += step) {
    int slot = -1, position = 0, request = -1;
    if (k < (unsigned)n_tok) {
      request = owner_of(s_tok, R, (int)k);
      const int len = a.lens[request];
      const int pos = len + ((int)k - s_tok[request]);
      const int have = (len + page - 1) >> a.page_shift, blk = pos >> a.page_shift;
      const int block = blk < have ? a.table[request * a.table_stride + blk]
                                   : taken(s_grow[request] + blk - have);
      if (block < 0 || block >= a.n_blocks) atomicCAS(a.status, kDevOk, kDevBadIndex);
      else slot = (block << a.page_shift) + (pos & (page - 1));
      position = a.base + pos;
    }
    a.slots[k] = slot;
    a.positions[k] = position;
    a.requests[k] = request;
  }
  for (unsigned k = at; k < (unsigned)n_take; k += step) {
    const int i = owner_of(s_grow, R, (int)k);
    const int have = (a.lens[i] + page - 1) >> a.page_shift;
    a.table[i * a.table_stride + have + ((int)k - s_grow[i])] = taken((int)k);
  }
  for (long p = count + at; p < count + n_give - n_take; p += step) {
    const int block = given((int)(p - count));
    if (block < 0 || block >= a.n_blocks) atomicCAS(a.status, kDevOk, kDevBadIndex);   // taken ones are told by their token
    a.free_blocks[p] = block;
  }
  for (unsigned i = at; i <= n_req; i += step) a.token_start[i] = s_tok[i];
  if (a.in_place) cg::this_cluster().sync();   // every CTA has read lens and the count
  for (unsigned i = at; i < n_req; i += step) a.lens_out[i] = a.lens[i] + a.delta[i];
  if (at == 0) a.free_count_out[0] = (int)(count + n_give - n_take);
}

}  // namespace ls

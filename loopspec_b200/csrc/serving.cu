// C entry points of the shared-prefix serving step: slot maps, per-head norm
// with rotation and K/V write, prefix attention. Each checks its arguments,
// picks the kernel variant and enqueues; none waits or allocates.

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "host.cuh"
#include "prefix_attn.cuh"
#include "prefix_tc.cuh"
#include "qk_norm.cuh"
#include "slots.cuh"

using namespace ls;
typedef __nv_bfloat16 bf16;

namespace {

int current_device() {
  int dev = 0;
  CK(cudaGetDevice(&dev));
  return dev;
}

// Facts of a device and grants to a kernel on it are looked up once a process.
constexpr int kMaxDevices = 64;

int sm_count() {
  static std::atomic<int> known[kMaxDevices];
  const int dev = current_device();
  int sms = dev < kMaxDevices ? known[dev].load(std::memory_order_relaxed) : 0;
  if (sms == 0) {
    CK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    if (dev < kMaxDevices) known[dev].store(sms, std::memory_order_relaxed);
  }
  return sms;
}

int cdiv(long a, long b) { return (int)((a + b - 1) / b); }

int page_shift_of(int page_size, const char* who) {
  int s = 0;
  while (s < 10 && (1 << s) < page_size) ++s;
  REQUIRE(page_size >= 1 && (1 << s) == page_size, LS_EINVAL,
          std::string(who) + ": page_size must be a power of two in [1, 1024]");
  return s;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
long type_bytes(int type) { return type == LS_F32 ? 4 : 2; }

// Let `kernel` have up to `most` bytes of dynamic shared memory on this device.
template <auto kernel>
void allow_smem(size_t most) {
  static std::atomic<bool> granted[kMaxDevices];
  const int dev = current_device();
  if (dev < kMaxDevices && granted[dev].load(std::memory_order_relaxed)) return;
  CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
  if (dev < kMaxDevices) granted[dev].store(true, std::memory_order_relaxed);
}

template <typename F>
int guarded(F f) {
  try {
    f();
  } catch (const std::exception& ex) {
    return fail_global(ex);
  } catch (...) {
    return fail_global(EngineError(LS_EINVAL, "unknown failure"));
  }
  return LS_OK;
}

// ------------------------------------------------------------------- slot maps
void run_build_slots(const ls_slots_args& p, cudaStream_t stream) {
  const char* who = "slot maps";
  REQUIRE(p.lens && p.delta && p.block_table && p.free_blocks && p.free_count && p.token_start &&
              p.lens_out && p.free_count_out && p.status,
          LS_EINVAL, "slot maps: null pointer argument");
  REQUIRE(p.max_tokens >= 0 && (p.max_tokens == 0 || (p.slots && p.positions && p.requests)), LS_EINVAL,
          "slot maps: max_tokens must not be negative and its buffers not null");
  REQUIRE(p.n_requests >= 1 && p.n_requests <= kSlotMaxRequests, LS_EINVAL,
          "slot maps: n_requests must be in [1, " + std::to_string(kSlotMaxRequests) + "]");
  REQUIRE(p.table_width >= 1 && p.table_stride >= p.table_width && p.free_capacity >= 0 && p.n_blocks >= 1,
          LS_EINVAL, "slot maps: table_width, table_stride, free_capacity or n_blocks out of range");
  const int shift = page_shift_of(p.page_size, who);
  const int64_t kTop = INT32_MAX;
  REQUIRE((int64_t)p.n_blocks << shift <= kTop && (int64_t)p.table_width << shift <= kTop &&
              (int64_t)p.n_requests * p.table_width <= kTop && p.base >= 0 &&
              (int64_t)p.base + ((int64_t)p.table_width << shift) <= kTop,
          LS_EINVAL, "slot maps: slots, positions and table entries must stay below 2^31");
  SlotArgs a{p.lens, p.delta, p.n_requests, p.block_table, (long)p.table_stride, p.table_width,
             p.free_blocks, p.free_capacity, p.free_count, p.n_blocks, shift, p.base, p.max_tokens,
             p.slots, p.positions, p.requests, p.token_start, p.lens_out, p.free_count_out, p.status, false};
  const size_t smem = slot_smem_bytes(p.n_requests);
  allow_smem<build_slots_kernel>(slot_smem_bytes(kSlotMaxRequests));   // 48 KB without it, the static part included
  a.in_place = p.lens_out == p.lens || p.free_count_out == p.free_count;
  // a token a thread, on as many SMs as that takes: each CTA repeats the sums,
  // but the token loop's dependent loads (length, block) are what takes time
  // (98000 tokens, with a graph launch: 10 us over the grid, 28 by the one cluster of in-place updates)
  const int work = std::max({p.max_tokens, p.n_requests, 1});
  int ctas = std::min(cdiv(work, kSlotThreads), sm_count());
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (a.in_place) {
    ctas = std::min(ctas, kSlotMaxCluster);
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)ctas, 1, 1};
    cfg.numAttrs = 2;
  }
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kSlotThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  CK(cudaLaunchKernelEx(&cfg, build_slots_kernel, a));
}

// ----------------------------------------------------------- norm and rotation
template <typename T, typename C, int HD, int U>
void launch_qk(const QkNormArgs& a, bool interleaved, cudaStream_t stream) {
  const long warps = (long)a.n_tokens * a.parts;
  REQUIRE(warps <= INT32_MAX, LS_EINVAL, "qk norm: too many tokens and heads for one launch");
  const dim3 grid((unsigned)cdiv(warps, kQkThreads / 32));
  if (interleaved) launch(qk_norm_rope_kernel<T, C, HD, true, U>, grid, dim3(kQkThreads), 0, stream, true, a);
  else launch(qk_norm_rope_kernel<T, C, HD, false, U>, grid, dim3(kQkThreads), 0, stream, true, a);
}

// One pass a warp while the passes fit the GPU at once; up to three for prompts,
// where loads in flight decide, as evenly as the heads go (61 tokens: 2.1 us with
// one, 2.9 with three; 8191 tokens of 48 heads: 44.0 and 37.7).
template <typename T, typename C, int HD>
void launch_qk(QkNormArgs a, bool interleaved, cudaStream_t stream) {
  const int passes = cdiv(a.nh + 2 * a.nkv, 512 / HD);
  a.parts = (long)a.n_tokens * passes <= 32L * sm_count() ? passes : cdiv(passes, 3);
  const int each = cdiv(passes, a.parts);
  if (each == 1) launch_qk<T, C, HD, 1>(a, interleaved, stream);
  else if (each == 2) launch_qk<T, C, HD, 2>(a, interleaved, stream);
  else launch_qk<T, C, HD, 3>(a, interleaved, stream);
}

template <typename T, typename C>
void launch_qk(const QkNormArgs& a, int hd, bool interleaved, cudaStream_t stream) {
  if (hd == 64) launch_qk<T, C, 64>(a, interleaved, stream);
  else launch_qk<T, C, 128>(a, interleaved, stream);
}

void run_qk_norm_rope(const ls_qk_norm_args& p, cudaStream_t stream) {
  REQUIRE(p.n_tokens >= 0, LS_EINVAL, "qk norm: n_tokens must not be negative");
  REQUIRE(p.n_heads >= 1 && p.n_kv_heads >= 1 && (p.head_dim == 64 || p.head_dim == 128), LS_EINVAL,
          "qk norm: head counts must be positive and head_dim 64 or 128");
  REQUIRE(p.qkv_type >= LS_BF16 && p.qkv_type <= LS_F32 && p.weight_type >= LS_BF16 && p.weight_type <= LS_F32 &&
              (p.cache_type == LS_BF16 || p.cache_type == LS_F16) &&
              (p.qkv_type == LS_F32 || p.qkv_type == p.cache_type),
          LS_EINVAL, "qk norm: the cache must be bf16 or f16, and qkv of its type or fp32");
  REQUIRE(p.rot >= 16 && p.rot % 16 == 0 && p.rot <= p.head_dim, LS_EINVAL,
          "qk norm: rot must be a multiple of 16 up to head_dim");
  REQUIRE(p.max_positions >= 1 && p.n_slots >= 1, LS_EINVAL, "qk norm: max_positions and n_slots must be positive");
  const int64_t qd = (int64_t)p.n_heads * p.head_dim, kd = (int64_t)p.n_kv_heads * p.head_dim;
  REQUIRE(p.qkv_stride >= qd + 2 * kd && p.q_out_stride >= qd && p.slot_stride >= kd, LS_EINVAL,
          "qk norm: a stride is smaller than its row");
  if (p.n_tokens == 0) return;
  REQUIRE(p.qkv && p.q_weight && p.k_weight && p.rope && p.positions && p.k_pool && p.v_pool && p.q_out && p.status,
          LS_EINVAL, "qk norm: null pointer argument");
  const long eb = type_bytes(p.qkv_type), cb = type_bytes(p.cache_type);
  REQUIRE(aligned16(p.qkv) && aligned16(p.q_weight) && aligned16(p.k_weight) && aligned16(p.rope) &&
              aligned16(p.k_pool) && aligned16(p.v_pool) && aligned16(p.q_out) && p.qkv_stride * eb % 16 == 0 &&
              p.q_out_stride * eb % 16 == 0 && p.slot_stride * cb % 16 == 0,
          LS_EINVAL, "qk norm: pointers and row strides must be 16-byte aligned");
  QkNormArgs a{p.qkv, (long)p.qkv_stride, p.n_tokens, p.n_heads, p.n_kv_heads, p.q_weight, p.k_weight,
               p.weight_type, p.eps, p.rope, p.max_positions, p.rot, p.positions, p.slots, p.k_pool, p.v_pool,
               (long)p.slot_stride, p.n_slots, p.q_out, (long)p.q_out_stride, p.status, 1};
  const bool il = p.interleaved != 0;
  if (p.qkv_type == LS_BF16) launch_qk<bf16, bf16>(a, p.head_dim, il, stream);
  else if (p.qkv_type == LS_F16) launch_qk<__half, __half>(a, p.head_dim, il, stream);
  else if (p.cache_type == LS_BF16) launch_qk<float, bf16>(a, p.head_dim, il, stream);
  else launch_qk<float, __half>(a, p.head_dim, il, stream);
}

// ------------------------------------------------------------ prefix attention
// How a call is cut into units: a function of its sizes and types alone.
struct PrefixPlan {
  int tc_tiles;     // 128-row tiles a CTA of the tcgen05 kernel takes; 0: the stream kernel does everything
  bool own;         // it takes one request's rows and also does that request's own positions
  int prefix_parts, prefix_chunk, suffix_parts, suffix_chunk, prefix_tiles, suffix_tiles;
  int rt;                     // eights of rows in a tile of the stream kernel
  int stream_sms;             // SMs the stream kernel is launched for
  size_t o_bytes, ml_bytes, total;
};

constexpr int kMaxParts = 64;   // of a request's own positions, and of what the tcgen05 kernel does

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Key ranges of `len` positions for `units` row tiles: as many as keep
// `resident` units on the GPU, none under `least` positions.
void cut(long units, int len, long resident, int least, int grain, int most, int& parts, int& chunk) {
  parts = chunk = 0;
  if (len == 0) return;
  const long want = std::max(1L, resident / std::max(1L, units));
  parts = (int)std::min<long>(want, std::min(most, std::max(1, cdiv(len, least))));
  chunk = cdiv(cdiv(len, parts), grain) * grain;
  parts = cdiv(len, chunk);
}

// Fewest keys of a stream unit: 64, or 32 where that leaves most SMs idle (4
// requests behind 333 positions: 10.3 -> 8.3 us; 16 behind 2048: 23.0 -> 24.5).
int least_keys(long units, int len, int sms) { return units * cdiv(len, 64) <= 2L * sms ? 32 : 64; }

// Measured costs, in cycles of an SM. A CTA of the tcgen05 kernel fills one and
// spends kAround besides its key tiles (lookups, first copies, results out).
// The stream kernel spends kStreamAround on every SM.
constexpr double kAround = 16000, kStreamAround = 6000, kJoinAround = 6000;

double tc_tile_cycles(int hd, int terms, int tc_tiles) {
  const double products = (hd == 128 ? 1030. : 520.) * terms * tc_tiles;   // both, at the tensor cores' rate
  const double softmax = terms > 1 ? 2000 : tc_tiles == 2 ? (hd == 128 ? 3400 : 3000) : 1800;
  return std::max(products * 1.1, softmax);
}

// ... and this a tile of 16 keys by 8 or 16 rows
double stream_tile_cycles(int terms, int rt) { return terms == 1 ? (rt == 1 ? 300 : 560) : (rt == 1 ? 450 : 1000); }

// How many key ranges the tcgen05 kernel cuts the shared prefix into, and the
// SMs left to the stream kernel, which does the requests' own positions beside
// it: the two share the GPU by SMs. Fewer, longer CTAs waste less around their
// tiles (33 requests of 5 drafts behind 5001 positions: 5 ranges beside the
// stream take 44000 cycles, 10 ranges and then the stream 50000). Returns the
// cycles it expects.
double share(PrefixPlan& p, int prefix_len, double tile_cycles, double stream_cycles, int sms, int units) {
  const int tiles = cdiv(prefix_len, kTcKeys);
  auto ranged = [&](int parts) { return kAround + tile_cycles * cdiv(tiles, parts); };
  const int most = std::max(1, std::min({sms / units, tiles, kMaxParts}));
  double best = 0;
  for (int parts = 1; parts <= most; ++parts) {
    const int ctas = units * cdiv(tiles, cdiv(tiles, parts));
    const double after = ranged(parts) * cdiv(ctas, sms) + stream_cycles / sms;
    // lengths are only bounded: never stretch the prefix far for the sake of the rest
    const double beside = ctas < sms && ranged(parts) <= 2 * ranged(most)
                              ? std::max(ranged(parts), stream_cycles / (sms - ctas)) : after;
    const double cycles = std::min(after, beside);
    if (best == 0 || cycles < best) {
      best = cycles;
      p.prefix_chunk = cdiv(tiles, parts) * kTcKeys;
      p.stream_sms = beside < after ? sms - ctas : sms;
    }
  }
  p.prefix_parts = cdiv(prefix_len, p.prefix_chunk);
  return best;
}

// Eights of rows in a row tile of the stream kernel: the rows there are, up to
// what q and O leave registers for.
int tile_eights(long rows) { return rows <= 8 ? 1 : 2; }

// terms: 1 for 16-bit q, else those of an fp32 q (see prefix_attn.cuh).
PrefixPlan make_plan(int n_tokens, int n_requests, int nh, int nkv, int hd, int prefix_len, int max_new,
                     int max_len, int terms, int sms) {
  PrefixPlan p{};
  const int G = nh / nkv;
  const long rows = (long)n_tokens * G;
  const long most_rows = (long)std::min(max_new, n_tokens) * G, mean_rows = cdiv(rows, n_requests);

  // one way: the prefix for all rows together, the requests' own positions by the stream kernel
  p.rt = tile_eights(most_rows);
  p.suffix_tiles = cdiv(most_rows, 8 * p.rt);
  p.stream_sms = sms;
  const double own_tiles = (double)n_requests * nkv * cdiv(mean_rows, 8 * p.rt) * max_len / 16 / 2;
  const double stream_cycles = max_len ? stream_tile_cycles(terms, p.rt) * own_tiles + kStreamAround * sms : 0;
  double cycles = stream_cycles / sms + kJoinAround;
  if (rows > 16 && prefix_len > 0) {
    p.tc_tiles = terms > 1 || rows <= kTcRows ? 1 : 2;
    p.prefix_tiles = cdiv(rows, kTcRows * p.tc_tiles);
    const int units = (int)std::min<long>((long)p.prefix_tiles * nkv, 1 << 20);
    cycles = share(p, prefix_len, tc_tile_cycles(hd, terms, p.tc_tiles), stream_cycles, sms, units) + kJoinAround;
  } else {
    // one launch for both if it reads the prefix no more than twice (from L2)
    p.prefix_tiles = cdiv(rows, 8 * p.rt);
    const long units = (long)p.prefix_tiles * nkv;
    cut(units, prefix_len, 12L * sms, least_keys(units, prefix_len, sms), 16, 4 * kMaxParts, p.prefix_parts,
        p.prefix_chunk);
  }
  // lengths are spread below max_len: two ranges a warp (12 an SM) even that out
  const long own_units = (long)p.suffix_tiles * nkv * n_requests;
  cut(own_units, max_len, 24L * p.stream_sms, least_keys(own_units, max_len, sms), 16, kMaxParts, p.suffix_parts,
      p.suffix_chunk);

  // the other way, for requests that bring about a tile of rows: each by itself, prefix and own positions
  if (most_rows > 16) {
    const int mt = terms > 1 || most_rows <= kTcRows ? 1 : 2;
    const int tiles = cdiv(prefix_len, kTcKeys) + cdiv(max_len, kTcKeys);
    const double units = (double)n_requests * nkv * cdiv(mean_rows, kTcRows * mt);
    for (int parts = 1; parts <= std::min(tiles, kMaxParts); ++parts) {
      const int each = cdiv(tiles, parts);
      const double ctas = units * cdiv(tiles, each);
      const double by_itself = (kAround + tc_tile_cycles(hd, terms, mt) * each) * std::ceil(ctas / sms) +
                               (parts > 1 ? kJoinAround : 0);
      if (by_itself < cycles) {
        cycles = by_itself;
        p.own = true;
        p.tc_tiles = mt;
        p.prefix_tiles = cdiv(most_rows, kTcRows * mt);
        p.prefix_chunk = each * kTcKeys;
        p.prefix_parts = cdiv(tiles, each);
        p.suffix_parts = 0;
      }
      if (ctas > 2.0 * sms) break;
    }
  }
  const bool direct = p.own && p.prefix_parts <= 1;   // whole results, no parts to keep
  const size_t part_rows = direct ? 0 : (size_t)(p.prefix_parts + p.suffix_parts) * n_tokens * nh;
  p.o_bytes = round256(part_rows * hd * sizeof(float));
  p.ml_bytes = round256(part_rows * sizeof(float2));
  p.total = p.o_bytes + p.ml_bytes;
  return p;
}

template <int HD, typename Q, typename C, int TERMS, int MT>
void launch_tc(const PrefixAttnArgs& a, cudaStream_t stream) {
  using L = TcLayout<HD, TERMS, MT>;
  allow_smem<prefix_tc_kernel<HD, Q, C, TERMS, MT>>(L::kSmem);
  // the register hand-over inside the kernel waits for good if the launch holds less than it shares out
  static const int regs = [] {
    cudaFuncAttributes attr = {};
    CK(cudaFuncGetAttributes(&attr, prefix_tc_kernel<HD, Q, C, TERMS, MT>));
    return attr.numRegs;
  }();
  REQUIRE(regs >= L::kLaunchRegs, LS_ECUDA,
          "prefix attention: built with " + std::to_string(regs) + " registers a thread, fewer than it shares out");
  const long units = (long)a.prefix_tiles * a.nkv * std::max(1, a.prefix_parts) * (a.own ? a.n_requests : 1);
  REQUIRE(units <= INT32_MAX, LS_EINVAL, "prefix attention: too many units for one launch");
  launch(prefix_tc_kernel<HD, Q, C, TERMS, MT>, dim3((unsigned)units), dim3(L::kThreads), (size_t)L::kSmem, stream,
         true, a);
}

// The stream kernel over the prefix, the requests' own positions or both.
// `behind`: a kernel of this call is ahead of it.
template <int HD, typename Q, typename C, int TERMS, int RT>
void launch_stream(PrefixAttnArgs a, bool prefix, bool suffix, bool behind, int sms, cudaStream_t stream) {
  const long units = (prefix ? (long)a.prefix_parts * a.prefix_tiles * a.nkv : 0) +
                     (suffix ? (long)a.suffix_parts * a.suffix_tiles * a.nkv * a.n_requests : 0);
  REQUIRE(units <= INT32_MAX / 2, LS_EINVAL, "prefix attention: too many units for one launch");   // and a stride past the last
  a.prefix_units = prefix;
  a.suffix_units = suffix;
  a.behind = behind;
  const size_t smem = unit_smem_bytes<HD, TERMS, RT>();
  allow_smem<prefix_stream_kernel<HD, Q, C, TERMS, RT>>(smem);
  const long ctas = std::min<long>((long)unit_ctas<HD, TERMS, RT>() * sms, cdiv(units, kUnitWarps));
  launch(prefix_stream_kernel<HD, Q, C, TERMS, RT>, dim3((unsigned)ctas), dim3(kUnitThreads), smem, stream, true, a);
}

template <int HD, typename Q, typename C, int TERMS>
void launch_stream(const PrefixAttnArgs& a, int rt, bool prefix, bool suffix, bool behind, int sms, cudaStream_t stream) {
  if (rt == 1) launch_stream<HD, Q, C, TERMS, 1>(a, prefix, suffix, behind, sms, stream);
  else launch_stream<HD, Q, C, TERMS, 2>(a, prefix, suffix, behind, sms, stream);
}

template <int HD, typename Q, typename C, int TERMS>
void launch_prefix(PrefixAttnArgs a, const PrefixPlan& plan, cudaStream_t stream) {
  if (plan.tc_tiles == 1) launch_tc<HD, Q, C, TERMS, 1>(a, stream);
  if constexpr (TERMS == 1) {
    if (plan.tc_tiles == 2) launch_tc<HD, Q, C, TERMS, 2>(a, stream);
  }
  if (a.direct) {
    launch(prefix_clear_kernel<HD, Q>, dim3((unsigned)std::min(a.n_tokens, sm_count())), dim3(kJoinThreads), 0, stream, true, a);
    return;
  }
  const bool prefix = plan.tc_tiles == 0 && a.prefix_parts > 0, suffix = a.suffix_parts > 0 && a.suffix_tiles > 0;
  const bool behind = plan.tc_tiles != 0;
  if (prefix || suffix) launch_stream<HD, Q, C, TERMS>(a, plan.rt, prefix, suffix, behind, plan.stream_sms, stream);
  a.behind = behind || prefix || suffix;
  constexpr int kGroups = kJoinThreads / (HD / 4);
  const dim3 rows((unsigned)a.n_tokens, (unsigned)a.nh), groups((unsigned)a.n_tokens, (unsigned)cdiv(a.nh, kGroups));
  // many parts come with few rows: a row's parts are shared out (4 requests behind
  // 333 positions: 6.7 us, 9.0 with a group a row; 16 behind 2048: 21.4 and 29.6)
  if (a.prefix_parts + a.suffix_parts > kJoinBatch)
    launch(prefix_join_kernel<HD, Q, C, true>, rows, dim3(kJoinThreads), 0, stream, true, a);
  else launch(prefix_join_kernel<HD, Q, C, false>, groups, dim3(kJoinThreads), 0, stream, true, a);
}

template <typename Q, typename C, int TERMS>
void launch_prefix(const PrefixAttnArgs& a, int hd, const PrefixPlan& plan, cudaStream_t stream) {
  if (hd == 64) launch_prefix<64, Q, C, TERMS>(a, plan, stream);
  else launch_prefix<128, Q, C, TERMS>(a, plan, stream);
}

void check_prefix_sizes(int n_tokens, int n_requests, int nh, int nkv, int hd, int prefix_len, int max_new,
                        int max_len) {
  REQUIRE(n_tokens >= 0 && n_requests >= 1 && nh >= 1 && nkv >= 1 && prefix_len >= 0 && max_new >= 0 && max_len >= 0,
          LS_EINVAL, "prefix attention: sizes must not be negative, requests and heads positive");
  REQUIRE(nh % nkv == 0, LS_EINVAL, "prefix attention: n_heads must be a multiple of n_kv_heads");
  REQUIRE(hd == 64 || hd == 128, LS_EINVAL, "prefix attention: head_dim must be 64 or 128");
  REQUIRE((int64_t)n_tokens * nh <= INT32_MAX, LS_EINVAL, "prefix attention: too many query rows");
}

bool nh_fits(int n_heads) { return n_heads <= 65535; }   // a grid dimension

void run_prefix_attention(const ls_prefix_attention_args& p, cudaStream_t stream) {
  check_prefix_sizes(p.n_tokens, p.n_requests, p.n_heads, p.n_kv_heads, p.head_dim, p.prefix_len, p.max_new,
                     p.max_len);
  REQUIRE((p.cache_type == LS_BF16 || p.cache_type == LS_F16) &&
              (p.q_type == LS_F32 || p.q_type == p.cache_type),
          LS_EINVAL, "prefix attention: the cache must be bf16 or f16, and q of its type or fp32");
  REQUIRE(p.n_slots >= 1 && std::isfinite(p.scale) && p.scale > 0.f, LS_EINVAL,
          "prefix attention: n_slots must be positive and the scale positive and finite");
  const int shift = page_shift_of(p.page_size, "prefix attention");
  const int64_t qd = (int64_t)p.n_heads * p.head_dim, kd = (int64_t)p.n_kv_heads * p.head_dim;
  REQUIRE(p.q_stride >= qd && p.out_stride >= qd && p.slot_stride >= kd &&
              p.table_stride >= cdiv(p.max_len, p.page_size),
          LS_EINVAL, "prefix attention: a stride is smaller than its row");
  REQUIRE(p.slot_stride <= 1 << 29 && nh_fits(p.n_heads), LS_EINVAL, "prefix attention: slot_stride or n_heads too large");
  if (p.n_tokens == 0) return;
  REQUIRE(p.q && p.k_pool && p.v_pool && p.lens && p.token_start && p.out && p.workspace && p.status &&
              (p.prefix_table || p.prefix_len == 0) && (p.block_table || p.max_len == 0),
          LS_EINVAL, "prefix attention: null pointer argument");
  const long eb = type_bytes(p.q_type);
  REQUIRE(aligned16(p.q) && aligned16(p.k_pool) && aligned16(p.v_pool) && aligned16(p.out) &&
              p.q_stride * eb % 16 == 0 && p.out_stride * eb % 16 == 0 && p.slot_stride * 2 % 16 == 0,
          LS_EINVAL, "prefix attention: pointers and row strides must be 16-byte aligned");
  const PrefixPlan plan = make_plan(p.n_tokens, p.n_requests, p.n_heads, p.n_kv_heads, p.head_dim, p.prefix_len,
                                    p.max_new, p.max_len, p.q_type != LS_F32 ? 1 : p.cache_type == LS_BF16 ? 3 : 2, sm_count());
  REQUIRE((reinterpret_cast<uintptr_t>(p.workspace) & 255) == 0, LS_EINVAL,
          "prefix attention: workspace must be 256-byte aligned");
  REQUIRE(p.workspace_bytes >= plan.total, LS_EINVAL,
          "prefix attention: workspace smaller than ls_prefix_attention_workspace_bytes()");
  char* w = static_cast<char*>(p.workspace);
  PrefixAttnArgs a{};
  a.q = p.q;
  a.q_stride = (long)p.q_stride;
  a.k_pool = p.k_pool;
  a.v_pool = p.v_pool;
  a.slot_stride = (long)p.slot_stride;
  a.n_slots = p.n_slots;
  a.prefix_table = p.prefix_table;
  a.prefix_len = p.prefix_len;
  a.block_table = p.block_table;
  a.table_stride = (long)p.table_stride;
  a.lens = p.lens;
  a.token_start = p.token_start;
  a.n_requests = p.n_requests;
  a.n_tokens = p.n_tokens;
  a.max_new = p.max_new;
  a.max_len = p.max_len;
  a.page_shift = shift;
  a.nh = p.n_heads;
  a.nkv = p.n_kv_heads;
  const uint32_t group = (uint32_t)(p.n_heads / p.n_kv_heads);
  a.g_magic = (uint32_t)(((1ull << 32) + group - 1) / group);
  a.scale_log2 = (float)((double)p.scale * 1.4426950408889634);
  a.out = p.out;
  a.out_stride = (long)p.out_stride;
  a.part_o = reinterpret_cast<float*>(w);
  a.part_ml = reinterpret_cast<float2*>(w + plan.o_bytes);
  a.prefix_parts = plan.prefix_parts;
  a.prefix_chunk = plan.prefix_chunk;
  a.suffix_parts = plan.suffix_parts;
  a.suffix_chunk = plan.suffix_chunk;
  a.prefix_tiles = plan.prefix_tiles;
  a.suffix_tiles = plan.suffix_tiles;
  a.own = plan.own;
  a.direct = plan.own && plan.prefix_parts <= 1;
  a.status = p.status;
  if (p.q_type == LS_BF16) launch_prefix<bf16, bf16, 1>(a, p.head_dim, plan, stream);
  else if (p.q_type == LS_F16) launch_prefix<__half, __half, 1>(a, p.head_dim, plan, stream);
  else if (p.cache_type == LS_BF16) launch_prefix<float, bf16, 3>(a, p.head_dim, plan, stream);
  else launch_prefix<float, __half, 2>(a, p.head_dim, plan, stream);
}

}  // namespace

extern "C" {

int ls_check_status(int32_t* status, void* stream) {
  return guarded([&] {
    REQUIRE(status, LS_EINVAL, "status: null pointer argument");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    int32_t code = 0;
    CK(cudaMemcpyAsync(&code, status, sizeof(code), cudaMemcpyDeviceToHost, s));
    CK(cudaStreamSynchronize(s));
    if (code == kDevOk) return;
    CK(cudaMemsetAsync(status, 0, sizeof(code), s));
    CK(cudaStreamSynchronize(s));
    switch (code) {
      case kDevNoBlocks:
        throw EngineError(LS_ECAPACITY, "device reported: the free blocks do not cover the requests' growth");
      case kDevTooManyTokens:
        throw EngineError(LS_ECAPACITY, "device reported: more new tokens than max_tokens");
      case kDevBadLength:
        throw EngineError(LS_EDEVICE, "device reported: a length, count or token range is out of its bounds");
      case kDevBadIndex:
        throw EngineError(LS_EDEVICE, "device reported: a position, block or slot is out of range");
      case kDevTimeoutFull:
      case kDevTimeoutEmpty:
      case kDevTimeoutAcc:
        throw EngineError(LS_EDEVICE, "device reported: a wait inside a kernel timed out");
      default:
        throw EngineError(LS_EDEVICE, "device reported: unknown error " + std::to_string(code));
    }
  });
}

int ls_build_slots(const ls_slots_args* args, void* stream) {
  return guarded([&] {
    REQUIRE(args, LS_EINVAL, "slot maps: null argument struct");
    run_build_slots(*args, static_cast<cudaStream_t>(stream));
  });
}

int ls_qk_norm_rope(const ls_qk_norm_args* args, void* stream) {
  return guarded([&] {
    REQUIRE(args, LS_EINVAL, "qk norm: null argument struct");
    run_qk_norm_rope(*args, static_cast<cudaStream_t>(stream));
  });
}

size_t ls_prefix_attention_workspace_bytes(int n_tokens, int n_requests, int n_heads, int n_kv_heads, int head_dim,
                                           int prefix_len, int max_new, int max_len) {
  size_t bytes = 0;
  guarded([&] {
    check_prefix_sizes(n_tokens, n_requests, n_heads, n_kv_heads, head_dim, prefix_len, max_new, max_len);
    for (const int terms : {1, 2, 3})   // enough for any type of q
      bytes = std::max({(size_t)256, bytes, make_plan(n_tokens, n_requests, n_heads, n_kv_heads, head_dim, prefix_len,
                                                      max_new, max_len, terms, sm_count()).total});
  });
  return bytes;   // 0: refused, see ls_last_error(NULL)
}

int ls_prefix_attention(const ls_prefix_attention_args* args, void* stream) {
  return guarded([&] {
    REQUIRE(args, LS_EINVAL, "prefix attention: null argument struct");
    run_prefix_attention(*args, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"

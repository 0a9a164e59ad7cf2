// fd_evict_tokens: choose the tokens of a paged cache that stay, per sequence
// and KV head, and copy them in order to new pages.
#include <algorithm>
#include <cstring>

#include "../../include/flashdec_b200.h"
#include "fd_host.h"
#include "fd_ptx.cuh"

namespace fd {
namespace {

struct EvictParams {
  uint8_t* k;
  int64_t ks0, ks1, ks2, ks3;  // bytes
  uint8_t* v;
  int64_t vs0, vs1, vs2, vs3;
  float* scores;
  int64_t scs0, scs1, scs2;
  const void* bt;
  int64_t bts0, bts1;
  const void* sl;
  int64_t sls;
  const void* nbt;
  int64_t nbts0, nbts1;
  int* kept;
  void* new_lens;
  int bt64, sl64, nbt64, nl64;
  int hkv, bs_log2, num_blocks, max_blocks, max_new_blocks;
  int budget, sinks, recent;
  int vec;        // rows are 16-byte aligned and contiguous
  int score_vec;  // four scores of a page: one 16-byte load
  int* status;
  int device;  // host side only
};

__device__ __forceinline__ int length_of(const EvictParams& p, int b) {
  const int64_t cap = static_cast<int64_t>(p.max_blocks) << p.bs_log2;
  return static_cast<int>(min(max(load_index(p.sl, p.sl64, b * p.sls), int64_t(0)), cap));
}
// tokens kept: never more than the new table holds
__device__ __forceinline__ int kept_of(const EvictParams& p, int n) {
  const int64_t cap = static_cast<int64_t>(p.max_new_blocks) << p.bs_log2;
  return static_cast<int>(min(static_cast<int64_t>(min(n, p.budget)), cap));
}
// physical page, or -1 (status bit) when the table entry is not a page
__device__ __forceinline__ int64_t page_of(const EvictParams& p, const void* table, int is64, int64_t at) {
  const int64_t id = load_index(table, is64, at);
  if (id >= 0 && id < p.num_blocks) return id;
  atomicOr(p.status, FD_STATUS_BAD_BLOCK_ID);
  return -1;
}

// Order-preserving map of a score to 32 bits: greater score, greater key; -0
// as +0, every NaN above the numbers.
__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 0xffffffffu;
  if (x == 0.f) return 0x80000000u;
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kSelectThreads = 512;
constexpr int kMaxCluster = 8;
// Four digits: sign and exponent, then 8, 8 and 7 bits.  Wider ones (11, 11,
// 10) need a pass less but cost more: every CTA reads the counts of its whole
// cluster, and 48 clusters of 8 took 51 us on that traffic.
constexpr int kDigits = 4;
constexpr int kSelectWords = 512 + 256 + 256 + 128;  // their histograms
constexpr int kKeyMost = 48 * 1024;  // keys a CTA keeps
constexpr int kShort = 2048;  // keys of the second digit's bin that are listed for the last two

// Exclusive sum over the threads of a CTA (in thread order) and the total.
__device__ __forceinline__ int block_exclusive(int x, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int y = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int z = __shfl_up_sync(0xffffffffu, y, d);
    if (lane >= d) y += z;
  }
  if (lane == 31) warp_sums[warp] = y;
  __syncthreads();
  constexpr int kW = kSelectThreads / 32;
  int w = lane < kW ? warp_sums[lane] : 0;
#pragma unroll
  for (int d = 1; d < kW; d <<= 1) {
    const int z = __shfl_up_sync(0xffffffffu, w, d);
    if (lane >= d) w += z;
  }
  total = __shfl_sync(0xffffffffu, w, kW - 1);
  const int before = __shfl_sync(0xffffffffu, w, (warp + kW - 1) % kW);
  __syncthreads();  // warp_sums may be written again
  return (warp > 0 ? before : 0) + y - x;
}

// One cluster per (KV head, sequence), each CTA a run of its tokens, whose keys
// it keeps in shared memory when they fit (`key_cap`).  The threshold key is
// found digit by digit: each CTA counts its keys, the
// cluster's counts are added through distributed shared memory, and every CTA
// finds the same digit.  Then one pass in order keeps the protected tokens
// (sinks and recent), the keys above the threshold and the first of the keys
// equal to it.  The counts are whole numbers: no order of the atomics changes
// the result.  A chain bounds it: the keys' two look-ups, then a cluster
// barrier and a scan for every digit and one for the counts (16
// sequences of 4400 tokens and 8 heads, 4 MB: 17 us cold, 10 in a stream of calls).
__global__ void __launch_bounds__(kSelectThreads, 3)
    evict_select_kernel(const __grid_constant__ EvictParams p, int key_cap) {
  extern __shared__ __align__(16) int dyn[];
  int* hist = dyn;                                                   // by digit
  uint32_t* list = reinterpret_cast<uint32_t*>(dyn + kSelectWords);  // [kShort]
  uint32_t* keys = list + kShort;                                    // [key_cap]
  __shared__ int warp_sums[32];
  __shared__ int pick[2];    // digit, keys still to take among that digit's
  __shared__ int counts[2];  // this CTA's sure keeps and threshold keys
  __shared__ int listed;     // keys that matched the first two digits
  const int tid = threadIdx.x;
  const int ranks = gridDim.x;  // the cluster
  const int rank = blockIdx.x;
  const int h = blockIdx.y;
  const int b = blockIdx.z;
  for (int i = tid; i < kSelectWords; i += kSelectThreads) hist[i] = 0;
  if (tid == 0) listed = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const int n = length_of(p, b);
  const int m = kept_of(p, n);
  int* kept = p.kept + (static_cast<int64_t>(b) * p.hkv + h) * p.budget;
  if (h == 0 && rank == 0 && tid == 0) {
    if (p.nl64) {
      static_cast<int64_t*>(p.new_lens)[b] = m;
    } else {
      static_cast<int*>(p.new_lens)[b] = m;
    }
  }
  // (64 bits: a budget may be within a step of INT_MAX)
  for (int64_t i = m + rank * kSelectThreads + tid; i < p.budget; i += ranks * kSelectThreads) kept[i] = -1;
  if (n <= m) {  // the whole cluster
    for (int i = rank * kSelectThreads + tid; i < m; i += ranks * kSelectThreads) kept[i] = i;
    return;
  }
  const int sinks = min(p.sinks, m);
  const int recent = min(p.recent, m - sinks);
  const int mid0 = sinks, mid1 = n - recent;
  const int run = ((n + ranks - 1) / ranks + 7) & ~7;
  const int t0 = min(rank * run, n), t1 = min(t0 + run, n);
  const bool cached = run <= key_cap;
  const int mask = (1 << p.bs_log2) - 1;
  // keys of the four tokens from t (t % 4 == 0: they share a page)
  auto load4 = [&](int t, uint32_t(&k)[4]) {
    const int64_t id =
        page_of(p, p.bt, p.bt64, b * p.bts0 + static_cast<int64_t>(t >> p.bs_log2) * p.bts1);
    if (id < 0) {
      k[0] = k[1] = k[2] = k[3] = 0u;
      return;
    }
    const float* src = p.scores + id * p.scs0 + h * p.scs1 + (t & mask) * p.scs2;
    if (p.score_vec) {
      const float4 x = *reinterpret_cast<const float4*>(src);
      k[0] = score_key(x.x);
      k[1] = score_key(x.y);
      k[2] = score_key(x.z);
      k[3] = score_key(x.w);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = score_key(src[i * p.scs2]);
    }
  };
  // the keys of two places, all look-ups and loads out before the first use
  auto load8 = [&](int t, int t2, uint32_t(&k)[2][4]) {
    const int at[2] = {t, t2};
    int64_t id[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      id[u] = at[u] < t1 ? load_index(p.bt, p.bt64, b * p.bts0 + static_cast<int64_t>(at[u] >> p.bs_log2) * p.bts1) : 0;
    float4 x[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (at[u] < t1 && id[u] >= 0 && id[u] < p.num_blocks) {
        const float* src = p.scores + id[u] * p.scs0 + h * p.scs1 + (at[u] & mask) * p.scs2;
        x[u] = p.score_vec ? *reinterpret_cast<const float4*>(src)
                           : make_float4(src[0], src[p.scs2], src[2 * p.scs2], src[3 * p.scs2]);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bool good = id[u] >= 0 && id[u] < p.num_blocks;
      if (!good && at[u] < t1) atomicOr(p.status, FD_STATUS_BAD_BLOCK_ID);
      k[u][0] = good ? score_key(x[u].x) : 0u;
      k[u][1] = good ? score_key(x[u].y) : 0u;
      k[u][2] = good ? score_key(x[u].z) : 0u;
      k[u][3] = good ? score_key(x[u].w) : 0u;
    }
  };
  auto four = [&](int t, uint32_t(&k)[4]) {
    if (cached) {
      const uint4 x = *reinterpret_cast<const uint4*>(keys + (t - t0));
      k[0] = x.x;
      k[1] = x.y;
      k[2] = x.z;
      k[3] = x.w;
    } else {
      load4(t, k);
    }
  };
  auto all_sync = [&] {  // the cluster's threads
    if (ranks == 1) {
      __syncthreads();
    } else {
      cluster_arrive();
      cluster_wait();
    }
  };
  // ---- the (m - sinks - recent)-th greatest key of [mid0, mid1) ----
  int need = m - sinks - recent;
  const bool any_mid = need > 0;
  uint32_t prefix = 0;
#pragma unroll 1
  for (int t8 = t0 + 4 * tid; t8 < t1; t8 += 8 * kSelectThreads) {  // keys, and the first digit's counts
    uint32_t k[2][4];
    load8(t8, t8 + 4 * kSelectThreads, k);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = t8 + 4 * kSelectThreads * u;
      if (t >= t1) break;
      if (cached) *reinterpret_cast<uint4*>(keys + (t - t0)) = make_uint4(k[u][0], k[u][1], k[u][2], k[u][3]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t + i >= mid0 && t + i < mid1) atomicAdd(&hist[k[u][i] >> 23], 1);
    }
  }
  int above = 0;  // of this CTA's keys, those that a thread's bins put above the threshold
  if (any_mid) {
    int* mine = hist;
#pragma unroll 1
    for (int digit = 0; digit < kDigits; ++digit) {
      const int shift = digit == 0 ? 23 : (digit == 1 ? 15 : (digit == 2 ? 7 : 0));
      const int width = digit == 0 ? 9 : (digit == 3 ? 7 : 8);
      const int bins = 1 << width;
      const uint32_t found = prefix >> shift >> width;  // the bits above this digit
      if (digit == 1 || (digit > 1 && listed > kShort)) {
        for (int t = t0 + 4 * tid; t < t1; t += 4 * kSelectThreads) {
          uint32_t k[4];
          four(t, k);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = k[i] >> shift;
            if ((x >> width) == found && t + i >= mid0 && t + i < mid1) {
              atomicAdd(&mine[x & (bins - 1)], 1);
              if (digit == 1) {
                const int at = atomicAdd(&listed, 1);
                if (at < kShort) list[at] = k[i];
              }
            }
          }
        }
      } else if (digit > 1) {
        for (int i = tid; i < listed; i += kSelectThreads) {
          const uint32_t x = list[i] >> shift;
          if ((x >> width) == found) atomicAdd(&mine[x & (bins - 1)], 1);
        }
      }
      all_sync();
      // thread i: bin bins - 1 - i, counted over the cluster
      int c = 0;
      if (tid < bins) {
        int x[kMaxCluster];
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) {
          x[r] = 0;
          if (r < ranks)
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x[r]) : "r"(map_to_rank(smem_u32(mine + bins - 1 - tid), r)) : "memory");
        }
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) c += x[r];
      }
      static_assert(kSelectThreads == 512, "a bin a thread");
      int total;
      const int before = block_exclusive(c, warp_sums, total);
      if (before < need && need <= before + c) {  // one thread
        pick[0] = bins - 1 - tid;
        pick[1] = need - before;
      }
      __syncthreads();
      if (tid < bins - 1 - pick[0]) above += mine[bins - 1 - tid];
      prefix |= static_cast<uint32_t>(pick[0]) << shift;
      need = pick[1];
      if (digit == kDigits - 1 && tid == 0) counts[1] = mine[pick[0]];  // keys equal to the threshold
      mine += bins;
      __syncthreads();
    }
  } else if (tid == 0) {
    counts[1] = 0;
  }
  // ---- keep `need` of the keys equal to `prefix` and all greater ones ----
  auto flags = [&](int t, uint32_t& sure, uint32_t& tie) {
    uint32_t k[4] = {0u, 0u, 0u, 0u};
    if (t < t1) four(t, k);
    sure = tie = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = t + i < t1;
      const bool mid = t + i >= mid0 && t + i < mid1;
      sure |= (in && (!mid || (any_mid && k[i] > prefix)) ? 1u : 0u) << i;
      tie |= (in && mid && any_mid && k[i] == prefix ? 1u : 0u) << i;
    }
  };
  int total_above;
  block_exclusive(above, warp_sums, total_above);
  if (tid == 0)  // with the protected tokens of the run
    counts[0] = total_above + max(min(t1, mid0) - t0, 0) + max(t1 - max(t0, mid1), 0);
  all_sync();
  int base = 0, ties = 0;  // sure keeps and threshold keys before this CTA's run
  for (int r = 0; r < rank; ++r) {
    int x, y;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(map_to_rank(smem_u32(&counts[0]), r)) : "memory");
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(y) : "r"(map_to_rank(smem_u32(&counts[1]), r)) : "memory");
    base += x;
    ties += y;
  }
  cluster_arrive();  // nobody reads this CTA's shared memory after the matching wait
  for (int c = t0; c < t1; c += 4 * kSelectThreads) {
    uint32_t sure, tie;
    flags(c + 4 * tid, sure, tie);
    int total;  // both counts in one sum: at most 2048 of each
    const int before = block_exclusive(__popc(sure) | (__popc(tie) << 16), warp_sums, total);
    int s = base + (before & 0xffff), w = ties + (before >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool is_sure = (sure >> i) & 1u, is_tie = (tie >> i) & 1u;
      if (is_sure || (is_tie && w < need)) kept[s + min(w, need)] = c + 4 * tid + i;
      s += is_sure;
      w += is_tie;
    }
    base += total & 0xffff;
    ties += total >> 16;
  }
  cluster_wait();
}

constexpr int kCopyWarps = 4;
constexpr int kCopyThreads = kCopyWarps * 32;
constexpr int kCopyRows = 8;    // rows of a batch
constexpr int kCopyStages = 2;  // batches a warp has in flight

template <int D>
constexpr size_t copy_smem_bytes() {
  return static_cast<size_t>(kCopyWarps) * kCopyStages * kCopyRows * 2 * D * 2;
}

// A warp copies K, V and score of 8 kept tokens at a time: lane i < 8 looks up
// row i's pages, cp.async brings the rows to the warp's ring in shared memory
// and they go out from there a batch later.  537 MB in 88 us, 6.1 TB/s read and
// written together, 0.94 of a plain copy's rate; reads and writes are both
// random 256-byte rows.  Rows held in registers instead (20 warps an SM, 4 KB
// each, and nothing in flight while they store) took 119 us; more bytes in
// flight than this (a third stage) make it slower.
template <int D>
__global__ void __launch_bounds__(kCopyThreads) evict_copy_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ __align__(16) uint8_t ring_all[];
  constexpr int kBatch = kCopyRows * 2 * D * 2;  // bytes: per row K then V
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int h = blockIdx.x;  // the heads of a page run together
  const int b = blockIdx.z;
  const int mask = (1 << p.bs_log2) - 1;
  uint8_t* ring = ring_all + warp * (kCopyStages * kBatch);
  pdl_wait();
  pdl_launch_dependents();
  const int m = kept_of(p, length_of(p, b));
  const int* kept = p.kept + (static_cast<int64_t>(b) * p.hkv + h) * p.budget;
  const int step = gridDim.y * kCopyWarps * kCopyRows;
  // lane i < 8: row i0 + i; offsets of its slot (bytes from the caches), -1: no row
  struct Rows {
    int64_t src, dst;  // pages
    int t;
    float score;
  };
  auto look = [&](int i0) -> Rows {
    Rows r = {-1, -1, 0, 0.f};
    const int i = i0 + lane;
    if (lane < kCopyRows && i < m) {
      r.dst = page_of(p, p.nbt, p.nbt64, b * p.nbts0 + static_cast<int64_t>(i >> p.bs_log2) * p.nbts1);
      r.t = kept[i];
      r.src = page_of(p, p.bt, p.bt64, b * p.bts0 + static_cast<int64_t>(r.t >> p.bs_log2) * p.bts1);
      if (r.src < 0 || r.dst < 0) {
        r.src = r.dst = -1;
      } else {
        r.score = p.scores[r.src * p.scs0 + h * p.scs1 + (r.t & mask) * p.scs2];
      }
    }
    return r;
  };
  constexpr int kChunks = D / 8;        // 16-byte chunks of a row
  constexpr int kSide = 16 / kChunks;   // rows a half warp moves at once: lanes 0-15 K, 16-31 V
  const bool is_v = lane >= 16;
  const int c = lane & (kChunks - 1);
  const int sub = (lane & 15) / kChunks;
  uint8_t* const base = (is_v ? p.v + h * p.vs1 : p.k + h * p.ks1) + c * 16;
  const int64_t s0 = is_v ? p.vs0 : p.ks0, s2 = is_v ? p.vs2 : p.ks2;
  uint8_t* const mine = ring + (is_v ? D * 2 : 0) + sub * (4 * D) + c * 16;  // + stage, + row
  auto load = [&](const Rows& r, int stage) {
    if (p.vec) {
#pragma unroll
      for (int j = 0; j < kCopyRows / kSide; ++j) {
        const int64_t from = __shfl_sync(0xffffffffu, r.src, j * kSide + sub);
        const int tok = __shfl_sync(0xffffffffu, r.t, j * kSide + sub);
        if (from >= 0)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                           smem_u32(mine + stage * kBatch + j * (kSide * 4 * D))),
                       "l"(base + from * s0 + (tok & mask) * s2)
                       : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int first = (blockIdx.y * kCopyWarps + warp) * kCopyRows;
  Rows rows[kCopyStages];  // batches in flight, and the next one's look-up
#pragma unroll
  for (int i = 0; i < kCopyStages; ++i) rows[i] = look(first + i * step);
#pragma unroll
  for (int i = 0; i < kCopyStages - 1; ++i) load(rows[i], i);
  int stage = 0;
  for (int i0 = first; i0 < m; i0 += step) {
    const Rows cur = rows[0];
    int ahead = stage + kCopyStages - 1;
    load(rows[kCopyStages - 1], ahead >= kCopyStages ? ahead - kCopyStages : ahead);
#pragma unroll
    for (int i = 0; i + 1 < kCopyStages; ++i) rows[i] = rows[i + 1];
    rows[kCopyStages - 1] = look(i0 + kCopyStages * step);
    if (p.vec) {
      // each lane reads back what it copied itself
      asm volatile("cp.async.wait_group %0;" ::"n"(kCopyStages - 1) : "memory");
#pragma unroll
      for (int j = 0; j < kCopyRows / kSide; ++j) {
        const int r = j * kSide + sub;
        const int64_t to = __shfl_sync(0xffffffffu, cur.dst, r);
        if (to >= 0)
          *reinterpret_cast<uint4*>(base + to * s0 + ((i0 + r) & mask) * s2) =
              *reinterpret_cast<const uint4*>(mine + stage * kBatch + j * (kSide * 4 * D));
      }
    } else {
      for (int r = 0; r < kCopyRows; ++r) {
        const int64_t from = __shfl_sync(0xffffffffu, cur.src, r), to = __shfl_sync(0xffffffffu, cur.dst, r);
        const int tok = __shfl_sync(0xffffffffu, cur.t, r);
        if (to < 0) continue;
        const uint8_t* k0 = p.k + from * p.ks0 + h * p.ks1 + (tok & mask) * p.ks2;
        uint8_t* k1 = p.k + to * p.ks0 + h * p.ks1 + ((i0 + r) & mask) * p.ks2;
        const uint8_t* v0 = p.v + from * p.vs0 + h * p.vs1 + (tok & mask) * p.vs2;
        uint8_t* v1 = p.v + to * p.vs0 + h * p.vs1 + ((i0 + r) & mask) * p.vs2;
        for (int d = lane; d < D; d += 32) {
          *reinterpret_cast<uint16_t*>(k1 + d * p.ks3) = *reinterpret_cast<const uint16_t*>(k0 + d * p.ks3);
          *reinterpret_cast<uint16_t*>(v1 + d * p.vs3) = *reinterpret_cast<const uint16_t*>(v0 + d * p.vs3);
        }
      }
    }
    if (cur.dst >= 0) p.scores[cur.dst * p.scs0 + h * p.scs1 + ((i0 + lane) & mask) * p.scs2] = cur.score;
    if (++stage == kCopyStages) stage = 0;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <int D>
int copy(const EvictParams& p, int num_seqs, int sms, cudaStream_t stream) {
  constexpr size_t smem = copy_smem_bytes<D>();
  // Six CTAs fit an SM (their registers); four times as many even out the
  // SMs (537 MB: 123 us with a third stage and four CTAs an SM, 114 with two
  // and six, 109 with 24, selection included)
  constexpr int kPerSm = 24;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(done, reinterpret_cast<const void*>(evict_copy_kernel<D>), smem, p.device);
  if (e != cudaSuccess) return cuda_status(e);
  const int64_t most = std::min<int64_t>(
      std::min<int64_t>(p.budget, static_cast<int64_t>(p.max_new_blocks) << p.bs_log2),
      static_cast<int64_t>(p.max_blocks) << p.bs_log2);
  const int per = kCopyWarps * kCopyRows;
  const int64_t units = static_cast<int64_t>(p.hkv) * num_seqs;
  const int64_t blocks = std::min((most + per - 1) / per, std::max<int64_t>(kPerSm * sms / units, 1));
  return cuda_status(launch_pdl(evict_copy_kernel<D>, dim3(p.hkv, static_cast<unsigned>(blocks), num_seqs),
                                dim3(kCopyThreads), smem, stream, p));
}

// Tokens a CTA of the selection holds: about 4096, and no more than a cluster
// of 8 has to.
int select(const EvictParams& p, int num_seqs, cudaStream_t stream) {
  const int64_t cap = static_cast<int64_t>(p.max_blocks) << p.bs_log2;
  int ranks = 1;
  while (ranks < kMaxCluster && cap > 4096 * ranks) ranks *= 2;
  const int64_t run = ((cap + ranks - 1) / ranks + 7) & ~int64_t(7);
  // past this the keys are read again for every digit
  const int key_cap = run <= kKeyMost ? static_cast<int>(run) : 0;
  const size_t smem = sizeof(int) * (kSelectWords + kShort + static_cast<size_t>(key_cap));
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(done, reinterpret_cast<const void*>(evict_select_kernel),
                                   sizeof(int) * (kSelectWords + kShort + kKeyMost), p.device);
  if (e != cudaSuccess) return cuda_status(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks, p.hkv, num_seqs);
  cfg.blockDim = dim3(kSelectThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, evict_select_kernel, p, key_cap));
}

}  // namespace
}  // namespace fd

extern "C" int fd_evict_tokens(const fd_evict_tokens_args* a, void* cuda_stream) {
  using namespace fd;
  if (!a || a->struct_size != static_cast<int32_t>(sizeof(fd_evict_tokens_args)))
    return FD_ERR_INVALID_ARGUMENT;
  if (a->elem_bytes != 2) return FD_ERR_UNSUPPORTED;
  if (a->head_dim != 64 && a->head_dim != 128) return FD_ERR_UNSUPPORTED;
  if (a->block_size != 8 && a->block_size != 16 && a->block_size != 32) return FD_ERR_UNSUPPORTED;
  if (a->num_seqs < 0 || a->num_kv_heads <= 0 || a->num_blocks <= 0 || a->max_blocks_per_seq <= 0 ||
      a->max_new_blocks_per_seq <= 0 || a->budget < 1 || a->sinks < 0 || a->recent < 0 ||
      static_cast<int64_t>(a->sinks) + a->recent > a->budget)
    return FD_ERR_INVALID_ARGUMENT;
  if (a->num_seqs > 65535 || a->num_kv_heads > 65535 ||
      static_cast<int64_t>(a->max_blocks_per_seq) * a->block_size > 0x3fffffff ||
      static_cast<int64_t>(a->max_new_blocks_per_seq) * a->block_size > 0x3fffffff)
    return FD_ERR_UNSUPPORTED;
  if (a->num_seqs == 0) return FD_OK;
  if (!a->k_cache || !a->v_cache || !a->scores || !a->block_tables || !a->seq_lens ||
      !a->new_block_tables || !a->kept || !a->new_seq_lens)
    return FD_ERR_INVALID_ARGUMENT;
  const DeviceInfo* dev = current_device_info();
  int* status = device_status_ptr();
  if (!dev || !status) return FD_ERR_CUDA;

  EvictParams p;
  std::memset(&p, 0, sizeof(p));
  p.k = static_cast<uint8_t*>(a->k_cache);
  p.ks0 = a->k_stride[0] * 2; p.ks1 = a->k_stride[1] * 2; p.ks2 = a->k_stride[2] * 2; p.ks3 = a->k_stride[3] * 2;
  p.v = static_cast<uint8_t*>(a->v_cache);
  p.vs0 = a->v_stride[0] * 2; p.vs1 = a->v_stride[1] * 2; p.vs2 = a->v_stride[2] * 2; p.vs3 = a->v_stride[3] * 2;
  p.scores = a->scores;
  p.scs0 = a->scores_stride[0]; p.scs1 = a->scores_stride[1]; p.scs2 = a->scores_stride[2];
  p.bt = a->block_tables;
  p.bts0 = a->block_tables_stride[0]; p.bts1 = a->block_tables_stride[1];
  p.bt64 = a->block_tables_index == FD_INDEX_I64;
  p.sl = a->seq_lens;
  p.sls = a->seq_lens_stride;
  p.sl64 = a->seq_lens_index == FD_INDEX_I64;
  p.nbt = a->new_block_tables;
  p.nbts0 = a->new_block_tables_stride[0]; p.nbts1 = a->new_block_tables_stride[1];
  p.nbt64 = a->new_block_tables_index == FD_INDEX_I64;
  p.kept = a->kept;
  p.new_lens = a->new_seq_lens;
  p.nl64 = a->new_seq_lens_index == FD_INDEX_I64;
  p.hkv = a->num_kv_heads;
  p.bs_log2 = a->block_size == 8 ? 3 : (a->block_size == 16 ? 4 : 5);
  p.num_blocks = a->num_blocks;
  p.max_blocks = a->max_blocks_per_seq;
  p.max_new_blocks = a->max_new_blocks_per_seq;
  p.budget = a->budget;
  p.sinks = a->sinks;
  p.recent = a->recent;
  auto aligned = [](const void* base, const int64_t* st) {
    return reinterpret_cast<uintptr_t>(base) % 16 == 0 && st[0] % 8 == 0 && st[1] % 8 == 0 &&
           st[2] % 8 == 0 && st[3] == 1;
  };
  p.vec = aligned(a->k_cache, a->k_stride) && aligned(a->v_cache, a->v_stride);
  p.status = status;
  p.device = dev->device;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  p.score_vec = reinterpret_cast<uintptr_t>(a->scores) % 16 == 0 && a->scores_stride[0] % 4 == 0 &&
                a->scores_stride[1] % 4 == 0 && a->scores_stride[2] == 1;
  int rc = select(p, a->num_seqs, stream);
  if (rc != FD_OK) return rc;
  return a->head_dim == 128 ? copy<128>(p, a->num_seqs, dev->num_sms, stream)
                            : copy<64>(p, a->num_seqs, dev->num_sms, stream);
}

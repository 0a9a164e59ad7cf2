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
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr int kSelectWords = 3 * kBins;  // histograms of the three digits

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
// found digit by digit (11, 11 and 10 bits): each CTA counts its keys, the
// cluster's counts are added through distributed shared memory, and every CTA
// finds the same digit.  Then one pass in order keeps the protected tokens
// (sinks and recent), the keys above the threshold and the first of the keys
// equal to it.  The counts are whole numbers: no order of the atomics changes
// the result.
__global__ void __launch_bounds__(kSelectThreads, 3)
    evict_select_kernel(const __grid_constant__ EvictParams p, int key_cap) {
  extern __shared__ __align__(16) int dyn[];
  int* hist = dyn;                                                // [3][kBins]
  uint32_t* keys = reinterpret_cast<uint32_t*>(dyn + kSelectWords);  // [key_cap]
  __shared__ int warp_sums[32];
  __shared__ int pick[2];    // digit, keys still to take among that digit's
  __shared__ int counts[2];  // this CTA's sure keeps and threshold keys
  const int tid = threadIdx.x;
  const int ranks = gridDim.x;  // the cluster
  const int rank = blockIdx.x;
  const int h = blockIdx.y;
  const int b = blockIdx.z;
  for (int i = tid; i < kSelectWords; i += kSelectThreads) hist[i] = 0;
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
  for (int i = m + rank * kSelectThreads + tid; i < p.budget; i += ranks * kSelectThreads) kept[i] = -1;
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
  if (cached) {
    for (int t = t0 + 4 * tid; t < t1; t += 4 * kSelectThreads) {
      uint32_t k[4];
      load4(t, k);
      *reinterpret_cast<uint4*>(keys + (t - t0)) = make_uint4(k[0], k[1], k[2], k[3]);
    }
  }
  __syncthreads();
  // ---- the (m - sinks - recent)-th greatest key of [mid0, mid1) ----
  int need = m - sinks - recent;
  const bool any_mid = need > 0;
  uint32_t prefix = 0;
  if (any_mid) {
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 21 : (digit == 1 ? 10 : 0);
      const int above = digit == 0 ? 32 : (digit == 1 ? 21 : 10);  // bits found so far lie above
      int* mine = hist + digit * kBins;
      for (int t = t0 + 4 * tid; t < t1; t += 4 * kSelectThreads) {
        uint32_t k[4];
        four(t, k);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t + i >= mid0 && t + i < mid1 && (above == 32 || (k[i] >> above) == (prefix >> above)))
            atomicAdd(&mine[(k[i] >> shift) & (above - shift == 11 ? 2047 : 1023)], 1);
      }
      cluster_arrive();
      cluster_wait();
      // bins from the top: thread i has bins top, top - 1, top - 2 and top - 3
      const int top = kBins - 1 - 4 * tid;
      static_assert(4 * kSelectThreads == kBins, "four bins a thread");
      int c[4] = {0, 0, 0, 0};
      for (int r = 0; r < ranks; ++r) {
        const uint32_t at = map_to_rank(smem_u32(mine + top - 3), r);
        int x[4];
        asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(x[3]), "=r"(x[2]), "=r"(x[1]), "=r"(x[0]) : "r"(at) : "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] += x[i];
      }
      int total;
      int before = block_exclusive(c[0] + c[1] + c[2] + c[3], warp_sums, total);
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // one bin of one thread holds the key
        if (before < need && need <= before + c[i]) {
          pick[0] = top - i;
          pick[1] = need - before;
        }
        before += c[i];
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(pick[0]) << shift;
      need = pick[1];
      __syncthreads();
    }
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
  int sure_n = 0, tie_n = 0;
  for (int t = t0 + 4 * tid; t < t1; t += 4 * kSelectThreads) {
    uint32_t sure, tie;
    flags(t, sure, tie);
    sure_n += __popc(sure);
    tie_n += __popc(tie);
  }
  int total_sure, total_tie;
  block_exclusive(sure_n, warp_sums, total_sure);
  block_exclusive(tie_n, warp_sums, total_tie);
  if (tid == 0) {
    counts[0] = total_sure;
    counts[1] = total_tie;
  }
  cluster_arrive();
  cluster_wait();
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

constexpr int kCopyThreads = 256;
constexpr int kCopyRows = 8;  // rows a warp has in flight

// A warp copies K, V and score of 8 kept tokens at a time: lane i < 8 looks up
// row i's pages, all rows' loads go out before the first store, and the next
// eight are looked up meanwhile.  A few CTAs an SM that loop: with one batch a
// warp and a CTA for every 64 rows the SMs stood at 23 % of their warps, waiting
// for new CTAs (131 us for 537 MB).
template <int D>
__global__ void __launch_bounds__(kCopyThreads) evict_copy_kernel(const __grid_constant__ EvictParams p) {
  const int lane = threadIdx.x & 31;
  const int h = blockIdx.x;  // the heads of a page run together
  const int b = blockIdx.z;
  const int mask = (1 << p.bs_log2) - 1;
  pdl_wait();
  pdl_launch_dependents();
  const int m = kept_of(p, length_of(p, b));
  const int* kept = p.kept + (static_cast<int64_t>(b) * p.hkv + h) * p.budget;
  const int step = gridDim.y * (kCopyThreads / 32) * kCopyRows;
  struct Rows {  // lane i < 8: row i0 + i
    int64_t src, dst;
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
  int i0 = (blockIdx.y * (kCopyThreads / 32) + (threadIdx.x >> 5)) * kCopyRows;
  Rows next = look(i0);
  for (; i0 < m; i0 += step) {
    const Rows cur = next;
    const int64_t src = cur.src, dst = cur.dst;
    const int t = cur.t;
    if (p.vec) {
      constexpr int kChunks = D / 8;      // 16-byte chunks of a row
      constexpr int kSide = 16 / kChunks; // rows a half warp moves at once: lanes 0-15 K, 16-31 V
      const bool is_v = lane >= 16;
      const int c = lane & (kChunks - 1);
      const int sub = (lane & 15) / kChunks;
      uint8_t* base = is_v ? p.v : p.k;
      const int64_t s0 = is_v ? p.vs0 : p.ks0, s1 = is_v ? p.vs1 : p.ks1, s2 = is_v ? p.vs2 : p.ks2;
      uint4 x[kCopyRows / kSide];
#pragma unroll
      for (int j = 0; j < kCopyRows / kSide; ++j) {
        const int r = j * kSide + sub;
        const int64_t from = __shfl_sync(0xffffffffu, src, r);
        const int tok = __shfl_sync(0xffffffffu, t, r);
        if (from >= 0) x[j] = __ldcs(reinterpret_cast<const uint4*>(base + from * s0 + h * s1 + (tok & mask) * s2 + c * 16));
      }
      next = look(i0 + step);
#pragma unroll
      for (int j = 0; j < kCopyRows / kSide; ++j) {
        const int r = j * kSide + sub;
        const int64_t to = __shfl_sync(0xffffffffu, dst, r);
        if (to >= 0) *reinterpret_cast<uint4*>(base + to * s0 + h * s1 + ((i0 + r) & mask) * s2 + c * 16) = x[j];
      }
    } else {
      next = look(i0 + step);
      for (int r = 0; r < kCopyRows; ++r) {
        const int64_t from = __shfl_sync(0xffffffffu, src, r), to = __shfl_sync(0xffffffffu, dst, r);
        const int tok = __shfl_sync(0xffffffffu, t, r);
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
    if (dst >= 0) p.scores[dst * p.scs0 + h * p.scs1 + ((i0 + lane) & mask) * p.scs2] = cur.score;
  }
}

// Tokens a CTA of the selection holds: about 4096, and no more than a cluster
// of 8 has to.
int select(const EvictParams& p, int num_seqs, cudaStream_t stream) {
  const int64_t cap = static_cast<int64_t>(p.max_blocks) << p.bs_log2;
  int ranks = 1;
  while (ranks < kMaxCluster && cap > 4096 * ranks) ranks *= 2;
  const int64_t run = ((cap + ranks - 1) / ranks + 7) & ~int64_t(7);
  // past this the keys are read again for every digit
  const int key_cap = run <= 48 * 1024 ? static_cast<int>(run) : 0;
  const size_t smem = sizeof(int) * (kSelectWords + static_cast<size_t>(key_cap));
  cudaError_t e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(smem));
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
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  p.score_vec = reinterpret_cast<uintptr_t>(a->scores) % 16 == 0 && a->scores_stride[0] % 4 == 0 &&
                a->scores_stride[1] % 4 == 0 && a->scores_stride[2] == 1;
  int rc = select(p, a->num_seqs, stream);
  if (rc != FD_OK) return rc;
  const int64_t most = std::min<int64_t>(
      std::min<int64_t>(p.budget, static_cast<int64_t>(p.max_new_blocks) << p.bs_log2),
      static_cast<int64_t>(p.max_blocks) << p.bs_log2);
  const int per = kCopyThreads / 32 * kCopyRows;
  const int64_t fill = (4 * dev->num_sms + p.hkv * a->num_seqs - 1) / (p.hkv * a->num_seqs);  // four CTAs an SM
  const int blocks = static_cast<int>(std::min((most + per - 1) / per, fill));
  const dim3 grid(p.hkv, std::max(blocks, 1), a->num_seqs);
  return cuda_status(a->head_dim == 128
                         ? launch_pdl(evict_copy_kernel<128>, grid, dim3(kCopyThreads), 0, stream, p)
                         : launch_pdl(evict_copy_kernel<64>, grid, dim3(kCopyThreads), 0, stream, p));
}

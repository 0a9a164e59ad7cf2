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
  int vec;  // rows are 16-byte aligned and contiguous
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

constexpr int kSelectThreads = 1024;

// One CTA per (KV head, sequence).  The threshold key is found digit by digit
// (four 8-bit histograms over the tokens that are neither sinks nor recent);
// then one pass in order keeps the protected tokens, the keys above the
// threshold and the first of the keys equal to it.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ EvictParams p) {
  __shared__ int hist[256];
  __shared__ int pick[2];  // digit, keys still to take among that digit's
  __shared__ int wsum[2][32];
  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int h = blockIdx.x;
  const int b = blockIdx.y;
  pdl_wait();
  pdl_launch_dependents();
  const int n = length_of(p, b);
  const int m = kept_of(p, n);
  int* kept = p.kept + (static_cast<int64_t>(b) * p.hkv + h) * p.budget;
  if (h == 0 && tid == 0) {
    if (p.nl64) {
      static_cast<int64_t*>(p.new_lens)[b] = m;
    } else {
      static_cast<int*>(p.new_lens)[b] = m;
    }
  }
  for (int i = m + tid; i < p.budget; i += kSelectThreads) kept[i] = -1;
  if (n <= m) {
    for (int i = tid; i < m; i += kSelectThreads) kept[i] = i;
    return;
  }
  const int sinks = min(p.sinks, m);
  const int recent = min(p.recent, m - sinks);
  const int mid0 = sinks, mid1 = n - recent;
  auto key_of = [&](int t) -> uint32_t {
    const int64_t id =
        page_of(p, p.bt, p.bt64, b * p.bts0 + static_cast<int64_t>(t >> p.bs_log2) * p.bts1);
    if (id < 0) return 0u;
    return score_key(p.scores[id * p.scs0 + h * p.scs1 + (t & ((1 << p.bs_log2) - 1)) * p.scs2]);
  };
  // the (m - sinks - recent)-th greatest key of [mid0, mid1)
  int need = m - sinks - recent;
  uint32_t prefix = 0;
  for (int shift = 24; need > 0 && shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int t = mid0 + tid; t < mid1; t += kSelectThreads) {
      const uint32_t k = key_of(t);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int left = need, d = 255;
      while (d > 0 && hist[d] < left) left -= hist[d--];
      pick[0] = d;
      pick[1] = left;
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(pick[0]) << shift;
    need = pick[1];
    __syncthreads();
  }
  // `need` keys equal to `prefix` are kept, all greater ones
  const bool any_mid = m - sinks - recent > 0;
  int base = 0, ties = 0;  // kept and equal keys before this chunk
  for (int c = 0; c < n; c += kSelectThreads) {
    const int t = c + tid;
    const bool mid = t >= mid0 && t < mid1;
    const uint32_t k = mid && any_mid ? key_of(t) : 0u;
    const bool sure = t < n && (!mid || (any_mid && k > prefix));
    const bool tie = mid && any_mid && k == prefix;
    const uint32_t below = (1u << lane) - 1u;
    const uint32_t bs = __ballot_sync(0xffffffffu, sure), bt = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) {
      wsum[0][warp] = __popc(bs);
      wsum[1][warp] = __popc(bt);
    }
    __syncthreads();
    int ws = 0, wt = 0, all_s = 0, all_t = 0;
    for (int w = 0; w < kSelectThreads / 32; ++w) {
      if (w < warp) {
        ws += wsum[0][w];
        wt += wsum[1][w];
      }
      all_s += wsum[0][w];
      all_t += wsum[1][w];
    }
    const int tie_rank = ties + wt + __popc(bt & below);
    const int ties_before = min(tie_rank, need) - min(ties, need);  // kept ties before t in this chunk
    const int at = base + ws + __popc(bs & below) + ties_before;
    if (sure || (tie && tie_rank < need)) {
      if (at < m) kept[at] = t;
    }
    base += all_s + min(ties + all_t, need) - min(ties, need);
    ties += all_t;
    __syncthreads();
  }
}

constexpr int kCopyThreads = 256;

// One warp per kept row: K, V and the score go to the new page.
template <int D>
__global__ void __launch_bounds__(kCopyThreads) evict_copy_kernel(const __grid_constant__ EvictParams p) {
  const int lane = threadIdx.x & 31;
  const int h = blockIdx.y;
  const int b = blockIdx.z;
  pdl_wait();
  pdl_launch_dependents();
  const int m = kept_of(p, length_of(p, b));
  const int mask = (1 << p.bs_log2) - 1;
  const int* kept = p.kept + (static_cast<int64_t>(b) * p.hkv + h) * p.budget;
  for (int i = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5); i < m;
       i += gridDim.x * (kCopyThreads / 32)) {
    const int t = kept[i];
    const int64_t src =
        page_of(p, p.bt, p.bt64, b * p.bts0 + static_cast<int64_t>(t >> p.bs_log2) * p.bts1);
    const int64_t dst =
        page_of(p, p.nbt, p.nbt64, b * p.nbts0 + static_cast<int64_t>(i >> p.bs_log2) * p.nbts1);
    if (src < 0 || dst < 0) continue;
    const uint8_t* k0 = p.k + src * p.ks0 + h * p.ks1 + (t & mask) * p.ks2;
    uint8_t* k1 = p.k + dst * p.ks0 + h * p.ks1 + (i & mask) * p.ks2;
    const uint8_t* v0 = p.v + src * p.vs0 + h * p.vs1 + (t & mask) * p.vs2;
    uint8_t* v1 = p.v + dst * p.vs0 + h * p.vs1 + (i & mask) * p.vs2;
    if (p.vec) {
      constexpr int kChunks = D / 8;  // 16-byte chunks of a row
      if (lane < kChunks) {
        *reinterpret_cast<uint4*>(k1 + lane * 16) = *reinterpret_cast<const uint4*>(k0 + lane * 16);
      } else if (lane - kChunks < kChunks) {
        *reinterpret_cast<uint4*>(v1 + (lane - kChunks) * 16) =
            *reinterpret_cast<const uint4*>(v0 + (lane - kChunks) * 16);
      }
    } else {
      for (int d = lane; d < D; d += 32) {
        *reinterpret_cast<uint16_t*>(k1 + d * p.ks3) = *reinterpret_cast<const uint16_t*>(k0 + d * p.ks3);
        *reinterpret_cast<uint16_t*>(v1 + d * p.vs3) = *reinterpret_cast<const uint16_t*>(v0 + d * p.vs3);
      }
    }
    if (lane == 0)
      p.scores[dst * p.scs0 + h * p.scs1 + (i & mask) * p.scs2] =
          p.scores[src * p.scs0 + h * p.scs1 + (t & mask) * p.scs2];
  }
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
  int rc = cuda_status(launch_pdl(evict_select_kernel, dim3(p.hkv, a->num_seqs), dim3(kSelectThreads), 0,
                                  stream, p));
  if (rc != FD_OK) return rc;
  const int64_t most = std::min<int64_t>(
      std::min<int64_t>(p.budget, static_cast<int64_t>(p.max_new_blocks) << p.bs_log2),
      static_cast<int64_t>(p.max_blocks) << p.bs_log2);
  const int per = kCopyThreads / 32;
  const int blocks = static_cast<int>(std::min<int64_t>((most + per - 1) / per, 1 << 20));
  const dim3 grid(std::max(blocks, 1), p.hkv, a->num_seqs);
  return cuda_status(a->head_dim == 128
                         ? launch_pdl(evict_copy_kernel<128>, grid, dim3(kCopyThreads), 0, stream, p)
                         : launch_pdl(evict_copy_kernel<64>, grid, dim3(kCopyThreads), 0, stream, p));
}

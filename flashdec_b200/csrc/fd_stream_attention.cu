// Attention over a bounded cache for few queries per sequence: one decoded
// token, or a handful of drafts (fd_window_attention), and one token with the
// attention weights kept (fd_scored_decode).
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "../../include/flashdec_b200.h"
#include "fd_host.h"
#include "fd_ptx.cuh"
#include "fd_stream.cuh"
#include "fd_stream.h"

namespace fd {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTok = 16;    // tokens per warp tile
constexpr int kStages = 3;  // tiles in flight per warp
constexpr int kMaxSplits = 64;

template <int D>
constexpr size_t ring_bytes() {
  return static_cast<size_t>(kWarps) * kStages * 2 * kTok * D * 2;
}
template <int D, int kM>
constexpr size_t split_smem_bytes() {
  // ring (later the merge buffer: kWarps x rows x (D + 2) floats) and q
  return ring_bytes<D>() + static_cast<size_t>(kM) * 16 * D * 2;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Byte offset of 16-byte chunk `c` of row `r` in a [rows][D] 16-bit tile: the
// chunk index is XORed with r % 8, so the 8 rows of an ldmatrix start on
// different banks.
template <int D>
__device__ __forceinline__ uint32_t tile_chunk(int r, int c) {
  return r * (D * 2) + ((c ^ (r & 7)) << 4);
}

// ---------------------------------------------------------------------------
// One CTA: rows [16 kM rb, +16 kM) of a (sequence, KV head), split `blockIdx.x`
// of the pages they see.  Row r is head r % group of query r / group, so K and
// V are read once for the whole group.  Tile i of 16 tokens goes to warp i % 4;
// each warp keeps three tiles in flight with cp.async and its own running
// max and sum (base 2), and the four merge at the end.
// ---------------------------------------------------------------------------
template <typename T, int D, int kM>
__global__ void __launch_bounds__(kThreads, 2) stream_split_kernel(const __grid_constant__ StreamParams p) {
  constexpr int kRows = 16 * kM;
  constexpr int kChunks = D / 8;
  constexpr uint32_t kTileBytes = kTok * D * 2;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* qsm = smem + ring_bytes<D>();
  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int g8 = lane >> 2;
  const int t4 = lane & 3;
  const int mi = lane >> 3;
  const int r8 = lane & 7;
  const int split = blockIdx.x;
  const int h = blockIdx.y / p.row_blocks;
  const int b = blockIdx.z;

  pdl_wait();
  pdl_launch_dependents();
  const StreamSeq s = sequence_of(p, b);
  const int rows_all = s.qlen * p.group;
  uint8_t* const kring = smem + warp * (kStages * 2 * kTileBytes);

  for (int rb = blockIdx.y - h * p.row_blocks; rb * kRows < rows_all; rb += p.row_blocks) {
    const int row0 = rb * kRows;
    const int rows = min(kRows, rows_all - row0);
    const StreamRange rg(s, row0, row0 + rows, p.group, p.window, p.sinks, p.bs_log2);
    const int tiles = ((rg.pages << p.bs_log2) + kTok - 1) / kTok;
    const int t0 = static_cast<int>(static_cast<int64_t>(split) * tiles / p.splits);
    const int t1 = static_cast<int>(static_cast<int64_t>(split + 1) * tiles / p.splits);

    // lanes 0 and 1 hold the (at most two) pages of a tile: {block, position of its first token}
    auto fetch = [&](int t, int& blk, int& pos) {
      blk = -1;
      pos = 0;
      const int i = p.bs_log2 >= 4 ? (t * kTok) >> p.bs_log2 : 2 * t + lane;
      if (lane < 2 && t < t1 && i < rg.pages) {
        const int page = rg.page(i);
        pos = p.bs_log2 >= 4 ? (page << p.bs_log2) + ((t * kTok) & ((1 << p.bs_log2) - 1))
                             : page << p.bs_log2;
        const int64_t id = load_index(p.bt, p.bt64, b * p.bts0 + page * p.bts1);
        if (id >= 0 && id < p.num_blocks) {
          blk = static_cast<int>(id);
        } else if (pos <= rg.pos1 && (pos + (1 << min(p.bs_log2, 4)) > rg.lo || pos < rg.sink_end)) {
          atomicOr(p.status, FD_STATUS_BAD_BLOCK_ID);
        }
      }
    };
    // position of tile token `tok`, or -1 when no row sees it or its page is bad
    auto token_pos = [&](int tok, int blk0, int blk1, int pos0, int pos1) -> int {
      const bool second = p.bs_log2 == 3 && tok >= 8;
      const int pos = second ? pos1 + tok - 8 : pos0 + tok;
      const bool seen = pos <= rg.pos1 && (pos >= rg.lo || pos < rg.sink_end);
      return (second ? blk1 : blk0) >= 0 && seen ? pos : -1;
    };
    auto issue = [&](int t, int blk, int pos) {
      const int blk0 = __shfl_sync(0xffffffffu, blk, 0), blk1 = __shfl_sync(0xffffffffu, blk, 1);
      const int pp0 = __shfl_sync(0xffffffffu, pos, 0), pp1 = __shfl_sync(0xffffffffu, pos, 1);
      if (t < t1) {
        uint8_t* kt = kring + ((t / kWarps) % kStages) * (2 * kTileBytes);
        uint8_t* vt = kt + kTileBytes;
        const int mask = (1 << p.bs_log2) - 1;
#pragma unroll
        for (int i = 0; i < kTok * kChunks / 32; ++i) {
          const int tok = (lane + 32 * i) / kChunks;
          const int c = (lane + 32 * i) % kChunks;
          const int tp = token_pos(tok, blk0, blk1, pp0, pp1);
          const int64_t blkid = p.bs_log2 == 3 && tok >= 8 ? blk1 : blk0;
          const T* ks = static_cast<const T*>(p.k);
          const T* vs = static_cast<const T*>(p.v);
          if (tp >= 0) {
            ks += blkid * p.ks0 + h * p.ks1 + (tp & mask) * p.ks2 + c * 8 * p.ks3;
            vs += blkid * p.vs0 + h * p.vs1 + (tp & mask) * p.vs2 + c * 8 * p.vs3;
          }
          const uint32_t off = tile_chunk<D>(tok, c);
          if (p.vec) {
            cp_async16(smem_u32(kt) + off, ks, tp >= 0 ? 16 : 0);
            cp_async16(smem_u32(vt) + off, vs, tp >= 0 ? 16 : 0);
          } else {
            const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(kt + off) = tp >= 0 ? gather8(ks, p.ks3) : zero;
            *reinterpret_cast<uint4*>(vt + off) = tp >= 0 ? gather8(vs, p.vs3) : zero;
          }
        }
      }
      cp_async_commit();
    };

    // ---- first tiles on their way, then q ----
    int blk[kStages], pos[kStages];  // pages of this warp's next tiles
#pragma unroll
    for (int i = 0; i < kStages; ++i) fetch(t0 + warp + i * kWarps, blk[i], pos[i]);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(t0 + warp + i * kWarps, blk[i], pos[i]);
    for (int e = tid; e < kRows * kChunks; e += kThreads) {
      const int r = e / kChunks, c = e % kChunks;
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows) {
        const int qt = (row0 + r) / p.group;
        const int head = h * p.group + (row0 + r) - qt * p.group;
        const T* src = static_cast<const T*>(p.q) + (s.q0 + qt) * p.qs0 + head * p.qs1 + c * 8 * p.qs2;
        x = p.qs2 == 1 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0
                ? *reinterpret_cast<const uint4*>(src)
                : gather8(src, p.qs2);
      }
      *reinterpret_cast<uint4*>(qsm + tile_chunk<D>(r, c)) = x;
    }
    __syncthreads();

    float o[kM][D / 8][4];
    float m[kM][2], l[kM][2];
    int pos_r[kM][2];  // query position of this thread's rows
#pragma unroll
    for (int a = 0; a < kM; ++a) {
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[a][j][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[a][e] = -INFINITY;
        l[a][e] = 0.f;
        pos_r[a][e] = s.n - s.qlen + (row0 + 16 * a + 8 * e + g8) / p.group;
      }
    }
    uint32_t qf[D / 16][4];  // one row tile: its fragments stay in registers
    auto load_q = [&](int a, int kk, uint32_t(&f)[4]) {
      ldsm_x4(smem_u32(qsm) + tile_chunk<D>(16 * a + (mi & 1) * 8 + r8, 2 * kk + (mi >> 1)), f[0],
              f[1], f[2], f[3]);
    };
    if constexpr (kM == 1) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) load_q(0, kk, qf[kk]);
    }

    for (int t = t0 + warp; t < t1; t += kWarps) {
      issue(t + (kStages - 1) * kWarps, blk[kStages - 1], pos[kStages - 1]);
      const int cb = blk[0], cp = pos[0];  // this tile's own pages, for the masks
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i) {
        blk[i] = blk[i + 1];
        pos[i] = pos[i + 1];
      }
      fetch(t + kStages * kWarps, blk[kStages - 1], pos[kStages - 1]);
      cp_async_wait<kStages - 1>();
      __syncwarp();
      uint8_t* kt = kring + ((t / kWarps) % kStages) * (2 * kTileBytes);
      uint8_t* vt = kt + kTileBytes;
      const int cb0 = __shfl_sync(0xffffffffu, cb, 0), cb1 = __shfl_sync(0xffffffffu, cb, 1);
      const int cp0 = __shfl_sync(0xffffffffu, cp, 0), cp1 = __shfl_sync(0xffffffffu, cp, 1);

      float sc[kM][2][4];
#pragma unroll
      for (int a = 0; a < kM; ++a)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[a][j][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4(smem_u32(kt) + tile_chunk<D>((mi >> 1) * 8 + r8, 2 * kk + (mi & 1)), b0, b1, b2, b3);
#pragma unroll
        for (int a = 0; a < kM; ++a) {
          if constexpr (kM == 1) {
            mma_16816<T>(sc[a][0], qf[kk], b0, b1);
            mma_16816<T>(sc[a][1], qf[kk], b2, b3);
          } else {
            uint32_t f[4];
            load_q(a, kk, f);
            mma_16816<T>(sc[a][0], f, b0, b1);
            mma_16816<T>(sc[a][1], f, b2, b3);
          }
        }
      }
      // ---- scale and masks ----
      int kp[2][2];  // positions of this thread's four tokens, -1: seen by no row
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) kp[j][e] = token_pos(8 * j + 2 * t4 + e, cb0, cb1, cp0, cp1);
      uint32_t vis = 0;  // bit (a, row half, j, e): the row sees the token
#pragma unroll
      for (int a = 0; a < kM; ++a)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = kp[j][e & 1];
            const int pos = pos_r[a][e >> 1];
            const bool on = key >= 0 && key <= pos && (key > pos - p.window || key < p.sinks);
            sc[a][j][e] = on ? sc[a][j][e] * p.scale_log2 : -INFINITY;
            vis |= (on ? 1u : 0u) << (a * 8 + j * 4 + e);
          }
      if (p.raw) {  // one query: row = head of the group, token position = key position
#pragma unroll
        for (int a = 0; a < kM; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int r = 16 * a + 8 * (e >> 1) + g8;
              if (r < rows && kp[j][e & 1] >= 0)
                p.raw[(static_cast<int64_t>(s.q0) * p.hq + h * p.group + row0 + r) * p.raw_tokens +
                      kp[j][e & 1]] = sc[a][j][e];
            }
      }
      // ---- running max and sum, P in the type of V ----
      uint32_t pf[kM][4];
#pragma unroll
      for (int a = 0; a < kM; ++a) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(fmaxf(sc[a][0][2 * e], sc[a][0][2 * e + 1]),
                           fmaxf(sc[a][1][2 * e], sc[a][1][2 * e + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float mn = fmaxf(m[a][e], mx);
          const float base = mn == -INFINITY ? 0.f : mn;
          const float alpha = exp2f(m[a][e] - base);
          m[a][e] = mn;
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float& x = sc[a][j][2 * e + i];
              x = exp2f(x - base);
              sum += x;
            }
          l[a][e] = l[a][e] * alpha + sum;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            o[a][j][2 * e] *= alpha;
            o[a][j][2 * e + 1] *= alpha;
          }
        }
        pf[a][0] = pack2<T>(sc[a][0][0], sc[a][0][1]);
        pf[a][1] = pack2<T>(sc[a][0][2], sc[a][0][3]);
        pf[a][2] = pack2<T>(sc[a][1][0], sc[a][1][1]);
        pf[a][3] = pack2<T>(sc[a][1][2], sc[a][1][3]);
      }
      // A token that some rows of the block see and others do not: an
      // infinity or NaN in its V row must not reach the others (0 * inf), so
      // such elements leave the tile and are added row by row.
      if (rg.pos0 != rg.pos1) {
        constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < kTok * kChunks / 32; ++i) {
          const uint4 x = *reinterpret_cast<const uint4*>(vt + (lane + 32 * i) * 16);
          odd |= nonfinite16(x.x, kExp) | nonfinite16(x.y, kExp) | nonfinite16(x.z, kExp) |
                 nonfinite16(x.w, kExp);
        }
        if (__any_sync(0xffffffffu, odd)) {
          for (int tok = 0; tok < kTok; ++tok) {
            const int src = (lane & ~3) | ((tok & 7) >> 1);  // same rows, the lane with this token
#pragma unroll
            for (int a = 0; a < kM; ++a)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float pv = 0.f;
                bool on = false;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                  for (int i = 0; i < 2; ++i) {
                    const float x = __shfl_sync(0xffffffffu, sc[a][j][2 * e + i], src);
                    const uint32_t w = __shfl_sync(0xffffffffu, vis, src);
                    if (j == (tok >> 3) && i == (tok & 1)) {
                      pv = x;
                      on = (w >> (a * 8 + j * 4 + 2 * e + i)) & 1u;
                    }
                  }
                if (!on) continue;
#pragma unroll
                for (int j = 0; j < D / 8; ++j)
#pragma unroll
                  for (int i = 0; i < 2; ++i) {
                    const float x = to_f32<T>(*reinterpret_cast<const T*>(
                        vt + tile_chunk<D>(tok, j) + (2 * t4 + i) * 2));
                    if (!isfinite(x)) o[a][j][2 * e + i] += pv * x;
                  }
              }
            __syncwarp();
          }
          for (int i = lane; i < kTok * D; i += 32) {
            T* x = reinterpret_cast<T*>(vt) + i;
            if (!isfinite(to_f32<T>(*x))) *x = from_f32<T>(0.f);
          }
          __syncwarp();
        }
      }
#pragma unroll
      for (int dp = 0; dp < D / 16; ++dp) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4_t(smem_u32(vt) + tile_chunk<D>((mi & 1) * 8 + r8, 2 * dp + (mi >> 1)), b0, b1, b2, b3);
#pragma unroll
        for (int a = 0; a < kM; ++a) {
          mma_16816<T>(o[a][2 * dp], pf[a], b0, b1);
          mma_16816<T>(o[a][2 * dp + 1], pf[a], b2, b3);
        }
      }
      __syncwarp();  // the stage is free
    }

    // ---- merge the warps: (max, sum, acc) per row through the ring ----
    cp_async_wait<0>();
    __syncthreads();
    float* acc = reinterpret_cast<float*>(smem);        // [warp][row][D]
    float* ml = acc + kWarps * kRows * D;               // [warp][row][2]
    static_assert(sizeof(float) * kWarps * kRows * (D + 2) <= split_smem_bytes<D, kM>(), "merge buffer");
#pragma unroll
    for (int a = 0; a < kM; ++a)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[a][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int r = 16 * a + 8 * e + g8;
        float* dst = acc + (warp * kRows + r) * D;
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
          *reinterpret_cast<float2*>(dst + 8 * j + 2 * t4) =
              make_float2(o[a][j][2 * e], o[a][j][2 * e + 1]);
        if (t4 == 0) {
          ml[(warp * kRows + r) * 2] = m[a][e];
          ml[(warp * kRows + r) * 2 + 1] = sum;
        }
      }
    __syncthreads();
    for (int e = tid; e < rows * D; e += kThreads) {
      const int r = e / D, d = e - r * D;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, ml[(w * kRows + r) * 2]);
      const float base = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2f(ml[(w * kRows + r) * 2] - base);
        sum += f * ml[(w * kRows + r) * 2 + 1];
        x += f * acc[(w * kRows + r) * D + d];
      }
      const int qt = (row0 + r) / p.group;
      const int head = h * p.group + (row0 + r) - qt * p.group;
      const int64_t row = static_cast<int64_t>(s.q0 + qt) * p.hq + head;
      if (p.splits == 1) {
        const float y = sum == 0.f ? 0.f : x / sum;
        static_cast<T*>(p.out)[(s.q0 + qt) * p.os0 + head * p.os1 + d * p.os2] = from_f32<T>(y);
        if (p.lse && d == 0) p.lse[row] = sum == 0.f ? INFINITY : base + log2f(sum);
      } else {
        p.part_acc[(row * p.splits + split) * D + d] = x;
        if (d == 0) {
          p.part_ml[(row * p.splits + split) * 2] = mx;
          p.part_ml[(row * p.splits + split) * 2 + 1] = sum;
        }
      }
    }
    __syncthreads();
  }
}

// Merge of the splits' partials: one warp per row of q.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) stream_merge_kernel(const __grid_constant__ StreamParams p) {
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.y;
  pdl_wait();
  pdl_launch_dependents();
  const StreamSeq s = sequence_of(p, b);
  for (int64_t r = blockIdx.x * kWarps + (threadIdx.x >> 5); r < static_cast<int64_t>(s.qlen) * p.hq;
       r += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t row = static_cast<int64_t>(s.q0) * p.hq + r;
    const float* ml = p.part_ml + row * p.splits * 2;
    const float* acc = p.part_acc + row * p.splits * D;
    float mx = -INFINITY;
    for (int i = 0; i < p.splits; ++i) mx = fmaxf(mx, ml[2 * i]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, x[D / 32];
#pragma unroll
    for (int j = 0; j < D / 32; ++j) x[j] = 0.f;
    for (int i = 0; i < p.splits; ++i) {
      const float f = exp2f(ml[2 * i] - base);
      sum += f * ml[2 * i + 1];
#pragma unroll
      for (int j = 0; j < D / 32; ++j) x[j] += f * acc[static_cast<int64_t>(i) * D + lane + 32 * j];
    }
    const int64_t qt = s.q0 + r / p.hq, head = r % p.hq;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
      static_cast<T*>(p.out)[qt * p.os0 + head * p.os1 + (lane + 32 * j) * p.os2] =
          from_f32<T>(sum == 0.f ? 0.f : x[j] / sum);
    if (p.lse && lane == 0) p.lse[row] = sum == 0.f ? INFINITY : base + log2f(sum);
  }
}

// scores[token] += sum over the group of exp2(raw - lse): one thread per token.
__global__ void __launch_bounds__(256) stream_scores_kernel(const __grid_constant__ StreamParams p) {
  const int h = blockIdx.y;
  const int b = blockIdx.z;
  pdl_wait();
  pdl_launch_dependents();
  const StreamSeq s = sequence_of(p, b);
  for (int t = blockIdx.x * 256 + threadIdx.x; t < s.n; t += gridDim.x * 256) {
    const int64_t id =
        load_index(p.bt, p.bt64, b * p.bts0 + static_cast<int64_t>(t >> p.bs_log2) * p.bts1);
    if (id < 0 || id >= p.num_blocks) continue;
    const int64_t row = static_cast<int64_t>(b) * p.hq + h * p.group;
    float w = 0.f;
    for (int g = 0; g < p.group; ++g) w += exp2f(p.raw[(row + g) * p.raw_tokens + t] - p.lse[row + g]);
    float* dst = p.scores + id * p.scs0 + h * p.scs1 + (t & ((1 << p.bs_log2) - 1)) * p.scs2;
    *dst = t == s.n - 1 ? w : *dst + w;
  }
}

struct StreamPlan {
  int m16;         // 16-row tiles per CTA: 1 or 2
  int row_blocks;  // grid extent
  int splits;
  bool prompt;     // many rows: prompt_attention, where it takes the layout
  int64_t max_query;
  int64_t raw_tokens;
  size_t acc_bytes, ml_bytes, raw_bytes, lse_bytes;
  size_t bytes() const { return acc_bytes + ml_bytes + raw_bytes + lse_bytes; }
};

int check(const fd_stream_attention_args* a, bool scored) {
  if (!a || a->struct_size != static_cast<int32_t>(sizeof(fd_stream_attention_args)))
    return FD_ERR_INVALID_ARGUMENT;
  if (a->dtype != FD_DTYPE_F16 && a->dtype != FD_DTYPE_BF16) return FD_ERR_UNSUPPORTED;
  if (a->head_dim != 64 && a->head_dim != 128) return FD_ERR_UNSUPPORTED;
  if (a->block_size != 8 && a->block_size != 16 && a->block_size != 32) return FD_ERR_UNSUPPORTED;
  if (a->num_seqs < 0 || a->num_q_heads <= 0 || a->num_kv_heads <= 0 || a->num_blocks <= 0 ||
      a->max_blocks_per_seq <= 0 || a->num_q_heads % a->num_kv_heads != 0)
    return FD_ERR_INVALID_ARGUMENT;
  if (a->num_seqs > 65535 || a->num_kv_heads > 65535 ||
      static_cast<int64_t>(a->max_blocks_per_seq) * a->block_size > 0x3fffffff)
    return FD_ERR_UNSUPPORTED;
  if (!scored) {
    if (a->window < 1 || a->sinks < 0 || a->max_query_len < 1 || a->num_tokens < 0)
      return FD_ERR_INVALID_ARGUMENT;
    if (!a->query_start_loc && a->num_tokens != a->num_seqs) return FD_ERR_INVALID_ARGUMENT;
    if (static_cast<int64_t>(a->num_tokens) * (a->num_q_heads / a->num_kv_heads) > 0x3fffffff)
      return FD_ERR_UNSUPPORTED;
  }
  return FD_OK;
}

int check_pointers(const fd_stream_attention_args* a, bool scored) {
  if (!a->q || !a->out || !a->k_cache || !a->v_cache || !a->block_tables || !a->seq_lens)
    return FD_ERR_INVALID_ARGUMENT;
  if (scored && !a->scores) return FD_ERR_INVALID_ARGUMENT;
  return FD_OK;
}

StreamPlan plan_of(const fd_stream_attention_args* a, bool scored, int sms) {
  StreamPlan pl;
  std::memset(&pl, 0, sizeof(pl));
  const int group = a->num_q_heads / a->num_kv_heads;
  const int64_t tokens = scored ? a->num_seqs : a->num_tokens;
  const int64_t mq = scored || !a->query_start_loc
                         ? 1
                         : std::min<int64_t>(a->max_query_len, std::max<int64_t>(tokens, 1));
  const int64_t rows = mq * group;
  pl.max_query = mq;
  pl.prompt = rows >= 256;
  pl.m16 = rows > 16 ? 2 : 1;
  const int per = 16 * pl.m16;
  pl.row_blocks = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, 65535 / a->num_kv_heads)));
  const int64_t cap = static_cast<int64_t>(a->max_blocks_per_seq) * a->block_size;
  int64_t seen = cap;
  if (!scored) {
    const int64_t most = std::min<int64_t>(a->window, cap) + std::min<int64_t>(a->sinks, cap) +
                         per / group + 2 * a->block_size;
    seen = std::min(cap, most);
  }
  const int64_t tiles = (seen + kTok - 1) / kTok;
  const int64_t units = static_cast<int64_t>(a->num_seqs) * a->num_kv_heads * pl.row_blocks;
  // two CTAs fit an SM; a split holds two tiles per warp at least
  int64_t splits = units > 0 ? 2 * sms / units : 1;
  splits = std::min<int64_t>(std::min<int64_t>(splits, tiles / (2 * kWarps)), kMaxSplits);
  pl.splits = static_cast<int>(std::max<int64_t>(splits, 1));
  const size_t q_rows = static_cast<size_t>(tokens) * a->num_q_heads;
  if (pl.splits > 1) {
    pl.acc_bytes = q_rows * pl.splits * a->head_dim * sizeof(float);
    pl.ml_bytes = q_rows * pl.splits * 2 * sizeof(float);
  }
  if (scored) {
    pl.raw_tokens = cap;
    pl.raw_bytes = q_rows * static_cast<size_t>(cap) * sizeof(float);
    pl.lse_bytes = q_rows * sizeof(float);
  }
  return pl;
}

template <typename T, int D, int kM>
int launch_split(const StreamParams& p, dim3 grid, cudaStream_t stream) {
  auto kern = stream_split_kernel<T, D, kM>;
  constexpr size_t smem = split_smem_bytes<D, kM>();
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(smem));
  if (e == cudaSuccess) e = launch_pdl(kern, grid, dim3(kThreads), smem, stream, p);
  return cuda_status(e);
}

template <typename T, int D>
int launch_typed(const StreamParams& p, const StreamPlan& pl, cudaStream_t stream) {
  const dim3 grid(pl.splits, p.hkv * pl.row_blocks, p.num_seqs);
  int rc = pl.m16 == 1 ? launch_split<T, D, 1>(p, grid, stream) : launch_split<T, D, 2>(p, grid, stream);
  if (rc != FD_OK || pl.splits == 1) return rc;
  const int64_t rows = static_cast<int64_t>(pl.row_blocks) * 16 * pl.m16 * p.hkv;
  const int blocks = static_cast<int>(std::min<int64_t>((rows + kWarps - 1) / kWarps, 65535));
  return cuda_status(launch_pdl(stream_merge_kernel<T, D>, dim3(blocks, p.num_seqs), dim3(kThreads), 0,
                                stream, p));
}

int run(const fd_stream_attention_args* a, bool scored, void* cuda_stream) {
  int rc = check(a, scored);
  if (rc != FD_OK) return rc;
  const bool one = scored || !a->query_start_loc;
  if (a->num_seqs == 0 || (!one && a->num_tokens == 0)) return FD_OK;
  rc = check_pointers(a, scored);
  if (rc != FD_OK) return rc;
  const DeviceInfo* dev = current_device_info();
  int* status = device_status_ptr();
  if (!dev || !status) return FD_ERR_CUDA;
  const StreamPlan pl = plan_of(a, scored, dev->num_sms);
  if (pl.bytes() > 0 && (!a->scratch || a->scratch_bytes < pl.bytes())) return FD_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->scratch) % 16 != 0) return FD_ERR_ALIGNMENT;

  StreamParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = a->q;
  p.qs0 = a->q_stride[0]; p.qs1 = a->q_stride[1]; p.qs2 = a->q_stride[2];
  p.out = a->out;
  p.os0 = a->out_stride[0]; p.os1 = a->out_stride[1]; p.os2 = a->out_stride[2];
  p.k = a->k_cache;
  p.ks0 = a->k_stride[0]; p.ks1 = a->k_stride[1]; p.ks2 = a->k_stride[2]; p.ks3 = a->k_stride[3];
  p.v = a->v_cache;
  p.vs0 = a->v_stride[0]; p.vs1 = a->v_stride[1]; p.vs2 = a->v_stride[2]; p.vs3 = a->v_stride[3];
  p.bt = a->block_tables;
  p.bts0 = a->block_tables_stride[0]; p.bts1 = a->block_tables_stride[1];
  p.bt64 = a->block_tables_index == FD_INDEX_I64;
  p.sl = a->seq_lens;
  p.sls = a->seq_lens_stride;
  p.sl64 = a->seq_lens_index == FD_INDEX_I64;
  p.num_seqs = a->num_seqs;
  p.num_tokens = one ? a->num_seqs : a->num_tokens;
  p.hq = a->num_q_heads;
  p.hkv = a->num_kv_heads;
  p.group = a->num_q_heads / a->num_kv_heads;
  p.bs_log2 = a->block_size == 8 ? 3 : (a->block_size == 16 ? 4 : 5);
  p.num_blocks = a->num_blocks;
  p.max_blocks = a->max_blocks_per_seq;
  p.window = p.sinks = 0;
  if (scored) {
    p.window = 0x3fffffff;
    p.scores = a->scores;
    p.scs0 = a->scores_stride[0]; p.scs1 = a->scores_stride[1]; p.scs2 = a->scores_stride[2];
  } else {
    p.window = static_cast<int>(std::min<int64_t>(a->window, 0x3fffffff));
    p.sinks = static_cast<int>(std::min<int64_t>(a->sinks, 0x3fffffff));
    p.qstart = a->query_start_loc;
    p.qss = a->query_start_loc_stride;
    p.qs64 = a->query_start_loc_index == FD_INDEX_I64;
  }
  p.row_blocks = pl.row_blocks;
  p.splits = pl.splits;
  auto aligned = [](const void* base, const int64_t* st) {
    return reinterpret_cast<uintptr_t>(base) % 16 == 0 && st[0] % 8 == 0 && st[1] % 8 == 0 &&
           st[2] % 8 == 0 && st[3] == 1;
  };
  p.vec = aligned(a->k_cache, a->k_stride) && aligned(a->v_cache, a->v_stride);
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  char* at = static_cast<char*>(a->scratch);
  p.part_acc = reinterpret_cast<float*>(at);
  p.part_ml = reinterpret_cast<float*>(at + pl.acc_bytes);
  if (scored) {
    p.raw = reinterpret_cast<float*>(at + pl.acc_bytes + pl.ml_bytes);
    p.lse = reinterpret_cast<float*>(at + pl.acc_bytes + pl.ml_bytes + pl.raw_bytes);
  }
  p.raw_tokens = pl.raw_tokens;
  p.status = status;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const bool bf16 = a->dtype == FD_DTYPE_BF16;
  if (pl.prompt && prompt_attention(p, bf16, a->head_dim, pl.max_query, stream, &rc)) return rc;
  if (a->head_dim == 128) {
    rc = bf16 ? launch_typed<__nv_bfloat16, 128>(p, pl, stream) : launch_typed<__half, 128>(p, pl, stream);
  } else {
    rc = bf16 ? launch_typed<__nv_bfloat16, 64>(p, pl, stream) : launch_typed<__half, 64>(p, pl, stream);
  }
  if (rc != FD_OK || !scored) return rc;
  const int chunks = static_cast<int>(std::min<int64_t>((pl.raw_tokens + 255) / 256, 1024));
  return cuda_status(launch_pdl(stream_scores_kernel, dim3(chunks, p.hkv, p.num_seqs), dim3(256), 0, stream, p));
}

int workspace(const fd_stream_attention_args* a, bool scored, size_t* bytes) {
  const int rc = check(a, scored);
  if (rc != FD_OK) return rc;
  if (!bytes) return FD_ERR_INVALID_ARGUMENT;
  const DeviceInfo* dev = current_device_info();
  if (!dev) return FD_ERR_CUDA;
  *bytes = a->num_seqs > 0 ? plan_of(a, scored, dev->num_sms).bytes() : 0;
  return FD_OK;
}

}  // namespace
}  // namespace fd

extern "C" {

int fd_window_attention_workspace(const fd_stream_attention_args* a, size_t* scratch_bytes) {
  return fd::workspace(a, false, scratch_bytes);
}
int fd_window_attention(const fd_stream_attention_args* a, void* cuda_stream) {
  return fd::run(a, false, cuda_stream);
}
int fd_scored_decode_workspace(const fd_stream_attention_args* a, size_t* scratch_bytes) {
  return fd::workspace(a, true, scratch_bytes);
}
int fd_scored_decode(const fd_stream_attention_args* a, void* cuda_stream) {
  return fd::run(a, true, cuda_stream);
}

}  // extern "C"

// Attention over a bounded cache for few queries per sequence: one decoded
// token, or a handful of drafts (fd_window_attention), and one token with the
// attention weights kept (fd_scored_decode).
#include <algorithm>
#include <climits>
#include <cstring>
#include <type_traits>

#include "../../include/flashdec_b200.h"
#include "fd_host.h"
#include "fd_ptx.cuh"
#include "fd_stream.cuh"
#include "fd_stream.h"

namespace fd {
namespace {

constexpr int kCluster = 0, kGrid = 1, kShares = 2;  // StreamParams::mode, see stream_split_kernel
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTok = 16;    // tokens per warp tile
constexpr int kStages = 3;  // tiles in flight per warp
constexpr int kMaxCluster = 8;      // splits that merge inside a cluster
constexpr int kMaxListed = 512;     // sequences of a launch
constexpr int kMinShare = 16;       // tiles of a CTA's share, at least
constexpr int kGridRun = 64;        // tiles of a CTA in kGrid, at most
constexpr int kSnap = 4;            // tiles: a cut this near to a unit's end moves there
constexpr int kRawBytes = 10 << 10; // scores a CTA may keep in shared memory
constexpr int kClusterRun = 512;    // tokens of a split of a cluster, at most
constexpr int kOldMost = kClusterRun / kThreads;
constexpr int kGroupMost = 16384;   // query heads a KV head, at most

template <int D>
constexpr size_t ring_bytes() {
  return static_cast<size_t>(kWarps) * kStages * 2 * kTok * D * 2;
}
// ring (later the merge buffer: kWarps x rows x (D + 2) floats) and q (one row
// tile: in the ring, see below); per row the offset of its output, the warps'
// and the cluster's weights, lse
template <int D, int kM>
constexpr size_t split_smem_bytes() {
  return ring_bytes<D>() + static_cast<size_t>(kM) * 16 *
                               ((kM > 1 ? D * 2 : 0) + sizeof(int64_t) + (kWarps + kMaxCluster + 2) * sizeof(float));
}
// what the other CTAs of a cluster send: (max, sum) per row and their part of
// this CTA's share of the rows' elements
__host__ __device__ constexpr int receive_ml(int splits, int rows) {  // floats; what follows starts on 16 bytes
  return (2 * splits * rows + 3) & ~3;
}
__host__ __device__ constexpr size_t receive_bytes(int splits, int rows, int D) {
  return sizeof(float) * (static_cast<size_t>(receive_ml(splits, rows)) + static_cast<size_t>(rows) * D + 4 * splits);
}

// Elements d .. d + 3 of a row.
template <typename T>
__device__ __forceinline__ void store4(T* row, int d, int64_t stride, int vec, float4 x) {
  if (vec) {
    *reinterpret_cast<uint2*>(row + d) = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
  } else {
    row[d * stride] = from_f32<T>(x.x);
    row[(d + 1) * stride] = from_f32<T>(x.y);
    row[(d + 2) * stride] = from_f32<T>(x.z);
    row[(d + 3) * stride] = from_f32<T>(x.w);
  }
}

// Tiles that a unit (row block x KV head) of a sequence is counted with: what
// its last row block sees, one at least (rows that see nothing are written too).
__device__ __forceinline__ int unit_tiles(const StreamParams& p, const StreamSeq& s, int rows) {
  const int all = s.qlen * p.group;
  if (all == 0) return 1;
  const StreamRange rg(s, (all - 1) / rows * rows, all, p.group, p.window, p.sinks, p.bs_log2);
  return max(((rg.pages << p.bs_log2) + kTok - 1) / kTok, 1);
}

// Tokens before a sequence's raw scores, from the tiles of the units before it
// (one query a sequence: as many units each as the group has row blocks).
__device__ __forceinline__ int64_t raw_tokens_before(const StreamParams& p, int64_t unit_tiles_before) {
  const uint64_t x = static_cast<uint64_t>(unit_tiles_before);
  return static_cast<int64_t>(p.blocks_magic ? __umul64hi(x, p.blocks_magic) : x) * kTok;
}

// Last i of [0, n) with first[i] <= x (first[0] <= x).
__device__ __forceinline__ int last_up_to(const int64_t* first, int n, int64_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  return lo;
}

// Byte offset of 16-byte chunk `c` of row `r` in a [rows][D] 16-bit tile: the
// chunk index is XORed with r % 8, so the 8 rows of an ldmatrix start on
// different banks.
template <int D>
__device__ __forceinline__ uint32_t tile_chunk(int r, int c) {
  return r * (D * 2) + ((c ^ (r & 7)) << 4);
}

// ---------------------------------------------------------------------------
// Works on segments: rows [16 kM rb, +16 kM) of a (sequence, KV head), a unit,
// against a run of the pages they see.  Row r is head r % group of query r /
// group, so K and V are read once for the whole group.  Tile i of 16 tokens
// goes to warp i % 4; each warp keeps three tiles in flight with cp.async and
// its own maximum and sum (base 2, the maximum followed only when a score
// passes it by 2^8), and the four merge at the end.
//
// p.mode:
//   kCluster  a unit per cluster, a segment per CTA; they merge through
//             distributed shared memory.
//   kGrid     a unit per p.splits CTAs, a segment each, as partials.
//   kShares   the tiles of all sequences in a row are cut into equal shares, one
//             per CTA and KV head, whatever the lengths: a CTA has a few
//             segments, of which only the first and the last can be parts of a
//             unit and leave partials.  The heads' CTAs of a share go over the
//             same pages together: with the heads one after another in the row,
//             24 sequences with interleaved heads took 151 us (139), 64 with a
//             plane a head 166 (161).  As many shares as CTAs fit: with four
//             times as many, one long sequence of 131071 tokens took 117 us
//             (97), 64 sequences of up to 4100 visible tokens 180 us (162).
// Partials go to stream_merge_kernel, or stream_finish_kernel with scores.
//
// Bounds: long windows, the reads of K and V, once each (64 sequences of up to
// 131072 tokens, window 4096, 32/8 heads of 128: 892 MB in 160 us, 5.6 TB/s; one
// sequence of 131071 tokens: 537 MB in 95 us, 5.7 TB/s); a short one, a chain of
// dependent steps - table, first tile, its product, two merges (one token,
// window 1024, 16/2 heads: 9.2 us, of which 0.16 are bytes).  Above 16 rows the
// instructions a tile weigh as much (24 sequences of up to 7 drafts, window 1500,
// 16/4 heads of 64: 20 us for 27 MB, merge included; DRAM 17 % busy).
// ---------------------------------------------------------------------------
template <typename T, int D, int kM>
__global__ void __launch_bounds__(kThreads, 2) stream_split_kernel(const __grid_constant__ StreamParams p) {
  constexpr int kRows = 16 * kM;
  constexpr int kChunks = D / 8;
  constexpr uint32_t kTileBytes = kTok * D * 2;
  extern __shared__ __align__(128) uint8_t smem[];
  int64_t* row_out = reinterpret_cast<int64_t*>(smem + ring_bytes<D>() + (kM > 1 ? kRows * D * 2 : 0));  // [row] element offset in out
  float* warp_weight = reinterpret_cast<float*>(row_out + kRows);      // [warp][row]
  float* weight = warp_weight + kWarps * kRows;                        // [split][row] of the cluster
  float* lse = weight + kMaxCluster * kRows;                           // [row]
  float* inv_sum = lse + kRows;                                        // [row], one split
  float* got_ml = reinterpret_cast<float*>(smem + split_smem_bytes<D, kM>());  // [split][rows_most][2]
  float* got = got_ml + receive_ml(p.splits, p.rows_most);                            // [split][share]
  float* raw = p.mode == kCluster ? got_ml + receive_bytes(p.splits, p.rows_most, D) / sizeof(float) : got_ml;  // [row][raw_tokens]
  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int g8 = lane >> 2;
  const int t4 = lane & 3;
  const int mi = lane >> 3;
  const int r8 = lane & 7;
  const int mask = (1 << p.bs_log2) - 1;
  int64_t* const upto = reinterpret_cast<int64_t*>(got_ml);  // [num_seqs + 1] tiles before a sequence's (no cluster)
  int* const unit = reinterpret_cast<int*>(upto + p.num_seqs + 1);  // [num_seqs] tiles of its units
  // a scale of 0 (uniform weights) stays above it: -inf * 0 is NaN; its sign goes to q
  const float scale = fmaxf(fabsf(p.scale_log2), 1e-30f);
  const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;

  const bool cluster = p.mode == kCluster, grid = p.mode == kGrid;
  if (cluster) cluster_arrive_relaxed();  // all its CTAs run before one of them is sent anything
  pdl_wait();
  pdl_launch_dependents();
  uint8_t* const kring = smem + warp * (kStages * 2 * kTileBytes);
  // this lane's part of a tile copy: chunk `cc` of rows cr, cr + kStep, ...
  constexpr int kStep = 32 / kChunks;
  const int cr = lane / kChunks, cc = lane % kChunks;
  const uint32_t copy_off = tile_chunk<D>(cr, cc);
  const uint32_t k_off = tile_chunk<D>((mi >> 1) * 8 + r8, mi & 1);
  const uint32_t v_off = tile_chunk<D>((mi & 1) * 8 + r8, mi >> 1);

  // what a cluster receives has room for as many rows as were announced: where
  // there are more, they are taken that many at a time
  const int block_rows = cluster ? p.rows_most : kRows;
  int b = 0, h = 0, rb = 0;
  StreamSeq s;
  int64_t at = 0, end = 0;  // this CTA's share of the tiles
  if (cluster || grid) {
    b = p.first_seq + blockIdx.z;
    h = blockIdx.y % p.hkv;
    rb = blockIdx.y / p.hkv;
    s = sequence_of(p, b);
  } else {
    for (int i = tid; i < p.num_seqs; i += kThreads) {
      s = sequence_of(p, p.first_seq + i);
      unit[i] = unit_tiles(p, s, kRows);
      upto[i + 1] = static_cast<int64_t>((s.qlen * p.group + kRows - 1) / kRows) * unit[i];
    }
    __syncthreads();
    if (warp == 0) {
      int64_t sum = 0;
      for (int i = 0; i < p.num_seqs; i += 32) {
        int64_t x = i + lane < p.num_seqs ? upto[i + lane + 1] : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
          if (lane >= d) x += y;
        }
        if (i + lane < p.num_seqs) upto[i + lane + 1] = sum + x;
        sum += __shfl_sync(0xffffffffu, x, 31);
      }
      if (lane == 0) upto[0] = 0;
    }
    __syncthreads();
    const int64_t total = upto[p.num_seqs];
    if (p.scores && blockIdx.x == 0)  // where a sequence's raw scores start
      for (int i = tid; i < p.num_seqs; i += kThreads) p.raw_start[i] = raw_tokens_before(p, upto[i]);
    const int shares = static_cast<int>(min(max(total / kMinShare, int64_t(1)), static_cast<int64_t>(gridDim.x / p.hkv)));
    const int c = blockIdx.x / p.hkv;
    h = blockIdx.x - c * p.hkv;
    if (c >= shares || total == 0) {
      if (blockIdx.x == 0 && tid == 0) *p.shares = 0;
      return;
    }
    auto cut = [&](int i) -> int64_t {
      int64_t x = total * i / shares;
      if (i == 0 || i == shares) return x;
      const int q = last_up_to(upto, p.num_seqs, x);
      const int past = static_cast<int>((x - upto[q]) % unit[q]);
      if (past < kSnap) return x - past;
      return unit[q] - past < kSnap ? x + unit[q] - past : x;
    };
    at = cut(c);
    end = cut(c + 1);
    if (h == 0 && tid == 0) {  // where the share starts
      const int i = last_up_to(upto, p.num_seqs, at);
      const int64_t past = at - upto[i];
      const int u = static_cast<int>(past / unit[i]);
      p.share_unit[c] = make_int3(i, u, static_cast<int>(past - static_cast<int64_t>(u) * unit[i]));
    }
    if (blockIdx.x == 0 && tid == 0) *p.shares = shares;
  }
  if (cluster) cluster_wait();
  for (;;) {
    int from = 0, to = 0, all = 0;  // the segment: tiles [from, to) of the unit's `all`
    if (!cluster && !grid) {
      if (at >= end) break;
      const int i = last_up_to(upto, p.num_seqs, at);
      b = p.first_seq + i;
      all = unit[i];
      const int64_t past = at - upto[i];
      rb = static_cast<int>(past / all);
      from = static_cast<int>(past - static_cast<int64_t>(rb) * all);
      to = static_cast<int>(min(static_cast<int64_t>(all), from + (end - at)));
      at += to - from;
      s = sequence_of(p, b);
    }
    const int rows_all = s.qlen * p.group;
    if (rb * block_rows >= rows_all) break;  // of a cluster or grid: the last row block is done
    // (grid: row blocks past the announced ones have no place for partials)
    const bool whole_unit = cluster ? false : grid ? rb >= p.row_blocks || p.splits == 1 : from == 0 && to == all;
    if (grid && whole_unit && blockIdx.x > 0) break;
    const int part = grid ? (blockIdx.z * gridDim.y + blockIdx.y) * p.splits + blockIdx.x
                          : 2 * blockIdx.x + (from == 0 ? 1 : 0);  // place of a partial
    {
      const int row0 = rb * block_rows;
      const int rows = min(block_rows, rows_all - row0);
      const StreamRange rg(s, row0, row0 + rows, p.group, p.window, p.sinks, p.bs_log2);
      const int tiles = ((rg.pages << p.bs_log2) + kTok - 1) / kTok;
      const int splits = p.splits, split = blockIdx.x;  // of a cluster
      const int per = max((tiles + splits - 1) / splits, 2 * kWarps);
      int t0 = min(from, tiles), t1 = to == all ? tiles : min(to, tiles);
      if (cluster || (grid && !whole_unit)) {
        t0 = min(split * per, tiles);
        t1 = min(t0 + per, tiles);
      }

      // lanes 0 and 1 hold the (at most two) pages of a tile: {block, position of its first token}
      auto fetch = [&](int t, int& blk, int& pos) {
        blk = -1;
        pos = 0;
        const int i = p.bs_log2 >= 4 ? (t * kTok) >> p.bs_log2 : 2 * t + lane;
        if (lane < 2 && t < t1 && i < rg.pages) {
          const int page = rg.page(i);
          pos = p.bs_log2 >= 4 ? (page << p.bs_log2) + ((t * kTok) & mask) : page << p.bs_log2;
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
      // all 16 tokens seen by some row (`all`: by every row) and their pages good
      auto whole = [&](int blk0, int blk1, int pos0, int pos1, bool all) -> bool {
        const int hi = all ? rg.pos0 : rg.pos1;
        const int lo = all ? max(rg.pos1 - p.window + 1, 0) : rg.lo;
        const int se = all ? min(p.sinks, rg.pos0 + 1) : rg.sink_end;
        auto run_ok = [&](int first, int n) { return first + n <= se || (first >= lo && first + n - 1 <= hi); };
        if (p.bs_log2 == 3) return blk0 >= 0 && blk1 >= 0 && run_ok(pos0, 8) && run_ok(pos1, 8);
        return blk0 >= 0 && run_ok(pos0, kTok);
      };
      auto issue = [&](int t, int blk, int pos) {
        const int blk0 = __shfl_sync(0xffffffffu, blk, 0), blk1 = __shfl_sync(0xffffffffu, blk, 1);
        const int pp0 = __shfl_sync(0xffffffffu, pos, 0), pp1 = __shfl_sync(0xffffffffu, pos, 1);
        if (t < t1) {
          uint8_t* kt = kring + ((t / kWarps) % kStages) * (2 * kTileBytes);
          constexpr int kN = kTok / kStep;
          if (p.vec && whole(blk0, blk1, pp0, pp1, false)) {
            const T* k0 = static_cast<const T*>(p.k) + blk0 * p.ks0 + h * p.ks1 + ((pp0 & mask) + cr) * p.ks2 + cc * 8;
            const T* v0 = static_cast<const T*>(p.v) + blk0 * p.vs0 + h * p.vs1 + ((pp0 & mask) + cr) * p.vs2 + cc * 8;
            const T* k1 = k0 + 8 * p.ks2;
            const T* v1 = v0 + 8 * p.vs2;
            if (p.bs_log2 == 3) {
              k1 = static_cast<const T*>(p.k) + blk1 * p.ks0 + h * p.ks1 + cr * p.ks2 + cc * 8;
              v1 = static_cast<const T*>(p.v) + blk1 * p.vs0 + h * p.vs1 + cr * p.vs2 + cc * 8;
            }
            const int64_t kstep = kStep * p.ks2, vstep = kStep * p.vs2;
            const uint32_t dst = smem_u32(kt);
#pragma unroll
            for (int i = 0; i < kN; ++i) {
              const uint32_t off = (copy_off + i * (kStep * D * 2)) ^ (((i * kStep) & 7) << 4);
              cp_async16(dst + off, i < kN / 2 ? k0 : k1);
              cp_async16(dst + kTileBytes + off, i < kN / 2 ? v0 : v1);
              if (i < kN / 2) {
                k0 += kstep;
                v0 += vstep;
              } else {
                k1 += kstep;
                v1 += vstep;
              }
            }
          } else {
            uint8_t* vt = kt + kTileBytes;
#pragma unroll 1
            for (int i = 0; i < kN; ++i) {
              const int tok = cr + i * kStep;
              const int tp = token_pos(tok, blk0, blk1, pp0, pp1);
              const int64_t blkid = p.bs_log2 == 3 && tok >= 8 ? blk1 : blk0;
              const T* ks = static_cast<const T*>(p.k);
              const T* vs = static_cast<const T*>(p.v);
              if (tp >= 0) {
                ks += blkid * p.ks0 + h * p.ks1 + (tp & mask) * p.ks2 + cc * 8 * p.ks3;
                vs += blkid * p.vs0 + h * p.vs1 + (tp & mask) * p.vs2 + cc * 8 * p.vs3;
              }
              const uint32_t off = tile_chunk<D>(tok, cc);
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
        }
        cp_async_commit();
      };

      // ---- q on its way, the first tiles on theirs, then q to shared memory ----
      constexpr int kQ = kRows * kChunks / kThreads;
      uint4 qx[kQ];
#pragma unroll
      for (int i = 0; i < kQ; ++i) {
        const int e = tid + i * kThreads, r = e / kChunks, c = e % kChunks;
        qx[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows) {
          const int qt = (row0 + r) / p.group;
          const int head = h * p.group + (row0 + r) - qt * p.group;
          const T* src = static_cast<const T*>(p.q) + (s.q0 + qt) * p.qs0 + head * p.qs1 + c * 8 * p.qs2;
          qx[i] = p.q_vec ? *reinterpret_cast<const uint4*>(src) : gather8(src, p.qs2);
        }
      }
      int blk[kStages], pos[kStages];  // pages of this warp's next tiles
#pragma unroll
      for (int i = 0; i < kStages; ++i) fetch(t0 + warp + i * kWarps, blk[i], pos[i]);
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i) issue(t0 + warp + i * kWarps, blk[i], pos[i]);
      // One row tile of q goes to the stage of warp 0's third tile, which is not
      // loaded before every warp has its fragments: two CTAs then fit an SM
      // with what a cluster's CTA receives.
      uint8_t* const qsm = kM > 1 ? smem + ring_bytes<D>()
                                  : smem + ((t0 / kWarps + kStages - 1) % kStages) * (2 * kTileBytes);
#pragma unroll
      for (int i = 0; i < kQ; ++i) {
        const int e = tid + i * kThreads;
        *reinterpret_cast<uint4*>(qsm + tile_chunk<D>(e / kChunks, e % kChunks)) =
            make_uint4(qx[i].x ^ flip, qx[i].y ^ flip, qx[i].z ^ flip, qx[i].w ^ flip);
      }
      __syncthreads();

      float o[kM][D / 8][4];
      float m[kM][2], l[kM][2];  // m in score units: P = exp2((S - m) scale)
      int pos_r[kM][2];          // query position of this thread's rows
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
        __syncthreads();
      }
      const float slack = 8.f / scale;
      // where this thread's rows' scores go (one query: row = head of the group,
      // list place = position), less the tile's; nowhere where the tables list more
      // pages than the cache has
      int64_t raw_tokens = p.raw_tokens;
      float* raw_at = nullptr;
      if (p.scores) {
        if (cluster) {
          raw_at = raw - t0 * kTok;
        } else {
          int64_t before = blockIdx.z * raw_tokens;
          if (!grid) {
            before = raw_tokens_before(p, upto[b - p.first_seq]);
            raw_tokens = static_cast<int64_t>(all) * kTok;
          }
          if (before + raw_tokens <= p.raw_room)
            raw_at = p.raw + before * p.hq + (h * p.group + row0) * raw_tokens;
        }
      }
      float* raw_row[kM][2];
#pragma unroll
      for (int a = 0; a < kM; ++a)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 16 * a + 8 * e + g8;
          raw_row[a][e] = nullptr;
          if (raw_at && r < rows) raw_row[a][e] = raw_at + r * raw_tokens + 2 * t4;
        }

      for (int t = t0 + warp; t < t1; t += kWarps) {
        issue(t + (kStages - 1) * kWarps, blk[kStages - 1], pos[kStages - 1]);
        const int cb0 = __shfl_sync(0xffffffffu, blk[0], 0), cb1 = __shfl_sync(0xffffffffu, blk[0], 1);
        const int cp0 = __shfl_sync(0xffffffffu, pos[0], 0), cp1 = __shfl_sync(0xffffffffu, pos[0], 1);
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
          ldsm_x4(smem_u32(kt) + (k_off ^ (kk << 5)), b0, b1, b2, b3);
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
        // ---- masks, where some row misses some token ----
        const bool edge = !whole(cb0, cb1, cp0, cp1, true);
        uint32_t vis = 0xffffffffu;  // bit (a, j, e): the row sees the token
        if (edge) {
          int kp[2][2];  // positions of this thread's four tokens, -1: seen by no row
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) kp[j][e] = token_pos(8 * j + 2 * t4 + e, cb0, cb1, cp0, cp1);
          vis = 0;
#pragma unroll
          for (int a = 0; a < kM; ++a)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int key = kp[j][e & 1];
                const int at = pos_r[a][e >> 1];
                const bool on = key >= 0 && key <= at && (key > at - p.window || key < p.sinks);
                if (!on) sc[a][j][e] = -INFINITY;
                vis |= (on ? 1u : 0u) << (a * 8 + j * 4 + e);
              }
        }
        if (p.scores) {  // rows are padded to whole tiles
#pragma unroll
          for (int a = 0; a < kM; ++a)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (raw_row[a][e]) {
                float* dst = raw_row[a][e] + static_cast<int64_t>(t) * kTok;
                *reinterpret_cast<float2*>(dst) = make_float2(sc[a][0][2 * e] * scale, sc[a][0][2 * e + 1] * scale);
                *reinterpret_cast<float2*>(dst + 8) = make_float2(sc[a][1][2 * e] * scale, sc[a][1][2 * e + 1] * scale);
              }
        }
        // ---- follow the maximum when it is 2^8 behind ----
        bool behind = false;
#pragma unroll
        for (int a = 0; a < kM; ++a)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            behind |= fmaxf(fmaxf(sc[a][0][2 * e], sc[a][0][2 * e + 1]),
                            fmaxf(sc[a][1][2 * e], sc[a][1][2 * e + 1])) > m[a][e] + slack;
        if (__any_sync(0xffffffffu, behind)) {
#pragma unroll
          for (int a = 0; a < kM; ++a)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(fmaxf(sc[a][0][2 * e], sc[a][0][2 * e + 1]),
                               fmaxf(sc[a][1][2 * e], sc[a][1][2 * e + 1]));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
              const float mn = fmaxf(m[a][e], mx);
              const float alpha = mn == -INFINITY ? 1.f : ex2((m[a][e] - mn) * scale);
              m[a][e] = mn;
              l[a][e] *= alpha;
#pragma unroll
              for (int j = 0; j < D / 8; ++j) {
                o[a][j][2 * e] *= alpha;
                o[a][j][2 * e + 1] *= alpha;
              }
            }
        }
        // ---- weights, rounded to the type of V for the product ----
        uint32_t pf[kM][4];
#pragma unroll
        for (int a = 0; a < kM; ++a) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float base = m[a][e] == -INFINITY ? 0.f : m[a][e] * scale;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float& x = sc[a][j][2 * e + i];
                x = ex2(fmaf(x, scale, -base));
                // The sum takes the weights as the product takes them, so that a
                // row with one great weight is not off by its rounding.  With
                // scores it is the exact sum: their weights are not rounded.
                l[a][e] += p.scores ? x : to_f32<T>(from_f32<T>(x));
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
        if (edge && rg.pos0 != rg.pos1) {
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
          ldsm_x4_t(smem_u32(vt) + (v_off ^ (dp << 5)), b0, b1, b2, b3);
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
      // with scores: the slots and old values of this thread's tokens, on their way
      float* slot[kOldMost];
      float old[kOldMost];
      if (cluster && p.scores) {
#pragma unroll
        for (int i = 0; i < kOldMost; ++i) {
          const int tok = t0 * kTok + tid + i * kThreads;
          slot[i] = nullptr;
          old[i] = 0.f;
          if (tok < min(t1 * kTok, s.n)) {
            const int64_t id = load_index(p.bt, p.bt64, b * p.bts0 + static_cast<int64_t>(tok >> p.bs_log2) * p.bts1);
            if (id >= 0 && id < p.num_blocks) {
              slot[i] = p.scores + id * p.scs0 + h * p.scs1 + (tok & mask) * p.scs2;
              if (tok < s.n - 1) old[i] = *slot[i];
            }
          }
        }
      }
      float* acc = reinterpret_cast<float*>(smem);  // [warp][row][D]
      float* ml = acc + kWarps * kRows * D;         // [warp][row][2]
      static_assert(sizeof(float) * kWarps * kRows * (D + 2) <= ring_bytes<D>(), "merge buffer");
#pragma unroll
      for (int a = 0; a < kM; ++a)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = l[a][e];
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          const int r = 16 * a + 8 * e + g8;
          if (r >= rows) continue;
          float* dst = acc + (warp * kRows + r) * D;
#pragma unroll
          for (int j = 0; j < D / 8; ++j)
            *reinterpret_cast<float2*>(dst + 8 * j + 2 * t4) =
                make_float2(o[a][j][2 * e], o[a][j][2 * e + 1]);
          if (t4 == 0) {
            ml[(warp * kRows + r) * 2] = m[a][e] * scale;
            ml[(warp * kRows + r) * 2 + 1] = sum;
          }
        }
      __syncthreads();
      if (tid < rows) {  // the row's weights, and where it goes
        const int r = tid;
        float pm[kWarps], mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          pm[w] = ml[(w * kRows + r) * 2];
          mx = fmaxf(mx, pm[w]);
        }
        const float base = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = ex2(pm[w] - base);
          warp_weight[w * kRows + r] = f;
          sum += f * ml[(w * kRows + r) * 2 + 1];
        }
        const int qt = (row0 + r) / p.group;
        const int head = h * p.group + (row0 + r) - qt * p.group;
        const int64_t row = static_cast<int64_t>(s.q0 + qt) * p.hq + head;
        row_out[r] = cluster || whole_unit ? (s.q0 + qt) * p.os0 + head * p.os1 : (static_cast<int64_t>(part) * kRows + r) * D;
        inv_sum[r] = sum == 0.f ? 0.f : 1.f / sum;
        if (cluster) {
          for (int i = 0; i < splits; ++i)
            st_cluster_v2(map_to_rank(smem_u32(got_ml + (split * p.rows_most + r) * 2), i), mx, sum);
        } else if (!whole_unit) {
          *reinterpret_cast<float2*>(p.part_ml + (static_cast<int64_t>(part) * kRows + r) * 2) = make_float2(mx, sum);
        } else if (p.scores) {
          p.row_lse[row] = sum == 0.f ? INFINITY : base + log2f(sum);
        }
      }
      __syncthreads();
      // elements 4 e4 .. + 3 of the rows' [rows][D]; rank i of a cluster gets [share i, + share)
      const int share = cluster ? (rows * (D / 4) + splits - 1) / splits * 4 : 0;
      T* const out = static_cast<T*>(p.out);
      for (int e4 = tid; e4 < rows * (D / 4); e4 += kThreads) {
        const int r = e4 / (D / 4), d = 4 * (e4 % (D / 4));
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = warp_weight[w * kRows + r];
          const float4 y = *reinterpret_cast<const float4*>(acc + (w * kRows + r) * D + d);
          x.x += f * y.x;
          x.y += f * y.y;
          x.z += f * y.z;
          x.w += f * y.w;
        }
        if (cluster) {
          const int to = 4 * e4 / share;
          st_cluster_v4(map_to_rank(smem_u32(got + split * share + 4 * e4 - to * share), to), x.x, x.y, x.z, x.w);
        } else if (whole_unit) {
          const float f = inv_sum[r];
          store4<T>(out + row_out[r], d, p.os2, p.out_vec, make_float4(x.x * f, x.y * f, x.z * f, x.w * f));
        } else {
          *reinterpret_cast<float4*>(p.part_acc + row_out[r] + d) = x;
        }
      }
      if (cluster) {
        // ---- merge the cluster's splits: everything needed has been sent here ----
        cluster_arrive();
        cluster_wait();
        if (tid < rows) {
          const int r = tid;
          float pm[kMaxCluster], pl[kMaxCluster], mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < kMaxCluster; ++i) {
            pm[i] = i < splits ? got_ml[(i * p.rows_most + r) * 2] : -INFINITY;
            pl[i] = i < splits ? got_ml[(i * p.rows_most + r) * 2 + 1] : 0.f;
            mx = fmaxf(mx, pm[i]);
          }
          const float base = mx == -INFINITY ? 0.f : mx;
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < kMaxCluster; ++i) {
            pm[i] = ex2(pm[i] - base);
            sum += pm[i] * pl[i];
          }
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
          for (int i = 0; i < kMaxCluster; ++i) weight[i * kRows + r] = pm[i] * inv;
          lse[r] = sum == 0.f ? INFINITY : base + log2f(sum);
        }
        __syncthreads();
        for (int e4 = tid; e4 < share / 4; e4 += kThreads) {
          const int e = split * share + 4 * e4;
          if (e >= rows * D) break;
          const int r = e / D, d = e % D;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int i = 0; i < kMaxCluster; ++i) {
            if (i >= splits) break;
            const float f = weight[i * kRows + r];
            const float4 y = *reinterpret_cast<const float4*>(got + i * share + 4 * e4);
            x.x += f * y.x;
            x.y += f * y.y;
            x.z += f * y.z;
            x.w += f * y.w;
          }
          store4<T>(out + row_out[r], d, p.os2, p.out_vec, x);
        }
        if (p.scores) {
#pragma unroll
          for (int i = 0; i < kOldMost; ++i) {
            if (!slot[i]) continue;
            float w = 0.f;
            for (int r = 0; r < rows; ++r) w += ex2(raw[r * p.raw_tokens + tid + i * kThreads] - lse[r]);
            *slot[i] = old[i] + w;
          }
        }
        if ((rb + p.row_blocks) * block_rows < rows_all) {  // the next rows are sent to the same place
          cluster_arrive();
          cluster_wait();
        }
      }
      if (cluster || grid) rb += p.row_blocks;
      __syncthreads();
    }
  }
}

// What remains after the split kernel where units were cut: one row a CTA, the
// segments of the row's unit shared out over the warps.  kGrid: CTA (unit, row);
// kShares: CTA ((c, head), row) has the unit that share c + 1 is the first to
// start inside, if it is.
template <typename T, int D>
__device__ __forceinline__ void merge_row(const StreamParams& p, int block, int r) {
  __shared__ float part[kWarps][D];
  __shared__ float part_ml[kWarps][2];
  constexpr int kPer = D / 32;
  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  int64_t place0, place1, step;  // places of the first and the second segment, and from there on
  int count, b, h;
  if (p.mode == kGrid) {
    const int units = p.row_blocks * p.hkv, u = block;
    b = u / units;
    h = u % p.hkv;
    place0 = (static_cast<int64_t>(u) * p.splits) * p.rows_cta + r;
    step = p.rows_cta;
    place1 = place0 + step;
    count = p.splits;
    r += u % units / p.hkv * p.rows_cta;
  } else {
    const int c = block / p.hkv + 1, shares = *p.shares;
    if (c >= shares) return;
    const int3 at = p.share_unit[c], before = p.share_unit[c - 1];
    if (at.z == 0 || (before.x == at.x && before.y == at.y && before.z > 0)) return;  // no cut, or not its first
    count = 1;  // the share before c, and those from c on that start inside the unit
    for (int i = c;; i += 32) {
      int3 x = make_int3(-1, 0, 0);
      if (i + lane < shares) x = p.share_unit[i + lane];
      const uint32_t same = __ballot_sync(0xffffffffu, x.x == at.x && x.y == at.y && x.z > 0);
      count += same == 0xffffffffu ? 32 : __ffs(~same) - 1;
      if (same != 0xffffffffu) break;
    }
    b = at.x;
    h = block % p.hkv;
    place0 = (2 * (static_cast<int64_t>(c - 1) * p.hkv + h) + 1) * p.rows_cta + r;
    place1 = 2 * (static_cast<int64_t>(c) * p.hkv + h) * p.rows_cta + r;
    step = static_cast<int64_t>(2) * p.hkv * p.rows_cta;
    r += at.y * p.rows_cta;
  }
  const StreamSeq s = sequence_of(p, p.first_seq + b);
  if (r >= s.qlen * p.group) return;
  // warp w: segments w, w + 4, ... with its own maximum; lane: D / 32 dims
  float m = -INFINITY, l = 0.f, x[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) x[j] = 0.f;
#pragma unroll 4
  for (int i = warp; i < count; i += kWarps) {
    const int64_t at = i == 0 ? place0 : place1 + (i - 1) * step;
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * at);
    float y[kPer];
    if constexpr (kPer == 4) {
      *reinterpret_cast<float4*>(y) = *reinterpret_cast<const float4*>(p.part_acc + at * D + lane * 4);
    } else {
      *reinterpret_cast<float2*>(y) = *reinterpret_cast<const float2*>(p.part_acc + at * D + lane * 2);
    }
    const float mn = fmaxf(m, ml.x), base = mn == -INFINITY ? 0.f : mn;
    const float f = ex2(m - base), w = ex2(ml.x - base);
    m = mn;
    l = l * f + ml.y * w;
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[j] = x[j] * f + y[j] * w;
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) part[warp][lane * kPer + j] = x[j];
  if (lane == 0) {
    part_ml[warp][0] = m;
    part_ml[warp][1] = l;
  }
  __syncthreads();
  if (tid >= D) return;
  float mx = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, part_ml[w][0]);
  const float base = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f, y = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const float f = ex2(part_ml[w][0] - base);
    sum += f * part_ml[w][1];
    y += f * part[w][tid];
  }
  const int qt = r / p.group, head = h * p.group + r - qt * p.group;
  static_cast<T*>(p.out)[(s.q0 + qt) * p.os0 + head * p.os1 + tid * p.os2] = from_f32<T>(sum == 0.f ? 0.f : y / sum);
}

// log2 of the sum of exp2 of row g of the unit's `count` partials, by a warp.
__device__ __forceinline__ float merged_lse(const StreamParams& p, int64_t place0, int64_t place1, int64_t step,
                                            int count, int lane) {
  float m = -INFINITY, l = 0.f;
  for (int i = lane; i < count; i += 32) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * (i == 0 ? place0 : place1 + (i - 1) * step));
    const float mn = fmaxf(m, ml.x), base = mn == -INFINITY ? 0.f : mn;
    l = l * ex2(m - base) + ml.y * ex2(ml.x - base);
    m = mn;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, d), l2 = __shfl_xor_sync(0xffffffffu, l, d);
    const float mn = fmaxf(m, m2), base = mn == -INFINITY ? 0.f : mn;
    l = l * ex2(m - base) + l2 * ex2(m2 - base);
    m = mn;
  }
  return l == 0.f ? INFINITY : (m == -INFINITY ? 0.f : m) + log2f(l);
}

// Every token's score gets the sum over the group of exp2(raw - lse), four
// neighbouring tokens a thread.  Bound by its reads of the raw scores (one
// sequence of 131071 tokens, 32/8 heads: 25 MB in 10 us, cold).  The weights have
// to wait for the whole row's sum, so the scores go through memory once; kept in
// the CTA instead where a cluster holds the row.  A CTA works out the sums of its
// rows itself, so it does not wait for the merge, which is in the same launch.
__device__ __forceinline__ void add_scores(const StreamParams& p, int chunk, int chunks, int h, int seq, float* lse) {
  const int tid = threadIdx.x;
  const int lane = tid & 31;
  const int b = p.first_seq + seq;
  const StreamSeq s = sequence_of(p, b);
  if (4 * chunk * kThreads >= s.n) return;
  const int64_t row0 = static_cast<int64_t>(b) * p.hq + h * p.group;
  for (int rb = 0; rb * p.rows_cta < p.group; ++rb) {
    int64_t place0 = 0, place1 = 0, step = 0;
    int count = 0;  // of partials; none: one CTA had the unit
    if (p.mode == kGrid) {
      if (p.splits > 1) {
        place0 = ((static_cast<int64_t>(seq) * p.row_blocks + rb) * p.hkv + h) * p.splits * p.rows_cta;
        step = p.rows_cta;
        place1 = place0 + step;
        count = p.splits;
      }
    } else {  // the shares that start inside the unit, and the one before them
      const int shares = *p.shares;
      int first = 0, inside = 0;
      for (int i = 0; i < shares; i += kThreads) {
        int3 x = make_int3(INT_MAX, 0, 0);
        if (i + tid < shares) x = p.share_unit[i + tid];
        const bool in = x.x == seq && x.y == rb && x.z > 0;
        first += __syncthreads_count(x.x < seq || (x.x == seq && (x.y < rb || (x.y == rb && x.z == 0))));
        inside += __syncthreads_count(in);
      }
      if (inside > 0) {
        place0 = (2 * (static_cast<int64_t>(first - 1) * p.hkv + h) + 1) * p.rows_cta;
        place1 = 2 * (static_cast<int64_t>(first) * p.hkv + h) * p.rows_cta;
        step = static_cast<int64_t>(2) * p.hkv * p.rows_cta;
        count = 1 + inside;
      }
    }
    const int rows = min(p.rows_cta, p.group - rb * p.rows_cta);
    for (int r = tid >> 5; r < rows; r += kWarps) {
      const float x = count > 0 ? merged_lse(p, place0 + r, place1 + r, step, count, lane)
                                : p.row_lse[row0 + rb * p.rows_cta + r];
      if (lane == 0) lse[rb * p.rows_cta + r] = x;
    }
  }
  __syncthreads();
  const bool grid = p.mode == kGrid;
  const int64_t raw_tokens = grid ? p.raw_tokens : unit_tiles(p, s, p.rows_cta) * kTok;
  const int64_t raw_at = grid ? seq * raw_tokens : p.raw_start[seq];
  if (raw_at + raw_tokens > p.raw_room) {
    if (tid == 0) atomicOr(p.status, FD_STATUS_BAD_BLOCK_ID);
    return;
  }
  const float* raw = p.raw + raw_at * p.hq + h * p.group * raw_tokens;
  for (int at = 4 * (chunk * kThreads + tid); at < s.n; at += 4 * chunks * kThreads) {
    const int64_t id =  // four tokens: one page
        load_index(p.bt, p.bt64, b * p.bts0 + static_cast<int64_t>(at >> p.bs_log2) * p.bts1);
    if (id < 0 || id >= p.num_blocks) continue;
    float* slot = p.scores + id * p.scs0 + h * p.scs1 + (at & ((1 << p.bs_log2) - 1)) * p.scs2;
    float old[4], w[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.score_vec) {
      *reinterpret_cast<float4*>(old) = *reinterpret_cast<const float4*>(slot);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) old[i] = slot[i * p.scs2];
    }
#pragma unroll 4
    for (int g = 0; g < p.group; ++g) {
      const float4 x = *reinterpret_cast<const float4*>(raw + g * raw_tokens + at);
      const float y = lse[g];
      w[0] += ex2(x.x - y);
      w[1] += ex2(x.y - y);
      w[2] += ex2(x.z - y);
      w[3] += ex2(x.w - y);
    }
    if (p.score_vec && at + 4 < s.n) {
      *reinterpret_cast<float4*>(slot) = make_float4(old[0] + w[0], old[1] + w[1], old[2] + w[2], old[3] + w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at + i < s.n) slot[i * p.scs2] = at + i == s.n - 1 ? w[i] : old[i] + w[i];
    }
  }
}

// Grid: (`merges` units, rows).
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) stream_merge_kernel(const __grid_constant__ StreamParams p) {
  pdl_wait();
  pdl_launch_dependents();
  merge_row<T, D>(p, blockIdx.x, blockIdx.y);
}

// The same with scores, in one launch (one sequence of 131071 tokens: 108 us, 113
// with a launch each): CTAs for `merges` units x `rows` of them, then for `chunks`
// x KV heads x sequences.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads)
    stream_finish_kernel(const __grid_constant__ StreamParams p, int merges, int rows, int chunks) {
  extern __shared__ float lse[];  // [group]
  pdl_wait();
  pdl_launch_dependents();
  int block = blockIdx.x;
  if (block < merges * rows) {
    merge_row<T, D>(p, block / rows, block % rows);
    return;
  }
  block -= merges * rows;
  const int unit = block / chunks;
  add_scores(p, block - unit * chunks, chunks, unit % p.hkv, unit / p.hkv, lse);
}

struct StreamPlan {
  int m16;         // 16-row tiles per CTA: 1 or 2
  int row_blocks;  // of the longest queries announced
  bool prompt;     // many rows: prompt_attention, where it takes the layout
  int64_t max_query;
  int64_t raw_tokens;  // of a table's row, or of a cluster's CTA
  int64_t raw_room;    // tokens of all sequences of a launch
  int mode;          // kCluster, kGrid or kShares
  int splits;        // CTAs of a unit, of a cluster or grid
  int rows_most;     // of a cluster's unit
  size_t more_smem;  // of a cluster's CTA
  int ctas;          // grid of kShares
  int parts;         // places of partials
  // scratch: (kShares) where each CTA's share starts, and their number; the
  // partials; for scores the rows' lse, (kShares) where each sequence's raw
  // scores start, and raw scores
  size_t meta_bytes, ml_bytes, acc_bytes, lse_bytes, start_bytes, raw_bytes;
  size_t bytes() const { return meta_bytes + ml_bytes + acc_bytes + lse_bytes + start_bytes + raw_bytes; }
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
  if (a->num_seqs > 65535 || a->num_kv_heads > 65535 || a->num_q_heads / a->num_kv_heads > kGroupMost ||
      static_cast<int64_t>(a->max_blocks_per_seq) * a->block_size > 0x3fffffff)
    return FD_ERR_UNSUPPORTED;
  if (!scored) {
    if (a->window < 1 || a->sinks < 0 || a->max_query_len < 1 || a->num_tokens < 0)
      return FD_ERR_INVALID_ARGUMENT;
    if (!a->query_start_loc && a->num_tokens != a->num_seqs) return FD_ERR_INVALID_ARGUMENT;
  }
  const int64_t tokens = scored ? a->num_seqs : std::max(a->num_tokens, a->num_seqs);
  if (tokens * a->num_q_heads > 0x3fffffff) return FD_ERR_UNSUPPORTED;
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
  const int64_t slots = 2 * sms;  // two CTAs fit an SM
  // Which kernel: by their times in us, as measured with 2 to 32 query heads a
  // KV head, 1 to 16 sequences and 4 to 256 queries at a window of 2048.  The
  // prompt kernel takes 6 + 1.9 a tile of 128 keys for each round of 256-row
  // blocks over the SMs (16 sequences, 8 KV heads: 41 us for 64 rows, 93 for
  // 512); this one 12 + 2.4 for every 16-token tile of its busiest warp (88 and
  // 490 there), 1.7 with heads of 64 (24 sequences' drafts: 20, 27 by the prompt
  // kernel).  Few rows of few sequences against a long window go to this one,
  // which splits the keys (1 sequence, 2 KV heads, 128 rows: 17 us, 38).
  if (!scored && rows > 16) {
    const int64_t blocks = (rows + 255) / 256 * a->num_kv_heads * a->num_seqs;
    const int64_t keys = std::min(cap, std::min<int64_t>(a->window, cap) +
                                           std::min<int64_t>(a->sinks, cap) + 256 / group + 2 * a->block_size);
    const double prompt_us =
        static_cast<double>((blocks + sms - 1) / sms) * (6 + 1.9 * static_cast<double>((keys + 127) / 128));
    const double split_us = 12 + (a->head_dim == 128 ? 2.4 : 1.7) * static_cast<double>(units * tiles) /
                                     static_cast<double>(kWarps * slots);
    pl.prompt = prompt_us < split_us;
  }
  const size_t q_rows = static_cast<size_t>(tokens) * a->num_q_heads;
  pl.raw_tokens = (cap + kTok - 1) / kTok * kTok;
  const int64_t row_most = std::min<int64_t>(rows, per);
  // Few units with short runs: the splits of each merge inside a cluster, with
  // no second launch (one token of one sequence: 9.2 us, 14.4 with partials).
  const int64_t in_cluster = std::min<int64_t>(tiles / (2 * kWarps), kMaxCluster);
  if (in_cluster > 1 && units * in_cluster <= slots) {
    const int64_t run = std::max<int64_t>((tiles + in_cluster - 1) / in_cluster, 2 * kWarps) * kTok;
    const size_t raw = scored ? static_cast<size_t>(run) * row_most * sizeof(float) : 0;
    // one CTA an SM if two do not fit: then clusters of 8 leave some SMs of a
    // GPC idle, and three quarters of them have to do
    const size_t base = a->head_dim == 128 ? (pl.m16 == 1 ? split_smem_bytes<128, 1>() : split_smem_bytes<128, 2>())
                                           : (pl.m16 == 1 ? split_smem_bytes<64, 1>() : split_smem_bytes<64, 2>());
    const size_t more = raw + receive_bytes(static_cast<int>(in_cluster), static_cast<int>(row_most), a->head_dim);
    const bool fits = 2 * (base + more + 1024) <= 228 * 1024 || units * in_cluster <= sms * 3 / 4;
    if (fits && run <= kClusterRun && raw <= kRawBytes) {
      pl.mode = kCluster;
      pl.rows_most = static_cast<int>(row_most);
      pl.splits = static_cast<int>(in_cluster);
      pl.more_smem = more;
      pl.raw_tokens = run;
      return pl;
    }
  }
  // A wave of CTAs with kGridRun tiles each at most: a grid of equal splits, which
  // needs no count of the batch's tiles first (24 sequences' drafts: 20 us,
  // 31 as shares).  More: shares.
  const int64_t even = std::max<int64_t>(std::min<int64_t>(slots / units, tiles / (2 * kWarps)), 1);
  if (units <= slots && (tiles + even - 1) / even <= kGridRun && a->num_seqs <= kMaxListed) {
    pl.mode = kGrid;
    pl.splits = static_cast<int>(even);
    pl.parts = static_cast<int>(units * even);
  } else {
    pl.mode = kShares;
    pl.splits = 1;
    const int64_t of_head = units / a->num_kv_heads * tiles;
    pl.ctas = static_cast<int>(std::min<int64_t>(std::max<int64_t>(of_head / kMinShare, 1),
                                                 std::max<int64_t>(slots / a->num_kv_heads, 1)) *
                               a->num_kv_heads);
    pl.parts = 2 * pl.ctas;
  }
  auto padded = [](size_t x) { return (x + 15) & ~size_t(15); };
  pl.meta_bytes = padded(pl.ctas * sizeof(int3) + sizeof(int));
  pl.ml_bytes = static_cast<size_t>(pl.parts) * per * 2 * sizeof(float);
  pl.acc_bytes = static_cast<size_t>(pl.parts) * per * a->head_dim * sizeof(float);
  if (scored) {
    pl.lse_bytes = padded(q_rows * sizeof(float));
    // Raw scores of the tables' tokens, but of no more than twice the cache's (no
    // two sequences share a page; whole tiles): block tables are as wide as the
    // longest context allowed (64 sequences of 500 tokens and 32 heads under
    // tables for 131072: 14 MB, not 1080).
    const int64_t seqs = std::min(a->num_seqs, kMaxListed);
    pl.raw_room = seqs * pl.raw_tokens;
    if (pl.mode == kShares) {
      pl.raw_room = std::min(pl.raw_room, 2 * static_cast<int64_t>(a->num_blocks) * a->block_size + seqs * kTok);
      pl.start_bytes = padded(seqs * sizeof(int64_t));
    }
    pl.raw_bytes = static_cast<size_t>(pl.raw_room) * a->num_q_heads * sizeof(float);
  }
  return pl;
}

template <typename T, int D, int kM>
int launch_split(const StreamParams& p, const StreamPlan& pl, cudaStream_t stream) {
  auto kern = stream_split_kernel<T, D, kM>;
  const size_t list = pl.mode == kShares ? (p.num_seqs + 1) * (sizeof(int64_t) + sizeof(int)) : 0;
  const size_t smem = split_smem_bytes<D, kM>() + pl.more_smem + list;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e =
      allow_smem(done, reinterpret_cast<const void*>(kern),
                 split_smem_bytes<D, kM>() + kRawBytes + receive_bytes(kMaxCluster, 16 * kM, D), p.device);
  if (e != cudaSuccess) return cuda_status(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = pl.mode == kShares ? dim3(pl.ctas) : dim3(pl.splits, p.hkv * pl.row_blocks, p.num_seqs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = pl.splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pl.mode == kCluster ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p));
}

template <typename T, int D>
int launch_typed(const StreamParams& p, const StreamPlan& pl, cudaStream_t stream) {
  if (p.scores && pl.mode != kCluster) {  // a sum per head of the group: 64 KB for the greatest one
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(done, reinterpret_cast<const void*>(stream_finish_kernel<T, D>),
                                     kGroupMost * sizeof(float), p.device);
    if (e != cudaSuccess) return cuda_status(e);
  }
  int rc = pl.m16 == 1 ? launch_split<T, D, 1>(p, pl, stream) : launch_split<T, D, 2>(p, pl, stream);
  if (rc != FD_OK || pl.mode == kCluster) return rc;
  const int64_t merges = pl.mode == kGrid ? (pl.splits == 1 ? 0 : static_cast<int64_t>(p.num_seqs) * p.hkv * pl.row_blocks)
                                          : pl.ctas - p.hkv;
  // rows of a row block: all of them where queries may be longer than announced
  const int64_t rows = p.qstart ? p.rows_cta : std::min<int64_t>(p.rows_cta, p.group);
  if (!p.scores) {
    if (merges > 0)
      rc = cuda_status(launch_pdl(stream_merge_kernel<T, D>,
                                  dim3(static_cast<unsigned>(merges), static_cast<unsigned>(rows)), dim3(kThreads), 0,
                                  stream, p));
    return rc;
  }
  // A CTA goes over 2 x 512 tokens of the longest sequence there can be, or more
  // where that would be many CTAs (of 64 sequences of 500 tokens under tables for
  // 131072, 65536 of which nearly all return at once: 106 us, 43 with narrow ones).
  const int64_t most = std::max<int64_t>(1, (1 << 15) / (static_cast<int64_t>(p.hkv) * p.num_seqs));
  const int64_t longest = std::min(pl.raw_tokens, static_cast<int64_t>(p.num_blocks) << p.bs_log2);
  const int64_t chunks = std::min<int64_t>((longest + 8 * kThreads - 1) / (8 * kThreads), most);
  const int64_t blocks = merges * rows + chunks * p.hkv * p.num_seqs;
  return cuda_status(launch_pdl(stream_finish_kernel<T, D>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads),
                                static_cast<size_t>(p.group) * sizeof(float), stream, p, static_cast<int>(merges),
                                static_cast<int>(rows), static_cast<int>(chunks)));
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
  p.group_magic = static_cast<uint32_t>(((uint64_t(1) << 32) + p.group - 1) / p.group);
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
  p.rows_most = pl.rows_most;
  p.rows_cta = 16 * pl.m16;
  p.score_vec = scored && reinterpret_cast<uintptr_t>(a->scores) % 16 == 0 && a->scores_stride[0] % 4 == 0 &&
                a->scores_stride[1] % 4 == 0 && a->scores_stride[2] == 1;
  p.mode = pl.mode;
  auto aligned = [](const void* base, const int64_t* st) {
    return reinterpret_cast<uintptr_t>(base) % 16 == 0 && st[0] % 8 == 0 && st[1] % 8 == 0 &&
           st[2] % 8 == 0 && st[3] == 1;
  };
  p.vec = aligned(a->k_cache, a->k_stride) && aligned(a->v_cache, a->v_stride);
  auto aligned3 = [](const void* base, const int64_t* st) {
    return reinterpret_cast<uintptr_t>(base) % 16 == 0 && st[0] % 8 == 0 && st[1] % 8 == 0 && st[2] == 1;
  };
  p.q_vec = aligned3(a->q, a->q_stride);
  p.out_vec = aligned3(a->out, a->out_stride);
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  char* at = static_cast<char*>(a->scratch);
  if (pl.mode != kCluster) {
    p.share_unit = reinterpret_cast<int3*>(at);
    p.shares = reinterpret_cast<int*>(p.share_unit + pl.ctas);
    at += pl.meta_bytes;
    p.part_ml = reinterpret_cast<float*>(at);
    at += pl.ml_bytes;
    p.part_acc = reinterpret_cast<float*>(at);
    at += pl.acc_bytes;
    p.row_lse = reinterpret_cast<float*>(at);
    at += pl.lse_bytes;
    p.raw_start = reinterpret_cast<int64_t*>(at);
    p.raw = reinterpret_cast<float*>(at + pl.start_bytes);
  }
  p.raw_tokens = pl.raw_tokens;
  p.raw_room = pl.raw_room;
  const uint64_t group_blocks = (p.group + p.rows_cta - 1) / p.rows_cta;
  p.blocks_magic = group_blocks > 1 ? UINT64_MAX / group_blocks + 1 : 0;
  p.status = status;
  p.device = dev->device;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const bool bf16 = a->dtype == FD_DTYPE_BF16;
  if (pl.prompt && prompt_attention(p, bf16, a->head_dim, pl.max_query, dev->num_sms, stream, &rc)) return rc;
  for (p.first_seq = 0; rc == FD_OK && p.first_seq < a->num_seqs; p.first_seq += kMaxListed) {
    p.num_seqs = std::min(a->num_seqs - p.first_seq, kMaxListed);
    if (a->head_dim == 128) {
      rc = bf16 ? launch_typed<__nv_bfloat16, 128>(p, pl, stream) : launch_typed<__half, 128>(p, pl, stream);
    } else {
      rc = bf16 ? launch_typed<__nv_bfloat16, 64>(p, pl, stream) : launch_typed<__half, 64>(p, pl, stream);
    }
  }
  return rc;
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

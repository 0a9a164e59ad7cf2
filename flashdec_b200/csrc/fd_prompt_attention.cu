// fd_window_attention for many queries per sequence (prompt chunks), on the
// 5th-generation tensor cores.
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "../../include/flashdec_b200.h"
#include "fd_host.h"
#include "fd_ptx.cuh"
#include "fd_stream.h"
#include "fd_stream.cuh"
#include "fd_tile.cuh"

namespace fd {
namespace {

// One item: 256 query rows (row = query x head of the group) of a (sequence, KV
// head) as two groups of 128, against the list of cache pages they see in
// tiles of 128 keys.  Per group: S = Q K^T (M 128, N 128) into TMEM, one thread
// per row takes it from there and writes P = exp2(S - m) back over it in the
// cache's type, in two halves, and O += P V accumulates in TMEM with P as the
// TMEM operand, the first half while the second is being computed.  The two
// groups alternate, so the tensor pipe works on one while the other does its
// softmax.  With two S buffers of 64 keys a group never waits for its own
// products, but a product of N 64 takes nearly as long as one of N 128 (it
// reads the same Q operand): 428 us on an 8k prompt against 378 at that point.
//
// One CTA an SM takes every gridDim.x-th item: while the softmax threads finish
// one, the K and V tiles and the queries of the next are on their way: 58 us for
// ragged prompts of 9 tiles an item, against 65 with a CTA for each item (whose
// start and end were a sixth of its time or more); 314 against 306 us for an 8k
// prompt of 17 tiles an item, which pays for the longer code instead (both
// figures of that time).
//
// What bounds it: the latency of a tile.  8k queries, window 2048, 32/8 heads:
// 241 GFLOP in 322-337 us, 0.44-0.46 of the rate of a large library product, with
// the tensor pipe busy 37 % of the time, the exponentials' pipe 38 % and the issue
// slots 32 %; 23, 25 and 25 % on ragged prompts of 9 tiles an item.  A group
// waits for its S, then for both halves of the scores, and has all 128 of them
// masked and their maximum found before the first exponential, and its
// products idle meanwhile; two groups do not cover that.  Some 200 bytes of a
// thread's state are spilled around the tile loop.
//
// K and V tiles are loaded again for every row block, from L2 mostly: the 8k
// prompt moves 1.2 GB through L2 and reads 146 MB of DRAM, where q, K and V are
// 101.
//
//   warp 0      TMA producer: K and V tiles alternate through a ring of slots
//   warp 1      issues the tcgen05.mma (one thread)
//   warps 2, 3  V tiles with keys that some row does not see, or with a page
//               that is not in the cache: rows that no row sees are zeroed, and
//               so is an infinity or NaN in another (a weight of 0 times it
//               would be NaN), which marks the item: its epilogue adds what the
//               rows that see it get
//   warps 4-7   softmax and epilogue of rows 0-127
//   warps 8-11  the same of rows 128-255
//
// TMEM columns: S/P of group g at 128 g, O of group g at 256 + 128 g.
constexpr int kPromptThreads = 384;
constexpr int kRows = 256;
constexpr int kKeys = 128;  // of a tile
constexpr int kMostSeqs = 256;  // of a launch

template <int D>
struct PromptSmem {
  static constexpr int kSlots = D == 128 ? 4 : 8;
  static constexpr uint32_t kHalf = 128 * 128;             // [128 rows][64 dims]
  static constexpr uint32_t kOperand = (D / 64) * kHalf;   // a Q group or a K or V tile
  static constexpr uint32_t kRing = 2 * kOperand;          // offset: two Q groups first
  static constexpr uint32_t kBars = kRing + kSlots * kOperand;
  static constexpr uint32_t kGood = kBars + 512;           // keys of 16 tiles whose page is in the cache
  static constexpr uint32_t kList = kGood + 256;           // row blocks before each sequence's
  static constexpr uint32_t kStage = kList + 4 * (kMostSeqs + 4);  // output rows, 4 KB a softmax warp
  static constexpr size_t kBytes = kStage + 8 * 4096 + 1024;       // and alignment
};

// 64 consecutive fp32 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&v)[64]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
#define R4(i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define R16(i) R4(i), R4(i + 4), R4(i + 8), R4(i + 12)
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : R16(0), R16(16), R16(32), R16(48)
      : "r"(taddr)
      : "memory");
#undef R16
#undef R4
}

// Two fp32 operations an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
        "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}

// 32 columns of this thread's TMEM lane <- registers.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// The products are issued by a whole warp of which one elected lane acts: the
// operands stay in uniform registers (from one lane of a divergent branch
// each product first moved its descriptors there, about 80 cycles a product).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
  return on;
}
// D[tmem] (+)= A[smem desc] x B[smem desc], by the lane with `on`.
__device__ __forceinline__ void umma_ss(uint32_t on, uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], %2, %3, %4, p;\n\t}\n" ::"r"(on),
      "r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// D[tmem] (+)= A[tmem] x B[smem desc], by the lane with `on`.
__device__ __forceinline__ void umma_ts(uint32_t on, uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], %3, %4, p;\n\t}\n" ::"r"(on),
      "r"(d_tmem), "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void umma_done(uint32_t on, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}\n" ::"r"(on),
      "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }

// The greater magnitude of each 16-bit half; NaN wins.
template <typename T>
__device__ __forceinline__ uint32_t max_abs(uint32_t a, uint32_t b) {
  uint32_t d;
  b &= 0x7fff7fffu;
  if constexpr (std::is_same<T, __half>::value) {
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  } else {
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  }
  return d;
}

// The first x bits, clamped to [0, 32].
__device__ __forceinline__ uint32_t low_bits(int x) {
  return x <= 0 ? 0u : (x >= 32 ? 0xffffffffu : (1u << x) - 1u);
}

// Whether the predicate holds for any of `threads` threads, which all wait here.
__device__ __forceinline__ bool barrier_any(int id, int threads, bool x) {
  uint32_t y;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(y)
      : "r"(id), "r"(threads), "r"(x ? 1u : 0u)
      : "memory");
  return y != 0;
}

// Wait for a barrier's phase whatever the abort flag says: copies in flight
// have to land before the CTA's shared memory is given up.
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 < kWaitLimitNs) {
  }
}

// S of the keys that are not `good` (4 x 32 bits) to -inf, for this thread's
// row, before the softmax takes it: in the mask there it cost the tiles
// without such keys 3 to 7 % (registers).
__device__ __noinline__ void drop_bad_keys(uint32_t s_addr, const uint32_t* good) {
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    const uint32_t on = good[c];
    if (on == ~0u) continue;
    float x[32];
    tmem_ld32(s_addr + 32 * c, x);
    uint32_t y[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) y[i] = (on >> i) & 1u ? __float_as_uint(x[i]) : 0xff800000u;
    tmem_st32(s_addr + 32 * c, y);
  }
  tmem_wait_st();
}

// What a row sees, in list coordinates (key i of tile j is list place 128 j +
// i): [0, sink_end) and [w0, w1].
struct RowView {
  int sink_end, w0, w1;
};
__device__ __forceinline__ RowView view_of(const StreamParams& p, const StreamRange& rg, int pos) {
  const int shift = (rg.sink_pages - rg.win_page) << p.bs_log2;
  RowView v;
  v.sink_end = min(p.sinks, pos + 1);
  v.w0 = max(pos - p.window + 1, 0) + shift;
  v.w1 = pos + shift;
  return v;
}

// Every row of the block sees list places [at, at + n).
__device__ __forceinline__ bool interior(const StreamParams& p, const StreamRange& rg, int at, int n) {
  const RowView first = view_of(p, rg, rg.pos0), last = view_of(p, rg, rg.pos1);
  return rg.pos0 >= 0 && (at + n <= first.sink_end || (at >= last.w0 && at + n - 1 <= first.w1));
}

// What the infinities and NaN that were zeroed in the item's V tiles give to
// the warp's rows [row0, row0 + rows), added to their outputs: only the tiles
// that some row sees in part are gone over (a few, whatever the window), a
// token at a time with a lane's D / 32 dims of it.  A weight is above 0 unless
// its score is -inf, so the outcome is an infinity or NaN whatever its size.
template <typename T, int D>
__device__ __noinline__ void add_nonfinite(const StreamParams& p, int b, int h, int rb, int row0, int rows, int lane) {
  constexpr int kN = D / 32;
  const StreamSeq s = sequence_of(p, b);
  const StreamRange rg(s, rb * kRows, min(rb * kRows + kRows, s.qlen * p.group), p.group, p.window, p.sinks, p.bs_log2);
  const RowView view = view_of(p, rg, s.n - s.qlen + (row0 + min(lane, rows - 1)) / p.group);  // of row `lane`
  uint32_t up[kN], down[kN];  // bit r: row r gets +inf, -inf; both: NaN
#pragma unroll
  for (int i = 0; i < kN; ++i) up[i] = down[i] = 0u;
  const int list = rg.pages << p.bs_log2;
#pragma unroll 1
  for (int place = 0; place < list; ++place) {
    if (place % kKeys == 0 && interior(p, rg, place, kKeys)) {
      place += kKeys - 1;
      continue;
    }
    const bool sees = place < view.sink_end || (place >= view.w0 && place <= view.w1);
    const uint32_t on = __ballot_sync(0xffffffffu, lane < rows && sees);
    if (on == 0u) continue;
    const int64_t id =
        load_index(p.bt, p.bt64, b * p.bts0 + static_cast<int64_t>(rg.page(place >> p.bs_log2)) * p.bts1);
    if (id < 0 || id >= p.num_blocks) continue;
    const int off = place & ((1 << p.bs_log2) - 1);
    const T* const k = static_cast<const T*>(p.k) + id * p.ks0 + h * p.ks1 + off * p.ks2;
    const T* const v = static_cast<const T*>(p.v) + id * p.vs0 + h * p.vs1 + off * p.vs2;
    float x[kN];
    bool odd = false;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      x[i] = to_f32<T>(v[(lane + 32 * i) * p.vs3]);
      odd |= !isfinite(x[i]);
    }
    if (!__any_sync(0xffffffffu, odd)) continue;
    uint32_t none = 0u;  // rows where the token's weight is 0
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
      if (!((on >> r) & 1u)) continue;
      const int qt = (row0 + r) / p.group, head = h * p.group + (row0 + r) - qt * p.group;
      const T* const q = static_cast<const T*>(p.q) + (s.q0 + qt) * p.qs0 + head * p.qs1;
      float y = 0.f;
#pragma unroll
      for (int i = 0; i < kN; ++i) y += to_f32<T>(q[(lane + 32 * i) * p.qs2]) * to_f32<T>(k[(lane + 32 * i) * p.ks3]);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) y += __shfl_xor_sync(0xffffffffu, y, d);
      if (y * p.scale_log2 == -INFINITY) none |= 1u << r;
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if (isfinite(x[i])) continue;
      up[i] |= x[i] < 0.f ? none : on;  // NaN: both
      down[i] |= x[i] > 0.f ? none : on;
    }
  }
#pragma unroll 1
  for (int r = 0; r < rows; ++r) {
    const int qt = (row0 + r) / p.group, head = h * p.group + (row0 + r) - qt * p.group;
    T* const out = static_cast<T*>(p.out) + (s.q0 + qt) * p.os0 + head * p.os1;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const bool u = (up[i] >> r) & 1u, d = (down[i] >> r) & 1u;
      if (!u && !d) continue;
      T* const y = out + (lane + 32 * i) * p.os2;
      *y = from_f32<T>(to_f32<T>(*y) + (u ? INFINITY : 0.f) + (d ? -INFINITY : 0.f));
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    prompt_kernel(const __grid_constant__ StreamParams p, const __grid_constant__ CUtensorMap tmap_k,
                  const __grid_constant__ CUtensorMap tmap_v, const int4 kperm, const int4 vperm) {
  using SM = PromptSmem<D>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kSlots = SM::kSlots;
  constexpr int kHalves = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::kBars);
  uint64_t* full = bars;                // [slot] TMA bytes
  uint64_t* empty = full + kSlots;      // [slot] the products that read it are done
  uint64_t* v_ready = empty + kSlots;   // [slot] V checked
  uint64_t* q_ready = v_ready + kSlots; // [group]
  uint64_t* s_full = q_ready + 2;       // [group] S in TMEM
  uint64_t* p_ready = s_full + 2;       // [group] P in TMEM (and O rescaled)
  uint64_t* pv_done = p_ready + 2;      // [group] O holds the tile
  uint64_t* drained = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  // [8] by the CTA's count of items with keys: count + 1 where values of such an
  // item were zeroed (add_nonfinite).  The loads are a few items ahead of the
  // group that works; the other one may lag (items of one group go past it),
  // so a group says how many it has `seen`, and a place that is taken again
  // before both have read it marks all later items.
  volatile int* marked = abort_flag + 1;
  volatile int* seen = marked + 8;  // [group]
  volatile int* all_marked = seen + 2;
  auto mark = [&](int count) {
    if (count >= 8 && (seen[0] < count - 7 || seen[1] < count - 7)) {
      *all_marked = 1;
      __threadfence_block();
    }
    marked[count & 7] = count + 1;
  };
  // Raised for good at the first page that is not in the cache: only then the
  // softmax looks at what good_keys says.
  volatile int* any_bad = all_marked + 1;
  // [16][4 x 32 bits] by the CTA's count of tiles: the tile's keys whose page is
  // in the cache.  A tile's product with V waits for those who read this, and
  // the producer is kSlots / 2 tiles ahead of them at most.
  uint32_t* const good_keys = reinterpret_cast<uint32_t*>(smem + SM::kGood);
  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  int* const upto = reinterpret_cast<int*>(smem + SM::kList);  // [num_seqs + 1] items before a sequence's

  if (tid == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), 1);
      mbar_init(smem_u32(&v_ready[i]), 2);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(smem_u32(&q_ready[g]), 128);
      mbar_init(smem_u32(&s_full[g]), 1);
      mbar_init(smem_u32(&p_ready[g]), 128);
      mbar_init(smem_u32(&pv_done[g]), 1);
    }
    mbar_init(smem_u32(drained), 1);
    fence_mbar_init();
    *abort_flag = 0;
    for (int i = 0; i < 8; ++i) marked[i] = 0;
    seen[0] = seen[1] = *all_marked = *any_bad = 0;
  }
  if (warp == 3) tmem_alloc(smem_u32(tmem_slot), 512);
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tmap_k);
    prefetch_tensormap(&tmap_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  // ---- the items: row blocks of a (sequence, KV head) are neighbours ----
  for (int i = tid; i < p.num_seqs; i += kPromptThreads)
    upto[i + 1] = (sequence_of(p, p.first_seq + i).qlen * p.group + kRows - 1) / kRows * p.hkv;
  __syncthreads();
  if (warp == 0) {
    int sum = 0;
    for (int i = 0; i < p.num_seqs; i += 32) {
      int x = i + lane < p.num_seqs ? upto[i + lane + 1] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      if (i + lane < p.num_seqs) upto[i + lane + 1] = sum + x;
      sum += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) upto[0] = 0;
  }
  __syncthreads();
  const int items = upto[p.num_seqs];
  struct Item {
    int b, h, rb, rows_all;
    StreamSeq s;
  };
  auto item_at = [&](int i) {
    Item im;
    int lo = 0, hi = p.num_seqs;  // upto[lo] <= i < upto[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (upto[mid] <= i) {
        lo = mid;
      } else {
        hi = mid;
      }
    }
    im.b = p.first_seq + lo;
    im.s = sequence_of(p, im.b);
    im.rows_all = im.s.qlen * p.group;
    const int blocks = (im.rows_all + kRows - 1) / kRows;
    im.h = (i - upto[lo]) / blocks;
    im.rb = (i - upto[lo]) - im.h * blocks;
    return im;
  };
  const int bs = 1 << p.bs_log2;
  const int tile_pages = kKeys >> p.bs_log2;
  auto range_of = [&](const Item& im) {
    return StreamRange(im.s, im.rb * kRows, min(im.rb * kRows + kRows, im.rows_all), p.group, p.window, p.sinks,
                       p.bs_log2);
  };

  // 128 x 88 + 256 x 208 registers: the launch's 384 x 168
  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 0) {
    // ======== producer: lane = (page of the tile, 64-dim half) ========
    const uint64_t policy = l2_policy_evict_first();
    const int my_half = lane & (kHalves - 1);
    const int my_page = lane / kHalves;
    uint32_t n = 0;  // tiles of either kind issued so far
    bool ok = true;
    for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const Item im = item_at(item);
      const StreamRange rg = range_of(im);
      const int tiles = (rg.pages + tile_pages - 1) / tile_pages;
      auto look = [&](int t) -> int64_t {  // -2: no page there
        const int i = t * tile_pages + my_page;
        if (my_page >= tile_pages || i >= rg.pages) return -2;
        return load_index(p.bt, p.bt64, im.b * p.bts0 + static_cast<int64_t>(rg.page(i)) * p.bts1);
      };
      int64_t next = look(0);
      for (int t = 0; ok && t < tiles; ++t) {
        const int64_t id = next;
        if (t + 1 < tiles) next = look(t + 1);
        const bool valid = id >= 0 && id < p.num_blocks;
        const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, valid));
        const uint32_t bad = __ballot_sync(0xffffffffu, id != -2 && !valid);
        if (bad != 0u && lane == 0) {
          *any_bad = 1;
          atomicOr(p.status, FD_STATUS_BAD_BLOCK_ID);
        }
        if (lane < 4) {
          uint32_t good = ~0u;
          if (bad != 0u) {  // 8 keys: never more than a page
#pragma unroll 1
            for (int i = 0; i < 32; i += 8)
              if ((bad >> (((32 * lane + i) >> p.bs_log2) * kHalves)) & 1u) good &= ~(0xffu << i);
          }
          good_keys[4 * ((n >> 1) & 15) + lane] = good;
        }
        __syncwarp();
        for (int kind = 0; ok && kind < 2; ++kind, ++n) {
          const int slot = n % kSlots;
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&empty[slot]), ((n / kSlots) & 1) ^ 1, p.status, abort_flag));
          if (!ok) break;
          const uint32_t bar = smem_u32(&full[slot]);
          if (lane == 0) mbar_arrive_expect_tx(bar, boxes * (bs * 128));
          __syncwarp();
          if (valid) {
            const int4 perm = kind ? vperm : kperm;
            const int blk = static_cast<int>(id);
            tma_load_4d(smem_u32(smem + SM::kRing + slot * SM::kOperand + my_half * SM::kHalf) + my_page * (bs * 128),
                        kind ? &tmap_v : &tmap_k, bar, my_half * 64, tmap_coord(perm.x, im.h, blk),
                        tmap_coord(perm.y, im.h, blk), tmap_coord(perm.z, im.h, blk), policy);
          }
        }
      }
    }
    if (*abort_flag) {
      for (uint32_t i = n > kSlots ? n - kSlots : 0; i < n; ++i)
        drain_wait(smem_u32(&full[i % kSlots]), (i / kSlots) & 1);
    }
  } else if (warp == 1) {
    // ======== tcgen05.mma, issued by one elected lane ========
    {
      const uint32_t on = elect_one();
      const uint32_t tm = uniform(tmem);
      constexpr uint32_t kIdO = umma_idesc_f16(kBf16, true, 128, D);
      const uint32_t base = uniform(smem_u32(smem));
      // Operand descriptors by addition: one built for each product (a dozen
      // dependent instructions) kept the tensor pipe waiting for this thread.
      const uint64_t q_desc = umma_smem_desc(base, 16, 1024, 2);
      const uint64_t k_desc = umma_smem_desc(base + SM::kRing, 16, 1024, 2);
      const uint64_t v_desc = umma_smem_desc(base + SM::kRing, SM::kHalf, 1024, 2);
      uint32_t n = 0;                 // next slot
      uint32_t it[2] = {0, 0};        // tiles done, per group
      uint32_t q_round[2] = {0, 0};   // items with keys so far that have the group
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, p.status, abort_flag));
        return ok;
      };
      for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
        const Item im = item_at(item);
        const StreamRange rg = range_of(im);
        const int keys = uniform(rg.pages << p.bs_log2);
        const int tiles = (keys + kKeys - 1) / kKeys;
        const int groups = uniform(im.rows_all - im.rb * kRows > 128 ? 2 : 1);
        if (tiles == 0) continue;
        const uint32_t q_parity[2] = {q_round[0] & 1, q_round[1] & 1};
        q_round[0] += 1;
        q_round[1] += groups == 2 ? 1 : 0;
        auto keys16 = [&](int t) { return (min(kKeys, keys - t * kKeys) + 15) >> 4; };  // of tile t
        auto issue_s = [&](int g, int t, uint32_t slot) {
          const uint32_t idesc = umma_idesc_f16(kBf16, false, 128, 16 * keys16(t));
          const uint64_t qa = q_desc + g * (SM::kOperand >> 4);
          const uint64_t ka = k_desc + slot * (SM::kOperand >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k >> 2) * SM::kHalf + (k & 3) * 32u;
            umma_ss(on, tm + 128 * g, qa + (off >> 4), ka + (off >> 4), idesc, k > 0);
          }
          umma_done(on, smem_u32(&s_full[g]));
        };
#pragma unroll
        for (int g = 0; g < 2; ++g)
          if (g < groups) wait(&q_ready[g], q_parity[g]);
        if (!wait(&full[n % kSlots], (n / kSlots) & 1)) break;
        tc_fence_after();
        for (int g = 0; g < groups; ++g) issue_s(g, 0, n % kSlots);
        umma_done(on, smem_u32(&empty[n % kSlots]));
        ++n;
        for (int t = 0; t < tiles; ++t, n += 2) {  // n: V of tile t
          const uint32_t vs = n % kSlots, ks = (n + 1) % kSlots;
          const bool more = t + 1 < tiles;
          if (!wait(&v_ready[vs], (n / kSlots) & 1)) break;
          if (more && !wait(&full[ks], ((n + 1) / kSlots) & 1)) break;
          const uint64_t va = v_desc + vs * (SM::kOperand >> 4);
          const int k16 = keys16(t);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (g >= groups || !ok) continue;
            const uint32_t pa = tm + 128 * g, oa = tm + 256 + 128 * g;
            if (!wait(&p_ready[g], it[g] & 1)) continue;
            ++it[g];
            tc_fence_after();
            umma_ts(on, oa, pa, va, kIdO, t > 0);
#pragma unroll
            for (int k = 1; k < 8; ++k)
              if (k < k16) umma_ts(on, oa, pa + 8 * k, va + k * 128, kIdO, 1);
            umma_done(on, smem_u32(&pv_done[g]));
            // The tensor pipe takes this warp's products in order: S of the
            // next tile lands on P only after the product above has read it.
            if (more) issue_s(g, t + 1, ks);
          }
          if (!ok) break;
          umma_done(on, smem_u32(&empty[vs]));
          if (more) umma_done(on, smem_u32(&empty[ks]));
        }
        --n;  // no K after the last V
      }
      if (*abort_flag) {  // products in flight still read shared memory and write TMEM
        umma_done(on, smem_u32(drained));
        drain_wait(smem_u32(drained), 0);
      }
    }
    __syncwarp();
  } else if (warp < 4) {
    // ======== V tiles on the edge of what the rows see, two warps ========
    constexpr uint32_t kExp = kBf16 ? 0x7f80u : 0x7c00u;
    uint32_t n = 0;
    bool ok = true;
    for (int item = blockIdx.x, live = -1; ok && item < items; item += gridDim.x) {
      const Item im = item_at(item);
      const StreamRange rg = range_of(im);
      const int tiles = (rg.pages + tile_pages - 1) / tile_pages;
      live += tiles > 0 ? 1 : 0;
      const int shift = (rg.sink_pages - rg.win_page) << p.bs_log2;
      const int list = rg.pages << p.bs_log2;
      // list places that some row of the block sees: [0, s1) and [w0, w1)
      const int s1 = min(rg.sink_end, list), w0 = rg.lo + shift, w1 = min(rg.pos1 + shift + 1, list);
      for (int t = 0; ok && t < tiles; ++t) {
        ++n;  // K
        const int slot = n % kSlots;
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[slot]), (n / kSlots) & 1, p.status, abort_flag));
        if (!ok) break;
        const bool edge = !interior(p, rg, t * kKeys, kKeys);
        const uint4 good4 = *reinterpret_cast<const uint4*>(good_keys + 4 * ((n >> 1) & 15));
        if (edge || (good4.x & good4.y & good4.z & good4.w) != ~0u) {
          uint8_t* v = smem + SM::kRing + slot * SM::kOperand + (lane >> 3) * 128 + (lane & 7) * 16;
          const int end = min(kKeys, (list - t * kKeys + 15) & ~15);
          uint32_t top = 0;  // the largest magnitudes so far, NaN above all
          // 16 keys of a 64-dim half at a time: lane = (key % 4, 16-byte chunk)
#pragma unroll 2
          for (int u = warp - 2; u < kHalves * (end >> 4); u += 2) {
            const int hf = kHalves == 2 ? u & 1 : 0;
            const int k0 = (kHalves == 2 ? u >> 1 : u) * 16;
            const int at = t * kKeys + k0;
            uint4* x = reinterpret_cast<uint4*>(v + hf * SM::kHalf + k0 * 128);
            const uint32_t good = (good_keys[4 * ((n >> 1) & 15) + (k0 >> 5)] >> (k0 & 16)) & 0xffffu;
            if (good == 0xffffu && (at + 16 <= s1 || (at >= w0 && at + 16 <= w1))) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint4 y = x[32 * i];
                top = max_abs<T>(max_abs<T>(max_abs<T>(max_abs<T>(top, y.x), y.y), y.z), y.w);
              }
            } else {
#pragma unroll 1
              for (int i = 0; i < 4; ++i) {
                const int place = at + 4 * i + (lane >> 3);
                if ((place < s1 || (place >= w0 && place < w1)) && ((good >> (4 * i)) & 1u)) {
                  const uint4 y = x[32 * i];
                  top = max_abs<T>(max_abs<T>(max_abs<T>(max_abs<T>(top, y.x), y.y), y.z), y.w);
                } else {
                  x[32 * i] = make_uint4(0u, 0u, 0u, 0u);
                }
              }
            }
          }
          // (a tile that every row sees has its product as it is)
          if (edge && __any_sync(0xffffffffu, nonfinite16(top, kExp))) {
            if (lane == 0) mark(live);
#pragma unroll 1
            for (int u = warp - 2; u < kHalves * (end >> 4); u += 2) {
              uint32_t* x = reinterpret_cast<uint32_t*>(v + (kHalves == 2 ? u & 1 : 0) * SM::kHalf +
                                                        (kHalves == 2 ? u >> 1 : u) * 16 * 128);
#pragma unroll 1
              for (int i = 0; i < 16; ++i) {
                uint32_t* y = x + 128 * (i >> 2) + (i & 3);
                const uint32_t w = *y;
                *y = ((w & kExp) == kExp ? 0u : w & 0xffffu) | ((w >> 16 & kExp) == kExp ? 0u : w & 0xffff0000u);
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(smem_u32(&v_ready[slot]));
        ++n;  // V
      }
    }
  } else {
    // ======== softmax: thread = row = TMEM lane ========
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int g = (warp - 4) >> 2;
    const int gt = tid - 128 - 128 * g;  // row of the group
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_addr = lane_addr + 128 * g, o_addr = lane_addr + 256 + 128 * g;
    // a scale of 0 (uniform weights) stays above it: -inf * 0 is NaN
    const float scale = fmaxf(fabsf(p.scale_log2), 1e-30f);
    const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;  // the scale's sign goes to q
    constexpr int kChunks = D / 8, kRowStep = 128 / kChunks;
    uint8_t* const q_area = smem + g * SM::kOperand + ((gt % kChunks) >> 3) * SM::kHalf;
    // element offset of row r of an item's group, whose first row is the one of
    // query qt0 and head rem0 (a small dividend: one multiplication)
    auto row_at = [&](const Item& x, int qt0, int rem0, int r, int64_t s0, int64_t s1) -> int64_t {
      const int add = p.group == 1 ? r : __umulhi(static_cast<uint32_t>(rem0 + r), p.group_magic);
      return (x.s.q0 + qt0 + add) * s0 + (x.h * p.group + rem0 + r - add * p.group) * s1;
    };
    // The group's queries of item x to its q area: cp.async where they are
    // aligned.  Hardly unrolled: it runs once per item, and unrolled sixteen
    // times its instruction fetches took 14k cycles.
    auto load_q = [&](const Item& x) {
      const int grow0 = x.rb * kRows + 128 * g;
      const int c = gt % kChunks, r0 = gt / kChunks;
      const int qt0 = grow0 / p.group, rem0 = grow0 - qt0 * p.group;
      if (p.q_vec) {
        const T* const src = static_cast<const T*>(p.q) + c * 8;
#pragma unroll 4
        for (int r = r0; r < 128; r += kRowStep) {
          const bool in = grow0 + r < x.rows_all;
          cp_async16(smem_u32(q_area) + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                     src + (in ? row_at(x, qt0, rem0, r, p.qs0, p.qs1) : 0), in ? 16 : 0);
        }
      } else {
#pragma unroll 1
        for (int r = r0; r < 128; r += kRowStep) {
          uint4 y = make_uint4(0u, 0u, 0u, 0u);
          if (grow0 + r < x.rows_all)
            y = gather8(static_cast<const T*>(p.q) + row_at(x, qt0, rem0, r, p.qs0, p.qs1) + c * 8 * p.qs2, p.qs2);
          *reinterpret_cast<uint4*>(q_area + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = y;
        }
      }
      cp_async_commit();
    };
    uint32_t it = 0;
    uint32_t skipped = 0;  // tiles of items without this group
    int live = -1;
    bool here = false;  // the queries of this item are on their way
    Item im = {0, 0, 0, 0, {0, 0, 0}};
    if (static_cast<int>(blockIdx.x) < items) im = item_at(blockIdx.x);
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
      bool ok = true;
      const Item cur = im;
      const StreamRange rg = range_of(cur);
      const int tiles = (rg.pages + tile_pages - 1) / tile_pages;
      live += tiles > 0 ? 1 : 0;
      const bool more = item + static_cast<int>(gridDim.x) < items;
      if (cur.rb * kRows + 128 * g >= cur.rows_all) {  // not a row of this group's
        if (gt == 0) seen[g] = live + 1;
        skipped += tiles;
        if (more) im = item_at(item + gridDim.x);
        continue;
      }
      const int rows_all = cur.rows_all;
      const int grow0 = cur.rb * kRows + 128 * g;
      // ---- q rows into the K-major operand (128B swizzle), 16 bytes a lane ----
      const int c = gt % kChunks, r0 = gt / kChunks;
      if (tiles > 0 && !here) load_q(cur);
      here = false;
      cp_async_wait<0>();
      if (flip && tiles > 0) {  // the chunks this thread brought itself
#pragma unroll 1
        for (int r = r0; r < 128; r += kRowStep) {
          uint4* x = reinterpret_cast<uint4*>(q_area + r * 128 + (((c & 7) ^ (r & 7)) << 4));
          *x = make_uint4(x->x ^ flip, x->y ^ flip, x->z ^ flip, x->w ^ flip);
        }
      }
      // Only for products that wait for it: a phase nobody waits for would let
      // the wait for the next one return at once.
      if (tiles > 0) {
        fence_proxy_async_smem();
        mbar_arrive(smem_u32(&q_ready[g]));
      }

      const int row = grow0 + gt;
      const int qt = min(row, rows_all - 1) / p.group;
      const RowView view = view_of(p, rg, cur.s.n - cur.s.qlen + qt);
      // list places that every row sees: [0, all_s) and [all_0, all_1)
      const RowView row_0 = view_of(p, rg, rg.pos0), row_n = view_of(p, rg, rg.pos1);
      const int all_s = rg.pos0 < 0 ? 0 : row_0.sink_end, all_0 = row_n.w0, all_1 = rg.pos0 < 0 ? 0 : row_0.w1 + 1;
      // the products of all tiles before `it` (S of tile `it` was issued after
      // that of tile it - 2, so the phase is the next one or the one before)
      auto pv_wait = [&] {
        return __all_sync(0xffffffffu, mbar_wait(smem_u32(&pv_done[g]), (it - 1) & 1, p.status, abort_flag)) != 0;
      };
      float m = -INFINITY;  // in score units: P = exp2((S - m) scale)
      float2 l2 = make_float2(0.f, 0.f);
      for (int t = 0; t < tiles; ++t, ++it) {
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[g]), it & 1, p.status, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (__any_sync(0xffffffffu, *any_bad)) drop_bad_keys(s_addr, good_keys + 4 * ((it + skipped) & 15));
        float v[kKeys];
        tmem_ld64(s_addr, *reinterpret_cast<float(*)[64]>(v));
        tmem_ld64(s_addr + 64, *reinterpret_cast<float(*)[64]>(v + 64));
        const int at = t * kKeys;
        if (!(at + kKeys <= all_s || (at >= all_0 && at + kKeys <= all_1))) {
#pragma unroll
          for (int c = 0; c < kKeys / 32; ++c) {
            const int place = at + 32 * c;
            const uint32_t on = low_bits(view.sink_end - place) |
                                (low_bits(view.w1 + 1 - place) & ~low_bits(view.w0 - place));
#pragma unroll
            for (int i = 0; i < 32; ++i) v[32 * c + i] = (on >> i) & 1u ? v[32 * c + i] : -INFINITY;
          }
        }
        float mx[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) mx[c] = fmaxf(v[c], v[c + 8]);
#pragma unroll
        for (int i = 16; i < kKeys; i += 16)
#pragma unroll
          for (int c = 0; c < 8; ++c) mx[c] = fmaxf(fmaxf(mx[c], v[i + c]), v[i + 8 + c]);
        const float top = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                            fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
        // The reference maximum follows the running one only when it is 2^8
        // behind: P stays below 2^8, and O is rescaled rarely.
        const bool first = m == -INFINITY;
        const bool behind = !first && (top - m) * scale > 8.f;
        if (first) m = top;
        if (__any_sync(0xffffffffu, behind)) {
          float alpha = 1.f;
          if (behind) {
            alpha = ex2((m - top) * scale);
            m = top;
          }
          l2 = make_float2(l2.x * alpha, l2.y * alpha);
          ok = pv_wait();  // the tiles before have to be in O first
          if (!ok) break;
          tc_fence_after();
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tmem_ld32(o_addr + 32 * c, o);
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(o[i] * alpha);
            tmem_st32(o_addr + 32 * c, w);
          }
          tmem_wait_st();
        }
        const float base = m == -INFINITY ? 0.f : m * scale;
        const float2 scale2 = make_float2(scale, scale), base2 = make_float2(-base, -base);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float2 x = fma2(make_float2(v[64 * c + 2 * i], v[64 * c + 2 * i + 1]), scale2, base2);
            x.x = ex2(x.x);
            x.y = ex2(x.y);
            sum[i & 1] = add2(sum[i & 1], x);
            w[i] = pack2<T>(x.x, x.y);
          }
          tmem_st32(s_addr + 32 * c, w);
        }
        l2 = add2(l2, add2(sum[0], sum[1]));
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&p_ready[g]));
      }
      // The last S of this item is done, so its queries make room for the next
      // item's while its last product and its epilogue run.
      if (more) im = item_at(item + gridDim.x);
      if (ok && tiles > 0 && more && im.rb * kRows + 128 * g < im.rows_all) {
        load_q(im);
        here = true;
      }
      if (ok && tiles > 0) ok = pv_wait();
      bool mend = false;
      if (tiles > 0) {
        mend = marked[live & 7] == live + 1;
        __threadfence_block();
        mend = mend || *all_marked != 0;
      }
      mend = __any_sync(0xffffffffu, mend);
      // all warps of the group go on or none
      if (barrier_any(1 + g, 128, !ok)) break;
      if (gt == 0) seen[g] = live + 1;
      const float l = l2.x + l2.y;
      tc_fence_after();
      // ---- O / l, 64 dims at a time through 4 KB of the warp's own, so that
      // 8 lanes write 128 bytes of a row: stored from TMEM rows directly, a
      // lane each, the epilogue took 11k cycles of a 100k-cycle row block ----
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int w0 = 32 * (warp & 3);  // the warp's first row of the group
      const int qt0 = grow0 / p.group, rem0 = grow0 - qt0 * p.group;
      uint8_t* const stage = smem + SM::kStage + (warp - 4) * 4096;
      T* const out = static_cast<T*>(p.out);
#pragma unroll 1
      for (int hf = 0; hf < D / 64; ++hf) {
#pragma unroll 1
        for (int q4 = 0; q4 < 2; ++q4) {
          float o[32];
          if (tiles > 0) {
            tmem_ld32(o_addr + 64 * hf + 32 * q4, o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = l == 0.f ? 0.f : o[i] * inv;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(stage + lane * 128 + (((4 * q4 + i) ^ (lane & 7)) << 4)) =
                make_uint4(pack2<T>(o[8 * i], o[8 * i + 1]), pack2<T>(o[8 * i + 2], o[8 * i + 3]),
                           pack2<T>(o[8 * i + 4], o[8 * i + 5]), pack2<T>(o[8 * i + 6], o[8 * i + 7]));
        }
        __syncwarp();
        const int cc = lane & 7;
#pragma unroll 4
        for (int i = lane >> 3; i < 32; i += 4) {
          if (grow0 + w0 + i >= rows_all) break;
          const T* y = reinterpret_cast<const T*>(stage + i * 128 + ((cc ^ (i & 7)) << 4));
          T* dst = out + row_at(cur, qt0, rem0, w0 + i, p.os0, p.os1);
          const int d = 64 * hf + 8 * cc;
          if (p.out_vec) {
            *reinterpret_cast<uint4*>(dst + d) = *reinterpret_cast<const uint4*>(y);
          } else {
#pragma unroll 1
            for (int k = 0; k < 8; ++k) dst[(d + k) * p.os2] = y[k];
          }
        }
        __syncwarp();
      }
      const int left = rows_all - grow0 - w0;
      if (mend && left > 0) add_nonfinite<T, D>(p, cur.b, cur.h, cur.rb, grow0 + w0, min(32, left), lane);
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 3) tmem_dealloc(tmem, 512);
}

template <typename T, int D>
int launch(const StreamParams& p, const CUtensorMap& mk, const CUtensorMap& mv, const int (&kp)[4],
           const int (&vp)[4], dim3 grid, cudaStream_t stream) {
  auto kern = prompt_kernel<T, D>;
  constexpr size_t smem = PromptSmem<D>::kBytes;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(done, reinterpret_cast<const void*>(kern), smem, p.device);
  if (e == cudaSuccess)
    e = launch_pdl(kern, grid, dim3(kPromptThreads), smem, stream, p, mk, mv, make_int4(kp[0], kp[1], kp[2], 0),
                   make_int4(vp[0], vp[1], vp[2], 0));
  return cuda_status(e);
}

}  // namespace

bool prompt_attention(const StreamParams& p, bool bf16, int D, int64_t max_query_len, int64_t sms,
                      cudaStream_t stream, int* rc) {
  CacheDesc kd;
  kd.base = p.k;
  kd.elem_bytes = 2;
  kd.is_bf16 = bf16;
  kd.head_dim = D;
  kd.block_size = 1 << p.bs_log2;
  kd.num_heads = p.hkv;
  kd.num_blocks = p.num_blocks;
  kd.plane_box = -1;
  CacheDesc vd = kd;
  vd.base = p.v;
  const int64_t ks[4] = {p.ks0, p.ks1, p.ks2, p.ks3}, vs[4] = {p.vs0, p.vs1, p.vs2, p.vs3};
  std::copy(ks, ks + 4, kd.stride);
  std::copy(vs, vs + 4, vd.stride);
  CUtensorMap mk, mv;
  int kp[4], vp[4];
  if (!get_cache_tensor_map(kd, &mk, kp) || !get_cache_tensor_map(vd, &mv, vp)) return false;
  StreamParams part = p;
  *rc = FD_OK;
  for (part.first_seq = 0; *rc == FD_OK && part.first_seq < p.num_seqs; part.first_seq += kMostSeqs) {
    part.num_seqs = std::min(p.num_seqs - part.first_seq, kMostSeqs);
    // row blocks of the announced queries, or of all rows of q where those are fewer
    const int64_t each = (max_query_len * p.group + kRows - 1) / kRows * part.num_seqs;
    const int64_t all = static_cast<int64_t>(p.num_tokens) * p.group / kRows + part.num_seqs;
    const dim3 grid(static_cast<unsigned>(std::max<int64_t>(std::min(std::min(each, all) * p.hkv, sms), 1)));
    if (D == 128) {
      *rc = bf16 ? launch<__nv_bfloat16, 128>(part, mk, mv, kp, vp, grid, stream)
                 : launch<__half, 128>(part, mk, mv, kp, vp, grid, stream);
    } else {
      *rc = bf16 ? launch<__nv_bfloat16, 64>(part, mk, mv, kp, vp, grid, stream)
                 : launch<__half, 64>(part, mk, mv, kp, vp, grid, stream);
    }
  }
  return true;
}

}  // namespace fd

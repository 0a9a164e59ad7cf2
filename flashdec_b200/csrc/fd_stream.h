// Shared by the bounded-cache attention kernels (fd_window_attention,
// fd_scored_decode): launch parameters and the key range of a block of query
// rows.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace fd {

struct StreamParams {
  const void* q;
  int64_t qs0, qs1, qs2;
  void* out;
  int64_t os0, os1, os2;
  const void* k;
  int64_t ks0, ks1, ks2, ks3;
  const void* v;
  int64_t vs0, vs1, vs2, vs3;
  const void* bt;
  int64_t bts0, bts1;
  const void* sl;
  int64_t sls;
  const void* qstart;  // null: one query per sequence
  int64_t qss;
  float* scores;  // null: no scores kept
  int64_t scs0, scs1, scs2;
  int bt64, sl64, qs64;
  int num_seqs, num_tokens, hq, hkv, group;
  uint32_t group_magic;  // ceil(2^32 / group): x / group = mulhi(x, magic) while x * group < 2^32 (not for group 1)
  int bs_log2, num_blocks, max_blocks;
  int window, sinks;
  int row_blocks;  // of the longest queries announced
  int splits;      // CTAs of a unit (cluster or grid)
  int vec;         // rows of K and V are 16-byte aligned and contiguous
  int q_vec, out_vec;  // the same of q and of out
  float scale_log2;
  int mode;         // how the split kernel's CTAs share the units (fd_stream_attention.cu)
  int first_seq;    // of this launch's num_seqs
  int rows_cta;     // rows of a row block
  int rows_most;    // rows of a cluster's row block
  int score_vec;    // four scores of a page: one 16-byte access
  int3* share_unit; // [share] where it starts: {sequence of the launch, row block x KV head, tile}
  int* shares;      // number of shares
  float* part_acc;  // [place][row of the unit][D]
  float* part_ml;   // [place][row of the unit][2]: max (base 2), sum
  float* row_lse;   // [query x head]: max + log2(sum), with scores
  float* raw;       // scaled scores (base 2): per sequence of the launch [head][its tokens]
  int64_t* raw_start;  // [sequence of the launch] tokens before its raw scores (kShares)
  int64_t raw_tokens;  // row length of raw (kGrid), or of its copy in shared memory
  int64_t raw_room;    // tokens that raw has room for
  uint64_t blocks_magic;  // ceil(2^64 / row blocks of a group); 0: one
  int* status;
  int device;  // host side only
};

// The sequence's queries: rows [q0, q0 + qlen) of q, tokens [n - qlen, n).
struct StreamSeq {
  int q0, qlen, n;
};

// The keys that rows [r0, r1) of a sequence's (query, group head) rows can
// see, as a list of cache pages: `sink_pages` from position 0, then the pages
// from `win_page` to the one of the last query.  Adjoining ranges are one
// (sink_pages 0, win_page 0), so no key is listed twice.
struct StreamRange {
  int pos0, pos1;      // positions of the first and the last row's query
  int lo;              // first key in the first row's window
  int sink_end;        // sinks seen: [0, sink_end)
  int sink_pages, win_page, pages;

  __host__ __device__ StreamRange(const StreamSeq& s, int r0, int r1, int group, int window,
                                  int sinks, int bs_log2) {
    pos0 = s.n - s.qlen + r0 / group;
    pos1 = s.n - s.qlen + (r1 - 1) / group;
    lo = pos0 - window + 1 > 0 ? pos0 - window + 1 : 0;
    sink_end = sinks < pos1 + 1 ? sinks : pos1 + 1;
    sink_pages = (sink_end + (1 << bs_log2) - 1) >> bs_log2;
    win_page = lo >> bs_log2;
    if (pos1 < 0) {  // no row sees a key
      sink_end = sink_pages = win_page = pages = 0;
      return;
    }
    if (sink_pages >= win_page) {
      if (sink_pages > 0) win_page = 0;
      sink_pages = 0;
    }
    pages = sink_pages + (pos1 >> bs_log2) + 1 - win_page;
  }
  // logical page of list entry i
  __host__ __device__ int page(int i) const { return i < sink_pages ? i : i - sink_pages + win_page; }
};

// fd_window_attention on tcgen05, for many rows per (sequence, KV head).  False
// when no tensor map describes the caches (nothing is launched); else *rc is
// the launch's status.
bool prompt_attention(const StreamParams& p, bool bf16, int head_dim, int64_t max_query_len, int64_t sms,
                      cudaStream_t stream, int* rc);

}  // namespace fd

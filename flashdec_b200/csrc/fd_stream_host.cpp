// Native host path of the bounded-cache operators (module
// flashdec_b200._hostpath): argument checks, output and workspace allocation
// and the library call of window_attention, scored_decode and evict_tokens in
// one C++ function each.  A decode step calls them once per layer, where the
// same checks in Python cost several times the launch.
//
// Misuse raises ValueError before any CUDA call.  The workspace is a tensor of
// the caching allocator taken on the current stream, so calls on different
// streams never share one and a CUDA graph keeps its own.
#include "fd_stream_host.h"

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <cstring>
#include <limits>
#include <string>

#include "flashdec_b200.h"

namespace {

using AttentionFn = int (*)(const fd_stream_attention_args*, void*);
using WorkspaceFn = int (*)(const fd_stream_attention_args*, size_t*);
using EvictFn = int (*)(const fd_evict_tokens_args*, void*);
using ErrorFn = const char* (*)(int);

AttentionFn g_window = nullptr, g_scored = nullptr;
WorkspaceFn g_window_ws = nullptr, g_scored_ws = nullptr;
EvictFn g_evict = nullptr;
ErrorFn g_error = nullptr;

void require(bool ok, const char* message) {
  if (!ok) throw py::value_error(message);
}

// FlashDecNativeError of _lib.check, raised from here
void check_status(int rc, const char* what) {
  if (rc == FD_OK) return;
  const std::string msg = std::string(what) + " failed: " + g_error(rc) + " (status " + std::to_string(rc) + ")";
  py::object cls = py::module_::import("flashdec_b200._lib").attr("FlashDecNativeError");
  PyErr_SetString(cls.ptr(), msg.c_str());
  throw py::error_already_set();
}

int index_code(const at::Tensor& t, const char* message) {
  if (t.scalar_type() == at::kInt) return FD_INDEX_I32;
  if (t.scalar_type() == at::kLong) return FD_INDEX_I64;
  throw py::value_error(message);
}

int32_t as_i32(int64_t v, const char* message) {
  require(v <= std::numeric_limits<int32_t>::max(), message);
  return static_cast<int32_t>(v);
}

bool same_device(const at::Tensor& a, const at::Tensor& b) {
  return b.is_cuda() && a.get_device() == b.get_device();
}

// A cache in logical order [block, kv_head, token, dim]
struct Cache {
  int64_t blocks, heads, tokens, dim;
  int64_t stride[4];
  Cache(const at::Tensor& t, bool dim_major) {
    const int ta = dim_major ? 3 : 2, da = dim_major ? 2 : 3;
    blocks = t.size(0);
    heads = t.size(1);
    tokens = t.size(ta);
    dim = t.size(da);
    stride[0] = t.stride(0);
    stride[1] = t.stride(1);
    stride[2] = t.stride(ta);
    stride[3] = t.stride(da);
  }
};

bool dim_major_of(const std::string& layout) {
  if (layout == "token_major") return false;
  if (layout == "dim_major") return true;
  throw py::value_error("kv_layout must be 'token_major' or 'dim_major'");
}

// K, V, block tables and lengths, common to the three operators.
void check_caches(const at::Tensor& k, const at::Tensor& v, const at::Tensor& block_tables,
                  const at::Tensor& seq_lens, const Cache& kc, const Cache& vc) {
  require(k.scalar_type() == v.scalar_type(), "k_cache and v_cache must have the same dtype");
  require(k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16,
          "the caches must be float16 or bfloat16");
  require(kc.blocks == vc.blocks && kc.heads == vc.heads && kc.tokens == vc.tokens && kc.dim == vc.dim,
          "k_cache and v_cache must have the same shape");
  require(kc.blocks > 0 && kc.heads > 0, "num_blocks and num_kv_heads must be positive");
  require(kc.tokens == 8 || kc.tokens == 16 || kc.tokens == 32, "block_size must be 8, 16 or 32");
  require(kc.dim == 64 || kc.dim == 128, "head_dim must be 64 or 128");
  require(block_tables.size(1) > 0, "max_blocks_per_seq must be positive");
  require(block_tables.size(0) == seq_lens.size(0),
          "block_tables and seq_lens must have one row/value per sequence");
}

void check_ranks(const at::Tensor& k, const at::Tensor& v, const at::Tensor& block_tables,
                 const at::Tensor& seq_lens) {
  require(k.is_cuda(), "k_cache must be a CUDA tensor");
  require(same_device(k, v) && same_device(k, block_tables) && same_device(k, seq_lens),
          "k_cache, v_cache, block_tables and seq_lens must be on the same CUDA device");
  require(k.dim() == 4 && v.dim() == 4, "k_cache and v_cache must be 4D tensors");
  require(block_tables.dim() == 2, "block_tables must have shape [num_seqs, max_blocks_per_seq]");
  require(seq_lens.dim() == 1, "seq_lens must have shape [num_seqs]");
}

void check_scores(const at::Tensor& k, const at::Tensor& scores, const Cache& kc) {
  require(same_device(k, scores), "scores must be on the device of k_cache");
  require(scores.dim() == 3 && scores.size(0) == kc.blocks && scores.size(1) == kc.heads &&
              scores.size(2) == kc.tokens,
          "scores must have shape [num_blocks, num_kv_heads, block_size]");
  require(scores.scalar_type() == at::kFloat, "scores must be float32");
}

template <size_t N>
void set_strides(int64_t (&dst)[N], const at::Tensor& t) {
  for (size_t i = 0; i < N; ++i) dst[i] = t.stride(static_cast<int64_t>(i));
}

// The part of an attention call that both operators share; returns out.
at::Tensor fill(fd_stream_attention_args* a, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                const at::Tensor& block_tables, const at::Tensor& seq_lens,
                const std::optional<double>& sm_scale, const std::string& kv_layout,
                const std::optional<at::Tensor>& out) {
  const bool dm = dim_major_of(kv_layout);
  check_ranks(k, v, block_tables, seq_lens);
  require(same_device(k, q), "q must be on the device of k_cache");
  require(q.dim() == 3, "q must have shape [num_tokens, num_q_heads, head_dim]");
  const Cache kc(k, dm), vc(v, dm);
  check_caches(k, v, block_tables, seq_lens, kc, vc);
  require(q.scalar_type() == k.scalar_type(), "q, k_cache and v_cache must have the same dtype");
  require(q.size(2) == kc.dim, "q, k_cache and v_cache must have the same head_dim");
  require(q.size(1) > 0 && q.size(1) % kc.heads == 0, "num_q_heads must be divisible by num_kv_heads");
  at::Tensor o;
  if (out.has_value()) {
    o = *out;
    require(same_device(q, o) && o.sizes() == q.sizes() && o.scalar_type() == q.scalar_type(),
            "out must have the shape, dtype and device of q");
  } else {
    o = at::empty(q.sizes(), q.options());
  }
  std::memset(a, 0, sizeof(*a));
  a->struct_size = static_cast<int32_t>(sizeof(*a));
  a->dtype = q.scalar_type() == at::kHalf ? FD_DTYPE_F16 : FD_DTYPE_BF16;
  a->num_seqs = as_i32(block_tables.size(0), "too many sequences");
  a->num_tokens = as_i32(q.size(0), "too many query tokens");
  a->num_q_heads = as_i32(q.size(1), "too many heads");
  a->num_kv_heads = as_i32(kc.heads, "too many heads");
  a->head_dim = static_cast<int32_t>(kc.dim);
  a->block_size = static_cast<int32_t>(kc.tokens);
  a->num_blocks = as_i32(kc.blocks, "too many blocks");
  a->max_blocks_per_seq = as_i32(block_tables.size(1), "block_tables rows are too long");
  a->sm_scale = static_cast<float>(sm_scale.has_value() ? *sm_scale : 1.0 / std::sqrt(static_cast<double>(kc.dim)));
  a->q = q.data_ptr();
  set_strides(a->q_stride, q);
  a->out = o.data_ptr();
  set_strides(a->out_stride, o);
  a->k_cache = k.data_ptr();
  std::memcpy(a->k_stride, kc.stride, sizeof(a->k_stride));
  a->v_cache = v.data_ptr();
  std::memcpy(a->v_stride, vc.stride, sizeof(a->v_stride));
  a->block_tables = block_tables.data_ptr();
  set_strides(a->block_tables_stride, block_tables);
  a->block_tables_index = index_code(block_tables, "block_tables must be int32 or int64");
  a->seq_lens = seq_lens.data_ptr();
  a->seq_lens_stride = seq_lens.stride(0);
  a->seq_lens_index = index_code(seq_lens, "seq_lens must be int32 or int64");
  return o;
}

void launch(fd_stream_attention_args* a, const at::Tensor& q, WorkspaceFn ws, AttentionFn fn,
            const char* what) {
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  size_t bytes = 0;
  check_status(ws(a, &bytes), what);
  at::Tensor scratch;
  if (bytes > 0) {
    scratch = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
    a->scratch = scratch.data_ptr();
    a->scratch_bytes = bytes;
  }
  check_status(fn(a, c10::cuda::getCurrentCUDAStream(q.get_device()).stream()), what);
}

at::Tensor window_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const at::Tensor& block_tables, const at::Tensor& seq_lens, int64_t window,
                            int64_t sinks, const std::optional<at::Tensor>& query_start_loc,
                            const std::optional<int64_t>& max_query_len,
                            const std::optional<double>& sm_scale, const std::string& kv_layout,
                            const std::optional<at::Tensor>& out) {
  fd_stream_attention_args a;
  require(window >= 1, "window must be at least 1");
  require(sinks >= 0, "sinks must not be negative");
  at::Tensor o = fill(&a, q, k, v, block_tables, seq_lens, sm_scale, kv_layout, out);
  a.window = window;
  a.sinks = sinks;
  a.max_query_len = 1;
  if (query_start_loc.has_value()) {
    const at::Tensor& st = *query_start_loc;
    require(same_device(q, st) && st.dim() == 1 && st.size(0) == block_tables.size(0) + 1,
            "query_start_loc must have shape [num_seqs + 1] on the device of q");
    require(max_query_len.has_value() && *max_query_len >= 1,
            "query_start_loc needs max_query_len, at least 1");
    a.query_start_loc = st.data_ptr();
    a.query_start_loc_stride = st.stride(0);
    a.query_start_loc_index = index_code(st, "query_start_loc must be int32 or int64");
    a.max_query_len = static_cast<int32_t>(
        std::min<int64_t>(*max_query_len, std::max<int64_t>(q.size(0), 1)));
  } else {
    require(q.size(0) == block_tables.size(0),
            "without query_start_loc, q must have one row per sequence");
    require(!max_query_len.has_value() || *max_query_len == 1,
            "without query_start_loc, max_query_len must be 1");
  }
  launch(&a, q, g_window_ws, g_window, "fd_window_attention");
  return o;
}

at::Tensor scored_decode(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                         const at::Tensor& scores, const at::Tensor& block_tables,
                         const at::Tensor& seq_lens, const std::optional<double>& sm_scale,
                         const std::string& kv_layout, const std::optional<at::Tensor>& out) {
  fd_stream_attention_args a;
  at::Tensor o = fill(&a, q, k, v, block_tables, seq_lens, sm_scale, kv_layout, out);
  require(q.size(0) == block_tables.size(0), "q must have one row per sequence");
  check_scores(k, scores, Cache(k, dim_major_of(kv_layout)));
  a.scores = static_cast<float*>(scores.data_ptr());
  set_strides(a.scores_stride, scores);
  launch(&a, q, g_scored_ws, g_scored, "fd_scored_decode");
  return o;
}

std::tuple<at::Tensor, at::Tensor> evict_tokens(const at::Tensor& k, const at::Tensor& v,
                                                const at::Tensor& scores, const at::Tensor& block_tables,
                                                const at::Tensor& seq_lens,
                                                const at::Tensor& new_block_tables, int64_t budget,
                                                int64_t sinks, int64_t recent,
                                                const std::string& kv_layout) {
  const bool dm = dim_major_of(kv_layout);
  require(budget >= 1, "budget must be at least 1");
  require(sinks >= 0 && recent >= 0, "sinks and recent must not be negative");
  require(sinks <= budget && recent <= budget - sinks, "sinks + recent must not exceed budget");
  check_ranks(k, v, block_tables, seq_lens);
  const Cache kc(k, dm), vc(v, dm);
  check_caches(k, v, block_tables, seq_lens, kc, vc);
  check_scores(k, scores, kc);
  require(same_device(k, new_block_tables) && new_block_tables.dim() == 2 &&
              new_block_tables.size(0) == block_tables.size(0) && new_block_tables.size(1) > 0,
          "new_block_tables must have shape [num_seqs, max_new_blocks_per_seq] on the device of k_cache");
  const int64_t longest = std::min(budget, block_tables.size(1) * kc.tokens);
  require(new_block_tables.size(1) * kc.tokens >= longest, "new_block_tables cannot hold budget tokens");
  fd_evict_tokens_args a;
  std::memset(&a, 0, sizeof(a));
  a.struct_size = static_cast<int32_t>(sizeof(a));
  a.elem_bytes = 2;
  a.num_seqs = as_i32(block_tables.size(0), "too many sequences");
  a.num_kv_heads = as_i32(kc.heads, "too many heads");
  a.head_dim = static_cast<int32_t>(kc.dim);
  a.block_size = static_cast<int32_t>(kc.tokens);
  a.num_blocks = as_i32(kc.blocks, "too many blocks");
  a.max_blocks_per_seq = as_i32(block_tables.size(1), "block_tables rows are too long");
  a.max_new_blocks_per_seq = as_i32(new_block_tables.size(1), "new_block_tables rows are too long");
  a.budget = as_i32(budget, "budget is too large");
  a.sinks = static_cast<int32_t>(sinks);
  a.recent = static_cast<int32_t>(recent);
  a.k_cache = k.data_ptr();
  std::memcpy(a.k_stride, kc.stride, sizeof(a.k_stride));
  a.v_cache = v.data_ptr();
  std::memcpy(a.v_stride, vc.stride, sizeof(a.v_stride));
  a.scores = static_cast<float*>(scores.data_ptr());
  set_strides(a.scores_stride, scores);
  a.block_tables = block_tables.data_ptr();
  set_strides(a.block_tables_stride, block_tables);
  a.block_tables_index = index_code(block_tables, "block_tables must be int32 or int64");
  a.seq_lens = seq_lens.data_ptr();
  a.seq_lens_stride = seq_lens.stride(0);
  a.seq_lens_index = index_code(seq_lens, "seq_lens must be int32 or int64");
  a.new_block_tables = new_block_tables.data_ptr();
  set_strides(a.new_block_tables_stride, new_block_tables);
  a.new_block_tables_index = index_code(new_block_tables, "new_block_tables must be int32 or int64");
  a.new_seq_lens_index = a.seq_lens_index;
  const c10::cuda::OptionalCUDAGuard guard(k.device());
  at::Tensor kept = at::empty({block_tables.size(0), kc.heads, budget}, k.options().dtype(at::kInt));
  at::Tensor lens = at::empty({block_tables.size(0)}, seq_lens.options());
  a.kept = static_cast<int32_t*>(kept.data_ptr());
  a.new_seq_lens = lens.data_ptr();
  check_status(g_evict(&a, c10::cuda::getCurrentCUDAStream(k.get_device()).stream()), "fd_evict_tokens");
  return {kept, lens};
}

void set_stream_entry_points(int64_t window, int64_t window_ws, int64_t scored, int64_t scored_ws,
                             int64_t evict, int64_t error) {
  g_window = reinterpret_cast<AttentionFn>(window);
  g_window_ws = reinterpret_cast<WorkspaceFn>(window_ws);
  g_scored = reinterpret_cast<AttentionFn>(scored);
  g_scored_ws = reinterpret_cast<WorkspaceFn>(scored_ws);
  g_evict = reinterpret_cast<EvictFn>(evict);
  g_error = reinterpret_cast<ErrorFn>(error);
}

}  // namespace

void bind_stream_operators(py::module_& m) {
  m.attr("STREAM_ARGS_BYTES") = static_cast<int64_t>(sizeof(fd_stream_attention_args));
  m.attr("EVICT_ARGS_BYTES") = static_cast<int64_t>(sizeof(fd_evict_tokens_args));
  m.def("set_stream_entry_points", &set_stream_entry_points);
  m.def("window_attention", &window_attention);
  m.def("scored_decode", &scored_decode);
  m.def("evict_tokens", &evict_tokens);
}

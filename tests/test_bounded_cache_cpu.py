"""The bounded-cache operators on the CPU: struct layouts, the C entry points'
argument checks, the key-range arithmetic, and the oracle's own properties.
No kernel is launched here."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

from flashdec_b200 import _lib
from oracle import bounded_cache as ref

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def test_struct_layouts(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    structs = {"fd_stream_attention_args": _lib.StreamAttentionArgs,
               "fd_evict_tokens_args": _lib.EvictTokensArgs}
    body = ""
    for cname, cls in structs.items():
        body += f'printf("{cname} sizeof %zu\\n", sizeof({cname}));\n'
        for f, _ in cls._fields_:
            body += f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));\n'
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "flashdec_b200.h"\n'
                   f"int main(void) {{ {body} return 0; }}\n")
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-std=c99", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        cname, field, value = line.split()
        cls = structs[cname]
        mine = ctypes.sizeof(cls) if field == "sizeof" else getattr(cls, field).offset
        assert mine == int(value), (cname, field)


def _attention_args():
    a = _lib.StreamAttentionArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype, a.head_dim, a.block_size = _lib.FD_DTYPE_BF16, 128, 32
    a.num_seqs = a.num_tokens = 1
    a.num_q_heads, a.num_kv_heads, a.num_blocks, a.max_blocks_per_seq = 8, 2, 4, 4
    a.window, a.max_query_len = 16, 1
    return a


@pytest.mark.parametrize("name", ["fd_window_attention", "fd_scored_decode"])
def test_attention_argument_checks(lib, name):
    fn, bad, uns = getattr(lib, name), _lib.FD_ERR_INVALID_ARGUMENT, _lib.FD_ERR_UNSUPPORTED
    assert fn(None, None) == bad
    assert fn(ctypes.byref(_attention_args()), None) == bad  # no pointers
    changes = [("struct_size", 8, bad), ("dtype", _lib.FD_DTYPE_F32, uns), ("head_dim", 96, uns),
               ("block_size", 12, uns), ("num_q_heads", 7, bad), ("num_kv_heads", 0, bad),
               ("num_seqs", -1, bad), ("num_blocks", 0, bad), ("max_blocks_per_seq", 1 << 30, uns),
               ("num_seqs", 70000, uns)]
    if name == "fd_window_attention":
        changes += [("window", 0, bad), ("sinks", -1, bad), ("max_query_len", 0, bad),
                    ("num_tokens", 2, bad)]
    for field, value, want in changes:
        a = _attention_args()
        setattr(a, field, value)
        assert fn(ctypes.byref(a), None) == want, field
        assert getattr(lib, name + "_workspace")(ctypes.byref(a), None) == want, field
    a = _attention_args()
    a.num_seqs = a.num_tokens = 0
    assert fn(ctypes.byref(a), None) == _lib.FD_OK  # nothing to do, no pointer needed


def test_evict_argument_checks(lib):
    def args():
        a = _lib.EvictTokensArgs()
        a.struct_size, a.elem_bytes = ctypes.sizeof(a), 2
        a.num_seqs, a.num_kv_heads, a.head_dim, a.block_size = 1, 2, 64, 8
        a.num_blocks, a.max_blocks_per_seq, a.max_new_blocks_per_seq, a.budget = 4, 4, 1, 8
        return a

    fn, bad, uns = lib.fd_evict_tokens, _lib.FD_ERR_INVALID_ARGUMENT, _lib.FD_ERR_UNSUPPORTED
    assert fn(None, None) == bad
    assert fn(ctypes.byref(args()), None) == bad
    for field, value, want in [("struct_size", 8, bad), ("elem_bytes", 4, uns), ("head_dim", 80, uns),
                               ("block_size", 4, uns), ("budget", 0, bad), ("sinks", -1, bad),
                               ("recent", 9, bad), ("num_seqs", 1 << 20, uns), ("num_kv_heads", 0, bad),
                               ("max_new_blocks_per_seq", 0, bad)]:
        a = args()
        setattr(a, field, value)
        assert fn(ctypes.byref(a), None) == want, field
    a = args()
    a.num_seqs = 0
    assert fn(ctypes.byref(a), None) == _lib.FD_OK


def test_key_range_lists_every_visible_page_once(tmp_path):
    """StreamRange (the kernels' page list) against the mask, over many small
    shapes, compiled for the host."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        pytest.skip("nvcc not available")
    src = tmp_path / "range.cu"
    src.write_text(r"""
#include <cstdio>
#include <vector>
#include "fd_stream.h"
int main() {
  long checked = 0;
  for (int bs = 3; bs <= 4; ++bs)
  for (int n = 0; n <= 70; n += 3)
  for (int q = 1; q <= 40; q += 3)
  for (int window = 1; window <= 80; window += 7)
  for (int sinks = 0; sinks <= 40; sinks += 4)
  for (int group = 1; group <= 3; group += 2)
  for (int r0 = 0; r0 < q * group; r0 += 16) {
    const int r1 = r0 + 16 < q * group ? r0 + 16 : q * group;
    fd::StreamSeq s{0, q, n};
    fd::StreamRange rg(s, r0, r1, group, window, sinks, bs);
    std::vector<int> count(32, 0);
    for (int i = 0; i < rg.pages; ++i) {
      const int pg = rg.page(i);
      if (pg < 0 || pg >= 32) { std::printf("page %d\n", pg); return 1; }
      ++count[pg];
    }
    for (int k = 0; k < n; ++k) {
      bool seen = false;
      for (int r = r0; r < r1; ++r) {
        const int pos = n - q + r / group;
        seen |= k <= pos && (k > pos - window || k < sinks);
      }
      const bool ranged = k <= rg.pos1 && (k >= rg.lo || k < rg.sink_end);
      if (seen != ranged && r1 - r0 <= group) { std::printf("range\n"); return 1; }
      if (seen && !ranged) { std::printf("missed\n"); return 1; }
      if (ranged && count[k >> bs] != 1) { std::printf("list %d\n", count[k >> bs]); return 1; }
      ++checked;
    }
    for (int c : count) if (c > 1) { std::printf("twice\n"); return 1; }
  }
  std::printf("ok %ld\n", checked);
  return 0;
}
""")
    exe = tmp_path / "range"
    subprocess.run([nvcc, "-std=c++17", "-I", str(ROOT / "flashdec_b200" / "csrc"), str(src), "-o", str(exe)],
                   check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0 and res.stdout.startswith("ok"), res.stdout


def test_oracle_window_is_causal_attention_when_wide():
    rng = np.random.default_rng(0)
    k, v = (rng.standard_normal((4, 2, 8, 16)) for _ in range(2))
    q = rng.standard_normal((20, 4, 16))
    table = np.array([[2, 0, 3]])
    wide, _ = ref.window_attention_ref(q, k, v, table, [20], 100, 0, [0, 20])
    for t in (0, 7, 19):
        one, _ = ref.window_attention_ref(q[t:t + 1], k, v, table, [t + 1], 100)
        assert np.allclose(wide[t], one[0], rtol=1e-12)
    # sinks as long as the stream make any window the whole of it
    sunk, _ = ref.window_attention_ref(q, k, v, table, [20], 1, 20, [0, 20])
    assert np.allclose(sunk, wide, rtol=1e-12)


def test_oracle_scores_are_the_weights():
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((4, 1, 8, 16)) for _ in range(2))
    q = rng.standard_normal((1, 3, 16))
    start = np.full((4, 1, 8), 5.0)
    _, _, s = ref.scored_decode_ref(q, k, v, start, np.array([[1, 3]]), [11])
    assert np.isclose((s - start)[[1, 3]].sum() + 5.0, 3.0)  # the newest token started at zero
    assert (s[[0, 2]] == 5.0).all()


def test_oracle_choice_order():
    nan, inf = float("nan"), float("inf")
    assert ref.evict_choice([1, 2, 3], 3, 0, 0) == [0, 1, 2]
    assert ref.evict_choice([0, 9, 9, 9, 0], 3, 1, 1) == [0, 1, 4]
    assert ref.evict_choice([0.0, -0.0, 0.0], 2, 0, 0) == [0, 1]
    assert ref.evict_choice([inf, nan, -inf, 5], 2, 0, 0) == [0, 1]
    assert ref.evict_choice([5, inf, 1, nan], 1, 0, 0) == [3]


def test_cpu_tensors_are_refused():
    torch = pytest.importorskip("torch")
    import flashdec_b200 as fd

    k = torch.zeros((2, 1, 8, 64), dtype=torch.bfloat16)
    bt, sl = torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        fd.window_attention(q, k, k, bt, sl, window=4)
    with pytest.raises(ValueError, match="CUDA"):
        fd.scored_decode(q, k, k, torch.zeros(2, 1, 8), bt, sl)
    with pytest.raises(ValueError, match="CUDA"):
        fd.evict_tokens(k, k, torch.zeros(2, 1, 8), bt, sl, bt, budget=1)

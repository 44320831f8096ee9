"""Sizes of the windowed attention that need no GPU: what the workspace queries take, and the
host's arithmetic on the largest grids."""
import subprocess
import sys

import pytest

from ml_engine_amd import build, hip

MOST = 2 ** 31 - 1
ROOT = hip.LIB_DIR.parent.parent


def query(name, *args):
    """A query in a process of its own, which an arithmetic trap would end."""
    code = f"import sys; sys.path.insert(0, {str(ROOT)!r}); from ml_engine_amd import hip; print(hip.lib().{name}{args})"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (name, args, r.returncode, r.stderr[-300:])
    return int(r.stdout)


@pytest.mark.parametrize("name,args", [
    ("mle_window_attention_step_ws_bytes", (1, 1, 1000, 2, 4, 64, 500, 0)),        # fewer heads than heads of keys
    ("mle_window_attention_step_ws_bytes", (1, 1, 1000, 6, 4, 64, 500, 0)),        # no whole groups
    ("mle_window_attention_step_ws_bytes", (1, 31, 1000, MOST, 1, 64, 500, 0)),
    ("mle_window_attention_step_ws_bytes", (MOST, 31, MOST, 1 << 16, 1, MOST, MOST, MOST)),
    ("mle_window_attention_ws_bytes", (1, 300, 2, 4, 64, 500, 0)),
    ("mle_window_attention_ws_bytes", (1, MOST, 2, 2, 64, 500, 0)),
    ("mle_window_attention_ws_bytes", (1, 300, 2, 2, 129, 500, 0)),
    ("mle_window_attention_ws_bytes", (MOST, MOST, MOST, 1, MOST, 500, MOST)),
])
def test_queries_of_sizes_that_the_calls_refuse(name, args):
    assert query(name, *args) == 0


def test_queries_of_the_largest_sizes():
    """The largest that the calls take: a number per row and head at least, and no overflow."""
    assert query("mle_window_attention_ws_bytes", 1, 1 << 30, 8, 8, 128, MOST, MOST) >= 8 * (8 << 30)
    assert query("mle_window_attention_step_ws_bytes", 1, 31, 1 << 30, 8, 1, 128, MOST, 0) > 0


def host_program(tmp_path, body, *includes):
    """What a program of the kernels' headers' host side prints."""
    src = tmp_path / "sizes.hip"
    src.write_text("".join(f'#include "{hip.LIB_DIR.parent / "csrc" / i}"\n' for i in includes)
                   + "#include <stdio.h>\nint main() {\n" + body + "\n}\n")
    exe = tmp_path / "sizes"
    subprocess.run([build.HIPCC, "--cuda-host-only", "-x", "hip", "-std=c++17", "-O1", "-w", f"-I{build.INCLUDE}", str(src),
                    "-o", str(exe)], check=True, capture_output=True, timeout=300)
    return [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout.split()]


def test_rows_of_a_tile_lie_at_whole_vectors(tmp_path):
    """The backward reads four rows' log-sums and Ds at once from an array of these."""
    size, align, lse, delta = host_program(
        tmp_path, 'typedef wattn::Rows<32> R; printf("%zu %zu %zu %zu", sizeof(R), alignof(R), offsetof(R, lse), offsetof(R, delta));',
        "window_bwd.hpp")
    assert align >= 16 and size % 16 == 0 and lse % 16 == 0 and delta % 16 == 0


def test_grids_of_more_than_32_bits(tmp_path):
    """One-token sequences of many narrow heads: more groups than an int holds."""
    got = host_program(tmp_path, """
  wattn::Args a{};
  a.batch = 1 << 24, a.kv_heads = 1 << 8, a.heads = 1 << 8, a.group = 1, a.rows = a.keys = 1, a.dim = 1, a.window = 1;
  wattn::Grid g(a, a.heads, 1, 8);
  printf("%lld %lld ", (long long)g.groups, (long long)g.total);
  const int64_t ids[] = {0, 7, 8, (1ll << 32) - 1, (1ll << 31) + 5};
  for (int64_t id : ids) {
    const wattn::Place p = g.place(id);
    printf("%lld %d ", (long long)p.group, p.item);
  }
  a.batch = (1 << 24) - 1, a.kv_heads = a.heads = 255;
  wattn::Grid odd(a, a.heads, 3, 8);
  const wattn::Place p = odd.place(odd.total - 1);
  printf("%lld %lld %d", (long long)odd.groups, (long long)p.group, p.item);
""", "window_kernels.hpp")
    assert got[:2] == [1 << 32, 1 << 32]
    assert got[2:12] == [x for i in (0, 7, 8, (1 << 32) - 1, (1 << 31) + 5) for x in (i, 0)]
    n = ((1 << 24) - 1) * 255
    assert got[12:] == [n, n - 1, 2]

"""The segments in which the kernels of 128- and 256-row tiles walk a piece's keys
(csrc/segments.hpp), in constant expressions, where a signed overflow does not
compile: up to the longest sequence that attention over chunks takes."""

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "neuronmlp-on-tpu_amd" / "csrc"
LONGEST = 0x7ffe0000  # tokens of a sequence
WALK = """
#include "segments.hpp"
using namespace svdmlp;
static_assert(kChunkTokensMost == 0x7ffe0000, "");
// Whether the segments of keys begin .. end cover them in order, whole tiles but for the last, in at most `ids` pages.
constexpr bool walk(int ids, int tile, int page, int begin, int end) {
  const int most = segment_keys(ids, page, tile);
  if (most < tile || most % tile != 0) return false;
  // a segment that begins at a page's last token
  if ((page - 1 + (long long)most - 1) / page + 1 > ids) return false;
  long long done = begin;
  for (int at = begin; at < end; at += most) {  // (as the kernels do)
    const int upto = end < at + most ? end : at + most;
    if (at != done || (done - begin) % tile != 0 || upto <= at) return false;
    done = upto;
  }
  return done == (end > begin ? end : begin);
}
// As it must not be: segments of as many keys as their pages have.
constexpr bool long_segments(int ids, int tile, int page, int keys) {
  const int most = (ids - 1) * page / tile * tile;
  int n = 0;
  for (int at = 0; at < keys; at += most) ++n;
  return n > 0;
}
"""


def _compile(tmp_path, text):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    (tmp_path / "walk.cpp").write_text(WALK + text)
    return subprocess.run([cxx, "-std=c++17", "-fsyntax-only", f"-I{CSRC}", str(tmp_path / "walk.cpp")], capture_output=True, text=True)


def _cases():
    for page in (1, 2, 3, 4, 5, 16, 48, 64, 1000, 32768, 65536, 131072, 262144, 262272, 1 << 24, 1 << 30, LONGEST):
        most = min(LONGEST, 65536 * page)  # (as wide as a table may be)
        ends = sorted({0, 1, 31, 64, most // 3, most // 2 + 1, most - 131072, most - 1, most})
        for end in ends:
            for begin in {0, 64, end - 1, end, end // 64 * 48, (end - 8000000) // 64 * 64}:
                if 0 <= begin and end <= most and begin <= end:
                    yield page, begin, end


@pytest.mark.parametrize("ids,tile", [(2048, 32), (4096, 64)])
def test_segments_cover_every_piece(tmp_path, ids, tile):
    text = "\n".join(f'static_assert(walk({ids}, {tile}, {page}, {begin}, {end}), "{page} {begin} {end}");' for page, begin, end in _cases())
    done = _compile(tmp_path, text)
    assert done.returncode == 0, done.stderr


@pytest.mark.parametrize("ids,tile", [(2048, 32), (4096, 64)])
def test_long_segments_would_overflow(tmp_path, ids, tile):
    done = _compile(tmp_path, f"static_assert(long_segments({ids}, {tile}, 32768, {LONGEST}));")
    assert done.returncode != 0 and "overflow" in done.stderr

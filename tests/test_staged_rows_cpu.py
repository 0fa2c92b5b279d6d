"""CPU-only: the shared memory that a staged row is given (texo_b200/csrc/row_ops.cuh) holds every
byte that the row's kernels touch, for every row length up to a few thousand values.

Reads past a block's shared memory return nothing wrong that a test on the GPU could see (what lies
behind a row's end is dropped), so the sizes are checked by arithmetic: a small host program
includes the header and compares its `staged_bytes` with the extents of the accesses."""
import subprocess

from texo_b200 import build

PROGRAM = r"""
#include <cstdio>
#include "row_ops.cuh"

// Bytes from the start of a staged row that a kernel touches at most.
static long long extent(int C, int size, bool pairs) {
  const long long bytes = (long long)C * size * (pairs ? 2 : 1);
  long long reach = (15 + bytes + 15) / 16 * 16;  // fetch_row: all granules of a row that starts at byte 15 of one
  auto covers = [&](long long end) { reach = end > reach ? end : reach; };
  const long long last = (C - 1) / 8 * 8;                // first value of the last group of eight outputs
  const long long granules = size * 2 / 4 + 1;           // that read_staged loads for eight values
  covers((pairs ? 2 * last + 8 : last) * size + granules * 16);
  covers(15 + (last + 8) * size * (pairs ? 2 : 1));      // clear_staged: to the end of the last group
  if (!pairs) covers((last + 8) * size);                 // store: whole groups
  covers(last + 8);                                      // store_quantised
  covers((long long)C / 16 * 16 + 16);                   // send_row of q: one granule more than it sends
  covers(bytes / 16 * 16 + 16);                          // and of y or z
  return reach;
}

int main() {
  int bad = 0;
  for (int pairs = 0; pairs < 2; ++pairs)
    for (int size = 2; size <= 4; size += 2)
      for (int C = 1; C <= 5000; ++C) {
        const long long room = texo::row::staged_bytes((long long)C * size * (pairs ? 2 : 1));
        if (room % 16 != 0 || room < extent(C, size, pairs)) {
          if (++bad <= 5) std::printf("C = %d, %d bytes, pairs = %d: room %lld, touched %lld\n", C, size, pairs, room,
                                      extent(C, size, pairs));
        }
      }
  std::printf("%d lengths outside\n", bad);
  return bad != 0;
}
"""


def test_staged_rows_stay_inside_their_room(tmp_path):
    source, program = tmp_path / "room.cu", tmp_path / "room"
    source.write_text(PROGRAM)
    subprocess.run([build._nvcc(), *build.NVCC_FLAGS, "-I", build.CSRC, "-o", str(program), str(source)], check=True,
                   capture_output=True, timeout=600)
    run = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout

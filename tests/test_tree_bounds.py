"""What the tree attention kernels look up again in the block table, from their own header on the host: keys before the
sequence's end only, whose blocks the table has."""
import os
import subprocess

from ferrisinfer_amd import build

PROGRAM = """
#include "fi_tree.h"
#include <cstdio>

int main() {
  for (int end = -70; end <= 300; ++end)
    for (int k0 = 0; k0 <= 320; k0 += 32) {
      const uint64_t bits = fi::keys_before(end, k0);
      for (int key = 0; key < 64; ++key) {
        if (((bits >> key) & 1) != (k0 + key < end)) return printf("end %d chunk %d key %d\\n", end, k0, key), 1;
        // the block of a key that is looked up, in a table just as wide as the keys
        for (int block : {1, 5, 16, 128})
          if (((bits >> key) & 1) && (k0 + key) / block >= (end + block - 1) / block) return printf("block of %d\\n", k0 + key), 1;
      }
    }
  return fi::keys_before(0x7fffffff, 0) != ~0ull || fi::keys_before(1 << 30, (1 << 30) - 1) != 1;
}
"""


def test_keys_that_are_looked_up_lie_before_the_end(tmp_path):
    source, program = tmp_path / "bounds.hip", tmp_path / "bounds"
    source.write_text(PROGRAM)
    csrc = os.path.join(os.path.dirname(build.__file__), "csrc")
    subprocess.run([build.hipcc(), "-std=c++17", "-x", "hip", "--offload-host-only", "-I", csrc, "-o", str(program), str(source)],
                   check=True, capture_output=True, text=True)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout

"""How the losses over logits are split over the machine (csrc/loss_plan.h): host arithmetic, compiled here with the host
compiler and walked through over multiprocessor counts, rows and lengths of rows.

* Where no weights are given, the streaming kernel always finds the rows' weight in memory: it does not count them.  A
  device of few multiprocessors (a slice of one) streams fewer rows than the register kernels count themselves.
* The streaming kernel's buffers (8 of partial results, 13 chunks of the ring) rest on shares of two chunks or more, and
  of more than four in a cluster, for every row of a call, wherever it starts within 16 bytes.
"""

import os
import subprocess

from conftest import PKG_DIR

SOURCE = r"""
#include <cstdio>

#include "loss_plan.h"

using namespace kdn;

int main() {
  const int64_t lengths[] = {1, 2, 255, 256, 257, 511, 513, 1024, 1025, 2047, 2048, 2049, 2050, 4000, 4097, 9215, 9216,
                             9217, 9218, 12000, 18431, 18432, 18433, 20000, 36864, 36865, 36866, 50000, 73728, 73729,
                             1 << 20, 1 << 28};
  const int64_t rows[] = {1, 2, 15, 63, 64, 100, 128, 200, 255, 256, 257, 296, 300, 1000, 4096, 9999, 1 << 20};
  long streamed_few = 0;
  for (int sms = 1; sms <= 160; ++sms)
    for (int64_t vecs : lengths)
      for (int64_t n : rows) {
        const LossShape a{n, vecs, sms};
        const Stream st = choose_stream(a);
        const Split s = choose_split(a), scan = choose_scan_split(a);
        auto fail = [&](const char* what) {
          std::printf("%s: sms %d, vectors %lld, rows %lld\n", what, sms, (long long)vecs, (long long)n);
          return 1;
        };
        if (st.parts > 0 && counts_rows_itself(a, st)) return fail("a streamed call without its rows' weight");
        if (st.parts == 0 && counts_rows_itself(a, st) != (n <= kFewRows)) return fail("the rule for few rows");
        if (st.parts > 0 && n <= kFewRows) ++streamed_few;
        for (const Split& x : {s, scan})
          if (x.parts < 1 || x.parts > kMaxCluster || (x.threads != 32 && x.threads != 128 && x.threads != 256 &&
                                                       x.threads != 512))
            return fail("a split");
        if (st.parts == 0) continue;
        if (st.parts > kMaxCluster || st.per > 9 * kChunk) return fail("a share longer than the ring allows");
        const int64_t group = group_rows(a, st), chunks = (st.per + kChunk - 1) / kChunk;
        if (group < 1 || (group > 1 && group * chunks > 8) || group > 32) return fail("a group");
        for (int64_t nvec = vecs - 1; nvec <= vecs; ++nvec)
          for (int rank = 0; rank < st.parts; ++rank) {
            const int64_t share = std::min<int64_t>(st.per, nvec - int64_t(rank) * st.per);
            if (share <= (st.parts > 1 ? 4 * kChunk : kChunk)) return fail("a share of too few chunks");
          }
      }
  if (streamed_few == 0) return std::printf("no call of few rows was streamed\n"), 1;
  std::puts("ok");
}
"""


def test_plan(tmp_path):
    source, program = tmp_path / "plan.cpp", tmp_path / "plan"
    source.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(PKG_DIR, "csrc"), str(source), "-o",
                    str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.stdout == "ok\n", done.stdout

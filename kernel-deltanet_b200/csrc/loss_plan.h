// loss_plan.h -- how the losses over vocabulary logits are split over the machine: host arithmetic on a call's sizes
// (losses.cu has the kernels).
#pragma once

#include <stdint.h>

#include <algorithm>

namespace kdn {

constexpr int kMaxCluster = 8;
constexpr int kNV = 8;                       // vectors of a share that a thread keeps in registers
constexpr int kPer = 4;                      // vectors that a thread of a role of the streaming kernel takes at a time
constexpr int kRoleThreads = 256;            // of its statistics and of its gradient role
constexpr int kChunk = kPer * kRoleThreads;  // vectors of its ring's chunks: 16 KiB
constexpr int64_t kFewRows = 256;

struct LossShape {
  int64_t n;     // rows
  int64_t vecs;  // the most 16-byte vectors that one reaches into
  int sms;
};

// How a row is split: threads of a CTA and CTAs of a row's cluster.
struct Split {
  int threads, parts;  // threads of a row's CTA (32: a warp of one with four rows), CTAs of a row's cluster
};

// Kernels that keep a row's share in registers.  Many short rows: a warp each (B200, policy loss with gradient, bf16,
// 16384 x 1000: 27 us against 74 with 128 threads a row; 16384 x 4096: 65 against 92, but 600 x 4096: 10.8 against
// 9.1).  Else enough threads to hold the row, over more CTAs where one is too small, but (few rows being spread over
// the SMs at best) no more than two CTAs an SM.
inline Split choose_split(const LossShape& a) {
  const int64_t vecs = a.vecs, sms = a.sms;
  if ((vecs <= 256 && a.n >= 2 * sms) || (vecs <= 512 && a.n >= 8 * sms)) return Split{32, 1};
  Split s{vecs <= 128 * kNV ? 128 : vecs <= 256 * kNV ? 256 : 512, 1};
  while (s.parts < kMaxCluster && vecs > int64_t(s.threads) * kNV * s.parts && a.n * s.parts < 2 * sms) s.parts *= 2;
  return s;
}

// Log-probabilities alone read a row once and keep nothing of it: where there are rows enough, small CTAs in as many
// rounds as it takes (at different places of their rows, those of an SM keep the memory busy).  B200, bf16:
// 16384 x 4096 26 us with a warp a row, 53 with 128 threads; 4096 x 32000 47 us with 128 threads, 65 with the row in
// the registers of 512; 2400 x 131072 101 us with 256 threads, 107 with 128, 326 with a cluster of four times 512.
inline Split choose_scan_split(const LossShape& a) {
  if (a.n < 2 * a.sms) return choose_split(a);
  const int64_t vecs = a.vecs;
  return Split{vecs <= 1024 ? 32 : vecs <= 8192 ? 128 : 256, 1};
}

// The CTAs of a row's cluster and the vectors of each one's share in the streaming kernel; parts = 0: the rows are too
// long for its ring, which has to hold a row's share and what is being copied of the next one's, or it does not pay:
// rows of up to 32 KiB, or fewer than two an SM.  Measured on B200, policy loss with gradient, bf16, streaming kernel
// against CTAs that keep a row in registers: 2400 x 4096 30.3 us against 18.8, 148 x 32000 11.5 against 9.4, 600 x
// 32000 26.8 against 26.1, 2400 x 32000 69.4 against 77.2, 2400 x 131072 236 against 330.  The choice does not depend
// on whether a gradient is asked for, so that the outputs do not either.
struct Stream {
  int parts, per;
};
inline Stream choose_stream(const LossShape& a) {
  const int64_t vecs = a.vecs;
  if (vecs <= 2048 || a.n < 2 * a.sms) return {0, 0};
  for (int parts = 1; parts <= kMaxCluster; parts *= 2) {
    const int64_t per = (vecs + parts - 1) / parts;
    if (per <= 9 * kChunk) return {parts, int(per)};
  }
  return {0, 0};
}

// Rows of one request: as many as make 128 KiB, as long as that leaves every SM sixteen requests to even out what
// ignored rows save.
inline int64_t group_rows(const LossShape& a, Stream s) {
  const int64_t chunks = (s.per + kChunk - 1) / kChunk, most = a.n * s.parts / (16 * a.sms);
  return std::max<int64_t>(1, std::min<int64_t>(8 / chunks, most));
}

// Without weights a row's weight is one over the number of rows that count.  The kernels that keep rows in registers
// count a few rows themselves; the streaming kernel, and more rows, read the weight from memory, where a launch before
// theirs puts it.
inline bool counts_rows_itself(const LossShape& a, Stream s) { return s.parts == 0 && a.n <= kFewRows; }

}  // namespace kdn

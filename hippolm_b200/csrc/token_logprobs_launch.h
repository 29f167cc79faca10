// Launch shape of the per-token scores (plain C++, so that a test can walk it on the host).
#pragma once

namespace hippo {
constexpr int kLpWarps = 8;                          // warps of a block at most

// Warps of a block: as many as fill the card (32 a multiprocessor), and one for 10 segments or more (two for the alternatives),
// which amortise its start and the joining of its lanes; a power of two, as others leave a multiprocessor's registers unused.
// 4096 rows of 16000, 5 alternatives: 2 warps 39.8 us, 8 warps 51.3; of 32000 4 warps 60.6, 1 warp 73.5, 8 warps 70.1; of 64000 and
// 20 alternatives 4 warps 111, 6 warps 122, 8 warps 116; 8 rows of 4096 2.5 with 4 and more, 3.8 with 1. Rounded down against not
// rounded, 5 alternatives: 600 rows of 16000 4 warps 10.3, 7 warps 13.1; 900 rows 4 warps 12.4, 5 warps 15.6; 1200 rows 2 warps 16.4,
// 3 warps 15.4; 1500 rows of 4096 2 warps 9.5, 3 warps 10.6.
inline int logprob_warps(long long rows, int parts, int segs, int sms, bool alternatives) {
  int least = 1;
  while (least < kLpWarps && least * 2 <= (segs + 9) / 10) least *= 2;
  if (alternatives && least < 2) least = 2;
  long long most = 32ll * sms / (rows * parts);      // fills the card
  if (most < least) most = least;
  if (most > segs) most = segs;
  int warps = 1;
  while (warps < kLpWarps && warps * 2 <= most) warps *= 2;
  return warps;
}
}  // namespace hippo

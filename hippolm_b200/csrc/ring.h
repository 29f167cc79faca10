// Places of a ring of asynchronous copies (plain C++, so that a test can walk it on the host).
#pragma once
#ifdef __CUDACC__
#define HIPPO_HD __host__ __device__ __forceinline__
#else
#define HIPPO_HD inline
#endif

namespace hippo {
struct RingPlace { int stage, parity; };

// Stage and barrier parity of the copy that was issued `ahead` copies (0 .. stages - 1) after the one that is waited for next, at
// (stage, phase). Stages before `stage` were consumed in this round already: what is under way there completes the next phase.
HIPPO_HD RingPlace ring_place(int stage, int phase, int ahead, int stages) {
  const int at = stage + ahead;
  return at < stages ? RingPlace{at, phase} : RingPlace{at - stages, phase ^ 1};
}
}  // namespace hippo

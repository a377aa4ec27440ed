// A ring of STAGES pieces of shared memory that one thread keeps busy: loads run LEAD pieces ahead of the stores that empty them.
// What loads, waits and stores is the caller's `Io`, so that the order can be run without a GPU too:
//   io.read<N>()                    waits until no more than N stores still read their stages
//   io.load(stage, from...)         starts the load of a piece and notes where it goes
//   io.wait(stage, parity) -> bool  waits, with a limit, for a load
//   io.store(stage)                 starts the store of a piece that is there
//   io.finish()                     waits until all stores have been written
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define NVLLM_RING __device__ __forceinline__
#else
#define NVLLM_RING inline
#endif

namespace nvllm {

template <int STAGES, int LEAD, class Io>
struct CopyRing {
  static_assert(LEAD < STAGES, "a stage whose store is being read");
  Io& io;
  uint32_t loaded = 0, stored = 0;  // pieces: 2^32 of 16 KB are far more than a memory holds
  bool ok = true;

  template <class... From>
  NVLLM_RING void piece(From... from) {
    io.template read<STAGES - LEAD - 1>();  // the store that had the stage before has read it
    io.load(static_cast<int>(loaded % STAGES), from...);
    if (++loaded - stored > LEAD) store();
  }
  NVLLM_RING void store() {
    const int s = static_cast<int>(stored % STAGES);
    if (!(ok = io.wait(s, phase(stored)))) return;
    io.store(s);
    ++stored;
  }
  // False where a wait ran out: what is left is not stored, but waited for, the piece whose wait ran out too, so that no load is in
  // flight when the block gives its shared memory up.
  NVLLM_RING bool end() {
    while (ok && stored < loaded) store();
    for (uint32_t m = stored; m < loaded; ++m) (void)io.wait(static_cast<int>(m % STAGES), phase(m));
    io.finish();
    return ok;
  }
  static NVLLM_RING uint32_t phase(uint32_t m) { return m / STAGES & 1; }
};

}  // namespace nvllm

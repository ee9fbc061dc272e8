// Which part of a warp's staging buffer its next block takes, and how many of
// its bulk stores may still be reading theirs.
//
// The buffer has two halves of 2 KB.  A block of 16-bit entries takes one of
// them, the halves in turn, so that its stores overlap the one before; a
// block of float32 entries takes both.  Bulk stores complete in order, and the
// wait before a block can let the latest stand, which is safe only where that
// one reads the other half: after a 16-bit block that a bulk store took.
// After a float32 block, whose store reads both halves, and after a block that
// the warp copied out itself, which leaves an older store the latest, it has
// to be waited for too.  (Plain C++: tests/test_staging_turn.py runs it on the
// host.)
#pragma once

#if defined(__CUDACC__)
#define ML_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define ML_HOST_DEVICE inline
#endif

namespace ml {

constexpr int STAGING_HALF = 2048;

struct StagingTurn {
  int turn = 0;
  bool other_half = false;     // the latest bulk store, if it runs, reads the half that is not next

  struct Place {
    int offset;                // of the block in the buffer, bytes
    int stand;                 // bulk stores that may still run when it is written: 0 or 1
  };
  // wide: float32 entries; bulk: a bulk store takes the block away.
  ML_HOST_DEVICE Place next(bool wide, bool bulk) {
    const Place p{wide ? 0 : turn * STAGING_HALF, !wide && other_half ? 1 : 0};
    other_half = !wide && bulk;
    turn ^= 1;
    return p;
  }
};

}  // namespace ml

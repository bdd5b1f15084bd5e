// Launches that overlap the end of the grid before them on the stream: of the new grid only what touches no
// memory runs before that grid is complete (its launch, its prologue).  For kernels whose CTAs take some time to
// set up: window prefill back to back, 4 prompts of 64 to 512 tokens, 13.4 us without and 12.9 with; 8 layers
// of rotary and decode of 8 sequences, 102.5 and 101 us.  The rotary kernels, which have nothing to set up, lose by it
// (64 tokens 4.7 and 6.0 us: a CTA that waits takes up room and is let go later than a new one starts).
#pragma once

#include "common.cuh"

namespace aici {

// In the kernel, before its first access to global memory: waits for the grids before this one, then lets the
// next one start its own prologue.  Every grid that is launched as a dependent does both in this order, so that what is
// complete for one is complete for all behind it.  One grid is an exception: window prefill beside a launch for the
// short sequences of the same call (window_chunk.cuh) reads its inputs without the wait and lets nobody start early.
// That is sound only because the launch right before it is not a dependent itself (programmaticStreamSerializationAllowed
// = 0): it began when all that came before was complete, so whatever starts behind its first CTAs may read the same
// inputs.  CTA 0 waits before it leaves, so that both are complete for what follows.
__device__ __forceinline__ void dependent_start() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

inline cudaLaunchAttribute dependent_launch() {
  cudaLaunchAttribute a = {};
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  return a;
}

}  // namespace aici

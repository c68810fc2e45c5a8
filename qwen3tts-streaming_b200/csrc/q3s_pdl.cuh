// q3s_pdl.cuh -- programmatic dependent launch, device side.
#pragma once

#include "q3s_device.cuh"

namespace q3s {

// Programmatic dependent launch.  A grid launched with that attribute may start
// while the one before it in the stream ends: grid_wait returns once that one is
// complete and its writes are visible.  grid_release lets the next such grid
// start.
//
// A grid that has started finds everything before its predecessor complete,
// because every grid releases after its own wait.  The one that does not, the
// key-split kernel beside the prefix kernel, was itself started by a release
// that came after a wait: what it reads, and what the join reads before its
// wait (offsets and lengths), is older than the prefix kernel's predecessor's end.
// Anything that the predecessor itself may write is read after the wait only,
// weights included: without a release the dependent starts when the
// predecessor's blocks have ended, which is before their writes are flushed.
Q3S_DEV void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
Q3S_DEV void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace q3s

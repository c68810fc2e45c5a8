// q3s_pdl.cuh -- programmatic dependent launch, device side.
#pragma once

#include "q3s_device.cuh"

namespace q3s {

// Programmatic dependent launch.  A grid launched with that attribute may start
// while the one before it in the stream ends: grid_wait returns once that one is
// complete and its writes are visible.  grid_release lets the next such grid
// start; every grid here releases only after it has waited, so that a grid that
// has started is behind everything before its predecessor.  Before its own wait
// a grid touches nothing but the weights of a product, which no grid that
// releases early writes.
Q3S_DEV void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
Q3S_DEV void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace q3s

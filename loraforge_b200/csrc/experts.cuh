// Host functions shared by the expert products' translation units.
#pragma once

#include "common.cuh"

namespace lfb {

// Expired bounded waits counted by the two units (synchronous).
int grouped_wait_timeouts(unsigned int* value, int reset);
int mx_wait_timeouts(unsigned int* value, int reset);

}  // namespace lfb

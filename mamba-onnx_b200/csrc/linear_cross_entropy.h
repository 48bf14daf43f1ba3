// Internal interface of the loss from hidden states (linear_cross_entropy.cu).
#pragma once

namespace mamba_lce {

// The kernels' error word (a bounded wait that gave up): its code, or -1 when
// it cannot be read; cleared when set.
int read_and_clear_error();

}  // namespace mamba_lce

// Host helpers shared by the translation units of the C-ABI library; defined in scanscam_b200.cu.
#pragma once

#include <stdint.h>

namespace ssb_host {

// Records the message that ssb_last_error() returns on this host thread, and returns `status`.
int fail(int status, const char *fmt, ...);
// SSB_OK, or SSB_ERR_LAUNCH with the runtime's text for the launch just made.
int check_launch(const char *what);
int sm_count();  // of the current device (148 where no device answers)

// Reads and clears the device status word of state_space.cu; the caller has synchronised.
// Returns a cudaError_t.
int take_state_space_status(int word[2]);

}  // namespace ssb_host

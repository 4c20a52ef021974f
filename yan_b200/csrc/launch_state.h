#pragma once
// What the library's translation units share of its state.

namespace yan {

// The current device's status word (a bounded wait that runs out writes it); null if the device cannot be asked.
int* status_word_of_current_device();
// The bound of the waits inside one kernel.
unsigned long long wait_timeout_ns();

}  // namespace yan

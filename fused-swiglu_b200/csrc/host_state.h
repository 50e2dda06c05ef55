// What the host code of the library's translation units shares: the current device's one-time set-up and the launch
// count.  Defined in api.cu.
#pragma once

namespace fsw {

// SM count of the current device after its one-time set-up; a negative status where it cannot be used.
int current_device_sms(int* num_sms);
void count_launch();

}  // namespace fsw

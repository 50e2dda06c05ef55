// What the host code of the library's translation units shares: the current device's one-time set-up and the launch
// count.  Defined in api.cu.
#pragma once

namespace fsw {

// The current device after its one-time set-up; the call returns a negative status where it cannot be used.
struct Device {
  int index, sms;
  unsigned* status;                  // where a bounded wait that gave up is recorded
  unsigned long long wait_limit_ns;  // how long such a wait may last
};
int current_device(Device* out);
void count_launch();
// Whether the next launch is to leave out a copy (fswiglu_test_expire_next_wait); one launch, then it is not.
bool take_withhold();

}  // namespace fsw

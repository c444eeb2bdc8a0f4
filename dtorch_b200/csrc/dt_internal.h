// What the translation units of libdtorch_b200.so share: the calling thread's error message and the launch count.
#pragma once

#include <string>

namespace dtb {

// Record `msg` as the calling thread's last error and return `status`.
int set_error(int status, const std::string& msg);

// After a launch: DT_ERR_CUDA with the runtime's message, or count the kernel and return DT_OK.
int check_launch(const char* what);

// SM count of the current device, and its ordinal.
int current_device(int* dev, int* sms);

}  // namespace dtb

// host.hpp — host helpers shared by the library's translation units (defined in
// starkv_abi.cu).
#pragma once
#include <cstdint>

namespace starkv {

// Records `msg` as the thread's last error and returns `code`.
int host_error(int code, const char* msg);
// STARKV_OK, or the launch error of the kernels launched so far (recorded).
int host_launch_status();
// STARKV_OK when the current device is an sm_100 GPU; *sms gets its SM count.
int host_device(int* sms);
// Time limit of one device-side wait, and the copy that a test withholds (-1: none).
unsigned long long host_wait_limit();
int host_skip_unit();

}  // namespace starkv

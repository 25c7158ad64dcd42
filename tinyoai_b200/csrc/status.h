// Status and thread-local error text shared by the library's source files
// (the store itself is in runtime.cu).
#pragma once

namespace tcu {

// Records `message` as the calling thread's last error and returns `code`.
int set_error(int code, const char* message);

// TCU_OK when `device` exists and is sm_100; checked once per device. Leaves
// the current device as it was.
int require_device(int device);

}  // namespace tcu

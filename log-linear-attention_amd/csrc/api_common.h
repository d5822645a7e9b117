// What the files of C-ABI entry points share: status codes and the thread's last message.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/hattn.h"

namespace hattn_api {

extern thread_local char g_err[512];

// Stores the message and returns the code.
int fail(int code, const char* fmt, ...);
// Clears the message; HATTN_OK.
int ok();
// HATTN_OK, or HATTN_ERR_HIP with the name of what failed.
int check_hip(hipError_t e, const char* what);

}  // namespace hattn_api

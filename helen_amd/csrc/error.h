// error.h -- the C ABI's error text: one thread-local message for every source of libhelen_hip.so (helen_last_error)
#pragma once

namespace helen {

// records the message and returns `code`
int fail(int code, const char* fmt, ...);

}  // namespace helen

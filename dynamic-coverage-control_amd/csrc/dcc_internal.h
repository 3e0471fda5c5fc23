// Internal to libdcc_hip.so (not installed): the error channel shared by every translation unit.
#pragma once
#include <string>

// Records `msg` as the calling thread's last error (returned by dcc_last_error()) and returns `code`.
int dcc_fail(int code, const std::string& msg);

// The same where nothing may be thrown (a handler, a C entry): the code alone if there is no memory for the message.
template <typename... Parts>
int dcc_fail_nothrow(int code, const Parts&... parts) noexcept {
    try {
        return dcc_fail(code, (std::string() + ... + parts));
    } catch (...) {
        return code;
    }
}

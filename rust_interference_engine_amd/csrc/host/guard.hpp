// guard.hpp — C++ exceptions end at the C ABI: an error code, and the message in the
// caller's buffer.
#pragma once

#include "../common.hpp"

#include <algorithm>
#include <cstring>
#include <exception>
#include <string>

namespace rie {

inline void write_err(char *err, size_t len, const std::string &m) {
    if (!err || !len) return;
    size_t n = std::min(len - 1, m.size());
    std::memcpy(err, m.data(), n);
    err[n] = 0;
}

template <class F>
int32_t guarded(char *err, size_t err_len, F &&f) {
    try {
        f();
        return E_OK;
    } catch (const Error &e) {
        write_err(err, err_len, e.msg);
        return e.code;
    } catch (const std::exception &e) {
        write_err(err, err_len, std::string("internal error: ") + e.what());
        return E_RUNTIME;
    } catch (...) {
        write_err(err, err_len, "internal error");
        return E_RUNTIME;
    }
}

}  // namespace rie

// jfh_status helpers shared by the files that define C entry points.
#pragma once

#include "jfh.h"

#include "jfh_format.hpp"

#include <cstdio>
#include <exception>
#include <new>
#include <stdexcept>
#include <string>

namespace jfh::capi {

inline jfh_status ok() {
    jfh_status s{};
    s.code = JFH_STATUS_OK;
    return s;
}

inline jfh_status error(int32_t code, const char* message) {
    jfh_status s{};
    s.code = code;
    std::snprintf(s.message, sizeof(s.message), "%s", message);
    return s;
}

template <typename F>
jfh_status guarded(F&& fn) {
    try {
        fn();
        return ok();
    } catch (const jfh::Error& e) {
        return error(static_cast<int32_t>(e.code()), e.what());
    } catch (const std::invalid_argument& e) {
        return error(JFH_STATUS_INVALID_ARGUMENT, e.what());
    } catch (const std::bad_alloc&) {
        return error(JFH_STATUS_OUT_OF_MEMORY, "host allocation failed");
    } catch (const std::exception& e) {
        return error(JFH_STATUS_DEVICE_ERROR, e.what());
    }
}

inline void require(bool condition, const char* message) {
    if (!condition) throw jfh::Error(jfh::Status::InvalidArgument, message);
}

inline void require(bool condition, const std::string& message) { require(condition, message.c_str()); }

}  // namespace jfh::capi

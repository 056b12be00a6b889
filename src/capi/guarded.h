// What every entry of the C interface of the training operators shares.
#pragma once

#include "b200ccl/types.h"
#include "core/check.h"

#include <cstdint>
#include <exception>
#include <stdexcept>
#include <string>

namespace b200ccl::kernels {
void set_last_error_message(const std::string& message);  // b2_last_error() of the calling thread
}

namespace b200ccl::capi {

// 0, or the code of what f threw, whose message b2_last_error() has then: no exception leaves a C entry.
template <typename F>
int guarded(const char* what, F&& f) {
    try {
        f();
        return 0;
    } catch (const std::invalid_argument& e) {
        kernels::set_last_error_message(std::string(what) + ": " + e.what());
        return 2;
    } catch (const std::exception& e) {
        kernels::set_last_error_message(std::string(what) + ": " + e.what());
        return 1;
    } catch (...) {
        kernels::set_last_error_message(std::string(what) + ": unknown failure");
        return 1;
    }
}

inline DType dtype_of(int code) {
    B2_REQUIRE(code >= 0 && code <= 2, "unsupported dtype");
    return static_cast<DType>(code);
}

inline bool aligned(const void* p, std::size_t n) { return reinterpret_cast<std::uintptr_t>(p) % n == 0; }

}  // namespace b200ccl::capi

#pragma once

#include <string.h>

#include <type_traits>
#include <utility>

#include "common.cuh"

namespace wick {

// An entry point NAME a second time as NAME_packed, whose arguments lie in places of 8 bytes one behind the other (whole numbers and pointers
// as such, floating-point numbers as doubles): one argument for the caller to convert, which for 25 of them costs a quarter.
template <typename A> inline A packed_argument(const int64_t* at) {
    if constexpr (std::is_pointer_v<A>) {
        return reinterpret_cast<A>(*at);
    } else if constexpr (std::is_floating_point_v<A>) {
        double d;
        memcpy(&d, at, sizeof d);
        return (A)d;
    } else {
        return (A)*at;
    }
}
template <typename... A, size_t... I> inline int call_packed(int (*f)(A...), const int64_t* args, std::index_sequence<I...>) {
    return f(packed_argument<A>(args + I)...);
}
template <typename... A> inline int call_packed(int (*f)(A...), const int64_t* args) { return call_packed(f, args, std::index_sequence_for<A...>{}); }

}  // namespace wick

#define WICK_PACKED(NAME) \
    WICK_API int NAME##_packed(const int64_t* args) { return ::wick::call_packed(NAME, args); }

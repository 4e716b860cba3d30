// Calls at the C boundary, which no exception passes (compiles without HIP).
#pragma once

#include <new>

#include "jamhip.h"

namespace jamhip {

// call(); of an exception note(text) and JAMHIP_EINVAL, as of a device allocation that fails. The texts fit the 15 characters that a std::string
// holds in itself, so that a note which assigns one needs no memory.
template <class F, class N> jamhip_status noexcept_call(F&& call, N&& note) noexcept {
    try {
        return call();
    } catch (const std::bad_alloc&) {
        note("out of memory");
    } catch (...) {
        note("internal error");
    }
    return JAMHIP_EINVAL;
}

}  // namespace jamhip

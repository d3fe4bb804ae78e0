// What every entry point of the C ABI shares: the message behind sar_last_error() and the wall no exception passes.
#pragma once
#include <exception>
#include <new>
#include <string>

#include "sar.h"

namespace sar {

int set_error(int code, const std::string& msg);   // keeps msg for sar_last_error() on this thread, returns code

// Runs the body of an entry point; no exception leaves the C ABI.
template <class F> int guarded(F&& body) {
    try { return body(); }
    catch (const std::bad_alloc&) { return set_error(SAR_ENOMEM, "out of host memory"); }
    catch (const std::exception& e) { return set_error(SAR_EINVAL, e.what()); }
    catch (...) { return set_error(SAR_EINVAL, "unexpected error"); }
}

}  // namespace sar

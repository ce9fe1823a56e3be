// What cck_last_error() says of the calling thread's last failure, for every translation unit of the library.
#pragma once

namespace cck {

int report(int code, const char* message) noexcept; // keeps the message, returns the code

} // namespace cck

// The thread-local error string behind tft_last_error, shared by the library's sources.
#ifndef TORCHFT_AMD_ERRORS_H_
#define TORCHFT_AMD_ERRORS_H_

namespace tft {

// Stores the message for tft_last_error and returns `code`.
__attribute__((visibility("hidden"), format(printf, 2, 3))) int fail(int code, const char* fmt, ...);

}  // namespace tft

#endif  // TORCHFT_AMD_ERRORS_H_

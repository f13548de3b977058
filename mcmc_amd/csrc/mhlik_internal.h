// mhlik_internal.h -- what the translation units of libmhlik.so share (not part of the C-ABI).
#pragma once

namespace mhlik {

// Records the text mhlik_last_error(NULL) returns on this thread, and returns `code`.
__attribute__((visibility("hidden"), format(printf, 2, 3))) int fail_no_ctx(int code, const char *fmt, ...);

} // namespace mhlik

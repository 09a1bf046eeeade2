// runtime.hip -- libdkz_dense.so's plumbing and error context.
#include "companion.hpp"

extern "C" const char *dkz_dense_last_error_context(void) { return dkz::g_context; }

// runtime.hip -- libdkz_lm.so's plumbing and error context.
#include "companion.hpp"
#include "dkz_lm.h"

extern "C" const char *dkz_lm_last_error_context(void) { return dkz::g_context; }

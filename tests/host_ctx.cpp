// A context without a device, for tests of the checks that every entry point
// makes before it touches one.
#include "wm_internal.h"

extern "C" void *host_ctx() { return new wm_ctx(); }

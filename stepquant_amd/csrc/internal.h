// Shared by the library's translation units; not part of its C ABI.
#ifndef STEPQUANT_INTERNAL_H
#define STEPQUANT_INTERNAL_H

// Sets sq_last_error() of the calling thread and returns `code`.
__attribute__((visibility("hidden"))) int sq_internal_fail(int code, const char *msg);

// The pending launch error of the calling thread, reported under `what`; 0 when there is none.
__attribute__((visibility("hidden"))) int sq_internal_launched(const char *what);

#endif

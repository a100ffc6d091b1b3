// Shared by the library's translation units; not part of its C ABI.
#ifndef STEPQUANT_INTERNAL_H
#define STEPQUANT_INTERNAL_H

#include <stdint.h>

// Sets sq_last_error() of the calling thread and returns `code`.
__attribute__((visibility("hidden"))) int sq_internal_fail(int code, const char *msg);

// The pending launch error of the calling thread, reported under `what`; 0 when there is none.
__attribute__((visibility("hidden"))) int sq_internal_launched(const char *what);

// Host checks of a plan's schedule (any number of rows that a plan may have); 0, or
// the error that sq_last_error() then tells.
struct sq_kv_schedule;
__attribute__((visibility("hidden"))) int sq_internal_check_schedule(const struct sq_kv_schedule *s, int64_t tokens,
                                                                     int64_t batch);

#endif

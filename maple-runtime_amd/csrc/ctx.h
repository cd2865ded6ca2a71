// ctx.h -- the library context (mmoe.hip) as other translation units see it: one device, one stream, one error text.
#pragma once
#include <hip/hip_runtime.h>

#pragma GCC visibility push(hidden)
int mm_ready();                            // sets the context up once; -1 without a device
int mm_device();                           // the device it lives on (after mm_ready)
void mm_error(const char *fmt, ...);       // mmoe_last_error's text, also to stderr
int mm_launch(int kid, const void *f, dim3 g, dim3 b, void **args);   // one kernel on the library stream; profiled as kid
#pragma GCC visibility pop

// What the other translation units of libsage_hip.so need of a context (defined in sage_hip.hip).
#pragma once
#include "../../include/sage_hip.h"

__attribute__((visibility("hidden"))) int sage_ctx_device(const sage_ctx* c);
__attribute__((visibility("hidden"))) int sage_ctx_compute_units(const sage_ctx* c);
__attribute__((visibility("hidden"))) int sage_ctx_fail(sage_ctx* c, int code, const char* msg) noexcept;   // records msg, returns code

// Host-side helpers shared by the library's translation units: the thread's
// last error and the launch check behind every entry point's status.
#pragma once

#include <stdint.h>

#include <string>

namespace tq {

// Sets the thread's message and returns `code`.
__attribute__((visibility("hidden"))) int fail(int code, const std::string& msg);
// TQ_OK, or TQ_ERR_LAUNCH with the pending HIP error's text; clears the message.
__attribute__((visibility("hidden"))) int launch_status(const char* what);
__attribute__((visibility("hidden"))) int device_cu_count();

// Workgroups per launch of the row kernels (fwht, append, unpack, rotary,
// gate, page appends).  A HIP launch holds at most 2^32 - 1 work-items; larger
// calls are cut into launches of at most this many workgroups, in stream order.
constexpr int64_t kMaxLaunchBlocks = int64_t(1) << 20;

}  // namespace tq

// workspace.cuh -- the caller-owned device scratch behind b2_workspace.
#pragma once

#include <stddef.h>

// Arrival counters beside the lent bytes: cleared when the workspace is
// created, and left cleared by every kernel that uses them, so no call has to
// clear them first.
constexpr int kWsCounters = 4096;

struct b2_workspace {
    void* ptr = nullptr;
    size_t bytes = 0;
    int* counters = nullptr;
};

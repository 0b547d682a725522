// kv_cache.hpp -- launchers of the cache-row kernels (kv_cache.hip), arguments checked by the callers.
#pragma once

#include <hip/hip_runtime.h>
#include <kernelcore/llm_kernels.h>

namespace kcamd {

int launchSetRowsQ40(const kcSetRowsQ40Args& a, hipStream_t s);
int launchGetRowsQ40(const kcGetRowsQ40Args& a, hipStream_t s);
int launchKvKeep(const kcKvKeepArgs& a, hipStream_t s);
int launchKvGather(const kcKvGatherArgs& a, hipStream_t s);

}  // namespace kcamd

// kserve.hpp -- launchers of the operators of a step of many requests over a paged cache (kv_pages.hip, krope_ext.hip, kflash_pages.hip,
// ksample.hip), arguments checked by the callers.
#pragma once

#include <hip/hip_runtime.h>
#include <kernelcore/llm_kernels.h>

#include <cstdint>

namespace kcamd {

int launchKvPages(const kcKvPagesArgs& a, hipStream_t s);
int launchRopeExt(const kcRopeExtArgs& a, hipStream_t s);
int launchFlashPages(const kcFlashPagesArgs& a, hipStream_t s);
size_t flashPagesPartBytes(const kcFlashPagesDims& d);
int launchSampleRows(const kcSampleRowsArgs& a, hipStream_t s);
size_t sampleRowsPartBytes(int rows, int n_vocab);

}  // namespace kcamd

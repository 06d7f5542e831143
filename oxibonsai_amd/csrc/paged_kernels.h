// paged_kernels.h — launch interface of a serving step's operators over a paged cache (see paged_kernels.hip, paged_attention.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/oxb_hip.h"

#define OXB_PAGED_MAX_REQUESTS 4096u
#define OXB_PAGED_MAX_GROUP 16u  // q heads to a kv head

hipError_t oxb_launch_paged_assign(const oxb_page_assign& a, hipStream_t st);
hipError_t oxb_launch_paged_rows(const oxb_paged_rows& a, hipStream_t st);
hipError_t oxb_launch_paged_attention(const oxb_paged_attention& a, hipStream_t st);
// Bytes of workspace: what any lengths can make the device's own split of the work need at these counts.
size_t oxb_paged_attention_workspace(const oxb_paged_attention& a);

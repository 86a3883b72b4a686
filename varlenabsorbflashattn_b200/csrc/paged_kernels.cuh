// Rotation of packed queries and keys, append to a paged key/value cache, attention over it: host-side launchers.
#pragma once
#include "common.cuh"

namespace vafa {

// Codes of the status word beside those of report_error(): a length, page or position that leaves its array.
constexpr int kBadCacheIndex = 4;
constexpr int kSiteRotary = 910, kSiteAppend = 911, kSiteDecode = 912;

int rotary_launch(const vafa_rotary_args* a, cudaStream_t s);
int paged_append_launch(const vafa_paged_append_args* a, cudaStream_t s);

size_t paged_decode_workspace(const vafa_paged_attn_args* a);
int paged_decode_launch(const vafa_paged_attn_args* a, cudaStream_t s);

}  // namespace vafa

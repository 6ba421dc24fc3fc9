// What the kernels that append tokens to the page pools share: where a token goes, and the copies that stage its rows.
#pragma once

#include <stdint.h>

namespace pal {

__device__ __forceinline__ void cp_async_16(void* smem_dst, const void* gmem_src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem_dst)), "l"(gmem_src)
               : "memory");
}

// (page, slot) of token t, or page = -1 when the token has to be skipped
template <bool kSlots>
__device__ __forceinline__ void token_destination(long long t, const int64_t* slot_mapping, const uint32_t* page_table,
                                                  const int32_t* write_positions, const uint32_t* query_to_seq_map,
                                                  int num_seqs, int tokens_per_page, long long num_pages,
                                                  int max_pages_per_seq, long long& page, int& slot) {
  page = -1;
  slot = 0;
  if (kSlots) {
    const long long s = slot_mapping[t];
    if (s < 0 || s >= num_pages * tokens_per_page) return;
    page = s / tokens_per_page;
    slot = (int)(s - page * tokens_per_page);
  } else {
    const uint32_t seq = query_to_seq_map[t];
    const int pos = write_positions[t];
    if (pos < 0 || seq >= (uint32_t)num_seqs) return;
    const int block = pos / tokens_per_page;
    if (block >= max_pages_per_seq) return;
    const long long pg = page_table[(long long)seq * max_pages_per_seq + block];
    if (pg >= num_pages) return;
    page = pg;
    slot = pos - block * tokens_per_page;
  }
}

}  // namespace pal

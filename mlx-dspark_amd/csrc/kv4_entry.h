// The 4-bit form of dsk_qkv_rope_append (kv4.hip), behind that entry's argument checks.
#pragma once

#include "common.h"

namespace dsk {

int kv4_append(const void* qkv, int splits, int B, int W, int nq, int nkv, int hd, const uint16_t* q_norm,
               const uint16_t* k_norm, const uint16_t* v_norm, float eps, const float* inv_freq,
               const int32_t* seq_lens, int pos_offset, const int32_t* block_table, int max_pages, int page,
               void* k_pool, void* v_pool, uint32_t* k_sb, uint32_t* v_sb, uint16_t* q_out, const float* x_ssq,
               int x_tiles, float x_eps, hipStream_t st);

}  // namespace dsk

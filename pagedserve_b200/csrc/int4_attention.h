// Shared declarations of the 4-bit attention translation units.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace psb {

struct Int4DecodeParams {
  const void* q;
  int64_t qsb, qsh;  // elements
  void* out;
  int64_t osb, osh;
  const uint8_t* codes;
  const void* params;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* ctx;
  int32_t batch, hq, hkv, group, block_size, head_dim, max_context;
  int64_t num_blocks;
  int64_t layer_tiles;  // layer * num_blocks * hkv
  float scale_log2;     // scale * log2(e)
  float* part;          // split partials
  int32_t* err;
};

struct Int4PrefillParams {
  const void* q;
  int64_t qst, qsh;
  void* out;
  int64_t ost, osh;
  const uint8_t* codes;
  const void* params;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* ctx;
  const int32_t* cu;
  int32_t num_seqs, total, max_seqlen, max_context, hq, hkv, block_size, head_dim;
  int64_t num_blocks;
  int64_t layer_tiles;
  float scale_log2;
  int32_t* err;
};

}  // namespace psb

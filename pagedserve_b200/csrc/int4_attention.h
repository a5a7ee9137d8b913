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
  uint64_t tile_div;    // tensor-core path: 2^32 / (block_size / 16), rounded up
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

// Tensor-core decode (int4_decode_fast.cu): whether a geometry is covered, its
// scratch bytes and the launch.  q rows and out rows start on 16 bytes.
bool int4_decode_fast_geometry(int dtype, int batch, int hkv, int group, int head_dim, int block_size,
                               int max_context, int num_layers, int64_t num_blocks);
size_t int4_decode_fast_workspace(int group, int head_dim);
int int4_decode_fast_launch(const Int4DecodeParams& p, int dtype, cudaStream_t s);

// Tensor-core prefill (int4_prefill_tc.cu): whether a geometry is covered, its
// scratch bytes and the launch.  q rows start on 16 bytes.
bool int4_prefill_tc_geometry(int dtype, int total, int num_seqs, int q_heads, int hkv, int head_dim, int block_size,
                              int max_context);
size_t int4_prefill_tc_workspace(int total, int num_seqs, int q_heads, int hkv, int max_context);
int int4_prefill_tc_launch(const Int4PrefillParams& p, int dtype, float* workspace, cudaStream_t s);

}  // namespace psb

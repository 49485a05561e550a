// Parameters of the attention over a shared prefix by many queries per key (5th-generation tensor cores).
#pragma once
#include "quant_cache.cuh"

namespace ra {

constexpr int kPrefixTile = 128;               // tokens of a K or V tile, and queries of a Q tile
constexpr int kPrefixHalf = kPrefixTile * 128; // one swizzled [128 rows][128 bytes] block
constexpr int kPrefixTileBytes = 2 * kPrefixHalf;

struct PrefixAttendParams {
  CUtensorMap kmap, vmap;   // boxes of 128 tokens of one head, 128 bytes wide
  const void* q;            // [batch, hq, 128]
  const float* k_scale;     // of codes: [hkv][tokens], scale_hstride floats between heads
  const float* v_scale;
  long long scale_hstride;
  float* part_o;            // [(kv head, query tile)][splits][128][128] un-normalised sums
  float* part_ml;           // same, [2]: maximum (log2 domain), weight
  unsigned* status;
  int n_tokens, queries;    // queries of a kv head: batch * group
  int query_tiles;          // ceil(queries / 128)
  int hq, hkv, group;
  int splits;
  float scale_log2e;
  int early;                // launched while the kernel before it still runs
};

// format: not int4, whose scales lie along the dims and cannot be applied to S
cudaError_t launch_prefix_attend(const PrefixAttendParams& P, int format, bool bf16, cudaStream_t stream);

}  // namespace ra

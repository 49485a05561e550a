// Parameters of decode attention over a prefix shared by the batch and each row's own cache.
#pragma once
#include "quant_cache.cuh"

namespace ra {

constexpr int kAttendTile = 64;                // tokens per pipeline stage
constexpr int kAttendWarps = 4;                // consumer warps, 16 tokens of a tile each
constexpr int kAttendThreads = 32 * (kAttendWarps + 1);
constexpr int kAttendMaxStages = 8;
// scales of a tile, K's and then V's
__host__ __device__ constexpr int attend_scale_floats(int format) { return 2 * kAttendTile * cache_row_scales(format); }
// What beginning and ending a work row costs, in tiles: loading its queries, merging the warps' sums.
constexpr int kAttendRowUnits = 2;
// CTAs per multiprocessor: three with 8 query columns (128 registers a thread), two with 16
__host__ __device__ constexpr int attend_ctas(int nq) { return nq == 1 ? 3 : 2; }

// One segment of the keys: the prefix (one cache, all batch rows' queries) or the rows' own caches.
// A work row is (cache, kv head, tile of queries).  The rows lie on a line, one behind the other, cache
// by cache, each as long as what it costs: kAttendRowUnits and then a unit for each tile of tokens.  CTA
// c of the first G = min(grid, total) takes the units [total c / G, total (c+1) / G), whatever rows they
// belong to, and leaves one partial for each row of which it has tiles, in slot row + c: along the line
// one of the two grows at every step, so the slots are distinct.
struct AttendSegment {
  CUtensorMap kmap, vmap;
  CacheView cache;
  const int* lens;          // [caches] or null: every cache is n_tokens long
  int caches;               // 1 for the prefix
  int queries;              // of a work row's (cache, kv head): group, or batch * group for the prefix
  int query_tiles;          // ceil(queries / (8 NQ))
  int grid;                 // CTAs
  int nstages;
  float* part_o;            // [slots][8 NQ][128] un-normalised sums
  float* part_ml;           // [slots][8 NQ][2] maximum (log2 domain), weight
  int* span;                // [rows][2]: first and last CTA with tiles of the row (of one with tokens)
};

struct CacheAttendParams {
  AttendSegment seg;
  const void* q;            // fp16 or bf16 [batch, hq, 128]
  unsigned* status;
  int hq, hkv, group;
  float scale_log2e;
  int after;                // launched while the prefix's kernel still runs: needs nothing of it, but
                            // ends behind it, so that the combine need only wait for this one
  int early;                // launched with the programmatic attribute
};

// What the combine reads of a segment.
struct CombineSegment {
  const float* part_o;      // null: no such segment
  const float* part_ml;
  const int* span;
  const int* lens;
  int query_tiles, qt, prefix;
  int splits;               // > 0: a row's partials lie in so many slots of its own
};
struct CombineParams {
  CombineSegment seg[2];
  void* out;
  int batch, hq, hkv, group;
};

cudaError_t launch_cache_attend(const CacheAttendParams& P, int format, bool bf16, int nq, cudaStream_t stream);
cudaError_t launch_cache_combine(const CombineParams& P, bool bf16, cudaStream_t stream);
int cache_attend_stages(int format, int nq);

}  // namespace ra

// Parameters of decode attention over a prefix shared by the batch and each row's own cache.
#pragma once
#include "quant_cache.cuh"

namespace ra {

constexpr int kAttendTile = 64;                // tokens per pipeline stage
constexpr int kAttendWarps = 4;                // consumer warps, 16 tokens of a tile each
constexpr int kAttendThreads = 32 * (kAttendWarps + 1);
constexpr int kAttendMaxStages = 8;
// CTAs per multiprocessor: three with 8 query columns (128 registers a thread), two with 16
__host__ __device__ constexpr int attend_ctas(int nq) { return nq == 1 ? 3 : 2; }

// One segment of the keys: the prefix (one cache, all batch rows' queries) or the rows' own caches.
// A work row is (cache, kv head, tile of queries); its tiles of tokens lie one behind the other, and so
// do the rows of a cache and the caches.  CTA c of the first G = min(grid, total) takes the tiles
// [total c / G, total (c+1) / G) of that line, whatever rows they belong to, and leaves one partial for each row it touches, in slot row + c:
// along the line one of the two grows at every step, so the slots are distinct.
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
  long long* line;          // [caches + 1]: tiles of (kv head, query tile) before each cache
};

struct CacheAttendParams {
  AttendSegment seg;
  const void* q;            // fp16 or bf16 [batch, hq, 128]
  unsigned* status;
  int hq, hkv, group;
  float scale_log2e;
};

// What the combine reads of a segment.
struct CombineSegment {
  const float* part_o;      // null: no such segment
  const float* part_ml;
  const long long* line;
  int queries, query_tiles, qt, grid, prefix;
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

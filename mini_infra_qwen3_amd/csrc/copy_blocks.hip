// Block copies inside the pools: block dst[i] = block src[i] of every layer, K and V.
//
// For forks (a continuation's copy of the block that its parent goes on writing) and for compaction (live blocks
// of the pool's upper part moved to free ones of its lower part); the reference has neither, its blocks are only
// handed out and freed (src/mini_infra/core/block_manager.py:35-76).  Bytes are copied as they are, so a pool's
// type and layout do not matter.
//
// Like the block records (kv_block_records.hip), kSplit workgroups share one layer's K or V block, 16 bytes a lane, but
// a layer's K or V is done for all pairs before the next: 1000 blocks of 28 layers of a 2200-block pool (1.84 GB each way)
// 666 us, 5.5 TB/s; with all layers of a pair in turn, as records lie, 728.  Splits of 8 to 32 with
// fewer threads, other stores and runs per XCD within 1%; one workgroup a block 693, ordinary loads 684, 512 or 1024 threads
// 685 to 704.  (Copies into randomly placed 32 KiB units reach 5.6 to 5.7 TB/s on this card.)
#include "mi_common.h"

namespace mi {
namespace {

constexpr int kThreads = 256;
constexpr int kSplit = 8;  // workgroups per block of one layer's K or V

struct CopyArgs {
  char* pool[2][kMaxLayersPerLaunch];  // [0] = key pools, [1] = value pools of this launch's layers
  const int64_t* src;
  const int64_t* dst;
  int64_t num_blocks;
  int64_t block_bytes;
  uint32_t pieces;  // block_bytes / sizeof(V)
  uint32_t pairs;
};

template <typename V>
__global__ __launch_bounds__(kThreads) void copy_blocks_kernel(const CopyArgs a) {
  const uint32_t part = blockIdx.x % kSplit;
  const uint32_t piece_id = blockIdx.x / kSplit;
  const uint32_t plane = piece_id / a.pairs;  // layer and K / V
  const uint32_t i = piece_id - plane * a.pairs;
  const int kv = plane & 1, layer = plane >> 1;
  const int64_t to = a.dst[i];
  int64_t from = a.src[i];
  if (from < 0 || from >= a.num_blocks) from = 0;                    // a read: the null block
  if (to < 0 || to >= a.num_blocks || to == from) return;            // a write: skipped
  const V* src = reinterpret_cast<const V*>(a.pool[kv][layer] + from * a.block_bytes);
  V* dst = reinterpret_cast<V*>(a.pool[kv][layer] + to * a.block_bytes);
  const uint32_t per_part = (a.pieces + kSplit - 1) / kSplit;
  const uint32_t p1 = min(a.pieces, (part + 1) * per_part);
  for (uint32_t p = part * per_part + threadIdx.x; p < p1; p += kThreads)
    store_stream<true>(dst + p, load_vec<true>(src + p));
}

}  // namespace
}  // namespace mi

extern "C" int32_t mi_copy_blocks(void* const* key_pools, void* const* value_pools, int64_t num_blocks,
                                  const int64_t* src_blocks, const int64_t* dst_blocks, int64_t num_pairs,
                                  int32_t num_layers, int64_t block_bytes, void* stream) {
  using namespace mi;
  const char* name = "mi_copy_blocks";
  if (num_pairs < 0 || num_layers < 0 || num_blocks < 0 || block_bytes < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: negative size", name);
  // A pool without blocks has no destination: every pair is skipped.
  if (num_pairs == 0 || num_layers == 0 || block_bytes == 0 || num_blocks == 0) return ok();
  if (!key_pools || !value_pools || !src_blocks || !dst_blocks)
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: null pointer argument", name);
  bool wide = block_bytes % 16 == 0;
  for (int l = 0; l < num_layers; ++l) {
    if (!key_pools[l] || !value_pools[l])
      return fail(MI_ERR_INVALID_ARGUMENT, "%s: null pointer for layer %d", name, l);
    wide = wide && aligned16(key_pools[l]) && aligned16(value_pools[l]);
  }
  const int64_t piece = wide ? 16 : (block_bytes % 4 == 0 ? 4 : (block_bytes % 2 == 0 ? 2 : 1));
  if (block_bytes / piece > 0x7fffffff)
    return fail(MI_ERR_UNSUPPORTED, "%s: block of %lld bytes not supported", name, static_cast<long long>(block_bytes));
  // A grid dimension holds fewer than 2^32 threads.
  const int most = num_layers < kMaxLayersPerLaunch ? num_layers : kMaxLayersPerLaunch;
  if (num_pairs > 0xffffffffll / kThreads / (kSplit * 2 * most))
    return fail(MI_ERR_UNSUPPORTED, "%s: too many pairs in one call", name);
  CopyArgs a{};
  a.src = src_blocks;
  a.dst = dst_blocks;
  a.num_blocks = num_blocks;
  a.block_bytes = block_bytes;
  a.pieces = static_cast<uint32_t>(block_bytes / piece);
  a.pairs = static_cast<uint32_t>(num_pairs);
  for (int l0 = 0; l0 < num_layers; l0 += kMaxLayersPerLaunch) {
    const int nl = num_layers - l0 < kMaxLayersPerLaunch ? num_layers - l0 : kMaxLayersPerLaunch;
    for (int l = 0; l < nl; ++l) {
      a.pool[0][l] = static_cast<char*>(key_pools[l0 + l]);
      a.pool[1][l] = static_cast<char*>(value_pools[l0 + l]);
    }
    const uint32_t groups = static_cast<uint32_t>(num_pairs * nl * 2 * kSplit);
    if (piece == 16)
      copy_blocks_kernel<u32x4><<<groups, kThreads, 0, as_stream(stream)>>>(a);
    else if (piece == 4)
      copy_blocks_kernel<uint32_t><<<groups, kThreads, 0, as_stream(stream)>>>(a);
    else if (piece == 2)
      copy_blocks_kernel<uint16_t><<<groups, kThreads, 0, as_stream(stream)>>>(a);
    else
      copy_blocks_kernel<uint8_t><<<groups, kThreads, 0, as_stream(stream)>>>(a);
    if (const int32_t rc = check_launch(name)) return rc;
  }
  return ok();
}

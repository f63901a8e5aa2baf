// The 4-bit pools' copies: quantising scatter of new K/V rows, and dequantising gather of whole blocks.
//
// Counterparts, for pools of 4-bit records (fp4_record.h), of mi_reshape_and_cache and mi_gather_blocks: the
// reference's PagedKVCachePool.write_prefill, its decode append and PagedKVCachePool.gather_blocks
// (src/mini_infra/worker/paged_kv_cache.py:54-95, src/mini_infra/model/qwen3.py:282-283).
//
// Both take a lane for eight values of a row (four code bytes), sixteen lanes for the row.
#include "fp4_record.h"

namespace mi {
namespace {

constexpr int kThreads = 256;
constexpr int kStoreTokens = kThreads / 16;  // tokens of a workgroup of the store
constexpr int kGatherThreads = 512;
constexpr int kGatherHeads = 8;              // KV heads of a workgroup of the gather

struct StoreArgs {
  const char* src[2][kMaxLayersPerLaunch];  // [0] keys, [1] values
  char* pool[2][kMaxLayersPerLaunch];
  int64_t row[2], head[2], pos[2];          // source strides, bytes
  const int64_t* token_rows;
  const int64_t* token_positions;
  const int64_t* slots;
  int64_t index_stride;
  int64_t num_tokens, num_rows, num_positions, num_slots;
  int32_t kv_heads;
};

// Eight source elements as fp32: kBytes 2 (kHalf: fp16, else bf16) or 4.  kWide: 16-byte aligned pieces.
enum class Source { kBf16, kFp16, kFp32 };
template <Source kType, bool kWide>
__device__ __forceinline__ void load8(float (&x)[8], const char* p) {
  if constexpr (kType == Source::kFp32) {
    if constexpr (kWide) {
      const u32x4 a = load_vec<true>(reinterpret_cast<const u32x4*>(p)), b = load_vec<true>(reinterpret_cast<const u32x4*>(p) + 1);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t ae = a[e], be = b[e];
        x[e] = __uint_as_float(ae);
        x[4 + e] = __uint_as_float(be);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = reinterpret_cast<const float*>(p)[e];
    }
  } else {
    uint32_t w[4];
    if constexpr (kWide) {
      const u32x4 a = load_vec<true>(reinterpret_cast<const u32x4*>(p));
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = a[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t lo = reinterpret_cast<const uint16_t*>(p)[2 * e], hi = reinterpret_cast<const uint16_t*>(p)[2 * e + 1];
        w[e] = lo | (hi << 16);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (kType == Source::kBf16) {
        x[2 * e] = bf16_lo(w[e]);
        x[2 * e + 1] = bf16_hi(w[e]);
      } else {
        x[2 * e] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[e])));
        x[2 * e + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[e] >> 16)));
      }
    }
  }
}

// One workgroup: kStoreTokens index entries of one KV head of one layer, K and V.  A wavefront's four rows are
// four entries; where they are the tokens of a quad of one block (a prompt's store), its V codes are 256
// contiguous bytes.
//
// Bound by memory: 3614 tokens of four prompts, 28 layers of 8 heads (525 MB) in 105 us, 5.0 TB/s.  How the work is laid out
// moves little: 2 or 4 layers a workgroup, a record's neighbours kept on one XCD, 128 to 1024 threads 101 to 110; K and V
// in workgroups of their own 125.  Ordinary loads take 112, nontemporal stores 124 (a record's lines are filled by several
// wavefronts, which the L2 joins).
template <Source kType, bool kWide>
__global__ __launch_bounds__(kThreads) void fp4_store_kernel(const StoreArgs a) {
  const int h = static_cast<int>(blockIdx.x % a.kv_heads);
  const int layer = blockIdx.y;
  const int64_t i = static_cast<int64_t>(blockIdx.x / a.kv_heads) * kStoreTokens + threadIdx.x / 16;
  const int j = threadIdx.x & 15;
  int64_t slot = -1, row = i, position = 0;
  if (i < a.num_tokens) {
    slot = a.slots[i * a.index_stride];
    if (a.token_rows) row = a.token_rows[i * a.index_stride];
    if (a.token_positions) position = a.token_positions[i * a.index_stride];
  }
  const bool live = slot >= 0 && slot < a.num_slots && row >= 0 && row < a.num_rows && position >= 0 &&
                    position < a.num_positions;  // one row of 16 lanes: all or none of a quad
  float x[2][8];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[c][e] = 0.0f;
    if (live) {
      constexpr int kBytes = kType == Source::kFp32 ? 4 : 2;
      load8<kType, kWide>(x[c], a.src[c][layer] + row * a.row[c] + h * a.head[c] + position * a.pos[c] + 8 * kBytes * j);
    }
  }
  const int64_t record = (slot / kFp4Tokens) * a.kv_heads + h;
  const int t = static_cast<int>(slot % kFp4Tokens);
#pragma unroll
  for (int c = 0; c < 2; ++c) fp4_store_piece(a.pool[c][layer] + record * kFp4Record, c == 1, t, j, x[c], live);
}

struct GatherArgs {
  const char* pool[2][kMaxLayersPerLaunch];
  char* out[2][kMaxLayersPerLaunch];
  const int64_t* block_ids;
  int64_t block_id_stride;
  int64_t num_blocks;
  int32_t nb;
  int32_t kv_heads;
  int32_t head_groups;  // ceil(kv_heads / kGatherHeads)
};

// One workgroup: up to kGatherHeads KV heads of one block of one table entry, K or V of one layer.  Their records are
// contiguous and go to LDS in whole 16-byte pieces; a row's 16 pieces of output are 16 lanes.
//
// Bound by memory: 1.75 GB (28 layers, 32 sequences of up to 1150 tokens, 8 heads) in 262 us, 6.7 TB/s, what a plain copy
// reaches; without LDS, a lane reading its own four code bytes, 422.  256 threads 291, and 315 with nontemporal loads (a
// record's second half is a line of its neighbour's); 4 heads a workgroup as fast here, but 12.2 us against 11.5 for one
// sequence of 1024 tokens; ordinary stores 359 against 315, nontemporal ones without sc1 335.
__global__ __launch_bounds__(kGatherThreads) void fp4_gather_kernel(const GatherArgs a) {
  __shared__ __align__(16) unsigned char s_rec[kGatherHeads * kFp4Record];
  const int layer = blockIdx.y / a.head_groups;
  const int h0 = static_cast<int>(blockIdx.y % a.head_groups) * kGatherHeads;
  const int heads = min(kGatherHeads, a.kv_heads - h0);
  const int c = blockIdx.z;
  const int64_t b = blockIdx.x / a.nb, j = blockIdx.x % a.nb;
  int64_t id = a.block_ids[b * a.block_id_stride + j];
  if (id < 0 || id >= a.num_blocks) id = 0;
  const u32x4* block = reinterpret_cast<const u32x4*>(a.pool[c][layer] + (id * a.kv_heads + h0) * kFp4Record);
  for (int x = threadIdx.x; x < heads * (kFp4Record / 16); x += kGatherThreads)
    reinterpret_cast<u32x4*>(s_rec)[x] = block[x];
  __syncthreads();
  char* out = a.out[c][layer] + (static_cast<int64_t>(blockIdx.x) * kFp4Tokens * a.kv_heads + h0) * (2 * kFp4Dim);
  const int octet = threadIdx.x & 15;
  for (int row = threadIdx.x >> 4; row < kFp4Tokens * heads; row += kGatherThreads / 16) {
    const int t = heads == kGatherHeads ? row / kGatherHeads : row / heads;
    const int h = row - t * heads;
    const unsigned char* rec = s_rec + h * kFp4Record;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(rec + fp4_code_at(c == 1, t, octet));
    const uint32_t scale = rec[fp4_scale_at(c == 1, t, octet)];
    store_stream<true>(reinterpret_cast<u32x4*>(out + (static_cast<int64_t>(t) * a.kv_heads + h) * (2 * kFp4Dim)) + octet,
                       fp4_unpack8(codes, e8m0_f32(scale)));
  }
}

template <Source kType>
void launch_store(const StoreArgs& a, bool wide, dim3 grid, hipStream_t s) {
  if (wide)
    fp4_store_kernel<kType, true><<<grid, kThreads, 0, s>>>(a);
  else
    fp4_store_kernel<kType, false><<<grid, kThreads, 0, s>>>(a);
}

constexpr int64_t kMaxGroups = 0xffffffffll / kThreads;  // a grid dimension holds fewer than 2^32 threads

}  // namespace
}  // namespace mi

extern "C" int32_t mi_reshape_and_cache_fp4(const void* const* key_src, const void* const* value_src,
                                            int64_t key_row_stride, int64_t key_head_stride, int64_t key_pos_stride,
                                            int64_t value_row_stride, int64_t value_head_stride,
                                            int64_t value_pos_stride, const int64_t* token_rows,
                                            const int64_t* token_positions, const int64_t* slot_mapping,
                                            int64_t index_stride, int64_t num_tokens, int64_t num_src_rows,
                                            int64_t num_src_positions, void* const* key_pools,
                                            void* const* value_pools, int32_t num_layers, int64_t num_slots,
                                            int32_t num_kv_heads, int32_t head_dim, int32_t src_type, void* stream) {
  using namespace mi;
  const char* name = "mi_reshape_and_cache_fp4";
  if (num_tokens < 0 || num_layers < 0 || num_slots < 0 || num_src_rows < 0 || num_src_positions < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: negative size", name);
  if (num_tokens == 0 || num_layers == 0 || num_src_rows == 0 || num_src_positions == 0) return ok();
  if (!key_src || !value_src || !key_pools || !value_pools || !slot_mapping)
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: null pointer argument", name);
  if (num_kv_heads <= 0) return fail(MI_ERR_INVALID_ARGUMENT, "%s: %d KV heads", name, num_kv_heads);
  if (head_dim != kFp4Dim) return fail(MI_ERR_UNSUPPORTED, "%s: head_dim %d, needs %d", name, head_dim, kFp4Dim);
  if (src_type != MI_TYPE_BF16 && src_type != MI_TYPE_FP16 && src_type != MI_TYPE_FP32)
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: source type %d", name, src_type);
  if (index_stride <= 0) return fail(MI_ERR_INVALID_ARGUMENT, "%s: index_stride must be > 0", name);
  const int64_t tiles = (num_tokens + kStoreTokens - 1) / kStoreTokens;
  if (tiles > kMaxGroups / num_kv_heads) return fail(MI_ERR_UNSUPPORTED, "%s: too many tokens", name);
  const int bytes = src_type == MI_TYPE_FP32 ? 4 : 2;

  StoreArgs a{};
  a.token_rows = token_rows;
  a.token_positions = token_positions;
  a.slots = slot_mapping;
  a.index_stride = index_stride;
  a.num_tokens = num_tokens;
  a.num_rows = num_src_rows;
  a.num_positions = num_src_positions;
  a.num_slots = num_slots;
  a.kv_heads = num_kv_heads;
  const int64_t strides[2][3] = {{key_row_stride, key_head_stride, key_pos_stride},
                                 {value_row_stride, value_head_stride, value_pos_stride}};
  bool wide = true;
  for (int c = 0; c < 2; ++c) {
    a.row[c] = strides[c][0] * bytes;
    a.head[c] = strides[c][1] * bytes;
    a.pos[c] = strides[c][2] * bytes;
    for (int64_t st : {a.row[c], a.head[c], a.pos[c]}) wide = wide && st % 16 == 0;
  }
  for (int l = 0; l < num_layers; ++l) {
    if (!key_src[l] || !value_src[l] || !key_pools[l] || !value_pools[l])
      return fail(MI_ERR_INVALID_ARGUMENT, "%s: null pointer for layer %d", name, l);
    if (!aligned16(key_pools[l]) || !aligned16(value_pools[l]))
      return fail(MI_ERR_UNSUPPORTED, "%s: pools must be 16-byte aligned", name);
    wide = wide && aligned16(key_src[l]) && aligned16(value_src[l]);
  }
  for (int l0 = 0; l0 < num_layers; l0 += kMaxLayersPerLaunch) {
    const int nl = num_layers - l0 < kMaxLayersPerLaunch ? num_layers - l0 : kMaxLayersPerLaunch;
    for (int l = 0; l < nl; ++l) {
      a.src[0][l] = static_cast<const char*>(key_src[l0 + l]);
      a.src[1][l] = static_cast<const char*>(value_src[l0 + l]);
      a.pool[0][l] = static_cast<char*>(key_pools[l0 + l]);
      a.pool[1][l] = static_cast<char*>(value_pools[l0 + l]);
    }
    const dim3 grid(static_cast<uint32_t>(tiles * num_kv_heads), nl, 1);
    if (src_type == MI_TYPE_BF16)
      launch_store<Source::kBf16>(a, wide, grid, as_stream(stream));
    else if (src_type == MI_TYPE_FP16)
      launch_store<Source::kFp16>(a, wide, grid, as_stream(stream));
    else
      launch_store<Source::kFp32>(a, wide, grid, as_stream(stream));
    if (const int32_t rc = check_launch(name)) return rc;
  }
  return ok();
}

extern "C" int32_t mi_gather_blocks_fp4(const void* const* key_pools, const void* const* value_pools,
                                        int64_t num_blocks, const int64_t* block_ids, int64_t block_id_stride,
                                        int32_t batch, int32_t num_gathered_blocks, void* const* key_out,
                                        void* const* value_out, int32_t num_layers, int32_t num_kv_heads,
                                        int32_t head_dim, void* stream) {
  using namespace mi;
  const char* name = "mi_gather_blocks_fp4";
  if (batch < 0 || num_gathered_blocks < 0 || num_layers < 0 || num_blocks < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: negative size", name);
  if (batch == 0 || num_gathered_blocks == 0 || num_layers == 0) return ok();
  if (const int32_t rc = reject_empty_pool(name, num_blocks, true)) return rc;
  if (!key_pools || !value_pools || !block_ids || !key_out || !value_out)
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: null pointer argument", name);
  if (num_kv_heads <= 0) return fail(MI_ERR_INVALID_ARGUMENT, "%s: %d KV heads", name, num_kv_heads);
  if (head_dim != kFp4Dim) return fail(MI_ERR_UNSUPPORTED, "%s: head_dim %d, needs %d", name, head_dim, kFp4Dim);
  if (block_id_stride < num_gathered_blocks)
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: block_id_stride < num_gathered_blocks", name);
  const int64_t groups = static_cast<int64_t>(batch) * num_gathered_blocks;
  if (groups > 0xffffffffll / kGatherThreads || num_kv_heads > 2048 * kGatherHeads)  // grid y: fewer than 65536
    return fail(MI_ERR_UNSUPPORTED, "%s: too many blocks", name);
  GatherArgs a{};
  a.block_ids = block_ids;
  a.block_id_stride = block_id_stride;
  a.num_blocks = num_blocks;
  a.nb = num_gathered_blocks;
  a.kv_heads = num_kv_heads;
  a.head_groups = (num_kv_heads + kGatherHeads - 1) / kGatherHeads;
  for (int l = 0; l < num_layers; ++l) {
    if (!key_pools[l] || !value_pools[l] || !key_out[l] || !value_out[l])
      return fail(MI_ERR_INVALID_ARGUMENT, "%s: null pointer for layer %d", name, l);
    if (!aligned16(key_pools[l]) || !aligned16(value_pools[l]) || !aligned16(key_out[l]) || !aligned16(value_out[l]))
      return fail(MI_ERR_UNSUPPORTED, "%s: pools and outputs must be 16-byte aligned", name);
  }
  for (int l0 = 0; l0 < num_layers; l0 += kMaxLayersPerLaunch) {
    const int nl = num_layers - l0 < kMaxLayersPerLaunch ? num_layers - l0 : kMaxLayersPerLaunch;
    for (int l = 0; l < nl; ++l) {
      a.pool[0][l] = static_cast<const char*>(key_pools[l0 + l]);
      a.pool[1][l] = static_cast<const char*>(value_pools[l0 + l]);
      a.out[0][l] = static_cast<char*>(key_out[l0 + l]);
      a.out[1][l] = static_cast<char*>(value_out[l0 + l]);
    }
    fp4_gather_kernel<<<dim3(static_cast<uint32_t>(groups), nl * a.head_groups, 2), kGatherThreads, 0, as_stream(stream)>>>(a);
    if (const int32_t rc = check_launch(name)) return rc;
  }
  return ok();
}

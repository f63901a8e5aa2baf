// Paged GQA decode attention over a cache of 4-bit records (fp4_record.h): one query token per sequence.
//
//   out[b, h] = sum_t softmax_t(scale q[b, h] . K_t) V_t    over the context's n tokens, in fp32
//
// with K_t, V_t the values that the records stand for.  The counterpart of mi_paged_decode_attention (the
// reference's gather, mask and attend: src/mini_infra/model/qwen3.py:219-292) for 136 bytes a token and KV head
// instead of 512.  At that size a bf16 kernel's arithmetic would be the bound, so none is spent on unpacking keys:
//
//  * S^T = K Q^T by one v_mfma_scale_f32_16x16x128_f8f6f4 per 16 tokens: A is the record's 1 KiB of K codes as it
//    lies in memory (16 bytes a lane) with the scale byte beside them, B is q in two 8-bit floats (split_query).
//    hi of head c is column c and lo column c + 8 (a KV head has at most 8 query heads here); one row rotation adds
//    the two products, and leaves every head twice, which does no harm.
//  * C has the tokens in the A layout of P V's product (v_mfma_f32_16x16x32_bf16 over two records: lane quad r
//    holds tokens 4 r .. 4 r + 3 of each), so the probabilities, rounded to bf16 (2^-9 of a weight, which the
//    average of many takes further down, and half of what the output's own rounding costs), feed it without moving.
//  * V: a lane loads the four tokens x eight dims that its part of B needs, two values a convert, and v_perm pairs
//    the tokens.  Output tile t takes dim 8 j + t as its column j: a lane ends with eight dims of a head side by side.
//  * The running maximum is raised only when a score passes it by 2^8 (with the sums scaled alike, exact).
//
// Work: a workgroup takes a KV head and a part of a sequence's blocks, its wavefronts every kWaves-th pair of
// blocks, each with its own softmax state; the states are joined in LDS.  A sequence of several parts leaves
// partials in the workspace, which a second launch joins.
#include "decode_block.h"
#include "fp4_record.h"

namespace mi {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxGroup = 8;        // query heads per KV head
constexpr int kMaxPartBlocks = 64;  // a lane holds one block id
constexpr int kMergeThreads = 128;

struct Fp4DecodeArgs {
  uint16_t* out;
  int64_t out_row;
  const uint16_t* query;
  int64_t q_row, q_head;
  const char* key_pool;
  const char* value_pool;
  int64_t num_blocks;
  const int64_t* block_tables;
  int64_t bt_stride;
  const int64_t* context_lens;
  int64_t ctx_stride;
  int32_t max_blocks;
  int32_t kv_heads;
  int32_t group;
  int32_t part_blocks;  // blocks of a part
  int32_t parts;        // parts per sequence
  float scale;          // |scale| log2 e; the queries carry the sign
  uint32_t q_sign;      // 0x80008000 when scale < 0
  float* ws_acc;        // [batch, heads, parts, 128]
  float* ws_ml;         // [batch, heads, parts, 2]: max (log2 units) and sum
};

__device__ __forceinline__ int64_t tokens_of(const Fp4DecodeArgs& a, int64_t b) {
  const int64_t n = a.context_lens[b * a.ctx_stride];
  return min(n, static_cast<int64_t>(a.max_blocks) * kFp4Tokens);
}

struct Piece {  // a lane's part of one block
  u32x4 k, v;
  uint32_t ks, vs;
};

// Two blocks (32 tokens from tok_base, those from n on hidden) of one KV head.  st as MfmaState: m of head
// lane % 8, l the lane's share of its sum, o[t][i]: head 4 (lane / 16) + i (rows 8 .. 15 repeat 0 .. 7), dim 8 (lane % 16) + t.
__device__ __forceinline__ void attend_pair(MfmaState& st, const i32x8& q, uint32_t q_scale, Piece (&x)[2], float scale,
                                            int64_t tok_base, int64_t n, int lane) {
  const int r = lane >> 4;
  const bool tail = tok_base + 2 * kFp4Tokens > n;  // uniform
  float s[8];
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    i32x8 k{};
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = x[b].k[e];
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q, acc, 4, 0, 0, x[b].ks, 0, q_scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[4 * b + i] = (acc[i] + dpp_f32<0x128>(acc[i])) * scale;  // row_ror:8
  }
  if (tail) {  // hidden tokens: no weight, and a value of zero whatever their bytes say
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (tok_base + 16 * b + 4 * r + i >= n) {
          s[4 * b + i] = -INFINITY;
          x[b].v[i] = 0;
          x[b].vs &= ~(0xffu << (8 * i));
        }
  }
  float mb = s[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) mb = fmaxf(mb, s[e]);
  if (__builtin_amdgcn_ballot_w64(mb > st.m + kRescaleSlack) != 0) {
    const float nm = fmaxf(st.m, xmax32(xmax16(mb)));
    const float al = nm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.m - nm);
    st.m = nm;
    st.l *= al;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float ai = __shfl(al, (4 * r + i) & 7);
#pragma unroll
      for (int t = 0; t < 8; ++t) st.o[t][i] *= ai;
    }
  }
  const float ref = st.m == -INFINITY ? 0.0f : st.m;
  f32x8 p;
#pragma unroll
  for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(s[e] - ref);
  st.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
  const bf16x8 pa = __builtin_convertvector(p, bf16x8);
  u32x4 w[2][4];  // [block][token 4 r + i]: dims 8 j .. 8 j + 7
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t codes = x[b].v[i];
      w[b][i] = fp4_unpack8(codes, e8m0_f32((x[b].vs >> (8 * i)) & 0xffu));
    }
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const uint32_t sel = (t & 1) ? 0x07060302u : 0x05040100u;
    u32x4 f;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f[2 * b] = __builtin_amdgcn_perm(w[b][1][t >> 1], w[b][0][t >> 1], sel);
      f[2 * b + 1] = __builtin_amdgcn_perm(w[b][3][t >> 1], w[b][2][t >> 1], sel);
    }
    st.o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa, __builtin_bit_cast(bf16x8, f), st.o[t], 0, 0, 0);
  }
}

__global__ __launch_bounds__(kThreads) void fp4_decode_kernel(const Fp4DecodeArgs a) {
  extern __shared__ float s_raw[];  // [kWaves][group][128], then [kWaves][group][2]
  float* s_ml = s_raw + kWaves * a.group * kHeadDim;
  const int g = static_cast<int>(blockIdx.x % a.kv_heads);
  const int64_t unit = blockIdx.x / a.kv_heads;
  const int64_t b = unit / a.parts;
  const int part = static_cast<int>(unit % a.parts);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int j = lane & 15, r = lane >> 4;
  const int64_t n = tokens_of(a, b);
  uint16_t* out = a.out + b * a.out_row + static_cast<int64_t>(g) * a.group * kHeadDim;
  const int blocks = n <= 0 ? 0 : static_cast<int>((n + kFp4Tokens - 1) / kFp4Tokens);
  const int first = part * a.part_blocks;  // < max_blocks
  if (first >= blocks) {                   // uniform
    if (part == 0)                         // an empty context: zero rows
      for (int c = threadIdx.x; c < a.group * 16; c += kThreads) *reinterpret_cast<u32x4*>(out + 8 * c) = u32x4{};
    return;
  }
  const int count = min(a.part_blocks, blocks - first);
  int64_t id = a.block_tables[b * a.bt_stride + first + min(lane, count - 1)];
  if (id < 0 || id >= a.num_blocks) id = 0;
  const uint32_t id_lo = static_cast<uint32_t>(id);  // fewer than 2^31 blocks
  const int c = j & 7;
  const SplitQuery split = split_query(a.query + b * a.q_row + (static_cast<int64_t>(g) * a.group + min(c, a.group - 1)) * a.q_head,
                                       c < a.group, a.q_sign, r);
  const i32x8 q = j < 8 ? split.hi : split.lo;
  const uint32_t q_scale = j < 8 ? split.hi_scale : split.lo_scale;
  MfmaState st;
  st.m = -INFINITY;
  st.l = 0.0f;
#pragma unroll
  for (int t = 0; t < 8; ++t) st.o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int64_t block_bytes = static_cast<int64_t>(a.kv_heads) * kFp4Record;
  auto load = [&](Piece (&x)[2], int i) {  // blocks i, i + 1 of the part; past its end the last one again, which is hidden
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t at = __builtin_amdgcn_readlane(id_lo, min(i + e, count - 1)) * block_bytes + g * kFp4Record;
      const char* k = a.key_pool + at;
      const char* v = a.value_pool + at;
      x[e].k = load_vec<true>(reinterpret_cast<const u32x4*>(k + 16 * lane));
      x[e].v = load_vec<true>(reinterpret_cast<const u32x4*>(v + 16 * lane));
      x[e].ks = *reinterpret_cast<const uint8_t*>(k + kFp4Codes + lane);
      x[e].vs = *reinterpret_cast<const uint32_t*>(v + kFp4Codes + 16 * r + 4 * (j >> 2));
    }
  };
  // The context's end as the part sees it: a pair past the part's own blocks is hidden.
  const int64_t end = min(n, static_cast<int64_t>(first + count) * kFp4Tokens);
  Piece x[2][2];
  if (2 * w < count) load(x[0], 2 * w);
  for (int i = 2 * w; i < count; i += 4 * kWaves) {
    if (i + 2 * kWaves < count) load(x[1], i + 2 * kWaves);
    attend_pair(st, q, q_scale, x[0], a.scale, static_cast<int64_t>(first + i) * kFp4Tokens, end, lane);
    if (i + 2 * kWaves >= count) break;
    if (i + 4 * kWaves < count) load(x[0], i + 4 * kWaves);
    attend_pair(st, q, q_scale, x[1], a.scale, static_cast<int64_t>(first + i + 2 * kWaves) * kFp4Tokens, end, lane);
  }
  const float l = xsum32_f32(xsum16_f32(st.l));  // lane: head lane % 8
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int h = 4 * r + i;
    const float lh = __shfl(l, h & 7), mh = __shfl(st.m, h & 7);
    if (h >= a.group) continue;
    float4* dst = reinterpret_cast<float4*>(s_raw + (w * a.group + h) * kHeadDim + 8 * j);
    dst[0] = make_float4(st.o[0][i], st.o[1][i], st.o[2][i], st.o[3][i]);
    dst[1] = make_float4(st.o[4][i], st.o[5][i], st.o[6][i], st.o[7][i]);
    if (j == 0) *reinterpret_cast<float2*>(s_ml + (w * a.group + h) * 2) = make_float2(mh, lh);
  }
  __syncthreads();
  const bool whole = blocks <= a.part_blocks;
  for (int x8 = threadIdx.x; x8 < a.group * 16; x8 += kThreads) {
    const int h = x8 >> 4, o8 = 8 * (x8 & 15);
    float M = -INFINITY;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) M = fmaxf(M, s_ml[(v * a.group + h) * 2]);
    float L = 0.0f, o[8] = {};
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float m = s_ml[(v * a.group + h) * 2];
      // A wavefront without a visible score has no sums, except where every score was NaN: then its sum is.
      const float e = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - M);
      L += e * s_ml[(v * a.group + h) * 2 + 1];
      const float* src = s_raw + (v * a.group + h) * kHeadDim + o8;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d] += e * src[d];
    }
    if (whole) {
      store_bf16x8(out + h * kHeadDim + o8, o, 1.0f / L);
    } else {
      const int64_t at = ((b * a.kv_heads + g) * a.group + h) * a.parts + part;
      float4* dst = reinterpret_cast<float4*>(a.ws_acc + at * kHeadDim + o8);
      dst[0] = make_float4(o[0], o[1], o[2], o[3]);
      dst[1] = make_float4(o[4], o[5], o[6], o[7]);
      if (o8 == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * at) = make_float2(M, L);
    }
  }
}

// Joins the parts of the sequences that have several: one workgroup per sequence and head, a thread per dim.
__global__ __launch_bounds__(kMergeThreads) void fp4_merge_kernel(const Fp4DecodeArgs a) {
  const int64_t heads = static_cast<int64_t>(a.kv_heads) * a.group;
  const int64_t b = blockIdx.x / heads, h = blockIdx.x % heads;
  const int64_t n = tokens_of(a, b);
  const int blocks = n <= 0 ? 0 : static_cast<int>((n + kFp4Tokens - 1) / kFp4Tokens);
  if (blocks <= a.part_blocks) return;
  const int parts = (blocks + a.part_blocks - 1) / a.part_blocks;
  const int64_t at = (b * heads + h) * a.parts;
  float M = -INFINITY;
  for (int p = 0; p < parts; ++p) M = fmaxf(M, a.ws_ml[2 * (at + p)]);
  float L = 0.0f, o = 0.0f;
  for (int p = 0; p < parts; ++p) {
    const float m = a.ws_ml[2 * (at + p)];
    const float e = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - M);
    L += e * a.ws_ml[2 * (at + p) + 1];
    o += e * a.ws_acc[(at + p) * kHeadDim + threadIdx.x];
  }
  a.out[b * a.out_row + h * kHeadDim + threadIdx.x] = static_cast<uint16_t>(f32_to_bf16_bits(o / L));
}

// Blocks of a part: enough parts for every CU to have several workgroups, at most a lane's ids.
int part_blocks_for(int32_t batch, int32_t max_blocks, int32_t num_kv_heads) {
  const int64_t units = static_cast<int64_t>(batch) * num_kv_heads * max_blocks;
  int64_t part = units / (4 * static_cast<int64_t>(device_cus()));
  part = part < 2 * kWaves ? 2 * kWaves : (part > kMaxPartBlocks ? kMaxPartBlocks : part);
  return static_cast<int>(part / (2 * kWaves) * (2 * kWaves));
}

}  // namespace
}  // namespace mi

extern "C" int64_t mi_paged_decode_fp4_workspace_bytes(int32_t batch, int32_t max_blocks, int32_t num_heads,
                                                       int32_t num_kv_heads) {
  using namespace mi;
  if (batch <= 0 || max_blocks <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0) return 0;
  const int part = part_blocks_for(batch, max_blocks, num_kv_heads);
  const int64_t parts = (max_blocks + part - 1) / part;
  if (parts == 1) return 0;
  return static_cast<int64_t>(batch) * num_heads * parts * (kHeadDim + 2) * static_cast<int64_t>(sizeof(float));
}

extern "C" int32_t mi_paged_decode_attention_fp4(void* out, int64_t out_row_stride, const void* query,
                                                 int64_t query_row_stride, int64_t query_head_stride,
                                                 const void* key_pool, const void* value_pool, int64_t num_blocks,
                                                 const int64_t* block_tables, int64_t block_table_stride,
                                                 int32_t max_blocks, const int64_t* context_lens,
                                                 int64_t context_lens_stride, int32_t batch, int32_t num_heads,
                                                 int32_t num_kv_heads, int32_t head_dim, float scale, void* workspace,
                                                 int64_t workspace_bytes, void* stream) {
  using namespace mi;
  const char* name = "mi_paged_decode_attention_fp4";
  if (batch < 0 || max_blocks < 0 || num_blocks < 0) return fail(MI_ERR_INVALID_ARGUMENT, "%s: negative size", name);
  if (batch == 0) return ok();
  if (const int32_t rc = reject_empty_pool(name, num_blocks, max_blocks > 0)) return rc;
  if (!out || !query || !key_pool || !value_pool || !context_lens || (max_blocks > 0 && !block_tables))
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: null pointer argument", name);
  if (head_dim != kHeadDim || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(MI_ERR_UNSUPPORTED, "%s: needs head_dim %d and num_heads a multiple of num_kv_heads (got head_dim %d, heads %d/%d)",
                name, kHeadDim, head_dim, num_heads, num_kv_heads);
  const int32_t group = num_heads / num_kv_heads;
  if (group > kMaxGroup)
    return fail(MI_ERR_UNSUPPORTED, "%s: %d query heads per KV head, at most %d", name, group, kMaxGroup);
  if (!aligned16(out) || !aligned16(query) || !aligned16(key_pool) || !aligned16(value_pool) || out_row_stride % 8 != 0 ||
      query_row_stride % 8 != 0 || query_head_stride % 8 != 0)
    return fail(MI_ERR_UNSUPPORTED, "%s: query/out/pools must be 16-byte aligned", name);
  if (max_blocks > 0 && block_table_stride < max_blocks)
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: block_table_stride < max_blocks", name);
  if (context_lens_stride <= 0) return fail(MI_ERR_INVALID_ARGUMENT, "%s: context_lens_stride must be > 0", name);
  if (num_blocks > 0x7fffffff) return fail(MI_ERR_UNSUPPORTED, "%s: pool too large", name);
  const float c = scale * kLog2e;
  if (!(c == c) || c - c != 0.0f) return fail(MI_ERR_INVALID_ARGUMENT, "%s: scale must be finite", name);
  const int64_t need = mi_paged_decode_fp4_workspace_bytes(batch, max_blocks, num_heads, num_kv_heads);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(MI_ERR_WORKSPACE, "%s: workspace of %lld bytes needed, got %lld", name, static_cast<long long>(need),
                static_cast<long long>(workspace_bytes));
  if (need > 0 && !aligned16(workspace)) return fail(MI_ERR_UNSUPPORTED, "%s: workspace must be 16-byte aligned", name);

  Fp4DecodeArgs a{};
  a.out = static_cast<uint16_t*>(out);
  a.out_row = out_row_stride;
  a.query = static_cast<const uint16_t*>(query);
  a.q_row = query_row_stride;
  a.q_head = query_head_stride;
  a.key_pool = static_cast<const char*>(key_pool);
  a.value_pool = static_cast<const char*>(value_pool);
  a.num_blocks = num_blocks;
  a.block_tables = block_tables;
  a.bt_stride = block_table_stride;
  a.context_lens = context_lens;
  a.ctx_stride = context_lens_stride;
  a.max_blocks = max_blocks;
  a.kv_heads = num_kv_heads;
  a.group = group;
  a.part_blocks = part_blocks_for(batch, max_blocks, num_kv_heads);
  a.parts = max_blocks > 0 ? (max_blocks + a.part_blocks - 1) / a.part_blocks : 1;
  a.scale = c < 0.0f ? -c : c;
  a.q_sign = c < 0.0f ? 0x80008000u : 0u;
  // A scale of zero (every weight alike) still has to leave hidden scores at -inf.
  if (a.scale < 1e-37f) a.scale = 1e-37f;
  if (a.parts > 1) {
    a.ws_acc = static_cast<float*>(workspace);
    a.ws_ml = a.ws_acc + static_cast<int64_t>(batch) * num_heads * a.parts * kHeadDim;
  }
  const int64_t groups = static_cast<int64_t>(batch) * num_kv_heads * a.parts;
  if (groups > 0xffffffffll / kThreads || static_cast<int64_t>(batch) * num_heads > 0xffffffffll / kMergeThreads)
    return fail(MI_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  hipStream_t s = as_stream(stream);
  const size_t lds = sizeof(float) * kWaves * group * (kHeadDim + 2);
  fp4_decode_kernel<<<static_cast<uint32_t>(groups), kThreads, lds, s>>>(a);
  if (const int32_t rc = check_launch(name)) return rc;
  if (a.parts > 1) {
    fp4_merge_kernel<<<static_cast<uint32_t>(batch * num_heads), kMergeThreads, 0, s>>>(a);
    if (const int32_t rc = check_launch(name)) return rc;
  }
  return ok();
}

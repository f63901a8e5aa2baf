// Paged GQA decode attention over a cache of 4-bit records (fp4_record.h): one query token per sequence.
//
//   out[b, h] = sum_t softmax_t(scale q[b, h] . K_t) V_t    over the context's n tokens, in fp32
//
// with K_t, V_t the values that the records stand for.  The counterpart of mi_paged_decode_attention (the
// reference's gather, mask and attend: src/mini_infra/model/qwen3.py:219-292) for 136 bytes a token and KV head
// instead of 512.  At that size a bf16 kernel's arithmetic would be the bound, so none is spent on unpacking keys:
//
//  * Bound by the reads: 256 sequences of 256 to 8192 tokens, 892.7 MB, in 151 us, 5.9 TB/s (the loads alone take 145); a
//    single sequence by the latency of its few dependent loads and of the launch (6.9 us).
//  * S^T = K Q^T by one v_mfma_scale_f32_16x16x128_f8f6f4 per 16 tokens: A is the record's 1 KiB of K codes as it
//    lies in memory (16 bytes a lane) with the scale byte beside them, B is q in two 8-bit floats (split_query).
//    hi of head c is column c and lo column c + 8 (a KV head has at most 8 query heads here); one row rotation adds
//    the two products, and leaves every head twice, which does no harm.
//  * C has the tokens in the A layout of P V's product (v_mfma_f32_16x16x32_bf16 over two records: lane quad r
//    holds tokens 4 r .. 4 r + 3 of each), so the probabilities, rounded to bf16 (half a step, 2^-8 of a weight at
//    most, as the output's own rounding; the average over many tokens takes it further down), feed it without moving.
//  * V: a lane loads the four tokens x eight dims that its part of B needs, two values a convert, and v_perm pairs
//    the tokens.  Output tile t takes dim 8 j + t as its column j: a lane ends with eight dims of a head side by side.
//  * The running maximum is raised only when a score passes it by 2^8 (with the sums scaled alike, exact).
//
// Work, in one of two forms (Plan):
//  * Parts: a workgroup takes a KV head and a part of a sequence's blocks, its wavefronts every n-th pair of blocks, each
//    with its own softmax state, joined in LDS.  A sequence of several parts leaves partials for a second launch.
//  * Streams: the blocks of all sequences, in order, are cut into as many equal ranges as the device holds wavefronts
//    (per KV head), whatever the lengths; a wavefront walks its range, sequence by sequence.  Sequences that
//    a range's end cuts leave partials, two a range at most, for the second launch.
#include <algorithm>

#include "decode_block.h"
#include "fp4_record.h"

namespace mi {
namespace {

constexpr int kMaxGroup = 8;      // query heads per KV head
// Registers: at most 128 and 168.  The stream form's loop takes 160 with the next sequence's query in them; at four
// wavefronts a SIMD (128, with spills) the 256-sequence case below took 189 us instead of 154, at two 159.
constexpr int kPartWavesPerSimd = 4;
constexpr int kStreamWavesPerSimd = 3;
constexpr int kIds = 64;          // block ids in a register, one a lane
constexpr int kStreamWaves = 4;   // wavefronts of a workgroup of the stream form
constexpr int kMaxStreamBatch = 4096;  // sequences whose prefix sums a workgroup holds in LDS
constexpr int kMinStreamBlocks = 8;    // blocks of a range at least
constexpr int kMergeThreads = 256;

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
  int32_t batch;
  int32_t part_blocks;  // parts form: blocks of a part, at most kIds per wavefront
  int32_t parts;        // parts per sequence
  int32_t streams;      // streams form: ranges per KV head at most; 0: the parts form
  float scale;          // |scale| log2 e; the queries carry the sign
  uint32_t q_sign;      // 0x80008000 when scale < 0
  // Partials: accumulators [slots, 128], and [slots, 2] of max (log2 units) and sum.  Parts: slot (b heads + h) parts + part.
  // Streams: slot 2 stream heads + h for the cut sequence that a range begins with, (2 stream + 1) heads + h for the one
  // that it ends with; and the sequences' first blocks in the list, [batch + 1].
  float* ws_acc;
  float* ws_ml;
  int32_t* ws_off;
};

__device__ __forceinline__ int64_t tokens_of(const Fp4DecodeArgs& a, int64_t b) {
  const int64_t n = a.context_lens[b * a.ctx_stride];
  return min(n, static_cast<int64_t>(a.max_blocks) * kFp4Tokens);
}

// A lane's part of two blocks: codes and scale bytes.
struct Pair {
  u32x4 k[2], v[2];
  uint32_t ks[2], vs[2];
};

__device__ __forceinline__ int blocks_of(int64_t n) {
  return n <= 0 ? 0 : static_cast<int>((n + kFp4Tokens - 1) / kFp4Tokens);
}

// The workgroup's queries as B operands of the scaled product, through LDS: thread 32 h + x takes dims 4 x .. 4 x + 3 of
// head h (zeros past the group).  split_query's numbers, without every wavefront making all of them.
struct QueryStage {
  uint32_t codes[2][kMaxGroup][kHeadDim / 4];  // [hi, lo][head]
  uint32_t scales[2][kMaxGroup];
};
__device__ __forceinline__ void stage_queries(QueryStage& s, const Fp4DecodeArgs& a, int64_t b, int g) {
  const int h = threadIdx.x >> 5, x = threadIdx.x & 31;
  if (h >= kMaxGroup) return;  // whole wavefronts
  typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
  u32x2v v{};
  if (h < a.group) {
    v = *reinterpret_cast<const u32x2v*>(a.query + b * a.q_row + (static_cast<int64_t>(g) * a.group + h) * a.q_head + 4 * x);
    v[0] ^= a.q_sign;
    v[1] ^= a.q_sign;
  }
  const uint32_t w0 = v[0], w1 = v[1];
  uint32_t amax = max(max(w0 & 0x7fffu, (w0 >> 16) & 0x7fffu), max(w1 & 0x7fffu, (w1 >> 16) & 0x7fffu));
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), d)));
  const SplitScale sc(amax);
  int hi, lo;
  split4(w0, w1, sc.up, hi, lo);
  s.codes[0][h][x] = hi;
  s.codes[1][h][x] = lo;
  if (x == 0) {
    s.scales[0][h] = sc.hi;
    s.scales[1][h] = sc.lo;
  }
}

// The raw scores of two blocks: s[4 b + i] of head lane % 8 and token 16 b + 4 (lane / 16) + i.
__device__ __forceinline__ void pair_scores(float (&s)[8], const i32x8& q, uint32_t q_scale, const Pair& x) {
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    i32x8 k{};
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = x.k[b][e];
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q, acc, 4, 0, 0, x.ks[b], 0, q_scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[4 * b + i] = acc[i] + dpp_f32<0x128>(acc[i]);  // row_ror:8
  }
}

// Softmax of a pair's scores: the weights as bf16.  st as MfmaState: m of head lane % 8, l the lane's share of its sum,
// o[t][i]: head 4 (lane / 16) + i (rows 8 .. 15 repeat 0 .. 7), dim 8 (lane % 16) + t.
__device__ __forceinline__ bf16x8 pair_weights(MfmaState& st, const float (&s)[8], float scale, int r) {
  float mb = s[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) mb = fmaxf(mb, s[e]);
  mb *= scale;
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
  for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], scale, -ref));
  st.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
  return __builtin_convertvector(p, bf16x8);
}

// P V of dims 8 j + 2 kPair and the next: eight values of each, unpacked two a convert, paired by token.
template <int kPair>
__device__ __forceinline__ void attend_dims(MfmaState& st, const bf16x8& p, const Pair& x, const float (&vs)[2][4]) {
  uint32_t w[2][4];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t codes = x.v[b][i];
      w[b][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, vs[b][i], kPair));
    }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t sel = e ? 0x07060302u : 0x05040100u;
    u32x4 f;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f[2 * b] = __builtin_amdgcn_perm(w[b][1], w[b][0], sel);
      f[2 * b + 1] = __builtin_amdgcn_perm(w[b][3], w[b][2], sel);
    }
    st.o[2 * kPair + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p, __builtin_bit_cast(bf16x8, f), st.o[2 * kPair + e], 0, 0, 0);
  }
}
__device__ __forceinline__ void attend_values(MfmaState& st, const bf16x8& p, const Pair& x) {
  float vs[2][4];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) vs[b][i] = e8m0_f32((x.vs[b] >> (8 * i)) & 0xffu);
  attend_dims<0>(st, p, x, vs);
  attend_dims<1>(st, p, x, vs);
  attend_dims<2>(st, p, x, vs);
  attend_dims<3>(st, p, x, vs);
}

// A wavefront's walk over blocks of one sequence and KV head: the pipeline's registers and addresses.
typedef const __attribute__((address_space(1))) char* global_t;
typedef const __attribute__((address_space(1))) u32x4* global4_t;
struct Walk {
  Pair x;
  uint32_t ids;  // block ids, one a lane
  int64_t block_bytes;
  const char* k_pool;  // at this KV head
  const char* v_pool;
  uint32_t code_off, ks_off, vs_off;

  __device__ __forceinline__ Walk(const Fp4DecodeArgs& a, int g, int lane) {
    block_bytes = static_cast<int64_t>(a.kv_heads) * kFp4Record;
    k_pool = a.key_pool + g * kFp4Record;
    v_pool = a.value_pool + g * kFp4Record;
    code_off = 16 * lane;
    ks_off = kFp4Codes + lane;
    vs_off = kFp4Codes + 16 * (lane >> 4) + 4 * ((lane & 15) >> 2);
  }
  // Id of block i of the `count` from row: past the end the last one (which is hidden there), outside the pool the null block.
  __device__ __forceinline__ static uint32_t fetch_id(const Fp4DecodeArgs& a, const int64_t* row, int count, int i) {
    const int64_t id = row[min(i, count - 1)];
    return id < 0 || id >= a.num_blocks ? 0u : static_cast<uint32_t>(id);  // fewer than 2^31 blocks
  }
  // Scalar bases and 32-bit lane offsets.
  __device__ __forceinline__ global_t base_of(const char* pool, int i) const {
    global_t p = (global_t)(pool + __builtin_amdgcn_readlane(ids, i) * block_bytes);
    asm("" : "+s"(p));
    return p;
  }
  __device__ __forceinline__ void load_k(int i) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const global_t p = base_of(k_pool, i + e);
      x.k[e] = __builtin_nontemporal_load((global4_t)(p + code_off));
      x.ks[e] = *reinterpret_cast<const __attribute__((address_space(1))) uint8_t*>(p + ks_off);
    }
  }
  __device__ __forceinline__ void load_v(int i) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const global_t p = base_of(v_pool, i + e);
      x.v[e] = __builtin_nontemporal_load((global4_t)(p + code_off));
      x.vs[e] = *reinterpret_cast<const __attribute__((address_space(1))) uint32_t*>(p + vs_off);
    }
  }
  // The pair in x, `left` tokens of which (32 or more: all) are visible; next(): loads K of the next pair.  A pair's K
  // registers take the next pair's as soon as its scores are there; its V registers after P V, by the caller.
  template <typename Next>
  __device__ __forceinline__ void attend(MfmaState& st, const i32x8& q, uint32_t q_scale, float scale, int64_t left, int r, Next next) {
    float s[8];
    pair_scores(s, q, q_scale, x);
    next();
    if (left < 2 * kFp4Tokens) {  // uniform.  Hidden tokens: no weight, and a value of zero whatever their bytes say
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (16 * (e >> 2) + 4 * r + (e & 3) >= left) {
          s[e] = -INFINITY;
          x.v[e >> 2][e & 3] = 0;
          x.vs[e >> 2] &= ~(0xffu << (8 * (e & 3)));
        }
    }
    const bf16x8 p = pair_weights(st, s, scale, r);
    attend_values(st, p, x);
  }
};

__device__ __forceinline__ void start(MfmaState& st) {
  st.m = -INFINITY;
  st.l = 0.0f;
#pragma unroll
  for (int t = 0; t < 8; ++t) st.o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

template <int kWaves>
__global__ __launch_bounds__(64 * kWaves, kPartWavesPerSimd) void fp4_part_kernel(const Fp4DecodeArgs a) {
  extern __shared__ float s_raw[];  // [kWaves][group][128], then [kWaves][group][2]
  __shared__ QueryStage s_q;
  constexpr int kThreads = 64 * kWaves;
  static_assert(kThreads >= 32 * kMaxGroup, "a thread for every four query elements");
  float* s_ml = s_raw + kWaves * a.group * kHeadDim;
  const uint32_t unit = blockIdx.x / static_cast<uint32_t>(a.kv_heads);
  const int g = static_cast<int>(blockIdx.x - unit * a.kv_heads);
  const int64_t b = unit / static_cast<uint32_t>(a.parts);
  const int part = static_cast<int>(unit % static_cast<uint32_t>(a.parts));
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int j = lane & 15, r = lane >> 4;
  const int first = part * a.part_blocks;  // < max_blocks, but for an empty table
  // Lanes 2 k and 2 k + 1 hold the ids of the wavefront's k-th pair, blocks 2 w + 2 k kWaves and the next.  They are read
  // before the context's length is known, a memory round trip earlier; what lies past it is not used.
  const int mine = 2 * w + kWaves * (lane & ~1) + (lane & 1);
  int64_t id = 0;
  if (a.max_blocks > 0) id = a.block_tables[b * a.bt_stride + min(first + mine, a.max_blocks - 1)];
  const int64_t n = tokens_of(a, b);
  uint16_t* out = a.out + b * a.out_row + static_cast<int64_t>(g) * a.group * kHeadDim;
  const int blocks = blocks_of(n);
  if (first >= blocks) {                   // uniform
    if (part == 0)                         // an empty context: zero rows
      for (int c = threadIdx.x; c < a.group * 16; c += kThreads) *reinterpret_cast<u32x4*>(out + 8 * c) = u32x4{};
    return;
  }
  const int count = min(a.part_blocks, blocks - first);
  Walk walk(a, g, lane);
  walk.ids = mine < count && id >= 0 && id < a.num_blocks ? static_cast<uint32_t>(id) : 0u;  // the null block, hidden there
  MfmaState st;
  start(st);
  // The context's end as the part sees it: a pair past the part's own blocks is hidden.
  const int64_t end = min(n - static_cast<int64_t>(first) * kFp4Tokens, static_cast<int64_t>(count) * kFp4Tokens);
  int i = 2 * w;
  walk.load_k(0);
  walk.load_v(0);
  stage_queries(s_q, a, b, g);
  __syncthreads();
  i32x8 q;
  {
    const u32x4 lo = *reinterpret_cast<const u32x4*>(&s_q.codes[j >> 3][j & 7][4 * r]);
    const u32x4 hi = *reinterpret_cast<const u32x4*>(&s_q.codes[j >> 3][j & 7][16 + 4 * r]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      q[e] = lo[e];
      q[4 + e] = hi[e];
    }
  }
  const uint32_t q_scale = s_q.scales[j >> 3][j & 7];
  // Loads without a condition, of the null block after the last pair: the waits then cover a pair's own loads only (64
  // sequences 14.4 us instead of 15.2, 21 of 64 heads 26.3 instead of 27.5).
  for (int k = 2; i < count; i += 2 * kWaves, k += 2) {
    const int ahead = min(k, kIds - 2);
    walk.attend(st, q, q_scale, a.scale, end - static_cast<int64_t>(i) * kFp4Tokens, r, [&] { walk.load_k(ahead); });
    walk.load_v(ahead);
  }
  const float l = xsum32_f32(xsum16_f32(st.l));  // lane: head lane % 8
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int h = 4 * r + i;
    if (h >= a.group) continue;
    float4* dst = reinterpret_cast<float4*>(s_raw + (w * a.group + h) * kHeadDim + 8 * j);
    dst[0] = make_float4(st.o[0][i], st.o[1][i], st.o[2][i], st.o[3][i]);
    dst[1] = make_float4(st.o[4][i], st.o[5][i], st.o[6][i], st.o[7][i]);
  }
  if (lane < a.group) *reinterpret_cast<float2*>(s_ml + (w * a.group + lane) * 2) = make_float2(st.m, l);
  __syncthreads();
  const bool whole = blocks <= a.part_blocks;
  for (int x2 = threadIdx.x; x2 < a.group * 64; x2 += kThreads) {  // two dims a thread
    const int h = x2 >> 6, o2 = 2 * (x2 & 63);
    float M = -INFINITY;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) M = fmaxf(M, s_ml[(v * a.group + h) * 2]);
    float L = 0.0f, o[2] = {};
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float m = s_ml[(v * a.group + h) * 2];
      // A wavefront without a visible score has no sums, except where every score was NaN: then its sum is.
      const float e = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - M);
      L += e * s_ml[(v * a.group + h) * 2 + 1];
      const float2 src = *reinterpret_cast<const float2*>(s_raw + (v * a.group + h) * kHeadDim + o2);
      o[0] += e * src.x;
      o[1] += e * src.y;
    }
    if (whole) {
      *reinterpret_cast<uint32_t*>(out + h * kHeadDim + o2) = pack_bf16x2(o[0] * (1.0f / L), o[1] * (1.0f / L));
    } else {
      const int64_t at = ((b * a.kv_heads + g) * a.group + h) * a.parts + part;
      *reinterpret_cast<float2*>(a.ws_acc + at * kHeadDim + o2) = make_float2(o[0], o[1]);
      if (o2 == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * at) = make_float2(M, L);
    }
  }
}

// The cut of `total` > 0 blocks into ranges, none empty: range s begins at s q + min(s, rem).
struct Cut {
  int count, q, rem;
  __device__ __forceinline__ Cut(int total, int streams) {
    count = max(min(streams, (total + kMinStreamBlocks - 1) / kMinStreamBlocks), 1);
    q = total / count;
    rem = total - q * count;
  }
  __device__ __forceinline__ int begin(int s) const { return s * q + min(s, rem); }
  __device__ __forceinline__ int of(int x) const {  // the range that holds block x
    const int wide = rem * (q + 1);
    return x < wide ? x / (q + 1) : rem + (x - wide) / q;
  }
};

__global__ __launch_bounds__(64 * kStreamWaves, kStreamWavesPerSimd) void fp4_stream_kernel(const Fp4DecodeArgs a) {
  extern __shared__ int s_off[];  // [batch + 1]: the sequences' first blocks in the list
  __shared__ int s_wave[kStreamWaves];
  constexpr int kThreads = 64 * kStreamWaves;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  int carry = 0;
  for (int base = 0; base < a.batch; base += kThreads) {
    const int b = base + threadIdx.x;
    int v = b < a.batch ? blocks_of(tokens_of(a, b)) : 0;
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(v, d);
      if (lane >= d) v += y;
    }
    if (lane == 63) s_wave[w] = v;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int k = 0; k < kStreamWaves; ++k) {
      before += k < w ? s_wave[k] : 0;
      carry += s_wave[k];
    }
    if (b < a.batch) s_off[b + 1] = before + v;
    __syncthreads();
  }
  if (threadIdx.x == 0) s_off[0] = 0;
  __syncthreads();
  const int total = carry;
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b <= a.batch; b += kThreads) a.ws_off[b] = s_off[b];
  if (total == 0) return;
  const Cut cut(total, a.streams);
  const int id = static_cast<int>(blockIdx.x) * kStreamWaves + w;  // consecutive wavefronts: the KV heads of a range
  const int stream = __builtin_amdgcn_readfirstlane(id / a.kv_heads);
  const int g = __builtin_amdgcn_readfirstlane(id % a.kv_heads);
  if (stream >= cut.count) return;
  const int begin = __builtin_amdgcn_readfirstlane(cut.begin(stream)), end = __builtin_amdgcn_readfirstlane(cut.begin(stream + 1));
  int b = 0;
  for (int hi = a.batch; hi - b > 1;) {  // s_off[b] <= begin < s_off[hi]
    const int mid = (b + hi) >> 1;
    if (s_off[mid] <= begin) b = mid; else hi = mid;
  }
  b = __builtin_amdgcn_readfirstlane(b);
  const int j = lane & 15, r = lane >> 4;
  const int64_t heads = static_cast<int64_t>(a.kv_heads) * a.group;
  // The range's blocks of one sequence; the next one's ids, query and first blocks are on their way before it ends.
  struct Segment {
    int b, at, first, count;  // sequence; first block in the list and in the sequence; blocks
    bool whole;
  };
  auto segment_at = [&](int b, int at) __attribute__((always_inline)) {
    while (s_off[b + 1] <= at) ++b;  // empty contexts
    b = __builtin_amdgcn_readfirstlane(b);
    const int seq0 = __builtin_amdgcn_readfirstlane(s_off[b]), seq1 = __builtin_amdgcn_readfirstlane(s_off[b + 1]);
    return Segment{b, at, at - seq0, min(end, seq1) - at, at == seq0 && seq1 <= end};
  };
  auto row_of = [&](const Segment& x) __attribute__((always_inline)) { return a.block_tables + x.b * a.bt_stride + x.first; };
  const int qh = min(j & 7, a.group - 1);
  const uint16_t* q_head = a.query + (static_cast<int64_t>(g) * a.group + qh) * a.q_head;
  const bool q_live = (j & 7) < a.group;
  Walk walk(a, g, lane);
  QueryWords words;
  Segment seg = segment_at(b, begin);
  walk.ids = Walk::fetch_id(a, row_of(seg), seg.count, lane);
  words.load(q_head + seg.b * a.q_row, q_live, a.q_sign, r);
  walk.load_k(0);
  walk.load_v(0);
  for (;;) {
    const int64_t* row = row_of(seg);
    const int count = seg.count;
    uint32_t ids_next = count > kIds ? Walk::fetch_id(a, row + kIds, count - kIds, lane) : 0u;
    i32x8 q;
    const SplitScale split = split_query(words, [&](int i, int hi, int lo) { q[i] = j < 8 ? hi : lo; });
    const uint32_t q_scale = j < 8 ? split.hi : split.lo;
    const bool another = seg.at + count < end;
    Segment next_seg = seg;
    uint32_t ids_ahead = 0;
    if (another) {
      next_seg = segment_at(seg.b + 1, seg.at + count);
      ids_ahead = Walk::fetch_id(a, row_of(next_seg), next_seg.count, lane);
      words.load(q_head + next_seg.b * a.q_row, q_live, a.q_sign, r);
    }
    const int64_t visible = min(tokens_of(a, seg.b) - static_cast<int64_t>(seg.first) * kFp4Tokens, static_cast<int64_t>(count) * kFp4Tokens);
    MfmaState st;
    start(st);
    // ahead: the next pair's place in the window of ids.  After the range's last pair the null block is loaded (see the
    // parts form; 154 us to 151 at 256 sequences).
    for (int i = 0, ahead = 2; i < count; i += 2, ahead += 2) {
      if (i + 2 >= count) {
        ahead = 0;
        walk.ids = ids_ahead;
      } else if (ahead == kIds) {
        ahead = 0;
        walk.ids = ids_next;
        if (count - i - 2 > kIds) ids_next = Walk::fetch_id(a, row + i + 2 + kIds, count - i - 2 - kIds, lane);
      }
      walk.attend(st, q, q_scale, a.scale, visible - static_cast<int64_t>(i) * kFp4Tokens, r, [&] { walk.load_k(ahead); });
      walk.load_v(ahead);
    }
    const float l = xsum32_f32(xsum16_f32(st.l));
    uint16_t* out = a.out + seg.b * a.out_row + static_cast<int64_t>(g) * a.group * kHeadDim + 8 * j;
    const int64_t slot = (2 * static_cast<int64_t>(stream) + (seg.at == begin ? 0 : 1)) * heads + static_cast<int64_t>(g) * a.group;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = 4 * r + i;
      const float lh = __shfl(l, h & 7), mh = __shfl(st.m, h & 7);
      if (h >= a.group) continue;
      const float o[8] = {st.o[0][i], st.o[1][i], st.o[2][i], st.o[3][i], st.o[4][i], st.o[5][i], st.o[6][i], st.o[7][i]};
      if (seg.whole) {
        store_bf16x8(out + h * kHeadDim, o, 1.0f / lh);
      } else {
        float4* dst = reinterpret_cast<float4*>(a.ws_acc + (slot + h) * kHeadDim + 8 * j);
        dst[0] = make_float4(o[0], o[1], o[2], o[3]);
        dst[1] = make_float4(o[4], o[5], o[6], o[7]);
        if (j == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * (slot + h)) = make_float2(mh, lh);
      }
    }
    if (!another) return;
    seg = next_seg;
  }
}

// Joins the partials of cut sequences (and writes the streams form's zero rows): one workgroup per sequence and head, 32
// threads with four dims each for every kMergeLanes-th partial.
__global__ __launch_bounds__(kMergeThreads) void fp4_merge_kernel(const Fp4DecodeArgs a) {
  constexpr int kMergeLanes = kMergeThreads / 32, kMergeWaves = kMergeThreads / 64;
  __shared__ float s_o[kMergeLanes][kHeadDim], s_l[kMergeLanes], s_m[kMergeWaves];
  const uint32_t heads = a.kv_heads * a.group;
  const int64_t b = blockIdx.x / heads, h = blockIdx.x % heads;
  uint16_t* out = a.out + b * a.out_row + h * kHeadDim;
  // Partial p is in slot `first` for p = 0, slot at + p step for the others.
  int64_t first, at, step;
  int parts;
  if (a.streams) {
    const int x0 = a.ws_off[b], x1 = a.ws_off[b + 1];
    if (x0 == x1) {
      if (threadIdx.x < kHeadDim) out[threadIdx.x] = 0;
      return;
    }
    const Cut cut(a.ws_off[a.batch], a.streams);
    const int s0 = cut.of(x0);
    parts = cut.of(x1 - 1) - s0 + 1;
    at = 2 * static_cast<int64_t>(s0) * heads + h;
    step = 2 * static_cast<int64_t>(heads);
    first = at + (cut.begin(s0) == x0 ? 0 : heads);  // the second slot, unless its range begins with this sequence
  } else {
    parts = (blocks_of(tokens_of(a, b)) + a.part_blocks - 1) / a.part_blocks;
    first = at = (b * heads + h) * a.parts;
    step = 1;
  }
  if (parts <= 1) return;  // written whole
  const auto slot = [&](int p) { return p == 0 ? first : at + p * step; };
  float M = -INFINITY;
  for (int p = threadIdx.x; p < parts; p += kMergeThreads) M = fmaxf(M, a.ws_ml[2 * slot(p)]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) M = fmaxf(M, __shfl_xor(M, d));
  if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMergeWaves; ++w) M = fmaxf(M, s_m[w]);
  const int lane = threadIdx.x >> 5, x = threadIdx.x & 31;
  float L = 0.0f;
  f32x4 o{};
  for (int p = lane; p < parts; p += kMergeLanes) {
    const int64_t at_p = slot(p);
    const float2 ml = *reinterpret_cast<const float2*>(a.ws_ml + 2 * at_p);
    const f32x4 v = *reinterpret_cast<const f32x4*>(a.ws_acc + at_p * kHeadDim + 4 * x);
    // A partial without a visible score has no sums, except where every score was NaN: then its sum is.
    const float e = ml.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ml.x - M);
    L += e * ml.y;
    o += e * v;
  }
  *reinterpret_cast<f32x4*>(&s_o[lane][4 * x]) = o;
  if (x == 0) s_l[lane] = L;
  __syncthreads();
  if (threadIdx.x >= kHeadDim) return;
  L = 0.0f;
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < kMergeLanes; ++k) {
    L += s_l[k];
    sum += s_o[k][threadIdx.x];
  }
  out[threadIdx.x] = static_cast<uint16_t>(f32_to_bf16_bits(sum / L));
}

// How a launch is cut, and the workspace that takes, by the (sequence, KV head) pairs P, the table's blocks M and their
// product (context lengths are on the device).  Measured, us a call (16 query / 8 KV heads but where noted; lengths in
// tokens, M their longest's blocks), whole sequences by 4 / by 8 wavefronts, parts of 16 / 32 / 64 blocks, streams:
//   whole, 8 wavefronts to 2 P a CU, then 4: a second launch and its joining cost 4 to 5 us, more than the tail of tables of
//   80 blocks, or of 256 where P fills the CUs, and in proportion between
//       1 x 417             M 27    P 8      6.5 /  6.9     8.4 /   6.5 /   6.5    10.2
//       8 x 32..1150           72      64   10.1 /  8.9    10.0 /  10.0 /  11.8    14.3
//      16 x 1000..2000        125     128   16.2 / 12.5    13.6 /  13.0 /  14.4    18.3
//      20 x 1200..2550        160     160      - / 16.1    15.7 (by rule)
//      31 x 2000..3900        244     248      - / 24.0    27.4 (by rule)
//      64 x 32..1150           72     512   15.4 / 14.7    21.4 /  19.6 /  22.2    22.5
//     128 x 32..1150           72    1024   21.9 / 24.5    32.0 /  27.6 /  35.2    30.2
//    1000 x 32..1150           72    8000    121 /  151     189 /   165 /   201     144
//      64 x 50..3500          219     512   31.9 / 31.1    39.8 /  32.9 /  41.1    34.4
//   parts: few pairs
//       1 x 4000              250       8   26.1 / 18.6     9.5 /  10.6 /  13.2    13.0
//       1 x 65000            4063       8           -      31.6 /  23.8 /  21.6    37.1
//       4 x 20000..40000     2500      32           -      40.5 /  33.1 /  30.8    35.9
//      21 x 256..8192, 64 query heads  512  168     - / 35.3   31.5 /  26.1 /  26.2    29.9
//   streams: long tables of many pairs, mostly empty
//      30 x 256..8192         512     240      - / 36.9    37.1 /  31.6 /  32.1    31.3
//     100 x 256..8192         512     800      - / 73.4    93.9 /  79.9 /  78.4    63.3
//     256 x 256..8192         512    2048      -  / 170     241 /   209 /   199     152
struct Plan {
  int32_t streams, part_blocks, parts, waves;
  int64_t slots, bytes;
  Plan(int32_t batch, int32_t max_blocks, int32_t num_heads, int32_t num_kv_heads) {
    const int64_t cus = device_cus();
    const int64_t pairs = static_cast<int64_t>(batch) * num_kv_heads;
    const int64_t units = pairs * max_blocks;
    streams = 0;
    parts = 1;
    waves = pairs <= 2 * cus ? 8 : 4;
    part_blocks = max_blocks > 0 ? max_blocks : 1;
    slots = bytes = 0;
    // whole: every wavefront's ids fit its lanes
    if (max_blocks <= std::min<int64_t>(std::max<int64_t>(pairs * 4 * kIds / cus, 80), 4 * kIds)) return;
    waves = 4;
    if (batch <= kMaxStreamBatch && units >= 120000 && static_cast<int64_t>(batch) * max_blocks < (int64_t{1} << 30)) {
      const int64_t s = cus * 4 * kStreamWavesPerSimd / num_kv_heads;
      streams = static_cast<int32_t>(s < 1 ? 1 : s);
      slots = 2 * static_cast<int64_t>(streams) * num_heads;
      bytes = slots * (kHeadDim + 2) * 4 + (static_cast<int64_t>(batch) + 1) * 4;
      return;
    }
    const int64_t part = (units / 1024 + 7) / 8 * 8;
    part_blocks = static_cast<int32_t>(part < 16 ? 16 : (part > 64 ? 64 : part));
    parts = (max_blocks + part_blocks - 1) / part_blocks;
    if (parts == 1) return;
    slots = static_cast<int64_t>(batch) * num_heads * parts;
    bytes = slots * (kHeadDim + 2) * 4;
  }
};

template <int kWaves>
int32_t launch_parts(const char* name, const Fp4DecodeArgs& a, hipStream_t s) {
  const int64_t groups = static_cast<int64_t>(a.batch) * a.kv_heads * a.parts;
  if (groups > 0xffffffffll / (64 * kWaves)) return fail(MI_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  const size_t lds = sizeof(float) * kWaves * a.group * (kHeadDim + 2);
  fp4_part_kernel<kWaves><<<static_cast<uint32_t>(groups), 64 * kWaves, lds, s>>>(a);
  return check_launch(name);
}

}  // namespace
}  // namespace mi

extern "C" int64_t mi_paged_decode_fp4_workspace_bytes(int32_t batch, int32_t max_blocks, int32_t num_heads,
                                                       int32_t num_kv_heads) {
  using namespace mi;
  if (batch <= 0 || max_blocks <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0) return 0;
  return Plan(batch, max_blocks, num_heads, num_kv_heads).bytes;
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
  const Plan plan(batch, max_blocks, num_heads, num_kv_heads);
  const int64_t need = plan.bytes;
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
  a.batch = batch;
  a.part_blocks = plan.part_blocks;
  a.parts = plan.parts;
  a.streams = plan.streams;
  a.scale = c < 0.0f ? -c : c;
  a.q_sign = c < 0.0f ? 0x80008000u : 0u;
  // A scale of zero (every weight alike) still has to leave hidden scores at -inf.
  if (a.scale < 1e-37f) a.scale = 1e-37f;
  if (need > 0) {
    a.ws_acc = static_cast<float*>(workspace);
    a.ws_ml = a.ws_acc + plan.slots * kHeadDim;
    a.ws_off = reinterpret_cast<int32_t*>(a.ws_ml + plan.slots * 2);
  }
  if (static_cast<int64_t>(batch) * num_heads > 0xffffffffll / kMergeThreads)
    return fail(MI_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  hipStream_t s = as_stream(stream);
  if (a.streams) {
    const uint32_t groups = static_cast<uint32_t>((static_cast<int64_t>(a.streams) * num_kv_heads + kStreamWaves - 1) / kStreamWaves);
    fp4_stream_kernel<<<groups, 64 * kStreamWaves, sizeof(int) * (batch + 1), s>>>(a);
    if (const int32_t rc = check_launch(name)) return rc;
  } else if (const int32_t rc = plan.waves == 8 ? launch_parts<8>(name, a, s) : launch_parts<4>(name, a, s)) {
    return rc;
  }
  if (need > 0) {
    fp4_merge_kernel<<<static_cast<uint32_t>(batch * num_heads), kMergeThreads, 0, s>>>(a);
    if (const int32_t rc = check_launch(name)) return rc;
  }
  return ok();
}

// Chunked-prefill attention whose history is a cache of 4-bit records (fp4_record.h).
//
// The counterpart of mi_chunked_prefill_attention (the reference's gather, concat, mask and attend:
// src/mini_infra/model/qwen3.py:219-255, 325-330, src/mini_infra/worker/paged_runner.py:83-89): row b is a
// left-padded bf16 chunk; query i >= pad sees the first nh tokens of its history and the chunk's keys pad .. i.
//   out[b, i, h] = sum_t softmax_t(scale q . K_t) V_t, in fp32, over both
//
// One flash-style kernel in two phases that share the softmax state: history tiles, then the chunk's.
//  * Workgroup: a row, a pair of query heads of one KV head, kQTile queries; wavefronts as (head, queries).  Both
//    heads share every tile of 64 keys in LDS.  Short chunks behind a long history have the tiles of a row cut into
//    parts, a workgroup each, and a second launch joins their partials.
//  * History keys are multiplied as they are stored (v_mfma_scale_f32_16x16x128_f8f6f4): a block's 1 KiB of codes
//    goes to LDS untouched and is the A operand, 16 bytes a lane, at its 16 scale bytes; B is the query in two 8-bit floats
//    (split_query).  Two such products take the time of the four bf16 ones, from a quarter of the LDS bytes.
//  * History values are unpacked to bf16 (exact) on their way to LDS, each once per workgroup, into the layout of the
//    chunk's: rows of 256 bytes, 16-byte pieces XOR-swizzled by the row, sixteen lanes a row (a thread's own eight bytes
//    in order put two rows' pieces on the same banks).  Tokens past nh become zeros there.
//  * Chunk tiles go from memory straight into LDS; keys before the row's first token read that token's row.
//  * P V by v_mfma_f32_16x16x32_bf16: the probabilities are rounded to bf16 (half a step, 2^-8 of a weight, as the
//    output's own rounding), V^T comes from LDS by transposing reads, and a ninth tile sums the rounded weights.
//  * Scores stay in fp32; the running maximum is raised only when a score passes it by 2^8.
//
// What bounds it (4 x 2048 queries behind 10240 tokens, 600 us, 1260 TFLOP/s; a large bf16 library product reaches 1348
// on this card): a wavefront's tile is 1088 cycles of matrix unit and about 270 issue slots of 4 cycles of vector work (32
// exponentials take four slots each), and the two wavefronts of a SIMD do them largely one after the other.  Timing copies
// of an earlier 635 us: without the softmax 563, without staging 535, without the products with K 517, with V 485.  No gains:
// a tile's products a round before its softmax (704 to 708 against 683, instructions interleaved by hand or not; in the narrow
// form with a third buffer, 2 chunks to 333 behind 1500, 33.7 against 30.0), other XOR patterns of the rows (607 to 617),
// LDS reads further ahead by hand (709 to 714 against 622), wave priorities (651 against 635), a barrier every two or
// three tiles (606, 639 against 601), two workgroups of half the queries a CU (630).
#include <algorithm>
#include <initializer_list>

#include "decode_block.h"
#include "fp4_record.h"

namespace mi {
namespace {

constexpr int kGroup = 2;     // query heads per workgroup (a pair of one GQA group)
constexpr int kKTile = 64;    // keys per tile
constexpr int kTileBlocks = kKTile / kFp4Tokens;
constexpr int kSpans = kKTile / 4;  // 1 KiB LDS spans (4 rows of 256 B) of a bf16 tile

// kNt: 16-query column tiles per wavefront; kWavesPerHead: wavefronts side by side on a head's queries; kKeySplit:
// wavefront groups that take every kKeySplit-th tile of the same queries and join their states at the end.
template <int kNtV, int kWavesPerHeadV, int kKeySplitV>
struct Shape {
  static constexpr int kNt = kNtV, kWavesPerHead = kWavesPerHeadV, kKeySplit = kKeySplitV;
  static constexpr int kQPerWave = 16 * kNt;
  static constexpr int kQTile = kQPerWave * kWavesPerHead;
  static constexpr int kGroupWaves = kGroup * kWavesPerHead;
  static constexpr int kGroupThreads = 64 * kGroupWaves;
  static constexpr int kThreads = kGroupThreads * kKeySplit;
  static constexpr int kTileBytes = kKTile * 256;           // a bf16 tile
  static constexpr int kGroupLds = 4 * kTileBytes;          // chunk phase: K and V, double-buffered
  static constexpr int kLdsBytes = kGroupLds * kKeySplit;
  static constexpr int kSpansPerWave = kSpans / kGroupWaves;
  // History phase: bytes and code words of a thread's part of a tile's 4 KiB of codes.
  static constexpr int kWords = kTileBlocks * kFp4Codes / kGroupThreads / 4;
  static constexpr int kHistK = kTileBlocks * kFp4Codes, kHistScales = kTileBlocks * 64;
  static constexpr int kHistBuffer = kHistK + kHistScales + kTileBytes;
  static_assert(kSpans % kGroupWaves == 0 && (kWords == 2 || kWords == 4) && 2 * kHistBuffer <= kGroupLds, "shapes");
};
using Wide = Shape<2, 4, 1>;       // 128 queries, 8 wavefronts
using Half = Shape<2, 2, 1>;       // 64 queries, 4 wavefronts
using HalfSplit = Shape<2, 2, 2>;  // 64 queries, 8 wavefronts, the keys in two halves
using Narrow = Shape<1, 2, 2>;     // 32 queries, 8 wavefronts, the keys in two halves
using Slim = Shape<1, 2, 1>;       // 32 queries, 4 wavefronts; the form for keys cut over workgroups
constexpr int kMergeThreads = 256;

struct Fp4PrefillArgs {
  uint16_t* out;
  int64_t out_row, out_tok;
  const uint16_t* query;
  int64_t q_row, q_head, q_tok;
  const uint16_t* key;
  int64_t k_row, k_head, k_tok;
  const uint16_t* value;
  int64_t v_row, v_head, v_tok;
  const char* key_pool;
  const char* value_pool;
  int64_t num_blocks;
  const int64_t* history_blocks;
  int64_t history_stride;
  int32_t max_history_blocks;
  const int64_t* start_lens;
  const int64_t* chunk_lens;
  int64_t lens_stride;
  const int64_t* chunk_first;  // ragged rows: row b's first token among chunk_tokens, in row 0 of the tensors; null: padded rows
  int64_t first_stride;
  int32_t chunk_tokens;
  int32_t padded_len;
  int32_t kv_heads;
  int32_t group;  // query heads per KV head
  int32_t pairs;  // workgroups per KV head: ceil(group / 2)
  float scale;    // |scale| log2 e; the queries carry the sign
  uint32_t q_sign;
  int32_t tiles;  // query tiles per row
  int32_t batch;
  int32_t parts;  // workgroups that share the keys of a query tile, each writing partials (1: the output)
  float* ws_acc;  // [batch, heads, padded_len, parts, 128]
  float* ws_ml;   // [batch, heads, padded_len, parts, 2]: max (log2 units) and sum
  int32_t round_pairs;  // (row, head pair) units per dispatch round of one workgroup queue
};

// Where row b lies: its tokens, and what position i of its padded form has to move by to be token i + shift of row `row`.
struct RowAt {
  int len, row, shift;
  __device__ __forceinline__ RowAt(const Fp4PrefillArgs& a, int b) {
    const int64_t top = a.chunk_first ? min(a.padded_len, a.chunk_tokens) : a.padded_len;
    const int64_t n = a.chunk_lens[b * a.lens_stride];
    len = static_cast<int>(n < 0 ? 0 : (n > top ? top : n));
    row = b;
    shift = 0;
    if (a.chunk_first) {
      const int64_t first = a.chunk_first[b * a.first_stride], last = a.chunk_tokens - len;
      row = 0;
      shift = static_cast<int>(first < 0 ? 0 : (first > last ? last : first)) - (a.padded_len - len);
    }
  }
};

// A wavefront-uniform pointer that the compiler may hold in vector registers, in scalar ones.
__device__ __forceinline__ const void* scalar_ptr(const void* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(u)));
  const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(u >> 32)));
  return reinterpret_cast<const void*>((hi << 32) | lo);
}

template <typename S>
__global__ __launch_bounds__(S::kThreads, 2) void fp4_prefill_kernel(const Fp4PrefillArgs a) {
  constexpr int kNt = S::kNt, kQPerWave = S::kQPerWave, kQTile = S::kQTile, kThreads = S::kThreads;
  constexpr int kKeySplit = S::kKeySplit, kSpansPerWave = S::kSpansPerWave, kWords = S::kWords;
  constexpr uint32_t kTileBytes = S::kTileBytes;
  extern __shared__ __align__(1024) unsigned char s_raw[];

  // Workgroup -> (row b, head pair hp, query tile qt): the tiles of a pair on one XCD, heaviest first within rounds
  // of as many pairs as the XCD's CUs hold (as mi_chunked_prefill_attention).
  int b, hp, qt, part;
  {
    const int tiles = a.tiles;
    const int per_row = a.kv_heads * a.pairs;
    const int rows_pairs = per_row * a.batch;
    const int pairs = rows_pairs * a.parts;
    const int lin = static_cast<int>(blockIdx.x);
    const bool by_xcd = pairs % kXcds == 0;
    const int units = by_xcd ? pairs / kXcds : pairs;
    const int slot = by_xcd ? lin / kXcds : lin;
    const int round_idx = slot / (a.round_pairs * tiles);
    const int within = slot - round_idx * a.round_pairs * tiles;
    const int round_size = min(a.round_pairs, units - round_idx * a.round_pairs);
    const int rank = within / round_size;
    const int unit = round_idx * a.round_pairs + (within - rank * round_size);
    const int pair = by_xcd ? unit * kXcds + lin % kXcds : unit;
    // (divisions run on the vector unit: back to scalars, which the addresses need)
    part = __builtin_amdgcn_readfirstlane(pair / rows_pairs);
    hp = __builtin_amdgcn_readfirstlane(pair % per_row);
    b = __builtin_amdgcn_readfirstlane(pair % rows_pairs / per_row);
    qt = __builtin_amdgcn_readfirstlane(tiles - 1 - rank);
  }
  const int q0 = qt * kQTile;
  const int L = a.padded_len;
  const RowAt place(a, b);
  const int64_t src_row = __builtin_amdgcn_readfirstlane(place.row), shift = __builtin_amdgcn_readfirstlane(place.shift);
  int64_t start64 = a.start_lens[b * a.lens_stride];
  const int pad = __builtin_amdgcn_readfirstlane(L - place.len);
  start64 = start64 < 0 ? 0 : start64;
  const int64_t hist_cap = static_cast<int64_t>(a.max_history_blocks) * kFp4Tokens;
  const int nh = __builtin_amdgcn_readfirstlane(static_cast<int>(start64 < hist_cap ? start64 : hist_cap));

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = w / S::kGroupWaves;  // wavefront group (key split)
  const int wt = w % S::kGroupWaves;  // wavefront of the group
  const int gt = tid - wk * S::kGroupThreads;
  const int hh = wt / S::kWavesPerHead;
  const int qs = wt % S::kWavesPerHead;
  const int g = __builtin_amdgcn_readfirstlane(hp / a.pairs);  // KV head
  const int j0 = (hp - g * a.pairs) * kGroup;  // first head of the pair within the group
  const bool head_live = j0 + hh < a.group;    // false for the spare half of an odd group
  const int h = g * a.group + min(j0 + hh, a.group - 1);
  const int ql = lane & 15;
  const int gq = lane >> 4;

  uint16_t* out_b = a.out + src_row * a.out_row + shift * a.out_tok;
  if (pad == L && a.chunk_first) return;  // no tokens: nothing to read or write
  if (q0 + kQTile <= pad) {  // the whole tile is padding: zero rows
    if (a.parts > 1 || a.chunk_first) return;  // the second launch's; or none
    for (int c = tid; c < kQTile * kGroup * (kHeadDim / 8); c += kThreads) {
      const int qi = q0 + c / (kGroup * (kHeadDim / 8));
      const int rem = c % (kGroup * (kHeadDim / 8));
      const int jj = j0 + rem / (kHeadDim / 8);
      if (qi < L && jj < a.group)
        *reinterpret_cast<u32x4*>(out_b + qi * a.out_tok + (g * a.group + jj) * kHeadDim + (rem % (kHeadDim / 8)) * 8) = u32x4{};
    }
    return;
  }

  const int qw0 = q0 + kQPerWave * qs;  // first query of this wavefront
  const uint16_t* q_rows = a.query + src_row * a.q_row + shift * a.q_tok + h * a.q_head;

  // oacc[0..7]: O^T dims 16 dt + 4 gq + i of query column ql; oacc[8]: the weights' sums (its A operand has ones in
  // rows 0, 4, 8, 12).
  f32x4 oacc[9][kNt];
#pragma unroll
  for (int dt = 0; dt < 9; ++dt)
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) oacc[dt][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const __bf16 one_or_zero = (ql & 3) == 0 ? static_cast<__bf16>(1.0f) : static_cast<__bf16>(0.0f);
  const bf16x8 ones_frag = {one_or_zero, one_or_zero, one_or_zero, one_or_zero,
                            one_or_zero, one_or_zero, one_or_zero, one_or_zero};
  float m_run[kNt];
#pragma unroll
  for (int nt = 0; nt < kNt; ++nt) m_run[nt] = -INFINITY;
  bf16x8 pf[kNt][2];
  const float scale = a.scale;

  // V (A of O^T = V^T P^T): lane L of a 16-lane group addresses row k0 + L / 4, dims 16 dt + 4 (L % 4) .. + 3, and receives
  // dim 16 dt + L of rows k0 .. k0 + 3; k0 = 32 ks2 + 4 gq, then + 16, are the keys in the products' order.
  const int vr = 4 * gq + (ql >> 2);
  uint32_t v_off[8];
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) v_off[dt] = vr * 256 + (((2 * dt + ((ql >> 1) & 1)) ^ vr) & 15) * 16 + (ql & 1) * 8;

  // Softmax of raw products x, keys key0 .. key0 + 63, of which query i sees [lo, last] (last < 0: [lo, i]): first masks
  // and the running maximum (rarely raised), then the weights.
  typedef f32x4 scores_t[4][kNt];
  auto raise_max = [&](scores_t& x, const int key0, const int lo, const int last, const bool need_mask) __attribute__((always_inline)) {
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(static_cast<int>(need_mask)) != 0, 0)) {
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) {
        const int qi = qw0 + 16 * nt + ql;
        const bool row_ok = (qi >= pad) & (qi < L);
        const int hi = last < 0 ? qi : last;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kpos = key0 + mt * 16 + 4 * gq + i;
            const bool vis = row_ok & (kpos >= lo) & (kpos <= hi);
            x[mt][nt][i] = vis ? x[mt][nt][i] : -INFINITY;
          }
      }
    }
    float mx[kNt];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) {
      float v = -INFINITY;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) v = fmaxf(v, x[mt][nt][i]);
      mx[nt] = v * scale;
      grow = grow || mx[nt] > m_run[nt] + kRescaleSlack;
    }
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) {
        const float mn = fmaxf(m_run[nt], xmax32(xmax16(mx[nt])));
        const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run[nt] - mn);
        m_run[nt] = mn;
#pragma unroll
        for (int dt = 0; dt < 9; ++dt) oacc[dt][nt] *= alpha;
      }
    }
  };
  auto weights = [&](scores_t& x) __attribute__((always_inline)) {
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2)
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) {
        const float ref = m_run[nt] == -INFINITY ? 0.0f : m_run[nt];
        f32x8 pv;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          pv[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * ks2 + (e >> 2)][nt][e & 3], scale, -ref));
        pf[nt][ks2] = __builtin_convertvector(pv, bf16x8);
      }
  };
  auto tile_values = [&](const char* sVb) __attribute__((always_inline)) {
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2) {
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(sVb + 32 * ks2 * 256 + v_off[dt]));
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(sVb + (32 * ks2 + 16) * 256 + v_off[dt]));
        const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int nt = 0; nt < kNt; ++nt)
          oacc[dt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[nt][ks2], oacc[dt][nt], 0, 0, 0);
      }
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt)
        oacc[8][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones_frag, pf[nt][ks2], oacc[8][nt], 0, 0, 0);
    }
  };
  unsigned char* lds = s_raw + wk * S::kGroupLds;
  const bool rows_edge = qw0 < pad || qw0 + kQPerWave - 1 >= L;  // some of the wavefront's queries are none

  // This workgroup's tiles of the row's: history tiles [h0, h1), then chunk tiles [c0, c1) (all, unless parts share them).
  const int hist_tiles = (nh + kKTile - 1) / kKTile;
  const int c_first = pad / kKTile;
  const int all_tiles = hist_tiles + (min(q0 + kQTile, L) - 1) / kKTile - c_first + 1;
  const int t_begin = static_cast<int>(static_cast<int64_t>(all_tiles) * part / a.parts);
  const int t_end = static_cast<int>(static_cast<int64_t>(all_tiles) * (part + 1) / a.parts);
  const int h0 = min(t_begin, hist_tiles), h1 = min(t_end, hist_tiles);
  const int c0 = c_first + max(t_begin - hist_tiles, 0), c1 = c_first + max(t_end - hist_tiles, 0);

  // ---- Phase 1: the history.  Per buffer: 4 KiB of K codes, 256 K scale bytes, the bf16 V tile.
  if (h1 > h0) {  // uniform
    const int seen = min(nh, h1 * kKTile);  // history keys that this workgroup shows its queries
    const int nhb = (nh + kFp4Tokens - 1) / kFp4Tokens;
    const int64_t block_bytes = static_cast<int64_t>(a.kv_heads) * kFp4Record;
    const int64_t* table = a.history_blocks + b * a.history_stride;
    // This thread's code words of the tile: in block my_blk (the wavefront's), K bytes my_at .. of its codes, and V of octet
    // gt % 16 and kWords tokens from tok on (16 lanes write a whole LDS row: no bank conflicts).
    constexpr int kBlockThreads = kFp4Codes / 4 / kWords;  // threads of a block
    const int my_blk = __builtin_amdgcn_readfirstlane(gt / kBlockThreads);
    const int my_at = gt % kBlockThreads * 4 * kWords;
    const int octet = gt & 15, tok = gt % kBlockThreads / 16 * kWords, quad = tok >> 2;
    const uint32_t v_from = 256 * quad + 16 * octet + 4 * (tok & 3);
    // Block ids of the tile that is loaded next, fetched a round ahead: this wavefront's block, and block lane / 16 (whose K
    // scales the lane moves).  Tiles past the last are the last again: their keys are hidden.
    int64_t id_mine, id_lane;
    auto fetch_ids = [&](const int t) __attribute__((always_inline)) {
      id_mine = table[min(t * kTileBlocks + my_blk, nhb - 1)];
      id_lane = table[min(t * kTileBlocks + gq, nhb - 1)];
    };
    const uint32_t blocks_end = static_cast<uint32_t>(a.num_blocks);  // < 2^31, checked by the entry point
    auto block_of = [&](const int64_t id) __attribute__((always_inline)) {
      return static_cast<uint64_t>(id) < blocks_end ? static_cast<uint32_t>(id) : 0u;
    };
    typedef uint32_t words_t __attribute__((ext_vector_type(kWords)));
    words_t kw{}, vw{};
    uint32_t vs = 0, ks = 0;
    const char* const k_base = a.key_pool + g * kFp4Record;
    const char* const v_base = a.value_pool + g * kFp4Record;
    const uint32_t vs_at = kFp4Codes + 16 * quad + 4 * (octet >> 2);
    auto load_tile = [&]() __attribute__((always_inline)) {
      const int64_t at = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(block_of(id_mine)))) * block_bytes;
      kw = *reinterpret_cast<const words_t*>(k_base + at + my_at);
      vw = *reinterpret_cast<const words_t*>(v_base + at + v_from);
      vs = *reinterpret_cast<const uint32_t*>(v_base + at + vs_at);
      ks = *reinterpret_cast<const uint32_t*>(k_base + block_of(id_lane) * block_bytes + kFp4Codes + 4 * ql);
    };
    // Byte offsets of this thread's rows in a V tile, and its shift to the first one's scale.
    uint32_t v_at[kWords];
#pragma unroll
    for (int e = 0; e < kWords; ++e) {
      const int row = kFp4Tokens * my_blk + tok + e;
      v_at[e] = row * 256 + ((octet ^ (row & 15)) * 16);
    }
    const uint32_t vs_shift = 8 * (tok & 3);
    auto store_tile = [&](const int t, unsigned char* buf) __attribute__((always_inline)) {
      *reinterpret_cast<words_t*>(buf + kFp4Codes * my_blk + my_at) = kw;
      *reinterpret_cast<uint32_t*>(buf + S::kHistK + 4 * lane) = ks;
      vs >>= vs_shift;
      if (__builtin_expect((t + 1) * kKTile > seen, 0)) {  // uniform
#pragma unroll
        for (int e = 0; e < kWords; ++e)
          if (t * kKTile + kFp4Tokens * my_blk + tok + e >= seen) {
            vw[e] = 0;
            vs &= ~(0xffu << (8 * e));
          }
      }
#pragma unroll
      for (int e = 0; e < kWords; ++e) {
        const uint32_t codes = vw[e];
        *reinterpret_cast<u32x4*>(buf + S::kHistK + S::kHistScales + v_at[e]) = fp4_unpack8(codes, e8m0_f32((vs >> (8 * e)) & 0xffu));
      }
    };
    i32x8 q_hi[kNt], q_lo[kNt];
    uint32_t hi_scale[kNt], lo_scale[kNt];
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) {
      const int qi = qw0 + 16 * nt + ql;
      QueryWords words;
      words.load(q_rows + static_cast<int64_t>(min(qi, L - 1)) * a.q_tok, qi < L && qi >= pad, a.q_sign, gq);
      const SplitScale split = split_query(words, [&](int i, int hi, int lo) {
        q_hi[nt][i] = hi;
        q_lo[nt][i] = lo;
      });
      hi_scale[nt] = split.hi;
      lo_scale[nt] = split.lo;
    }
    auto products = [&](scores_t& x, const unsigned char* buf) __attribute__((always_inline)) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const u32x4 kc = *reinterpret_cast<const u32x4*>(buf + kFp4Codes * mt + 16 * lane);
        const int sc = buf[S::kHistK + 64 * mt + lane];
        i32x8 kf{};
#pragma unroll
        for (int e = 0; e < 4; ++e) kf[e] = kc[e];
#pragma unroll
        for (int nt = 0; nt < kNt; ++nt) {
          f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
          acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kf, q_lo[nt], acc, 4, 0, 0, sc, 0, lo_scale[nt]);
          x[mt][nt] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kf, q_hi[nt], acc, 4, 0, 0, sc, 0, hi_scale[nt]);
        }
      }
    };
    // In round i this group's tile is t = h0 + wk + i kKeySplit: it is in LDS, the next one goes there in the round, the one after
    // into registers.  Every wavefront does every round (a group's last may be hidden as a whole).
    fetch_ids(h0 + wk);
    load_tile();
    fetch_ids(h0 + wk + kKeySplit);
    store_tile(h0 + wk, lds);
    load_tile();
    fetch_ids(h0 + wk + 2 * kKeySplit);
    __syncthreads();
    const int rounds = (h1 - h0 + kKeySplit - 1) / kKeySplit;
    scores_t sacc;
    for (int i = 0; i < rounds; ++i) {
      const int t = h0 + wk + i * kKeySplit;
      unsigned char* const cur = lds + (i & 1) * S::kHistBuffer;
      products(sacc, cur);
      store_tile(t + kKeySplit, lds + ((i & 1) ^ 1) * S::kHistBuffer);
      load_tile();
      fetch_ids(t + 3 * kKeySplit);
      raise_max(sacc, t * kKTile, 0, seen - 1, (t + 1) * kKTile > seen || rows_edge);
      weights(sacc);
      tile_values(reinterpret_cast<const char*>(cur + S::kHistK + S::kHistScales));
      __syncthreads();
    }
  }

  // ---- Phase 2: the chunk, bf16 tiles in double-buffered LDS (two K tiles, then two V tiles).
  {
    const int c_lo = c0;
    const int n_tiles = c1 - c0;
    bf16x8 qf[kNt][4];
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) {
      const int qi = qw0 + 16 * nt + ql;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        u32x4 v{};
        if (qi < L && qi >= pad) {
          v = *reinterpret_cast<const u32x4*>(q_rows + static_cast<int64_t>(qi) * a.q_tok + ks * 32 + gq * 8);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] ^= a.q_sign;
        }
        qf[nt][ks] = __builtin_bit_cast(bf16x8, v);
      }
    }
    const int drow = lane >> 4;
    const int dchunk = lane & 15;
    const uint16_t* k_rows = a.key + src_row * a.k_row + shift * a.k_tok + g * a.k_head;
    const uint16_t* v_rows = a.value + src_row * a.v_row + shift * a.v_tok + g * a.v_head;
    const uint32_t k_tok = static_cast<uint32_t>(a.k_tok);  // < 2^24, checked by the entry point
    const uint32_t v_tok = static_cast<uint32_t>(a.v_tok);
    typedef __attribute__((address_space(3))) void* lds_ptr_t;
    const uint32_t k_lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr_t)(lds + kSpansPerWave * wt * 1024)));
    const uint32_t v_lds0 = k_lds0 + 2 * kTileBytes;
    // Lane i of span m of a tile fetches row 4 m + i / 16, 16-byte piece (i % 16) ^ (row % 16), which lands swizzled.
    // Rows before the first token read it, rows past the last read that (their keys are hidden).
    auto dma_tile = [&](const int t, const int buf) __attribute__((always_inline)) {
      const int key0 = (c_lo + t) * kKTile;
      const int row0 = min(max(key0, pad), L - 1);
      const void* kbase = scalar_ptr(k_rows + static_cast<int64_t>(row0) * k_tok);
      const void* vbase = scalar_ptr(v_rows + static_cast<int64_t>(row0) * v_tok);
#pragma unroll
      for (int i = 0; i < kSpansPerWave; ++i) {
        const int r = 4 * (kSpansPerWave * wt + i) + drow;
        const uint32_t c16 = static_cast<uint32_t>((dchunk ^ (r & 15)) * 16);
        const uint32_t kc = static_cast<uint32_t>(min(max(key0 + r, pad), L - 1) - row0);
        dma16<5>(kbase, 2 * kc * k_tok + c16, __builtin_amdgcn_readfirstlane(k_lds0 + buf * kTileBytes + i * 1024));
        dma16<5>(vbase, 2 * kc * v_tok + c16, __builtin_amdgcn_readfirstlane(v_lds0 + buf * kTileBytes + i * 1024));
      }
    };
    uint32_t k_off[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) k_off[ks] = ql * 256 + (((4 * ks + gq) ^ ql) & 15) * 16;
    const char* k_tiles = reinterpret_cast<const char*>(lds);
    const char* v_tiles = k_tiles + 2 * kTileBytes;
    auto tile_step = [&](const int t, const int buf) __attribute__((always_inline)) {
      if (t + kKeySplit < n_tiles) dma_tile(t + kKeySplit, buf ^ 1);
      scores_t sacc;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int nt = 0; nt < kNt; ++nt) sacc[mt][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          const bf16x8 kf = *reinterpret_cast<const bf16x8*>(k_tiles + buf * kTileBytes + mt * 4096 + k_off[ks]);
#pragma unroll
          for (int nt = 0; nt < kNt; ++nt)
            sacc[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[nt][ks], sacc[mt][nt], 0, 0, 0);
        }
      const int key0 = (c_lo + t) * kKTile;
      raise_max(sacc, key0, pad, -1, key0 + kKTile - 1 > qw0 || key0 < pad || rows_edge);
      weights(sacc);
      tile_values(v_tiles + buf * kTileBytes);
    };
    // The loads into LDS are the asm's, which the compiler does not count: each wavefront waits for its own before a
    // tile's barrier (vmcnt(0) as an instruction it sees first, so that it counts its own loads as done too).
    auto round_end = [&] {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    };
    if (wk < n_tiles) dma_tile(wk, 0);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    round_end();
    for (int t0 = 0; t0 < n_tiles; t0 += 2 * kKeySplit) {
      if (kKeySplit == 1 || t0 + wk < n_tiles) tile_step(t0 + wk, 0);
      round_end();
      if (t0 + kKeySplit < n_tiles) {
        if (kKeySplit == 1 || t0 + kKeySplit + wk < n_tiles) tile_step(t0 + kKeySplit + wk, 1);
        round_end();
      }
    }
  }
  if constexpr (kKeySplit > 1) {
    // Join the groups' states: group 0's wavefronts fold in the others', which they leave in LDS over the tiles.
    constexpr int kStateFloats = 33 * kNt * 64;
    static_assert((kKeySplit - 1) * S::kGroupWaves * (kStateFloats + 64 * kNt) * 4 <= S::kLdsBytes, "the states fit the tiles");
    float* st = reinterpret_cast<float*>(s_raw) + ((wk > 0 ? wk - 1 : 0) * S::kGroupWaves + wt) * (kStateFloats + 64 * kNt) + lane;
    if (wk > 0) {
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) {
#pragma unroll
        for (int e = 0; e < 32; ++e) st[(33 * nt + e) * 64] = oacc[e >> 2][nt][e & 3];
        st[(33 * nt + 32) * 64] = oacc[8][nt][0];
        st[(33 * kNt + nt) * 64] = m_run[nt];
      }
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int k = 1; k < kKeySplit; ++k) {
      const float* other = st + (k - 1) * S::kGroupWaves * (kStateFloats + 64 * kNt);
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) {
        const float mo = other[(33 * kNt + nt) * 64];
        const float mn = fmaxf(m_run[nt], mo);
        // A state without a maximum has no sums, except where every score was NaN: then they are NaN.
        const float e0 = m_run[nt] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run[nt] - mn);
        const float e1 = mo == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mo - mn);
        m_run[nt] = mn;
#pragma unroll
        for (int e = 0; e < 32; ++e)
          oacc[e >> 2][nt][e & 3] = e0 * oacc[e >> 2][nt][e & 3] + e1 * other[(33 * nt + e) * 64];
        oacc[8][nt][0] = e0 * oacc[8][nt][0] + e1 * other[(33 * nt + 32) * 64];
      }
    }
  }
  if (a.parts > 1) {  // unnormalised sums; padding rows are the second launch's
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) {
      const int qi = qw0 + 16 * nt + ql;
      if (qi >= L || qi < pad || !head_live) continue;
      const int64_t slot = ((static_cast<int64_t>(b) * a.kv_heads * a.group + h) * L + qi) * a.parts + part;
      float* acc = a.ws_acc + slot * kHeadDim + 4 * gq;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(acc + 16 * dt) = oacc[dt][nt];
      if (gq == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * slot) = make_float2(m_run[nt], oacc[8][nt][0]);
    }
    return;
  }
  // ---- normalise and write: lane holds query qw0 + 16 nt + ql, dims 16 dt + 4 gq + i; padding rows are zeros
#pragma unroll
  for (int nt = 0; nt < kNt; ++nt) {
    const int qi = qw0 + 16 * nt + ql;
    if (qi >= L || !head_live) continue;
    const bool real = qi >= pad;  // a padding row's sums are zeros, but a NaN among the values is in them too
    if (!real && a.chunk_first) continue;
    const float inv = 1.0f / oacc[8][nt][0];
    uint16_t* orow = out_b + qi * a.out_tok + h * kHeadDim + 4 * gq;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      uint2 v;
      v.x = real ? pack_bf16x2(oacc[dt][nt][0] * inv, oacc[dt][nt][1] * inv) : 0u;
      v.y = real ? pack_bf16x2(oacc[dt][nt][2] * inv, oacc[dt][nt][3] * inv) : 0u;
      *reinterpret_cast<uint2*>(orow + dt * 16) = v;
    }
  }
}

// Joins the parts of every query: 32 threads, four dims each, for a query of a head.
__global__ __launch_bounds__(kMergeThreads) void fp4_prefill_merge_kernel(const Fp4PrefillArgs a) {
  const int64_t heads = static_cast<int64_t>(a.kv_heads) * a.group;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kMergeThreads / 32) + threadIdx.x / 32;  // (b, query, head)
  if (row >= heads * a.padded_len * a.batch) return;
  const int64_t h = row % heads, qi = row / heads % a.padded_len, b = row / heads / a.padded_len;
  const int x = threadIdx.x & 31;
  const RowAt place(a, static_cast<int>(b));
  uint16_t* out = a.out + place.row * a.out_row + (qi + place.shift) * a.out_tok + h * kHeadDim + 4 * x;
  if (qi < a.padded_len - place.len) {
    if (!a.chunk_first) *reinterpret_cast<uint2*>(out) = uint2{0u, 0u};
    return;
  }
  const int64_t at = ((b * heads + h) * a.padded_len + qi) * a.parts;
  float M = -INFINITY;
  for (int p = 0; p < a.parts; ++p) M = fmaxf(M, a.ws_ml[2 * (at + p)]);
  float L = 0.0f;
  f32x4 o{};
  for (int p = 0; p < a.parts; ++p) {
    const float2 ml = *reinterpret_cast<const float2*>(a.ws_ml + 2 * (at + p));
    // A part without a visible key has no sums, except where every score was NaN: then its sum is.
    const float e = ml.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ml.x - M);
    L += e * ml.y;
    o += e * *reinterpret_cast<const f32x4*>(a.ws_acc + (at + p) * kHeadDim + 4 * x);
  }
  const float inv = 1.0f / L;
  *reinterpret_cast<uint2*>(out) = uint2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
}

template <typename S>
int32_t launch(const char* name, Fp4PrefillArgs& a, hipStream_t s) {
  a.tiles = (a.padded_len + S::kQTile - 1) / S::kQTile;
  const int64_t pairs = static_cast<int64_t>(a.kv_heads) * a.pairs * a.batch * a.parts;
  const int64_t groups = a.tiles * pairs;
  if (groups > 0xffffffffll / S::kThreads || groups > 0x3fffffff)
    return fail(MI_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  const bool by_xcd = pairs % kXcds == 0;
  const int64_t units = by_xcd ? pairs / kXcds : pairs;
  const int64_t cus = by_xcd ? device_cus() / kXcds : device_cus();
  a.round_pairs = static_cast<int32_t>(std::max(std::min(cus / a.tiles, units), int64_t{1}));
  if (const int32_t rc = allow_lds<&fp4_prefill_kernel<S>>(S::kLdsBytes, name)) return rc;
  fp4_prefill_kernel<S><<<static_cast<uint32_t>(groups), S::kThreads, S::kLdsBytes, s>>>(a);
  if (const int32_t rc = check_launch(name)) return rc;
  if (a.parts == 1) return ok();
  const int64_t rows = static_cast<int64_t>(a.kv_heads) * a.group * a.padded_len * a.batch;
  const int64_t merges = (rows * 32 + kMergeThreads - 1) / kMergeThreads;
  fp4_prefill_merge_kernel<<<static_cast<uint32_t>(merges), kMergeThreads, 0, s>>>(a);
  return check_launch(name);
}

enum class Form { kWide, kHalf, kHalfSplit, kNarrow, kSlim };

// The workgroup shape of a launch, by the workgroups it would have in the narrow and the wide shape, and the parts of its keys.
// Measured, us (16 query, 8 KV heads; rows x queries behind tokens of history, and the workgroups that decide),
// wide / half / half split / narrow, and the keys cut into 4 / 8 / 16 parts:
//   parts: twice the CUs' narrow workgroups, three parts at least, of six tiles at least, or twelve where the narrow
//   workgroups alone keep more than 3/8 of the CUs busy (a second launch and its joining, and the partials, cost 8 us)
//     1 x 1 behind 4000        8 narrow      138 / 105 /  76 /  53      27 / 20 / 18
//     1 x 16 behind 20000      8             645 / 490 / 331 / 215      96 / 55 / 37
//     1 x 60 behind 4000      16             140 / 110 /  79 /  52      29 / 24 / 23
//     4 x 60 behind 2000      64              78 /  61 /  47 /  31      26 / 27 / 37
//     1 x 300 behind 4000     80             148 / 116 /  84 /  57      40 / 42 / 49
//     1 x 256 behind 1200     64                              23      21 (3 parts)
//     1 x 333 behind 1500     88                              29      29 (4)
//     2 x 256 behind 3000    128                              40      38 (4)
//     1 x 512 behind 8000    128             219 / 153 / 123 /  88      63 / 68 / 81
//   narrow: one round of its workgroups (cus; 11/8 of that without much history)
//     4 x 128 behind 1200    128 narrow                       23      28 (3 parts)
//     3 x 160 behind 1500    120                              26      30 (4)
//     2 x 256 behind 1500    128                              26      30 (4)
//     5 x 100 behind 2000    160                              32      33 (3)
//     2 x 333 behind 1500    176              68 /  53 /  41 /  29      35 / 39 / 56
//     1 x 1000               256              41 /  34 /  26 /  19
//   half: short rows without history
//     15 x 128               120 wide         14 /  10 /  12 /  14
//     64 x 128               512              34 /  29 /  44 /  52
//     40 x 256               640              50 /  39 /  57 /  71
//   half split: up to half of cus wide workgroups, up to 17/16 of them for rows of more than 256; then half for shorter ones
//     3 x 450                 96              24 /  19 /  16 /  18
//     16 x 128 behind 1000   128              46 /  34 /  32 /  40
//     1 x 2000 behind 2000   128             142 / 114 /  81 /  81
//     20 x 128 behind 2000   160              72 /  64 /  72 /  78
//     3 x 700                144              30 /  27 /  23 /  25
//     2 x 1800 behind 4000   240             198 / 170 / 137 / 184
//     1 x 4096               256             105 /  94 /  82 / 108
//     3 x 1408 behind 6000   264             322 / 244 / 233 / 301
//   half: a second wide round at most 9/16 full
//     3 x 2048               384              77 /  76 /  86 /  99
//     25 x 256 behind 2000   400             135 / 125 / 153 / 188
//   wide beyond
//     4 x 1600               416              63 /  68 /  71 /  92
//     4 x 1900 behind 1000   480             122 / 143 / 144 / 194
//     4 x 2048 behind 10240  512             600 / 630 / 639 / 878
struct Plan {
  Form form;
  int32_t parts = 1;
  int64_t slots = 0;  // partials
  Plan(int32_t batch, int32_t padded_len, int32_t num_heads, int32_t num_kv_heads, int32_t max_history_blocks) {
    const int64_t cus = device_cus();
    const int64_t pairs = static_cast<int64_t>(num_kv_heads) * ((num_heads / num_kv_heads + kGroup - 1) / kGroup) * batch;
    const int64_t wide = pairs * ((padded_len + Wide::kQTile - 1) / Wide::kQTile);
    const int64_t narrow = pairs * ((padded_len + Narrow::kQTile - 1) / Narrow::kQTile);
    const int64_t history = static_cast<int64_t>(max_history_blocks) * kFp4Tokens;
    const int64_t part_tiles = 8 * narrow <= 3 * cus ? 6 : 12;
    const int64_t most = std::min(2 * cus / narrow, (history + padded_len) / (part_tiles * kKTile));
    if (most >= 3) {
      form = Form::kSlim;
      parts = static_cast<int32_t>(most);
      slots = static_cast<int64_t>(batch) * num_heads * padded_len * parts;
    } else if (8 * narrow <= (2 * history >= padded_len ? 8 : 11) * cus) {
      form = Form::kNarrow;
    } else if (history == 0 && padded_len <= 256) {
      form = Form::kHalf;
    } else if (2 * wide <= cus) {
      form = Form::kHalfSplit;
    } else if (16 * wide <= 17 * cus) {
      form = padded_len > 256 ? Form::kHalfSplit : Form::kHalf;
    } else {
      form = 16 * wide <= 25 * cus ? Form::kHalf : Form::kWide;
    }
  }
  int64_t bytes() const { return slots * (kHeadDim + 2) * static_cast<int64_t>(sizeof(float)); }
};

// The entry points below: chunk_first null for padded rows.
int32_t run_prefill(const char* name, void* out, int64_t out_row_stride, int64_t out_tok_stride, const void* query,
                    int64_t query_row_stride, int64_t query_head_stride, int64_t query_tok_stride, const void* key,
                    int64_t key_row_stride, int64_t key_head_stride, int64_t key_tok_stride, const void* value,
                    int64_t value_row_stride, int64_t value_head_stride, int64_t value_tok_stride, const void* key_pool,
                    const void* value_pool, int64_t num_blocks, const int64_t* history_blocks, int64_t history_stride,
                    int32_t max_history_blocks, const int64_t* start_lens, const int64_t* chunk_lens, int64_t lens_stride,
                    const int64_t* chunk_first, int64_t first_stride, int32_t chunk_tokens, int32_t batch,
                    int32_t padded_len, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, float scale,
                    void* workspace, int64_t workspace_bytes, void* stream) {
  if (batch < 0 || padded_len < 0 || max_history_blocks < 0 || num_blocks < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: negative size", name);
  if (batch == 0 || padded_len == 0) return ok();
  if (const int32_t rc = reject_empty_pool(name, num_blocks, max_history_blocks > 0)) return rc;
  if (!out || !query || !key || !value || !start_lens || !chunk_lens ||
      (max_history_blocks > 0 && (!history_blocks || !key_pool || !value_pool)))
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: null pointer argument", name);
  if (head_dim != kHeadDim || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(MI_ERR_UNSUPPORTED, "%s: needs head_dim %d and num_heads a multiple of num_kv_heads (got head_dim %d, heads %d/%d)",
                name, kHeadDim, head_dim, num_heads, num_kv_heads);
  for (int64_t st : {out_row_stride, out_tok_stride, query_row_stride, query_head_stride, query_tok_stride, key_row_stride,
                     key_head_stride, key_tok_stride, value_row_stride, value_head_stride, value_tok_stride})
    if (st % 8 != 0) return fail(MI_ERR_UNSUPPORTED, "%s: strides must be multiples of 8", name);
  for (const void* t : {static_cast<const void*>(out), query, key, value})
    if (!aligned16(t)) return fail(MI_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned", name);
  if (max_history_blocks > 0 && (!aligned16(key_pool) || !aligned16(value_pool)))
    return fail(MI_ERR_UNSUPPORTED, "%s: pools must be 16-byte aligned", name);
  if (num_blocks > 0x7fffffff) return fail(MI_ERR_UNSUPPORTED, "%s: pool too large", name);
  if (max_history_blocks > 0 && history_stride < max_history_blocks)
    return fail(MI_ERR_INVALID_ARGUMENT, "%s: history_stride < max_history_blocks", name);
  if (static_cast<int64_t>(max_history_blocks) * kFp4Tokens + padded_len > 0x7fffffff - 2 * kKTile)
    return fail(MI_ERR_UNSUPPORTED, "%s: %d history blocks and %d positions are too many", name, max_history_blocks, padded_len);
  if (lens_stride <= 0) return fail(MI_ERR_INVALID_ARGUMENT, "%s: lens_stride must be > 0", name);
  if (key_tok_stride < 0 || key_tok_stride >= (1 << 24) || value_tok_stride < 0 || value_tok_stride >= (1 << 24))
    return fail(MI_ERR_UNSUPPORTED, "%s: key/value token strides must be in [0, 2^24)", name);
  const float c = scale * kLog2e;
  if (!(c - c == 0.0f)) return fail(MI_ERR_INVALID_ARGUMENT, "%s: scale must be finite", name);

  Fp4PrefillArgs a{};
  a.out = static_cast<uint16_t*>(out);
  a.out_row = out_row_stride;
  a.out_tok = out_tok_stride;
  a.query = static_cast<const uint16_t*>(query);
  a.q_row = query_row_stride;
  a.q_head = query_head_stride;
  a.q_tok = query_tok_stride;
  a.key = static_cast<const uint16_t*>(key);
  a.k_row = key_row_stride;
  a.k_head = key_head_stride;
  a.k_tok = key_tok_stride;
  a.value = static_cast<const uint16_t*>(value);
  a.v_row = value_row_stride;
  a.v_head = value_head_stride;
  a.v_tok = value_tok_stride;
  a.key_pool = static_cast<const char*>(key_pool);
  a.value_pool = static_cast<const char*>(value_pool);
  a.num_blocks = num_blocks;
  a.history_blocks = history_blocks;
  a.history_stride = history_stride;
  a.max_history_blocks = max_history_blocks;
  a.start_lens = start_lens;
  a.chunk_lens = chunk_lens;
  a.lens_stride = lens_stride;
  a.chunk_first = chunk_first;
  a.first_stride = first_stride;
  a.chunk_tokens = chunk_tokens;
  a.padded_len = padded_len;
  a.kv_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.pairs = (a.group + kGroup - 1) / kGroup;
  // A scale of zero (every weight alike) still has to leave hidden scores at -inf.
  a.scale = std::max(c < 0.0f ? -c : c, 1e-37f);
  a.q_sign = c < 0.0f ? 0x80008000u : 0u;
  a.batch = batch;
  if (static_cast<int64_t>(num_kv_heads) * a.pairs * batch > 0x3fffffff)
    return fail(MI_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  const Plan plan(batch, padded_len, num_heads, num_kv_heads, max_history_blocks);
  if (plan.slots > 0) {
    if (!workspace || workspace_bytes < plan.bytes())
      return fail(MI_ERR_WORKSPACE, "%s: workspace of %lld bytes needed, got %lld", name, static_cast<long long>(plan.bytes()),
                  static_cast<long long>(workspace_bytes));
    if (!aligned16(workspace)) return fail(MI_ERR_UNSUPPORTED, "%s: workspace must be 16-byte aligned", name);
    a.ws_acc = static_cast<float*>(workspace);
    a.ws_ml = a.ws_acc + plan.slots * kHeadDim;
  }
  a.parts = plan.parts;
  hipStream_t s = as_stream(stream);
  switch (plan.form) {
    case Form::kWide: return launch<Wide>(name, a, s);
    case Form::kHalf: return launch<Half>(name, a, s);
    case Form::kHalfSplit: return launch<HalfSplit>(name, a, s);
    case Form::kNarrow: return launch<Narrow>(name, a, s);
    default: return launch<Slim>(name, a, s);
  }
}

}  // namespace
}  // namespace mi

extern "C" int64_t mi_chunked_prefill_fp4_workspace_bytes(int32_t batch, int32_t padded_len, int32_t num_heads,
                                                          int32_t num_kv_heads, int32_t max_history_blocks) {
  using namespace mi;
  if (batch <= 0 || padded_len <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      max_history_blocks < 0)
    return 0;
  return Plan(batch, padded_len, num_heads, num_kv_heads, max_history_blocks).bytes();
}

extern "C" int32_t mi_chunked_prefill_attention_fp4(
    void* out, int64_t out_row_stride, int64_t out_tok_stride, const void* query, int64_t query_row_stride,
    int64_t query_head_stride, int64_t query_tok_stride, const void* key, int64_t key_row_stride,
    int64_t key_head_stride, int64_t key_tok_stride, const void* value, int64_t value_row_stride,
    int64_t value_head_stride, int64_t value_tok_stride, const void* key_pool, const void* value_pool,
    int64_t num_blocks, const int64_t* history_blocks, int64_t history_stride, int32_t max_history_blocks,
    const int64_t* start_lens, const int64_t* chunk_lens, int64_t lens_stride, int32_t batch, int32_t padded_len,
    int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, float scale, void* workspace, int64_t workspace_bytes,
    void* stream) {
  return mi::run_prefill("mi_chunked_prefill_attention_fp4", out, out_row_stride, out_tok_stride, query, query_row_stride,
                         query_head_stride, query_tok_stride, key, key_row_stride, key_head_stride, key_tok_stride, value,
                         value_row_stride, value_head_stride, value_tok_stride, key_pool, value_pool, num_blocks,
                         history_blocks, history_stride, max_history_blocks, start_lens, chunk_lens, lens_stride, nullptr, 0,
                         0, batch, padded_len, num_heads, num_kv_heads, head_dim, scale, workspace, workspace_bytes, stream);
}

extern "C" int32_t mi_ragged_prefill_attention_fp4(
    void* out, int64_t out_tok_stride, const void* query, int64_t query_head_stride, int64_t query_tok_stride,
    const void* key, int64_t key_head_stride, int64_t key_tok_stride, const void* value, int64_t value_head_stride,
    int64_t value_tok_stride, int32_t num_tokens, const void* key_pool, const void* value_pool, int64_t num_blocks,
    const int64_t* history_blocks, int64_t history_stride, int32_t max_history_blocks, const int64_t* start_lens,
    const int64_t* chunk_lens, int64_t lens_stride, const int64_t* chunk_first, int64_t first_stride, int32_t batch,
    int32_t max_len, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, float scale, void* workspace,
    int64_t workspace_bytes, void* stream) {
  using namespace mi;
  const char* name = "mi_ragged_prefill_attention_fp4";
  if (num_tokens < 0) return fail(MI_ERR_INVALID_ARGUMENT, "%s: negative size", name);
  if (batch > 0 && !chunk_first) return fail(MI_ERR_INVALID_ARGUMENT, "%s: null pointer argument", name);
  if (first_stride <= 0) return fail(MI_ERR_INVALID_ARGUMENT, "%s: first_stride must be > 0", name);
  if (num_tokens == 0) return ok();
  return run_prefill(name, out, 0, out_tok_stride, query, 0, query_head_stride, query_tok_stride, key, 0, key_head_stride,
                     key_tok_stride, value, 0, value_head_stride, value_tok_stride, key_pool, value_pool, num_blocks,
                     history_blocks, history_stride, max_history_blocks, start_lens, chunk_lens, lens_stride, chunk_first,
                     first_stride, num_tokens, batch, max_len, num_heads, num_kv_heads, head_dim, scale, workspace,
                     workspace_bytes, stream);
}

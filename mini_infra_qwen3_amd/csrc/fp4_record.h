// The 4-bit block record: 16 tokens of one KV head, K or V, in 1088 bytes (4.25 bits a value).
//
// A row of 128 values is four groups of 32 dims.  Group g has one power of two s_g = 2^(c_g - 127), c_g a byte
// (E8M0), and 32 codes of 4 bits (E2M1: sign, two exponent bits, one mantissa bit; magnitudes 0, 0.5, 1, 1.5, 2,
// 3, 4, 6); a value is its code's number times s_g.  This is the operand format of the scaled matrix instructions
// (v_mfma_scale_f32_16x16x128_f8f6f4) and of the packed converts (v_cvt_scalef32_pk_bf16_fp4), so keys go into
// the products as they are stored and values take half an instruction each.
//
// Quantisation: with a = max |x| of the group,
//   c = clamp(((bits(fp32 a) + 2^21) >> 23) - 2, 1, 252)
// is the smallest exponent at which a rounds to at most 6 (a / s in [3.5, 7), or below where c is clamped to 1),
// and a code is x / s rounded to nearest, ties to the even code, saturated at 6 (which only c = 252 needs).  A
// group with an infinity or NaN gets c = 255, the format's NaN: every value of it reads as NaN.
//
// Record, 1024 code bytes, then 64 scale bytes; two codes a byte, the even dim in the low four bits:
//   K: codes [4 groups][16 tokens][16 bytes], scales [4 groups][16 tokens]: 16 bytes a lane for lane = 16 group +
//      token are the A operand of the scaled product, and the scale byte beside them is that lane's.
//   V: codes [4 token quads][16 dim octets][4 tokens][4 bytes], scales [4 quads][4 groups][4 tokens]: 16 bytes a
//      lane for lane = 16 quad + octet are the four tokens that the lane's share of P V sums over.
// A token's bytes are whole bytes of its own in both, so tokens are written in any order.
#pragma once

#include "mi_common.h"

namespace mi {
namespace {

constexpr int kFp4Record = 1088;
constexpr int kFp4Codes = 1024;
constexpr int kFp4Tokens = 16;  // tokens of a record
constexpr int kFp4Dim = 128;
constexpr uint32_t kFp4NanScale = 255;

// fp32 of an E8M0 code as the converts' scale operand (code 0 is 2^-127, which they take from exponent 0).
__device__ __forceinline__ float e8m0_f32(uint32_t code) { return __uint_as_float(code << 23); }

// The scale code of a group whose largest magnitude has these fp32 bits.
__device__ __forceinline__ uint32_t fp4_scale_code(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return kFp4NanScale;
  const int c = static_cast<int>((amax_bits + (1u << 21)) >> 23) - 2;
  return static_cast<uint32_t>(min(max(c, 1), 252));
}

// Eight values at a finite scale as eight codes.
__device__ __forceinline__ uint32_t fp4_pack8(const float (&x)[8], float scale) {
  uint32_t r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], scale, 3);
}

// Eight codes as eight bf16 (exact: a code has two significant bits).
__device__ __forceinline__ u32x4 fp4_unpack8(uint32_t codes, float scale) {
  u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  return r;
}

// Byte offsets within a record of the four code bytes of token t, dims 8 j .. 8 j + 7, and of their scale.
__device__ __forceinline__ int fp4_code_at(bool value, int t, int j) {
  return value ? 256 * (t >> 2) + 16 * j + 4 * (t & 3) : 256 * (j >> 2) + 16 * t + 4 * (j & 3);
}
__device__ __forceinline__ int fp4_scale_at(bool value, int t, int j) {
  return kFp4Codes + (value ? 16 * (t >> 2) + 4 * (j >> 2) + (t & 3) : 16 * (j >> 2) + t);
}

// Quantises a row's piece j, dims 8 j .. 8 j + 7, into token t of a record.  Called by the sixteen lanes of a row together: a
// group of 32 dims is the four lanes of a DPP quad, its largest magnitude two quad permutes away, in integer bits, which
// order magnitudes and put every NaN above every number.
__device__ __forceinline__ void fp4_store_piece(char* record, bool value, int t, int j, const float (&x)[8], bool live) {
  uint32_t amax = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(x[e]) & 0x7fffffffu);
  amax = max(amax, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(amax), 0xB1, 0xf, 0xf, false)));
  amax = max(amax, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(amax), 0x4E, 0xf, 0xf, false)));
  const uint32_t scale = fp4_scale_code(amax);
  const uint32_t codes = scale == kFp4NanScale ? 0u : fp4_pack8(x, e8m0_f32(scale));
  if (live) {
    *reinterpret_cast<uint32_t*>(record + fp4_code_at(value, t, j)) = codes;
    if ((j & 3) == 0) *reinterpret_cast<uint8_t*>(record + fp4_scale_at(value, t, j)) = static_cast<uint8_t>(scale);
  }
}

// A query against K records: q = 2^s (hi + lo / 16), hi the nearest e4m3 numbers and lo the nearest ones of what is
// left, as B operands of the scaled product (lane quad r holds dims 16 r .. + 15 and 64 + 16 r .. + 15, the order
// that the instruction reads 8-bit operands in).  bf16 has 8 significant bits and e4m3 4, and the largest element's
// hi is in [128, 256), so an element is exact down to 2^-14 of the largest, and off by at most 2^-23 of it below.
// An infinity or NaN makes both scales NaN, and with them every score.
//
// The scaled product adds eight terms (dims 8 j .. 8 j + 7) at a time, dropping what lies 2^-13 below their largest, and
// the sixteen sums in fp32 (measured in bounds, term by term against exact sums).  That is off by at most 7 x 2^-13 of each
// octet's largest term, so by 2^-10 of sum |q k| at the very most: fewer bits than the kernels' other sums keep, taken
// because the operands have fewer, q being bf16 and off by up to 2^-8 of every term before it gets here.  lo's terms, 2^-4
// of hi's, are summed on their own and go in as the fp32 addend.
typedef int i32x8 __attribute__((ext_vector_type(8)));
struct SplitScale {
  float up;         // 2^-s: brings the largest element to [128, 256)
  uint32_t hi, lo;  // scale codes
  // amax: the largest magnitude's bf16 bits.  Below 2^-103 the scale stays (up and lo's code in range; elements sink).
  __device__ __forceinline__ explicit SplitScale(uint32_t amax) {
    const int e = max(static_cast<int>(amax >> 7), 24);
    up = __uint_as_float(static_cast<uint32_t>(2 * 127 + 7 - e) << 23);
    const bool finite = amax < 0x7f80u;
    hi = finite ? static_cast<uint32_t>(e - 7) : kFp4NanScale;
    lo = finite ? static_cast<uint32_t>(e - 11) : kFp4NanScale;
  }
};
// Four elements (two bf16 pairs) as four hi and four lo codes.
__device__ __forceinline__ void split4(uint32_t w0, uint32_t w1, float up, int& hi, int& lo) {
  const float x0 = bf16_lo(w0) * up, x1 = bf16_hi(w0) * up, x2 = bf16_lo(w1) * up, x3 = bf16_hi(w1) * up;
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(x0, x1, 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(x2, x3, hi, true);
  const float r0 = x0 - __builtin_amdgcn_cvt_f32_fp8(hi, 0), r1 = x1 - __builtin_amdgcn_cvt_f32_fp8(hi, 1);
  const float r2 = x2 - __builtin_amdgcn_cvt_f32_fp8(hi, 2), r3 = x3 - __builtin_amdgcn_cvt_f32_fp8(hi, 3);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(r0 * 16.0f, r1 * 16.0f, 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(r2 * 16.0f, r3 * 16.0f, lo, true);
}
// Lane quad r's part of a head's 128 elements (16-byte aligned; not read when !live: zeros), signs flipped by `flip`
// (0x80008000 or 0).
struct QueryWords {
  uint32_t w[16];
  __device__ __forceinline__ void load(const uint16_t* q, bool live, uint32_t flip, int r) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const u32x4 v = live ? *reinterpret_cast<const u32x4*>(q + 64 * (p >> 1) + 16 * r + 8 * (p & 1)) : u32x4{};
#pragma unroll
      for (int e = 0; e < 4; ++e) w[4 * p + e] = v[e] ^ flip;
    }
  }
};
// put(i, hi, lo) for a lane's code words i = 0 .. 7; returns the scales.  Every lane of the wavefront must be active; the four
// lanes of a column (lane % 16) hold the same query.
template <typename Put>
__device__ __forceinline__ SplitScale split_query(const QueryWords& q, Put put) {
  uint32_t amax = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) amax = max(amax, max(q.w[e] & 0x7fffu, (q.w[e] >> 16) & 0x7fffu));
  amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 16)));
  amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 32)));
  const SplitScale s(amax);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    int hi, lo;
    split4(q.w[2 * i], q.w[2 * i + 1], s.up, hi, lo);
    put(i, hi, lo);
  }
  return s;
}

}  // namespace
}  // namespace mi

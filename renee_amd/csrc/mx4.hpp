// Label matrices in microscaled 4-bit floating point (MX4): quantisation, and products of embeddings with them.
//
// 32 consecutive dims of a label are a block: a scale 2^(byte - 127) and 32 numbers of a sign, two exponent bits and one mantissa
// bit (0, 0.5, 1, 1.5, 2, 3, 4, 6).  byte - 127 = floor(log2 of the block's largest magnitude) - 2, at least -127, so that the largest
// number is 4 or 6; numbers are rounded to the nearest, ties to an even mantissa, and those above 6 become 6.  A block that
// holds an infinity or a NaN has byte 255 and stands for 32 NaNs; a block of zeros has byte 0.
//
// Embeddings enter a product in blocks of the same kind, quantised as they are loaded: in 4 bits, or in 8 (four exponent
// bits, three mantissa bits, up to 448: byte - 127 = floor(log2 of the largest) - 8).  Then z[b][l] = sum over blocks of 2^(sx + sw) times
// the sum of 32 products, which is what v_mfma_scale_f32_16x16x128_f8f6f4 does: 16 rows x 16 labels x four blocks, sums in fp32.
// With 4-bit embeddings products are quarters and sums are exact unless scales lie some 2^8 apart.  With 8-bit ones the
// matrix pipe drops what lies below about 2^-14 of the largest of neighbouring products (measured), well under fp16's half step.
//
// Layout.  Lane (i, q) = i + 16 q of the MFMA holds row i, block q of the step.  Labels go in units of 64, four tiles of 16 for one
// wave, dims in steps of four blocks, and codes and scales lie in the order in which lanes take them:
//   codes   [unit][step][tile 4][row 16][block 4][16 bytes]    the last step has as many blocks as are left of the width
//   scales  [unit][step][block 4][row 16][tile 4]              a lane's dword: one byte for each tile, the MFMA's operand selector
// so that a fetch of a wave is 1 KB in a row, 24 KB of a unit at 768 dims follow each other, and a scale takes no instruction but its load.
// Row 4 q + r of tile 2 p + t is label 32 p + 8 q + 4 t + r of the unit: of two tiles' sums a lane then holds eight consecutive labels.
#pragma once
#include <type_traits>
#include <utility>

#include "mx4_layout.hpp"
#include "pipe_core.hpp"
#include "topk.hpp"

namespace xfc {

constexpr uint32_t MX_NAN = 255;

typedef int int4v __attribute__((ext_vector_type(4)));
typedef int int8v __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------------------------
// blocks
// ---------------------------------------------------------------------------------------------
struct Float8 { float v[8]; };

// Eight consecutive numbers of type TYPE (xfc_type), as floats.
template <int TYPE>
__device__ __forceinline__ Float8 load8(const void* p) {
  Float8 f;
  if constexpr (TYPE == XFC_F32) {
    const float4v lo = reinterpret_cast<const float4v*>(p)[0], hi = reinterpret_cast<const float4v*>(p)[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) { f.v[e] = lo[e]; f.v[4 + e] = hi[e]; }
  } else if constexpr (TYPE == XFC_BF16) {
    const uint4v q = *reinterpret_cast<const uint4v*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) { f.v[2 * e] = __uint_as_float(q[e] << 16); f.v[2 * e + 1] = __uint_as_float(q[e] & 0xffff0000u); }
  } else {
    const half8 h = *reinterpret_cast<const half8*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = (float)h[e];
  }
  return f;
}
template <int TYPE>
__device__ __forceinline__ void store8(void* p, const Float8& f) {
  if constexpr (TYPE == XFC_F32) {
    reinterpret_cast<float4v*>(p)[0] = float4v{f.v[0], f.v[1], f.v[2], f.v[3]};
    reinterpret_cast<float4v*>(p)[1] = float4v{f.v[4], f.v[5], f.v[6], f.v[7]};
  } else if constexpr (TYPE == XFC_BF16) {
    typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
    bf16x8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (__bf16)f.v[e];
    *reinterpret_cast<bf16x8*>(p) = h;
  } else {
    half8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (half_t)f.v[e];
    *reinterpret_cast<half8*>(p) = h;
  }
}
constexpr int type_bytes(int type) { return type == XFC_F32 ? 4 : 2; }

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {  // over four neighbouring lanes
  const uint32_t a = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true);  // quad_perm 1, 0, 3, 2
  v = a > v ? a : v;
  const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true);  // quad_perm 2, 3, 0, 1
  return b > v ? b : v;
}

// The scale byte of a block that lies in four neighbouring lanes, eight numbers each, and the factor that conversions divide by.
// Magnitudes are compared as bits: infinities and NaNs come out on top.  Where the scale would be no normal float, numbers and
// factor are multiplied by 2^64, which leaves the quotient as it is.
template <int EMAX>
__device__ __forceinline__ uint32_t block_scale(Float8& f, float& by) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = __float_as_uint(f.v[e]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  m = quad_max(m);
  const int exponent = (int)(m >> 23);
  uint32_t byte = exponent > EMAX ? exponent - EMAX : 0;
  by = __uint_as_float(byte << 23);
  if (byte == 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] *= 0x1p64f;
    by = 0x1p-63f;
  }
  return exponent == 255 ? MX_NAN : m == 0 ? 0 : byte;
}
__device__ __forceinline__ uint32_t to_fp4(const Float8& f, float by) {  // eight numbers, the first in the lowest bits
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f.v[0], f.v[1], by, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f.v[2], f.v[3], by, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f.v[4], f.v[5], by, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f.v[6], f.v[7], by, 3);
}
// (The conversion makes a NaN of what lies above 448: that is cut off first.)
__device__ __forceinline__ uint64_t to_fp8(Float8 f, float by) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f.v[e] = __builtin_amdgcn_fmed3f(f.v[e], -448.f * by, 448.f * by);
  typedef short short2v __attribute__((ext_vector_type(2)));
  short2v lo = {0, 0}, hi = {0, 0};
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, f.v[0], f.v[1], by, false);
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, f.v[2], f.v[3], by, true);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, f.v[4], f.v[5], by, false);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, f.v[6], f.v[7], by, true);
  return (uint64_t)__builtin_bit_cast(uint32_t, lo) | ((uint64_t)__builtin_bit_cast(uint32_t, hi) << 32);
}
// The same of eight halves, without making floats of them: half the instructions.  Their blocks' scales are normal floats.
template <int EMAX>
__device__ __forceinline__ uint32_t block_scale(const half8& h, float& by) {
  typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
  const uint4v q = __builtin_bit_cast(uint4v, h) & 0x7fff7fffu;
  auto larger = [](uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, a), __builtin_bit_cast(ushort2v, b)));
  };
  const uint32_t two = larger(larger(q[0], q[1]), larger(q[2], q[3]));
  const uint32_t m = quad_max((two >> 16) > (two & 0xffffu) ? two >> 16 : two & 0xffffu);
  const uint32_t exponent = __float_as_uint((float)__builtin_bit_cast(half_t, (uint16_t)m)) >> 23;
  const uint32_t byte = exponent - EMAX;  // (m = 0: not used)
  by = m == 0 ? 1.f : __uint_as_float((exponent == 255 ? 127u : byte) << 23);
  return exponent == 255 ? MX_NAN : m == 0 ? 0 : byte;
}
__device__ __forceinline__ uint32_t to_fp4(const half8& h, float by) {
  typedef half_t half2v __attribute__((ext_vector_type(2)));
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, half2v{h[0], h[1]}, by, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, half2v{h[2], h[3]}, by, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, half2v{h[4], h[5]}, by, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, half2v{h[6], h[7]}, by, 3);
}
// (448 times the scale is a half, or rounds to one that no number of the block exceeds.)
__device__ __forceinline__ uint64_t to_fp8(const half8& h, float by) {
  typedef short short2v __attribute__((ext_vector_type(2)));
  typedef half_t half2v __attribute__((ext_vector_type(2)));
  const half_t most = (half_t)(448.f * by);
  half8 c;
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = most;
  c = __builtin_elementwise_max(__builtin_elementwise_min(h, c), -c);
  short2v lo = {0, 0}, hi = {0, 0};
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(lo, half2v{c[0], c[1]}, by, false);
  lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(lo, half2v{c[2], c[3]}, by, true);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(hi, half2v{c[4], c[5]}, by, false);
  hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(hi, half2v{c[6], c[7]}, by, true);
  return (uint64_t)__builtin_bit_cast(uint32_t, lo) | ((uint64_t)__builtin_bit_cast(uint32_t, hi) << 32);
}
// 2^(byte - 127), NaN for 255
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == MX_NAN ? 0x7fc00000u : byte == 0 ? 0x00400000u : byte << 23);
}
// Eight numbers of a block, from their codes.
__device__ __forceinline__ Float8 from_fp4(uint32_t codes, float scale) {
  Float8 f;
  auto pair = [&](auto at) {
    const auto p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, decltype(at)::value);
    f.v[2 * decltype(at)::value] = p[0] * scale;
    f.v[2 * decltype(at)::value + 1] = p[1] * scale;
  };
  pair(std::integral_constant<int, 0>{});
  pair(std::integral_constant<int, 1>{});
  pair(std::integral_constant<int, 2>{});
  pair(std::integral_constant<int, 3>{});
  return f;
}

// ---------------------------------------------------------------------------------------------
// label matrix -> MX4 and back
// ---------------------------------------------------------------------------------------------
// A workgroup takes a step of a unit: 64 labels x 128 dims.  Of each tile a wave takes four rows, four consecutive labels, a lane eight
// dims of one: 256 bytes of a label in a row are read (fp16), 256 bytes of codes written, and after four tiles a lane in four has
// a dword of scales.  Bound by the stream: of 131,072 x 768 halves 201 MB are read and 53 written in 60 us, 4.2 TB/s (a plain copy reaches 4.8
// here), and back, out of the Infinity Cache, in 38; 655,363 x 768 fp32, 2.0 GB and 0.27, in 463 us, 4.9 TB/s.  4,097 x 200 takes 3.5 us, little more
// than an empty launch.
struct MxArgs {
  const void* W; void* out; int64_t ldw;  // quantize: W, dequantize: out
  uint8_t* codes; uint8_t* scales;
  int64_t L; int d, blocks, steps;
};

template <int TYPE>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(MxArgs a) {
  const int64_t unit = blockIdx.x / (unsigned)a.steps;
  const int step = blockIdx.x % (unsigned)a.steps;
  const int lane = threadIdx.x & 63, row = 4 * (threadIdx.x >> 6) + (lane >> 4), block = (lane >> 2) & 3, part = lane & 3;
  const int k = step * MX_STEP + block * MX_BLOCK + part * 8;
  const int wide = mx_wide(step, a.blocks);
  Float8 f[MX_TILES];
#pragma unroll
  for (int t = 0; t < MX_TILES; ++t) {
    const int64_t label = unit * MX_UNIT + mx_label(t, row);
    f[t] = Float8{};
    if (label < a.L && k < a.d) f[t] = load8<TYPE>(reinterpret_cast<const char*>(a.W) + (label * a.ldw + k) * type_bytes(TYPE));
  }
  uint32_t bytes = 0;
  uint8_t* const codes = a.codes + unit * mx_code_bytes(a.d) + mx_step_codes(step);
#pragma unroll
  for (int t = 0; t < MX_TILES; ++t) {
    float by;
    const uint32_t byte = block_scale<2>(f[t], by);
    bytes |= byte << (8 * t);
    if (block < wide) *reinterpret_cast<uint32_t*>(codes + ((t * 16 + row) * wide + block) * 16 + part * 4) = to_fp4(f[t], by);
  }
  if (part == 0) *reinterpret_cast<uint32_t*>(a.scales + unit * mx_scale_bytes(a.d) + mx_step_scales(step) + block * 64 + row * 4) = bytes;
}

template <int TYPE>
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(MxArgs a) {
  const int64_t unit = blockIdx.x / (unsigned)a.steps;
  const int step = blockIdx.x % (unsigned)a.steps;
  const int lane = threadIdx.x & 63, row = 4 * (threadIdx.x >> 6) + (lane >> 4), block = (lane >> 2) & 3, part = lane & 3;
  const int k = step * MX_STEP + block * MX_BLOCK + part * 8;
  const int wide = mx_wide(step, a.blocks);
  if (block >= wide || k >= a.d) return;
  const uint32_t bytes = *reinterpret_cast<const uint32_t*>(a.scales + unit * mx_scale_bytes(a.d) + mx_step_scales(step) + block * 64 + row * 4);
  const uint8_t* const codes = a.codes + unit * mx_code_bytes(a.d) + mx_step_codes(step);
#pragma unroll
  for (int t = 0; t < MX_TILES; ++t) {
    const int64_t label = unit * MX_UNIT + mx_label(t, row);
    const uint32_t c = *reinterpret_cast<const uint32_t*>(codes + ((t * 16 + row) * wide + block) * 16 + part * 4);
    const Float8 f = from_fp4(c, scale_value((bytes >> (8 * t)) & 255u));
    if (label >= a.L) continue;
    store8<TYPE>(reinterpret_cast<char*>(a.out) + (label * a.ldw + k) * type_bytes(TYPE), f);
  }
}

// ---------------------------------------------------------------------------------------------
// embeddings in blocks, as the B side of the product
// ---------------------------------------------------------------------------------------------
// A fragment is 16 rows x one step: 1 KB of codes in 4 bits, 2 KB in 8, lane after lane.  In 8 bits the MFMA takes dims 16 q .. 16 q
// + 15 of the step from lane (i, q)'s first sixteen bytes and 64 + 16 q .. from the other sixteen (checked on hardware), so that block b is
// half b / 2 of lanes (i, 2 (b % 2)) and (i, 2 (b % 2) + 1); its scale is lane (i, b)'s all the same.
template <bool X8>
struct MxRows {
  static constexpr int FRAG = X8 ? 2048 : 1024;
  static constexpr int EMAX = X8 ? 8 : 2;
  // Where the eight numbers `part` of row i's block stand.
  static __device__ __forceinline__ int at(int i, int block, int part) {
    if constexpr (X8) return (block >> 1) * 1024 + ((2 * (block & 1) + (part >> 1)) * 16 + i) * 16 + (part & 1) * 8;
    else return (block * 16 + i) * 16 + part * 4;
  }
  // Quantises them (four neighbouring lanes hold a block; V: Float8 or half8) and returns the scale byte.
  template <class V>
  static __device__ __forceinline__ uint32_t put(unsigned char* frag, V f, int i, int block, int part) {
    float by;
    const uint32_t byte = block_scale<EMAX>(f, by);
    if constexpr (X8) *reinterpret_cast<uint64_t*>(frag + at(i, block, part)) = to_fp8(f, by);
    else *reinterpret_cast<uint32_t*>(frag + at(i, block, part)) = to_fp4(f, by);
    return byte;
  }
  static __device__ __forceinline__ int8v get(const unsigned char* frag, int lane) {
    const int4v lo = *reinterpret_cast<const int4v*>(frag + lane * 16);
    if constexpr (X8) {
      const int4v hi = *reinterpret_cast<const int4v*>(frag + 1024 + lane * 16);
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return __builtin_shufflevector(lo, lo, 0, 1, 2, 3, -1, -1, -1, -1);
  }
};

// c + labels (codes a, scale byte T of sa) . rows (codes b, scale byte J of sb)
template <bool X8, int T, int J>
__device__ __forceinline__ float4v mx_mfma(const int4v& a, uint32_t sa, const int8v& b, uint32_t sb, const float4v& c) {
  const int8v a8 = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b, c, 4, X8 ? 0 : 4, T, (int)sa, J, (int)sb);
}

// Eight numbers of a row of an embedding matrix of any type.
__device__ __forceinline__ Float8 load8_of(const void* X, int type, int64_t at) {
  if (type == XFC_F32) return load8<XFC_F32>(reinterpret_cast<const float*>(X) + at);
  if (type == XFC_BF16) return load8<XFC_BF16>(reinterpret_cast<const uint16_t*>(X) + at);
  return load8<XFC_F16>(reinterpret_cast<const half_t*>(X) + at);
}

// ---------------------------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------------------------
// A uniform address as the scalar half of a fetch's address: the compiler adds it up per lane otherwise.
__device__ __forceinline__ const XFC_GLB uint8_t* scalar(const uint8_t* p) {
  const XFC_GLB uint8_t* g = (const XFC_GLB uint8_t*)p;
  asm volatile("" : "+s"(g));
  return g;
}

// MX_LOGITS: logits.  MX_LOGITS_MAX: the same for a selection, numbers only (a NaN becomes -inf), with the largest of every 32.
// MX_MAXIMA: the largest sum of every unit, or of every half of one.  MX_HALF_MAXIMA: the largest of every 32 as a logit, no number counts
// as -inf.
enum MxOut { MX_LOGITS, MX_LOGITS_MAX, MX_MAXIMA, MX_HALF_MAXIMA };

struct MxProductArgs {
  const void* X; int type; int64_t ldx;  // M rows of K
  const uint8_t* codes; const uint8_t* scales;
  half_t* out; int64_t ldo;              // logits
  half_t* hmax; float* bmax; int64_t ldb; // beside logits; alone: one float for a unit, two, or two halves
  bool fine;                              // MX_MAXIMA: of half units, which run = 1 alone has
  int M, N, K;
  int units, blocks, steps;
  int tiles_m, slots;                    // row tiles; workgroups of a row tile on an XCD
  int run;                               // units in a row that a wave takes, 1 or 4
};

constexpr int MX_WAVES = 8, MX_SLOTS = 2;

// The first n of eight halves, to a place that begins on 16 bytes.
__device__ __forceinline__ void store_first(half_t* to, const half8& h, int n) {
  const uint4v v = __builtin_bit_cast(uint4v, h);
  if (n >= 8) {
    *reinterpret_cast<uint4v*>(to) = v;
  } else if (n > 0) {
    typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
    uint2v left = {v[0], v[1]};
    if (n & 4) {
      *reinterpret_cast<uint2v*>(to) = left;
      left = uint2v{v[2], v[3]};
      to += 4;
    }
    uint32_t last = left[0];
    if (n & 2) {
      *reinterpret_cast<uint32_t*>(to) = last;
      last = left[1];
      to += 2;
    }
    if (n & 1) *reinterpret_cast<uint16_t*>(to) = (uint16_t)last;
  }
}

// The largest of a lane's eight labels of half p of a unit, for its row of row tile j.
template <int NT>
__device__ __forceinline__ float mx_largest(const float4v (&acc)[MX_TILES][NT], int j, int p) {
  const float4v lo = acc[2 * p][j < NT ? j : NT - 1], hi = acc[2 * p + 1][j < NT ? j : NT - 1];
  return max3_num(max3_num(lo[0], lo[1], lo[2]), lo[3], max3_num(hi[0], hi[1], max_num(hi[2], hi[3])));
}
// ... over the four lanes that have the row: of four row tiles, lane group g ends up with tile 4 n + g.
template <class Of>
__device__ __forceinline__ float mx_over_lanes(int n, Of&& of) {
  return fold16(fold32(of(4 * n), of(4 * n + 2)), fold32(of(4 * n + 1), of(4 * n + 3)));
}
// Both halves' maxima as logits, in a float's place; no number is -inf.
template <int NT>
__device__ __forceinline__ float mx_half_maxima(const float4v (&acc)[MX_TILES][NT], int n) {
  typedef half_t half2v __attribute__((ext_vector_type(2)));
  const float least = -__builtin_huge_valf();
  const half2v two = {(half_t)max_num(mx_over_lanes(n, [&](int j) { return mx_largest(acc, j, 0); }), least),
                      (half_t)max_num(mx_over_lanes(n, [&](int j) { return mx_largest(acc, j, 1); }), least)};
  return __builtin_bit_cast(float, two);
}
// The maxima above are inline asm, in front of which the compiler puts no wait states: the last MFMAs' results are waited for here.  Labels behind the last
// are made no numbers.
template <int NT>
__device__ __forceinline__ void mx_before_maxima(float4v (&acc)[MX_TILES][NT], int label0, int labels, int q) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 15");
  __builtin_amdgcn_sched_barrier(0);
  if (label0 + MX_UNIT > labels) {
#pragma unroll
    for (int t = 0; t < MX_TILES; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool in = label0 + mx_label(t, 4 * q + r) < labels;
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[t][j][r] = in ? acc[t][j][r] : __builtin_nanf("");
      }
  }
}

// Bound, with few rows, by the stream of codes: 16 rows x 131,072 x 768 12.8 us for 54 MB of them and 4 of logits, 4.5 TB/s.  With many, logits
// by the memory that they go to (512 x 1,310,720: 1.34 GB of them beside 0.53 of codes, 455 us at best, 530 to 590 with a warm chip), maxima by the
// matrix pipes' power: 1024 x 2,812,281 x 768 with 4-bit rows took 990 to 1,080 us, 4.1 to 4.5 PFLOP/s (registers alone
// reach 7 PFLOP/s on random numbers, 9.6 on zeros); without the fetches it was 200 us less, without the maxima 90: mx4_wide_kernel has such calls now.
//
// A workgroup keeps its rows' fragments in the LDS and its waves, which never meet again, stream units of 64 labels past them, straight
// into the A side's registers: two steps on their way, across units.  (Three or six took as long where there is much to do, and longer where
// there is little, by the size of the code: 16 rows x 131,072 labels 12.8, 13.5, 17.7 us.)
template <int NT, bool X8, int OUT>
__global__ void __launch_bounds__(64 * MX_WAVES, NT >= 4 ? 2 : 4) mx4_product_kernel(MxProductArgs a) {
  using Rows = MxRows<X8>;
  constexpr int NS = (NT + 3) / 4;  // dwords of row scales of a step
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[];
  unsigned char* const frags = smem_raw;
  unsigned char* const row_scales = smem_raw + a.steps * NT * Rows::FRAG;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, q = lane >> 4;
  const int xcd = blockIdx.x & 7, local = blockIdx.x >> 3;
  const int row0 = (local % a.tiles_m) * 16 * NT;
  const int workers = 8 * a.slots * MX_WAVES, worker = (xcd * a.slots + local / a.tiles_m) * MX_WAVES + wave;
  const int run = a.run, skip = (workers - 1) * run + 1;  // from the last unit of a run to the first of the next
  auto next = [&](int u) { return (u + 1) & (run - 1) ? u + 1 : u + skip; };
  int unit = worker * run;

  // Fetch cursor.  Past the last unit it repeats that one, so that as many loads are on their way as ever.
  const int64_t unit_codes = mx_code_bytes(a.K), unit_scales = mx_scale_bytes(a.K);
  const int whole = a.blocks >> 2, wide = a.blocks & 3;  // steps of four blocks, blocks of the step behind them
  const uint32_t at_whole = (uint32_t)(4 * i + q) * 16, at_rest = (uint32_t)(wide * i + (q < wide ? q : wide - 1)) * 16;
  int f_unit = unit < a.units ? unit : a.units - 1, f_step = 0;
  struct Slot { int4v w[MX_TILES]; uint32_t s; };
  Slot slot[MX_SLOTS];
  auto fetch = [&](Slot& to) __attribute__((always_inline)) {
    const uint8_t* const c = a.codes + (int64_t)f_unit * unit_codes + f_step * 4096;
    const uint8_t* const s = a.scales + (int64_t)f_unit * unit_scales + f_step * 256;
    const bool rest = f_step == whole;
    const uint32_t at = rest ? at_rest : at_whole, tile = rest ? (uint32_t)wide * 256 : 1024u;
#pragma unroll
    for (int t = 0; t < MX_TILES; ++t) to.w[t] = *reinterpret_cast<const XFC_GLB int4v*>(scalar(c + t * tile) + at);
    to.s = *reinterpret_cast<const XFC_GLB uint32_t*>(scalar(s) + (uint32_t)lane * 4);
    if (++f_step == a.steps) {
      f_step = 0;
      if (next(f_unit) < a.units) f_unit = next(f_unit);
    }
  };
#pragma unroll
  for (int s = 0; s < MX_SLOTS; ++s) fetch(slot[s]);

  // The rows' blocks, four lanes each, 16 lanes a step of a row, 32 rows at a time, FILL steps on their way; behind the last row, dim or
  // block there are zeros.
  constexpr int FILL = 3;
  auto fill = [&](auto load) __attribute__((always_inline)) {
    const int part = tid & 3, block = (tid >> 2) & 3, k = block * MX_BLOCK + part * 8;
    for (int r = tid >> 4; r < 16 * NT; r += 4 * MX_WAVES) {
      const int j = r >> 4;
      for (int s0 = 0; s0 < a.steps; s0 += FILL) {
        decltype(load((int64_t)0)) v[FILL];
#pragma unroll
        for (int n = 0; n < FILL; ++n) {
          v[n] = {};
          if (row0 + r < a.M && (s0 + n) * MX_STEP + k < a.K) v[n] = load((int64_t)(row0 + r) * a.ldx + (s0 + n) * MX_STEP + k);
        }
#pragma unroll
        for (int n = 0; n < FILL; ++n) {
          const int step = s0 + n;
          if (step >= a.steps) break;
          const uint32_t byte = Rows::put(frags + (step * NT + j) * Rows::FRAG, v[n], r & 15, block, part);
          if (part == 0) row_scales[((step * NS + (j >> 2)) * 64 + block * 16 + (r & 15)) * 4 + (j & 3)] = (unsigned char)byte;
        }
      }
    }
  };
  if (a.type == XFC_F16) fill([&](int64_t at) { return *reinterpret_cast<const half8*>(reinterpret_cast<const half_t*>(a.X) + at); });
  else if (a.type == XFC_BF16) fill([&](int64_t at) { return load8<XFC_BF16>(reinterpret_cast<const uint16_t*>(a.X) + at); });
  else fill([&](int64_t at) { return load8<XFC_F32>(reinterpret_cast<const float*>(a.X) + at); });
  __syncthreads();

  float4v acc[MX_TILES][NT];
  [[maybe_unused]] float4v best[NS];  // of up to four units in a row
  int step = 0;

  // Row fragments run AHEAD of the MFMAs that read them, over the steps' ends: a step's first ones are read under the last MFMAs of the one before.
  constexpr int RING = NT < 4 ? NT : 4, AHEAD = (RING + 1) / 2;
  int8v ring[RING];
  uint32_t sb[2][NS];
  auto read_rows = [&](int of, auto jt) { ring[decltype(jt)::value % RING] = Rows::get(frags + (of * NT + decltype(jt)::value) * Rows::FRAG, lane); };
  auto read_scales = [&](int of, uint32_t (&to)[NS]) {
#pragma unroll
    for (int n = 0; n < NS; ++n) to[n] = *reinterpret_cast<const uint32_t*>(row_scales + ((of * NS + n) * 64 + lane) * 4);
  };
  [&]<int... J>(std::integer_sequence<int, J...>) { (read_rows(0, std::integral_constant<int, J>{}), ...); }(std::make_integer_sequence<int, AHEAD>{});
  read_scales(0, sb[0]);
  auto multiply = [&](const Slot& w, auto first) __attribute__((always_inline)) {
    const int after = step + 1 == a.steps ? 0 : step + 1;
    read_scales(after, sb[1]);
    auto row_tile = [&](auto jt) {
      constexpr int J = decltype(jt)::value, NEXT = (J + AHEAD) % NT;
      const int8v b = ring[J % RING];
      read_rows(J + AHEAD < NT ? step : after, std::integral_constant<int, NEXT>{});
      auto tile = [&](auto tt) {
        constexpr int T = decltype(tt)::value;
        acc[T][J] = mx_mfma<X8, T, J % 4>(w.w[T], w.s, b, sb[0][J / 4], decltype(first)::value ? float4v{0.f, 0.f, 0.f, 0.f} : acc[T][J]);
      };
      [&]<int... T>(std::integer_sequence<int, T...>) { (tile(std::integral_constant<int, T>{}), ...); }(std::make_integer_sequence<int, MX_TILES>{});
      if constexpr (NT > 1) __builtin_amdgcn_sched_barrier(0);
    };
    [&]<int... J>(std::integer_sequence<int, J...>) { (row_tile(std::integral_constant<int, J>{}), ...); }(std::make_integer_sequence<int, NT>{});
#pragma unroll
    for (int n = 0; n < NS; ++n) sb[0][n] = sb[1][n];
  };

  auto epilogue = [&]() __attribute__((always_inline)) {
    // (Made anew each time: kept over the loop, the rows' addresses would take the registers of the fragments under way.)
    int lane_now = lane;
    asm volatile("" : "+v"(lane_now));
    const int i = lane_now & 15, q = lane_now >> 4;
    const int label0 = unit * MX_UNIT;
    const bool edge = label0 + MX_UNIT > a.N;
    if constexpr (OUT == MX_MAXIMA || OUT == MX_HALF_MAXIMA) {
      mx_before_maxima(acc, label0, a.N, q);
      if (OUT == MX_MAXIMA && a.fine) {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          const float m0 = mx_over_lanes(n, [&](int j) { return mx_largest(acc, j, 0); }), m1 = mx_over_lanes(n, [&](int j) { return mx_largest(acc, j, 1); });
          const int row = row0 + 64 * n + lane_now;
          if (4 * n + q < NT && row < a.M) *reinterpret_cast<float2v*>(a.bmax + (int64_t)row * a.ldb + 2 * (int64_t)unit) = float2v{m0, m1};
        }
      } else {
        const int r4 = unit & (run - 1);
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          float m;
          if constexpr (OUT == MX_MAXIMA) m = mx_over_lanes(n, [&](int j) { return max_num(mx_largest(acc, j, 0), mx_largest(acc, j, 1)); });
          else m = mx_half_maxima(acc, n);
#pragma unroll
          for (int r = 0; r < 4; ++r) best[n][r] = r4 == r ? m : best[n][r];
        }
        const int after = next(unit);
        if (after != unit + 1 || run == 1 || after >= a.units) {
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            const int row = row0 + 64 * n + lane_now;
            if (4 * n + q >= NT || row >= a.M) continue;
            float* const to = a.bmax + (int64_t)row * a.ldb + (unit - r4);
            if (run == 1) *to = best[n][0];
            else *reinterpret_cast<float4v*>(to) = best[n];
          }
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        half8 h[2];  // of row i's two halves of the unit
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
          for (int r = 0; r < 4; ++r) { h[p][r] = (half_t)acc[2 * p][j][r]; h[p][4 + r] = (half_t)acc[2 * p + 1][j][r]; }
          if constexpr (OUT == MX_LOGITS_MAX) {
#pragma unroll
            for (int e = 0; e < 8; ++e) h[p][e] = h[p][e] == h[p][e] ? h[p][e] : (half_t)-__builtin_huge_valf();
          }
        }
        const int row = row0 + 16 * j + i;
        if (OUT == MX_LOGITS_MAX || !edge) {  // (a selection's rows have room for whole units)
          // Neighbouring lanes swap halves: a store is eight rows of 128 bytes, whole lines, where it was sixteen of 64.  (512 x 1,310,720 x
          // 768: 588 -> 529 us.  Past the caches they take as long.)
          const bool odd = i & 1;
          const uint4v lo = __builtin_bit_cast(uint4v, h[0]), hi = __builtin_bit_cast(uint4v, h[1]);
          uint4v even_row, odd_row;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t got = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(odd ? lo[e] : hi[e]), 0xb1, 0xf, 0xf, true);  // quad_perm 1, 0, 3, 2
            even_row[e] = odd ? got : lo[e];
            odd_row[e] = odd ? hi[e] : got;
          }
          const int first = row & ~1;
          half_t* const to = a.out + (int64_t)first * a.ldo + label0 + (odd ? 32 : 0) + 8 * q;
          if (first < a.M) *reinterpret_cast<uint4v*>(to) = even_row;
          if (first + 1 < a.M) *reinterpret_cast<uint4v*>(to + a.ldo) = odd_row;
        } else if (row < a.M) {
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const int col = label0 + 32 * p + 8 * q;
            store_first(a.out + (int64_t)row * a.ldo + col, h[p], a.N - col);
          }
        }
        if constexpr (OUT == MX_LOGITS_MAX) {
          if (edge) {
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
              for (int e = 0; e < 8; ++e) h[p][e] = label0 + 32 * p + 8 * q + e < a.N ? h[p][e] : (half_t)-__builtin_huge_valf();
          }
          const uint32_t v = pk_fold32(pk_max(h[0]), pk_max(h[1]));
          const half_t m = pk_larger(pk_fold16(v, v));
          if (a.hmax && row < a.M && (q & 1) == 0) a.hmax[(int64_t)row * a.ldb + 2 * (int64_t)unit + (q >> 1)] = m;
        }
      }
    }
  };

  auto turn = [&](Slot& w) __attribute__((always_inline)) {
    if (unit < a.units) {
      if (step == 0) multiply(w, std::true_type{});
      else multiply(w, std::false_type{});
      if (++step == a.steps) {
        epilogue();
        step = 0;
        unit = next(unit);
      }
    }
    fetch(w);  // (whatever way was taken: else the compiler could not tell how many are on their way, and would wait for all)
  };
  static_assert(MX_SLOTS == 2, "turns");
  while (unit < a.units) {  // (written out: a loop of this size would stay one, with the slots in scratch memory)
    turn(slot[0]);
    turn(slot[1]);
  }
}

// Maxima of many rows of 4 bits and many labels: the rows stay in registers, 64 of them a wave for as long as the kernel runs, and the codes are streamed through
// the LDS, two units at a time (a section) that all eight waves multiply with: 512 rows a workgroup where the kernel above has 128, so that a quarter of the codes
// cross from the L2s, for as many bytes out of the LDS.  (1024 x 2,812,281 x 768 1,071 -> 958 us, 512 x 1,310,720 282 -> 260; the first 13 of them
// quantise rows, which is why there have to be many labels.  With 8 bits, 256 rows a workgroup, 1.00 to 1.05 of the kernel above; logits 564 -> 730, whose rows
// are written in shorter pieces.)
template <int STEPS>
struct MxSection {
  static constexpr int UNITS = 2, CODES = UNITS * STEPS * 4096, SCALES = (UNITS * STEPS * 256 + 1023) / 1024 * 1024, BYTES = CODES + SCALES;
  static constexpr int SLOTS = 3;      // one in use, two on their way
  static constexpr int FETCHES = STEPS + 1;  // of a wave
  static_assert(SLOTS * BYTES <= 160 * 1024, "LDS");
};
constexpr int MX_WIDE_TILES = 4, MX_WIDE_ROWS = MX_WAVES * 16 * MX_WIDE_TILES;

// f(0) ... f(N - 1), as constants: what indexes registers has to be written out, which the compiler leaves off with loops of that size.
template <int N, class Fn>
__device__ __forceinline__ void written_out(Fn&& f) {
  [&]<int... I>(std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }(std::make_integer_sequence<int, N>{});
}

template <int STEPS, int OUT>
__global__ void __launch_bounds__(64 * MX_WAVES) mx4_wide_kernel(MxProductArgs a) {
  using Rows = MxRows<false>;
  using Section = MxSection<STEPS>;
  constexpr int NR = MX_WIDE_TILES;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, q = lane >> 4;
  const int xcd = blockIdx.x & 7, local = blockIdx.x >> 3;
  const int row0 = ((local % a.tiles_m) * MX_WAVES + wave) * 16 * NR;
  const int workers = 8 * a.slots, worker = xcd * a.slots + local / a.tiles_m;
  const int sections = (a.units + Section::UNITS - 1) / Section::UNITS;
  const int64_t unit_codes = mx_code_bytes(a.K), unit_scales = mx_scale_bytes(a.K);

  // A section's tiles lie in the LDS as lanes read them, one after the other, whatever the width (of a block that is none any other).  Past the last
  // section that one is fetched again, so that as many fetches are on their way as ever; of a unit that is none, the one before.
  const int whole = a.blocks >> 2, wide = a.blocks & 3;  // steps of four blocks, blocks of the step behind them
  const uint32_t at_whole = (uint32_t)(4 * i + q) * 16, at_rest = (uint32_t)(wide * i + (q < wide ? q : wide - 1)) * 16;
  auto fetch = [&](int section, int slot) __attribute__((always_inline)) {
    const int sec = section < sections ? section : sections - 1;
    const int units = a.units - sec * Section::UNITS < Section::UNITS ? a.units - sec * Section::UNITS : Section::UNITS;
    unsigned char* const to = smem_raw + slot * Section::BYTES;
    const uint8_t* const c = a.codes + (int64_t)sec * Section::UNITS * unit_codes;
    const uint8_t* const s = a.scales + (int64_t)sec * Section::UNITS * unit_scales;
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {  // tiles, dealt to the waves
      const int at = (wave >> 2) + 2 * n, u = at >= STEPS && units > 1 ? 1 : 0, step = at >= STEPS ? at - STEPS : at, tile = wave & 3;
      const bool rest = step >= whole;
      load16_to_lds(c + u * unit_codes + (rest ? whole * 4096 + tile * wide * 256 : step * 4096 + tile * 1024), rest ? at_rest : at_whole,
                    to + (wave + MX_WAVES * n) * 1024);
    }
    // (waves that have no part of the scales fetch the first once more)
    const uint32_t part = wave * 1024 < Section::SCALES ? wave * 1024 : 0, at = part + lane * 16, last = (uint32_t)(units * unit_scales) - 16;
    load16_to_lds(s, at < last ? at : last, to + Section::CODES + part);
  };
  fetch(worker, 0);

  // The wave's rows, quantised as in the kernel above, a tile at a time through its part of the other slots.
  int8v rows[STEPS][NR];
  uint32_t row_scales[STEPS] = {};
  constexpr int ROOM = (Section::SLOTS - 1) * Section::BYTES / MX_WAVES / 16 * 16;
  static_assert(ROOM >= STEPS * (Rows::FRAG + 64), "room for a tile");
  unsigned char* const stage = smem_raw + Section::BYTES + wave * ROOM;
  unsigned char* const stage_scales = stage + STEPS * Rows::FRAG;
  auto lds_done = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
  auto fill = [&](auto many, auto load) __attribute__((always_inline)) {
    constexpr int N = decltype(many)::value;  // rows of a lane on their way
    const int part = lane & 3, block = (lane >> 2) & 3, k = block * MX_BLOCK + part * 8;
    written_out<NR>([&](auto jt) __attribute__((always_inline)) {
      constexpr int j = decltype(jt)::value;
#pragma unroll
      for (int r0 = lane >> 4; r0 < 16; r0 += 4 * N) {
        decltype(load((int64_t)0)) v[N][STEPS];
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int row = row0 + 16 * j + r0 + 4 * n;
#pragma unroll
          for (int s = 0; s < STEPS; ++s) {
            v[n][s] = {};
            if (row < a.M && s * MX_STEP + k < a.K) v[n][s] = load((int64_t)row * a.ldx + s * MX_STEP + k);
          }
        }
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int s = 0; s < STEPS; ++s) {
            const uint32_t byte = Rows::put(stage + s * Rows::FRAG, v[n][s], r0 + 4 * n, block, part);
            if (part == 0) stage_scales[s * 64 + block * 16 + r0 + 4 * n] = (unsigned char)byte;
          }
      }
      lds_done();
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        rows[s][j] = Rows::get(stage + s * Rows::FRAG, lane);
        row_scales[s] |= (uint32_t)stage_scales[s * 64 + lane] << (8 * j);
      }
      lds_done();
    });
  };
  if (a.type == XFC_F16) fill(std::integral_constant<int, 4>{}, [&](int64_t at) { return *reinterpret_cast<const half8*>(reinterpret_cast<const half_t*>(a.X) + at); });
  else fill(std::integral_constant<int, 1>{}, [&](int64_t at) { return load8_of(a.X, a.type, at); });
  asm volatile("s_barrier" ::: "memory");
#pragma unroll
  for (int s = 1; s < Section::SLOTS; ++s) fetch(worker + s * workers, s);

  struct Slot { int4v w[MX_TILES]; uint32_t s; };
  Slot slot[2];
  auto read = [&](const unsigned char* c, int u, int step, Slot& to) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < MX_TILES; ++t) to.w[t] = *reinterpret_cast<const int4v*>(c + ((u * STEPS + step) * MX_TILES + t) * 1024 + lane * 16);
    to.s = *reinterpret_cast<const uint32_t*>(c + Section::CODES + u * (int)unit_scales + step * 256 + lane * 4);
  };
  float4v acc[MX_TILES][NR];
  int in = 0;
  // What this wave has asked for of the first section is there, and after the barrier what all have.
  wait_vmcnt<(Section::SLOTS - 1) * Section::FETCHES>();
  asm volatile("s_barrier" ::: "memory");
  for (int section = worker; section < sections; section += workers) {
    const unsigned char* const c = smem_raw + in * Section::BYTES;
    float4v best = {};
    read(c, 0, 0, slot[0]);
    written_out<Section::UNITS>([&](auto ut) __attribute__((always_inline)) {
      constexpr int U = decltype(ut)::value;
      written_out<STEPS>([&](auto st) __attribute__((always_inline)) {
        constexpr int STEP = decltype(st)::value, NOW = (U * STEPS + STEP) & 1;
        if constexpr (STEP + 1 < STEPS) read(c, U, STEP + 1, slot[NOW ^ 1]);
        else if constexpr (U + 1 < Section::UNITS) read(c, U + 1, 0, slot[NOW ^ 1]);
        __builtin_amdgcn_sched_barrier(0);
        written_out<NR>([&](auto jt) __attribute__((always_inline)) {
          written_out<MX_TILES>([&](auto tt) __attribute__((always_inline)) {
            constexpr int J = decltype(jt)::value, T = decltype(tt)::value;
            acc[T][J] = mx_mfma<false, T, J>(slot[NOW].w[T], slot[NOW].s, rows[STEP][J], row_scales[STEP], STEP == 0 ? float4v{0.f, 0.f, 0.f, 0.f} : acc[T][J]);
          });
        });
        __builtin_amdgcn_sched_barrier(0);
      });
      mx_before_maxima(acc, (section * Section::UNITS + U) * MX_UNIT, a.N, q);
      if constexpr (OUT == MX_MAXIMA) best[U] = mx_over_lanes(0, [&](int j) { return max_num(mx_largest(acc, j, 0), mx_largest(acc, j, 1)); });
      else best[U] = mx_half_maxima(acc, 0);
    });
    // The next section is there, and all have read this one.  (Fetches and stores return in order.)
    wait_vmcnt<(Section::SLOTS - 2) * Section::FETCHES>();
    asm volatile("s_barrier" ::: "memory");
    fetch(section + Section::SLOTS * workers, in);
    in = in + 1 == Section::SLOTS ? 0 : in + 1;
    const int row = row0 + lane;
    if (row < a.M) *reinterpret_cast<float2v*>(a.bmax + (int64_t)row * a.ldb + 2 * (int64_t)section) = float2v{best[0], best[1]};
  }
  wait_vmcnt<0>();  // of fetches into the LDS that no wave has any more
}

// The scores of sixteen labels of a row formed again, for topk_pick_kernel and below: any sixteen, each lane of the A side fetches its own.  The
// row, quantised once, stands in all sixteen columns; a sum's MFMAs and their order are those of mx4_product_kernel.
template <bool X8>
struct MxScores {
  const void* X; int type; int64_t ldx;
  const uint8_t* codes; const uint8_t* scales;

  static constexpr int MANY = 2;  // groups of labels whose fetches are on their way together
  static __device__ __forceinline__ unsigned char* room() {
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[];
    return smem_raw;
  }
  // bytes of a step: block q's numbers behind each other, then four scale bytes
  static constexpr int STEP_BYTES = (X8 ? 128 : 64) + 16;
  __host__ __device__ static int64_t lds(int64_t d) { return (int64_t)mx_steps(d) * STEP_BYTES; }

  __device__ __forceinline__ void open(const PickArgs& a, int row) const {
    unsigned char* const at = room();
    for (int w = threadIdx.x; w < mx_steps(a.K) * 16; w += blockDim.x) {
      const int part = w & 3, block = (w >> 2) & 3, step = w >> 4, k = w * 8;
      Float8 f = {};
      if (k < a.K) f = load8_of(X, type, (int64_t)row * ldx + k);
      float by;
      const uint32_t byte = block_scale<X8 ? 8 : 2>(f, by);
      unsigned char* const s = at + step * STEP_BYTES;
      if constexpr (X8) *reinterpret_cast<uint64_t*>(s + (block * 4 + part) * 8) = to_fp8(f, by);
      else *reinterpret_cast<uint32_t*>(s + (block * 4 + part) * 4) = to_fp4(f, by);
      if (part == 0) s[STEP_BYTES - 16 + block] = (unsigned char)byte;
    }
  }
  // Labels first .. first + 15, first a multiple of 16: lane (., q) has four of them, first + 4 q on.
  static __device__ __forceinline__ int place(int part, int lane) { return 16 * part + 4 * (lane >> 4); }
  __device__ __forceinline__ void score(const PickArgs& a, const int (&first)[MANY], int lane, float4v (&z)[MANY]) const {
    const int blocks = mx_blocks(a.K), steps = mx_steps(a.K), i = lane & 15, q = lane >> 4;
    const unsigned char* const at = room();
    const uint8_t* c[MANY];
    const uint8_t* s[MANY];
    int tile[MANY], row[MANY];
#pragma unroll
    for (int m = 0; m < MANY; ++m) {
      const int64_t unit = first[m] / MX_UNIT;
      const int within = first[m] % MX_UNIT + i;
      tile[m] = mx_tile(within);
      row[m] = mx_row(within);
      c[m] = codes + unit * mx_code_bytes(a.K);
      s[m] = scales + unit * mx_scale_bytes(a.K) + q * 64 + row[m] * 4 + tile[m];
      z[m] = float4v{0.f, 0.f, 0.f, 0.f};
    }
    constexpr int AT_ONCE = 6;  // steps on their way together
    for (int s0 = 0; s0 < steps; s0 += AT_ONCE) {
      int4v w[MANY][AT_ONCE];
      uint32_t sa[MANY][AT_ONCE];
#pragma unroll
      for (int m = 0; m < MANY; ++m)
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          const int step = s0 + j < steps ? s0 + j : steps - 1, wide = blocks - 4 * step < 4 ? blocks - 4 * step : 4;
          w[m][j] = *reinterpret_cast<const int4v*>(c[m] + mx_code_at(tile[m], row[m], 4 * step + (q < wide ? q : wide - 1), blocks));
          sa[m][j] = s[m][step * 256];
        }
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        if (s0 + j >= steps) break;
        const unsigned char* const x = at + (s0 + j) * STEP_BYTES;
        int8v b;
        if constexpr (X8) {
          const int4v lo = *reinterpret_cast<const int4v*>(x + q * 16), hi = *reinterpret_cast<const int4v*>(x + 64 + q * 16);
          b = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
          const int4v lo = *reinterpret_cast<const int4v*>(x + q * 16);
          b = __builtin_shufflevector(lo, lo, 0, 1, 2, 3, -1, -1, -1, -1);
        }
        const uint32_t sb = x[STEP_BYTES - 16 + q];
#pragma unroll
        for (int m = 0; m < MANY; ++m) z[m] = mx_mfma<X8, 0, 0>(w[m][j], sa[m][j], b, sb, z[m]);
      }
    }
  }
};

// ---------------------------------------------------------------------------------------------
// 8 < K <= MX_SELECT_K without logits: the K best blocks of 32 labels by their maxima, their scores formed again
// ---------------------------------------------------------------------------------------------
// Why that is exact: as in topk.hpp, with scores rounded to fp16; the K-th best maximum is no larger than the K-th best score, so
// that of the K blocks' scores only those that reach it are put in order.
//
// One workgroup per row.  The K-th largest of the threads' own largest maxima, to eleven bits, is no larger than the K-th maximum; the blocks that
// reach it, a few more than K, are listed and ranked by comparing each with all.  Only if there is no room for them (rows of many
// equal scores) are the maxima counted by their upper eleven bits and then, in the bin that the K-th is in, by the lower five, and of those
// at the K-th key the first ones taken.  The waves then form the scores, a block at a time each.  Bound by fetching K x 32 labels
// a row, after some 25 us for the blocks: 512 rows x 40,960 blocks, K = 100, 668 MB of codes and scales, 136 us.  (Blocks of 16 would halve that, but
// their maxima cost the product more than they save; blocks in the order of labels, for the rows to share fetches, 137 us.)
//
// More rows than the chip has CUs: two workgroups of 512 threads to a CU, one finds its blocks while the other fetches; else one of 1024.  (K = 100, us by
// 512 / by 1024, with the product: 512 rows x 1,310,720 x 768 363 / 373, 300 292 / 305, 256 239 / 216, 32 209 / 174; 512 x 320,001 x 64 53 / 62.)
constexpr int MX_SELECT_K = 256, MX_SELECT_BLOCK = 32, MX_SELECT_LIST = 512, MX_SELECT_BINS = 2048;

// (of PickArgs: bmax, two halves a float; n_blocks; N, K, topk, numy, out_v, out_i)
struct MxSelectLds {
  union {
    unsigned long long cand[MX_SELECT_K * MX_SELECT_BLOCK];
    struct {  // before there are any
      int hist[MX_SELECT_BINS];
      unsigned long long list[MX_SELECT_LIST];
    };
  };
  int block[MX_SELECT_K];
  int wave_tot[16];
  int bin, above, n_block, n_cand;
};

// fp16 bits as a key that orders like the value, -0 as +0, and back.
__device__ __forceinline__ uint32_t half_key(uint32_t h) {
  if (h == 0x8000u) h = 0u;
  return (h & 0x8000u) ? (~h & 0xffffu) : (h | 0x8000u);
}
__device__ __forceinline__ float half_unkey(uint32_t k) {
  const uint16_t h = (uint16_t)((k & 0x8000u) ? (k & 0x7fffu) : ~k);
  return (float)__builtin_bit_cast(half_t, h);
}

template <bool X8, int THREADS>
__global__ void __launch_bounds__(THREADS) mx4_select_kernel(PickArgs a, MxScores<X8> scores) {
  MxSelectLds& S = *reinterpret_cast<MxSelectLds*>(MxScores<X8>::room() + MxScores<X8>::lds(a.K));  // a multiple of 16
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int K = a.topk;  // there are more blocks
  const uint32_t* const maxima = reinterpret_cast<const uint32_t*>(a.bmax) + (int64_t)row * a.ldb;  // two blocks each
  const int quads = (a.n_blocks + 7) / 8;
  auto for_each = [&](auto&& f) {
    for (int w = tid; w < quads; w += THREADS) {
      const uint4v v = *reinterpret_cast<const uint4v*>(maxima + 4 * w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t h = (v[e >> 1] >> (16 * (e & 1))) & 0xffffu;
        if (8 * w + e < a.n_blocks) f(half_key(h), 8 * w + e);
      }
    }
  };
  // The bin of the K-th, counted down from the last; above: how many lie in higher ones.  Wave 0.
  auto find_bin = [&](int bins, int base) {
    if (wave == 0) {
      const int per = bins / 64;
      int mine = 0;
      for (int j = 0; j < per; ++j) mine += S.hist[lane * per + j];
      int from = mine;  // of this lane's bins and all higher ones
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int v = __shfl_down(from, off, 64);
        if (lane + off < 64) from += v;
      }
      const unsigned long long reach = __ballot(base + from >= K);
      if (lane == 63 - __builtin_clzll(reach | 1ull)) {
        int above = base + from - mine, b = lane * per + per - 1;
        for (; b > lane * per; --b) {
          if (above + S.hist[b] >= K) break;
          above += S.hist[b];
        }
        S.bin = b;
        S.above = above;
      }
    }
    __syncthreads();
  };
  // The same by counting all maxima; leaves the blocks and returns the K-th key.
  auto by_counts = [&]() -> uint32_t {
    for (int i = tid; i < MX_SELECT_BINS; i += THREADS) S.hist[i] = 0;
    if (tid == 0) S.n_block = 0;
    __syncthreads();
    for_each([&](uint32_t key, int) { atomicAdd(&S.hist[key >> 5], 1); });
    __syncthreads();
    find_bin(MX_SELECT_BINS, 0);
    const int top = S.bin, above = S.above;
    __syncthreads();
    if (tid < 64) S.hist[tid] = 0;
    __syncthreads();
    for_each([&](uint32_t key, int) { if ((int)(key >> 5) == top) atomicAdd(&S.hist[key & 31], 1); });
    __syncthreads();
    find_bin(64, above);
    const uint32_t least = (uint32_t)top * 32 + (uint32_t)S.bin;
    const int at_least = K - S.above;  // blocks at the K-th key that are taken, the first ones
    // (the list's order is of no matter)
    int taken = 0;
    for (int w0 = 0; w0 < quads; w0 += THREADS) {
      uint32_t here = 0, equal = 0;  // of this thread's eight blocks: above the key, at it
      if (w0 + tid < quads) {
        const uint4v v = *reinterpret_cast<const uint4v*>(maxima + 4 * (w0 + tid));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t key = half_key((v[e >> 1] >> (16 * (e & 1))) & 0xffffu);
          if (8 * (w0 + tid) + e < a.n_blocks) {
            here |= (key > least ? 1u : 0u) << e;
            equal |= (key == least ? 1u : 0u) << e;
          }
        }
      }
      // the equal ones' ranks, in the order of blocks
      int mine = __builtin_popcount(equal), rank = mine;
      const bool any = __syncthreads_or(mine != 0 && taken < at_least);
      if (any) {
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const int v = __shfl_up(rank, off, 64);
          if (lane >= off) rank += v;
        }
        if (lane == 63) S.wave_tot[wave] = rank;
        __syncthreads();
        int before = taken, all = 0;
        for (int w = 0; w < THREADS / 64; ++w) {
          before += w < wave ? S.wave_tot[w] : 0;
          all += S.wave_tot[w];
        }
        before += rank - mine;
        for (uint32_t left = equal; left && before < at_least; left &= left - 1, ++before) here |= left & (0u - left);
        taken += all;
      }
      for (; here; here &= here - 1) S.block[atomicAdd(&S.n_block, 1)] = 8 * (w0 + tid) + __builtin_ctz(here);
      __syncthreads();
    }
    return least;
  };
  for (int i = tid; i < MX_SELECT_BINS; i += THREADS) S.hist[i] = 0;
  if (tid == 0) S.n_block = S.n_cand = 0;
  scores.open(a, row);
  uint32_t largest = 0;
  for_each([&](uint32_t key, int) { largest = key > largest ? key : largest; });
  __syncthreads();
  if (tid < quads) atomicAdd(&S.hist[largest >> 5], 1);
  __syncthreads();
  find_bin(MX_SELECT_BINS, 0);
  const uint32_t bound = (uint32_t)S.bin * 32;
  for_each([&](uint32_t key, int block) {
    if (key < bound) return;
    const int at = atomicAdd(&S.n_block, 1);
    if (at < MX_SELECT_LIST) S.list[at] = ((unsigned long long)key << 32) | (uint32_t)~block;
  });
  __syncthreads();
  const int listed = S.n_block;
  __syncthreads();
  uint32_t least;
  if (listed <= MX_SELECT_LIST) {
    if (tid < listed) {
      const unsigned long long mine = S.list[tid];
      int rank = 0;
      for (int o = 0; o < listed; ++o) rank += S.list[o] > mine;
      if (rank < K) S.block[rank] = (int)~(uint32_t)mine;
      if (rank == K - 1) S.bin = (int)(mine >> 32);
    }
    __syncthreads();
    least = (uint32_t)S.bin;
  } else {
    least = by_counts();
  }
  const int n_block = K;
  for (int u = wave; u < n_block; u += THREADS / 64) {
    const int block = __builtin_amdgcn_readfirstlane(S.block[u]) * MX_SELECT_BLOCK;
    const int first[2] = {block, block + 16};
    float4v z[2];
    scores.score(a, first, lane, z);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      if ((lane & 15) != 0) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int label = first[m] + 4 * (lane >> 4) + r;
        const half_t h = z[m][r] == z[m][r] ? (half_t)z[m][r] : (half_t)-__builtin_huge_valf();
        const uint32_t key = half_key(__builtin_bit_cast(uint16_t, h));
        if (label < a.N && key >= least) S.cand[atomicAdd(&S.n_cand, 1)] = ((unsigned long long)key << 32) | (uint32_t)~label;
      }
    }
  }
  __syncthreads();
  auto write = [&](int at, unsigned long long c) {
    const int64_t label = (int64_t)(uint32_t)~(uint32_t)c;
    a.out_v[(int64_t)row * K + at] = half_unkey((uint32_t)(c >> 32));
    a.out_i[(int64_t)row * K + at] = label < a.numy ? label : a.numy - 1;
  };
  const int n = S.n_cand;
  if (n <= THREADS) {
    if (tid < n) {
      const unsigned long long mine = S.cand[tid];
      int rank = 0;
      for (int o = 0; o < n; ++o) rank += S.cand[o] > mine;
      if (rank < K) write(rank, mine);
    }
    return;
  }
  // bitonic over the next power of two
  int size = 64;
  while (size < n) size <<= 1;
  for (int i = n + tid; i < size; i += THREADS) S.cand[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = tid; i < size; i += THREADS) {
        const int o = i ^ j;
        if (o > i) {
          const unsigned long long x = S.cand[i], y = S.cand[o];
          if ((x < y) == ((i & k) == 0)) { S.cand[i] = y; S.cand[o] = x; }
        }
      }
      __syncthreads();
    }
  for (int i = tid; i < K; i += THREADS) write(i, S.cand[i]);
}

}  // namespace xfc

// Narrow label matrices and label preferences: the C entry points of mx4.hpp and preference.hpp.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include <stdio.h>

#include "../../include/xfc_mi355x.h"
#include "launch.hpp"
#include "mx4.hpp"
#include "preference.hpp"

using namespace xfc;

namespace {

bool type_ok(int t) { return t == XFC_F16 || t == XFC_BF16 || t == XFC_F32; }
// A row stride in elements, and whether rows of that type can be read in 16-byte pieces.
bool rows_ok(const void* p, int type, int64_t ld) { return aligned16(p) && ld % (16 / type_bytes(type)) == 0; }

// Calls f with XFC_F16, XFC_BF16 or XFC_F32 as a constant.
template <class Fn>
int by_type(int type, Fn&& f) {
  if (type == XFC_F32) return f(std::integral_constant<int, XFC_F32>{});
  if (type == XFC_BF16) return f(std::integral_constant<int, XFC_BF16>{});
  return f(std::integral_constant<int, XFC_F16>{});
}

// A launch has fewer than 2^32 threads: matrices go in ranges of units, selections in ranges of rows.
constexpr int64_t MX_GRID = ((int64_t)1 << 24) - 1, SELECT_ROWS = (int64_t)1 << 21;

int check_mx(const void* W, int type, int64_t ldw, int64_t L, int64_t d, const void* codes, const void* scales, bool& empty) {
  empty = false;
  if (!dims_ok(L) || !dims_ok(d) || !type_ok(type)) return XFC_ERR_INVALID;
  if (L == 0) { empty = true; return XFC_OK; }
  if (d == 0 || !W || !codes || !scales) return XFC_ERR_INVALID;
  if (d % 8 || !rows_ok(W, type, ldw) || !aligned16(codes) || !aligned16(scales)) return XFC_ERR_ALIGN;
  if (ldw < d) return XFC_ERR_SHAPE;
  if (mx_steps(d) > MX_GRID) return XFC_ERR_LIMIT;
  return XFC_OK;
}

template <class Launch>
int by_units(const MxArgs& all, int type, Launch&& launch) {
  const int64_t units = MX_GRID / all.steps;
  for (int64_t l0 = 0; l0 < all.L; l0 += units * MX_UNIT) {
    MxArgs a = all;
    const int64_t u0 = l0 / MX_UNIT, bytes = l0 * a.ldw * type_bytes(type);
    a.W = a.W ? reinterpret_cast<const char*>(a.W) + bytes : nullptr;
    a.out = a.out ? reinterpret_cast<char*>(a.out) + bytes : nullptr;
    a.codes += u0 * mx_code_bytes(a.d);
    a.scales += u0 * mx_scale_bytes(a.d);
    a.L = all.L - l0 < units * MX_UNIT ? all.L - l0 : units * MX_UNIT;
    const int rc = launch(dim3((unsigned)(ceil_div(a.L, MX_UNIT) * (int64_t)a.steps)), a);
    if (rc) return rc;
  }
  return XFC_OK;
}

// How a product is cut.  Rows: tiles of 16, 32, 64 or 128, as many as the batch fills and the LDS holds.  Label units: dealt to the waves
// of every workgroup of a row tile.
struct MxPlan {
  int nt;              // tiles of 16 rows of a workgroup; 0: the width does not fit
  int tiles_m, slots;
  int64_t lds;
};
int64_t mx_lds_of(int nt, bool x8, int64_t d) {
  const int64_t frag = x8 ? MxRows<true>::FRAG : MxRows<false>::FRAG;
  return (int64_t)mx_steps(d) * (nt * frag + (nt + 3) / 4 * 256);
}
MxPlan mx_plan(int64_t rows, int64_t L, int64_t d, bool x8, int run, int cus) {
  MxPlan p = {};
  for (p.nt = 8; p.nt > 0; p.nt /= 2) {
    const int64_t room = p.nt >= 4 ? FULL_LDS : FULL_LDS / 2;
    if (mx_lds_of(p.nt, x8, d) <= room && (p.nt == 1 || rows > 8 * p.nt)) break;
  }
  if (p.nt == 0) {
    p.nt = 1;  // one workgroup to a CU
    if (mx_lds_of(1, x8, d) > FULL_LDS) { p.nt = 0; return p; }
  }
  p.lds = mx_lds_of(p.nt, x8, d);
  p.tiles_m = ceil_div(rows, 16 * p.nt);
  const int per_xcd = (p.nt >= 4 || 2 * p.lds > FULL_LDS ? 1 : 2) * (cus / 8 > 0 ? cus / 8 : 1);
  const int most = ceil_div(ceil_div(L, MX_UNIT), 8 * MX_WAVES * run);  // workgroups of an XCD that have anything to do
  p.slots = per_xcd / p.tiles_m;
  if (p.slots > most) p.slots = most;
  if (p.slots < 1) p.slots = 1;
  return p;
}

// A kernel whose LDS goes by the call: the limit is raised to all there is.
template <auto Kernel, class A>
int launch_lds(dim3 g, dim3 b, int64_t lds, hipStream_t st, const A& args) {
  const hipError_t e = raise_lds_limit<Kernel>(FULL_LDS);
  if (e != hipSuccess) {
    fprintf(stderr, "xfc: cannot raise the dynamic LDS limit: %s\n", hipGetErrorString(e));
    return XFC_ERR_HIP;
  }
  hipLaunchKernelGGL(Kernel, g, b, (unsigned)lds, st, args);
  return check_launch();
}

template <bool X8, int OUT>
int launch_product(const MxPlan& p, const MxProductArgs& a, hipStream_t st) {
  const dim3 g((unsigned)(8 * p.slots * p.tiles_m)), b(64 * MX_WAVES);
  switch (p.nt) {
    case 1: return launch_lds<mx4_product_kernel<1, X8, OUT>>(g, b, p.lds, st, a);
    case 2: return launch_lds<mx4_product_kernel<2, X8, OUT>>(g, b, p.lds, st, a);
    case 4: return launch_lds<mx4_product_kernel<4, X8, OUT>>(g, b, p.lds, st, a);
    default: return launch_lds<mx4_product_kernel<8, X8, OUT>>(g, b, p.lds, st, a);
  }
}
int launch_product(int out, bool x8, const MxPlan& p, const MxProductArgs& a, hipStream_t st) {
  if (x8) {
    if (out == MX_HALF_MAXIMA) return launch_product<true, MX_HALF_MAXIMA>(p, a, st);
    if (out == MX_LOGITS) return launch_product<true, MX_LOGITS>(p, a, st);
    if (out == MX_LOGITS_MAX) return launch_product<true, MX_LOGITS_MAX>(p, a, st);
    return launch_product<true, MX_MAXIMA>(p, a, st);
  }
  if (out == MX_HALF_MAXIMA) return launch_product<false, MX_HALF_MAXIMA>(p, a, st);
  if (out == MX_LOGITS) return launch_product<false, MX_LOGITS>(p, a, st);
  if (out == MX_LOGITS_MAX) return launch_product<false, MX_LOGITS_MAX>(p, a, st);
  return launch_product<false, MX_MAXIMA>(p, a, st);
}

// Maxima by mx4_wide_kernel: rows that fill its tiles as well as those of 128, and units enough to a workgroup to make up for its rows' quantisation.
// (Time of top-5 with mx4_product_kernel over that with it.  Units to a workgroup 16: 400 rows x 262,144 labels x 768 0.95, 512 1.01; 18: 400 x 300,001 x 512 1.00, x 384 1.01; 32:
// 512 x 524,288 x 768 1.04, 1000 x 262,144 1.03; 80: 512 x 1,310,720 x 768 1.11, x 256 1.09; 160 and more 1.12 to 1.39.  Rows that fill fewer tiles of 128: 768 x 700,001 x 768
// 0.98, 640 0.88.)
bool mx_wide(int64_t rows, int64_t units, int steps, int cus) {
  const int64_t tiles = ceil_div(rows, MX_WIDE_ROWS);
  return steps >= 2 && steps <= 6 && round_up(rows, MX_WIDE_ROWS) == round_up(rows, 128) && units * tiles >= (int64_t)20 * cus;
}
template <int STEPS, int OUT>
int launch_wide(const MxProductArgs& args, int cus, hipStream_t st) {
  MxProductArgs a = args;
  const int per_xcd = cus / 8 > 0 ? cus / 8 : 1, most = ceil_div(ceil_div(a.units, MxSection<STEPS>::UNITS), 8);
  a.tiles_m = ceil_div(a.M, MX_WIDE_ROWS);
  a.slots = per_xcd / a.tiles_m;
  if (a.slots > most) a.slots = most;
  if (a.slots < 1) a.slots = 1;
  return launch_lds<mx4_wide_kernel<STEPS, OUT>>(dim3((unsigned)(8 * a.slots * a.tiles_m)), dim3(64 * MX_WAVES), MxSection<STEPS>::SLOTS * MxSection<STEPS>::BYTES, st, a);
}
template <int OUT>
int launch_wide(const MxProductArgs& a, int cus, hipStream_t st) {
  switch (a.steps) {
    case 2: return launch_wide<2, OUT>(a, cus, st);
    case 3: return launch_wide<3, OUT>(a, cus, st);
    case 4: return launch_wide<4, OUT>(a, cus, st);
    case 5: return launch_wide<5, OUT>(a, cus, st);
    default: return launch_wide<6, OUT>(a, cus, st);
  }
}

// Rows of one launch: the row tiles of an XCD's workgroups.
constexpr int64_t MX_ROWS = 2048;

// All rows of a product, in as many launches as it takes.
int mx_product(int out, bool x8, const void* X, int type, int64_t ldx, const void* codes, const void* scales, half_t* logits, int64_t ldo,
               half_t* hmax, float* bmax, int64_t ldb, int64_t B, int64_t L, int64_t d, int run, bool fine, hipStream_t st) {
  for (int64_t r0 = 0; r0 < B; r0 += MX_ROWS) {
    const int64_t rows = B - r0 < MX_ROWS ? B - r0 : MX_ROWS;
    const MxPlan p = mx_plan(rows, L, d, x8, run, num_cus());
    if (p.nt == 0) return XFC_ERR_LIMIT;
    MxProductArgs a = {};
    a.X = reinterpret_cast<const char*>(X) + r0 * ldx * type_bytes(type); a.type = type; a.ldx = ldx;
    a.codes = (const uint8_t*)codes; a.scales = (const uint8_t*)scales;
    a.out = logits ? logits + r0 * ldo : nullptr; a.ldo = ldo;
    a.hmax = hmax ? hmax + r0 * ldb : nullptr; a.bmax = bmax ? bmax + r0 * ldb : nullptr; a.ldb = ldb;
    a.M = (int)rows; a.N = (int)L; a.K = (int)d;
    a.units = ceil_div(L, MX_UNIT); a.blocks = mx_blocks(d); a.steps = mx_steps(d);
    a.tiles_m = p.tiles_m; a.slots = p.slots; a.run = run; a.fine = fine;
    if (!x8 && !fine && (out == MX_MAXIMA || out == MX_HALF_MAXIMA) && mx_wide(rows, a.units, a.steps, num_cus())) {
      const int rc = out == MX_MAXIMA ? launch_wide<MX_MAXIMA>(a, num_cus(), st) : launch_wide<MX_HALF_MAXIMA>(a, num_cus(), st);
      if (rc) return rc;
      continue;
    }
    const int rc = launch_product(out, x8, p, a, st);
    if (rc) return rc;
  }
  return XFC_OK;
}

int check_product(const void* X, int type, int64_t ldx, const void* codes, const void* scales, int64_t B, int64_t L, int64_t d, int bits) {
  if (!dims_ok(B) || !dims_ok(L) || !dims_ok(d) || !type_ok(type) || (bits != 4 && bits != 8)) return XFC_ERR_INVALID;
  if (B == 0 || L == 0) return XFC_OK;
  if (!X || !codes || !scales || d <= 0) return XFC_ERR_INVALID;
  if (d % 8 || !rows_ok(X, type, ldx) || !aligned16(codes) || !aligned16(scales)) return XFC_ERR_ALIGN;
  if (ldx < d) return XFC_ERR_SHAPE;
  if (mx_lds_of(1, bits == 8, d) > FULL_LDS || L > TOPK_RANGE_MAX) return XFC_ERR_LIMIT;
  return XFC_OK;
}

// Maxima of a row, as floats: whole runs of units, whole pieces of 16 bytes.  K <= 8: where they are few a float for each half of a unit, from
// which fewer labels' scores have to be formed again, else for each unit (top-5 of 64 rows x 131,072 x 768 28 us by halves, 32 by units, of
// 1024 88 and 96; 512 x 320,001 x 384 and more: no difference, and twice the room).  K > 8: two halves in a float's place.
constexpr int64_t MX_FINE = (int64_t)1 << 27;
bool mx_fine(int64_t B, int64_t L, int64_t K) { return K <= TOPK_MAX && (B <= 32 || B * L <= MX_FINE); }
int64_t mx_maxima(int64_t B, int64_t L, int64_t K) {
  const int64_t units = ceil_div(L, MX_UNIT);
  return round_up(mx_fine(B, L, K) ? 2 * units : units, 4);
}
// Beside logits, halves; rows of whole 16-byte pieces, which select_rows reads.
int64_t mx_half_maxima(int64_t L) { return round_up(2 * (int64_t)ceil_div(L, MX_UNIT), 8); }

// What mx4_select_kernel takes at most: its own, and the row's numbers at 16,384 dims (8 bits: 9,088).
constexpr int MX_SELECT_LDS = 96 * 1024;
static_assert(sizeof(MxSelectLds) + 128 * MxScores<false>::STEP_BYTES <= MX_SELECT_LDS && sizeof(MxSelectLds) + 71 * MxScores<true>::STEP_BYTES <= MX_SELECT_LDS, "LDS budget");

}  // namespace

int xfc::init_labels() {
  hipError_t e = hipSuccess;
  auto keep = [&](hipError_t r) { if (e == hipSuccess) e = r; };
  auto products = [&](auto x8, auto out) {
    constexpr bool X8 = decltype(x8)::value;
    constexpr int OUT = decltype(out)::value;
    keep(raise_lds_limit<mx4_product_kernel<1, X8, OUT>>(FULL_LDS));
    keep(raise_lds_limit<mx4_product_kernel<2, X8, OUT>>(FULL_LDS));
    keep(raise_lds_limit<mx4_product_kernel<4, X8, OUT>>(FULL_LDS));
    keep(raise_lds_limit<mx4_product_kernel<8, X8, OUT>>(FULL_LDS));
  };
  auto both = [&](auto out) { products(std::true_type{}, out); products(std::false_type{}, out); };
  both(std::integral_constant<int, MX_LOGITS>{});
  both(std::integral_constant<int, MX_LOGITS_MAX>{});
  both(std::integral_constant<int, MX_MAXIMA>{});
  both(std::integral_constant<int, MX_HALF_MAXIMA>{});
  auto wide = [&](auto out) {
    constexpr int OUT = decltype(out)::value;
    keep(raise_lds_limit<mx4_wide_kernel<2, OUT>>(FULL_LDS));
    keep(raise_lds_limit<mx4_wide_kernel<3, OUT>>(FULL_LDS));
    keep(raise_lds_limit<mx4_wide_kernel<4, OUT>>(FULL_LDS));
    keep(raise_lds_limit<mx4_wide_kernel<5, OUT>>(FULL_LDS));
    keep(raise_lds_limit<mx4_wide_kernel<6, OUT>>(FULL_LDS));
  };
  wide(std::integral_constant<int, MX_MAXIMA>{});
  wide(std::integral_constant<int, MX_HALF_MAXIMA>{});
  keep(raise_lds_limit<mx4_select_kernel<true, 512>>(MX_SELECT_LDS));
  keep(raise_lds_limit<mx4_select_kernel<true, 1024>>(MX_SELECT_LDS));
  keep(raise_lds_limit<mx4_select_kernel<false, 512>>(MX_SELECT_LDS));
  keep(raise_lds_limit<mx4_select_kernel<false, 1024>>(MX_SELECT_LDS));
  return e == hipSuccess ? XFC_OK : XFC_ERR_HIP;
}

extern "C" {

size_t xfc_mx4_code_bytes(int64_t L, int64_t d) {
  if (!dims_ok(L) || !dims_ok(d)) return 0;
  return (size_t)ceil_div(L, MX_UNIT) * (size_t)mx_code_bytes(d);
}
size_t xfc_mx4_scale_bytes(int64_t L, int64_t d) {
  if (!dims_ok(L) || !dims_ok(d)) return 0;
  return (size_t)ceil_div(L, MX_UNIT) * (size_t)mx_scale_bytes(d);
}

int xfc_mx4_quantize(const void* W, int type, int64_t ldw, int64_t L, int64_t d, void* codes, void* scales, void* stream) {
  bool empty;
  const int rc = check_mx(W, type, ldw, L, d, codes, scales, empty);
  if (rc || empty) return rc;
  const MxArgs a = {W, nullptr, ldw, (uint8_t*)codes, (uint8_t*)scales, L, (int)d, mx_blocks(d), mx_steps(d)};
  return by_type(type, [&](auto t) {
    return by_units(a, type, [&](dim3 g, const MxArgs& part) {
      return launch_k<mx4_quantize_kernel<decltype(t)::value>>(g, dim3(256), 0, reinterpret_cast<hipStream_t>(stream), part);
    });
  });
}

int xfc_mx4_dequantize(const void* codes, const void* scales, int64_t L, int64_t d, void* W, int type, int64_t ldw, void* stream) {
  bool empty;
  const int rc = check_mx(W, type, ldw, L, d, codes, scales, empty);
  if (rc || empty) return rc;
  const MxArgs a = {nullptr, W, ldw, (uint8_t*)const_cast<void*>(codes), (uint8_t*)const_cast<void*>(scales), L, (int)d, mx_blocks(d), mx_steps(d)};
  return by_type(type, [&](auto t) {
    return by_units(a, type, [&](dim3 g, const MxArgs& part) {
      return launch_k<mx4_dequantize_kernel<decltype(t)::value>>(g, dim3(256), 0, reinterpret_cast<hipStream_t>(stream), part);
    });
  });
}

int xfc_mx4_logits(const void* X, int type, int64_t ldx, const void* codes, const void* scales, void* out, int64_t ldo,
                   int64_t B, int64_t L, int64_t d, int embed_bits, void* stream) {
  const int rc = check_product(X, type, ldx, codes, scales, B, L, d, embed_bits);
  if (rc || B == 0 || L == 0) return rc;
  if (!out) return XFC_ERR_INVALID;
  if (ldo % 8 || !aligned16(out)) return XFC_ERR_ALIGN;
  if (ldo < L) return XFC_ERR_SHAPE;
  return mx_product(MX_LOGITS, embed_bits == 8, X, type, ldx, codes, scales, (half_t*)out, ldo, nullptr, nullptr, 0, B, L, d, 1, false,
                    reinterpret_cast<hipStream_t>(stream));
}

// K > 8: by logits, or by maxima of 32 labels and the K best blocks' scores formed again.  Writing logits takes 2 L bytes a row, fetching the blocks 17 d K;
// a row's blocks are one workgroup's, which few rows wait for.  (us by maxima / by logits.  512 rows x 768 dims: 131,072 labels, K = 10 67 / 74,
// 50 106 / 80; 320,001, K = 50 145 / 179, 100 189 / 180; 1,310,720, K = 200 481 / 650.  x 64: 131,072, K = 100 54 / 58, 200 78 / 66.  32 rows x 768:
// 131,072, K = 10 28 / 30; 1,310,720, K = 50 154 / 169, 100 174 / 171.  1 row x 1,310,720 x 768, K = 10 130 / 109.)
static bool mx_by_maxima(int64_t B, int64_t L, int64_t d, int64_t K) {
  return K > TOPK_MAX && K <= MX_SELECT_K && B >= 32 && L >= (B < 128 ? 2 : 1) * K * (1000 + 5 * d);
}
// By logits: those of this many rows, and the maxima of their blocks
static size_t mx_logit_rows_bytes(int64_t rows, int64_t L, int64_t K) {
  const size_t logits = (size_t)rows * (size_t)round_up(L, MX_UNIT) * 2;
  return (size_t)round_up((int64_t)logits, 16) + (select_takes_maxima(K, ceil_div(L, LOGIT_BLOCK)) ? (size_t)rows * (size_t)mx_half_maxima(L) * 2 : 0);
}

// Rows whose logits a call asks for room for: all where they are 2 GiB or 512 rows at most, else even turns of that.  (In two turns / all at once, 768 dims, K = 300:
// 1024 rows x 1,310,720 labels 1,336 / 1,402 us, 1536 2,144 / 2,513, 1024 x 2.8 M 2,715 / 2,949 and 2.8 / 5.9 GB, 600 x 2.8 M 1,760 / 1,755.  Of 768 and 256 rows
// the first takes 1,426.)
static int64_t mx_turn_rows(int64_t B, int64_t L, int64_t K) {
  const int64_t fit = (int64_t)(((size_t)2 << 30) / mx_logit_rows_bytes(256, L, K)) * 256, most = fit > 512 ? fit : 512;
  const int64_t turns = ceil_div(B, most);
  return turns == 1 ? B : round_up(ceil_div(B, turns), 256);
}

size_t xfc_mx4_topk_workspace_bytes(int64_t B, int64_t L, int64_t d, int64_t K) {
  if (!dims_ok(B) || !dims_ok(L) || !dims_ok(d) || K < 1 || K > SEL_MAX_K || B == 0 || L == 0) return 0;
  if (K <= TOPK_MAX || mx_by_maxima(B, L, d, K)) return (size_t)B * (size_t)mx_maxima(B, L, K) * 4;
  return mx_logit_rows_bytes(mx_turn_rows(B, L, K), L, K);
}

int xfc_mx4_topk(const void* X, int type, int64_t ldx, const void* codes, const void* scales, int64_t B, int64_t L, int64_t d,
                 int64_t numy, int K, int embed_bits, float* values, int64_t* indices, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_product(X, type, ldx, codes, scales, B, L, d, embed_bits);
  if (rc || B == 0) return rc;
  if (K < 1 || K > SEL_MAX_K || L < K || numy < 1 || !values || !indices) return XFC_ERR_INVALID;
  const bool maxima = K <= TOPK_MAX || mx_by_maxima(B, L, d, K);
  const size_t turn = mx_logit_rows_bytes(256, L, K), all = mx_logit_rows_bytes(B, L, K);  // 256 rows' logits, all rows'
  if (!workspace || workspace_bytes < (maxima ? xfc_mx4_topk_workspace_bytes(B, L, d, K) : B <= 256 ? all : turn)) return XFC_ERR_WORKSPACE;
  if (!aligned16(workspace)) return XFC_ERR_ALIGN;
  const bool x8 = embed_bits == 8;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (!maxima) {
    const int64_t ldb = mx_half_maxima(L);
    int64_t block = B;
    if (workspace_bytes < all) block = (int64_t)(workspace_bytes / turn) * 256;
    if (block > SELECT_ROWS) block = SELECT_ROWS;
    const int64_t ldl = round_up(L, MX_UNIT);
    for (int64_t r0 = 0; r0 < B; r0 += block) {
      const int64_t rows = B - r0 < block ? B - r0 : block;
      half_t* const logits = (half_t*)workspace;
      half_t* const hmax = select_takes_maxima(K, ceil_div(L, LOGIT_BLOCK)) ? logits + rows * ldl : nullptr;
      rc = mx_product(MX_LOGITS_MAX, x8, reinterpret_cast<const char*>(X) + r0 * ldx * type_bytes(type), type, ldx, codes, scales,
                      logits, ldl, hmax, nullptr, ldb, rows, L, d, 1, false, st);
      if (rc) return rc;
      rc = select_rows(logits, ldl, (int)rows, (int)L, numy, K, hmax, ldb, values + r0 * K, indices + r0 * K, st);
      if (rc) return rc;
    }
    return XFC_OK;
  }
  float* const bmax = (float*)workspace;
  const int64_t ldb = mx_maxima(B, L, K);
  const bool fine = mx_fine(B, L, K);
  const int block = K > TOPK_MAX ? MX_SELECT_BLOCK : fine ? MX_UNIT / 2 : MX_UNIT;
  rc = mx_product(K > TOPK_MAX ? MX_HALF_MAXIMA : MX_MAXIMA, x8, X, type, ldx, codes, scales, nullptr, 0, nullptr, bmax, ldb, B, L, d,
                  !fine && L >= (1 << 20) ? 4 : 1, fine, st);
  if (rc) return rc;
  auto pick = [&](auto s, int64_t r0, int64_t rows) {
    using S = decltype(s);
    PickArgs k = {};
    k.bmax = bmax + r0 * ldb; k.ldb = ldb; k.n_blocks = ceil_div(L, block); k.N = (int)L; k.K = (int)d; k.topk = K;
    k.begin = k.end = 1; k.numy = numy; k.out_v = values + r0 * K; k.out_i = indices + r0 * K;
    if (K > TOPK_MAX) {
      auto select = [&](auto threads) {
        constexpr int T = decltype(threads)::value;
        constexpr auto kernel = mx4_select_kernel<std::is_same_v<S, MxScores<true>>, T>;
        if (raise_lds_limit<kernel>(MX_SELECT_LDS) != hipSuccess) return (int)XFC_ERR_HIP;
        hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(T), (unsigned)(S::lds(d) + sizeof(MxSelectLds)), st, k, s);
        return check_launch();
      };
      if (rows > num_cus()) return select(std::integral_constant<int, 512>{});
      return select(std::integral_constant<int, 1024>{});
    }
    if (fine) hipLaunchKernelGGL((topk_pick_kernel<MX_UNIT / 2, S>), dim3((unsigned)rows), dim3(512), (unsigned)S::lds(d), st, k, s);  // 11 KB at most
    else hipLaunchKernelGGL((topk_pick_kernel<MX_UNIT, S>), dim3((unsigned)rows), dim3(512), (unsigned)S::lds(d), st, k, s);
    return check_launch();
  };
  for (int64_t r0 = 0; r0 < B && !rc; r0 += SELECT_ROWS) {
    const int64_t rows = B - r0 < SELECT_ROWS ? B - r0 : SELECT_ROWS;
    const void* const x = reinterpret_cast<const char*>(X) + r0 * ldx * type_bytes(type);
    rc = x8 ? pick(MxScores<true>{x, type, ldx, (const uint8_t*)codes, (const uint8_t*)scales}, r0, rows)
            : pick(MxScores<false>{x, type, ldx, (const uint8_t*)codes, (const uint8_t*)scales}, r0, rows);
  }
  return rc;
}

// Pairs of a wave: as many as a lane each holds, fewer where they would leave the chip's waves without any.  (65,536 pairs of 1024 rows x 768,
// both kernels: 72 us in 8192 chunks, whose parts of rows have to be added up, 59 in 4096, 50 in 2048.)
static int pref_chunk(int64_t P) {
  int chunk = 64;
  while (chunk > 4 && ceil_div(P, chunk) < 2048) chunk /= 2;
  return chunk;
}
size_t xfc_preference_workspace_bytes(int64_t B, int64_t P, int64_t d) {
  if (!dims_ok(B) || !dims_ok(P) || !dims_ok(d)) return 16;
  const int64_t chunks = ceil_div(P, pref_chunk(P));
  return (size_t)round_up(chunks * 8, 16) + (size_t)round_up(P * 4, 16) + (size_t)(chunks * 2 * d * 4) + 16;
}

int xfc_preference(const void* X, int type, int64_t ldx, const void* W, int64_t ldw, const void* scales, int64_t L, int64_t d,
                   const int32_t* rowptr, const int32_t* chosen, const int32_t* rejected, const float* reference, const float* weight,
                   int64_t B, int64_t P, float beta, float smoothing, float scale, float* loss, float* margin,
                   void* dX, int dx_type, int64_t lddx, void* G, int64_t ldg, void* workspace, size_t workspace_bytes, void* stream) {
  if (!dims_ok(B) || !dims_ok(L) || !dims_ok(d) || !dims_ok(P) || !type_ok(type) || (dX && !type_ok(dx_type))) return XFC_ERR_INVALID;
  if (!loss || (B > 0 && (!X || !W || !rowptr)) || (P > 0 && (!chosen || !rejected)) || d <= 0 || L <= 0 || B > 0x3ffffe) return XFC_ERR_INVALID;  // (threads of a launch)
  if (!(fabsf(beta) <= 3.4e38f) || !(smoothing >= 0.f && smoothing <= 1.f)) return XFC_ERR_INVALID;
  if (B > 0 && (d % 8 || !rows_ok(X, type, ldx) || !aligned16(W) || (scales ? !aligned16(scales) : ldw % 8 != 0) ||
                (dX && !rows_ok(dX, dx_type, lddx)))) return XFC_ERR_ALIGN;
  if (B > 0 && (ldx < d || (!scales && ldw < d) || (dX && lddx < d) || (G && ldg < L))) return XFC_ERR_SHAPE;
  if (d > 4096 || P > (1 << 30)) return XFC_ERR_LIMIT;
  if (!workspace || workspace_bytes < xfc_preference_workspace_bytes(B, P, d)) return XFC_ERR_WORKSPACE;
  if (!aligned16(workspace)) return XFC_ERR_ALIGN;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  PrefArgs a = {};
  a.X = X; a.type = type; a.ldx = ldx; a.W = W; a.ldw = ldw; a.scales = (const uint8_t*)scales; a.L = L; a.d = (int)d;
  a.rowptr = rowptr; a.chosen = chosen; a.rejected = rejected; a.reference = reference; a.weight = weight;
  a.B = (int)B; a.P = (int)P; a.chunk = pref_chunk(P); a.chunks = ceil_div(P, a.chunk);
  a.beta = beta; a.smoothing = smoothing; a.scale = scale; a.margin = margin;
  a.dX = dX; a.dx_type = dx_type; a.lddx = lddx; a.G = (half_t*)G; a.ldg = ldg; a.loss = loss;
  a.part_loss = (double*)workspace;
  a.slope = (float*)((char*)workspace + round_up((int64_t)a.chunks * 8, 16));
  a.part_dx = (float*)((char*)a.slope + round_up(P * 4, 16));
  if (a.chunks > 0) {
    const dim3 g((unsigned)ceil_div(a.chunks, PREF_WAVES)), b(64 * PREF_WAVES);
    auto launch = [&](auto c) {
      constexpr int C = decltype(c)::value;
      return scales ? launch_k<preference_kernel<C, true>>(g, b, 0, st, a) : launch_k<preference_kernel<C, false>>(g, b, 0, st, a);
    };
    const int rc = d <= 512 ? launch(std::integral_constant<int, 1>{}) : d <= 1024 ? launch(std::integral_constant<int, 2>{})
                 : d <= 2048 ? launch(std::integral_constant<int, 4>{}) : launch(std::integral_constant<int, 8>{});
    if (rc) return rc;
  }
  // Behind them: a workgroup for each row, several where rows are few, as they may be long.
  const int64_t rows = G || dX ? B : 0, pieces = d / 8;
  const int threads = G ? PREF_FINISH : PREF_FINISH / 2;
  a.slices = 1;
  if (dX) {
    const int64_t want = rows > 0 ? ceil_div(512, rows) : 1, most = ceil_div(pieces, 8), least = ceil_div(pieces, threads);
    a.slices = (int)(want > most ? most : want < least ? least : want);
  }
  a.width = ceil_div(pieces, a.slices);
  return launch_k<preference_finish_kernel>(dim3((unsigned)(rows * a.slices + 1)), dim3(threads), 0, st, a);
}

}  // extern "C"

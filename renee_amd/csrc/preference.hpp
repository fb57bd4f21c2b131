// The preference loss over (row, chosen label, rejected label) pairs, and its gradients.
//
//   m = x_b . (w_c - w_r) - reference          (log pi(c) - log pi(r) of a softmax over the labels: its normaliser cancels)
//   loss = sum a [-(1 - e) log sigmoid(beta m) - e log sigmoid(-beta m)]
//   slope = a beta (sigmoid(beta m) - (1 - e))  = d loss / d m
//   dX_b = scale sum slope (w_c - w_r);         or G[b][c] += slope, G[b][r] -= slope, from which dX and dW follow
//
// Bound by fetching two rows of labels per pair from anywhere.  A wave takes pairs of one row, four at a time, whole rows of
// weights in its registers; the difference that makes the margin makes the gradient too, so rows are fetched once.  Everything is summed
// in fp32 in a fixed order (the loss in double): a row's pairs by waves in turn, waves by number, splits by number.
#pragma once
#include "mx4.hpp"

namespace xfc {

constexpr int PREF_WAVES = 4;
constexpr int pref_pairs(int pieces) { return pieces <= 2 ? 4 : 8 / pieces; }  // as many as the registers hold
constexpr int PREF_TILE = 512;  // pairs of a row whose entries of G are joined at a time

struct PrefArgs {
  const void* X; int type; int64_t ldx;
  const void* W; int64_t ldw; const uint8_t* scales;  // scales: W holds MX4 codes
  int64_t L; int d;
  const int32_t* rowptr; const int32_t* chosen; const int32_t* rejected;
  const float* reference; const float* weight;        // may be null: 0, 1
  int B, P, splits;
  float beta, smoothing, scale;
  float* margin;                                       // may be null
  void* dX; int dx_type; int64_t lddx;                 // may be null
  half_t* G; int64_t ldg;                              // may be null
  float* loss;
  float* slope; double* part_loss; float* part_dx;     // workspace: P; B x splits; B x splits x d with several splits and dX
};

// Pairs of a row, whatever rowptr holds.
__device__ __forceinline__ void pref_range(const PrefArgs& a, int row, int& begin, int& end) {
  begin = a.rowptr[row];
  end = a.rowptr[row + 1];
  begin = begin < 0 ? 0 : begin;
  end = end > a.P ? a.P : end;
  end = end < begin ? begin : end;
}

// Eight dims from k on of a label.
template <bool MX>
__device__ __forceinline__ Float8 pref_load(const PrefArgs& a, int label, int k) {
  if constexpr (MX) {
    const int blocks = mx_blocks(a.d), within = label % MX_UNIT, tile = mx_tile(within), row = mx_row(within), block = k / MX_BLOCK;
    const uint8_t* const c = reinterpret_cast<const uint8_t*>(a.W) + label / MX_UNIT * mx_code_bytes(a.d);
    const uint8_t* const s = a.scales + label / MX_UNIT * mx_scale_bytes(a.d);
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(c + mx_code_at(tile, row, block, blocks) + (k % MX_BLOCK) / 2);
    return from_fp4(codes, scale_value(s[mx_scale_at(tile, row, block)]));
  } else {
    return load8<XFC_F16>(reinterpret_cast<const half_t*>(a.W) + (int64_t)label * a.ldw + k);
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// C pieces of 512 dims.
template <int C, bool MX>
__global__ void __launch_bounds__(64 * PREF_WAVES) preference_kernel(PrefArgs a) {
  constexpr int PAIRS = pref_pairs(C);
  __shared__ float sums[PREF_WAVES][C * 512];
  __shared__ double losses[PREF_WAVES];
  const int row = blockIdx.x, split = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int begin, end;
  pref_range(a, row, begin, end);
  const int per = (end - begin + a.splits - 1) / a.splits;
  const int first = begin + split * per, last = first + per < end ? first + per : end;

  Float8 x[C], acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int k = 512 * c + 8 * lane;
    x[c] = Float8{};
    acc[c] = Float8{};
    if (k < a.d) x[c] = load8_of(a.X, a.type, (int64_t)row * a.ldx + k);
  }
  double loss = 0.0;
  // 64 pairs at a time: their lists by one load each, every fourth of them this wave's
  for (int p0 = first; p0 < last; p0 += 64 * PREF_WAVES) {
    const int p = p0 + lane * PREF_WAVES + wave;
    const bool in = p < last;
    const int cl = in ? a.chosen[p] : -1, rl = in ? a.rejected[p] : -1;
    const float ref = in && a.reference ? a.reference[p] : 0.f, wt = in && a.weight ? a.weight[p] : 1.f;
    unsigned long long left = __ballot(cl >= 0 && cl < a.L && rl >= 0 && rl < a.L && wt != 0.f);
    float my_margin = 0.f, my_slope = 0.f;
    while (left) {
      int at[PAIRS], n = 0;
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        at[j] = left ? __builtin_ctzll(left) : at[j > 0 ? j - 1 : 0];
        n += left != 0;
        left &= left - 1;
      }
      Float8 diff[PAIRS][C];
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        const int lc = __builtin_amdgcn_readlane(cl, at[j]), lr = __builtin_amdgcn_readlane(rl, at[j]);
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int k = 512 * c + 8 * lane;  // (no branches: all of the pairs' loads are on their way together)
          const Float8 u = pref_load<MX>(a, lc, k < a.d ? k : 0), v = pref_load<MX>(a, lr, k < a.d ? k : 0);
#pragma unroll
          for (int e = 0; e < 8; ++e) diff[j][c].v[e] = k < a.d ? u.v[e] - v.v[e] : 0.f;
        }
      }
      float z[PAIRS];
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        z[j] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e) z[j] = fmaf(x[c].v[e], diff[j][c].v[e], z[j]);
        z[j] = wave_sum(z[j]);
      }
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        if (j < n) {
          const float m = z[j] - __shfl(ref, at[j], 64), t = a.beta * m, w = __shfl(wt, at[j], 64);
          const float small = expf(-fabsf(t)), sig = t >= 0.f ? 1.f / (1.f + small) : small / (1.f + small);
          // (a positive margin's slope is -(1 - sigmoid) + e: formed so, what is left at sigmoid near 1 keeps its bits)
          const float g = w * a.beta * (t >= 0.f ? a.smoothing - small / (1.f + small) : sig - (1.f - a.smoothing));
          loss += (double)(w * (log1pf(small) + (t >= 0.f ? a.smoothing * t : -(1.f - a.smoothing) * t)));
          if (lane == at[j]) { my_margin = m; my_slope = g; }
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[c].v[e] = fmaf(g, diff[j][c].v[e], acc[c].v[e]);
        }
      }
    }
    if (in) {
      if (a.margin) a.margin[p] = my_margin;
      if (a.G) a.slope[p] = my_slope;
    }
  }
  if (a.margin && split == 0) {  // pairs that no row has
    if (row == 0)
      for (int p = tid; p < a.P && p < begin; p += 64 * PREF_WAVES) a.margin[p] = 0.f;
    if (row == a.B - 1)
      for (int p = end + tid; p < a.P; p += 64 * PREF_WAVES) a.margin[p] = 0.f;
  }
  if (lane == 0) losses[wave] = loss;
  if (a.dX) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<float4v*>(&sums[wave][512 * c + 8 * lane + e]) = float4v{acc[c].v[e], acc[c].v[e + 1], acc[c].v[e + 2], acc[c].v[e + 3]};
  }
  __syncthreads();
  if (tid == 0) {
    double t = 0.0;
    for (int w = 0; w < PREF_WAVES; ++w) t += losses[w];
    a.part_loss[(int64_t)row * a.splits + split] = t;
  }
  if (a.dX) {
    for (int k = tid; k < a.d; k += 64 * PREF_WAVES) {
      float t = 0.f;
      for (int w = 0; w < PREF_WAVES; ++w) t += sums[w][k];
      if (a.splits > 1) {
        a.part_dx[((int64_t)row * a.splits + split) * a.d + k] = t;
      } else {
        t *= a.scale;
        const int64_t to = (int64_t)row * a.lddx + k;
        if (a.dx_type == XFC_F32) reinterpret_cast<float*>(a.dX)[to] = t;
        else if (a.dx_type == XFC_BF16) reinterpret_cast<__bf16*>(a.dX)[to] = (__bf16)t;
        else reinterpret_cast<half_t*>(a.dX)[to] = (half_t)t;
      }
    }
  }
}

// What is left after the pairs, a workgroup per row: the sum of the splits' dX, and G.  A row's entries of G, two a pair, are
// joined PREF_TILE pairs at a time: each is compared with all others, the first of a label adds up all of them in their order and
// rounds G once.  Workgroup B sums the loss.
__global__ void __launch_bounds__(256) preference_finish_kernel(PrefArgs a) {
  __shared__ int32_t label[2 * PREF_TILE];
  __shared__ float slope[2 * PREF_TILE];
  __shared__ double sums[4];
  const int row = blockIdx.x, tid = threadIdx.x;
  if (row == (int)gridDim.x - 1) {
    double t = 0.0;
    for (int64_t i = tid; i < (int64_t)a.B * a.splits; i += 256) t += a.part_loss[i];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) t += __shfl_xor(t, off, 64);
    if ((tid & 63) == 0) sums[tid >> 6] = t;
    __syncthreads();
    if (tid == 0) *a.loss = (float)(((sums[0] + sums[1]) + sums[2]) + sums[3]);
    return;
  }
  if (a.dX && a.splits > 1) {
    for (int k = tid; k < a.d; k += 256) {
      float t = 0.f;
      for (int s = 0; s < a.splits; ++s) t += a.part_dx[((int64_t)row * a.splits + s) * a.d + k];
      t *= a.scale;
      const int64_t to = (int64_t)row * a.lddx + k;
      if (a.dx_type == XFC_F32) reinterpret_cast<float*>(a.dX)[to] = t;
      else if (a.dx_type == XFC_BF16) reinterpret_cast<__bf16*>(a.dX)[to] = (__bf16)t;
      else reinterpret_cast<half_t*>(a.dX)[to] = (half_t)t;
    }
  }
  if (!a.G) return;
  int begin, end;
  pref_range(a, row, begin, end);
  half_t* const g = a.G + (int64_t)row * a.ldg;
  for (int p0 = begin; p0 < end; p0 += PREF_TILE) {
    const int n = end - p0 < PREF_TILE ? end - p0 : PREF_TILE;
    __syncthreads();
    for (int e = tid; e < n; e += 256) {
      const int c = a.chosen[p0 + e], r = a.rejected[p0 + e];
      const bool ok = c >= 0 && c < a.L && r >= 0 && r < a.L && (!a.weight || a.weight[p0 + e] != 0.f);
      const float s = ok ? a.slope[p0 + e] : 0.f;
      label[2 * e] = ok ? c : -1;
      label[2 * e + 1] = ok ? r : -1;
      slope[2 * e] = s;
      slope[2 * e + 1] = -s;
    }
    __syncthreads();
    for (int e = tid; e < 2 * n; e += 256) {
      const int mine = label[e];
      float t = 0.f;
      bool owner = mine >= 0;
      for (int o = 0; o < 2 * n; ++o) {
        const bool same = label[o] == mine;
        owner = owner && !(same && o < e);
        t += same ? slope[o] : 0.f;
      }
      if (owner) g[mine] = (half_t)((float)g[mine] + t);
    }
  }
}

}  // namespace xfc

// The preference loss over (row, chosen label, rejected label) pairs, and its gradients.
//
//   m = x_b . (w_c - w_r) - reference          (log pi(c) - log pi(r) of a softmax over the labels: its normaliser cancels)
//   loss = sum a [-(1 - e) log sigmoid(beta m) - e log sigmoid(-beta m)]
//   slope = a beta (sigmoid(beta m) - (1 - e))  = d loss / d m
//   dX_b = scale sum slope (w_c - w_r);         or G[b][c] += slope, G[b][r] -= slope, from which dX and dW follow
//
// Bound by fetching two rows of labels per pair from anywhere.  A wave takes a chunk of consecutive pairs whatever rows they are of (rows have
// very unequal numbers of them), four at a time, whole rows of weights in its registers; the difference that makes the margin makes the
// gradient too, so rows are fetched once.  Where a row's pairs end the wave stores its dX, or, of a row that the chunk has only
// a part of, that part: preference_finish_kernel adds those up.  Everything is summed in fp32 in a fixed order (the loss in double): pairs in
// their order within a chunk, chunks in theirs.
//
// 65,536 pairs of 1024 rows over 1,310,720 fp16 labels x 768: 26 us and 5 behind them (201 MB of rows asked for, a half of which the caches have; 43 with the
// functions of a pair in all lanes and differences by conversions, which took as much of the vector units as the sums); 512 rows' pairs into G, 131,072
// labels: 9.4 and 5.8; 32 rows over MX4 labels: 9.5 and 5, the latency of a chunk's loads.
#pragma once
#include "mx4.hpp"

namespace xfc {

constexpr int PREF_WAVES = 4;
constexpr int pref_pairs(int pieces) { return pieces <= 2 ? 4 : 8 / pieces; }  // as many as the registers hold
constexpr int PREF_FINISH = 1024;  // threads with G, half of them without
constexpr int PREF_TILE = 512;  // pairs of a row whose entries of G are joined at a time
constexpr int PREF_COMPARED = 256;  // ... by comparing each with all others: 9 us, as long as sorting any number takes; 512 37

struct PrefArgs {
  const void* X; int type; int64_t ldx;
  const void* W; int64_t ldw; const uint8_t* scales;  // scales: W holds MX4 codes
  int64_t L; int d;
  const int32_t* rowptr; const int32_t* chosen; const int32_t* rejected;
  const float* reference; const float* weight;        // may be null: 0, 1
  int B, P;
  int chunk, chunks;                                   // pairs of a wave; waves
  int slices, width;                                   // workgroups of a row behind them; of so many pieces of eight dims
  float beta, smoothing, scale;
  float* margin;                                       // may be null
  void* dX; int dx_type; int64_t lddx;                 // may be null
  half_t* G; int64_t ldg;                              // may be null
  float* loss;
  float* slope; double* part_loss; float* part_dx;     // workspace: P; chunks; chunks x 2 x d, the parts of a chunk's first and last row
};

// Pairs of a row, whatever rowptr holds.
__device__ __forceinline__ void pref_range(const PrefArgs& a, int row, int& begin, int& end) {
  begin = a.rowptr[row];
  end = a.rowptr[row + 1];
  begin = begin < 0 ? 0 : begin;
  end = end > a.P ? a.P : end;
  end = end < begin ? begin : end;
}

// Eight dims from k on of a label in MX4.
__device__ __forceinline__ Float8 pref_load(const PrefArgs& a, int label, int k) {
  const int blocks = mx_blocks(a.d), within = label % MX_UNIT, tile = mx_tile(within), row = mx_row(within), block = k / MX_BLOCK;
  const uint8_t* const c = reinterpret_cast<const uint8_t*>(a.W) + label / MX_UNIT * mx_code_bytes(a.d);
  const uint8_t* const s = a.scales + label / MX_UNIT * mx_scale_bytes(a.d);
  const uint32_t codes = *reinterpret_cast<const uint32_t*>(c + mx_code_at(tile, row, block, blocks) + (k % MX_BLOCK) / 2);
  return from_fp4(codes, scale_value(s[mx_scale_at(tile, row, block)]));
}

// u - v of halves as a float, in one instruction where conversions would be two more.  (LO: the lower ones of two, else the upper ones.)
template <bool LO>
__device__ __forceinline__ float pref_minus(uint32_t u, uint32_t v) {
  float r;
  if constexpr (LO) asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel_hi:[1,0,1]" : "=v"(r) : "v"(u), "v"(v));
  else asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[1,0,1] op_sel_hi:[1,0,1]" : "=v"(r) : "v"(u), "v"(v));
  return r;
}
// Eight dims from k on of the difference of two labels.
template <bool MX>
__device__ __forceinline__ Float8 pref_difference(const PrefArgs& a, int chosen, int rejected, int k) {
  Float8 f;
  if constexpr (MX) {
    const Float8 u = pref_load(a, chosen, k), v = pref_load(a, rejected, k);
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = u.v[e] - v.v[e];
  } else {
    const half_t* const w = reinterpret_cast<const half_t*>(a.W) + k;
    const uint4v u = *reinterpret_cast<const uint4v*>(w + (int64_t)chosen * a.ldw), v = *reinterpret_cast<const uint4v*>(w + (int64_t)rejected * a.ldw);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f.v[2 * e] = pref_minus<true>(u[e], v[e]);
      f.v[2 * e + 1] = pref_minus<false>(u[e], v[e]);
    }
  }
  return f;
}

// The wave's sum, uniform: within rows of 16 lanes, then across them.
__device__ __forceinline__ float wave_sum(float v) {
  auto step = [&](auto ctrl, auto rows) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});  // row_shr:1, 2, 4, 8
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row_bcast:15, 31
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Eight neighbouring elements of a row of dX.
__device__ __forceinline__ void pref_store(const PrefArgs& a, int64_t at, const Float8& f) {
  if (a.dx_type == XFC_F32) store8<XFC_F32>(reinterpret_cast<float*>(a.dX) + at, f);
  else if (a.dx_type == XFC_BF16) store8<XFC_BF16>(reinterpret_cast<uint16_t*>(a.dX) + at, f);
  else store8<XFC_F16>(reinterpret_cast<half_t*>(a.dX) + at, f);
}

// C pieces of 512 dims.
template <int C, bool MX>
__global__ void __launch_bounds__(64 * PREF_WAVES) preference_kernel(PrefArgs a) {
  constexpr int PAIRS = pref_pairs(C);
  const int lane = threadIdx.x & 63, chunk = blockIdx.x * PREF_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (chunk >= a.chunks) return;
  const int p0 = chunk * a.chunk, p1 = p0 + a.chunk < a.P ? p0 + a.chunk : a.P;  // a.chunk <= 64
  // a pair for each lane
  const bool in = p0 + lane < p1;
  const int cl = in ? a.chosen[p0 + lane] : -1, rl = in ? a.rejected[p0 + lane] : -1;
  const float ref = in && a.reference ? a.reference[p0 + lane] : 0.f, wt = in && a.weight ? a.weight[p0 + lane] : 1.f;
  // The first row from `from` on that ends behind pair p (B: none), of 64 rows looked at at a time.
  auto search = [&](int from, int p) {
    for (int left = a.B - from; left > 0;) {
      const int step = (left + 63) / 64, mid = (lane + 1) * step - 1;
      const int past = __builtin_popcountll(__ballot(mid < left && a.rowptr[from + (mid < left ? mid : 0) + 1] <= p));
      from += past * step;
      left = left - past * step < step - 1 ? left - past * step : step - 1;
    }
    return __builtin_amdgcn_readfirstlane(from);
  };
  int row = search(0, p0);
  const unsigned long long usable = __ballot(cl >= 0 && cl < a.L && rl >= 0 && rl < a.L && wt != 0.f);
  float my_margin = 0.f, my_slope = 0.f;
  double loss = 0.0;
  for (int p = p0; p < p1 && row < a.B;) {
    int begin, end;
    pref_range(a, row, begin, end);
    begin = __builtin_amdgcn_readfirstlane(begin);
    end = __builtin_amdgcn_readfirstlane(end);
    if (begin >= p1) break;  // nor has any row from here on
    const int first = p > begin ? p : begin, last = end < p1 ? end : p1;  // of the row, in this chunk
    if (first >= last) {
      // None of this row's, and what lies before it is no row's.  The next row that has any is most often near; if not it is searched for: going through
      // the rows one after the other took 0.14 us for each.
      p = first;
      const int next = row + 1 + lane;
      const unsigned long long near = __ballot(next < a.B && a.rowptr[next + 1] > p);
      row = near ? row + 1 + __builtin_ctzll(near) : search(row + 1, p);
      continue;
    }
    unsigned long long left = usable & (~0ull << (first - p0)) & (~0ull >> (64 - (last - p0)));
    Float8 acc[C];
    Float8 x[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int k = 512 * c + 8 * lane;
      acc[c] = Float8{};
      x[c] = Float8{};
      if (k < a.d) x[c] = load8_of(a.X, a.type, (int64_t)row * a.ldx + k);
    }
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
          diff[j][c] = pref_difference<MX>(a, lc, lr, k < a.d ? k : 0);
        }
      }
      float z[PAIRS];
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        z[j] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float part = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) part = fmaf(x[c].v[e], diff[j][c].v[e], part);
          z[j] += 512 * c + 8 * lane < a.d ? part : 0.f;
        }
        z[j] = wave_sum(z[j]);
      }
      // The pairs' own lanes, all at once: these functions are as much work as a pair's sums.
      bool mine = false;
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        m = lane == at[j] ? z[j] : m;
        mine = mine || lane == at[j];
      }
      m -= ref;
      const float t = a.beta * m, small = expf(-fabsf(t)), rest = small / (1.f + small);  // rest: 1 - sigmoid(|t|)
      // (a positive margin's slope is -(1 - sigmoid) + e: formed so, what is left at sigmoid near 1 keeps its bits)
      const float g = wt * a.beta * (t >= 0.f ? a.smoothing - rest : rest - (1.f - a.smoothing));
      const float l = wt * (log1pf(small) + (t >= 0.f ? a.smoothing * t : -(1.f - a.smoothing) * t));
      if (mine) {
        my_margin = m;
        my_slope = g;
        loss += (double)l;
      }
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        if (j < n) {
          const float gj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(g), at[j]));
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[c].v[e] = fmaf(gj, diff[j][c].v[e], acc[c].v[e]);
        }
      }
    }
    if (a.dX) {
      const bool whole = begin >= p0 && end <= p1;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int k = 512 * c + 8 * lane;
        if (k >= a.d) continue;
        if (whole) {
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[c].v[e] *= a.scale;
          pref_store(a, (int64_t)row * a.lddx + k, acc[c]);
        } else {
          float* const to = a.part_dx + (2 * (int64_t)chunk + (begin >= p0 ? 1 : 0)) * a.d + k;
          store8<XFC_F32>(to, acc[c]);
        }
      }
    }
    p = last;
    ++row;
  }
  if (in) {
    if (a.margin) a.margin[p0 + lane] = my_margin;
    if (a.G) a.slope[p0 + lane] = my_slope;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) loss += __shfl_xor(loss, off, 64);
  if (lane == 0) a.part_loss[chunk] = loss;
}

// More entries of G: sorted by label, a thread each, within a wave by exchanges between lanes.  Sums over equal labels then double in reach step by step (a label that
// far away is the same only if all between are), and the last entry of a label has its sum.
__device__ __forceinline__ void pref_join_sorted(const int32_t* label, const float* slope, int entries, float* room, half_t* g) {
  static_assert(PREF_FINISH == 2 * PREF_TILE, "a thread for each entry");
  unsigned long long* const keys = reinterpret_cast<unsigned long long*>(room);
  uint32_t* const sorted = reinterpret_cast<uint32_t*>(keys + PREF_FINISH);
  float* const sums = reinterpret_cast<float*>(sorted + PREF_FINISH);  // two of them
  const int i = threadIdx.x;
  unsigned long long key = i < entries ? ((unsigned long long)(uint32_t)label[i] << 32) | (unsigned)i : ~0ull;  // no label: behind all others
  for (int k = 2; k <= PREF_FINISH; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      unsigned long long other;
      if (j < 64) {
        other = __shfl_xor(key, j, 64);
      } else {
        __syncthreads();
        keys[i] = key;
        __syncthreads();
        other = keys[i ^ j];
      }
      const bool lower = ((i & k) == 0) == ((i & j) == 0);  // of the two, the smaller one stays
      key = (other < key) == lower ? other : key;
    }
  const uint32_t mine = (uint32_t)(key >> 32);
  float t = (uint32_t)key < (uint32_t)entries ? slope[(uint32_t)key] : 0.f;
  sorted[i] = mine;
  int half = 0;
  for (int off = 1; off < PREF_FINISH; off <<= 1, half ^= PREF_FINISH) {
    sums[half + i] = t;
    __syncthreads();
    if (i >= off && sorted[i - off] == mine) t += sums[half + i - off];
  }
  if (mine < 0x80000000u && (i + 1 == PREF_FINISH || sorted[i + 1] != mine)) g[mine] = (half_t)((float)g[mine] + t);
}

// What is left after the pairs: dX of rows without pairs and of those that several chunks have a part of, and G.  A workgroup has `width` pieces of eight dims of a row: one
// thread for each adds up to four parts, more are dealt to all the threads there are and joined through the LDS, in an order that the arguments alone decide.  (8192 pairs
// of one row x 768, both kernels: 570 us with one thread for each piece and one workgroup for the row, 21.)
// A row's entries of G, two a pair, are joined PREF_TILE pairs at a time, and G is rounded once for each label.  Of few each is compared with all others, the first of a
// label adds up all of them; more are sorted.  (64 rows of 1024 pairs, both kernels: 116 us by comparing, 61.)  The last workgroup sums the loss.
__global__ void __launch_bounds__(PREF_FINISH) preference_finish_kernel(PrefArgs a) {
  __shared__ __attribute__((aligned(16))) int32_t label[2 * PREF_TILE];
  __shared__ __attribute__((aligned(16))) float slope[2 * PREF_TILE];
  __shared__ __attribute__((aligned(16))) float join[PREF_FINISH * 8];
  __shared__ double sums[PREF_FINISH / 64];
  const int tid = threadIdx.x, threads = blockDim.x;
  if (blockIdx.x == gridDim.x - 1) {
    double t = 0.0;
    for (int i = tid; i < a.chunks; i += threads) t += a.part_loss[i];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) t += __shfl_xor(t, off, 64);
    if ((tid & 63) == 0) sums[tid >> 6] = t;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < threads / 64; ++w) t += sums[w];
      *a.loss = (float)t;
    }
    return;
  }
  const int row = blockIdx.x / (unsigned)a.slices, slice = blockIdx.x % (unsigned)a.slices;
  int begin, end;
  pref_range(a, row, begin, end);
  if (a.dX) {
    constexpr int AT_ONCE = 4;
    const int first = begin / a.chunk, last = end > begin ? (end - 1) / a.chunk : first;
    if (begin == end || first < last) {
      const int groups = threads / a.width, group = tid / a.width, piece = slice * a.width + tid % a.width, k = 8 * piece;
      const int parts = begin < end ? last - first + 1 : 0, per = parts <= AT_ONCE ? AT_ONCE : (parts + groups - 1) / groups;
      Float8 t = {};
      if (group < groups && k < a.d) {
        const int until = first + (group + 1) * per < first + parts ? first + (group + 1) * per : first + parts;
        for (int c0 = first + group * per; c0 < until; c0 += AT_ONCE) {
          Float8 part[AT_ONCE];
#pragma unroll
          for (int j = 0; j < AT_ONCE; ++j) {
            const int c = c0 + j < until ? c0 + j : c0;
            part[j] = load8<XFC_F32>(a.part_dx + (2 * (int64_t)c + (c == first ? 1 : 0)) * a.d + k);
          }
#pragma unroll
          for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) t.v[e] += c0 + j < until ? part[j].v[e] : 0.f;
        }
      }
      if (parts > AT_ONCE) {
        store8<XFC_F32>(join + 8 * tid, t);
        __syncthreads();
        if (group == 0) {
          for (int g = 1; g < groups; ++g) {
            const Float8 other = load8<XFC_F32>(join + 8 * (g * a.width + tid));
#pragma unroll
            for (int e = 0; e < 8; ++e) t.v[e] += other.v[e];
          }
        }
      }
      if (group == 0 && k < a.d) {
#pragma unroll
        for (int e = 0; e < 8; ++e) t.v[e] *= a.scale;
        pref_store(a, (int64_t)row * a.lddx + k, t);
      }
    }
  }
  if (!a.G || slice) return;
  half_t* const g = a.G + (int64_t)row * a.ldg;
  for (int p0 = begin; p0 < end; p0 += PREF_TILE) {
    const int n = end - p0 < PREF_TILE ? end - p0 : PREF_TILE, quads = (n + 1) / 2;
    __syncthreads();
    for (int e = tid; e < 2 * quads; e += threads) {  // an odd number of pairs is filled up with one that is none
      const int c = e < n ? a.chosen[p0 + e] : -1, r = e < n ? a.rejected[p0 + e] : -1;
      const bool ok = c >= 0 && c < a.L && r >= 0 && r < a.L && (!a.weight || a.weight[p0 + e] != 0.f);
      const float s = ok ? a.slope[p0 + e] : 0.f;
      label[2 * e] = ok ? c : -1;
      label[2 * e + 1] = ok ? r : -1;
      slope[2 * e] = s;
      slope[2 * e + 1] = -s;
    }
    __syncthreads();
    if (n > PREF_COMPARED) {
      pref_join_sorted(label, slope, 4 * quads, join, g);
      continue;
    }
    for (int e = tid >> 2; e < 2 * n; e += threads / 4) {  // four neighbouring lanes an entry, every fourth quad each
      const int mine = label[e];
      float t = 0.f;
      int first = e;
#pragma unroll 4
      for (int o = tid & 3; o < quads; o += 4) {
        const int4v l = reinterpret_cast<const int4v*>(label)[o];
        const float4v s = reinterpret_cast<const float4v*>(slope)[o];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          first = l[j] == mine && 4 * o + j < first ? 4 * o + j : first;
          t += l[j] == mine ? s[j] : 0.f;
        }
      }
#pragma unroll
      for (int off = 1; off < 4; off <<= 1) {
        t += __shfl_xor(t, off, 64);
        const int other = __shfl_xor(first, off, 64);
        first = other < first ? other : first;
      }
      if ((tid & 3) == 0 && first == e && mine >= 0) g[mine] = (half_t)((float)g[mine] + t);
    }
  }
}

}  // namespace xfc

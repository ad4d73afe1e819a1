// Linear layer + softmax cross entropy over many classes, with gradients, without keeping the [n, C] logits.
//
//   l_ic = x_i . W_c + b_c      lse_i = log sum_c exp l_ic      ce_i = w[y_i] (lse_i - l_i,y_i)      loss = sum ce / sum w[y]
//   G_ic = s w[y_i] / sum w (exp(l_ic - lse_i) - [c = y_i])     dx = G W       dW = G^T x            db = sum_i G_i
//
// In general two sweeps over the classes.  The first computes logit tiles on the matrix pipe and keeps of each 64-class strip of a row
// its maximum and its sum of exponentials (8 bytes for 64 logits) and the target's logit; the strips of a row are then joined.
// The second computes the tiles again, now against the known lse, and writes G for one piece of the classes at a time (bounded
// scratch), which two products turn into dx (summed over the pieces in fp32) and dW.  8 n C D flops instead of 6: the price of
// not keeping the logits.  Two cases need one sweep: up to 256 classes a tile holds whole rows, and fp32 rows of 256 columns and more whose
// G is one piece keep the first sweep's exponentials in its place and rescale them.
//
// fp32 operands are scaled by a power of two per tensor (in the logits: also per row where rows differ much, pack_row_scale), cut into two
// fp16 planes once per call (mma.h), G likewise: binary32's own accuracy on the fp16 pipe.  bf16 operands are multiplied as they are and G is rounded to bf16 for its two products: relative
// 2^-8 at most, and next to nothing at the entries p - 1 of the targets, which lie next to -1.  With class weights those entries are
// anything, and where a class has one row their rounding is as large as the result's own; then (and for up to 8 rows) the operands are copied
// into one fp16 plane (exact for bf16 values down to 2^-28 of the row's largest, or the tensor's), and G rounded to fp16 (2^-11): 3 passes
// over W more (4096 x 32000 x 1024: 1059 us against 990; 33 x 100000 x 2048: 746 against 446).  db and every sum stay fp32.
//
// Rows with a negative target are left out whatever they hold (x is copied with those rows zero); a target >= C makes its row's
// loss NaN, and with it the mean and the gradients.  No atomics: partial sums are written out and added in a fixed order.
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "mma.h"
#include "tiles.h"

namespace suave {

namespace {

using namespace mma;

constexpr int kStrip = 64;          // classes of one (max, sum) pair
constexpr int kClassPad = 256;      // bias and G are padded to whole tiles of classes
constexpr int kAmaxBlocks = 512;    // partial maxima per tensor
constexpr int64_t kScanElems = 65536;  // x and W together: up to here every packing block finds the maximum itself (a launch less)
constexpr size_t kPieceBytes = (size_t)192 << 20;  // G of one piece: what the 256 MB memory-side cache holds beside its operands

struct Scalars {
  float x_scale, w_scale;    // powers of two the tensors' fp16 operands are multiplied by (1 for bf16 ones)
  int x_split, w_split;      // rows of x / W far below the tensor's largest have scales of their own in the logits' operand (pack_row_scale)
  float g_unit;              // loss_scale * max_w / total / g_scale: what one unit of the stored G is worth
  float max_w;               // largest |class weight| (1 without gradients and without class weights): G is stored relative to it
};

// G is stored relative to the largest row weight (entries in [-1, 1]), in fp16 times 2^14: normal down to 2^-28 in one plane; in two off by
// 2^-23 of itself, or 2^-39 of the largest.  A class that no row gives a chance (p = 2^-20) has its row of dW to 2^-19 of itself, then,
// and one with p below 2^-39 has zeros there.
__host__ __device__ constexpr float g_scale(int type) { return type == kF16 ? 16384.0f : 1.0f; }
// a value in one plane, or two
template <int TYPE, int NP>
__device__ __forceinline__ void g_bits(float v, uint16_t& hi, uint16_t& lo) {
  if constexpr (NP == 2) planes(v, hi, lo);
  else if constexpr (TYPE == kF16) hi = f16_bits((_Float16)v);
  else hi = bf16_bits(v);
}

struct PackArgs {
  const void* src[2];        // x, W
  int64_t ld[2];             // elements
  int64_t rows[2];
  char* dst[2];              // null: not packed.  The operands of the logits
  char* same[2];             // null: not wanted.  Those of the gradients' products where the rows of dst differ in scale: one scale
  float* unit[2];            // [n], [C_pad]: what one unit of a row of dst is worth
  int64_t dst_ld[2];         // bytes
  int blocks0;               // blocks of tensor 0
  int D, Dp;
  const int32_t* targets;    // rows of tensor 0 with a negative target are zero
  float* amax;               // [5][kAmaxBlocks]: largest of x, W, class weights; smallest row (by its largest element) of x, W
  int scan;                  // no k_lce_amax launch: the blocks look for the maxima themselves
  const float* class_weight;
  Scalars* scal;
  const float* bias;         // null: zero
  float* bias_pad;           // [round_up(C, kClassPad)], -inf past C
  int C, C_pad;
};

__device__ __forceinline__ int64_t row_of(int64_t chunk, int64_t chunks, int q) {  // 32-bit division where it reaches
  return chunks <= 0xffffffffll ? (int64_t)((uint32_t)chunk / (uint32_t)q) : chunk / q;
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(uint16_t v) { return bf16_value(v); }
__device__ __forceinline__ float finite_abs(float v) {
  v = fabsf(v);
  return v < INFINITY ? v : 0.f;  // (a NaN compares false)
}

// lanes that share a row of q chunks of eight: a power of two, up to a wave
__device__ __forceinline__ int row_lanes(int q) { return q >= 64 ? 64 : q <= 1 ? 1 : 1 << (32 - __builtin_clz(q - 1)); }

// the maximum over the `L` neighbouring lanes that share a row, in each of them: within 16 lanes without LDS
template <int CTRL>
__device__ __forceinline__ float max_dpp(float v) {
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true)));
}
__device__ __forceinline__ float row_max(float v, int L) {
  if (L > 1) v = max_dpp<0xb1>(v);   // lane ^ 1
  if (L > 2) v = max_dpp<0x4e>(v);   // lane ^ 2
  if (L > 4) v = max_dpp<0x141>(v);  // mirrored within 8: the other four
  if (L > 8) v = max_dpp<0x140>(v);  // mirrored within 16: the other eight
  if (L > 16) v = fmaxf(v, __shfl_xor(v, 16, 64));
  if (L > 32) v = fmaxf(v, __shfl_xor(v, 32, 64));
  return v;
}

// chunk c (eight values, c < ceil(D / 8)) of a row, zeros past D
template <class T>
__device__ __forceinline__ void load_chunk(const PackArgs& a, const T* row, int c, T (&v)[8]) {
  const int d0 = c * 8;
  if (d0 + 8 <= a.D) {
    load8(row + d0, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = d0 + i < a.D ? row[d0 + i] : (T)0;
  }
}

// Largest finite |value| of each row of x (of those that count) or W: mx their largest, mn the smallest that is not zero.  `block` of
// `blocks`; row_lanes lanes share a row, four rows in flight.
template <class T>
__device__ __forceinline__ void scan_rows(const PackArgs& a, int t, int block, int blocks, float& mx, float& mn) {
  const T* src = static_cast<const T*>(a.src[t]);
  const int q = (a.D + 7) / 8, L = row_lanes(q), l = threadIdx.x & (L - 1);
  const int64_t rows = a.rows[t], step = (int64_t)blocks * (256 / L), mine = threadIdx.x / L;
  constexpr int U = 4;
  for (int64_t base = (int64_t)block * (256 / L); base < rows; base += U * step) {  // (the same number of turns for every lane of a wave)
    float m[U];
    const T* row[U];
    bool in[U], gone[U];  // (rows without a target are read like the others: a load that waits for the target takes twice as long)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = base + mine + u * step;
      in[u] = r < rows;
      row[u] = src + (in[u] ? r : 0) * a.ld[t];
      gone[u] = t == 0 && in[u] && a.targets[r] < 0;
      m[u] = 0.f;
    }
    for (int c = l; c < q; c += L) {
      T v[U][8];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = (T)0;
        if (!in[u]) continue;
        if (a.D >= 8) load8(row[u] + min(c * 8, a.D - 8), v[u]);  // (the last chunk may repeat some of the one before)
        else load_chunk(a, row[u], c, v[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) m[u] = fmaxf(m[u], finite_abs(as_float(v[u][i])));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = row_max(gone[u] ? 0.f : m[u], L);
      mx = fmaxf(mx, m[u]);
      if (m[u] > 0.f) mn = fminf(mn, m[u]);
    }
  }
}
__device__ __forceinline__ float wave_max(float v) { return row_max(v, 64); }
// 256 threads; every thread gets the maxima of a and w and the minimum of b
__device__ __forceinline__ void block_extremes(float& a, float& b, float& w, float (&part)[3][4]) {
  a = wave_max(a);
  b = wave_max(-b);
  w = wave_max(w);
  if ((threadIdx.x & 63) == 0) { part[0][threadIdx.x >> 6] = a; part[1][threadIdx.x >> 6] = b; part[2][threadIdx.x >> 6] = w; }
  __syncthreads();
  a = fmaxf(fmaxf(part[0][0], part[0][1]), fmaxf(part[0][2], part[0][3]));
  b = -fmaxf(fmaxf(part[1][0], part[1][1]), fmaxf(part[1][2], part[1][3]));
  w = fmaxf(fmaxf(part[2][0], part[2][1]), fmaxf(part[2][2], part[2][3]));
}

template <class T>
__global__ __launch_bounds__(256) void k_lce_amax(PackArgs a) {
  __shared__ float part[3][4];
  const int t = (int)blockIdx.x >= kAmaxBlocks, b = blockIdx.x - t * kAmaxBlocks;
  float m = 0.f, mn = INFINITY, w = 0.f;
  if (t == 0 && a.class_weight)
    for (int64_t c = (int64_t)b * 256 + threadIdx.x; c < a.C; c += (int64_t)kAmaxBlocks * 256) w = fmaxf(w, finite_abs(a.class_weight[c]));
  scan_rows<T>(a, t, b, kAmaxBlocks, m, mn);
  block_extremes(m, mn, w, part);
  if (threadIdx.x == 0) {
    a.amax[blockIdx.x] = m;
    a.amax[3 * kAmaxBlocks + blockIdx.x] = mn;
    if (t == 0) a.amax[2 * kAmaxBlocks + b] = w;
  }
}

// the power of two that brings amax into [2^13, 2^14) (products of two such and their sums stay far inside binary32)
__device__ __forceinline__ float plane_scale(float amax) {
  if (!(amax > 0.f)) return 1.0f;
  int e;
  (void)frexpf(amax, &e);  // amax = f 2^e, f in [1/2, 1)
  return ldexpf(1.0f, min(14 - e, 120));
}

// A tensor has ONE scale as long as its rows are of a size: fp16 holds both planes of what lies up to 2^14 below the largest element in
// full.  Rows of x are independent in the logits, though, and so are the classes: a row whose largest element is kSplit times smaller than
// the tensor's gets a scale of its own there, or one large row would cost all others their low planes (64 x 1000 x 32 with one
// row 10^6 times the others: their lse off by 3.7e-5 instead of 2.5e-6).  The gradients' products add over these rows (dW over x's, dx
// over W's), so they take operands of one scale: what a small row loses there is 2^-38 of the largest.  Looking for such rows and
// the units' way through the epilogue cost 4096 x 1000 x 128 one microsecond of 60, 1777 x 20011 x 501 five of 466.
constexpr float kSplit = 256.0f;
__device__ __forceinline__ bool split_rows(float mx, float mn) { return mn < mx * (1.0f / kSplit); }
__device__ __forceinline__ float pack_row_scale(float row_max, float mx, float scale) {
  return row_max > 0.f && row_max < mx * (1.0f / kSplit) ? plane_scale(row_max) : scale;
}
template <class T, int PLANES>
__device__ __forceinline__ void store_chunk(char* o, const T (&v)[8], float scale, int Dp) {
  uint16_t hi[8], lo[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (PLANES > 0) g_bits<kF16, PLANES>(as_float(v[i]) * scale, hi[i], lo[i]);
    else hi[i] = v[i];
  }
  *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(hi);
  if constexpr (PLANES == 2) *reinterpret_cast<uint4*>(o + (size_t)Dp * 2) = *reinterpret_cast<const uint4*>(lo);
}

// PLANES 1, 2: scaled fp16; 0: as it is
template <class T, int PLANES>
__global__ __launch_bounds__(256) void k_lce_pack(PackArgs a) {
  const int t = (int)blockIdx.x >= a.blocks0;
  const int b = blockIdx.x - (t ? a.blocks0 : 0), nb = t ? (int)gridDim.x - a.blocks0 : a.blocks0;
  float scale = 1.0f, max_w = 1.0f, largest = 0.f;
  bool split = false;
  if constexpr (PLANES > 0) {
    __shared__ float part[3][4];
    float m = 0.f, mn = INFINITY, w = 0.f;
    if (a.scan) {
      scan_rows<T>(a, t, 0, 1, m, mn);
      if (t == 0 && a.class_weight)
        for (int c = threadIdx.x; c < a.C; c += 256) w = fmaxf(w, finite_abs(a.class_weight[c]));
    } else {
      for (int i = threadIdx.x; i < kAmaxBlocks; i += 256) {
        m = fmaxf(m, a.amax[t * kAmaxBlocks + i]);
        mn = fminf(mn, a.amax[(3 + t) * kAmaxBlocks + i]);
        w = fmaxf(w, a.amax[2 * kAmaxBlocks + i]);
      }
    }
    block_extremes(m, mn, w, part);
    largest = m;
    split = split_rows(m, mn);
    scale = plane_scale(m);
    max_w = a.class_weight && w > 0.f ? w : 1.0f;
  }
  if (b == 0 && threadIdx.x == 0) {
    if (t == 0) {
      a.scal->x_scale = scale;
      a.scal->x_split = split;
      a.scal->max_w = max_w;
    } else {
      a.scal->w_scale = scale;
      a.scal->w_split = split;
    }
  }
  if (t) {
    for (int64_t c = (int64_t)b * 256 + threadIdx.x; c < a.C_pad; c += (int64_t)nb * 256)
      a.bias_pad[c] = c < a.C ? (a.bias ? a.bias[c] : 0.f) : -INFINITY;
  }
  if constexpr (PLANES > 0) {
    const int64_t units = t ? a.C_pad : a.rows[0], from = split ? a.rows[t] : 0;  // (rows of their own scale say theirs below)
    for (int64_t r = from + (int64_t)b * 256 + threadIdx.x; r < units; r += (int64_t)nb * 256) a.unit[t][r] = 1.0f / scale;
  }
  if (a.dst[t] == nullptr) return;
  const T* src = static_cast<const T*>(a.src[t]);
  const int q = a.Dp / 8;  // 16-byte chunks of a row
  const int64_t rows = a.rows[t], ld = a.ld[t];
  if constexpr (PLANES > 0) {
    if (split) {  // row_lanes lanes share a row: its maximum, then its planes (read again, from L2)
      const int L = row_lanes(q), l = threadIdx.x & (L - 1), per = 256 / L;
      for (int64_t base = (int64_t)b * per; base < rows; base += (int64_t)nb * per) {
        const int64_t r = base + threadIdx.x / L;
        const bool in = r < rows && !(t == 0 && a.targets[r] < 0);
        const T* p = src + (in ? r : 0) * ld;
        float m = 0.f;
        for (int c = l; in && c < q; c += L) {
          T v[8];
          load_chunk(a, p, c, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(as_float(v[i])));
        }
        m = row_max(m, L);
        if (r >= rows) continue;
        const float rs = pack_row_scale(m, largest, scale);
        if (l == 0) a.unit[t][r] = 1.0f / rs;
        for (int c = l; c < q; c += L) {
          T v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = (T)0;
          if (in) load_chunk(a, p, c, v);
          const int64_t o = r * a.dst_ld[t] + c * 16;
          store_chunk<T, PLANES>(a.dst[t] + o, v, rs, a.Dp);
          if (a.same[t]) store_chunk<T, PLANES>(a.same[t] + o, v, scale, a.Dp);
        }
      }
      return;
    }
  }
  const int64_t chunks = rows * q;
  for (int64_t e = (int64_t)b * 256 + threadIdx.x; e < chunks; e += (int64_t)nb * 256) {
    const int64_t r = row_of(e, chunks, q);
    const int c = (int)(e - r * q);
    T v[8];
    const bool gone = t == 0 && a.targets[r] < 0;
    load_chunk(a, src + r * ld, c, v);
    if (gone) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (T)0;
    }
    store_chunk<T, PLANES>(a.dst[t] + r * a.dst_ld[t] + c * 16, v, scale, a.Dp);
  }
}

struct TotalArgs {   // loss and the unit of G, from the partial sums of k_lce_rows
  const double* part; int blocks;  // [blocks][2]: sum of ce, sum of w
  const float* weight_sum; float loss_scale, loss_rows; float gs;
  float* loss; double* loss_sum; Scalars* scal;
};
// Every thread of a block of 256 or more takes part; the first 256 add, in a fixed order.
__device__ __forceinline__ void total_loss(const TotalArgs& a, double (&sce)[4], double (&sw)[4]) {
  if (threadIdx.x < 256) {
    double ce = 0.0, w = 0.0;
    for (int i = threadIdx.x; i < a.blocks; i += 256) {
      ce += a.part[2 * i];
      w += a.part[2 * i + 1];
    }
    for (int off = 32; off > 0; off >>= 1) {
      ce += __shfl_xor(ce, off, 64);
      w += __shfl_xor(w, off, 64);
    }
    if ((threadIdx.x & 63) == 0) { sce[threadIdx.x >> 6] = ce; sw[threadIdx.x >> 6] = w; }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const double ce = ((sce[0] + sce[1]) + sce[2]) + sce[3], w = ((sw[0] + sw[1]) + sw[2]) + sw[3];
    const double total = a.weight_sum ? (double)*a.weight_sum : w;
    const bool none = total == 0.0;  // (NaN stays NaN)
    const double loss = none ? 0.0 : ce / total;
    if (a.loss) *a.loss = (float)loss;
    if (a.loss_sum) *a.loss_sum += loss * (double)a.loss_rows;
    a.scal->g_unit = none ? 0.f : (float)((double)a.loss_scale * (double)a.scal->max_w / total / (double)a.gs);
  }
}
__global__ __launch_bounds__(256) void k_lce_total(TotalArgs a) {
  __shared__ double sce[4], sw[4];
  total_loss(a, sce, sw);
}

struct RowArgs {
  const float2* strips; int n_strips;
  int64_t n;
  const int32_t* targets; int C;
  const float* class_weight;
  const float* target_logit;
  float* row_loss;   // or null
  float* lse_out;    // or null
  float2* row;       // (lse, w / max_w)
  double* part;      // [blocks][2]: sum of ce, sum of w over the block's rows
  const Scalars* scal;
};
// What a row's lse and its target's logit give: the row's outputs, and its terms of the two sums
__device__ __forceinline__ void finish_row(const RowArgs& a, int64_t m, float lse, float target_logit, float& ce, float2& row, float& weight) {
  const int y = a.targets[m];
  float w = 0.f, l = 0.f;
  if (y >= a.C) {
    w = l = NAN;
  } else if (y >= 0) {
    w = a.class_weight ? a.class_weight[y] : 1.0f;
    l = w == 0.f ? 0.f : w * (lse - target_logit);
  }
  if (a.row_loss) a.row_loss[m] = l;
  if (a.lse_out) a.lse_out[m] = lse;
  row = make_float2(lse, w / a.scal->max_w);
  ce = l;
  weight = w;
}

struct LogitArgs {
  const char* x; int64_t ldx;      // packed [n][..], bytes
  const char* w; int64_t ldw;
  uint32_t plane;                  // bytes hi -> lo in a row of x and W
  int64_t n;
  int C, D;
  int c0, c1;                      // classes of this launch
  int group;
  const Scalars* scal;
  const float* bias;               // padded
  const float* x_unit;             // [n], scaled fp16 operands: what one unit of a row of x is worth
  const float* w_unit;             // padded
  const int32_t* targets;
  // first sweep
  float2* strips;                  // [strip][n] (max, sum exp(l - max))
  float* target_logit;             // [n]
  // second sweep
  const float2* row;               // (lse, row weight / largest class weight)
  char* g; int64_t ldg; uint32_t g_plane;  // [n][c1 - c0 rounded up], bytes
  float* db;                       // [row tiles of a wave][C_pad]
  int64_t db_ld;
  int totals;                      // 1: the first block of the launch finishes the loss instead
  TotalArgs total;
  RowArgs rows;                    // whole rows in one tile
};

// the units are powers of two
template <int TYPE>
__device__ __forceinline__ float logit(float acc, float x_unit, float w_unit, float bias) {
  if constexpr (TYPE == kF16) return fmaf(acc, x_unit * w_unit, bias);
  else return acc + bias;
}

// G of a tile from its logits and its rows' (lse, weight), and the column sums that db is made of
template <class T>
__device__ __forceinline__ void write_gradients(const LogitArgs& a, const typename T::acc_t (&acc)[T::MI][T::NI], const float4 (&bias)[T::NI],
                                                const float4 (&unit)[T::NI], int tm, int cw, const float2* row_tab, const int* target_tab,
                                                const float* unit_tab, char* stages) {
  constexpr bool P = T::NP == 2;
  typedef RowStage<uint16_t, kStrip> Rows;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / T::WN, g = lane >> 4;
  const int64_t m_base = (int64_t)tm * T::BM;
  char* stage = stages + wave * (T::NP * Rows::kBytes);
  float cs[T::NI][4];
#pragma unroll
  for (int j = 0; j < T::NI; ++j)
#pragma unroll
    for (int u = 0; u < 4; ++u) cs[j][u] = 0.f;
#pragma unroll
  for (int i = 0; i < T::MI; ++i) {
    const int m0 = wm * (T::MI * 16) + 16 * i, ml = m0 + (lane & 15);
    const float2 rw = row_tab[ml];
    const int at = target_tab[ml] - cw;
    const float x_unit = T::TYPE == kF16 ? unit_tab[ml] : 1.0f;
    float p[T::NI][4];
#pragma unroll
    for (int j = 0; j < T::NI; ++j) {
      const float* bj = reinterpret_cast<const float*>(&bias[j]);
      const float* wj = reinterpret_cast<const float*>(&unit[j]);
#pragma unroll
      for (int u = 0; u < 4; ++u) p[j][u] = __expf(logit<T::TYPE>(acc[i][j][u], x_unit, wj[u], bj[u]) - rw.x);
    }
    if (__any(at >= 0 && at < kStrip)) {
#pragma unroll
      for (int j = 0; j < T::NI; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (16 * j + 4 * g + u == at) p[j][u] -= 1.0f;
    }
    const bool counts = rw.y != 0.f;  // a row without weight contributes nothing, whatever it holds
#pragma unroll
    for (int j = 0; j < T::NI; ++j) {
      uint16_t hi[4], lo[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float gv = counts ? p[j][u] * rw.y : 0.f;
        cs[j][u] += gv;
        g_bits<T::TYPE, T::NP>(gv * g_scale(T::TYPE), hi[u], lo[u]);
      }
      Rows::put(stage, lane & 15, 16 * j + 4 * g, hi);
      if constexpr (P) Rows::put(stage + Rows::kBytes, lane & 15, 16 * j + 4 * g, lo);
    }
    const int rows = (int)max<int64_t>(0, min<int64_t>(16, a.n - m_base - m0));
    char* out = a.g + (m_base + m0) * a.ldg + (int64_t)(cw - a.c0) * 2;
    Rows::flush(stage, out, a.ldg, rows, kStrip, lane);
    if constexpr (P) Rows::flush(stage + Rows::kBytes, out + a.g_plane, a.ldg, rows, kStrip, lane);
  }
  if (a.db != nullptr) {  // column sums over the wave's rows: lanes of equal g hold the same columns
#pragma unroll
    for (int j = 0; j < T::NI; ++j) {
      float4 s;
      float* sp = reinterpret_cast<float*>(&s);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float v = cs[j][u];
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
        sp[u] = v;
      }
      if ((lane & 15) == 0) *reinterpret_cast<float4*>(a.db + (int64_t)(tm * T::WM + wm) * a.db_ld + cw + 16 * j + 4 * g) = s;
    }
  }
}

// One tile of logits; SWEEP 0: strip statistics, 1: G, 3: statistics and the exponentials they are made of, for k_lce_scale; 2: statistics
// and G, for tiles that hold whole rows (few classes: no second product and two
// launches less; 1000 x 250 x 256 f32: 38 us against 53 in two sweeps).  What the epilogue needs of bias, targets and rows is asked for before the
// product, one value per thread, and spread through LDS behind it: the matrix pipe covers the latency.
template <class T, int SWEEP>
__global__ __launch_bounds__(T::kThreads, 2) void k_lce_logits(LogitArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  int block = blockIdx.x, blocks = gridDim.x;
  if constexpr (SWEEP == 1) {
    if (a.totals) {
      if (block == 0) {
        double* d = reinterpret_cast<double*>(lds);
        total_loss(a.total, *reinterpret_cast<double(*)[4]>(d), *reinterpret_cast<double(*)[4]>(d + 4));
        return;
      }
      --block; --blocks;
    }
  }
  const int tiles_m = (int)((a.n + T::BM - 1) / T::BM), tiles_n = (a.c1 - a.c0 + T::BN - 1) / T::BN;
  int tm, tn;
  tile_of(block, blocks, tiles_m, tiles_n, a.group, tm, tn);
  const int64_t m_base = (int64_t)tm * T::BM;
  const int c_base = a.c0 + tn * T::BN;
  const int t = threadIdx.x;
  static_assert(T::BM <= T::kThreads && T::BN <= T::kThreads, "one value per thread");
  const bool has_row = t < T::BM && m_base + t < a.n;
  const float my_bias = t < T::BN ? a.bias[c_base + t] : 0.f;
  const int my_target = has_row ? a.targets[m_base + t] : -1;
  float2 my_row = make_float2(0.f, 0.f);
  if (SWEEP == 1 && has_row) my_row = a.row[m_base + t];
  constexpr bool kScaled = T::TYPE == kF16;
  const float my_x_unit = kScaled && has_row ? a.x_unit[m_base + t] : 0.f;
  const float my_w_unit = kScaled && t < T::BN ? a.w_unit[c_base + t] : 0.f;
  const Operand A{a.x + m_base * a.ldx, (uint32_t)a.ldx, (int)min<int64_t>(T::BM, a.n - m_base), a.plane};
  const Operand B{a.w + (int64_t)c_base * a.ldw, (uint32_t)a.ldw, a.C - c_base, a.plane};
  typename T::acc_t acc[T::MI][T::NI];
  T::run(lds, A, B, a.D, acc);
  const int lane = t & 63, wave = t >> 6;
  const int wm = wave / T::WN, wn = wave % T::WN;
  const int g = lane >> 4;
  static_assert(T::NI * 16 == kStrip, "a wave owns one strip");
  float2* row_tab = reinterpret_cast<float2*>(lds);
  float* bias_tab = reinterpret_cast<float*>(row_tab + T::BM);
  int* target_tab = reinterpret_cast<int*>(bias_tab + T::BN);
  float* w_unit_tab = reinterpret_cast<float*>(target_tab + T::BM);  // scaled operands only
  float* x_unit_tab = w_unit_tab + (kScaled ? T::BN : 0);
  float2* strip_tab = reinterpret_cast<float2*>(x_unit_tab + (kScaled ? T::BM : 0));  // whole rows only
  float* logit_tab = reinterpret_cast<float*>(strip_tab + T::WN * T::BM);
  constexpr int kTabs = T::BM * 12 + T::BN * 4 + (kScaled ? (T::BM + T::BN) * 4 : 0) + (SWEEP == 2 ? T::BM * (8 * T::WN + 4) : 0);
  static_assert(kTabs % 16 == 0 && kTabs + T::WM * T::WN * T::NP * RowStage<uint16_t, kStrip>::kBytes <= T::kLds, "tables and stages fit the tile's LDS");
  if (t < T::BN) {
    bias_tab[t] = my_bias;
    if (kScaled) w_unit_tab[t] = my_w_unit;
  }
  if (t < T::BM) {
    target_tab[t] = my_target;
    if (kScaled) x_unit_tab[t] = my_x_unit;
    if (SWEEP == 1) row_tab[t] = my_row;
  }
  __syncthreads();
  const int cw = c_base + wn * kStrip;
  float4 bias[T::NI], unit[T::NI];
#pragma unroll
  for (int j = 0; j < T::NI; ++j) {
    bias[j] = *reinterpret_cast<const float4*>(bias_tab + wn * kStrip + 16 * j + 4 * g);
    unit[j] = kScaled ? *reinterpret_cast<const float4*>(w_unit_tab + wn * kStrip + 16 * j + 4 * g) : make_float4(1.f, 1.f, 1.f, 1.f);
  }
  if constexpr (SWEEP != 1) {
#pragma unroll
    for (int i = 0; i < T::MI; ++i) {
      const int ml = wm * (T::MI * 16) + 16 * i + (lane & 15);
      const int64_t m = m_base + ml;
      const float x_unit = kScaled ? x_unit_tab[ml] : 1.0f;
      float v[T::NI][4], mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < T::NI; ++j) {
        const float* bj = reinterpret_cast<const float*>(&bias[j]);
        const float* wj = reinterpret_cast<const float*>(&unit[j]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          v[j][u] = logit<T::TYPE>(acc[i][j][u], x_unit, wj[u], bj[u]);
          mx = fmaxf(mx, v[j][u]);
        }
      }
      const int at = target_tab[ml] - cw;  // the target's place in the strip
      if (__any(at >= 0 && at < kStrip)) {
#pragma unroll
        for (int j = 0; j < T::NI; ++j)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (16 * j + 4 * g + u == at) (SWEEP == 2 ? logit_tab[ml] : a.target_logit[m]) = v[j][u];
      }
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float base = mx == -INFINITY ? 0.f : mx;  // a strip that is -inf throughout contributes exp(-inf) = 0
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < T::NI; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          v[j][u] = __expf(v[j][u] - base);
          s += v[j][u];
        }
      s += __shfl_xor(s, 16, 64);
      s += __shfl_xor(s, 32, 64);
      if constexpr (SWEEP == 3) {
        typedef RowStage<uint16_t, kStrip> Rows;
        char* stage = lds + kTabs + wave * (T::NP * Rows::kBytes);
#pragma unroll
        for (int j = 0; j < T::NI; ++j) {
          uint16_t hi[4], lo[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) planes(v[j][u] * g_scale(kF16), hi[u], lo[u]);
          Rows::put(stage, lane & 15, 16 * j + 4 * g, hi);
          Rows::put(stage + Rows::kBytes, lane & 15, 16 * j + 4 * g, lo);
        }
        const int64_t m0 = m_base + wm * (T::MI * 16) + 16 * i;
        const int rows = (int)max<int64_t>(0, min<int64_t>(16, a.n - m0));
        char* out = a.g + m0 * a.ldg + (int64_t)cw * 2;
        Rows::flush(stage, out, a.ldg, rows, kStrip, lane);
        Rows::flush(stage + Rows::kBytes, out + a.g_plane, a.ldg, rows, kStrip, lane);
      }
      if (SWEEP == 2) {
        if (g == 0) strip_tab[wn * T::BM + ml] = make_float2(base, s);
      } else {
        if (g == 0 && m < a.n && cw < a.c1) a.strips[(int64_t)(cw / kStrip) * a.n + m] = make_float2(base, s);
      }
    }
  }
  if constexpr (SWEEP == 2) {
    static_assert(T::BM <= 64, "one wave finishes the rows");
    __syncthreads();
    if (t < 64) {
      double ce = 0.0, w = 0.0;
      if (has_row) {
        float mx = -INFINITY, s = 0.f;
#pragma unroll
        for (int k = 0; k < T::WN; ++k)
          if (strip_tab[k * T::BM + t].y != 0.f) mx = fmaxf(mx, strip_tab[k * T::BM + t].x);
#pragma unroll
        for (int k = 0; k < T::WN; ++k)
          if (strip_tab[k * T::BM + t].y != 0.f) s += strip_tab[k * T::BM + t].y * __expf(strip_tab[k * T::BM + t].x - mx);
        float l, rw;
        finish_row(a.rows, m_base + t, s == 0.f ? -INFINITY : mx + logf(s), logit_tab[t], l, row_tab[t], rw);
        ce = l;
        w = rw;
      } else if (t < T::BM) {
        row_tab[t] = make_float2(0.f, 0.f);
      }
      for (int off = 32; off > 0; off >>= 1) {
        ce += __shfl_xor(ce, off, 64);
        w += __shfl_xor(w, off, 64);
      }
      if (t == 0) {
        a.rows.part[2 * tm] = ce;
        a.rows.part[2 * tm + 1] = w;
      }
    }
    if (a.g == nullptr) return;
    __syncthreads();
  }
  if constexpr (SWEEP == 1 || SWEEP == 2) {
    write_gradients<T>(a, acc, bias, unit, tm, cw, row_tab, target_tab, x_unit_tab, lds + kTabs);
  }
}

struct ScaleArgs {
  char* g; int64_t ldg; uint32_t g_plane;
  int64_t n;
  int n_strips, groups;            // groups: of 256 classes
  const float2* strips;
  const float2* row;
  const float* target_logit;
  const int32_t* targets;
  float* db; int64_t db_ld;        // [ceil(n / kScaleRows)][db_ld], or null
  TotalArgs total;
};
constexpr int kScaleRows = 32;

// G from the exponentials of a sweep that kept them, in place: exp(l - strip's max) exp(strip's max - lse) instead of a second product.
// A block takes 32 rows x 256 classes, a thread eight neighbouring classes of every eighth row.  Only for planes, whose rounding
// (2^-23) may be made twice, and where all the classes are one piece.  Bound by the memory-side cache: 1777 x 20011 50 us for 285 MB,
// against 177 us for the second sweep at 501 columns (and 34 more in the first one for the writing).  The first block finishes the loss.
__global__ __launch_bounds__(256) void k_lce_scale(ScaleArgs a) {
  __shared__ double tot[8];
  __shared__ float sums[8][256];
  if (blockIdx.x == 0) {
    total_loss(a.total, *reinterpret_cast<double(*)[4]>(tot), *reinterpret_cast<double(*)[4]>(tot + 4));
    return;
  }
  const int b = blockIdx.x - 1;
  const int64_t rb = b / a.groups;
  const int cl = threadIdx.x & 31, rr = threadIdx.x >> 5;
  const int c = (b - (int)rb * a.groups) * 256 + cl * 8, strip = c / kStrip;
  float cs[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) cs[u] = 0.f;
  constexpr int U = 4;
#pragma unroll
  for (int h = 0; h < kScaleRows / 8 / U; ++h) {
    uint4 hi[U], lo[U];
    float2 st[U], rw[U];
    int y[U];
    float tl[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t m = rb * kScaleRows + (h * U + u) * 8 + rr;
      const bool in = m < a.n;
      const char* p = a.g + (in ? m : 0) * a.ldg + (int64_t)c * 2;
      hi[u] = *reinterpret_cast<const uint4*>(p);
      lo[u] = *reinterpret_cast<const uint4*>(p + a.g_plane);
      st[u] = in && strip < a.n_strips ? a.strips[(int64_t)strip * a.n + m] : make_float2(0.f, 0.f);
      rw[u] = in ? a.row[m] : make_float2(0.f, 0.f);
      y[u] = in ? a.targets[m] : -1;
      tl[u] = in ? a.target_logit[m] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t m = rb * kScaleRows + (h * U + u) * 8 + rr;
      if (m >= a.n) continue;
      // (a strip without any class, or with all its logits -inf, holds zeros; without any logit in the row the result is NaN)
      const bool none = strip >= a.n_strips || (st[u].y == 0.f && rw[u].x > -INFINITY);
      const float f = none || rw[u].y == 0.f ? 0.f : __expf(st[u].x - rw[u].x) * rw[u].y;
      const bool zero = none || rw[u].y == 0.f;  // a row without weight contributes nothing, whatever it holds
      const int at = y[u] - c;
      const uint16_t* ph = reinterpret_cast<const uint16_t*>(&hi[u]);
      const uint16_t* pl = reinterpret_cast<const uint16_t*>(&lo[u]);
      uint16_t oh[8], ol[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v = ((float)__builtin_bit_cast(_Float16, ph[i]) + (float)__builtin_bit_cast(_Float16, pl[i])) * f;
        if (i == at) v = (__expf(tl[u] - rw[u].x) - 1.0f) * (rw[u].y * g_scale(kF16));
        if (zero) v = i == at && rw[u].y != 0.f ? v : 0.f;
        cs[i] += v;
        planes(v, oh[i], ol[i]);
      }
      char* p = a.g + m * a.ldg + (int64_t)c * 2;
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(oh);
      *reinterpret_cast<uint4*>(p + a.g_plane) = *reinterpret_cast<const uint4*>(ol);
    }
  }
  if (a.db == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[rr][cl * 8 + i] = cs[i];
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) s += sums[k][threadIdx.x];
  a.db[rb * a.db_ld + (c - cl * 8) + threadIdx.x] = s * (1.0f / g_scale(kF16));
}

// lse of R rows per block (1024 threads: R rows x 1024 / R strip groups), their loss terms and weights: 16 rows, or 4 for batches that
// would fill few CUs with 16 (33 x 100000: 6 us against 8).  The sums over all blocks are left to the next launch: a ticket that lets
// the last block do it costs every block a release and an acquire at device scope (4096 rows: 18 us, this 7).
template <int R>
__global__ __launch_bounds__(1024) void k_lce_rows(RowArgs a) {
  constexpr int G = 1024 / R;
  __shared__ float2 ms[G][R + 1];
  const int r = threadIdx.x % R, q = threadIdx.x / R;
  const int64_t m = (int64_t)blockIdx.x * R + r;
  float mx = -INFINITY, s = 0.f;
  if (m < a.n) {
    constexpr int U = 8;  // strips in flight
    for (int t0 = q; t0 < a.n_strips; t0 += G * U) {
      float2 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = t0 + G * u < a.n_strips ? a.strips[(int64_t)(t0 + G * u) * a.n + m] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (v[u].y == 0.f) continue;  // nothing of the strip counts (all -inf); NaN goes on
        const float nm = fmaxf(mx, v[u].x);
        s = s * (mx == -INFINITY ? 0.f : __expf(mx - nm)) + v[u].y * __expf(v[u].x - nm);
        mx = nm;
      }
    }
  }
  ms[q][r] = make_float2(mx, s);
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const int part = threadIdx.x / R;  // 64 / R lanes per row, 16 groups each
  float M = -INFINITY, S = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) M = fmaxf(M, ms[part * 16 + k][r].x);
#pragma unroll
  for (int off = R; off < 64; off <<= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
#pragma unroll
  for (int k = 0; k < 16; ++k)
    if (ms[part * 16 + k][r].y != 0.f) S += ms[part * 16 + k][r].y * __expf(ms[part * 16 + k][r].x - M);
#pragma unroll
  for (int off = R; off < 64; off <<= 1) S += __shfl_xor(S, off, 64);
  double ce = 0.0, wsum = 0.0;
  if (part == 0 && m < a.n) {
    const float lse = S == 0.f ? -INFINITY : M + logf(S);
    float l, w;
    finish_row(a, m, lse, a.target_logit[m], l, a.row[m], w);
    ce = l;
    wsum = w;
  }
  for (int off = R / 2; off > 0; off >>= 1) {
    ce += __shfl_xor(ce, off, 64);
    wsum += __shfl_xor(wsum, off, 64);
  }
  if (threadIdx.x == 0) {
    a.part[2 * blockIdx.x] = ce;
    a.part[2 * blockIdx.x + 1] = wsum;
  }
}

struct GradArgs {
  const char* a; int64_t lda; uint32_t a_plane;
  const char* b; int64_t ldb; uint32_t b_plane;
  const char* b_same;          // what takes b's place where b's rows differ in scale (Scalars), or null
  int64_t M;
  int N, K, splits, group;     // split s takes K range [s, s + 1) * round_up(ceil(K / splits), 64)
  float* slab; int64_t slab_stride; int ld_slab;  // fp32 [splits][M][ld_slab]; null: out is written
  int accumulate;              // add to what the slab holds (an earlier piece of the classes)
  void* out; int64_t ld_out;   // T_out [M][N]
  int out_bf16, out_vec;       // out_vec: rows may be stored four elements at a time
  int which;                   // 0: dx (the classes' operand is W), 1: dW (x)
};

__device__ __forceinline__ float grad_factor(const Scalars& s, int which) { return s.g_unit / (which ? s.x_scale : s.w_scale); }

__device__ __forceinline__ void store4(void* out, int64_t at, const float (&v)[4], int n_valid, int bf16, int vec) {
  if (bf16) {
    uint16_t* o = static_cast<uint16_t*>(out) + at;
    uint16_t h[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) h[u] = bf16_bits(v[u]);
    if (vec && n_valid >= 4) *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(h);
    else
      for (int u = 0; u < 4; ++u)
        if (u < n_valid) o[u] = h[u];
  } else {
    float* o = static_cast<float*>(out) + at;
    if (vec && n_valid >= 4) *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
    else
      for (int u = 0; u < 4; ++u)
        if (u < n_valid) o[u] = v[u];
  }
}

template <class T>
__device__ __forceinline__ void grad_tile(const GradArgs& a, int block, char* lds, int b_split, const Scalars* scal) {
  const int tiles_m = (int)((a.M + T::BM - 1) / T::BM), tiles_n = (a.N + T::BN - 1) / T::BN;
  const int per = tiles_m * tiles_n;
  const int split = block / per;
  int tm, tn;
  tile_of(block - split * per, per, tiles_m, tiles_n, a.group, tm, tn);
  const int64_t m_base = (int64_t)tm * T::BM;
  const int n_base = tn * T::BN;
  const int kper = ((a.K + a.splits - 1) / a.splits + 63) / 64 * 64;
  const int k0 = min(split * kper, a.K), k1 = min(k0 + kper, a.K);
  const char* b_base = a.b_same && b_split ? a.b_same : a.b;
  Operand A, B;
  if (T::ACOL) A = Operand{a.a + (int64_t)k0 * a.lda + m_base * 2, (uint32_t)a.lda, (int)min<int64_t>((a.M - m_base + 7) / 8 * 16, 1 << 20), a.a_plane};
  else A = Operand{a.a + m_base * a.lda + (int64_t)k0 * 2, (uint32_t)a.lda, (int)min<int64_t>(T::BM, a.M - m_base), a.a_plane};
  if (T::BCOL) B = Operand{b_base + (int64_t)k0 * a.ldb + (int64_t)n_base * 2, (uint32_t)a.ldb, (a.N - n_base + 7) / 8 * 16, a.b_plane};
  else B = Operand{b_base + (int64_t)n_base * a.ldb + (int64_t)k0 * 2, (uint32_t)a.ldb, a.N - n_base, a.b_plane};
  typename T::acc_t acc[T::MI][T::NI];
  T::run(lds, A, B, k1 - k0, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / T::WN, wn = wave % T::WN;
  const float f = a.slab ? 1.0f : grad_factor(*scal, a.which);
#pragma unroll
  for (int i = 0; i < T::MI; ++i) {
    const int64_t m = m_base + wm * (T::MI * 16) + 16 * i + (lane & 15);
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < T::NI; ++j) {
      const int n = n_base + wn * (T::NI * 16) + 16 * j + 4 * (lane >> 4);
      if (n >= a.N) continue;
      if (a.slab) {
        float4* o = reinterpret_cast<float4*>(a.slab + split * a.slab_stride + m * a.ld_slab + n);
        float4 v = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
        if (a.accumulate) {
          const float4 p = *o;
          v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w;
        }
        *o = v;
      } else {
        const float v[4] = {acc[i][j][0] * f, acc[i][j][1] * f, acc[i][j][2] * f, acc[i][j][3] * f};
        store4(a.out, m * a.ld_out + n, v, a.N - n, a.out_bf16, a.out_vec);
      }
    }
  }
}

// dx and dW of one piece of the classes in one launch: they only share G
template <class TX, class TW>
__global__ __launch_bounds__(TX::kThreads, 2) void k_lce_grads(GradArgs dx, GradArgs dw, int dx_blocks, int totals, TotalArgs total) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int x_split = total.scal->x_split, w_split = total.scal->w_split;
  const int block = (int)blockIdx.x - totals;
  if (block < 0) {  // finishes the loss instead: nothing else in this launch needs it
    double* d = reinterpret_cast<double*>(lds);
    total_loss(total, *reinterpret_cast<double(*)[4]>(d), *reinterpret_cast<double(*)[4]>(d + 4));
  } else if (block < dx_blocks) {
    grad_tile<TX>(dx, block, lds, w_split, total.scal);
  } else {
    grad_tile<TW>(dw, block - dx_blocks, lds, x_split, total.scal);
  }
}

struct FinishArgs {  // out = factor * sum over the slabs, for dx and dW; db = unit * sum over the row tiles
  const float* slab[2]; int n_slabs[2]; int64_t slab_stride[2]; int64_t rows[2]; int ld_slab; int N;
  void* out[2]; int64_t ld_out[2]; int vec[2];
  int out_bf16;
  const float* db; int64_t db_ld; int db_rows, C;
  float* dbias;
  float gs;
  int blk1, blk2;  // blocks [0, blk1) dx, [blk1, blk2) dW, [blk2, grid) db
  const Scalars* scal;
};

__global__ __launch_bounds__(256) void k_lce_finish(FinishArgs a) {
  if ((int)blockIdx.x >= a.blk2) {
    const int c = ((int)blockIdx.x - a.blk2) * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
    __shared__ float part[4][64];
    float s = 0.f;
    if (c < a.C)
      for (int r = q; r < a.db_rows; r += 4) s += a.db[(int64_t)r * a.db_ld + c];
    part[q][threadIdx.x & 63] = s;
    __syncthreads();
    if (q == 0 && c < a.C) a.dbias[c] = (((part[0][threadIdx.x] + part[1][threadIdx.x]) + part[2][threadIdx.x]) + part[3][threadIdx.x]) * (a.scal->g_unit * a.gs);
    return;
  }
  const int w = (int)blockIdx.x >= a.blk1;
  const int64_t b = blockIdx.x - (w ? a.blk1 : 0), nb = w ? a.blk2 - a.blk1 : a.blk1;
  const float f = grad_factor(*a.scal, w);
  const int q = a.ld_slab / 4;
  for (int64_t e = b * 256 + threadIdx.x; e < a.rows[w] * q; e += nb * 256) {
    const int64_t r = e / q;
    const int n = (int)(e - r * q) * 4;
    if (n >= a.N) continue;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < a.n_slabs[w]; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(a.slab[w] + k * a.slab_stride[w] + r * a.ld_slab + n);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const float v[4] = {s.x * f, s.y * f, s.z * f, s.w * f};
    store4(a.out[w], r * a.ld_out[w] + n, v, a.N - n, a.out_bf16, a.vec[w]);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------

struct Layout {  // offsets into the workspace, bytes
  size_t scal, amax, bias, x_unit, w_unit, xp, wp, x_same, w_same, strips, target, row, part, g, db, dx_slab, dw_slab, total;
  int Dp, C_pad, n_strips, piece, pieces;
  int dx_splits, dw_splits;
  int64_t ldp, ldg;      // bytes
  uint32_t plane, g_plane;
  bool pack_w, dw_direct;
  TileId grad_tile;
  int row_blocks, db_rows;
  bool whole;            // one sweep: a tile holds whole rows
  bool keep;             // one sweep: the exponentials stay in G's scratch until lse is known
  int tile_s, tile_g;    // LogitTile of the two sweeps (one per call: the db partials of all pieces have the same rows)
};

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Tile height and width of the logit products.  Up to 16 and 64 rows the tile is as low as the batch and 256 classes wide
// (the weights stream past once; a taller tile would multiply rows that are not there); otherwise 256 x 256 with eight
// waves once that gives every CU a tile, else 128 x 128 (two blocks per CU), or 64 x 128 while there are not enough tiles for
// every CU either (512 x 4000 x 256 f32: 61 us against 65).  Up to 256 classes a tile of 256 holds whole rows.
enum LogitTile : int { kLow16, kLow64, kMid64, kMid128, kBig256 };
constexpr int kLogitM[] = {16, 64, 64, 128, 256}, kLogitWM[] = {1, 1, 2, 2, 2};  // rows, waves side by side in them
LogitTile logit_tile(int64_t n, int64_t classes) {
  if (n <= 16) return kLow16;
  if (n <= 64) return kLow64;
  if (ceil_div(n, 256) * ceil_div(classes, 256) >= kCUs) return kBig256;
  return ceil_div(n, 128) * ceil_div(classes, 128) >= kCUs ? kMid128 : kMid64;
}
// (1000 x 250 x 256: 38 us by 16 rows against 43; 4096 x 256 x 128: 54 against 48)
LogitTile whole_tile(int64_t n) { return n <= 1024 ? kLow16 : kLow64; }

int rows_per_block(int64_t n) { return n <= 1024 ? 4 : 16; }  // of k_lce_rows

// Tile and K splits of the two gradient products of a piece.  A split takes whole multiples of 64 values of K, so a product of
// K values has at most K / 64 of them; dW is not split when the classes come in several pieces (its rows are then plenty).
void pick_grad(int64_t n, int cp, int dim, int planes, bool dx, bool dw, bool one_piece, Layout& L) {
  double best = 1e30;
  const int step = planes == 2 ? 32 : 64;
  for (int t = 0; t < kTileIds; ++t) {
    Work w[2];
    int count = 0, at_dx = -1, at_dw = -1;
    if (dx) { at_dx = count; w[count++] = {ceil_div(n, kTileM[t]) * ceil_div(dim, kTileN[t]), ceil_div(cp, step), 4.0 * n * dim}; }
    if (dw) { at_dw = count; w[count++] = {ceil_div(cp, kTileM[t]) * ceil_div(dim, kTileN[t]), ceil_div(n, step), 4.0 * cp * dim}; }
    for (int sx = 1; sx <= (dx ? 32 : 1); sx *= 2) {
      if (sx > 1 && sx * 64 > cp) break;
      for (int sw = 1; sw <= (dw && one_piece ? 32 : 1); sw *= 2) {
        if (sw > 1 && sw * 64 > n) break;
        int split[2] = {1, 1};
        if (at_dx >= 0) split[at_dx] = sx;
        if (at_dw >= 0) split[at_dw] = sw;
        const double us = estimate_us((TileId)t, planes, w, split, count);
        if (us < best * 0.98) { best = us; L.grad_tile = (TileId)t; L.dx_splits = sx; L.dw_splits = sw; }
      }
    }
  }
}

// Whether a bf16 call's gradients go through fp16 (the head of this file): with class weights, and with few rows, where a row of
// dweight is a few entries of G times rows of x and may happen to round exactly (1 x 1000 x 500: off by 5.6e-4 instead of 3.4e-4).
// Measured against the result's own rounding (300 x 32, 1000 x 500, 5000 x 128; 1 .. 4000 rows): up to 8 rows, in fp16, off by 1.00 - 1.02
// times that; from 9 rows on, in bf16, dx by 1.01 - 1.22 and dweight by 1.02 - 1.35 times, its rows of classes without a target by 1.1 -
// 1.7.  More rows do not change that (every term of a sum has its own error), so above 8 it is speed that decides.
bool bf16_in_half(const suave_linear_ce_t& h) { return (h.dx || h.dweight || h.dbias) && (h.class_weight || h.n_rows <= 8); }

void make_layout(const suave_linear_ce_t& h, Layout& L) {
  const bool f32 = h.dtype == SUAVE_DTYPE_F32;
  const int np = f32 ? 2 : 1;
  const bool grad = h.dx || h.dweight || h.dbias;
  const int64_t n = std::max<int64_t>(h.n_rows, 1);
  L.Dp = round_up(h.dim, 8);
  L.C_pad = round_up(h.n_classes, kClassPad);
  L.n_strips = (int)ceil_div(h.n_classes, kStrip);
  L.ldp = (int64_t)L.Dp * 2 * np;
  L.plane = (uint32_t)(L.Dp * 2);
  L.pack_w = f32 || bf16_in_half(h) || h.dim % 8 != 0 || h.ld_weight % 8 != 0 || (reinterpret_cast<uintptr_t>(h.weight) & 15) != 0;
  const int64_t per_class = n * 2 * np;
  // (at most 2^20 classes: 256 rows of a piece lie within the 2^31 bytes a tile addresses)
  const int64_t piece = std::min<int64_t>(1 << 20, std::max<int64_t>(kClassPad, (int64_t)(kPieceBytes / per_class) / kClassPad * kClassPad));
  L.pieces = (int)ceil_div(L.C_pad, std::min<int64_t>(piece, L.C_pad));
  L.piece = (int)(ceil_div(ceil_div(L.C_pad, L.pieces), kClassPad) * kClassPad);
  L.pieces = (int)ceil_div(L.C_pad, L.piece);
  L.ldg = (int64_t)L.piece * 2 * np;
  L.g_plane = (uint32_t)(L.piece * 2);
  const int cp = std::min(L.piece, (int)h.n_classes);
  L.grad_tile = kT64;
  L.dx_splits = L.dw_splits = 1;
  if (h.dx || h.dweight) pick_grad(n, cp, h.dim, np, h.dx != nullptr, h.dweight != nullptr, L.pieces == 1, L);
  L.whole = h.n_classes <= 256;
  L.dw_direct = L.dw_splits == 1 && !L.whole;  // (in one sweep the unit of G is not known before the gradients' launch ends)
  L.tile_s = L.whole ? whole_tile(n) : logit_tile(n, h.n_classes);
  L.tile_g = L.whole ? L.tile_s : logit_tile(n, cp);
  // (pays where the second product costs more than the pass over G: fp32 1777 x 20011 x 501: 493 us against 576, 4096 x 1000 x 256: 82
  // against 81, 4096 x 1000 x 16: 64 against 57.  Two planes only: db is summed from what is kept)
  L.keep = f32 && grad && L.pieces == 1 && !L.whole && h.dim >= 256;
  L.db_rows = L.keep ? (int)ceil_div(n, kScaleRows) : (int)ceil_div(n, kLogitM[L.tile_g]) * kLogitWM[L.tile_g];
  L.row_blocks = (int)ceil_div(n, L.whole ? kLogitM[L.tile_s] : rows_per_block(n));
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o += up256(bytes); return at; };
  L.scal = take(sizeof(Scalars));
  L.amax = take(sizeof(float) * 5 * kAmaxBlocks);
  L.bias = take(sizeof(float) * L.C_pad);
  L.xp = take((size_t)n * L.ldp);
  L.wp = L.pack_w ? take((size_t)h.n_classes * L.ldp) : 0;
  L.x_unit = L.w_unit = L.x_same = L.w_same = 0;
  if (f32 || bf16_in_half(h)) {
    L.x_unit = take(sizeof(float) * n);
    L.w_unit = take(sizeof(float) * L.C_pad);
  }
  L.strips = take(sizeof(float2) * (size_t)L.n_strips * n);
  L.target = take(sizeof(float) * n);
  L.row = take(sizeof(float2) * n);
  L.part = take(sizeof(double) * 2 * L.row_blocks);
  L.g = L.db = L.dx_slab = L.dw_slab = 0;
  if (grad) {
    L.g = take((size_t)n * L.ldg);
    L.db = take(sizeof(float) * (size_t)L.db_rows * L.C_pad);
    if (h.dx) L.dx_slab = take(sizeof(float) * (size_t)L.dx_splits * n * L.Dp);
    if (h.dweight && !L.dw_direct) L.dw_slab = take(sizeof(float) * (size_t)L.dw_splits * h.n_classes * L.Dp);
  }
  if (f32 || bf16_in_half(h)) {
    if (h.dweight) L.x_same = take((size_t)n * L.ldp);
    if (h.dx) L.w_same = take((size_t)h.n_classes * L.ldp);
  }
  L.total = o;
}

int check_args(const suave_linear_ce_t* h) {
  SUAVE_REQUIRE(h != nullptr, "linear_ce: null argument");
  SUAVE_REQUIRE(h->dtype == SUAVE_DTYPE_F32 || h->dtype == SUAVE_DTYPE_BF16, "linear_ce: dtype must be SUAVE_DTYPE_F32 or SUAVE_DTYPE_BF16");
  SUAVE_REQUIRE(h->n_classes >= 1 && h->n_classes <= (1 << 24), "linear_ce: n_classes must be in 1..2^24");
  SUAVE_REQUIRE(h->dim >= 1 && h->dim <= 32768, "linear_ce: dim must be in 1..32768");
  SUAVE_REQUIRE(h->n_rows >= 0 && h->n_rows <= (1 << 24), "linear_ce: n_rows must be in 0..2^24");
  SUAVE_REQUIRE(h->n_rows * h->n_classes <= ((int64_t)1 << 38), "linear_ce: n_rows * n_classes must be at most 2^38");  // (2^32 threads a launch)
  SUAVE_REQUIRE(h->ld_x >= h->dim && h->ld_weight >= h->dim, "linear_ce: a row stride is shorter than the row");
  SUAVE_REQUIRE(h->ld_x <= (1 << 22) && h->ld_weight <= (1 << 22), "linear_ce: row strides of x and weight must be at most 2^22 elements");
  SUAVE_REQUIRE(!h->dx || h->ld_dx >= h->dim, "linear_ce: ld_dx < dim");
  SUAVE_REQUIRE(!h->dweight || h->ld_dweight >= h->dim, "linear_ce: ld_dweight < dim");
  return 0;
}

// `done`: per kernel, a static of the caller (allow_lds)
int launch_tile(const void* fn, int grid, int threads, int lds, void** args, std::atomic<uint64_t>& done, hipStream_t s) {
  SUAVE_CHECK_HIP(allow_lds(fn, lds, done));
  SUAVE_CHECK_HIP(hipLaunchKernel(fn, dim3(grid), dim3(threads), args, lds, s));
  return 0;
}

template <class T, int SWEEP>
int launch_logits_tile(LogitArgs a, hipStream_t s) {
  const int64_t grid = ceil_div(a.n, T::BM) * ceil_div(a.c1 - a.c0, T::BN) + a.totals;
  a.group = 8;
  void* args[] = {&a};
  static std::atomic<uint64_t> done{0};
  return launch_tile(reinterpret_cast<const void*>(k_lce_logits<T, SWEEP>), (int)grid, T::kThreads, T::kLds, args, done, s);
}

template <int TYPE, int NP, int SWEEP>
int launch_logits(const LogitArgs& a, int tile, hipStream_t s) {
  switch (tile) {
    case kLow16: return launch_logits_tile<Tile<TYPE, NP, false, false, 16, 256, 1, 4>, SWEEP>(a, s);
    case kLow64: return launch_logits_tile<Tile<TYPE, NP, false, false, 64, 256, 1, 4>, SWEEP>(a, s);
    case kMid64: return launch_logits_tile<Tile<TYPE, NP, false, false, 64, 128, 2, 2>, SWEEP>(a, s);
    case kMid128: return launch_logits_tile<Tile<TYPE, NP, false, false, 128, 128, 2, 2>, SWEEP>(a, s);
    default: return launch_logits_tile<Tile<TYPE, NP, false, false, 256, 256, 2, 4>, SWEEP>(a, s);
  }
}

template <int TYPE, int NP>
int launch_whole(const LogitArgs& a, int tile, hipStream_t s) {
  return tile == kLow16 ? launch_logits_tile<Tile<TYPE, NP, false, false, 16, 256, 1, 4>, 2>(a, s)
                        : launch_logits_tile<Tile<TYPE, NP, false, false, 64, 256, 1, 4>, 2>(a, s);
}

template <int TYPE, int NP, int BM, int BN, int WM, int WN>
int launch_grads_tile(GradArgs dx, GradArgs dw, int totals, TotalArgs total, hipStream_t s) {
  typedef Tile<TYPE, NP, false, true, BM, BN, WM, WN> X;
  typedef Tile<TYPE, NP, true, true, BM, BN, WM, WN> W;
  dx.group = dw.group = 8;
  int dx_blocks = (int)(ceil_div(dx.M, BM) * ceil_div(dx.N, BN) * dx.splits);  // (M = 0: not wanted)
  const int blocks = dx_blocks + (int)(ceil_div(dw.M, BM) * ceil_div(dw.N, BN) * dw.splits) + totals;
  void* args[] = {&dx, &dw, &dx_blocks, &totals, &total};
  static std::atomic<uint64_t> done{0};
  return launch_tile(reinterpret_cast<const void*>(k_lce_grads<X, W>), blocks, X::kThreads, X::kLds, args, done, s);
}
template <int TYPE, int NP>
int launch_grads(const GradArgs& dx, const GradArgs& dw, TileId tile, int totals, const TotalArgs& total, hipStream_t s) {
  switch (tile) {
    case kT64: return launch_grads_tile<TYPE, NP, 64, 64, 2, 2>(dx, dw, totals, total, s);
    case kT96: return launch_grads_tile<TYPE, NP, 96, 96, 2, 2>(dx, dw, totals, total, s);
    case kT64x128: return launch_grads_tile<TYPE, NP, 64, 128, 2, 2>(dx, dw, totals, total, s);
    case kT128: return launch_grads_tile<TYPE, NP, 128, 128, 2, 2>(dx, dw, totals, total, s);
    default: return launch_grads_tile<TYPE, NP, 256, 256, 2, 4>(dx, dw, totals, total, s);
  }
}

// What follows the statistics where gradients are wanted: G piece by piece, its two products, the results
template <int TYPE, int NP>
int run_gradients(const suave_linear_ce_t& h, const Layout& L, LogitArgs& a, bool products, hipStream_t s) {
  const bool bf = h.dtype == SUAVE_DTYPE_BF16;
  const int64_t n = h.n_rows;
  char* ws = static_cast<char*>(h.workspace);
  const Scalars* scal = a.scal;
  if (L.keep) {
    const ScaleArgs k{a.g, L.ldg, L.g_plane, n, L.n_strips, L.C_pad / 256, a.strips, a.row, a.target_logit, h.targets, a.db, a.db_ld, a.total};
    hipLaunchKernelGGL(k_lce_scale, dim3((unsigned)(1 + ceil_div(n, kScaleRows) * k.groups)), dim3(256), 0, s, k);
    SUAVE_CHECK_HIP(hipGetLastError());
  }
  auto vec_ok = [&](const void* ptr, int64_t ld) {
    return ld % 4 == 0 && (reinterpret_cast<uintptr_t>(ptr) & (bf ? 7 : 15)) == 0;
  };
  for (int piece = 0; piece < L.pieces; ++piece) {
    a.c0 = piece * L.piece;
    a.c1 = std::min(a.c0 + L.piece, (int)h.n_classes);
    a.totals = piece == 0;
    if (!L.whole && !L.keep)
      if (int rc = launch_logits<TYPE, NP, 1>(a, L.tile_g, s)) return rc;
    const int cp = a.c1 - a.c0;
    GradArgs gx{}, gw{};
    if (h.dx) {
      GradArgs& g = gx;
      g.a = a.g; g.lda = L.ldg; g.a_plane = L.g_plane;
      g.b = a.w + (int64_t)a.c0 * a.ldw; g.ldb = a.ldw; g.b_plane = L.plane;
      g.b_same = TYPE == kF16 ? ws + L.w_same + (int64_t)a.c0 * L.ldp : nullptr;
      g.M = n; g.N = h.dim; g.K = cp; g.splits = L.dx_splits;
      g.slab = reinterpret_cast<float*>(ws + L.dx_slab); g.slab_stride = n * L.Dp; g.ld_slab = L.Dp; g.accumulate = piece > 0;
      g.which = 0;
    }
    if (h.dweight) {
      GradArgs& g = gw;
      g.a = a.g; g.lda = L.ldg; g.a_plane = L.g_plane;
      g.b = a.x; g.ldb = L.ldp; g.b_plane = L.plane;
      g.b_same = TYPE == kF16 ? ws + L.x_same : nullptr;
      g.M = cp; g.N = h.dim; g.K = (int)n; g.splits = L.dw_splits;
      if (!L.dw_direct) {
        g.slab = reinterpret_cast<float*>(ws + L.dw_slab); g.slab_stride = (int64_t)h.n_classes * L.Dp; g.ld_slab = L.Dp;
      }
      g.out = static_cast<char*>(h.dweight) + (int64_t)a.c0 * h.ld_dweight * (bf ? 2 : 4); g.ld_out = h.ld_dweight;
      g.out_bf16 = bf; g.out_vec = vec_ok(h.dweight, h.ld_dweight);
      g.which = 1;
    }
    if (products)
      if (int rc = launch_grads<TYPE, NP>(gx, gw, L.grad_tile, L.whole, a.total, s)) return rc;
  }
  FinishArgs f{};
  f.scal = scal; f.out_bf16 = bf; f.ld_slab = L.Dp; f.N = h.dim; f.gs = g_scale(TYPE);
  int blocks = 0;
  if (h.dx) {
    f.slab[0] = reinterpret_cast<float*>(ws + L.dx_slab); f.n_slabs[0] = L.dx_splits; f.slab_stride[0] = n * L.Dp; f.rows[0] = n;
    f.out[0] = h.dx; f.ld_out[0] = h.ld_dx; f.vec[0] = vec_ok(h.dx, h.ld_dx);
    blocks += (int)std::min<int64_t>(ceil_div(n * (L.Dp / 4), 256), 4096);
  }
  f.blk1 = blocks;
  if (h.dweight && !L.dw_direct) {
    f.slab[1] = reinterpret_cast<float*>(ws + L.dw_slab); f.n_slabs[1] = L.dw_splits; f.slab_stride[1] = (int64_t)h.n_classes * L.Dp;
    f.rows[1] = h.n_classes; f.out[1] = h.dweight; f.ld_out[1] = h.ld_dweight; f.vec[1] = vec_ok(h.dweight, h.ld_dweight);
    blocks += (int)std::min<int64_t>(ceil_div((int64_t)h.n_classes * (L.Dp / 4), 256), 4096);
  }
  f.blk2 = blocks;
  if (h.dbias) {
    f.db = reinterpret_cast<const float*>(ws + L.db); f.db_ld = L.C_pad; f.db_rows = L.db_rows; f.C = h.n_classes; f.dbias = h.dbias;
    blocks += (int)ceil_div(h.n_classes, 64);
  }
  if (blocks > 0) {
    hipLaunchKernelGGL(k_lce_finish, dim3(blocks), dim3(256), 0, s, f);
    SUAVE_CHECK_HIP(hipGetLastError());
  }
  return 0;
}


template <int TYPE, int NP>
int run_linear_ce(const suave_linear_ce_t& h, const Layout& L, hipStream_t s) {
  constexpr bool F = TYPE == kF16;  // scaled fp16
  const bool bf = h.dtype == SUAVE_DTYPE_BF16;
  const bool grad = h.dx || h.dweight || h.dbias;
  const int64_t n = h.n_rows;
  char* ws = static_cast<char*>(h.workspace);
  Scalars* scal = reinterpret_cast<Scalars*>(ws + L.scal);
  PackArgs p{};
  p.src[0] = h.x; p.src[1] = h.weight; p.ld[0] = h.ld_x; p.ld[1] = h.ld_weight; p.rows[0] = n; p.rows[1] = h.n_classes;
  p.dst[0] = ws + L.xp; p.dst[1] = L.pack_w ? ws + L.wp : nullptr; p.dst_ld[0] = p.dst_ld[1] = L.ldp;
  if (F) {
    for (int t = 0; t < 2; ++t) p.unit[t] = reinterpret_cast<float*>(ws + (t ? L.w_unit : L.x_unit));
    p.same[0] = h.dweight ? ws + L.x_same : nullptr;
    p.same[1] = h.dx ? ws + L.w_same : nullptr;
  }
  p.D = h.dim; p.Dp = L.Dp; p.targets = h.targets; p.amax = reinterpret_cast<float*>(ws + L.amax); p.scal = scal;
  p.class_weight = F ? h.class_weight : nullptr;
  p.scan = (n + h.n_classes) * h.dim <= kScanElems;
  p.bias = h.bias; p.bias_pad = reinterpret_cast<float*>(ws + L.bias); p.C = h.n_classes; p.C_pad = L.C_pad;
  if (F && !p.scan) {
    if (bf) hipLaunchKernelGGL(k_lce_amax<uint16_t>, dim3(2 * kAmaxBlocks), dim3(256), 0, s, p);
    else hipLaunchKernelGGL(k_lce_amax<float>, dim3(2 * kAmaxBlocks), dim3(256), 0, s, p);
    SUAVE_CHECK_HIP(hipGetLastError());
  }
  p.blocks0 = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(n * (L.Dp / 8), 256), 1024));
  const int64_t wblocks = L.pack_w ? ceil_div((int64_t)h.n_classes * (L.Dp / 8), 256) : ceil_div(L.C_pad, 256);
  const int grid = p.blocks0 + (int)std::max<int64_t>(1, std::min<int64_t>(wblocks, 4096));
  if (NP == 2) hipLaunchKernelGGL((k_lce_pack<float, 2>), dim3(grid), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((k_lce_pack<uint16_t, F ? 1 : 0>), dim3(grid), dim3(256), 0, s, p);
  SUAVE_CHECK_HIP(hipGetLastError());

  LogitArgs a{};
  a.x = ws + L.xp; a.ldx = L.ldp;
  a.w = L.pack_w ? ws + L.wp : static_cast<const char*>(h.weight);
  a.ldw = L.pack_w ? L.ldp : h.ld_weight * 2;
  a.plane = L.plane; a.n = n; a.C = h.n_classes; a.D = h.dim; a.c0 = 0; a.c1 = h.n_classes; a.scal = scal;
  a.bias = p.bias_pad; a.targets = h.targets; a.x_unit = p.unit[0]; a.w_unit = p.unit[1];
  a.strips = reinterpret_cast<float2*>(ws + L.strips);
  a.target_logit = reinterpret_cast<float*>(ws + L.target);
  a.row = reinterpret_cast<const float2*>(ws + L.row);

  RowArgs& r = a.rows;
  r.strips = a.strips; r.n_strips = L.n_strips; r.n = n; r.targets = h.targets; r.C = h.n_classes;
  r.class_weight = h.class_weight; r.target_logit = a.target_logit; r.row_loss = h.row_loss; r.lse_out = h.lse;
  r.row = reinterpret_cast<float2*>(ws + L.row); r.part = reinterpret_cast<double*>(ws + L.part); r.scal = scal;
  a.total = TotalArgs{r.part, L.row_blocks, h.weight_sum, h.loss_scale, h.loss_rows, g_scale(TYPE), h.loss, h.loss_sum, scal};
  a.db_ld = L.C_pad;
  a.ldg = L.ldg; a.g_plane = L.g_plane;
  if (grad) {
    a.g = ws + L.g;
    a.db = h.dbias ? reinterpret_cast<float*>(ws + L.db) : nullptr;
  }
  const bool products = h.dx || h.dweight;
  if (L.whole) {
    if (int rc = launch_whole<TYPE, NP>(a, L.tile_s, s)) return rc;
  } else {
    if constexpr (NP == 2) {
      if (int rc = L.keep ? launch_logits<TYPE, NP, 3>(a, L.tile_s, s) : launch_logits<TYPE, NP, 0>(a, L.tile_s, s)) return rc;
    } else {
      if (int rc = launch_logits<TYPE, NP, 0>(a, L.tile_s, s)) return rc;
    }
    if (rows_per_block(n) == 4) hipLaunchKernelGGL(k_lce_rows<4>, dim3(L.row_blocks), dim3(1024), 0, s, r);
    else hipLaunchKernelGGL(k_lce_rows<16>, dim3(L.row_blocks), dim3(1024), 0, s, r);
    SUAVE_CHECK_HIP(hipGetLastError());
  }
  if (!grad || (L.whole && !products)) {
    hipLaunchKernelGGL(k_lce_total, dim3(1), dim3(256), 0, s, a.total);
    SUAVE_CHECK_HIP(hipGetLastError());
    if (!grad) return 0;
  }

  return run_gradients<TYPE, NP>(h, L, a, products, s);
}

}  // namespace

int linear_ce_workspace(const suave_linear_ce_t* h, size_t* bytes) {
  if (int rc = check_args(h)) return rc;
  SUAVE_REQUIRE(bytes != nullptr, "linear_ce: bytes is null");
  Layout L;
  make_layout(*h, L);
  *bytes = L.total;
  return 0;
}

__global__ __launch_bounds__(256) void k_lce_empty(float* loss, float* dbias, int C, void* dweight, int64_t ld, int D, int bf16) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  if (t == 0 && loss) *loss = 0.f;
  if (dbias)
    for (int64_t c = t; c < C; c += step) dbias[c] = 0.f;
  if (dweight)
    for (int64_t e = t; e < (int64_t)C * D; e += step) {
      const int64_t r = e / D, d = e - r * D;
      if (bf16) static_cast<uint16_t*>(dweight)[r * ld + d] = 0;
      else static_cast<float*>(dweight)[r * ld + d] = 0.f;
    }
}

int launch_linear_ce(const suave_linear_ce_t* h, hipStream_t s) {
  if (int rc = check_args(h)) return rc;
  if (h->n_rows == 0) {  // an empty batch: loss 0, zero gradients
    hipLaunchKernelGGL(k_lce_empty, dim3(256), dim3(256), 0, s, h->loss, h->dbias, h->n_classes, h->dweight, h->ld_dweight, h->dim,
                       (int)(h->dtype == SUAVE_DTYPE_BF16));
    SUAVE_CHECK_HIP(hipGetLastError());
    return 0;
  }
  SUAVE_REQUIRE(h->x && h->weight && h->targets, "linear_ce: x / weight / targets is null");
  const uintptr_t align = h->dtype == SUAVE_DTYPE_BF16 ? 1 : 3;
  for (const void* ptr : {h->x, h->weight, static_cast<const void*>(h->dx), static_cast<const void*>(h->dweight)})
    SUAVE_REQUIRE((reinterpret_cast<uintptr_t>(ptr) & align) == 0, "linear_ce: x / weight / dx / dweight is not aligned to its elements");
  SUAVE_REQUIRE(h->dx != h->x && h->dx != h->weight && h->dweight != h->x && h->dweight != h->weight && (!h->dx || h->dx != h->dweight),
                "linear_ce: an output is an input or another output");
  Layout L;
  make_layout(*h, L);
  SUAVE_REQUIRE(h->workspace && (reinterpret_cast<uintptr_t>(h->workspace) & 255) == 0, "linear_ce: workspace is null or not 256-byte aligned");
  SUAVE_REQUIRE(h->workspace_bytes >= L.total, "linear_ce: workspace too small (suave_linear_ce_workspace_bytes)");
  if (h->dtype == SUAVE_DTYPE_F32) return run_linear_ce<kF16, 2>(*h, L, s);
  return bf16_in_half(*h) ? run_linear_ce<kF16, 1>(*h, L, s) : run_linear_ce<kBf16, 1>(*h, L, s);
}

}  // namespace suave

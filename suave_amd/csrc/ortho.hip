// Orthogonalised updates: Newton-Schulz products, and the Muon step built on them.
//
//   X_0 = U / (|U|_F + eps)      A = X X^T      B = a I + b A + c A A      X <- B X,     (a, b, c) = (3.4445, -4.7750, 2.0315)
//
// drives every singular value of U towards 1 (after five steps into about 0.7 .. 1.2) and keeps the singular vectors.  X is
// kept in the orientation of U; A and B live on the short side, so a tall U uses A = X^T X and X <- X B.  A and B are
// symmetric: only tiles on and above the diagonal are computed, what lies below it is written as the mirror image, which takes a
// step from 2 s^2 l + 2 s^3 + 2 s^2 l to s^2 l + s^3 + 2 s^2 l flops (s the short side, l the long one).  All matrices of a
// call go through the same launches: three per step for the whole list.
//
// Arithmetic (mma.h).  fp32 matrices: every factor as two fp16 planes, which keeps binary32's accuracy -- the iteration
// multiplies small singular directions, and rounding noise in them, by up to a^5 = 485.  bf16 matrices from a short side of 128 on: one fp16 plane (11 bits;
// the result is rounded to 8): a relative error of about 1.3e-3 where the rounding of the result is 1.7e-3.  Factors are stored times a power of two:
// X times 2^(12 - e), A times 2^(12 - 2 e), B times 2^12, with 2^e the size of X (e = 0 unless |U|_F is below eps): entries of
// X are at most about 1.3 in magnitude, and start at 1 / sqrt(rows cols), which 2^12 keeps clear of fp16's subnormals.
#include <algorithm>
#include <cmath>
#include <utility>

#include "kernels.h"
#include "mma.h"
#include "tiles.h"

namespace suave {

namespace {

using namespace mma;

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr int kMaxMats = 24;      // matrices of one group of launches
constexpr int kMaxSteps = 16;
constexpr int kNormBlocks = 512;  // partial sums per matrix
constexpr float kS = 4096.0f;

struct Mat {
  const void* in;       // U (orthogonalize) or the gradient (muon)
  void* out;            // result or parameter
  float* mom;           // muon: momentum
  int64_t ld_in, ld_out, ld_mom;
  char* x[2];           // planes of X, [rows][pitch]
  char* a;              // [short][pitch_s]
  char* b;
  int rows, cols;
  int id;               // index of its partial sums and sizes
  float lr;             // muon: learning rate times shape factor
  float decay;          // muon: 1 - learning rate * weight decay
};

struct Group {
  Mat m[kMaxMats];
  int32_t begin[kMaxMats + 1];  // first block of each matrix in this launch
  int n;
  double* part;                 // [kMaxMats][kNormBlocks]
  int32_t* exps;                // [kMaxMats][kMaxSteps + 1]: e of X_k
  double eps;
  float momentum;
  int nesterov, muon, bf16, steps, k;  // k: the step
};

__device__ __forceinline__ int find_mat(const Group& g, int b) {
  int i = 0;
  while (i + 1 < g.n && b >= g.begin[i + 1]) ++i;
  return i;
}
__host__ __device__ inline int pitch(int cols, int np) { return (cols + 7) / 8 * 8 * 2 * np; }  // bytes of a stored row

__device__ __forceinline__ float in_value(const Group& g, const Mat& m, int64_t r, int c) {
  if (g.bf16) return bf16_value(static_cast<const uint16_t*>(m.in)[r * m.ld_in + c]);
  const float v = static_cast<const float*>(m.in)[r * m.ld_in + c];
  if (!g.muon) return v;
  const float mom = m.mom[r * m.ld_mom + c];  // already this step's
  return g.nesterov ? fmaf(g.momentum, mom, v) : mom;
}

// blocks of k_ortho_norm for a matrix: 2048 elements each, eight per thread
__host__ __device__ inline int norm_blocks(int rows, int cols) {
  const int64_t b = ((int64_t)rows * cols + 2047) / 2048;
  return b < kNormBlocks ? (int)b : kNormBlocks;
}

// Eight neighbours of U's row r from column c0 (zeros past the row); muon: from the gradient and this step's momentum
__device__ __forceinline__ void in_values(const Group& g, const Mat& m, int64_t r, int c0, float (&v)[8]) {
  if (c0 + 8 <= m.cols) {
    if (g.bf16) {
      uint16_t w[8];
      load8(static_cast<const uint16_t*>(m.in) + r * m.ld_in + c0, w);
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = bf16_value(w[u]);
      return;
    }
    load8(static_cast<const float*>(m.in) + r * m.ld_in + c0, v);
    if (g.muon) {
      float mom[8];
      load8(m.mom + r * m.ld_mom + c0, mom);
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = g.nesterov ? fmaf(g.momentum, mom[u], v[u]) : mom[u];
    }
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = c0 + u < m.cols ? in_value(g, m, r, c0 + u) : 0.f;
  }
}

// Partial sums of squares (double: neither overflow nor loss over 2^24 values); muon: the momentum first.  Chunks of eight
// neighbours, two in flight per thread.
__global__ __launch_bounds__(256) void k_ortho_norm(Group g) {
  const int i = find_mat(g, blockIdx.x);
  const Mat& m = g.m[i];
  const int b = blockIdx.x - g.begin[i], nb = g.begin[i + 1] - g.begin[i];
  const int q = (m.cols + 7) / 8;
  const int64_t chunks = (int64_t)m.rows * q, step = (int64_t)nb * 256;
  double s = 0.0;
  for (int64_t e0 = (int64_t)b * 256 + threadIdx.x; e0 < chunks; e0 += 2 * step) {
    float v[2][8], mom[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t e = e0 + h * step;
#pragma unroll
      for (int u = 0; u < 8; ++u) v[h][u] = mom[h][u] = 0.f;
      if (e >= chunks) continue;
      const int64_t r = chunks < (1ll << 31) ? (int64_t)((uint32_t)e / (uint32_t)q) : e / q;
      const int c0 = (int)(e - r * q) * 8;
      if (!g.muon) {
        in_values(g, m, r, c0, v[h]);
      } else {
        const float* gr = static_cast<const float*>(m.in) + r * m.ld_in + c0;
        const float* mo = m.mom + r * m.ld_mom + c0;
        if (c0 + 8 <= m.cols) {
          load8(gr, v[h]);
          load8(mo, mom[h]);
        } else {
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (c0 + u < m.cols) { v[h][u] = gr[u]; mom[h][u] = mo[u]; }
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t e = e0 + h * step;
      if (e >= chunks) continue;
      if (g.muon) {
        const int64_t r = chunks < (1ll << 31) ? (int64_t)((uint32_t)e / (uint32_t)q) : e / q;
        const int c0 = (int)(e - r * q) * 8;
        float* mo = m.mom + r * m.ld_mom + c0;
        f32x4_any w[2];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float mn = fmaf(g.momentum, mom[h][u], v[h][u]);
          w[u / 4][u % 4] = mn;
          v[h][u] = g.nesterov ? fmaf(g.momentum, mn, v[h][u]) : mn;
        }
        if (c0 + 8 <= m.cols) {
          *reinterpret_cast<f32x4_any*>(mo) = w[0];
          *reinterpret_cast<f32x4_any*>(mo + 4) = w[1];
        } else {
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (c0 + u < m.cols) mo[u] = w[u / 4][u % 4];
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) s += (double)v[h][u] * (double)v[h][u];
    }
  }
  __shared__ double part[4];
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) g.part[m.id * kNormBlocks + b] = (part[0] + part[1]) + (part[2] + part[3]);
}

// from the sum of squares of U: what U is multiplied by to give the stored X_0, and the sizes e of X_0 .. X_steps
__device__ __forceinline__ double start_scale(double sum, double eps, int steps, int* exps) {
  const double norm = sqrt(sum), full = norm + eps;
  double f = norm / full;  // |X_0|_F
  int e0 = 0;
  for (int k = 0; k <= steps; ++k) {
    int e = 0;
    if (f > 0.0 && f < 1.0) { (void)frexp(f, &e); e = max(e, -100); }
    if (!(e < 0)) e = 0;
    if (k == 0) e0 = e;
    exps[k] = e;
    f *= (double)kNsA;
  }
  return isfinite(sum) ? ldexp(1.0 / full, 12 - e0) : (double)NAN;  // anything not finite: the whole result is NaN
}
__device__ __forceinline__ void write_result(const Group& g, const Mat& m, int r, int c, float v) {
  if (g.bf16) {
    static_cast<uint16_t*>(m.out)[(int64_t)r * m.ld_out + c] = bf16_bits(v);
  } else {
    float* o = static_cast<float*>(m.out) + (int64_t)r * m.ld_out + c;
    *o = g.muon ? fmaf(-m.lr, v, *o * m.decay) : v;
  }
}

// four neighbours, as one access each way
__device__ __forceinline__ void write_results(const Group& g, const Mat& m, int r, int c, const float (&v)[4]) {
  if (c + 4 > m.cols) {
    for (int u = 0; c + u < m.cols; ++u) write_result(g, m, r, c + u, v[u]);
  } else if (g.bf16) {
    typedef uint16_t u16x4_any __attribute__((ext_vector_type(4), aligned(2)));
    *reinterpret_cast<u16x4_any*>(static_cast<uint16_t*>(m.out) + (int64_t)r * m.ld_out + c) = u16x4_any{bf16_bits(v[0]), bf16_bits(v[1]), bf16_bits(v[2]), bf16_bits(v[3])};
  } else {
    f32x4_any* o = reinterpret_cast<f32x4_any*>(static_cast<float*>(m.out) + (int64_t)r * m.ld_out + c);
    f32x4_any w = f32x4_any{v[0], v[1], v[2], v[3]};
    if (g.muon) {
      const f32x4_any p = *o;
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u] = fmaf(-m.lr, v[u], p[u] * m.decay);
    }
    *o = w;
  }
}

// X_0 in planes, pads zero; the sizes of X_0 .. X_steps.  The norm is a chain of a few microseconds in every block, so two chunks
// per thread are asked for in front of it and the grid fits the card in one round; the scaling is two exact-range binary32 steps (in
// doubles the kernel was bound by their conversions: 2 x (1024 x 4096) bf16 18 us, this 11).
constexpr int kPackBlocks = 512;  // per matrix
template <int NP>
__global__ __launch_bounds__(256) void k_ortho_pack(Group g) {
  const int i = find_mat(g, blockIdx.x);
  const Mat& m = g.m[i];
  const int b = blockIdx.x - g.begin[i], nb = g.begin[i + 1] - g.begin[i];
  const int cp = (m.cols + 7) / 8 * 8, q = cp / 8;
  const int64_t chunks = (int64_t)m.rows * q, step = (int64_t)nb * 256;
  const int pit = pitch(m.cols, NP);
  constexpr int U = 2;
  float in[U][8];
  int64_t r[U];
  int c0[U];
  auto load = [&](int64_t e0) {
#pragma unroll
    for (int h = 0; h < U; ++h) {
      const int64_t e = e0 + h * step;
      if (e >= chunks) continue;
      r[h] = chunks < (1ll << 31) ? (int64_t)((uint32_t)e / (uint32_t)q) : e / q;
      c0[h] = (int)(e - r[h] * q) * 8;
      in_values(g, m, r[h], c0[h], in[h]);
    }
  };
  int64_t e0 = (int64_t)b * 256 + threadIdx.x;
  load(e0);
  __shared__ double sc, part[4];
  {
    double s = 0.0;
    const int n = norm_blocks(m.rows, m.cols);
    for (int k = threadIdx.x; k < n; k += 256) s += g.part[m.id * kNormBlocks + k];
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      int e[kMaxSteps + 1];
      sc = start_scale((part[0] + part[1]) + (part[2] + part[3]), g.eps, b == 0 ? g.steps : 0, e);
      if (b == 0)
        for (int k = 0; k <= g.steps; ++k) g.exps[m.id * (kMaxSteps + 1) + k] = e[k];
    }
  }
  __syncthreads();
  // scale = sm 2^se: the power of two first, so neither a subnormal U nor a huge scale leaves binary32
  int se = 0;
  const float sm = (float)frexp(sc, &se);
  while (e0 < chunks) {
#pragma unroll
    for (int h = 0; h < U; ++h) {
      if (e0 + h * step >= chunks) continue;
      uint16_t hi[8], lo[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float v = c0[h] + u < m.cols ? ldexpf(in[h][u], se) * sm : 0.f;
        if constexpr (NP == 2) planes(v, hi[u], lo[u]);
        else hi[u] = f16_bits((_Float16)v);
      }
      char* o = m.x[0] + r[h] * pit + c0[h] * 2;
      *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(hi);
      if constexpr (NP == 2) *reinterpret_cast<uint4*>(o + cp * 2) = *reinterpret_cast<const uint4*>(lo);
    }
    e0 += U * step;
    load(e0);
  }
}

// stores four consecutive elements (n .. n + 3) of row m, elements past `cols` as zero; n < round_up(cols, 8)
template <int NP>
__device__ __forceinline__ void store_planes(char* base, int pit, int cols, int64_t m, int n, const float (&v)[4]) {
  uint16_t hi[4], lo[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float x = n + u < cols ? v[u] : 0.f;
    if constexpr (NP == 2) planes(x, hi[u], lo[u]);
    else hi[u] = f16_bits((_Float16)x);
  }
  char* o = base + m * pit + n * 2;
  *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(hi);
  if constexpr (NP == 2) *reinterpret_cast<uint2*>(o + (cols + 7) / 8 * 16) = *reinterpret_cast<const uint2*>(lo);
}
// the mirror image: elements (n .. n + 3, m)
template <int NP>
__device__ __forceinline__ void store_mirror(char* base, int pit, int cols, int m, int n, const float (&v)[4]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (n + u >= cols) continue;
    char* o = base + (int64_t)(n + u) * pit + m * 2;
    if constexpr (NP == 2) {
      uint16_t hi, lo;
      planes(v[u], hi, lo);
      *reinterpret_cast<uint16_t*>(o) = hi;
      *reinterpret_cast<uint16_t*>(o + (cols + 7) / 8 * 16) = lo;
    } else {
      *reinterpret_cast<uint16_t*>(o) = f16_bits((_Float16)v[u]);
    }
  }
}

// (m, n .. n + 3) of a symmetric matrix and their mirror image.  Each pair of elements comes from the one above the diagonal: in two planes
// the two sums differ in the order of their cross terms, and which of them a tile computes depends on its size.
// `side`: fragments above (1), on (0) or below (-1) the diagonal.
template <int NP>
__device__ __forceinline__ void store_symmetric(char* base, int pit, int s, int m, int n, const float (&v)[4], int side) {
  if (side > 0) {
    store_planes<NP>(base, pit, s, m, n, v);
    store_mirror<NP>(base, pit, s, m, n, v);
  } else if (side == 0) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = n + u;
      if (c < m) continue;
      const float x = c < s ? v[u] : 0.f;
      uint16_t hi, lo = 0;
      if constexpr (NP == 2) planes(x, hi, lo);
      else hi = f16_bits((_Float16)x);
      auto put = [&](int r, int k) {
        char* o = base + (int64_t)r * pit + k * 2;
        *reinterpret_cast<uint16_t*>(o) = hi;
        if constexpr (NP == 2) *reinterpret_cast<uint16_t*>(o + (s + 7) / 8 * 16) = lo;
      };
      put(m, c);
      if (c > m && c < s) put(c, m);
    }
  }
}

template <class T, int GROUPS, int PARTS>
__device__ __forceinline__ void run_tile(char* lds, const Operand& A, const Operand& B, int K, typename T::acc_t (&acc)[T::MI][T::NI]) {
  if constexpr (GROUPS > 1) T::template run_split<GROUPS, PARTS>(lds, A, B, K, acc);
  else T::run(lds, A, B, K, acc);
}

// tile t of the T (T + 1) / 2 on and above the diagonal
__device__ __forceinline__ void upper_tile(int t, int T, int& tm, int& tn) {
  tm = 0;
  while (t >= T - tm) { t -= T - tm; ++tm; }
  tn = tm + t;
}

// Waves per SIMD that a block's registers must leave room for: 1024 threads, or two blocks of 512, on a CU
constexpr int min_waves(int threads, int parts) { return threads >= 1024 || parts > 1 ? 4 : 2; }

// POLY 0: A from X; 1: B from A
template <int NP, int BM, int WM, int WN, int POLY, int GROUPS, int PARTS>
__global__ __launch_bounds__(64 * WM * WN * GROUPS, min_waves(64 * WM * WN * GROUPS, PARTS)) void k_ortho_sym(Group g) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  typedef Tile<kF16, NP, false, false, BM, BM, WM, WN> R;
  typedef Tile<kF16, NP, true, true, BM, BM, WM, WN> C;
  const int i = find_mat(g, blockIdx.x);
  const Mat& m = g.m[i];
  const int s = min(m.rows, m.cols), T = (s + BM - 1) / BM;
  const int ps = pitch(s, NP);
  int tm, tn;
  upper_tile(die_order(blockIdx.x - g.begin[i], T * (T + 1) / 2), T, tm, tn);
  const int m0 = tm * BM, n0 = tn * BM;
  f32x4 acc[R::MI][R::NI];
  if (POLY) {
    const uint32_t plane = (s + 7) / 8 * 16;
    run_tile<R, GROUPS, PARTS>(lds, Operand{m.a + (int64_t)m0 * ps, (uint32_t)ps, s - m0, plane}, Operand{m.a + (int64_t)n0 * ps, (uint32_t)ps, s - n0, plane}, s, acc);
  } else {
    const int px = pitch(m.cols, NP);
    const uint32_t plane = (m.cols + 7) / 8 * 16;
    const char* x = m.x[g.k & 1];
    if (m.rows <= m.cols)
      run_tile<R, GROUPS, PARTS>(lds, Operand{x + (int64_t)m0 * px, (uint32_t)px, s - m0, plane}, Operand{x + (int64_t)n0 * px, (uint32_t)px, s - n0, plane}, m.cols, acc);
    else
      run_tile<C, GROUPS, PARTS>(lds, Operand{x + m0 * 2, (uint32_t)px, (s - m0 + 7) / 8 * 16, plane}, Operand{x + n0 * 2, (uint32_t)px, (s - n0 + 7) / 8 * 16, plane}, m.rows, acc);
  }
  const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) % (WM * WN), group = (threadIdx.x >> 6) / (WM * WN);
  const int wm = wave / WN, wn = wave % WN;
  const int e = g.exps[m.id * (kMaxSteps + 1) + g.k];
  const float fb = ldexpf(kNsB, 2 * e), fc = ldexpf(kNsC, max(4 * e - 12, -126));
  const int sp = (s + 7) / 8 * 8;
#pragma unroll
  for (int mi = 0; mi < R::MI; ++mi) {
    const int r = m0 + wm * (R::MI * 16) + 16 * mi + (lane & 15);
    if (r >= s) continue;
#pragma unroll
    for (int j = 0; j < R::NI; ++j) {
      if (GROUPS > 1 && (R::MI * j + mi) % GROUPS != group) continue;
      const int n = n0 + wn * (R::NI * 16) + 16 * j + 4 * (lane >> 4);
      const int above = (n0 + wn * (R::NI * 16) + 16 * j) - (m0 + wm * (R::MI * 16) + 16 * mi), side = (above > 0) - (above < 0);
      if (n >= sp || side < 0) continue;
      float v[4];
      if (POLY) {
        uint16_t hi[4], lo[4];
        const char* o = m.a + (int64_t)r * ps + n * 2;
        *reinterpret_cast<uint2*>(hi) = *reinterpret_cast<const uint2*>(o);
        if (NP == 2) *reinterpret_cast<uint2*>(lo) = *reinterpret_cast<const uint2*>(o + sp * 2);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float av = (float)__builtin_bit_cast(_Float16, hi[u]);
          if (NP == 2) av += (float)__builtin_bit_cast(_Float16, lo[u]);
          v[u] = fmaf(fc, acc[mi][j][u], fb * av) + (r == n + u ? kNsA * kS : 0.f);
        }
        store_symmetric<NP>(m.b, ps, s, r, n, v, side);
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = acc[mi][j][u] * (1.0f / kS);
        store_symmetric<NP>(m.a, ps, s, r, n, v, side);
      }
    }
  }
}

// X <- B X (wide) or X B (tall); the last step writes the result or takes the step on the parameter
template <int NP, int BM, int BN, int WM, int WN, bool LAST, int GROUPS>
__global__ __launch_bounds__(64 * WM * WN * GROUPS, min_waves(64 * WM * WN * GROUPS, 1)) void k_ortho_update(Group g) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  typedef Tile<kF16, NP, false, true, BM, BN, WM, WN> W;
  typedef Tile<kF16, NP, false, false, BM, BN, WM, WN> H;
  const int i = find_mat(g, blockIdx.x);
  const Mat& m = g.m[i];
  const int s = min(m.rows, m.cols);
  const int ps = pitch(s, NP), px = pitch(m.cols, NP);
  const uint32_t plane_s = (s + 7) / 8 * 16, plane_x = (m.cols + 7) / 8 * 16;
  const int tiles_m = (m.rows + BM - 1) / BM, tiles_n = (m.cols + BN - 1) / BN;
  int tm, tn;
  tile_of(blockIdx.x - g.begin[i], tiles_m * tiles_n, tiles_m, tiles_n, 8, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const char* x = m.x[g.k & 1];
  f32x4 acc[W::MI][W::NI];
  if (m.rows <= m.cols)
    run_tile<W, GROUPS, 1>(lds, Operand{m.b + (int64_t)m0 * ps, (uint32_t)ps, s - m0, plane_s}, Operand{x + (int64_t)n0 * 2, (uint32_t)px, (m.cols - n0 + 7) / 8 * 16, plane_x}, s, acc);
  else
    run_tile<H, GROUPS, 1>(lds, Operand{x + (int64_t)m0 * px, (uint32_t)px, m.rows - m0, plane_x}, Operand{m.b + (int64_t)n0 * ps, (uint32_t)ps, s - n0, plane_s}, s, acc);
  const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) % (WM * WN), group = (threadIdx.x >> 6) / (WM * WN);
  const int wm = wave / WN, wn = wave % WN;
  const int e = g.exps[m.id * (kMaxSteps + 1) + g.k], e1 = LAST ? 12 : g.exps[m.id * (kMaxSteps + 1) + g.k + 1];
  const float f = ldexpf(1.0f, max(e - e1 - 12, -126));
  const int cp = (m.cols + 7) / 8 * 8;
  // a wave's planes leave in whole rows; blocks of several groups hold every other fragment only and store them as they are
  constexpr bool kStaged = !LAST && GROUPS == 1;
  typedef RowStage<uint16_t, W::NI * 16> Rows;
  static_assert(!kStaged || WM * WN * NP * Rows::kBytes <= W::kLds, "the stages fit the tile's LDS");
  char* stage = lds + wave * (NP * Rows::kBytes);
  const int n_wave = n0 + wn * (W::NI * 16);
#pragma unroll
  for (int mi = 0; mi < W::MI; ++mi) {
    const int r0 = m0 + wm * (W::MI * 16) + 16 * mi, r = r0 + (lane & 15);
    if (!kStaged && r >= m.rows) continue;
#pragma unroll
    for (int j = 0; j < W::NI; ++j) {
      if (GROUPS > 1 && (W::MI * j + mi) % GROUPS != group) continue;
      const int n = n_wave + 16 * j + 4 * (lane >> 4);
      if (!kStaged && n >= (LAST ? m.cols : cp)) continue;
      float v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = acc[mi][j][u] * f;
      if constexpr (LAST) {
        write_results(g, m, r, n, v);
      } else if constexpr (kStaged) {
        uint16_t hi[4], lo[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float x = n + u < m.cols ? v[u] : 0.f;
          if constexpr (NP == 2) planes(x, hi[u], lo[u]);
          else hi[u] = f16_bits((_Float16)x);
        }
        Rows::put(stage, lane & 15, n - n_wave, hi);
        if constexpr (NP == 2) Rows::put(stage + Rows::kBytes, lane & 15, n - n_wave, lo);
      } else {
        store_planes<NP>(m.x[(g.k & 1) ^ 1], px, m.cols, r, n, v);
      }
    }
    if constexpr (kStaged) {
      const int rows = max(0, min(16, m.rows - r0)), cols = max(0, cp - n_wave);
      char* o = m.x[(g.k & 1) ^ 1] + (int64_t)r0 * px + n_wave * 2;
      Rows::flush(stage, o, px, rows, cols, lane);
      if constexpr (NP == 2) Rows::flush(stage + Rows::kBytes, o + cp * 2, px, rows, cols, lane);
    }
  }
}

// ---- one block per matrix ------------------------------------------------------------------------------------------
// A matrix whose planes fit a CU's LDS goes through the whole iteration in one launch: X (short side s in rows) and one s x s
// buffer that holds A and then B stay in LDS, fp32 accumulators in registers.  What bounds it is the chain of barriers and LDS
// reads, a few microseconds per step, instead of three launches per step; column strips of X are independent in X <- B X, so a
// wave replaces its strips in place.  64 x 64 f32: 23 us against 73 us by launches.
constexpr int kSmallWaves = 8;
constexpr int kSmallLds = 156 * 1024;

struct SmallShape {
  int sp, lp, px, pa, bytes;  // padded sides, row pitches (bytes) of a plane of X and of A, LDS bytes
};
__host__ __device__ inline SmallShape small_shape(int rows, int cols, int np) {
  SmallShape h;
  const int s = rows < cols ? rows : cols, l = rows < cols ? cols : rows;
  h.sp = (s + 31) / 32 * 32;
  h.lp = (l + 31) / 32 * 32;
  // 32 bytes past a multiple of 128: four rows of a transposed read, and eight of a row read, fall on distinct banks
  h.px = (h.lp * 2 + 127) / 128 * 128 + 32;
  h.pa = (h.sp * 2 + 127) / 128 * 128 + 32;
  h.bytes = h.sp > 128 || h.lp > 4096 ? 1 << 30 : np * h.sp * (h.px + h.pa) + kSmallWaves * 1024 + 512;
  return h;
}

// fragment of 16 rows from row0, K values 32 kk ..: rows contiguous in K
__device__ __forceinline__ i32x4 small_rows(const char* base, int pitch, int row0, int kk, int lane) {
  return *reinterpret_cast<const i32x4*>(base + (row0 + (lane & 15)) * pitch + kk * 64 + (lane >> 4) * 16);
}
// fragment of 16 columns from col0, K = rows 32 kk ..
__device__ __forceinline__ i32x4 small_cols(const char* base, int pitch, int col0, int kk, int lane) {
  const int i = lane & 15, k = kk * 32 + 8 * (lane >> 4) + (i >> 2);
  s16x4 v[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const char* p = base + (k + 4 * h) * pitch + (col0 + 4 * (i & 3)) * 2;
    v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_char*)const_cast<char*>(p));
  }
  const s16x8 w = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(i32x4, w);
}
template <int NP>
__device__ __forceinline__ f32x4 small_mul(const i32x4 (&b)[NP], const i32x4 (&a)[NP], f32x4 c) {
  if constexpr (NP == 2) {
    c = mul<kF16>(b[1], a[0], c);
    c = mul<kF16>(b[0], a[1], c);
  }
  return mul<kF16>(b[0], a[0], c);
}
// KA: 32-row blocks of the short side (1 .. 4)
template <int NP, int KA>
__device__ __forceinline__ void small_matrix(const Group& g, const Mat& m, char* lds) {
  constexpr int T = 2 * KA, U = T * (T + 1) / 2;                                  // 16 x 16 tiles: per side, on and above the diagonal
  constexpr int kSplit = U >= kSmallWaves ? 1 : kSmallWaves / U;                 // waves per tile of the Gram product
  constexpr int kItems = (U + kSmallWaves - 1) / kSmallWaves;
  constexpr int kThreads = 64 * kSmallWaves;
  const int rows = m.rows, cols = m.cols;
  const bool tall = rows > cols;
  const int s = tall ? cols : rows;
  const SmallShape h = small_shape(rows, cols, NP);
  const int xplane = h.sp * h.px, aplane = h.sp * h.pa;
  char* X = lds;
  char* A = X + NP * xplane;
  f32x4* part = reinterpret_cast<f32x4*>(A + NP * aplane);                       // [waves][64]
  double* red = reinterpret_cast<double*>(part + kSmallWaves * 64);              // [waves]
  double* scale_at = red + kSmallWaves;
  int* exps = reinterpret_cast<int*>(scale_at + 1);                              // [kMaxSteps + 1]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  for (int i = tid; i < NP * (xplane + aplane) / 16; i += kThreads) reinterpret_cast<uint4*>(lds)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  // U as it is into X's place (binary32: upper halves in the first plane, lower halves in the second), its sum of squares;
  // eight loads in flight per thread
  const int total = rows * cols;
  double ss = 0.0;
  for (int e0 = tid; e0 < total; e0 += 8 * kThreads) {
    float v[8], mo[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int e = e0 + u * kThreads, r = e / cols, c = e - r * cols;
      v[u] = mo[u] = 0.f;
      if (e < total) {
        if (g.bf16) v[u] = bf16_value(static_cast<const uint16_t*>(m.in)[(int64_t)r * m.ld_in + c]);
        else v[u] = static_cast<const float*>(m.in)[(int64_t)r * m.ld_in + c];
        if (g.muon) mo[u] = m.mom[(int64_t)r * m.ld_mom + c];
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int e = e0 + u * kThreads, r = e / cols, c = e - r * cols;
      if (e >= total) continue;
      if (g.muon) {
        const float mn = fmaf(g.momentum, mo[u], v[u]);
        m.mom[(int64_t)r * m.ld_mom + c] = mn;
        v[u] = g.nesterov ? fmaf(g.momentum, mn, v[u]) : mn;
      }
      ss += (double)v[u] * (double)v[u];
      const uint32_t bits = __float_as_uint(v[u]);
      const int at = (tall ? c : r) * h.px + (tall ? r : c) * 2;
      *reinterpret_cast<uint16_t*>(X + at) = (uint16_t)(bits >> 16);
      if (NP == 2) *reinterpret_cast<uint16_t*>(X + xplane + at) = (uint16_t)bits;
    }
  }
  for (int off = 32; off > 0; off >>= 1) ss += __shfl_xor(ss, off, 64);
  if (lane == 0) red[wave] = ss;
  __syncthreads();
  if (tid == 0) {
    double t = 0.0;
    for (int k = 0; k < kSmallWaves; ++k) t += red[k];
    *scale_at = start_scale(t, g.eps, g.steps, exps);
  }
  __syncthreads();
  const double scale = *scale_at;
  for (int i = tid; i < s * (h.lp / 4); i += kThreads) {  // four neighbours of a row at a time (pads are zero and stay zero, unless NaN)
    const int r = i / (h.lp / 4), at = r * h.px + (i - r * (h.lp / 4)) * 8;
    uint16_t hi[4], lo[4] = {0, 0, 0, 0};
    *reinterpret_cast<uint2*>(hi) = *reinterpret_cast<const uint2*>(X + at);
    if (NP == 2) *reinterpret_cast<uint2*>(lo) = *reinterpret_cast<const uint2*>(X + xplane + at);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float v = (float)((double)__uint_as_float(((uint32_t)hi[u] << 16) | lo[u]) * scale);
      if constexpr (NP == 2) planes(v, hi[u], lo[u]);
      else hi[u] = f16_bits((_Float16)v);
    }
    *reinterpret_cast<uint2*>(X + at) = *reinterpret_cast<const uint2*>(hi);
    if (NP == 2) *reinterpret_cast<uint2*>(X + xplane + at) = *reinterpret_cast<const uint2*>(lo);
  }
  __syncthreads();

  const int strips = h.lp / 16, kx = h.lp / 32;
  // a 16 x 16 tile of a symmetric matrix: four neighbours of row r from column c, and their mirror image
  auto put_tile = [&](int tm, int tn, const f32x4& v) {
    const int r = 16 * tm + (lane & 15), c = 16 * tn + 4 * (lane >> 4);
    uint16_t hi[4], lo[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if constexpr (NP == 2) planes(v[u], hi[u], lo[u]);
      else hi[u] = f16_bits((_Float16)v[u]);
    }
    *reinterpret_cast<uint2*>(A + r * h.pa + c * 2) = *reinterpret_cast<const uint2*>(hi);
    if constexpr (NP == 2) *reinterpret_cast<uint2*>(A + aplane + r * h.pa + c * 2) = *reinterpret_cast<const uint2*>(lo);
    if (tm != tn) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        *reinterpret_cast<uint16_t*>(A + (c + u) * h.pa + r * 2) = hi[u];
        if constexpr (NP == 2) *reinterpret_cast<uint16_t*>(A + aplane + (c + u) * h.pa + r * 2) = lo[u];
      }
    }
  };
  for (int k = 0; k < g.steps; ++k) {
    const int e = exps[k];
    f32x4 acc[kItems];
    // A = X X^T
#pragma unroll
    for (int q = 0; q < kItems; ++q) {
      const int item = wave + q * kSmallWaves;
      acc[q] = f32x4{0, 0, 0, 0};
      if (item >= U * kSplit) continue;
      int tm, tn;
      upper_tile(item % U, T, tm, tn);
      const int p = item / U, k0 = kx * p / kSplit, k1 = kx * (p + 1) / kSplit;
#pragma unroll 4
      for (int kk = k0; kk < k1; ++kk) {
        i32x4 a[NP], b[NP];
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) {
          a[pl] = small_rows(X + pl * xplane, h.px, 16 * tm, kk, lane);
          b[pl] = small_rows(X + pl * xplane, h.px, 16 * tn, kk, lane);
        }
        acc[q] = small_mul<NP>(b, a, acc[q]);
      }
    }
    if constexpr (kSplit > 1) {  // (one item per wave then: the later parts hand theirs to the first)
      part[wave * 64 + lane] = acc[0];
      __syncthreads();
      if (wave < U)
        for (int p = 1; p < kSplit; ++p) acc[0] += part[(wave + p * U) * 64 + lane];
    }
#pragma unroll
    for (int q = 0; q < kItems; ++q) {
      const int item = wave + q * kSmallWaves;
      if (item >= U) continue;
      int tm, tn;
      upper_tile(item, T, tm, tn);
      put_tile(tm, tn, acc[q] * (1.0f / kS));
    }
    __syncthreads();
    // B = a I + b A + c A A, over A
    const float fb = ldexpf(kNsB, 2 * e), fc = ldexpf(kNsC, max(4 * e - 12, -126));
#pragma unroll
    for (int q = 0; q < kItems; ++q) {
      const int item = wave + q * kSmallWaves;
      acc[q] = f32x4{0, 0, 0, 0};
      if (item >= U) continue;
      int tm, tn;
      upper_tile(item, T, tm, tn);
#pragma unroll
      for (int kk = 0; kk < KA; ++kk) {
        i32x4 a[NP], b[NP];
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) {
          a[pl] = small_rows(A + pl * aplane, h.pa, 16 * tm, kk, lane);
          b[pl] = small_rows(A + pl * aplane, h.pa, 16 * tn, kk, lane);
        }
        acc[q] = small_mul<NP>(b, a, acc[q]);
      }
      const int r = 16 * tm + (lane & 15), c = 16 * tn + 4 * (lane >> 4);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float av = (float)*reinterpret_cast<const _Float16*>(A + r * h.pa + (c + u) * 2);
        if (NP == 2) av += (float)*reinterpret_cast<const _Float16*>(A + aplane + r * h.pa + (c + u) * 2);
        acc[q][u] = fmaf(fc, acc[q][u], fb * av) + (r == c + u && r < s ? kNsA * kS : 0.f);
      }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kItems; ++q) {
      const int item = wave + q * kSmallWaves;
      if (item >= U) continue;
      int tm, tn;
      upper_tile(item, T, tm, tn);
      put_tile(tm, tn, acc[q]);
    }
    __syncthreads();
    // X <- B X, a strip of 16 columns at a time
    const bool last = k + 1 == g.steps;
    const float f = ldexpf(1.0f, max(e - (last ? 12 : exps[k + 1]) - 12, -126));
    for (int st = wave; st < strips; st += kSmallWaves) {
      i32x4 x[KA][NP];
#pragma unroll
      for (int kk = 0; kk < KA; ++kk)
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) x[kk][pl] = small_cols(X + pl * xplane, h.px, 16 * st, kk, lane);
      f32x4 y[T];
#pragma unroll
      for (int tm = 0; tm < T; ++tm) {
        y[tm] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < KA; ++kk) {
          i32x4 b[NP];
#pragma unroll
          for (int pl = 0; pl < NP; ++pl) b[pl] = small_rows(A + pl * aplane, h.pa, 16 * tm, kk, lane);
          y[tm] = small_mul<NP>(x[kk], b, y[tm]);
        }
      }
#pragma unroll
      for (int tm = 0; tm < T; ++tm) {
        const int r = 16 * tm + (lane & 15), c = 16 * st + 4 * (lane >> 4);
        if (!last) {
          uint16_t hi[4], lo[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if constexpr (NP == 2) planes(y[tm][u] * f, hi[u], lo[u]);
            else hi[u] = f16_bits((_Float16)(y[tm][u] * f));
          }
          *reinterpret_cast<uint2*>(X + r * h.px + c * 2) = *reinterpret_cast<const uint2*>(hi);
          if constexpr (NP == 2) *reinterpret_cast<uint2*>(X + xplane + r * h.px + c * 2) = *reinterpret_cast<const uint2*>(lo);
        } else if (r < s) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int lr = tall ? c + u : r, lc = tall ? r : c + u;
            if (lr < rows && lc < cols) write_result(g, m, lr, lc, y[tm][u] * f);
          }
        }
      }
    }
    __syncthreads();
  }
}

template <int NP>
__global__ __launch_bounds__(64 * kSmallWaves) void k_ortho_small(Group g) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const Mat& m = g.m[blockIdx.x];
  switch ((min(m.rows, m.cols) + 31) / 32) {
    case 1: small_matrix<NP, 1>(g, m, lds); break;
    case 2: small_matrix<NP, 2>(g, m, lds); break;
    case 3: small_matrix<NP, 3>(g, m, lds); break;
    default: small_matrix<NP, 4>(g, m, lds); break;
  }
}

// ---- short sides up to 16 -------------------------------------------------------------------------------------------
// X_k = P_k X_0 with P_k = B_k .. B_1, and every B is a polynomial of A_0 = X_0 X_0^T: the whole iteration is one of s x s matrices,
// all of which commute, and U is read once and multiplied once.  In doubles throughout: P is large where U is small (3.44^5), so
// P U cancels.  A block per matrix, U in LDS.  Short sides are where the roundings of planes do not average out: 3 x 40 f32 is off by
// 5e-8 here, by 1.6e-6 in two fp16 planes; 16 x 2000 f32: 57 us, against 126 by launches.  Up to 32 the s x s products take longer than the
// matrix pipe's whole iteration (32 x 32: 54 us against 15).
constexpr int kTinyThreads = 512, kTinySide = 16, kTinyValues = 35840;
int tiny_pitch(int l) { return l | 1; }  // odd: the rows of a column fall on distinct banks
bool is_tiny(int rows, int cols) {
  const int s = std::min(rows, cols), l = std::max(rows, cols);
  return s <= kTinySide && (int64_t)s * tiny_pitch(l) <= kTinyValues;
}
constexpr int kTinyFixed = 4 * kTinySide * (kTinySide + 1) * 8, kTinyLds = kTinyFixed + kTinyValues * 4;
static_assert(kTinyLds <= 160 * 1024 && kSmallLds <= 160 * 1024, "a CU's LDS");
int tiny_lds(int s, int l) { return kTinyFixed + s * tiny_pitch(l) * 4; }

__global__ __launch_bounds__(kTinyThreads) void k_ortho_tiny(Group g) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const Mat& m = g.m[blockIdx.x];
  constexpr int S = kTinySide;
  constexpr double kA = 3.4445, kB = -4.7750, kC = 2.0315;  // (binary32's differ by up to 2^-25: more than all the rest)
  constexpr int W = S + 1;                 // row pitch of the s x s matrices: a column falls on distinct banks
  constexpr int R = S / 8;                 // a wave holds the S x S sums as 8 x 8 lanes of R x R
  constexpr int kWaves = kTinyThreads / 64;
  const int rows = m.rows, cols = m.cols, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool tall = rows > cols;
  const int s = tall ? cols : rows, l = tall ? rows : cols, pitch = l | 1;
  double* A = reinterpret_cast<double*>(lds);
  double* B = A + S * W;
  double* P = B + S * W;
  double* T = P + S * W;
  float* U = reinterpret_cast<float*>(T + S * W);
  auto at = [](int i) { return i / S * W + i % S; };  // entry i of the S x S
  for (int i = tid; i < S * S; i += kTinyThreads) {
    A[at(i)] = 0.0;
    P[at(i)] = i / S == i % S ? 1.0 : 0.0;
  }
  // U[i][k]: i the short side; eight loads in flight per thread
  const int total = s * l;
  for (int e0 = tid; e0 < total; e0 += 8 * kTinyThreads) {
    float v[8], mo[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int e = e0 + u * kTinyThreads, r = e / cols, c = e - r * cols;
      v[u] = mo[u] = 0.f;
      if (e < total) {
        if (g.bf16) v[u] = bf16_value(static_cast<const uint16_t*>(m.in)[(int64_t)r * m.ld_in + c]);
        else v[u] = static_cast<const float*>(m.in)[(int64_t)r * m.ld_in + c];
        if (g.muon) mo[u] = m.mom[(int64_t)r * m.ld_mom + c];
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int e = e0 + u * kTinyThreads, r = e / cols, c = e - r * cols;
      if (e >= total) continue;
      if (g.muon) {
        const float mn = fmaf(g.momentum, mo[u], v[u]);
        m.mom[(int64_t)r * m.ld_mom + c] = mn;
        v[u] = g.nesterov ? fmaf(g.momentum, mn, v[u]) : mn;
      }
      U[(tall ? c : r) * pitch + (tall ? r : c)] = v[u];
    }
  }
  __syncthreads();
  {  // U U^T: every wave its columns, then the waves' sums in their order (rows past s repeat the last one and are not used)
    const int i0 = R * (lane >> 3), j0 = R * (lane & 7);
    double acc[R][R];
#pragma unroll
    for (int a = 0; a < R; ++a)
#pragma unroll
      for (int b = 0; b < R; ++b) acc[a][b] = 0.0;
    for (int k = wave; k < l; k += kWaves) {
      double x[R], y[R];
#pragma unroll
      for (int a = 0; a < R; ++a) {
        x[a] = (double)U[min(i0 + a, s - 1) * pitch + k];
        y[a] = (double)U[min(j0 + a, s - 1) * pitch + k];
      }
#pragma unroll
      for (int a = 0; a < R; ++a)
#pragma unroll
        for (int b = 0; b < R; ++b) acc[a][b] = fma(x[a], y[b], acc[a][b]);
    }
    for (int w = 0; w < kWaves; ++w) {
      if (w == wave) {
#pragma unroll
        for (int a = 0; a < R; ++a)
#pragma unroll
          for (int b = 0; b < R; ++b)
            if (i0 + a < s && j0 + b < s) A[(i0 + a) * W + j0 + b] += acc[a][b];
      }
      __syncthreads();
    }
  }
  double sum = 0.0;
  for (int i = 0; i < s; ++i) sum += A[i * W + i];
  const double f = isfinite(sum) ? 1.0 / (sqrt(sum) + (double)g.eps) : (double)NAN;  // anything not finite: the whole result is NaN
  __syncthreads();
  for (int i = tid; i < S * S; i += kTinyThreads) A[at(i)] *= f * f;
  __syncthreads();
  // entry (i0, j0) of a product of two of them by 256 threads (the second factor is symmetric: rows of both)
  static_assert(S * S == 256 && kTinyThreads == 512, "two products at a time");
  const int half = tid >> 8, i0 = (tid & 255) / S, j0 = tid % S, own = i0 * W + j0;
  auto product = [&](const double* x, const double* y) {
    double d = 0.0;
#pragma unroll
    for (int k = 0; k < S; ++k) d = fma(x[i0 * W + k], y[j0 * W + k], d);
    return d;
  };
  for (int step = 0; step < g.steps; ++step) {
    if (half == 0) B[own] = fma(kC, product(A, A), kB * A[own]) + (i0 == j0 ? kA : 0.0);
    __syncthreads();
    const double d = product(half == 0 ? A : P, B);  // A B beside P B
    __syncthreads();
    (half == 0 ? T : P)[own] = d;
    __syncthreads();
    if (half == 0) A[own] = product(T, B);
    __syncthreads();
  }
  for (int k = tid; k < l; k += kTinyThreads) {
    double x[S];
#pragma unroll
    for (int i = 0; i < S; ++i) x[i] = i < s ? (double)U[i * pitch + k] * f : 0.0;
    for (int r = 0; r < s; ++r) {
      double y = 0.0;
#pragma unroll
      for (int i = 0; i < S; ++i) y = fma(P[r * W + i], x[i], y);
      write_result(g, m, tall ? k : r, tall ? r : k, (float)y);
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

size_t mat_bytes(int rows, int cols, int np) {
  const int s = std::min(rows, cols);
  return 2 * up256((size_t)rows * pitch(cols, np)) + 2 * up256((size_t)s * pitch(s, np));
}
size_t head_bytes() { return up256(sizeof(double) * kMaxMats * kNormBlocks) + up256(sizeof(int32_t) * kMaxMats * (kMaxSteps + 1)); }

bool is_small(int rows, int cols, int np) { return is_tiny(rows, cols) || small_shape(rows, cols, np).bytes <= kSmallLds; }

// Planes of a matrix: float32 two.  bfloat16 one, an error (fp16's 2^-11 through the steps) that adds little to the result's own rounding
// -- but on short sides it does not average out: 4 x 400 was 4 times, 96 x 39 1.6 times as far off as that rounding alone, from 128
// on it is 1.3 times at most.  Short sides take two; they are bound by latency.
constexpr int kOnePlaneSide = 128;
int planes_of(int rows, int cols, bool bf16) { return bf16 && std::min(rows, cols) >= kOnePlaneSide ? 1 : 2; }

// The matrices that do not fit one block go through the launches in groups of kMaxMats of the same planes, one group after the
// other in the same workspace
template <class F>
size_t workspace_bytes(int n, int np, bool bf16, F shape) {
  size_t most = 0, b = 0;
  int in_group = 0;
  for (int i = 0; i < n; ++i) {
    if (planes_of(shape(i).first, shape(i).second, bf16) != np || is_small(shape(i).first, shape(i).second, np)) continue;
    if (in_group == kMaxMats) { b = 0; in_group = 0; }
    b += mat_bytes(shape(i).first, shape(i).second, np);
    ++in_group;
    most = std::max(most, b);
  }
  return head_bytes() + most;
}

// What a matrix asks of a launch: its products with A = X X^T, with B from A, and X <- B X
enum Phase : int { kGram, kPoly, kUpdate };
int64_t tiles_of(const Mat& m, Phase p, int bm, int bn) {
  if (p == kUpdate) return ceil_div(m.rows, bm) * ceil_div(m.cols, bn);
  const int64_t T = ceil_div(std::min(m.rows, m.cols), bm);
  return T * (T + 1) / 2;
}
int64_t steps_of(const Mat& m, Phase p, int planes) {
  return ceil_div(p == kGram ? std::max(m.rows, m.cols) : std::min(m.rows, m.cols), planes == 2 ? 32 : 64);
}
double launch_us(double blocks_per_cu, int64_t steps, int planes, int tile, int groups) {
  const double alone = kAlone[planes - 1][tile], share = kShare[planes - 1][tile], per = (double)ceil_div(steps, groups);
  const double on_cu = blocks_per_cu < 6 ? std::ceil(blocks_per_cu) : blocks_per_cu;  // whole blocks per CU while there are few
  return std::max(per * alone, on_cu * per * groups * share) + (groups > 1 ? 2 * alone : 0.0);
}
// Into how many groups of waves the blocks of a matrix's product cut K (Tile::run_split: a step of the block costs a CU as much as
// that many steps of the tile and takes as long as one; about two steps more join the sums): 4 on 64 x 64 tiles, 2 on 96 x 96, 1 on
// any.  Decided by the matrix alone, so that its result does not depend on what else is in the list: the order of the sums of an
// element does not depend on the tile, only on the groups, and symmetric results are computed above the diagonal only.
int groups_of(const Mat& m, Phase p, int planes) {
  const int64_t steps = steps_of(m, p, planes);
  double us = 1e30;
  for (int t = 0; t < kTileIds; ++t) us = std::min(us, launch_us((double)tiles_of(m, p, kTileM[t], kTileN[t]) / kCUs, steps, planes, t, 1));
  const double two = launch_us((double)tiles_of(m, p, 96, 96) / kCUs, steps, planes, kT96, 2);
  const double four = launch_us((double)tiles_of(m, p, 64, 64) / kCUs, steps, planes, kT64, 4);
  // (a microsecond for staying with the other small matrices of a list: a launch of its own costs more)
  return four < us + 1.0 && four <= two + 1.0 ? 4 : two < us * 0.98 ? 2 : 1;
}
// The tile of the ungrouped launches: the smallest estimated time for the whole list
int pick_tile(const Group& g, Phase p, int planes) {
  int best = kT64;
  double us = 1e30;
  for (int t = 0; t < kTileIds; ++t) {
    if (t == kT64x128 && p != kUpdate) continue;
    int64_t tiles = 0, steps = 1;
    for (int i = 0; i < g.n; ++i) {
      tiles += tiles_of(g.m[i], p, kTileM[t], kTileN[t]);
      steps = std::max(steps, steps_of(g.m[i], p, planes));
    }
    const double e = launch_us((double)tiles / kCUs, steps, planes, t, 1);
    if (e < us * 0.98) { us = e; best = t; }
  }
  return best;
}

// `most`: the largest lds of any launch of the kernel, where it depends on the matrices
template <auto kernel>
int launch(Group& g, int grid, int threads, int lds, hipStream_t s, int most = 0) {
  static std::atomic<uint64_t> done{0};
  SUAVE_REQUIRE(most == 0 || lds <= most, "orthogonalize: a launch asks for more LDS than its kernel was allowed");
  SUAVE_CHECK_HIP(allow_lds(reinterpret_cast<const void*>(kernel), most ? most : lds, done));
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), lds, s, g);
  SUAVE_CHECK_HIP(hipGetLastError());
  return 0;
}

template <class F>
int set_begin(Group& g, F blocks) {
  int64_t b = 0;
  for (int i = 0; i < g.n; ++i) {
    g.begin[i] = (int32_t)b;
    b += blocks(g.m[i]);
  }
  g.begin[g.n] = (int32_t)b;
  return (int)b;
}

template <int NP, int POLY, int BM, int WM, int WN, int GROUPS, int PARTS = 1>
int launch_sym_tile(Group& g, hipStream_t s) {
  const int grid = set_begin(g, [](const Mat& m) { return tiles_of(m, kGram, BM, BM); });
  return launch<k_ortho_sym<NP, BM, WM, WN, POLY, GROUPS, PARTS>>(g, grid, 64 * WM * WN * GROUPS, GROUPS * Tile<kF16, NP, false, false, BM, BM, WM, WN>::kLds, s);
}
template <int NP, bool LAST, int BM, int BN, int WM, int WN, int GROUPS>
int launch_update_tile(Group& g, hipStream_t s) {
  const int grid = set_begin(g, [](const Mat& m) { return tiles_of(m, kUpdate, BM, BN); });
  return launch<k_ortho_update<NP, BM, BN, WM, WN, LAST, GROUPS>>(g, grid, 64 * WM * WN * GROUPS,
                                                                  GROUPS * Tile<kF16, NP, false, true, BM, BN, WM, WN>::kLds, s);
}
template <int NP, int POLY>
int launch_sym(Group& g, int groups, hipStream_t s) {
  if (groups == 4) {
    // one block per CU; a list with more of them takes two quarters of K in turn, two blocks per CU (2 x (1024 x 4096) bf16: 272 blocks in
    // 32 us, against 38 with a second round for the last 16)
    int64_t blocks = 0;
    for (int i = 0; i < g.n; ++i) blocks += tiles_of(g.m[i], kGram, 64, 64);
    return blocks > kCUs ? launch_sym_tile<NP, POLY, 64, 2, 2, 2, 2>(g, s) : launch_sym_tile<NP, POLY, 64, 2, 2, 4>(g, s);
  }
  if (groups == 2) return launch_sym_tile<NP, POLY, 96, 2, 2, 2>(g, s);
  switch (pick_tile(g, POLY ? kPoly : kGram, NP)) {
    case kT64: return launch_sym_tile<NP, POLY, 64, 2, 2, 1>(g, s);
    case kT96: return launch_sym_tile<NP, POLY, 96, 2, 2, 1>(g, s);
    case kT128: return launch_sym_tile<NP, POLY, 128, 2, 2, 1>(g, s);
    default: return launch_sym_tile<NP, POLY, 256, 2, 4, 1>(g, s);
  }
}
template <int NP, bool LAST>
int launch_update(Group& g, int groups, hipStream_t s) {
  if (groups == 4) return launch_update_tile<NP, LAST, 64, 64, 2, 2, 4>(g, s);
  if (groups == 2) return launch_update_tile<NP, LAST, 96, 96, 2, 2, 2>(g, s);
  switch (pick_tile(g, kUpdate, NP)) {
    case kT64: return launch_update_tile<NP, LAST, 64, 64, 2, 2, 1>(g, s);
    case kT96: return launch_update_tile<NP, LAST, 96, 96, 2, 2, 1>(g, s);
    case kT64x128: return launch_update_tile<NP, LAST, 64, 128, 2, 2, 1>(g, s);
    case kT128: return launch_update_tile<NP, LAST, 128, 128, 2, 2, 1>(g, s);
    default: return launch_update_tile<NP, LAST, 256, 256, 2, 4, 1>(g, s);
  }
}

template <int NP>
int run_group(Group& g, char* ws, hipStream_t s) {
  g.part = reinterpret_cast<double*>(ws);
  g.exps = reinterpret_cast<int32_t*>(ws + up256(sizeof(double) * kMaxMats * kNormBlocks));
  char* at = ws + head_bytes();
  for (int i = 0; i < g.n; ++i) {
    Mat& m = g.m[i];
    m.id = i;
    const int sh = std::min(m.rows, m.cols);
    for (int k = 0; k < 2; ++k) { m.x[k] = at; at += up256((size_t)m.rows * pitch(m.cols, NP)); }
    m.a = at; at += up256((size_t)sh * pitch(sh, NP));
    m.b = at; at += up256((size_t)sh * pitch(sh, NP));
  }
  int grid = set_begin(g, [](const Mat& m) { return norm_blocks(m.rows, m.cols); });
  hipLaunchKernelGGL(k_ortho_norm, dim3(grid), dim3(256), 0, s, g);
  SUAVE_CHECK_HIP(hipGetLastError());
  grid = set_begin(g, [](const Mat& m) { return std::min<int64_t>(kPackBlocks, std::max<int64_t>(1, ceil_div((int64_t)m.rows * ((m.cols + 7) / 8), 256))); });
  hipLaunchKernelGGL(k_ortho_pack<NP>, dim3(grid), dim3(256), 0, s, g);
  SUAVE_CHECK_HIP(hipGetLastError());
  Group part[3];  // the matrices of a phase by groups 1, 2, 4
  for (int k = 0; k < g.steps; ++k)
    for (Phase p : {kGram, kPoly, kUpdate}) {
      for (int c = 0; c < 3; ++c) {
        part[c] = g;
        part[c].n = 0;
        part[c].k = k;
      }
      for (int i = 0; i < g.n; ++i) {
        Group& to = part[groups_of(g.m[i], p, NP) >> 1];
        to.m[to.n++] = g.m[i];
      }
      for (int c = 0; c < 3; ++c) {
        if (part[c].n == 0) continue;
        const int groups = 1 << c;
        int rc;
        if (p == kGram) rc = launch_sym<NP, 0>(part[c], groups, s);
        else if (p == kPoly) rc = launch_sym<NP, 1>(part[c], groups, s);
        else rc = k + 1 < g.steps ? launch_update<NP, false>(part[c], groups, s) : launch_update<NP, true>(part[c], groups, s);
        if (rc) return rc;
      }
    }
  return 0;
}

// `fill(i, mat)` describes matrix i; `base` holds what the matrices of the call share
template <int NP, class F>
int run_list(int n, const Group& base, F fill, char* ws, hipStream_t s) {
  enum { kTiny, kSmall, kLarge, kKinds };
  Group groups[kKinds] = {base, base, base};
  for (Group& g : groups) g.n = 0;
  auto flush = [&](int kind) {
    Group& g = groups[kind];
    if (g.n == 0) return 0;
    int rc;
    if (kind == kTiny) {
      int lds = 0;
      for (int i = 0; i < g.n; ++i) lds = std::max(lds, tiny_lds(std::min(g.m[i].rows, g.m[i].cols), std::max(g.m[i].rows, g.m[i].cols)));
      rc = launch<k_ortho_tiny>(g, g.n, kTinyThreads, lds, s, kTinyLds);
    } else if (kind == kSmall) {
      int lds = 0;
      for (int i = 0; i < g.n; ++i) lds = std::max(lds, small_shape(g.m[i].rows, g.m[i].cols, NP).bytes);
      rc = launch<k_ortho_small<NP>>(g, g.n, 64 * kSmallWaves, lds, s, kSmallLds);
    } else {
      rc = run_group<NP>(g, ws, s);
    }
    g.n = 0;
    return rc;
  };
  for (int i = 0; i < n; ++i) {
    Mat m{};
    fill(i, m);
    if (planes_of(m.rows, m.cols, base.bf16) != NP) continue;
    const int kind = is_tiny(m.rows, m.cols) ? kTiny : is_small(m.rows, m.cols, NP) ? kSmall : kLarge;
    Group& g = groups[kind];
    g.m[g.n++] = m;
    if (g.n == kMaxMats)
      if (int rc = flush(kind)) return rc;
  }
  for (int kind = 0; kind < kKinds; ++kind)
    if (int rc = flush(kind)) return rc;
  return 0;
}

int check_dims(int32_t rows, int32_t cols) {
  SUAVE_REQUIRE(rows >= 1 && cols >= 1, "orthogonalize: a matrix needs at least one row and one column");
  SUAVE_REQUIRE(std::min(rows, cols) <= 32768 && std::max(rows, cols) <= (1 << 20), "orthogonalize: the sides of a matrix must be at most 32768 (short) and 2^20 (long)");
  return 0;
}
int check_run(int32_t n, int32_t steps, float eps, const void* ws, size_t bytes, size_t need) {
  SUAVE_REQUIRE(n >= 0, "orthogonalize: negative number of matrices");
  SUAVE_REQUIRE(steps >= 1 && steps <= kMaxSteps, "orthogonalize: steps must be in 1..16");
  SUAVE_REQUIRE(eps > 0.f && std::isfinite(eps), "orthogonalize: eps must be positive");
  SUAVE_REQUIRE(n == 0 || (ws && (reinterpret_cast<uintptr_t>(ws) & 255) == 0), "orthogonalize: workspace is null or not 256-byte aligned");
  SUAVE_REQUIRE(bytes >= need || n == 0, "orthogonalize: workspace too small");
  return 0;
}

}  // namespace

int orthogonalize_workspace(const suave_ortho_matrix_t* mats, int32_t n, int32_t dtype, size_t* bytes) {
  SUAVE_REQUIRE(dtype == SUAVE_DTYPE_F32 || dtype == SUAVE_DTYPE_BF16, "orthogonalize: dtype must be SUAVE_DTYPE_F32 or SUAVE_DTYPE_BF16");
  SUAVE_REQUIRE(n >= 0 && (n == 0 || mats) && bytes, "orthogonalize: null argument");
  for (int i = 0; i < n; ++i)
    if (int rc = check_dims(mats[i].rows, mats[i].cols)) return rc;
  const bool bf16 = dtype == SUAVE_DTYPE_BF16;
  auto shape = [&](int i) { return std::make_pair(mats[i].rows, mats[i].cols); };
  *bytes = std::max(workspace_bytes(n, 2, bf16, shape), bf16 ? workspace_bytes(n, 1, bf16, shape) : 0);
  return 0;
}

int launch_orthogonalize(const suave_ortho_matrix_t* mats, int32_t n, int32_t dtype, int32_t steps, float eps, void* ws, size_t ws_bytes, hipStream_t s) {
  size_t need = 0;
  if (int rc = orthogonalize_workspace(mats, n, dtype, &need)) return rc;
  if (int rc = check_run(n, steps, eps, ws, ws_bytes, need)) return rc;
  for (int i = 0; i < n; ++i) {
    SUAVE_REQUIRE(mats[i].in && mats[i].out, "orthogonalize: a matrix is null");
    SUAVE_REQUIRE(mats[i].ld_in >= mats[i].cols && mats[i].ld_out >= mats[i].cols, "orthogonalize: a row stride is shorter than the row");
    for (int j = 0; j < i; ++j)
      SUAVE_REQUIRE(mats[i].out != mats[j].out && mats[i].out != mats[j].in && mats[i].in != mats[j].out, "orthogonalize: an output is another matrix of the list");
  }
  Group base{};
  base.eps = eps; base.steps = steps; base.bf16 = dtype == SUAVE_DTYPE_BF16;
  auto fill = [&](int i, Mat& m) {
    m.in = mats[i].in; m.out = mats[i].out; m.ld_in = mats[i].ld_in; m.ld_out = mats[i].ld_out; m.rows = mats[i].rows; m.cols = mats[i].cols;
  };
  if (int rc = run_list<2>(n, base, fill, static_cast<char*>(ws), s)) return rc;
  return base.bf16 ? run_list<1>(n, base, fill, static_cast<char*>(ws), s) : 0;
}

int muon_workspace(const suave_muon_matrix_t* mats, int32_t n, size_t* bytes) {
  SUAVE_REQUIRE(n >= 0 && (n == 0 || mats) && bytes, "muon_step: null argument");
  for (int i = 0; i < n; ++i)
    if (int rc = check_dims(mats[i].rows, mats[i].cols)) return rc;
  *bytes = workspace_bytes(n, 2, false, [&](int i) { return std::make_pair(mats[i].rows, mats[i].cols); });
  return 0;
}

int launch_muon(const suave_muon_matrix_t* mats, int32_t n, float momentum, int nesterov, float weight_decay, int32_t steps, float eps, void* ws,
                size_t ws_bytes, hipStream_t s) {
  size_t need = 0;
  if (int rc = muon_workspace(mats, n, &need)) return rc;
  if (int rc = check_run(n, steps, eps, ws, ws_bytes, need)) return rc;
  SUAVE_REQUIRE(momentum >= 0.f && momentum < 1.f, "muon_step: momentum must be in [0, 1)");
  SUAVE_REQUIRE(weight_decay >= 0.f && std::isfinite(weight_decay), "muon_step: weight_decay must not be negative");
  for (int i = 0; i < n; ++i) {
    const suave_muon_matrix_t& h = mats[i];
    SUAVE_REQUIRE(h.param && h.grad && h.momentum, "muon_step: param / grad / momentum is null");
    SUAVE_REQUIRE(h.ld_param >= h.cols && h.ld_grad >= h.cols && h.ld_momentum >= h.cols, "muon_step: a row stride is shorter than the row");
    SUAVE_REQUIRE(std::isfinite(h.lr) && h.lr >= 0.f, "muon_step: lr must not be negative");
    SUAVE_REQUIRE(h.param != h.grad && h.param != h.momentum && h.grad != h.momentum, "muon_step: param, grad and momentum must be three matrices");
    for (int j = 0; j < i; ++j) {
      const suave_muon_matrix_t& o = mats[j];
      SUAVE_REQUIRE(h.param != o.param && h.momentum != o.momentum && h.param != o.momentum && h.momentum != o.param,
                    "muon_step: a matrix is in the list twice");
      SUAVE_REQUIRE(h.grad != o.param && h.grad != o.momentum && o.grad != h.param && o.grad != h.momentum,
                    "muon_step: a gradient is another matrix's param or momentum");
    }
  }
  Group base{};
  base.eps = eps; base.steps = steps; base.muon = 1; base.momentum = momentum; base.nesterov = nesterov;
  auto fill = [&](int i, Mat& m) {
    const suave_muon_matrix_t& h = mats[i];
    m.in = h.grad; m.out = h.param; m.mom = h.momentum; m.ld_in = h.ld_grad; m.ld_out = h.ld_param; m.ld_mom = h.ld_momentum;
    m.rows = h.rows; m.cols = h.cols;
    m.lr = (float)((double)h.lr * std::sqrt(std::max(1.0, (double)h.rows / h.cols)));
    m.decay = (float)(1.0 - (double)h.lr * weight_decay);
  };
  return run_list<2>(n, base, fill, static_cast<char*>(ws), s);
}

}  // namespace suave

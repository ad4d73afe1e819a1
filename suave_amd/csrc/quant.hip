// Matrix product in 8-bit integers with a scale per row of either operand (per token and per output channel): the serving
// form of a linear layer.
//
//   s_r = max_k |x_rk| (1/127)   q_rk = rint(x_rk / s_r)     out_rn = s_r w_n sum_k q_rk Q_nk + b_n
//
// k_quantize_rows writes q and s.  The scale is the binary32 product with the binary32 1/127 -- what torch makes of amax / 127.0 on
// the device, so scales laid out with it agree in every bit -- and q the exact nearest integer of
// x / s (ties to even): the quotient by the reciprocal decides except next to a half-integer, where the sign of the exactly
// rounded x - (q +- 1/2) s does; so q does not depend on how the division is evaluated.  A row of zeros has scale 0, a row
// that holds an infinity or a NaN gets that as its scale and q = 0: its outputs are NaN.
//
// The sums are exact int32 (127^2 * 2^17 < 2^31).  Two kernels, by the number of rows:
//  * up to 64 rows and few channels the call is a chain of latencies: k_linear_rows.  A block owns 64 channels, its four waves
//    a quarter of K each; a wave loads the 16 x 64 byte fragments of Q straight into registers (no LDS: nothing is reused)
//    and those of q through L2; the four partial sums meet in LDS.
//  * otherwise the tile product of mma.h: with few rows and many channels 16 x 256 or 64 x 256 tiles, bound by reading Q once;
//    above, square tiles, bound by the matrix pipe or, for short K, by writing the result.
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "mma.h"
#include "tiles.h"

namespace suave {

namespace {

using namespace mma;

struct QuantArgs {
  const void* x;
  int64_t ld;
  int64_t rows;
  int cols;
  int8_t* q;
  int64_t ldq;
  float* scale;
  int vec;  // rows may be read 16 bytes at a time
};

// Adding 1.5 * 2^23 rounds to an integer (ties to even) and leaves it in the low bits.  The quotient by the reciprocal is off
// by at most 127 * 2^-24 < 8e-6: away from a half-integer it decides.
constexpr float kRound = 12582912.0f;
constexpr float kStep = 1.0f / 127.0f;
__device__ __forceinline__ uint32_t quantize_near(float x, float inv, float& off) {
  const float t = fmaf(x, inv, kRound);
  off = fmaxf(off, fabsf(fmaf(x, inv, kRound - t)));
  return __float_as_uint(t);
}
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t ab = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), cd = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
  return __builtin_amdgcn_perm(cd, ab, 0x05040100u);
}
__device__ __forceinline__ uint32_t quantize_exact(float x, float s, float inv) {
  const float k = fminf(fmaxf(rintf(x * inv), -127.f), 127.f);
  const float up = fmaf(-(k + 0.5f), s, x), down = fmaf(-(k - 0.5f), s, x);  // signs are exact: one rounding each
  const int ki = (int)k, odd = ki & 1;
  const int r = ki + ((up > 0.f) | ((up == 0.f) & odd)) - ((down < 0.f) | ((down == 0.f) & odd));
  return (uint32_t)min(max(r, -127), 127);
}

template <class T> __device__ __forceinline__ float as_float(T v);
template <> __device__ __forceinline__ float as_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float as_float<uint16_t>(uint16_t v) { return bf16_value(v); }

template <class T>
__device__ __forceinline__ void load8(const T* row, int k0, int cols, int vec, float (&v)[8]) {  // zeros past the row
  if (vec && k0 + 8 <= cols) {
    constexpr int per = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8 / per; ++i) {
      const uint4 u = *reinterpret_cast<const uint4*>(row + k0 + i * per);
      const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int j = 0; j < per; ++j) v[i * per + j] = as_float<T>(t[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k0 + i < cols ? as_float<T>(row[k0 + i]) : 0.f;
  }
}

// What a row's largest |x| (bits) gives: its scale, and how its values are quantised.  Rows whose scale is next to or below binary32's
// smallest normal number are taken 2^100 times larger, values and scale, which is exact: neither the reciprocal nor the
// residuals leave the range then.  A subnormal scale has few bits -- largest |x| 190 2^-149: 1.496 2^-149 rounds to 2^-149 -- so values
// reach 190 steps there; they saturate at 127.
struct RowScale {
  float scale, s, inv;
  bool tiny, none;  // none: nothing to quantise (zeros, or an infinity or a NaN among them): q = 0
};
__device__ __forceinline__ RowScale row_scale(uint32_t mx) {
  RowScale r;
  r.scale = __uint_as_float(mx) * kStep;
  r.tiny = r.scale < 1e-30f;
  r.s = r.tiny ? r.scale * 0x1p100f : r.scale;
  r.none = mx >= 0x7f800000u || r.s == 0.f;
  r.inv = 1.0f / r.s;
  return r;
}
__device__ __forceinline__ uint2 quantize8(float (&u)[8], const RowScale& r) {
  if (r.none) return make_uint2(0, 0);
  if (r.tiny) {
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] *= 0x1p100f;
  }
  uint32_t k[8];
  float off = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) k[i] = quantize_near(u[i], r.inv, off);
  if (r.tiny || off > 0.49998f) {  // (tiny: quantize_near keeps the low byte of any integer, quantize_exact saturates)
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = quantize_exact(u[i], r.s, r.inv);
  }
  return make_uint2(low_bytes(k[0], k[1], k[2], k[3]), low_bytes(k[4], k[5], k[6], k[7]));
}

// W waves share a row; a lane keeps P runs of 8 values, all loaded at once, and quantises them from its registers.  What a
// row holds beyond W P 512 values is read twice.
template <class T, int W, int P>
__global__ __launch_bounds__(256) void k_quantize_rows(QuantArgs a) {
  __shared__ uint32_t part[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * (4 / W) + wave / W;
  const int t = (wave % W) * 64 + lane;
  constexpr int kRun = W * 64 * 8;
  const bool in = r < a.rows;
  const T* row = static_cast<const T*>(a.x) + (in ? r : 0) * a.ld;
  float v[P][8];
#pragma unroll
  for (int p = 0; p < P; ++p) load8<T>(row, p * kRun + t * 8, a.cols, a.vec, v[p]);
  // |x| as an integer: monotonic, infinity above every number and NaN above infinity, so neither is lost in the maximum
  uint32_t mx = 0;
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(v[p][i]) & 0x7fffffffu);
  for (int k0 = P * kRun + t * 8; k0 < a.cols; k0 += kRun) {
    float u[8];
    load8<T>(row, k0, a.cols, a.vec, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(u[i]) & 0x7fffffffu);
  }
  for (int off = 32; off > 0; off >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, off, 64));
  if constexpr (W > 1) {
    if (lane == 0) part[wave] = mx;
    __syncthreads();
    const int w0 = wave / W * W;
#pragma unroll
    for (int i = 0; i < W; ++i) mx = max(mx, part[w0 + i]);
  }
  if (!in) return;
  const RowScale rs = row_scale(mx);
  if (t == 0) a.scale[r] = rs.scale;
  const int end = (a.cols + 15) / 16 * 16;
  auto write = [&](int k0, float (&u)[8]) { *reinterpret_cast<uint2*>(a.q + r * a.ldq + k0) = quantize8(u, rs); };
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (p * kRun + t * 8 < end) write(p * kRun + t * 8, v[p]);
  for (int k0 = P * kRun + t * 8; k0 < end; k0 += kRun) {
    float u[8];
    load8<T>(row, k0, a.cols, a.vec, u);
    write(k0, u);
  }
}

struct ProductArgs {
  const int8_t* x; int64_t ldx;   // quantised rows [M][ldx], zero from K to the next multiple of 16
  const float* xs;
  const int8_t* w; int64_t ldw;
  const float* ws;
  const float* bias;
  int64_t M;
  int N, K;
  void* out; int64_t ld_out;
  int bf16, vec;   // vec: rows of out may be stored four elements at a time (1), 16 bytes at a time (2)
  int group;
};

__device__ __forceinline__ void store_out(const ProductArgs& a, int64_t m, int n, const float (&v)[4]) {
  if (a.bf16) {
    uint16_t* o = static_cast<uint16_t*>(a.out) + m * a.ld_out + n;
    uint16_t h[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) h[u] = bf16_bits(v[u]);
    if (a.vec && n + 4 <= a.N) *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(h);
    else
      for (int u = 0; u < 4; ++u)
        if (n + u < a.N) o[u] = h[u];
  } else {
    float* o = static_cast<float*>(a.out) + m * a.ld_out + n;
    if (a.vec && n + 4 <= a.N) *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
    else
      for (int u = 0; u < 4; ++u)
        if (n + u < a.N) o[u] = v[u];
  }
}

template <class T>
__global__ __launch_bounds__(T::kThreads, 2) void k_linear_tile(ProductArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int tiles_m = (int)((a.M + T::BM - 1) / T::BM), tiles_n = (a.N + T::BN - 1) / T::BN;
  int tm, tn;
  tile_of(blockIdx.x, gridDim.x, tiles_m, tiles_n, a.group, tm, tn);
  const int64_t m_base = (int64_t)tm * T::BM;
  const int n_base = tn * T::BN;
  const Operand A{reinterpret_cast<const char*>(a.x) + m_base * a.ldx, (uint32_t)a.ldx, (int)min<int64_t>(T::BM, a.M - m_base), 0};
  const Operand B{reinterpret_cast<const char*>(a.w) + (int64_t)n_base * a.ldw, (uint32_t)a.ldw, a.N - n_base, 0};
  typename T::acc_t acc[T::MI][T::NI];
  T::run(lds, A, B, a.K, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / T::WN, wn = wave % T::WN;
  float sw[T::NI][4], b[T::NI][4];
#pragma unroll
  for (int j = 0; j < T::NI; ++j)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int n = n_base + wn * (T::NI * 16) + 16 * j + 4 * (lane >> 4) + u;
      sw[j][u] = n < a.N ? a.ws[n] : 0.f;
      b[j][u] = n < a.N && a.bias ? a.bias[n] : 0.f;
    }
  const int n_wave = n_base + wn * (T::NI * 16);
  typedef RowStage<uint16_t, T::NI * 16> Half;
  typedef RowStage<float, T::NI * 16> Full;
  char* stage = lds + wave * Full::kBytes;
  static_assert(T::WM * T::WN * Full::kBytes <= T::kLds, "the stages fit the tile's LDS");
#pragma unroll
  for (int i = 0; i < T::MI; ++i) {
    const int64_t m0 = m_base + wm * (T::MI * 16) + 16 * i, m = m0 + (lane & 15);
    const float sx = m < a.M ? a.xs[m] : 0.f;
#pragma unroll
    for (int j = 0; j < T::NI; ++j) {
      const int n = n_wave + 16 * j + 4 * (lane >> 4);
      float v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = fmaf((float)acc[i][j][u], sx * sw[j][u], b[j][u]);
      if (a.vec < 2) {
        if (m < a.M && n < a.N) store_out(a, m, n, v);
      } else if (a.bf16) {
        const uint16_t h[4] = {bf16_bits(v[0]), bf16_bits(v[1]), bf16_bits(v[2]), bf16_bits(v[3])};
        Half::put(stage, lane & 15, n - n_wave, h);
      } else {
        Full::put(stage, lane & 15, n - n_wave, v);
      }
    }
    if (a.vec == 2 && m0 < a.M && n_wave < a.N) {
      const int rows = (int)min<int64_t>(16, a.M - m0), cols = a.N - n_wave;
      if (a.bf16) Half::flush(stage, reinterpret_cast<char*>(static_cast<uint16_t*>(a.out) + m0 * a.ld_out + n_wave), a.ld_out * 2, rows, cols, lane);
      else Full::flush(stage, reinterpret_cast<char*>(static_cast<float*>(a.out) + m0 * a.ld_out + n_wave), a.ld_out * 4, rows, cols, lane);
    }
  }
}

constexpr int kRowChannels = 64;

// Rows quantised inside k_linear_rows: a wave per row, 512 values at a time, read a second time (L2) for the rounding
constexpr int kFusedRow = 1024, kFusedValues = 4096;  // longest row, all rows together
template <class T>
__device__ __forceinline__ void quantize_in_block(const QuantArgs& a, char* q, int pitch, float* scale) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int end = (a.cols + 15) / 16 * 16;
  for (int r = wave; r < (int)a.rows; r += 4) {
    const T* row = static_cast<const T*>(a.x) + r * a.ld;
    float v[2][8];
    uint32_t mx = 0;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      load8<T>(row, p * 512 + lane * 8, a.cols, a.vec, v[p]);
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(v[p][i]) & 0x7fffffffu);
    }
    for (int off = 32; off > 0; off >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, off, 64));
    const RowScale rs = row_scale(mx);
    if (lane == 0) scale[r] = rs.scale;
#pragma unroll
    for (int p = 0; p < 2; ++p)
      if (p * 512 + lane * 8 < end) *reinterpret_cast<uint2*>(q + r * pitch + p * 512 + lane * 8) = quantize8(v[p], rs);
  }
}

// MT x 16 rows at most, 64 channels per block.  FUSED: the rows are quantised here, by every block for itself, instead of in a launch
// of their own (1 x 1000 x 256: 14 us a call against 16, host included).
template <int MT, bool FUSED>
__global__ __launch_bounds__(256, 2) void k_linear_rows(ProductArgs a, QuantArgs x_in, int x_bf16) {
  __shared__ int part[4][4][MT * 4 * 64];  // [wave][channel tile][MT x 4 accumulators x lane]
  __shared__ __attribute__((aligned(16))) char fused_q[FUSED ? kFusedValues + 16 * 32 : 16];
  __shared__ float fused_scale[16];
  if constexpr (FUSED) {
    const int pitch = (a.K + 15) / 16 * 16 + 16;
    if (x_bf16) quantize_in_block<uint16_t>(x_in, fused_q, pitch, fused_scale);
    else quantize_in_block<float>(x_in, fused_q, pitch, fused_scale);
    __syncthreads();
    a.ldx = pitch;
  }
  const int8_t* xbase = FUSED ? reinterpret_cast<const int8_t*>(fused_q) : a.x;
  const float* xscale = FUSED ? fused_scale : a.xs;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * kRowChannels;
  const int chunks = (a.K + 15) / 16;                     // 16-byte chunks of a row
  const int steps = (chunks + 3) / 4;                     // 64 bytes of K each
  const int per = (steps + 3) / 4;
  const int s0 = min(wave * per, steps), s1 = min(s0 + per, steps);
  const int8_t* wp[4];
  const int8_t* xp[MT];
#pragma unroll
  for (int j = 0; j < 4; ++j) wp[j] = a.w + (int64_t)min(n0 + 16 * j + r, a.N - 1) * a.ldw;
#pragma unroll
  for (int i = 0; i < MT; ++i) xp[i] = xbase + min<int64_t>(16 * i + r, a.M - 1) * a.ldx;
  i32x4 acc[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  constexpr int U = MT == 1 ? 8 : 4;  // K steps in flight
  for (int s = s0; s < s1; s += U) {
    i32x4 w[U][4], x[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = (s + u) * 4 + g;
      const bool in = s + u < s1 && c < chunks;           // past the row: q is taken as zero, so whatever Q gives does not count
      const int64_t off = (int64_t)(in ? c : 0) * 16;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[u][j] = *reinterpret_cast<const i32x4*>(wp[j] + off);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        x[u][i] = *reinterpret_cast<const i32x4*>(xp[i] + off);
        if (!in) x[u][i] = i32x4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mul<kI8>(w[u][j], x[u][i], acc[i][j]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u) part[wave][j][(i * 4 + u) * 64 + lane] = acc[i][j][u];
  __syncthreads();
  // wave j finishes channel tile j
  const int n = n0 + 16 * wave + 4 * g;
  if (n >= a.N) return;
  float sw[4], b[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    sw[u] = n + u < a.N ? a.ws[n + u] : 0.f;
    b[u] = n + u < a.N && a.bias ? a.bias[n + u] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = 16 * i + r;
    if (m >= a.M) continue;
    const float sx = xscale[m];
    float v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int e = (i * 4 + u) * 64 + lane;
      const int sum = (part[0][wave][e] + part[1][wave][e]) + (part[2][wave][e] + part[3][wave][e]);
      v[u] = fmaf((float)sum, sx * sw[u], b[u]);
    }
    store_out(a, m, n, v);
  }
}

template <class T>
int launch_tile(ProductArgs a, hipStream_t s) {
  const int64_t grid = (a.M + T::BM - 1) / T::BM * ((a.N + T::BN - 1) / T::BN);
  a.group = 8;
  static std::atomic<uint64_t> done{0};
  SUAVE_CHECK_HIP(allow_lds(reinterpret_cast<const void*>(k_linear_tile<T>), T::kLds, done));
  hipLaunchKernelGGL(k_linear_tile<T>, dim3((unsigned)grid), dim3(T::kThreads), T::kLds, s, a);
  SUAVE_CHECK_HIP(hipGetLastError());
  return 0;
}

// A wave per row; four where the rows are few (the chain of one row is then what takes the time) or long
template <class T, int W>
void launch_quantize_w(const QuantArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.rows + 4 / W - 1) / (4 / W)));
  const int runs = (a.cols + W * 512 - 1) / (W * 512);
  if (runs <= 1) hipLaunchKernelGGL((k_quantize_rows<T, W, 1>), grid, dim3(256), 0, s, a);
  else if (runs <= 2) hipLaunchKernelGGL((k_quantize_rows<T, W, 2>), grid, dim3(256), 0, s, a);
  else if (runs <= 4) hipLaunchKernelGGL((k_quantize_rows<T, W, 4>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_quantize_rows<T, W, 8>), grid, dim3(256), 0, s, a);
}
template <class T>
void launch_quantize(QuantArgs a, hipStream_t s) {
  const int64_t rows = a.rows, step = 1 << 23;  // a launch is limited to 2^32 threads
  for (int64_t r = 0; r < rows; r += step) {
    QuantArgs p = a;
    p.x = static_cast<const T*>(a.x) + r * a.ld;
    p.rows = std::min(step, rows - r);
    p.q += r * a.ldq;
    p.scale += r;
    if (rows <= 512 || a.cols > 4096) launch_quantize_w<T, 4>(p, s);
    else launch_quantize_w<T, 1>(p, s);
  }
}

int vec_rows(const void* x, int32_t dtype, int64_t ld) {
  return (ld * (dtype == SUAVE_DTYPE_BF16 ? 2 : 4)) % 16 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

int check_call(const suave_linear_quantized_t* h) {
  SUAVE_REQUIRE(h != nullptr, "linear_quantized: null argument");
  SUAVE_REQUIRE(h->dtype == SUAVE_DTYPE_F32 || h->dtype == SUAVE_DTYPE_BF16, "linear_quantized: dtype must be SUAVE_DTYPE_F32 or SUAVE_DTYPE_BF16");
  SUAVE_REQUIRE(h->n_rows >= 0 && h->n_rows <= (1 << 24), "linear_quantized: n_rows must be in 0..2^24");
  SUAVE_REQUIRE(h->n_in >= 1 && h->n_in <= 131072, "linear_quantized: n_in must be in 1..131072 (exact 32-bit sums)");
  SUAVE_REQUIRE(h->n_out >= 1 && h->n_out <= (1 << 24), "linear_quantized: n_out must be in 1..2^24");
  SUAVE_REQUIRE(h->n_rows * h->n_out <= ((int64_t)1 << 40), "linear_quantized: n_rows * n_out must be at most 2^40");
  SUAVE_REQUIRE(h->ld_x >= h->n_in && h->ld_out >= h->n_out, "linear_quantized: a row stride is shorter than the row");
  SUAVE_REQUIRE(h->ld_weight >= h->n_in && h->ld_weight % 16 == 0 && h->ld_weight <= (1 << 22),
                "linear_quantized: ld_weight must be a multiple of 16, at least n_in and at most 2^22");
  return 0;
}

}  // namespace

int launch_quantize_rows(const void* x, int32_t dtype, int64_t rows, int32_t cols, int64_t ld_x, int8_t* q, int64_t ld_q, float* scale,
                         hipStream_t s) {
  SUAVE_REQUIRE(dtype == SUAVE_DTYPE_F32 || dtype == SUAVE_DTYPE_BF16, "quantize_rows: dtype must be SUAVE_DTYPE_F32 or SUAVE_DTYPE_BF16");
  SUAVE_REQUIRE(rows >= 0 && rows <= (1 << 30), "quantize_rows: rows must be in 0..2^30");
  SUAVE_REQUIRE(cols >= 1 && cols <= (1 << 24), "quantize_rows: cols must be in 1..2^24");
  SUAVE_REQUIRE(ld_x >= cols, "quantize_rows: ld_x < cols");
  SUAVE_REQUIRE(ld_q % 16 == 0 && ld_q >= cols, "quantize_rows: ld_q must be a multiple of 16 and at least cols");
  if (rows == 0) return 0;
  SUAVE_REQUIRE(x && q && scale, "quantize_rows: x / q / scale is null");
  SUAVE_REQUIRE((reinterpret_cast<uintptr_t>(q) & 15) == 0, "quantize_rows: q must be 16-byte aligned");
  QuantArgs a{x, ld_x, rows, cols, q, ld_q, scale, 0};
  a.vec = vec_rows(x, dtype, ld_x);
  if (dtype == SUAVE_DTYPE_BF16) launch_quantize<uint16_t>(a, s);
  else launch_quantize<float>(a, s);
  SUAVE_CHECK_HIP(hipGetLastError());
  return 0;
}

int linear_quantized_workspace(const suave_linear_quantized_t* h, size_t* bytes) {
  if (int rc = check_call(h)) return rc;
  SUAVE_REQUIRE(bytes != nullptr, "linear_quantized: bytes is null");
  *bytes = up256((size_t)h->n_rows * round_up(h->n_in, 16)) + up256(sizeof(float) * h->n_rows);
  return 0;
}

int launch_linear_quantized(const suave_linear_quantized_t* h, hipStream_t s) {
  size_t need = 0;
  if (int rc = linear_quantized_workspace(h, &need)) return rc;
  if (h->n_rows == 0) return 0;
  SUAVE_REQUIRE(h->x && h->weight && h->weight_scale && h->out, "linear_quantized: x / weight / weight_scale / out is null");
  SUAVE_REQUIRE((reinterpret_cast<uintptr_t>(h->weight) & 15) == 0, "linear_quantized: weight must be 16-byte aligned");
  // (few short rows are quantised by every block for itself, while others already write out)
  for (const void* in : {h->x, static_cast<const void*>(h->weight), static_cast<const void*>(h->weight_scale), static_cast<const void*>(h->bias)})
    SUAVE_REQUIRE(h->out != in, "linear_quantized: the output is an input");
  SUAVE_REQUIRE(h->workspace && (reinterpret_cast<uintptr_t>(h->workspace) & 255) == 0, "linear_quantized: workspace is null or not 256-byte aligned");
  SUAVE_REQUIRE(h->workspace_bytes >= need, "linear_quantized: workspace too small (suave_linear_quantized_workspace_bytes)");
  const int ldq = round_up(h->n_in, 16);
  int8_t* q = static_cast<int8_t*>(h->workspace);
  float* xs = reinterpret_cast<float*>(q + up256((size_t)h->n_rows * ldq));
  ProductArgs a{};
  a.x = q; a.ldx = ldq; a.xs = xs; a.w = h->weight; a.ldw = h->ld_weight; a.ws = h->weight_scale; a.bias = h->bias;
  a.M = h->n_rows; a.N = h->n_out; a.K = h->n_in; a.out = h->out; a.ld_out = h->ld_out; a.bf16 = h->dtype == SUAVE_DTYPE_BF16;
  const int per = a.bf16 ? 8 : 4;  // elements of 16 bytes
  a.vec = h->ld_out % per == 0 && (reinterpret_cast<uintptr_t>(h->out) & 15) == 0 ? 2
          : h->ld_out % 4 == 0 && (reinterpret_cast<uintptr_t>(h->out) & (a.bf16 ? 7 : 15)) == 0 ? 1 : 0;
  const unsigned blocks = (unsigned)((h->n_out + kRowChannels - 1) / kRowChannels);
  // Few rows: with 256 channels for half the CUs at least, tiles as low as the batch stream the weights best (16 x 100000 x 2048: 47
  // us against 74 by k_linear_rows, 64 x 100000 x 1000: 38 against 54); with fewer, blocks of 64 channels and K over the waves
  // (1 x 5000 x 4096: 21 us against 29).
  const bool many = (a.N + 255) / 256 >= 128;
  if (a.M <= 16 && !many && a.K <= kFusedRow && a.M * a.K <= kFusedValues) {
    QuantArgs x{h->x, h->ld_x, a.M, a.K, nullptr, 0, nullptr, vec_rows(h->x, h->dtype, h->ld_x)};
    hipLaunchKernelGGL((k_linear_rows<1, true>), dim3(blocks), dim3(256), 0, s, a, x, a.bf16);
    SUAVE_CHECK_HIP(hipGetLastError());
    return 0;
  }
  if (int rc = launch_quantize_rows(h->x, h->dtype, h->n_rows, h->n_in, h->ld_x, q, ldq, xs, s)) return rc;
  if (a.M <= 16 && many) return launch_tile<Tile<kI8, 1, false, false, 16, 256, 1, 4>>(a, s);
  if (a.M <= 64 && many) return launch_tile<Tile<kI8, 1, false, false, 64, 256, 1, 4>>(a, s);
  if (a.M <= 16) hipLaunchKernelGGL((k_linear_rows<1, false>), dim3(blocks), dim3(256), 0, s, a, QuantArgs{}, 0);
  else if (a.M <= 32) hipLaunchKernelGGL((k_linear_rows<2, false>), dim3(blocks), dim3(256), 0, s, a, QuantArgs{}, 0);
  else if (a.M <= 64) hipLaunchKernelGGL((k_linear_rows<4, false>), dim3(blocks), dim3(256), 0, s, a, QuantArgs{}, 0);
  else {
    // the tile with the smallest estimated time
    int best = kT64;
    double us = 1e30;
    for (int t = 0; t < kTileIds; ++t) {
      if (t == kT64x128) continue;
      const Work w{(a.M + kTileM[t] - 1) / kTileM[t] * ((a.N + kTileN[t] - 1) / kTileN[t]), (a.K + 127) / 128, 0.0};
      const int one = 1;
      const double e = estimate_us((TileId)t, 1, &w, &one, 1);
      if (e < us * 0.98) { us = e; best = t; }
    }
    switch (best) {
      case kT64: return launch_tile<Tile<kI8, 1, false, false, 64, 64, 2, 2>>(a, s);
      case kT96: return launch_tile<Tile<kI8, 1, false, false, 96, 96, 2, 2>>(a, s);
      case kT128: return launch_tile<Tile<kI8, 1, false, false, 128, 128, 2, 2>>(a, s);
      default: return launch_tile<Tile<kI8, 1, false, false, 256, 256, 2, 4>>(a, s);
    }
  }
  SUAVE_CHECK_HIP(hipGetLastError());
  return 0;
}

}  // namespace suave

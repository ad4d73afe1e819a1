// Tile product shared by the many-class head (lce.hip), the orthogonalised update (ortho.hip) and the 8-bit integer
// product (quant.hip):  acc[m][n] = sum_k A[m][k] B[n][k]  for one BM x BN tile of a block.
//
// Mathematics: the matrix pipe multiplies bf16, fp16 or int8 fragments into fp32 / int32 accumulators.  A binary32
// operand enters as TWO fp16 planes, x = hi + lo (each 11 bits, round to nearest: |x - hi - lo| <= 2^-24 |x| while the
// caller's power-of-two scale keeps lo clear of fp16's subnormals), and a product is hi hi + hi lo + lo hi: the dropped
// lo lo term is below 2^-24 of the product as well, so the result carries binary32's own error.
//
// Operands come in two storage forms.  "Row" form: [rows][K], K contiguous.  "Column" form: [K][rows], rows contiguous
// (the gradient products read the same stored matrices along their other axis); those fragments are transposed on the
// way out of LDS by ds_read_b64_tr_b16: 16 lanes read 4 k-rows x 16 columns, lane i gets column i.
//
// A K step is 128 bytes per row whatever the type: 64 bf16 / fp16, 32 values in two planes, 128 int8.  Tiles go from
// global memory to LDS directly (buffer_load ... lds, 16 bytes per lane), ST - 1 steps ahead.  The DMA writes lane i
// at base + 16 i, so the bank swizzle is a permutation of the SOURCE chunks: row form slot s of row r holds chunk
// s ^ (r & 7); column form slot s of k-row r holds chunk s ^ (2 (r & 3) [^ 8 ((r >> 3) & 1)]).  Chunks past the edge of an
// operand along K read as zero (an offset beyond the buffer resource's range), rows past the edge are clamped to the
// last one (their products are never written).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace suave {
namespace mma {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

enum Type : int { kBf16 = 0, kF16 = 1, kI8 = 2 };

template <int TYPE> struct Acc { typedef f32x4 type; };
template <> struct Acc<kI8> { typedef i32x4 type; };

// One operand of a tile.  base: the first byte of the tile's first row (row form: at K index k_begin; column form: at
// k-row k_begin).  ld: bytes between stored rows.  rows: valid rows of the tile (row form) / valid bytes of a stored row
// from base (column form, a multiple of 16).  plane: bytes from a hi element to its lo element (two planes only).
struct Operand {
  const char* base;
  uint32_t ld;
  int rows;
  uint32_t plane;
};

constexpr uint32_t kOutside = 0x80000000u;  // any offset >= the resource's range reads zero

__device__ __forceinline__ const char* uniform_ptr(const char* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return reinterpret_cast<const char*>(((uint64_t)hi << 32) | lo);
}

typedef __attribute__((address_space(3))) char lds_char;

__device__ __forceinline__ void dma16(const char* base, uint32_t voff, char* lds) {
  __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, (int)0x80000000u, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds_char*)lds, 16, voff, 0, 0, 0);
}

// The staging of one operand: EXT rows (row form) or columns (column form) of a tile, NP planes, by NW waves.
template <int TYPE, int NP, bool COL, int EXT, int NW>
struct Stage {
  static constexpr int kBytes = EXT * 128;              // LDS bytes of a step
  static constexpr int kInstr = kBytes / 1024;          // wave instructions of a step
  static constexpr int kPer = (kInstr + NW - 1) / NW;   // per wave
  static constexpr int kES = TYPE == kI8 ? 1 : 2;
  static constexpr int kStepK = 128 / NP / kES;         // K elements of a step
  static_assert(!COL || (kES == 2 && EXT >= 64), "column form: 16-bit elements, 64 columns at least");

  static __device__ __forceinline__ uint32_t col_swizzle(int r) { return (2 * (r & 3)) ^ (EXT >= 128 ? 8 * ((r >> 3) & 1) : 0); }

  // source offset of lane's chunk of instruction i (of this wave) for a full step, and whether K-masked: kleft elements remain
  static __device__ __forceinline__ uint32_t offset(const Operand& o, int i, int wave, int lane, int kleft) {
    const int instr = i * NW + wave;
    if constexpr (!COL) {
      const int r = instr * 8 + (lane >> 3);
      const int c = (lane & 7) ^ (r & 7);
      const int pl = NP == 2 ? c >> 2 : 0;
      const uint32_t kb = (uint32_t)(NP == 2 ? c & 3 : c) * 16;
      if ((int)(kb / kES) >= kleft) return kOutside;
      return (uint32_t)min(r, o.rows - 1) * o.ld + kb + (pl ? o.plane : 0u);
    } else {
      const int f = instr * 64 + lane;
      const int r = f / (EXT / 8);  // k-row, planes one behind the other
      const uint32_t c = (uint32_t)(f % (EXT / 8)) ^ col_swizzle(r);
      const int pl = NP == 2 ? r / kStepK : 0;
      const int k = NP == 2 ? r - pl * kStepK : r;
      if (k >= kleft) return kOutside;
      const uint32_t cb = c * 16;
      return (uint32_t)k * o.ld + ((int)cb < o.rows ? cb : 0u) + (pl ? o.plane : 0u);
    }
  }
  static __device__ __forceinline__ uint64_t advance(const Operand& o) {  // bytes from one step to the next
    if constexpr (!COL) return (uint64_t)kStepK * kES;
    else return (uint64_t)kStepK * o.ld;
  }
};

// A fragment: row / column tile index t (16 wide), sub-step kk of 64 bytes per row (one plane) or plane index kk
template <int TYPE, int NP, bool COL, int EXT>
__device__ __forceinline__ i32x4 fragment(const char* lds, int row0, int kk, int lane) {
  if constexpr (!COL) {
    const int r = row0 + (lane & 15);
    const int c = kk * 4 + (lane >> 4);
    return *reinterpret_cast<const i32x4*>(lds + r * 128 + ((c ^ (r & 7)) << 4));
  } else {
    const int i = lane & 15;
    const uint32_t c = (uint32_t)(row0 >> 3) + ((i & 3) >> 1);
    const int k0 = kk * 32 + 8 * (lane >> 4) + (i >> 2);
    s16x4 v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = k0 + 4 * h;
      const uint32_t sw = (2 * (r & 3)) ^ (EXT >= 128 ? 8 * ((r >> 3) & 1) : 0);
      const char* p = lds + r * (EXT * 2) + ((c ^ sw) << 4) + 8 * (i & 1);
      v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_char*)const_cast<char*>(p));
    }
    s16x8 w = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(i32x4, w);
  }
}

template <int TYPE>
__device__ __forceinline__ typename Acc<TYPE>::type mul(i32x4 a, i32x4 b, typename Acc<TYPE>::type c) {
  if constexpr (TYPE == kBf16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else if constexpr (TYPE == kF16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// A block of WM x WN waves computes BM x BN; a wave MI x NI fragments of 16 x 16.  Lane layout of acc[mi][ni]:
// m = wave_m0 + 16 mi + (lane & 15), n = wave_n0 + 16 ni + 4 (lane >> 4) + j: four consecutive n per lane.
template <int TYPE_, int NP_, bool ACOL_, bool BCOL_, int BM_, int BN_, int WM_, int WN_, int ST_>
struct Tile {
  static constexpr int TYPE = TYPE_, NP = NP_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, ST = ST_;
  static constexpr bool ACOL = ACOL_, BCOL = BCOL_;
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  static_assert(MI * WM * 16 == BM && NI * WN * 16 == BN, "whole fragments");
  typedef Stage<TYPE, NP, ACOL, BM, WM * WN> SA;
  typedef Stage<TYPE, NP, BCOL, BN, WM * WN> SB;
  typedef typename Acc<TYPE>::type acc_t;
  static constexpr int kStepK = SA::kStepK;
  static constexpr int kStepBytes = SA::kBytes + SB::kBytes;
  static constexpr int kLds = ST * kStepBytes;
  // DMA instructions a wave has in flight per step (waves that issue fewer simply wait for less)
  static constexpr int kPerStep = SA::kPer + SB::kPer;
  static constexpr bool kEven = SA::kInstr % (WM * WN) == 0 && SB::kInstr % (WM * WN) == 0;

  static __device__ __forceinline__ void load(const Operand& A, const Operand& B, const char* pa, const char* pb, char* lds, int wave, int lane,
                                              const uint32_t (&oa)[SA::kPer], const uint32_t (&ob)[SB::kPer], int kleft) {
    const bool full = kleft >= kStepK;
#pragma unroll
    for (int i = 0; i < SA::kPer; ++i) {
      if (SA::kInstr % (WM * WN) != 0 && i * WM * WN + wave >= SA::kInstr) break;
      dma16(pa, full ? oa[i] : SA::offset(A, i, wave, lane, kleft), lds + (i * WM * WN + wave) * 1024);
    }
#pragma unroll
    for (int i = 0; i < SB::kPer; ++i) {
      if (SB::kInstr % (WM * WN) != 0 && i * WM * WN + wave >= SB::kInstr) break;
      dma16(pb, full ? ob[i] : SB::offset(B, i, wave, lane, kleft), lds + SA::kBytes + (i * WM * WN + wave) * 1024);
    }
  }

  template <int N, int PER>
  static __device__ __forceinline__ void schedule() {  // N times: PER matrix instructions, one LDS read
    if constexpr (N > 0) {
      __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      schedule<N - 1, PER>();
    }
  }
  static __device__ __forceinline__ void step(const char* lds, int wm, int wn, int lane, acc_t (&acc)[MI][NI]) {
    const char* la = lds;
    const char* lb = lds + SA::kBytes;
    const int m0 = wm * (MI * 16), n0 = wn * (NI * 16);
    if constexpr (NP == 1) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        i32x4 b[NI], a[MI];
#pragma unroll
        for (int j = 0; j < NI; ++j) b[j] = fragment<TYPE, NP, BCOL, BN>(lb, n0 + 16 * j, kk, lane);
#pragma unroll
        for (int i = 0; i < MI; ++i) a[i] = fragment<TYPE, NP, ACOL, BM>(la, m0 + 16 * i, kk, lane);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j) acc[i][j] = mul<TYPE>(b[j], a[i], acc[i][j]);
      }
      // issue order: the first sub-step's B fragments and two A fragments, then one fragment read behind every few
      // products (left alone the compiler waits for each A fragment right before its products: 4096^3 bf16 132 -> 116 us,
      // int8 71 -> 64 us; the two-plane form has three products per fragment pair and gains nothing)
      constexpr int ra = ACOL ? 2 : 1, rb = BCOL ? 2 : 1;
      constexpr int head = NI * rb + (MI > 1 ? 2 : 1) * ra, rest = 2 * (NI * rb + MI * ra) - head, mf = 2 * MI * NI;
      constexpr int per = (mf - 4) / rest > 1 ? (mf - 4) / rest : 1;
      __builtin_amdgcn_sched_group_barrier(0x100, head, 0);
      schedule<rest, per>();
      __builtin_amdgcn_sched_group_barrier(0x008, mf, 0);
    } else {  // kk is the plane: row form chunks 0..3 hi, 4..7 lo; column form k-rows 0..31 hi, 32..63 lo
      i32x4 bh[NI], bl[NI];
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        bh[j] = fragment<TYPE, NP, BCOL, BN>(lb, n0 + 16 * j, 0, lane);
        bl[j] = fragment<TYPE, NP, BCOL, BN>(lb, n0 + 16 * j, 1, lane);
      }
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const i32x4 ah = fragment<TYPE, NP, ACOL, BM>(la, m0 + 16 * i, 0, lane);
        const i32x4 al = fragment<TYPE, NP, ACOL, BM>(la, m0 + 16 * i, 1, lane);
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          acc[i][j] = mul<TYPE>(bl[j], ah, acc[i][j]);
          acc[i][j] = mul<TYPE>(bh[j], al, acc[i][j]);
          acc[i][j] = mul<TYPE>(bh[j], ah, acc[i][j]);
        }
      }
    }
  }

  // K elements from the operands' bases.  Every thread of the block takes part; lds: kLds bytes, 16-byte aligned.
  static __device__ __forceinline__ void run(char* lds, Operand A, Operand B, int K, acc_t (&acc)[MI][NI]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = acc_t{0, 0, 0, 0};
    uint32_t oa[SA::kPer], ob[SB::kPer];
#pragma unroll
    for (int i = 0; i < SA::kPer; ++i) oa[i] = SA::offset(A, i, wave, lane, kStepK);
#pragma unroll
    for (int i = 0; i < SB::kPer; ++i) ob[i] = SB::offset(B, i, wave, lane, kStepK);
    const char* pa = uniform_ptr(A.base);
    const char* pb = uniform_ptr(B.base);
    const uint64_t da = SA::advance(A), db = SB::advance(B);
    const int steps = (K + kStepK - 1) / kStepK;
    int issued = 0;
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) {
      if (s < steps) {
        load(A, B, pa, pb, lds + s * kStepBytes, wave, lane, oa, ob, K - s * kStepK);
        pa += da; pb += db; ++issued;
      }
    }
    for (int s = 0; s < steps; ++s) {
      // step s has landed when at most the steps issued behind it are still in flight
      if (ST == 2 || !kEven || s + ST - 1 > steps) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      else if constexpr (ST == 3) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kPerStep) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kPerStep) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (issued < steps) {  // into the slot that step s - 1 has left (all waves are past it: the barrier above)
        load(A, B, pa, pb, lds + (issued % ST) * kStepBytes, wave, lane, oa, ob, K - issued * kStepK);
        pa += da; pb += db; ++issued;
      }
      step(lds + (s % ST) * kStepBytes, wm, wn, lane, acc);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's reads of the slot are done before the next barrier
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
};

// Block -> tile: the blocks an XCD gets (every eighth) walk one contiguous range of tiles, `group` row tiles side by side
// within it, so that the operand panels a die's L2 holds are shared by its blocks in flight.
__device__ __forceinline__ void tile_of(int b, int n_blocks, int tiles_m, int tiles_n, int group, int& tm, int& tn) {
  const int q = n_blocks / 8, r = n_blocks % 8, x = b % 8, i = b / 8;
  const int t = x * q + min(x, r) + i;
  const int per = group * tiles_n, g = t / per, rem = t - g * per;
  const int gm = min(group, tiles_m - g * group);
  tm = g * group + rem % gm;
  tn = rem / gm;
}

__device__ __forceinline__ uint16_t bf16_bits(float x) {
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}
__device__ __forceinline__ float bf16_value(uint16_t u) { return __builtin_bit_cast(float, (uint32_t)u << 16); }
__device__ __forceinline__ uint16_t f16_bits(_Float16 x) { return __builtin_bit_cast(uint16_t, x); }
// hi and lo planes of x; an infinite hi keeps lo zero
__device__ __forceinline__ void planes(float x, uint16_t& hi, uint16_t& lo) {
  const _Float16 h = (_Float16)x;
  const float r = x - (float)h;
  hi = f16_bits(h);
  lo = __builtin_isinf((float)h) ? 0 : f16_bits((_Float16)r);
}

}  // namespace mma
}  // namespace suave

// Tile product shared by the many-class head (lce.hip), the orthogonalised update (ortho.hip) and the 8-bit integer
// product (quant.hip):  acc[m][n] = sum_k A[m][k] B[n][k]  for one BM x BN tile of a block.
//
// Mathematics: the matrix pipe multiplies bf16, fp16 or int8 fragments into fp32 / int32 accumulators.  A binary32
// operand enters as TWO fp16 planes of 11 bits, x = hi + lo, each rounded to nearest.  For 2^e <= |x| < 2^(e+1): |x - hi| <= 2^(e-11), so lo
// is off by 2^(e-23) at most and |x - hi - lo| <= 2^-23 |x|.  That takes |x| >= 1/4; below it lo is subnormal and off by up to 2^-25 whatever
// x is, which the caller's power-of-two scale keeps far below its largest values.  A product is hi hi + hi lo + lo hi; the dropped lo lo is
// at most 2^-22 of it.  These are worst cases of single products, 2 to 4 times binary32's; they have either sign, and a sum of many
// is off by what binary32's own rounding of it is off by.
//
// Operands come in two storage forms.  "Row" form: [rows][K], K contiguous.  "Column" form: [K][rows], rows contiguous
// (the gradient products read the same stored matrices along their other axis); those fragments are transposed on the
// way out of LDS by ds_read_b64_tr_b16: 16 lanes read 4 k-rows x 16 columns, lane i gets column i.
//
// A K step is 128 bytes per row whatever the type: 64 bf16 / fp16, 32 values in two planes, 128 int8.  Tiles go from
// global memory to LDS directly (buffer_load ... lds, 16 bytes per lane), into two slots.  The DMA writes lane i
// at base + 16 i, so the bank swizzle is a permutation of the SOURCE chunks: row form slot s of row r holds chunk
// s ^ (r & 7), column form by col_chunk.  Chunks past the edge of an
// operand along K read as zero (an offset beyond the buffer resource's range), rows past the edge are clamped to the
// last one (their products are never written).
//
// What it reaches (256 x 256 tile, eight waves, 8192 x 8192 x 4096, stores of the fp32 result included): bf16 1200 TFLOP/s, int8 1950,
// two fp16 planes 1510 of their three products; a library product reaches 1400 / 2160 / 1490 on this card.  Matrix pipe busy 61 %
// (bf16) and 69 % (planes) of the cycles at the 2.0 - 2.2 GHz it runs at under this load; the rest is the feed: without the
// transfers the bf16 loop runs at 1530, with every transfer hitting L2 at 1280.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

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

// Column form, k-row r: the chunk in a slot, and the slot of a chunk.  Rows of 64 and of n 128 columns start on the same bank: the
// four rows of a transposed read are set apart by exchanging pairs of chunks.  Rows of 96 columns (192 bytes) alternate
// between two halves of the banks by themselves; every second pair of rows is turned by one pair of chunks.
template <int EXT>
__device__ __forceinline__ uint32_t col_chunk(uint32_t slot, int r) {
  if constexpr (EXT == 96) return r & 2 ? (slot < 2 ? slot + 10 : slot - 2) : slot;
  else return slot ^ (2 * (r & 3)) ^ (EXT >= 128 ? 8 * ((r >> 3) & 1) : 0);
}
template <int EXT>
__device__ __forceinline__ uint32_t col_slot(uint32_t chunk, int r) {
  if constexpr (EXT == 96) return r & 2 ? (chunk < 10 ? chunk + 2 : chunk - 10) : chunk;
  else return chunk ^ (2 * (r & 3)) ^ (EXT >= 128 ? 8 * ((r >> 3) & 1) : 0);
}

constexpr uint32_t kOutside = 0x80000000u;  // any offset >= the resource's range reads zero

__device__ __forceinline__ const char* uniform_ptr(const char* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return reinterpret_cast<const char*>(((uint64_t)hi << 32) | lo);
}

typedef __attribute__((address_space(3))) char lds_char;

__device__ __forceinline__ i32x4 resource(const char* base) {  // raw buffer of 2^31 bytes from base
  const uint64_t v = reinterpret_cast<uint64_t>(base);
  return i32x4{(int)(uint32_t)v, (int)((uint32_t)(v >> 32) & 0xffffu), (int)0x80000000u, 0x00020000};
}
__device__ __forceinline__ uint32_t lds_offset(const char* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const lds_char*)p);
}
// 16 bytes per lane from base + voff to LDS at lds + 16 lane.
__device__ __forceinline__ void dma16_scheduled(const char* base, uint32_t voff, char* lds) {
  __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, (int)0x80000000u, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds_char*)lds, 16, voff, 0, 0, 0);
}
// The same, written as an instruction because the compiler, which would
// otherwise know of the transfer, waits for ALL transfers before any transposed LDS read (8192 x 8192 x 4096 bf16 with a
// column-form operand: 569 us, against 457 us).  It has no result register; callers wait by vmcnt and a barrier before the LDS is read.
// The wait states cover m0 and a resource that a vector instruction has just written; m0 is given back as it was.
__device__ __forceinline__ void dma16(i32x4 rsrc, uint32_t voff, uint32_t lds) {
  uint32_t keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "s"(lds), "v"(voff), "s"(rsrc));
}

// The staging of one operand: EXT rows (row form) or columns (column form) of a tile, NP planes, by NW waves.
template <int TYPE, int NP, bool COL, int EXT, int NW>
struct Stage {
  static constexpr int kBytes = EXT * 128;              // LDS bytes of a step
  static constexpr int kInstr = kBytes / 1024;          // wave instructions of a step
  static constexpr int kPer = (kInstr + NW - 1) / NW;   // per wave
  static constexpr int kES = TYPE == kI8 ? 1 : 2;
  static constexpr int kStepK = 128 / NP / kES;         // K elements of a step
  static_assert(!COL || (kES == 2 && (EXT == 64 || EXT == 96 || EXT % 128 == 0)), "column form: 16-bit elements, 64, 96 or n 128 columns");

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
      const uint32_t c = col_chunk<EXT>(f % (EXT / 8), r);
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
      const char* p = lds + r * (EXT * 2) + (col_slot<EXT>(c, r) << 4) + 8 * (i & 1);
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
template <int TYPE_, int NP_, bool ACOL_, bool BCOL_, int BM_, int BN_, int WM_, int WN_>
struct Tile {
  static constexpr int TYPE = TYPE_, NP = NP_, BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr bool ACOL = ACOL_, BCOL = BCOL_;
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  static_assert(MI * WM * 16 == BM && NI * WN * 16 == BN, "whole fragments");
  typedef Stage<TYPE, NP, ACOL, BM, WM * WN> SA;
  typedef Stage<TYPE, NP, BCOL, BN, WM * WN> SB;
  typedef typename Acc<TYPE>::type acc_t;
  static constexpr int kStepK = SA::kStepK;
  static constexpr int kStepBytes = SA::kBytes + SB::kBytes;
  static constexpr int kLds = 2 * kStepBytes;
  static constexpr int kPerStep = SA::kPer + SB::kPer;  // DMA instructions of a wave and step
  static constexpr bool kEven = SA::kInstr % (WM * WN) == 0 && SB::kInstr % (WM * WN) == 0;

  // DMA instruction i (of kPerStep) of this wave
  template <int I>
  static __device__ __forceinline__ void dma(i32x4 ra, i32x4 rb, uint32_t lds, int wave, const uint32_t (&oa)[SA::kPer], const uint32_t (&ob)[SB::kPer]) {
    if constexpr (I < SA::kPer) {
      if (SA::kInstr % (WM * WN) == 0 || I * WM * WN + wave < SA::kInstr) dma16(ra, oa[I], lds + (I * WM * WN + wave) * 1024);
    } else if constexpr (I < kPerStep) {
      constexpr int J = I - SA::kPer;
      if (SB::kInstr % (WM * WN) == 0 || J * WM * WN + wave < SB::kInstr) dma16(rb, ob[J], lds + SA::kBytes + (J * WM * WN + wave) * 1024);
    }
  }
  template <int I0, int I1>
  static __device__ __forceinline__ void dmas(i32x4 ra, i32x4 rb, uint32_t lds, int wave, const uint32_t (&oa)[SA::kPer], const uint32_t (&ob)[SB::kPer]) {
    if constexpr (I0 < I1) {
      dma<I0>(ra, rb, lds, wave, oa, ob);
      dmas<I0 + 1, I1>(ra, rb, lds, wave, oa, ob);
    }
  }
  static __device__ __forceinline__ void offsets(const Operand& A, const Operand& B, int wave, int lane, int kleft, uint32_t (&oa)[SA::kPer],
                                                 uint32_t (&ob)[SB::kPer]) {
#pragma unroll
    for (int i = 0; i < SA::kPer; ++i) oa[i] = SA::offset(A, i, wave, lane, kleft);
#pragma unroll
    for (int i = 0; i < SB::kPer; ++i) ob[i] = SB::offset(B, i, wave, lane, kleft);
  }

  struct Frags { i32x4 b[NI], a[MI]; };
  // fragment q of a half step (one plane: kk the half, two planes: kk the plane): B's NI first, then A's MI
  static __device__ __forceinline__ void read(const char* lds, int wm, int wn, int kk, int lane, int q, Frags& f) {
    if (q < NI) f.b[q] = fragment<TYPE, NP, BCOL, BN>(lds + SA::kBytes, wn * (NI * 16) + 16 * q, kk, lane);
    else f.a[q - NI] = fragment<TYPE, NP, ACOL, BM>(lds, wm * (MI * 16) + 16 * (q - NI), kk, lane);
  }
  static __device__ __forceinline__ void read_all(const char* lds, int wm, int wn, int kk, int lane, Frags& f) {
#pragma unroll
    for (int q = 0; q < NI + MI; ++q) read(lds, wm, wn, kk, lane, q, f);
  }

  // Half a step: the products of `now`, while the other half (or the next step's first) is read into `then` and, if DMA, a step's
  // DMA is issued.  A wave issues in order: DMA instructions in a row fill the address unit's queue and hold up the products
  // behind them, and a fragment read right before its products is waited for.  So each of the MI groups of products is followed
  // by its share of both, and the compiler may not move them across (8192 x 8192 x 4096 bf16: transfers in a row and one barrier
  // in front of each step 490 us, this 450 us; the transfers in front of the products 456 us).
  template <int I, bool DMA>
  static __device__ __forceinline__ void half(const char* lds, int wm, int wn, int kk, int lane, const Frags& now, Frags& then, acc_t (&acc)[MI][NI],
                                              i32x4 ra, i32x4 rb, uint32_t slot, int wave, const uint32_t (&oa)[SA::kPer], const uint32_t (&ob)[SB::kPer]) {
    if constexpr (I < MI) {
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[I][j] = mul<TYPE>(now.b[j], now.a[I], acc[I][j]);
#pragma unroll
      for (int q = (I * (NI + MI) + MI - 1) / MI; q < ((I + 1) * (NI + MI) + MI - 1) / MI; ++q) read(lds, wm, wn, kk, lane, q, then);
      if constexpr (DMA) dmas<I * kPerStep / MI, (I + 1) * kPerStep / MI>(ra, rb, slot, wave, oa, ob);
      __builtin_amdgcn_sched_barrier(0);
      half<I + 1, DMA>(lds, wm, wn, kk, lane, now, then, acc, ra, rb, slot, wave, oa, ob);
    }
  }
  // Two planes: a step's fragments (row form chunks 0..3 hi, 4..7 lo; column form k-rows 0..31 hi, 32..63 lo), three products
  // for each pair.  The transfers of the next step are placed by the compiler: the reads of this step all come first or
  // between its products, so nothing waits for a transfer before the next turn.
  static __device__ __forceinline__ void planes_load(const char* pa, const char* pb, char* lds, int wave, const uint32_t (&oa)[SA::kPer],
                                                     const uint32_t (&ob)[SB::kPer]) {
#pragma unroll
    for (int i = 0; i < SA::kPer; ++i)
      if (SA::kInstr % (WM * WN) == 0 || i * WM * WN + wave < SA::kInstr) dma16_scheduled(pa, oa[i], lds + (i * WM * WN + wave) * 1024);
#pragma unroll
    for (int i = 0; i < SB::kPer; ++i)
      if (SB::kInstr % (WM * WN) == 0 || i * WM * WN + wave < SB::kInstr)
        dma16_scheduled(pb, ob[i], lds + SA::kBytes + (i * WM * WN + wave) * 1024);
  }
  static __device__ __forceinline__ void planes_step(const char* lds, int wm, int wn, int lane, acc_t (&acc)[MI][NI]) {
    Frags h, l;
    read_all(lds, wm, wn, 0, lane, h);
    read_all(lds, wm, wn, 1, lane, l);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        acc[i][j] = mul<TYPE>(l.b[j], h.a[i], acc[i][j]);
        acc[i][j] = mul<TYPE>(h.b[j], l.a[i], acc[i][j]);
        acc[i][j] = mul<TYPE>(h.b[j], h.a[i], acc[i][j]);
      }
  }
  // issue order of a planes step: B's and the first two A fragments, then the other reads and the transfers spread evenly
  // between the products
  template <int I, int M, int D, int V>
  static __device__ __forceinline__ void spread() {
    if constexpr (I < M) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if constexpr ((I + 1) * D / M > I * D / M) __builtin_amdgcn_sched_group_barrier(0x100, (I + 1) * D / M - I * D / M, 0);
      if constexpr ((I + 1) * V / M > I * V / M) __builtin_amdgcn_sched_group_barrier(0x010, (I + 1) * V / M - I * V / M, 0);
      spread<I + 1, M, D, V>();
    }
  }
  static __device__ __forceinline__ void planes_order() {
    constexpr int da_reads = 2 * MI * (ACOL ? 2 : 1), db_reads = 2 * NI * (BCOL ? 2 : 1), first = db_reads + da_reads / MI * (MI > 1 ? 2 : 1);
    __builtin_amdgcn_sched_group_barrier(0x100, first, 0);
    spread<0, 3 * MI * NI, da_reads + db_reads - first, kEven ? kPerStep : 0>();
    __builtin_amdgcn_sched_barrier(0);
  }
  // one plane, a whole step: its fragments, then `transfers` (behind the reads: the compiler lets a transposed read wait for
  // earlier transfers), then its products
  template <class F>
  static __device__ __forceinline__ void both_halves(const char* lds, int wm, int wn, int lane, acc_t (&acc)[MI][NI], F transfers) {
    Frags f[2];
    read_all(lds, wm, wn, 0, lane, f[0]);
    read_all(lds, wm, wn, 1, lane, f[1]);
    transfers();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = mul<TYPE>(f[kk].b[j], f[kk].a[i], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  }
  static __device__ __forceinline__ void turn() {  // this wave's DMA has landed and its LDS reads are done; then everybody's
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }

  // For products of few tiles, whose time is the chain of K steps: K is cut into GROUPS x PARTS ranges of `per` steps, the block has
  // GROUPS times the waves of a tile, and group g takes PARTS neighbouring ranges, one after the other, in LDS of its own (kLds bytes
  // each, at lds); the partial sums meet in LDS.  Every group walks `per` steps of a range, those past K as zeros, so all waves
  // pass the same barriers.  On return acc holds the whole sums of this group's share of the fragments: those with
  // (MI j + i) % GROUPS == g.  The ranges are added in their order, so the result depends on GROUPS x PARTS only.
  template <int GROUPS, int PARTS>
  static __device__ __forceinline__ void run_split(char* lds, Operand A, Operand B, int K, acc_t (&acc)[MI][NI]) {
    const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = all / (WM * WN), wave = all % (WM * WN);
    const int wm = wave / WN, wn = wave % WN;
    const int steps = (K + kStepK - 1) / kStepK, per = (steps + GROUPS * PARTS - 1) / (GROUPS * PARTS);
    char* mine = lds + group * kLds;
    acc_t sum[PARTS][MI][NI];
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) sum[part][i][j] = acc_t{0, 0, 0, 0};
      const int first = (group * PARTS + part) * per;
      const char* pa = uniform_ptr(A.base + SA::advance(A) * first);
      const char* pb = uniform_ptr(B.base + SB::advance(B) * first);
      uint32_t oa[SA::kPer], ob[SB::kPer];
      auto load = [&](int s) {
        planes_load(pa + SA::advance(A) * s, pb + SB::advance(B) * s, mine + (s & 1) * kStepBytes, wave, oa, ob);
      };
      if (part > 0) turn();  // the last step of the range before is read
      offsets(A, B, wave, lane, K - first * kStepK, oa, ob);
      load(0);
      // steps that lie inside K for every group come first: their transfers need no masks and are spread between the products
      const int whole = min(per, max(0, K / kStepK - ((GROUPS - 1) * PARTS + part) * per));
      int s = 0;
      if (whole > 1) offsets(A, B, wave, lane, kStepK, oa, ob);
      for (; s + 1 < whole; ++s) {
        turn();
        if constexpr (NP == 2) {
          planes_step(mine + (s & 1) * kStepBytes, wm, wn, lane, sum[part]);
          load(s + 1);
          planes_order();
        } else {
          both_halves(mine + (s & 1) * kStepBytes, wm, wn, lane, sum[part], [&] { load(s + 1); });
        }
      }
      for (; s < per; ++s) {
        turn();
        auto next = [&] {
          if (s + 1 < per) {
            offsets(A, B, wave, lane, K - (first + s + 1) * kStepK, oa, ob);
            load(s + 1);
          }
        };
        if constexpr (NP == 2) {
          planes_step(mine + (s & 1) * kStepBytes, wm, wn, lane, sum[part]);
          next();
        } else {
          both_halves(mine + (s & 1) * kStepBytes, wm, wn, lane, sum[part], next);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    turn();
    acc_t* sums = reinterpret_cast<acc_t*>(lds);  // [range][wave][fragment][lane]
    static_assert(WM * WN * MI * NI * 64 * 16 * PARTS <= kLds, "the partial sums fit the groups' slots");
    auto at = [&](int range, int i, int j) { return ((range * WM * WN + wave) * MI * NI + MI * j + i) * 64 + lane; };
#pragma unroll
    for (int part = 0; part < PARTS; ++part)
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) sums[at(group * PARTS + part, i, j)] = sum[part][i][j];
    turn();
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        acc[i][j] = acc_t{0, 0, 0, 0};
        if ((MI * j + i) % GROUPS != group) continue;
#pragma unroll
        for (int r = 0; r < GROUPS * PARTS; ++r) acc[i][j] += sums[at(r, i, j)];
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
    const int steps = (K + kStepK - 1) / kStepK;
    if (steps == 0) return;
    uint32_t oa[SA::kPer], ob[SB::kPer];
    offsets(A, B, wave, lane, steps > 1 ? kStepK : K, oa, ob);
    const char* pa = uniform_ptr(A.base);
    const char* pb = uniform_ptr(B.base);
    const uint64_t da = SA::advance(A), db = SB::advance(B);
    const uint32_t slot0 = lds_offset(lds);
    int s = 0;
    if constexpr (NP == 1) {
      dmas<0, kPerStep>(resource(pa), resource(pb), slot0, wave, oa, ob);
      // The slot of step s is free as soon as every wave holds its second half in registers, so there is ONE barrier per step,
      // in the middle of its products: behind it the DMA of step s + 2 starts and the first half of step s + 1 is read while
      // the second half of step s is multiplied.  No product waits for LDS, and a DMA has a whole step to land.
      if (steps > 1) {
        pa += da; pb += db;
        if (steps == 2) offsets(A, B, wave, lane, K - kStepK, oa, ob);
        dmas<0, kPerStep>(resource(pa), resource(pb), slot0 + kStepBytes, wave, oa, ob);
      }
      if (kEven && steps > 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kPerStep) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      Frags f0, f1;
      read_all(lds, wm, wn, 0, lane, f0);
      __builtin_amdgcn_sched_barrier(0);
      for (; s < steps - 3; ++s) {
        half<0, false>(lds + (s & 1) * kStepBytes, wm, wn, 1, lane, f0, f1, acc, i32x4{}, i32x4{}, 0, wave, oa, ob);
        turn();
        pa += da; pb += db;
        half<0, true>(lds + (~s & 1) * kStepBytes, wm, wn, 0, lane, f1, f0, acc, resource(pa), resource(pb), slot0 + (s & 1) * kStepBytes, wave, oa, ob);
      }
      for (; s < steps - 1; ++s) {  // the last step may be short: its chunks past K are masked
        half<0, false>(lds + (s & 1) * kStepBytes, wm, wn, 1, lane, f0, f1, acc, i32x4{}, i32x4{}, 0, wave, oa, ob);
        turn();
        if (s + 2 < steps) {
          pa += da; pb += db;
          offsets(A, B, wave, lane, K - (s + 2) * kStepK, oa, ob);
          dmas<0, kPerStep>(resource(pa), resource(pb), slot0 + (s & 1) * kStepBytes, wave, oa, ob);
        }
        half<0, false>(lds + (~s & 1) * kStepBytes, wm, wn, 0, lane, f1, f0, acc, i32x4{}, i32x4{}, 0, wave, oa, ob);
      }
      half<0, false>(lds + (s & 1) * kStepBytes, wm, wn, 1, lane, f0, f1, acc, i32x4{}, i32x4{}, 0, wave, oa, ob);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = mul<TYPE>(f1.b[j], f1.a[i], acc[i][j]);
    } else {
      planes_load(pa, pb, lds, wave, oa, ob);
      for (; s < steps - 2; ++s) {
        turn();
        pa += da; pb += db;
        planes_step(lds + (s & 1) * kStepBytes, wm, wn, lane, acc);
        planes_load(pa, pb, lds + (~s & 1) * kStepBytes, wave, oa, ob);
        planes_order();
      }
      for (; s < steps; ++s) {  // the last step may be short: its chunks past K are masked
        turn();
        if (s + 1 < steps) {
          pa += da; pb += db;
          offsets(A, B, wave, lane, K - (s + 1) * kStepK, oa, ob);
          planes_load(pa, pb, lds + (~s & 1) * kStepBytes, wave, oa, ob);
        }
        planes_step(lds + (s & 1) * kStepBytes, wm, wn, lane, acc);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();  // the caller may reuse the LDS
    asm volatile("" ::: "memory");
  }
};

// Block -> tile: the blocks an XCD gets (every eighth) walk one contiguous range of tiles, `group` row tiles side by side
// within it, so that the operand panels a die's L2 holds are shared by its blocks in flight.
__device__ __forceinline__ int die_order(int b, int n_blocks) {
  const int q = n_blocks / 8, r = n_blocks % 8, x = b % 8, i = b / 8;
  return x * q + min(x, r) + i;
}
__device__ __forceinline__ void tile_of(int b, int n_blocks, int tiles_m, int tiles_n, int group, int& tm, int& tn) {
  const int t = die_order(b, n_blocks);
  const int per = group * tiles_n, g = t / per, rem = t - g * per;
  const int gm = min(group, tiles_m - g * group);
  tm = g * group + rem % gm;
  tn = rem / gm;
}

// Eight neighbours in 16-byte loads, wherever the row begins (the memory system takes them at element alignment)
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x8_any __attribute__((ext_vector_type(8), aligned(2)));
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const f32x4_any a = *reinterpret_cast<const f32x4_any*>(p), b = *reinterpret_cast<const f32x4_any*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
__device__ __forceinline__ void load8(const uint16_t* p, uint16_t (&v)[8]) {
  const u16x8_any a = *reinterpret_cast<const u16x8_any*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = a[i];
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

// Rows of a wave's tile leave through LDS: a lane holds four neighbours of one row (8 bytes of 16-bit values), stored as they are a
// wave instruction touches 16 rows by 32 bytes.  Staged 16 rows at a time (wave-private, no barrier) they leave as whole rows of
// COLS elements, 16 bytes per lane.  The pitch keeps the 16 rows of a write on distinct banks.
template <class E, int COLS>
struct RowStage {
  static constexpr int kRowBytes = COLS * (int)sizeof(E), kPitch = kRowBytes + 16, kBytes = 16 * kPitch;
  static constexpr int kLanes = kRowBytes / 16;  // lanes per row
  static_assert(kRowBytes % 16 == 0, "whole 16-byte pieces");
  // four neighbours of row r (0 .. 15) from column c (a multiple of 4)
  static __device__ __forceinline__ void put(char* lds, int r, int c, const E (&v)[4]) {
    if constexpr (sizeof(E) == 2) *reinterpret_cast<uint2*>(lds + r * kPitch + c * 2) = *reinterpret_cast<const uint2*>(v);
    else *reinterpret_cast<float4*>(lds + r * kPitch + c * 4) = *reinterpret_cast<const float4*>(v);
  }
  // rows 0 .. rows - 1, columns 0 .. cols - 1 to out (16-byte aligned rows of ld bytes)
  static __device__ __forceinline__ void flush(const char* lds, char* out, int64_t ld, int rows, int cols, int lane) {
    asm volatile("" ::: "memory");  // the reads below are of other lanes' writes: a wave's LDS operations run in order, so order is all they need
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int p = 0; p < (16 * kLanes + 63) / 64; ++p) {
      const int at = p * 64 + lane, r = at / kLanes, c = (at % kLanes) * (16 / (int)sizeof(E));
      if (r >= rows || c >= cols) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(lds + r * kPitch + c * sizeof(E));
      char* o = out + r * ld + c * sizeof(E);
      if (c + 16 / (int)sizeof(E) <= cols) {
        *reinterpret_cast<uint4*>(o) = v;
      } else {
        const E* e = reinterpret_cast<const E*>(&v);
        for (int u = 0; c + u < cols; ++u) reinterpret_cast<E*>(o)[u] = e[u];
      }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
};

// Dynamic LDS beyond 64 KB has to be allowed once per kernel and device; `done` is the caller's record for one kernel.  bytes: the most
// that ANY launch of the kernel asks for (later calls do not raise it).
inline hipError_t allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  if (bytes <= 64 * 1024) return hipSuccess;
  int dev = 0;
  if (const hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return hipSuccess;
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

}  // namespace mma
}  // namespace suave

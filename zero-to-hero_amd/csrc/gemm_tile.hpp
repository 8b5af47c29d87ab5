// The matrix product under the layer operators: C[m,n] = sum_k X[m,k] W[n,k]
// on the matrix cores, with the operator's epilogue applied to the sums.  Each
// operand's rows are contiguous along k (fp32, bf16, fp16 or int8), or, for
// the products of a backward pass, it is stored the other way about, k-rows of
// consecutive m or n (not for int8).
//
// Everything is laid out in 16-byte chunks of a row: 4 fp32, 8 16-bit or 16
// int8 elements.  A lane of the matrix instructions below holds one chunk of
// row lane % 32 or lane % 16 (32x32x16 and 16x16x32 on 16-bit types, 32x32x32
// and 16x16x64 on int8 take the whole chunk; fp32 takes four instructions, one
// element each: the order of k inside a step is free as long as both operands
// share it).  So one kernel
// serves all types.  W is the instruction's first operand, so a lane ends up
// with four consecutive columns n of one row m: a vector store, and one call
// of the dropout generator.
//
// A workgroup computes a BM x BN tile over K steps of 128 bytes, a whole line
// of memory per row (half lines were fetched twice: 1127 against 988 us for
// 8192 x 4096 x 16384 in bf16).  The tiles go from memory to one of two LDS
// buffers without passing through registers (buffer loads with the LDS bit: 64
// lanes, 16 bytes each, to consecutive LDS addresses; through registers the
// LDS writes cost 5 to 8% of 8192 x 8192 x 4096).  A row's chunk c sits in slot
// c ^ (row % 8), which spreads the rows that a fragment read touches over all
// banks; since the LDS side of the load is fixed, the lanes permute the
// addresses they load from instead.  The buffer descriptor ends with the
// operand's last row and lanes past the end of a row ask for an offset behind
// it: the hardware gives zero for both, so partial tiles need no other path.
//
// An operand stored by k-rows is kept that way in LDS (nothing is transposed
// in memory) and turned while it is read: 16-bit fragments by the transposing
// LDS read, in which sixteen lanes fetch four k-rows of sixteen columns and
// each receives one column's four values; fp32 by single words.
#pragma once

#include <type_traits>

#include "layers.hpp"

namespace ppo {

struct GemmArgs {
  const char* x;    // [M] rows
  const char* w0;   // [N] rows
  const char* w1;   // second matrix of a gated product, [N] rows
  int64_t xpitch, wpitch;  // bytes, multiples of 16
  int64_t kbytes;   // of a row, a multiple of 16
  int64_t k;        // k-rows of an operand that is stored by them
  int ranges;       // K is so many ranges of kbytes and k: W's are w0 and w1 in turn,
  int64_t x_range;  //    X's lie x_range bytes apart in its rows
  int M, N;         // N: output columns
  int tiles_m, tiles_n;
  int steps_per_split;     // K steps that one split takes
  char* partial;    // [splits][1 or 2][M][N4] 32-bit sums, or null: no split
};

constexpr int kStepBytes = 128;  // of a row, in one step

// Sums of one matrix instruction: kEdge x kEdge outputs over 64 lanes, 4 or
// 16 a lane, in groups of four consecutive columns n of one row m.
template <class T, int kEdge>
struct AccOf;
template <class T>
struct AccOf<T, 16> { typedef float type __attribute__((ext_vector_type(4))); };
template <class T>
struct AccOf<T, 32> { typedef float type __attribute__((ext_vector_type(16))); };
template <>
struct AccOf<int8_t, 16> { typedef int type __attribute__((ext_vector_type(4))); };
template <>
struct AccOf<int8_t, 32> { typedef int type __attribute__((ext_vector_type(16))); };
template <class T, int kEdge = 16>
using Acc = typename AccOf<T, kEdge>::type;

// c += w x over the k of one chunk per lane: row lane % kEdge of W and of X,
// chunk lane / kEdge of a run.
template <class T, int kEdge>
__device__ __forceinline__ Acc<T, kEdge> mfma(v4i w, v4i x, Acc<T, kEdge> c) {
  if constexpr (sizeof(T) == 4) {
    const v4f a = __builtin_bit_cast(v4f, w), b = __builtin_bit_cast(v4f, x);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if constexpr (kEdge == 16)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
      else
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  } else if constexpr (sizeof(T) == 1) {
    if constexpr (kEdge == 16)
      return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_i32_32x32x32_i8(w, x, c, 0, 0, 0);
  } else if constexpr (__is_same(T, fp16)) {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    const v8 a = __builtin_bit_cast(v8, w), b = __builtin_bit_cast(v8, x);
    if constexpr (kEdge == 16)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  } else {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    const v8 a = __builtin_bit_cast(v8, w), b = __builtin_bit_cast(v8, x);
    if constexpr (kEdge == 16)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
}

// Four consecutive columns of a lane's sums.
template <class T, int kEdge>
__device__ __forceinline__ Acc<T> four(const Acc<T, kEdge>& c, int group) {
  Acc<T> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = c[4 * group + i];
  return r;
}

// Descriptor of `bytes` (below 2^31) from p on; loads behind it give zero.
__device__ __forceinline__ v4i buffer_of(const char* p, uint32_t bytes) {
  const uint64_t a = (uint64_t)p;
  v4i r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32) & 0xffff);
  r[2] = __builtin_amdgcn_readfirstlane((int)bytes);
  r[3] = 0x00020000;
  return r;
}

// 64 lanes, 16 bytes each from buffer + offset, to LDS at lds + 16 * lane
// (`lds` is the same in all lanes).  Nothing in registers is written; the
// data has arrived after a barrier below that waits for it.  A load may read the
// descriptor five wait states after the vector instruction that wrote it
// (v_readfirstlane, or v_readlane of a spilled one) at the earliest, and the
// compiler does not look into the block: the block waits them itself (8192 x 4096
// -> 8192 gated forward 899 -> 912 us, backward 1898 -> 1911, int8 242 -> 244).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is reserved, and written all the same)
__device__ __forceinline__ void load_to_lds(uint32_t lds, v4i buffer, uint32_t offset) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 3\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer)
      : "m0");
}
#pragma clang diagnostic pop

// Waits until at most kLeft of this wave's loads are under way, and for its
// LDS reads, then for the whole workgroup.
template <int kLeft>
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLeft) : "memory");
}

// How one operand's tile of kRows rows of C (or columns) goes to LDS and from
// there to fragments.  kT: stored by k-rows.
template <class T, int kRows, int kWaves, bool kT>
struct Side {
  static constexpr int kSize = (int)sizeof(T);
  static constexpr int kLoads = kRows / 8 / kWaves;       // of a wave per step
  static constexpr int kPerLine = kRows * kSize / 16;     // chunks of a k-row (kT)
  static constexpr int kLines = 64 / kPerLine;            // k-rows that one load covers (kT)
  static constexpr int kSwing = kSize == 2 ? 64 : 128;    // bytes that 32 columns take (kT)
  static_assert(!kT || (kSize >= 2 && kPerLine <= 64), "");

  static __device__ __forceinline__ uint32_t stride(uint32_t pitch) {  // from load to load
    return (uint32_t)(kT ? kLines : 8) * pitch;
  }
  // k-rows k..k+3 of a fragment's columns lie 32 columns apart, so that they
  // do not meet in one bank
  static __device__ __forceinline__ int swing(int k) {
    return kSize == 4 ? k >> 2 & 1 : kRows >= 128 ? k & 3 : k >> 1 & 1;
  }
  // what a lane fetches with load i, relative to the tile's start: its place
  // in LDS is fixed (16 * lane), so the lanes permute what they ask for
  static __device__ __forceinline__ uint32_t offset(int wave, int lane, int i, uint32_t pitch) {
    if (kT) {
      const int k = (wave * kLoads + i) * kLines + lane / kPerLine, c = lane % kPerLine * 16;
      return (uint32_t)k * pitch + (uint32_t)((c / kSwing ^ swing(k)) * kSwing + c % kSwing);
    }
    return (uint32_t)((wave * kLoads + i) * 8 + (lane >> 3)) * pitch;
  }
  static __device__ __forceinline__ uint32_t chunk(int lane) {  // (not kT) within a step
    return (uint32_t)((lane & 7) ^ (lane >> 3)) * 16;
  }
  // one chunk of rows (columns) 32 * block .. + 31 in phase 0..3: row lane % 32,
  // chunk 2 * phase + lane / 32
  static __device__ __forceinline__ v4i read(char* tile, int lane, int block, int phase) {
    const int kq = lane >> 5;
    if constexpr (!kT) {
      const int r = lane & 31;
      return *reinterpret_cast<const v4i*>(tile + (block * 32 + r) * kStepBytes +
                                           ((phase * 2 + kq) ^ (r & 7)) * 16);
    } else if constexpr (kSize == 2) {
      typedef short v4s __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) v4s lds_v4s;
      const int i = lane & 15, k = phase * 16 + kq * 8 + i / 4;
      char* at = tile + k * kRows * 2 + (block ^ swing(k)) * kSwing + (lane >> 4 & 1) * 32 + i % 4 * 8;
      struct { v4s lo, hi; } r;
      r.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at);
      r.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 4 * kRows * 2));
      return __builtin_bit_cast(v4i, r);
    } else {
      const int k = (phase * 2 + kq) * 4;
      const char* at = tile + k * kRows * 4 + (block ^ swing(k)) * kSwing + (lane & 31) * 4;
      v4i r;
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = *reinterpret_cast<const int*>(at + j * kRows * 4);
      return r;
    }
  }
};

// Waits for this wave's LDS reads and writes, then for the workgroup.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

constexpr uint32_t kBehind = 0x80000000u;  // an offset that no descriptor reaches

// Workgroup -> tile.  Workgroups go round-robin over the eight XCDs, each
// with an L2 of its own: an XCD takes a run of consecutive tiles, and a run
// walks blocks of kGroup row tiles by columns, so that the tiles in flight on
// one XCD share rows and columns.
__device__ __forceinline__ void tile_of(const GemmArgs& a, int id, int& tm, int& tn) {
  constexpr int kXcds = 8, kGroup = 8;
  const int n = a.tiles_m * a.tiles_n;
  const int xcd = id % kXcds, q = n / kXcds, r = n % kXcds;
  const int t = xcd * q + min(xcd, r) + id / kXcds;
  const int per = kGroup * a.tiles_n, first = t / per * kGroup;
  const int rows = min(kGroup, a.tiles_m - first);
  tm = first + t % per % rows;
  tn = t % per / rows;
}

// One 32-bit sum block to its place among the partial sums of a split.
template <class A>
__device__ __forceinline__ void store_partial(const GemmArgs& a, int split, int half, int halves,
                                              int m, int n, A v) {
  const int64_t n4 = round_up(a.N, 4);
  const int64_t at = ((((int64_t)split * halves + half) * a.M + m) * n4 + n) * 4;
  *reinterpret_cast<A*>(a.partial + at) = v;
}

// Epi, the operator's epilogue: kGated (two W matrices, one output), kBatch
// (rows that a lane takes at once),
//   Cols columns(int n), what columns n..n+3 bring along (a bias, scales),
//   Row row(int m), what row m does (kRows: whether that is anything),
// both plain 32-bit or 64-bit values that are fetched before the stores begin,
//   void apply(n, const Cols&, const int (&m)[B], const bool (&live)[B],
//              const Row (&)[B], const Acc<T> (&c)[B] [, const Acc<T> (&second)[B]])
// for columns n..n+3 of B rows m, of which the live ones are stored (n < N for
// those; columns past N - 1 are its to skip).
//
// A step is four phases, each one 16-byte chunk per lane of every fragment.
// While the matrix cores work on one phase, the fragments of the next are read
// from LDS, a read or a load in the shadow of each matrix instruction.  The
// workgroup meets once a step, before the last phase: every wave has then read
// the buffer to its end and the other buffer's loads have arrived.  The loads
// of the step after next go into the freed buffer during the last phase and
// the first of the next step (issued at once they hold up the instructions
// behind them; later they arrive late).
//
// `block` of `blocks` workgroups that share the tiles of split `split`; lds: two
// buffers of (BM + BN) * kStepBytes.
template <class T, int BM, int BN, int kWavesM, int kWavesN, bool kXT, bool kWT, class Epi>
__device__ __forceinline__ void gemm_tile(const GemmArgs& a, const Epi& epi,
                                          char (*lds)[(BM + BN) * kStepBytes], int block,
                                          int blocks, int split) {
  constexpr int kWaves = kWavesM * kWavesN;
  constexpr int kEdge = 32;  // of a matrix instruction's block
  constexpr int TM = BM / kWavesM / kEdge, TN = BN / kWavesN / kEdge;
  constexpr int kPhases = 4;
  typedef Side<T, BM, kWaves, kXT> X;
  typedef Side<T, BN, kWaves, kWT> W;
  constexpr int kLoads = X::kLoads + W::kLoads;
  constexpr int kFrags = TM + TN, kMfmas = TM * TN;
  constexpr int kEarly = kLoads / 2;  // loads of a step in the last phase before it
  constexpr bool kGated = Epi::kGated;
  constexpr int kCols = kGated ? BN / 2 : BN;  // output columns of a tile
  constexpr int kBuffer = (BM + BN) * kStepBytes;
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0, "");
  static_assert(!kGated || (TN % 2 == 0 && !kWT), "");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / kWavesN, wn = wave % kWavesN;
  constexpr int kStepK = kStepBytes / (int)sizeof(T);
  const int per_range = (int)(kXT ? div_up(a.k, kStepK) : div_up(a.kbytes, kStepBytes));
  const int steps = per_range * a.ranges;
  const int first = split * a.steps_per_split;
  const int count = max(0, min(steps - first, a.steps_per_split));

  // --- loads ------------------------------------------------------------------------
  const uint32_t xp = (uint32_t)a.xpitch, wp = (uint32_t)a.wpitch;
  typedef v4i Buffer;
  // one operand's source for a step: an operand of k-contiguous rows has one
  // descriptor and a moving offset, one of k-rows a descriptor per step
  struct Source { Buffer b0, b1; uint32_t off; };
  int m0, n0;  // of the tile that is loaded
  Buffer bx, bw0, bw1;
  auto locate = [&](int id) {
    int tm, tn;
    tile_of(a, id, tm, tn);
    m0 = tm * BM;
    n0 = tn * kCols;
    const uint32_t w_bytes = (uint32_t)min(kCols, a.N - n0) * wp;
    bx = kXT ? buffer_of(a.x, 0)
             : buffer_of(a.x + m0 * a.xpitch, (uint32_t)min(BM, a.M - m0) * xp);
    bw0 = kWT ? bx : buffer_of(a.w0 + n0 * a.wpitch, w_bytes);
    bw1 = kGated ? buffer_of(a.w1 + n0 * a.wpitch, w_bytes) : bw0;
  };
  auto by_rows = [&](const char* base, int64_t pitch, int64_t col_bytes, int local, bool live) {
    const int64_t k0 = (int64_t)local * kStepK;
    const int64_t left = live ? (a.k - k0) * pitch - col_bytes : 0;
    return buffer_of(base + k0 * pitch + col_bytes,
                     (uint32_t)max((int64_t)0, min(left, (int64_t)0x7fffffff)));
  };
  // steps past the last ask for nothing
  auto source = [&](int step, Source& x, Source& w) {
    const bool live = step < count;
    const int at = first + step;
    const int range = a.ranges > 1 ? at / per_range : 0, local = at - range * per_range;
    const uint32_t kb = (uint32_t)local * kStepBytes + X::chunk(lane);
    const uint32_t k_off = live && kb < (uint32_t)a.kbytes ? kb : kBehind;
    const int64_t behind = range * a.x_range;
    x = {bx, bx, k_off + (uint32_t)behind};
    w = {bw0, bw1, k_off};
    if (kXT)
      x.off = 0, x.b0 = by_rows(a.x, a.xpitch, (int64_t)m0 * (int)sizeof(T) + behind, local, live);
    if (kWT)
      w.off = 0, w.b0 = by_rows(range & 1 ? a.w1 : a.w0, a.wpitch, (int64_t)n0 * (int)sizeof(T),
                                local, live);
  };
  const uint32_t lds0 =
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)&lds[0][0];
  // load i of a step (X's first)
  auto load = [&](int i, int buf, const Source& x, const Source& w) {
    const uint32_t to = lds0 + buf * kBuffer + (i < X::kLoads ? (wave * X::kLoads + i) * 1024
                        : BM * kStepBytes + (wave * W::kLoads + i - X::kLoads) * 1024);
    if (i < X::kLoads) return load_to_lds(to, x.b0, X::offset(wave, lane, i, xp) + x.off);
    const int iw = i - X::kLoads;
    if (!kGated) return load_to_lds(to, w.b0, W::offset(wave, lane, iw, wp) + w.off);
    // a wave's columns: half from the first matrix, half from the second
    constexpr int kSpan = TN * kEdge, kHalf = kSpan / 2;
    const int j = (wave * W::kLoads + iw) * 8;  // first of the eight LDS rows
    const int col = j / kSpan * kHalf + j % kHalf;
    load_to_lds(to, j % kSpan >= kHalf ? w.b1 : w.b0,
                (uint32_t)(col + (lane >> 3)) * wp + w.off);
  };

  // --- fragments --------------------------------------------------------------------
  const int r = lane & (kEdge - 1), kq = lane / kEdge;
  struct Frags { v4i w[TN], x[TM]; };
  Frags f[2];
  // fragment g of a phase: W's first
  auto read = [&](Frags& to, int g, char* buf, int phase) {
    if (g < TN)
      to.w[g] = W::read(buf + BM * kStepBytes, lane, wn * TN + g, phase);
    else
      to.x[g - TN] = X::read(buf, lane, wm * TM + g - TN, phase);
  };

  Acc<T, kEdge> acc[TM][TN];
  auto multiply = [&](const Frags& from, int e) {
    acc[e / TN][e % TN] = mfma<T, kEdge>(from.w[e % TN], from.x[e / TN], acc[e / TN][e % TN]);
    __builtin_amdgcn_sched_barrier(0);
  };
  // The matrix instructions of a phase in their order; behind each goes what it
  // is to cover: the reads behind the first of every pair, the rest (`other`,
  // called with the share of the phase that is over) behind the second.
  auto phase = [&](const Frags& from, Frags& to, char* buf, int p, auto&& other) {
#pragma unroll
    for (int e = 0; e < kMfmas; ++e) {
      multiply(from, e);
      // reads: evenly over the even slots (all slots if there are too few)
      constexpr int kEven = (kMfmas + 1) / 2;
      if (e % 2 == 0) {
#pragma unroll
        for (int g = e / 2 * kFrags / kEven; g < (e / 2 + 1) * kFrags / kEven; ++g)
          read(to, g, buf, p);
      }
      if (e % 2 == 1 || kMfmas == 1) other(e / 2, kMfmas / 2 > 0 ? kMfmas / 2 : 1);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // --- epilogue ---------------------------------------------------------------------
  // Through LDS, 32 rows of the wave's block at a time: a lane then holds
  // columns next to its neighbours' (whole lines are stored), and the
  // operator's arithmetic is a loop whose code is there once, not once for
  // every register.  A wave reads only what it wrote.  Row r's chunks (16
  // bytes) are permuted by r % 16 to spread the banks.
  constexpr int kSpan = TN * kEdge, kOut = kGated ? kSpan / 2 : kSpan;
  constexpr int kLanes = kOut / 4, kRows = 64 / kLanes, kBatch = Epi::kBatch;
  static_assert(kWaves * kEdge * kSpan * 4 <= kBuffer && kEdge % (kRows * kBatch) == 0, "");
  typedef Acc<T> A4;
  A4* mine = reinterpret_cast<A4*>(&lds[0][0] + wave * kEdge * kSpan * 4);
  constexpr int kRowSets = (TM * kEdge + 63) / 64;
  auto finish = [&](int em0, int en0, const typename Epi::Cols& cols,
                    const typename Epi::Row (&states)[kRowSets], bool more) {
    const int n = en0 + wn * kOut + lane % kLanes * 4;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          mine[r * (kSpan / 4) + ((j * 8 + g * 2 + kq) ^ (r & 15))] =
              four<T, kEdge>(acc[i][j], g);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      // (the next tile's first loads have then arrived, with most of the stores)
      if (i == TM - 1 && more) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll 1
      for (int row0 = 0; row0 < kEdge; row0 += kRows * kBatch) {
        typename Epi::Row rows[kBatch];
        int m[kBatch];
        bool live[kBatch];
        A4 c[kBatch], c2[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int row = row0 + b * kRows + lane / kLanes, at = i * kEdge + row;
          m[b] = em0 + wm * TM * kEdge + at;
          live[b] = m[b] < a.M && n < a.N;
          if constexpr (Epi::kRows) rows[b] = __shfl(states[i * kEdge / 64], at & 63, 64);
          c[b] = mine[row * (kSpan / 4) + ((lane % kLanes) ^ (row & 15))];
          if constexpr (kGated) c2[b] = mine[row * (kSpan / 4) + ((kLanes + lane % kLanes) ^ (row & 15))];
        }
        if (a.partial) {
#pragma unroll
          for (int b = 0; b < kBatch; ++b)
            if (live[b]) {
              store_partial(a, split, 0, kGated ? 2 : 1, m[b], n, c[b]);
              if constexpr (kGated) store_partial(a, split, 1, 2, m[b], n, c2[b]);
            }
        } else if constexpr (kGated) {
          epi.apply(n, cols, m, live, rows, c, c2);
        } else {
          epi.apply(n, cols, m, live, rows, c);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  };

  // --- tiles ------------------------------------------------------------------------
  // Where the grid is smaller than the tiles, a workgroup takes several, and
  // the first step of the next is loaded (into the second buffer) while the
  // epilogue of the last uses the first.  A tile's steps go to the buffers in
  // turn, the second first.
  constexpr bool kLoop = BM * BN >= 256 * 256;
  const int tiles = a.tiles_m * a.tiles_n;
  Source x, w;
  locate(block);
  source(0, x, w);
#pragma unroll
  for (int i = 0; i < kLoads; ++i) load(i, 1, x, w);
  for (int id = block;; id += blocks) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = Acc<T, kEdge>(0);
    source(1, x, w);
#pragma unroll
    for (int i = 0; i < kEarly; ++i) load(i, 0, x, w);
    if (id == block) stage_barrier<kEarly>();
#pragma unroll
    for (int g = 0; g < kFrags; ++g) read(f[0], g, lds[1], 0);
    for (int step = 0; step < count; ++step) {
      const int b = step & 1 ^ 1;
      char* cur = lds[b];
      char* other = lds[b ^ 1];
#pragma unroll
      for (int p = 0; p < kPhases - 1; ++p)
        phase(f[p & 1], f[(p + 1) & 1], cur, p + 1, [&](int slot, int slots) {
          if (p > 0) return;
          constexpr int kRest = kLoads - kEarly;
#pragma unroll
          for (int i = slot * kRest / slots; i < (slot + 1) * kRest / slots; ++i)
            load(kEarly + i, b ^ 1, x, w);
        });
      stage_barrier<0>();
      source(step + 2, x, w);
      phase(f[1], f[0], other, 0, [&](int slot, int slots) {
#pragma unroll
        for (int i = slot * kEarly / slots; i < (slot + 1) * kEarly / slots; ++i) load(i, b, x, w);
      });
    }
    // what the epilogue needs beside the sums is fetched before its LDS is free
    // and the next tile's loads are under way: waiting for it later would wait
    // for those
    const int em0 = m0, en0 = n0;
    const bool more = kLoop && id + blocks < tiles;
    typename Epi::Cols cols = epi.columns(min(en0 + wn * kOut + lane % kLanes * 4, a.N - 1));
    typename Epi::Row states[kRowSets];
    if constexpr (Epi::kRows) {
#pragma unroll
      for (int i = 0; i < kRowSets; ++i)
        states[i] = epi.row(min(em0 + wm * TM * kEdge + i * 64 + lane, a.M - 1));
    }
    stage_barrier<0>();
    if constexpr (Epi::kRows) {
#pragma unroll
      for (int i = 0; i < kRowSets; ++i) asm volatile("" : "+v"(states[i]));
    }
    cols.arrived();
    if (more) {
      locate(id + blocks);
      source(0, x, w);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) load(i, 1, x, w);
    }
    finish(em0, en0, cols, states, more);
    if (!more) break;
    lds_barrier();
  }
}

template <class T, int BM, int BN, int kWavesM, int kWavesN, bool kXT, bool kWT, class Epi>
__global__ void __launch_bounds__(kWavesM* kWavesN * 64)
    gemm_tile_kernel(const GemmArgs a, const Epi epi) {
  __shared__ __align__(1024) char lds[2][(BM + BN) * kStepBytes];
  gemm_tile<T, BM, BN, kWavesM, kWavesN, kXT, kWT>(a, epi, lds, blockIdx.x, gridDim.x, blockIdx.y);
}

// The two products of a backward pass, dY W and dY^T X, in one launch: apart,
// neither fills the chip for as long as it runs, unless it is cut into splits
// whose sums are joined (a training step of 256 x 128 -> 256 in fp32 35 -> 26 us, of
// 4096 x 1024 -> 2048 in bf16 183 -> 151).  The first `span` workgroups are those
// of the product whose workgroups have more steps.  `extra`, a small task of
// `blocks` workgroups that needs neither, goes before them.
struct GemmPair {
  GemmArgs x, w;
  int splits_x, splits_w, span;
  bool w_first;
};
template <class T, int BM, int BN, int kWavesM, int kWavesN, class Epi, class Extra>
__global__ void __launch_bounds__(kWavesM* kWavesN * 64)
    gemm_pair_kernel(const GemmPair p, const Epi ex, const Epi ew, const Extra extra) {
  __shared__ __align__(1024) char lds[2][(BM + BN) * kStepBytes];
  const int block = (int)blockIdx.x - (extra.blocks + 7) / 8 * 8;
  if (block < 0) {
    if ((int)blockIdx.x < extra.blocks)
      extra.template run<kWavesM * kWavesN * 64>(blockIdx.x, &lds[0][0]);
    return;
  }
  const bool behind = block >= p.span, second = behind != p.w_first;
  const int at = block - (behind ? p.span : 0);
  const int tiles = second ? p.w.tiles_m * p.w.tiles_n : p.x.tiles_m * p.x.tiles_n;
  const int wide = (tiles + 7) / 8 * 8;  // (a split's tiles start on the first XCD)
  const int split = at / wide, id = at % wide;
  if (id >= tiles) return;
  if (second)
    gemm_tile<T, BM, BN, kWavesM, kWavesN, true, true>(p.w, ew, lds, id, tiles, split);
  else
    gemm_tile<T, BM, BN, kWavesM, kWavesN, false, true>(p.x, ex, lds, id, tiles, split);
}

// The epilogue of one row's four columns.
template <class T, class Epi, int kHalves>
__device__ __forceinline__ void apply_one(const Epi& epi, int m, int n,
                                          const typename Epi::Cols& cols, bool live,
                                          const Acc<T> (&sum)[kHalves]) {
  const int ms[1] = {m};
  const bool lives[1] = {live};
  typename Epi::Row rows[1];
  if constexpr (Epi::kRows) rows[0] = epi.row(m);
  const Acc<T> c[1] = {sum[0]};
  if constexpr (kHalves == 2) {
    const Acc<T> c2[1] = {sum[1]};
    epi.apply(n, cols, ms, lives, rows, c, c2);
  } else {
    epi.apply(n, cols, ms, lives, rows, c);
  }
}

// Joins the splits of K in their order and applies the epilogue.
template <class T, class Epi>
__device__ __forceinline__ void gemm_join(const GemmArgs& a, const Epi& epi, int splits) {
  constexpr int kHalves = Epi::kGated ? 2 : 1;
  const int64_t groups = div_up(a.N, 4), n4 = groups * 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= a.M * groups) return;
  const int m = (int)(id / groups), n = (int)(id % groups) * 4;
  Acc<T> sum[kHalves];
  for (int s = 0; s < splits; ++s)
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int64_t at = ((((int64_t)s * kHalves + h) * a.M + m) * n4 + n) * 4;
      const Acc<T> v = *reinterpret_cast<const Acc<T>*>(a.partial + at);
      sum[h] = s ? sum[h] + v : v;
    }
  apply_one<T>(epi, m, n, epi.columns(n), true, sum);
}

template <class T, class Epi>
__global__ void __launch_bounds__(256) gemm_join_kernel(const GemmArgs a, const Epi epi,
                                                        int splits) {
  gemm_join<T>(a, epi, splits);
}

template <class T, class Epi>
__global__ void __launch_bounds__(256) gemm_join_pair_kernel(const GemmPair p, const Epi ex,
                                                             const Epi ew) {
  const bool second = p.splits_x == 1 || blockIdx.y == 1;  // (the only one, or both)
  if (second)
    gemm_join<T>(p.w, ew, p.splits_w);
  else
    gemm_join<T>(p.x, ex, p.splits_x);
}

constexpr int kRunBytes = 128;  // of K that a wave of the rows kernel takes at a time

// Sixteen bytes of a row that ends `left` bytes from p on; zeros behind.
__device__ __forceinline__ v4i load16_upto(const char* p, int left) {
  if (left >= 16) return *reinterpret_cast<const v4i_any*>(p);
  union { v4i v; char c[16]; } r;
  r.v = v4i{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < left) r.c[i] = p[i];
  return r.v;
}

// The same by few loads: the row, of `bytes` bytes, has its last sixteen shifted
// where fewer are left.
__device__ __forceinline__ v4i load16_of_row(const char* p, int left, int bytes, bool odd) {
  if (left <= 0) return v4i{0, 0, 0, 0};
  if (bytes < 16) return load16_upto(p, left);
  const int gone = left < 16 ? 16 - left : 0;
  const char* at = p - gone;
  const v4i v = odd || gone ? load16_shifted(at) : *reinterpret_cast<const v4i_any*>(at);
  uint64_t part[2];
  __builtin_memcpy(part, &v, 16);
  if (gone >= 8) {
    part[0] = part[1] >> (gone - 8) * 8;
    part[1] = 0;
  } else if (gone) {
    part[0] = part[0] >> gone * 8 | part[1] << (8 - gone) * 8;
    part[1] >>= gone * 8;
  }
  v4i r;
  __builtin_memcpy(&r, part, 16);
  return r;
}

// Up to three matrices of rows of `bytes` bytes to rows at a pitch, zeros behind
// each row, in one launch (blockIdx.y).  odd: some row starts off 4 bytes.
struct PadArgs {
  const char* in[3];
  char* out[3];
  int64_t rows[3];
};
inline __global__ void __launch_bounds__(256) pad_rows_kernel(const PadArgs a, int bytes, int pitch,
                                                              bool odd) {
  const char* in = a.in[blockIdx.y];
  char* out = a.out[blockIdx.y];
  // a workgroup takes as many rows at once as 256 threads of 16 bytes cover
  const int chunks = pitch / 16;
  int per_row = 256;
  while (per_row / 2 >= chunks && per_row > 1) per_row >>= 1;
  const int at = threadIdx.x & (per_row - 1), lanes = 256 / per_row;
  for (int64_t r = (int64_t)blockIdx.x * lanes + threadIdx.x / per_row; r < a.rows[blockIdx.y];
       r += (int64_t)gridDim.x * lanes)
    for (int c = at * 16; c < pitch; c += per_row * 16) {
      *reinterpret_cast<v4i*>(out + r * pitch + c) =
          load16_of_row(in + r * bytes + c, bytes - c, bytes, odd);
    }
}

inline int pad_rows(const PadArgs& a, int64_t bytes, int64_t pitch, hipStream_t stream) {
  int64_t rows = 0;
  uintptr_t starts = (uintptr_t)bytes;
  for (int i = 0; i < 3; ++i) {
    rows = a.rows[i] > rows ? a.rows[i] : rows;
    starts |= (uintptr_t)a.in[i];
  }
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)(rows < 4096 ? rows : 4096), 3), dim3(256), 0,
                     stream, a, (int)bytes, (int)pitch, (starts & 3) != 0);
  return last_launch_status();
}

// Few rows of X (at most 16 * MT): every weight is read once, so the time is
// that of reading W.  A workgroup takes 16 columns and its waves share K in
// runs of 128 bytes; W goes straight to registers (no reuse for LDS to serve)
// from rows of any alignment, and the waves' sums meet in LDS.  Rows of X
// beyond M repeat the last one and are not stored.  kOdd: rows that start off 4
// bytes.
template <class T, int MT, int kWaves, bool kOdd, class Epi>
__global__ void __launch_bounds__(kWaves * 64) gemm_rows_kernel(const GemmArgs a, const Epi epi) {
  constexpr int kHalves = Epi::kGated ? 2 : 1;
  __shared__ Acc<T> red[kWaves][MT * kHalves][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, kq = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int64_t wrow = min(n0 + r16, a.N - 1);
  const char* w[2] = {a.w0 + wrow * a.wpitch + kq * 16,
                      kHalves == 2 ? a.w1 + wrow * a.wpitch + kq * 16 : nullptr};
  const char* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) x[i] = a.x + (int64_t)min(i * 16 + r16, a.M - 1) * a.xpitch + kq * 16;
  const typename Epi::Cols cols = epi.columns(min(n0 + kq * 4, a.N - 1));
  Acc<T> acc[MT][kHalves];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int h = 0; h < kHalves; ++h) acc[i][h] = Acc<T>{0, 0, 0, 0};

  const int kbytes = (int)a.kbytes;
  const int full = kbytes / kRunBytes;  // whole runs
  // kRuns runs' loads are under way before the first is used
  constexpr int kRuns = MT == 1 ? 4 : MT == 2 ? 3 : 2;
  auto load = [](const char* p) -> v4i {
    if constexpr (kOdd) return load16_shifted(p);
    return *reinterpret_cast<const v4i_any*>(p);
  };
  auto take = [&](int s, auto runs) {
    constexpr int R = decltype(runs)::value;
    v4i wf[R][kHalves][2], xf[R][MT][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t k = (int64_t)(s + r * kWaves) * kRunBytes;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
          wf[r][h][ks] = load(w[h] + k + ks * 64);
#pragma unroll
        for (int i = 0; i < MT; ++i)
          xf[r][i][ks] = load(x[i] + k + ks * 64);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
            acc[i][h] = mfma<T, 16>(wf[r][h][ks], xf[r][i][ks], acc[i][h]);
  };
  int s = wave;
  for (; s + (kRuns - 1) * kWaves < full; s += kRuns * kWaves)
    take(s, std::integral_constant<int, kRuns>{});
  for (; s < full; s += kWaves) take(s, std::integral_constant<int, 1>{});
  if (full * kRunBytes < kbytes && wave == full % kWaves) {  // the run that ends inside
    const int64_t k = (int64_t)full * kRunBytes;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int left = kbytes - (int)k - ks * 64 - kq * 16;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const v4i xf = load16_upto(x[i] + k + ks * 64, left);
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
          acc[i][h] = mfma<T, 16>(load16_upto(w[h] + k + ks * 64, left), xf, acc[i][h]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int h = 0; h < kHalves; ++h) red[wave][i * kHalves + h][lane] = acc[i][h];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    if (wave != i % kWaves) continue;
    Acc<T> sum[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      sum[h] = red[0][i * kHalves + h][lane];
#pragma unroll
      for (int v = 1; v < kWaves; ++v) sum[h] += red[v][i * kHalves + h][lane];
    }
    const int m = i * 16 + r16, n = n0 + kq * 4;
    if (m < a.M && n < a.N) apply_one<T>(epi, m, n, cols, true, sum);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct GemmPlan {
  int tile;     // 0: rows kernel, else the tile's edge
  int splits;
  size_t partial_bytes;
  double us;    // expected
};

constexpr int kCus = 256;
constexpr int kRowsMax = 64;       // rows that the rows kernel takes
constexpr int64_t kMaxRows = (int64_t)1 << 27;   // of either operand
constexpr int64_t kMaxPitch = (int64_t)1 << 22;  // 256 rows of a tile stay below 2^31 bytes

// What a workgroup of a tile takes, in us (plan_gemm): 8- and 16-bit types and
// fp32, of rows along k and of k-rows (fitted to 440 cuts of 18 backward passes).
struct TileCost { int tile, per_cu; double step, alone, fixed, lone; };
constexpr TileCost kTileCosts[2][2][3] = {
    {{{256, 1, 0.95, 1.11, 17.6, 10.7}, {128, 2, 0.32, 0.52, 4.2, 7.8}, {64, 5, 0.19, 0.44, 1.75, 4.6}},
     {{256, 1, 7.2, 7.2, 17.6, 10.7}, {128, 2, 1.8, 2.0, 4.2, 7.8}, {64, 5, 0.90, 1.08, 1.75, 4.6}}},
    {{{256, 1, 1.32, 1.28, 17.6, 11.6}, {128, 2, 0.49, 0.79, 4.7, 7.8}, {64, 5, 0.20, 0.68, 1.33, 6.8}},
     {{256, 1, 4.65, 7.4, 21.0, 8.3}, {128, 2, 2.05, 2.16, 2.3, 4.1}, {64, 5, 0.60, 1.43, 1.2, 2.0}}}};
inline double join_cost(int splits, int64_t M, int64_t wrows) {
  return splits > 1 ? splits * 8.0 * (double)M * wrows / 13.6e6 : 0.0;
}
inline size_t partial_size(int splits, int64_t M, int64_t wrows) {
  return splits > 1 ? (size_t)splits * M * round_up(wrows, 8) * 4 : 0;
}

// How a product of M rows and `wrows` rows of W (both matrices of a gated one
// together) over `kbytes` is cut: the tile and the number of splits of K with
// the least expected time in us.  A workgroup takes `step` a K step and `fixed`
// for its start and epilogue while it shares its CU (what the CU gets done),
// and at least `alone` a step and `lone` where it waits for memory; a split
// adds a launch, and its partial sums are written and read again (in the
// caches).  The numbers are fitted to 60 products of 64 to 11000 rows, 64 to
// 16384 columns and 1 to 96 steps, each in up to 12 cuts: the cut chosen takes
// 1.5% longer than the best on average.  Measured on MI355X (us, bf16 unless
// said), tile 256 / 128 / 64 without split: gated 4096 x 1024 -> 2048 41 / 42 / 60,
// 1024 x 2048 -> 2048 49 / 28 / 26, fp32 4096 x 512 -> 1024 134 / 74 / 102; 128 in
// two splits 79, 33 and 90; fp32 1024 x 1024 -> 512 in 64s and one, two or four
// splits 40 / 43 / 31.  The rows kernel's time is that of reading W, or of one
// workgroup's K where the columns are few, more where a single matrix does not
// share the reads of x, and two to three times that for rows that start off 4
// bytes (16 and 64 x 1023 -> 1365 gated bf16 9 and 25 us, 1024 -> 1365 5 and 8).  The tiles, which want a padded copy of
// rows off 16 bytes, have to be 15% better by this estimate, which is for weights
// that the caches hold (from HBM the rows kernel loses least).  1, 16, 32 and 64 rows
// of 4096 -> 8192 gated 24, 25, 32 and 47, against 25, 26, 26 and 27 for tiles of 64 in
// two or four splits; with weights from HBM 28, 31, 36 and 51 against 31, 32, 33 and
// 38; of 16384 -> 512 gated 34, 44, 58 and 87 against 18, 20, 20 and 20 in sixteen.
enum GemmKind { kOneMatrix, kTwoMatrices, kByKRows };
inline GemmPlan plan_gemm(int64_t M, int64_t wrows, int64_t row_bytes, bool fp32, GemmKind kind) {
  const int64_t kbytes = round_up(row_bytes, 16);
  GemmPlan p = {-1, 1, 0, 0.0};
  double best = 0.0;
  if (M <= kRowsMax && kind != kByKRows) {
    p.tile = 0;
    const int set = M <= 16 ? 0 : M <= 32 ? 1 : 2;
    const double reads[2][3] = {{1.25, 2.0, 3.3}, {1.03, 1.25, 1.8}};
    const double row[2][3] = {{0.75, 1.3, 2.1}, {1.15, 1.75, 2.6}};
    const double odd[] = {1.8, 2.2, 3.0};
    const double all = 1.0 + (double)wrows * kbytes / 5.6e6 * reads[kind][set];
    const double one = 2.4 + (double)kbytes / 1024.0 * row[kind][set];
    best = fmax(all, one) * (row_bytes % 4 ? odd[set] : 1.0) / 1.15;
    if (row_bytes != kbytes) best -= 4.0 + 2.0 * (double)wrows * kbytes / 5.3e6;
  }
  const double steps = (double)div_up(kbytes, kStepBytes);
  for (const TileCost& c : kTileCosts[kind == kByKRows][fp32]) {
    for (int splits = 1; splits <= 16; splits *= 2) {
      if (splits > 1 && steps < 4.0 * splits) break;
      const double groups = (double)(div_up(M, c.tile) * div_up(wrows, c.tile)) * splits;
      const double each = ceil(steps / splits);
      const double busy = ceil(groups / kCus) * (each * c.step + c.fixed);
      const double waits = ceil(groups / (kCus * c.per_cu)) * (each * c.alone + c.lone);
      const double join = (splits > 1 ? 4.0 : 0.0) + join_cost(splits, M, wrows);
      const double time = fmax(busy, waits) + join;
      if (p.tile < 0 || time < best) {
        best = time;
        p.tile = c.tile;
        p.splits = splits;
      }
    }
  }
  p.partial_bytes = partial_size(p.splits, M, wrows);
  p.us = best;
  return p;
}

// The same for the two products of a backward pass in one launch (tile 0: they
// run apart).  Both share the tile; a round of workgroups takes the mean of
// theirs.  Over 18 backward passes in up to 48 cuts the one chosen takes 2.3%
// longer than the best.
struct PairPlan {
  int tile, splits_x, splits_w;
  size_t partial_x, partial_w;  // bytes
};
inline PairPlan plan_pair(int64_t Mx, int64_t Nx, int64_t bytes_x, int64_t Mw, int64_t Nw,
                          int64_t bytes_w, bool fp32, double apart) {
  PairPlan p = {0, 1, 1, 0, 0};
  double best = apart;
  const double kx = (double)div_up(bytes_x, kStepBytes), kw = (double)div_up(bytes_w, kStepBytes);
  for (const TileCost& c : kTileCosts[1][fp32]) {
    const double gx = (double)(div_up(Mx, c.tile) * div_up(Nx, c.tile)),
                 gw = (double)(div_up(Mw, c.tile) * div_up(Nw, c.tile));
    for (int sx = 1; sx <= 16 && (sx == 1 || kx >= 4.0 * sx); sx *= 2)
      for (int sw = 1; sw <= 16 && (sw == 1 || kw >= 4.0 * sw); sw *= 2) {
        const double groups = gx * sx + gw * sw, ex = ceil(kx / sx), ew = ceil(kw / sw);
        const double each = (gx * sx * ex + gw * sw * ew) / groups;
        const double busy = ceil(groups / kCus) * (each * c.step + c.fixed);
        const double waits = fmax(ceil(groups / (kCus * c.per_cu)) * (each * c.alone + c.lone),
                                  fmax(ex, ew) * c.alone + c.lone);
        const double join =
            sx * sw > 1 ? 4.0 + 2.0 * (join_cost(sx, Mx, Nx) + join_cost(sw, Mw, Nw)) : 0.0;
        const double time = fmax(busy, waits) + join;
        if (time < best) {
          best = time;
          p = {c.tile, sx, sw, partial_size(sx, Mx, Nx), partial_size(sw, Mw, Nw)};
        }
      }
  }
  return p;
}

// Checks what the kernels assume of sizes (a grid's threads are counted in 32
// bits: 128 for each of the smallest tiles, 16 for a column of the rows kernel).
inline bool gemm_fits(int64_t M, int64_t N, int64_t pitch_bytes) {
  return M <= kMaxRows && N <= kMaxRows && pitch_bytes < kMaxPitch &&
         div_up(M, 64) * div_up(N, 32) < ((int64_t)1 << 25);
}

template <class T, bool kXT>
void cut_gemm(GemmArgs& a, bool gated, int tile, int splits) {
  const int64_t range_steps = kXT ? div_up(a.k, kStepBytes / (int)sizeof(T))
                                  : div_up(a.kbytes, kStepBytes);
  a.steps_per_split = (int)div_up(range_steps * a.ranges, splits);
  a.tiles_m = (int)div_up(a.M, tile);
  a.tiles_n = (int)div_up(a.N, gated ? tile / 2 : tile);
}

// p: plan_gemm's for these sizes.
template <class T, bool kXT = false, bool kWT = false, class Epi>
int launch_gemm(GemmArgs a, const Epi& epi, const GemmPlan& p, char* partial, hipStream_t stream) {
  if (a.ranges == 0) a.ranges = 1;
  a.partial = p.splits > 1 ? partial : nullptr;
  if constexpr (!kXT && !kWT) {
    if (p.tile == 0) {
      const dim3 grid((unsigned)div_up(a.N, 16));
      // Eight waves where a CU has one workgroup and each wave four runs of K or
      // more (four and eight, with weights from HBM, gated: 1 x 4096 -> 2048 bf16 15.3
      // and 12.9 us, fp32 29.3 and 23.1; 32 x 4096 -> 4096 bf16 25.5 and 22.4; for 16
      // rows alike, 2048 -> 4096 11.6 and 12.0; below 32 runs 1 x 1024 -> 4096 6.5 and
      // 7.0, with more workgroups 16 x 4096 -> 8192 31 and 34), except for many rows of
      // fp32, which the matrix cores bind (64 x 2050 -> 1000 42 and 44, 6116 -> 3376 94
      // and 107).
      const bool eight = div_up(a.N, 16) <= kCus && a.kbytes >= 32 * kRunBytes &&
                         !(sizeof(T) == 4 && a.M > 32);
      const bool odd = sizeof(T) < 4 && (((uintptr_t)a.x | (uintptr_t)a.w0 | (uintptr_t)a.w1 |
                                          (uintptr_t)a.xpitch | (uintptr_t)a.wpitch) & 3);
      auto go = [&](auto sets, auto waves) {
        constexpr int MT = decltype(sets)::value, kWaves = decltype(waves)::value;
        constexpr bool kOdd = sizeof(T) < 4;
        if (odd)
          hipLaunchKernelGGL((gemm_rows_kernel<T, MT, kWaves, kOdd, Epi>), grid, dim3(kWaves * 64),
                             0, stream, a, epi);
        else
          hipLaunchKernelGGL((gemm_rows_kernel<T, MT, kWaves, false, Epi>), grid, dim3(kWaves * 64),
                             0, stream, a, epi);
      };
      auto with_waves = [&](auto sets) {
        if (eight) go(sets, std::integral_constant<int, 8>{});
        else go(sets, std::integral_constant<int, 4>{});
      };
      if (a.M <= 16) with_waves(std::integral_constant<int, 1>{});
      else if (a.M <= 32) with_waves(std::integral_constant<int, 2>{});
      else with_waves(std::integral_constant<int, 4>{});
      return last_launch_status();
    }
  }
  cut_gemm<T, kXT>(a, Epi::kGated, p.tile, p.splits);
  // (256: a workgroup of the largest tile has a CU to itself and takes tile after tile)
  const int tiles = a.tiles_m * a.tiles_n;
  const dim3 grid((unsigned)(p.tile == 256 && tiles > kCus ? kCus : tiles), (unsigned)p.splits);
  if (p.tile == 256)
    hipLaunchKernelGGL((gemm_tile_kernel<T, 256, 256, 2, 2, kXT, kWT, Epi>), grid, dim3(256), 0,
                       stream, a, epi);
  else if (p.tile == 128)
    hipLaunchKernelGGL((gemm_tile_kernel<T, 128, 128, 2, 2, kXT, kWT, Epi>), grid, dim3(256), 0,
                       stream, a, epi);
  else
    hipLaunchKernelGGL((gemm_tile_kernel<T, 64, 64, 2, 1, kXT, kWT, Epi>), grid, dim3(128), 0,
                       stream, a, epi);
  if (p.splits > 1) {
    const int64_t n = (int64_t)a.M * div_up(a.N, 4);
    hipLaunchKernelGGL((gemm_join_kernel<T, Epi>), dim3((unsigned)div_up(n, 256)), dim3(256), 0,
                       stream, a, epi, p.splits);
  }
  return last_launch_status();
}

// x and w: the products of a backward pass, their partial sums where the plan splits.
template <class T, class Epi, class Extra>
int launch_pair(GemmArgs x, GemmArgs w, const Epi& ex, const Epi& ew, const PairPlan& plan,
                const Extra& extra, hipStream_t stream) {
  cut_gemm<T, false>(x, false, plan.tile, plan.splits_x);
  cut_gemm<T, true>(w, false, plan.tile, plan.splits_w);
  GemmPair p = {x, w, plan.splits_x, plan.splits_w, 0, w.steps_per_split > x.steps_per_split};
  const int64_t span_x = round_up(x.tiles_m * x.tiles_n, 8) * plan.splits_x,
                span_w = round_up(w.tiles_m * w.tiles_n, 8) * plan.splits_w;
  p.span = (int)(p.w_first ? span_w : span_x);
  const dim3 grid((unsigned)(round_up(extra.blocks, 8) + span_x + span_w));
  if (plan.tile == 256)
    hipLaunchKernelGGL((gemm_pair_kernel<T, 256, 256, 2, 2, Epi, Extra>), grid, dim3(256), 0,
                       stream, p, ex, ew, extra);
  else if (plan.tile == 128)
    hipLaunchKernelGGL((gemm_pair_kernel<T, 128, 128, 2, 2, Epi, Extra>), grid, dim3(256), 0,
                       stream, p, ex, ew, extra);
  else
    hipLaunchKernelGGL((gemm_pair_kernel<T, 64, 64, 2, 1, Epi, Extra>), grid, dim3(128), 0, stream,
                       p, ex, ew, extra);
  if (plan.splits_x > 1 || plan.splits_w > 1) {
    const int64_t nx = plan.splits_x > 1 ? (int64_t)x.M * div_up(x.N, 4) : 0,
                  nw = plan.splits_w > 1 ? (int64_t)w.M * div_up(w.N, 4) : 0;
    hipLaunchKernelGGL((gemm_join_pair_kernel<T, Epi>),
                       dim3((unsigned)div_up(nx > nw ? nx : nw, 256), nx && nw ? 2 : 1), dim3(256),
                       0, stream, p, ex, ew);
  }
  return last_launch_status();
}

}  // namespace ppo

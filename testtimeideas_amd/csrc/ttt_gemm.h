// ttt_gemm.h — the tile product that the linear cross entropy's kernels are
// made of: a BM x BN tile of  sum_k Mop[m][k] Nop[n][k]  over a list of
// segments, on the 16-bit matrix cores of gfx950.
//
// Both operands are row-major with k contiguous.  A segment is a pair of
// operands and their common k; the sum runs over all segments in order.  That
// one form covers
//   - a plain product (one segment);
//   - a contraction over two stacked ranges, [H | G] [W ; B] (two segments);
//   - fp32 operands, each held as three bf16 parts whose sum is the value: six
//     segments, the part products above 2^-24 of the whole, smallest first.
//
// MFMA 16x16x32: a lane (c = lane % 16, g = lane / 16) holds the results of
// four consecutive m (4g ..) of one n (c).  So the M operand is chosen to be
// the one whose index is contiguous in the output, and a token's sums over the
// vocabulary stay in one lane plus two lane swaps.
//
// A step is 64 k: both tiles go straight from global memory to LDS (1 KB per
// wave instruction: eight rows of 128 bytes, 16-byte chunks permuted by the
// row's low three bits against bank conflicts), two buffers, the next step's
// loads issued before this step's products.  Rows past an operand's end and
// chunks past its k read as zeros through the buffer's range check.
#pragma once

#include "ttt_common.h"

namespace ttt {

constexpr int kStepK = 64;  // k of one step: 128 bytes of a row

struct Seg {
  const void *m, *n;  // first rows of the operands
  int64_t ldm, ldn;   // row strides in elements
  int k;              // a multiple of 8
};

constexpr int kMaxSegs = 12;

struct SegList {
  Seg s[kMaxSegs];
  int n;      // segments
  int steps;  // 64-k steps of all of them
};

// One operand's share of a step's loads: this lane's byte offsets.
template <int ROWS, int NW>
struct RowLoader {
  static constexpr int kInstr = ROWS * 128 / 1024;
  static constexpr int kPerWave = kInstr / NW;
  static_assert(kPerWave * NW == kInstr, "tile shape");
  uint32_t off[kPerWave];

  // rows_valid rows of stride ld elements
  __device__ __forceinline__ void rows(int rows_valid, int64_t ld, int wave) {
    const int lane = threadIdx.x & 63, r8 = lane >> 3;
    const uint32_t ldb = (uint32_t)(ld * 2);
#pragma unroll
    for (int q = 0; q < kPerWave; ++q) {
      const int r = 8 * (wave + NW * q) + r8;
      off[q] = r < rows_valid ? (uint32_t)r * ldb + 16u * (uint32_t)((lane & 7) ^ r8) : kBufRange;
    }
  }
  // base: the tile's first row at this step's k; past: this lane's chunk lies past the segment's k
  __device__ __forceinline__ void issue(char* lds, const char* base, bool past, int wave) const {
#if defined(__HIP_DEVICE_COMPILE__)
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), (short)0, (int)kBufRange, kBufWord3);
#pragma unroll
    for (int q = 0; q < kPerWave; ++q)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)(lds + 1024 * (wave + NW * q)), 16,
                                               past ? kBufPast : (int)off[q], 0, 0, 0);
#endif
  }
};

template <typename T, int BM_, int BN_, int WM_, int WN_>
struct TileProduct {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NW = WM * WN;
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  typedef typename Elem<T>::frag frag;

  // The four step buffers, in distinct arrays: the compiler waits for pending
  // direct loads before an LDS read that may alias their destination.
  struct Lds {
    char *m0, *m1, *n0, *n1;
  };

  int wave, wm, wn;
  int m0, n0, mrows, nrows;  // the tile's corner and the rows it has of each operand
  RowLoader<BM, NW> lm;
  RowLoader<BN, NW> ln;

  __device__ __forceinline__ TileProduct(int m0_, int n0_, int M, int N) : m0(m0_), n0(n0_) {
    wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    wm = wave % WM;
    wn = wave / WM;
    mrows = M - m0;
    nrows = N - n0;
  }

  // Position in the segment list.
  int seg, k0;
  const char *bm, *bn;

  __device__ __forceinline__ void enter(const SegList& l) {
    const Seg& s = l.s[seg];
    bm = (const char*)s.m + ((int64_t)m0 * s.ldm + k0) * 2;
    bn = (const char*)s.n + ((int64_t)n0 * s.ldn + k0) * 2;
    lm.rows(mrows, s.ldm, wave);
    ln.rows(nrows, s.ldn, wave);
  }
  __device__ __forceinline__ void seek(const SegList& l, int step) {
    seg = 0;
    for (int n; seg + 1 < l.n && step >= (n = (l.s[seg].k + kStepK - 1) / kStepK); ++seg) step -= n;
    k0 = step * kStepK;
    enter(l);
  }
  // Issue the loads of the current step and move to the next.
  __device__ __forceinline__ void issue(const SegList& l, char* sm, char* sn, bool last) {
    const int lane = threadIdx.x & 63;
    const int k = l.s[seg].k;
    const bool past = k0 + 8 * ((lane & 7) ^ (lane >> 3)) >= k;
    lm.issue(sm, bm, past, wave);
    ln.issue(sn, bn, past, wave);
    k0 += kStepK;
    bm += kStepK * 2;
    bn += kStepK * 2;
    if (k0 >= k && !last) {
      ++seg;
      k0 = 0;
      enter(l);
    }
  }

  __device__ __forceinline__ void multiply(f32x4 (&acc)[MI][NI], const char* sm, const char* sn) const {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const char* pm = sm + (wm * MI * 16 + c) * 128;
    const char* pn = sn + (wn * NI * 16 + c) * 128;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int slot = 16 * ((4 * kk + g) ^ (c & 7));
      frag fm[MI], fn[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) fm[i] = *(const frag*)(pm + i * 2048 + slot);
#pragma unroll
      for (int i = 0; i < NI; ++i) fn[i] = *(const frag*)(pn + i * 2048 + slot);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = Elem<T>::mma(acc[i][j], fm[i], fn[j]);
    }
  }

  // acc += the steps lo .. hi - 1 of the list.  Ends with every wave past its
  // last read of the buffers.
  __device__ __forceinline__ void run(f32x4 (&acc)[MI][NI], const SegList& l, int lo, int hi, const Lds& s) {
    if (lo >= hi) return;  // uniform
    seek(l, lo);
    issue(l, s.m0, s.n0, lo + 1 >= hi);
    for (int t = lo; t < hi; t += 2) {
      dma_wait();
      __syncthreads();
      if (t + 1 < hi) issue(l, s.m1, s.n1, t + 2 >= hi);
      multiply(acc, s.m0, s.n0);
      if (t + 1 >= hi) break;
      dma_wait();
      __syncthreads();
      if (t + 2 < hi) issue(l, s.m0, s.n0, t + 3 >= hi);
      multiply(acc, s.m1, s.n1);
    }
    __syncthreads();
  }

  __device__ __forceinline__ static void zero(f32x4 (&acc)[MI][NI]) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // First m (of four) of acc[i][*] and the n of acc[*][j] in this lane.
  __device__ __forceinline__ int m_of(int i) const { return m0 + (wm * MI + i) * 16 + 4 * ((threadIdx.x & 63) >> 4); }
  __device__ __forceinline__ int n_of(int j) const { return n0 + (wn * NI + j) * 16 + (threadIdx.x & 15); }
};

// Tile (tm, tn) of workgroup `id` among tm_count x tn_count.  Workgroups go to
// the eight XCDs in turn, each with an L2 of its own: an XCD gets a run of
// neighbouring tiles, walked in blocks of kGroup tn, so that the tiles in
// flight on it share operand rows.
__device__ __forceinline__ void tile_of(int id, int tm_count, int tn_count, int* tm, int* tn) {
  constexpr int kXcd = 8, kGroup = 4;
  const int total = tm_count * tn_count;
  const int per = total / kXcd, rest = total % kXcd;
  const int x = id % kXcd, i = id / kXcd;
  const int t = x * per + (x < rest ? x : rest) + i;
  const int block = kGroup * tm_count, b = t / block, in = t % block;
  const int wide = tn_count - b * kGroup < kGroup ? tn_count - b * kGroup : kGroup;
  *tn = b * kGroup + in % wide;
  *tm = in / wide;
}

}  // namespace ttt

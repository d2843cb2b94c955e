// ttt_gemm.h — the tile products that the linear cross entropy's kernels are
// made of: a BM x BN tile of  sum_k Mop[m][k] Nop[n][k]  over a list of
// segments, on the 16-bit matrix cores of gfx950.
//
// An operand is a row-major matrix in either order: its rows are m (or n) and
// k is contiguous, or its rows are k and m is contiguous ("turned").  So no
// product needs a transposed copy, and one order of G serves both dX = G W and
// dW = G^T X.  A segment is a pair of operands and their common k; the sum
// runs over all segments in order, which covers a contraction over two stacked
// ranges, [H | G] [W ; B], without stacking them.
//
// MFMA 16x16x32: a lane (c = lane % 16, g = lane / 16) holds the results of
// four consecutive m (4g ..) of one n (c).  So the M operand is chosen to be
// the one whose index is contiguous in the output, and a token's sums over the
// vocabulary stay in one lane plus two lane swaps.
//
// TileProduct (16-bit types): a step is 64 k.  Both tiles go straight from
// global memory to LDS (1 KB per wave instruction, 16-byte chunks permuted
// against bank conflicts), two buffers, the next step's loads issued before
// this step's products.  Turned tiles are read with ds_read_b64_tr_b16.  What
// lies past an operand's end reads as zeros through the buffer's range check.
//
// SplitProduct (fp32): a value is the sum of three bf16 parts, exactly
// (split_pair), and a product the sum of the six part products above 2^-22 of
// it, smallest first, in fp32: six times the matrix work of bf16, where the
// fp32 instruction takes sixteen.  A step is 32 k: values go to registers two
// steps ahead, are split once, among the products of the step before theirs,
// and stored as three tiles of parts; either order of an operand ends up the
// same there.
#pragma once

#include "ttt_common.h"

namespace ttt {

struct Seg {
  const void *m, *n;  // first elements of the operands
  int64_t ldm, ldn;   // row strides in elements
  int k;
};

constexpr int kMaxSegs = 2;

struct SegList {
  Seg s[kMaxSegs];
  int n;
};

// Steps of STEP k in a list.
template <int STEP>
__host__ __device__ __forceinline__ int list_steps(const SegList& l) {
  int t = 0;
  for (int i = 0; i < l.n; ++i) t += (l.s[i].k + STEP - 1) / STEP;
  return t;
}

// What the two products share: the waves' places in the tile, and the walk
// over the segments.  Derived classes have enter() and the loads of a step.
template <int BM_, int BN_, int WM_, int WN_, int STEP_>
struct TileBase {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NW = WM * WN, kStep = STEP_;
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;

  int wave, wm, wn;
  int m0, n0, mrows, nrows;  // the tile's corner and the rows it has of each operand
  int seg, k0;               // position in the segment list

  __device__ __forceinline__ TileBase(int m0_, int n0_, int M, int N) : m0(m0_), n0(n0_) {
    wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    wm = wave % WM;
    wn = wave / WM;
    mrows = M - m0;
    nrows = N - n0;
  }
  __device__ __forceinline__ void seek(const SegList& l, int step) {
    seg = 0;
    for (int n; seg + 1 < l.n && step >= (n = (l.s[seg].k + kStep - 1) / kStep); ++seg) step -= n;
    k0 = step * kStep;
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

// One 16-bit operand's share of a step's loads: this lane's byte offsets.
//   plain:  LDS [R rows][64 k], chunk ^ (row & 7)
//   turned: LDS [64 k][R], chunk ^ swz(k): the sixteen rows of a transposing
//           read (k = 0-3, 8-11, 16-19, 24-27 past its first) are spread over
//           eight 32-byte places
template <int R, int NW, bool TURNED>
struct Loader {
  static constexpr int kInstr = R * 128 / 1024, kPerWave = kInstr / NW;
  static_assert(kPerWave * NW == kInstr, "tile shape");
  static constexpr int kRowBytes = TURNED ? R * 2 : 128, kChunks = kRowBytes / 16;
  uint32_t off[kPerWave];
  int64_t step;  // bytes from a step's first element to the next one's

  static __device__ __forceinline__ int swz(int k) {
    return ((k & 1) << 1) | (((k >> 1) & 1) << 2) | (((k >> 3) & 1) << 3);
  }
  // Row and chunk that instruction q fetches in this lane.  They are needed
  // where a segment begins or ends only: `lane` is made opaque there, or they
  // would be kept in registers all along.
  static __device__ __forceinline__ int fresh_lane() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
  }
  static __device__ __forceinline__ int row_of(int q, int wave, int lane) {
    return (1024 * (wave + NW * q) + 16 * lane) / kRowBytes;
  }
  static __device__ __forceinline__ int chunk_of(int row, int lane) {
    return lane % kChunks ^ (TURNED ? swz(row) : row & 7);
  }
  // valid: rows (turned: columns) of the tile that exist
  __device__ __forceinline__ void enter(int valid, int64_t ld, int wave) {
    step = TURNED ? 128 * ld : 128;
    const int lane = fresh_lane();
#pragma unroll
    for (int q = 0; q < kPerWave; ++q) {
      const int r = row_of(q, wave, lane), ch = chunk_of(r, lane);
      const bool in = TURNED ? 8 * ch < valid : r < valid;
      off[q] = in ? (uint32_t)r * (uint32_t)(ld * 2) + 16u * (uint32_t)ch : kBufRange;
    }
  }
  // base: the tile's first element at this step; left: k from here to the segment's end
  __device__ __forceinline__ void issue(char* lds, const char* base, int left, int wave) const {
#if defined(__HIP_DEVICE_COMPILE__)
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), (short)0, (int)kBufRange, kBufWord3);
    if (left >= 64) {
#pragma unroll
      for (int q = 0; q < kPerWave; ++q)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)(lds + 1024 * (wave + NW * q)), 16, (int)off[q], 0, 0,
                                                 0);
    } else {
      const int lane = fresh_lane();
#pragma unroll
      for (int q = 0; q < kPerWave; ++q) {
        const int row = row_of(q, wave, lane);
        const bool in = TURNED ? row < left : 8 * chunk_of(row, lane) < left;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)(lds + 1024 * (wave + NW * q)), 16,
                                                 in ? (int)off[q] : kBufPast, 0, 0, 0);
      }
    }
#endif
  }
};

template <typename T, int BM_, int BN_, int WM_, int WN_, bool MT, bool NT>
struct TileProduct : TileBase<BM_, BN_, WM_, WN_, 64> {
  typedef TileBase<BM_, BN_, WM_, WN_, 64> B;
  using B::BM;
  using B::BN;
  using B::MI;
  using B::NI;
  using B::NW;
  typedef typename Elem<T>::frag frag;
  static constexpr int kBytesM = BM * 128, kBytesN = BN * 128;  // of one buffer

  // The step buffers, in distinct arrays: the compiler waits for pending
  // direct loads before an LDS read that may alias their destination.
  struct Lds {
    char *m0, *m1, *n0, *n1;
  };

  Loader<BM, NW, MT> lm;
  Loader<BN, NW, NT> ln;
  const char *bm, *bn;
  int kseg;  // the segment's k

  __device__ __forceinline__ TileProduct(int m0, int n0, int M, int N) : B(m0, n0, M, N) {}

  __device__ __forceinline__ void enter(const SegList& l) {
    const Seg& s = l.s[this->seg];
    const int64_t k0 = this->k0;
    kseg = s.k;
    bm = (const char*)s.m + (MT ? k0 * s.ldm + this->m0 : this->m0 * s.ldm + k0) * 2;
    bn = (const char*)s.n + (NT ? k0 * s.ldn + this->n0 : this->n0 * s.ldn + k0) * 2;
    lm.enter(this->mrows, s.ldm, this->wave);
    ln.enter(this->nrows, s.ldn, this->wave);
  }
  // Issue the loads of the current step and move to the next.
  __device__ __forceinline__ void issue(const SegList& l, char* sm, char* sn, bool last) {
    const int left = kseg - this->k0;
    lm.issue(sm, bm, left, this->wave);
    ln.issue(sn, bn, left, this->wave);
    this->k0 += 64;
    bm += lm.step;
    bn += ln.step;
    if (left <= 64 && !last) {
      ++this->seg;
      this->k0 = 0;
      enter(l);
    }
  }

  // This lane's byte offset of a fragment's eight k (of row c, from 8 g) in the
  // tile of an operand whose fragments start at row r0 of R.  Fragment i is at
  // the offset + 2048 i, turned: offset ^ 32 i; 32 k on: ^ 64, turned: + 64 R.
  template <int R, bool TURNED>
  static __device__ __forceinline__ int lane_offset(int r0) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    if constexpr (!TURNED) return (r0 + c) * 128 + 16 * (g ^ (c & 7));
    const int k = 8 * g + (c >> 2);  // k + 4 and k + 32 have the same permutation
    return k * (R * 2) + 16 * (((r0 >> 3) + ((c & 3) >> 1)) ^ Loader<R, NW, true>::swz(k)) + 8 * (c & 1);
  }
  template <int R, bool TURNED>
  static __device__ __forceinline__ frag read(const char* s, int off, int i, int kk) {
    if constexpr (!TURNED) {
      return *(const frag*)(s + (off ^ (64 * kk)) + 2048 * i);
    } else {
      const char* a = s + (off ^ (32 * i)) + kk * 64 * R;
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(a));
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(a + 8 * R));
      const i16x4 both[2] = {lo, hi};
      frag f;
      __builtin_memcpy(&f, both, 16);
      return f;
    }
  }

  // A step is four quarters: 32 k of one half of the M fragments.  The reads
  // of a quarter's fragments are issued among the products of the quarter
  // before, across the barrier too, so that neither unit waits for the other.
  static constexpr int MH = MI / 2;
  struct Frags {
    frag n[2][NI];  // of k 0-31 and 32-63
    frag m[2][MH];  // of the even and odd quarters
    int om, on;     // lane_offset of the operands
  };
  template <int Q>
  __device__ __forceinline__ void read_quarter(Frags& f, const char* sm, const char* sn) const {
    constexpr int kk = Q >> 1, h = Q & 1;
    if constexpr (h == 0)
#pragma unroll
      for (int i = 0; i < NI; ++i) f.n[kk][i] = read<BN, NT>(sn, f.on, i, kk);
#pragma unroll
    for (int i = 0; i < MH; ++i) f.m[h][i] = read<BM, MT>(sm, f.om, h * MH + i, kk);
  }
  template <int Q>
  static __device__ __forceinline__ void multiply(f32x4 (&acc)[MI][NI], const Frags& f) {
    constexpr int kk = Q >> 1, h = Q & 1;
#pragma unroll
    for (int i = 0; i < MH; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[h * MH + i][j] = Elem<T>::mma(acc[h * MH + i][j], f.m[h][i], f.n[kk][j]);
  }
  // The order of the reads of quarter Q (two for a turned fragment) and the
  // products of the quarter before.
  template <int Q>
  static __device__ __forceinline__ void interleave() {
    constexpr int kReads = MH * (MT ? 2 : 1) + (Q & 1 ? 0 : NI * (NT ? 2 : 1)), kProducts = MH * NI;
    constexpr int kPer = kProducts / kReads < 1 ? 1 : kProducts / kReads;
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, kPer, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kProducts, 0);
    __builtin_amdgcn_sched_barrier(0);
  }

  // One step of run(): its tile is in (sm, sn) once the loads are waited for,
  // the next one's go to (om, on).
  template <bool FIRST>
  __device__ __forceinline__ void step(f32x4 (&acc)[MI][NI], Frags& f, const SegList& l, const char* sm, const char* sn,
                                       char* om, char* on, int left) {
    dma_wait();
    __syncthreads();
    if (left > 1) issue(l, om, on, left <= 2);
    // the turned reads' addresses are formed here, in every step: kept across
    // the loop, one for each fragment and buffer, they do not fit the registers
    if constexpr (MT) asm volatile("" : "+v"(f.om));
    if constexpr (NT) asm volatile("" : "+v"(f.on));
    __builtin_amdgcn_sched_barrier(0);
    read_quarter<0>(f, sm, sn);
    if constexpr (!FIRST) {
      multiply<3>(acc, f);
      interleave<0>();
    }
    read_quarter<1>(f, sm, sn);
    multiply<0>(acc, f);
    interleave<1>();
    read_quarter<2>(f, sm, sn);
    multiply<1>(acc, f);
    interleave<2>();
    read_quarter<3>(f, sm, sn);
    multiply<2>(acc, f);
    interleave<3>();
  }

  // acc += the steps lo .. hi - 1 of the list.  Ends with every wave past its
  // last read of the buffers.
  __device__ __forceinline__ void run(f32x4 (&acc)[MI][NI], const SegList& l, int lo, int hi, const Lds& s) {
    if (lo >= hi) return;  // uniform
    this->seek(l, lo);
    enter(l);
    issue(l, s.m0, s.n0, lo + 1 >= hi);
    Frags f;
    f.om = lane_offset<BM, MT>(this->wm * MI * 16);
    f.on = lane_offset<BN, NT>(this->wn * NI * 16);
    step<true>(acc, f, l, s.m0, s.n0, s.m1, s.n1, hi - lo);
    int left = hi - lo - 1;
    for (; left > 1; left -= 2) {
      step<false>(acc, f, l, s.m1, s.n1, s.m0, s.n0, left);
      step<false>(acc, f, l, s.m0, s.n0, s.m1, s.n1, left - 1);
    }
    if (left > 0) step<false>(acc, f, l, s.m1, s.n1, s.m0, s.n0, 1);
    multiply<3>(acc, f);
    __syncthreads();
  }
};

// One fp32 operand's share of a step: 16-byte chunks (eight k of a row) of
// parts, kTasks per thread.  LDS, per part: [R rows][32 k], chunk ^ (row >> 1 & 3).
template <int R, int THREADS, bool TURNED>
struct SplitLoader {
  static constexpr int kTasks = R * 4 / THREADS;
  static_assert(kTasks * THREADS == R * 4 && kTasks >= 1, "tile shape");
  static_assert(!TURNED || kTasks % 2 == 0 || kTasks == 1, "tile shape");
  static constexpr int kPlane = R * 64;  // bytes of a part's tile
  float v[kTasks][8];
  float f[kTasks][8];  // LIVE: the k's factors

  // Row and chunk of a task.  plain: four lanes share a row's 128 bytes;
  // turned: neighbouring lanes have neighbouring rows.
  static __device__ __forceinline__ int row_of(int t) {
    const int i = (int)threadIdx.x + t * THREADS;
    return TURNED ? i % R : i >> 2;
  }
  static __device__ __forceinline__ int chunk_of(int t) {
    const int i = (int)threadIdx.x + t * THREADS;
    return TURNED ? i / R : i & 3;
  }
  // base: the tile's first element at this step; rows past valid and k past left are zeros, and so, with LIVE,
  // are the k whose `live` factor is 0 (live at this step).  WHOLE: nothing is past anything.
  template <bool WHOLE, bool LIVE>
  __device__ __forceinline__ void load(const float* base, int64_t ld, int valid, int left, const float* live) {
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
      const int r = row_of(t), k = 8 * chunk_of(t);
      if constexpr (!TURNED) {
        const float* p = base + r * ld + k;
        if (WHOLE || (r < valid && k + 8 <= left)) {
          __builtin_memcpy(&v[t][0], p, 16);
          __builtin_memcpy(&v[t][4], p + 4, 16);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[t][j] = r < valid && k + j < left ? p[j] : 0.f;
        }
      } else {
        const float* p = base + k * ld + r;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[t][j] = WHOLE || (r < valid && k + j < left) ? p[j * ld] : 0.f;
          if constexpr (LIVE) f[t][j] = WHOLE || k + j < left ? live[k + j] : 0.f;
        }
      }
    }
  }
  // SIGNED: the values' signs are changed by `sign` (its highest bit).
  template <bool LIVE, bool SIGNED>
  __device__ __forceinline__ void store(char* lds, uint32_t sign) const {
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
      const int r = row_of(t), ch = chunk_of(t);
      u32x4 h, m, l;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t a, b, c;
        float x = v[t][2 * j], y = v[t][2 * j + 1];
        if constexpr (LIVE) {
          x = f[t][2 * j] != 0.f ? x : 0.f;
          y = f[t][2 * j + 1] != 0.f ? y : 0.f;
        }
        if constexpr (SIGNED) {
          x = __uint_as_float(__float_as_uint(x) ^ sign);
          y = __uint_as_float(__float_as_uint(y) ^ sign);
        }
        split_pair(x, y, a, b, c);
        h[j] = a;
        m[j] = b;
        l[j] = c;
      }
      char* p = lds + r * 64 + 16 * (ch ^ ((r >> 1) & 3));
      *(u32x4*)p = h;
      *(u32x4*)(p + kPlane) = m;
      *(u32x4*)(p + 2 * kPlane) = l;
    }
  }
};

template <int BM_, int BN_, int WM_, int WN_, bool MT, bool NT>
struct SplitProduct : TileBase<BM_, BN_, WM_, WN_, 32> {
  typedef TileBase<BM_, BN_, WM_, WN_, 32> B;
  using B::BM;
  using B::BN;
  using B::MI;
  using B::NI;
  using B::NW;
  static constexpr int kThreads_ = 64 * NW;
  static constexpr int kBytesM = BM * 64 * 3, kBytesN = BN * 64 * 3;

  struct Lds {
    char *m0, *m1, *n0, *n1;
  };
  struct Regs {  // a step's values
    SplitLoader<BM, kThreads_, MT> m;
    SplitLoader<BN, kThreads_, NT> n;
  };

  const float* live;  // factors of the k of a turned M operand, or null

  __device__ __forceinline__ SplitProduct(int m0, int n0, int M, int N, const float* live_)
      : B(m0, n0, M, N), live(live_) {}

  // Both operands turned is a sum over the rows of X (or A): those that do not
  // count are left out.
  static constexpr bool kLive = MT && NT;

  const float *bm, *bn;  // the tile's first elements at this step
  int64_t ldm, ldn, incm, incn;
  int kseg;

  __device__ __forceinline__ void enter(const SegList& l) {
    const Seg& s = l.s[this->seg];
    const int64_t k0 = this->k0;
    kseg = s.k;
    ldm = s.ldm;
    ldn = s.ldn;
    incm = MT ? 32 * ldm : 32;
    incn = NT ? 32 * ldn : 32;
    bm = (const float*)s.m + (MT ? k0 * ldm + this->m0 : this->m0 * ldm + k0);
    bn = (const float*)s.n + (NT ? k0 * ldn + this->n0 : this->n0 * ldn + k0);
  }
  // Load the current step's values and move to the next.
  template <bool WHOLE>
  __device__ __forceinline__ void load(const SegList& l, Regs& r) {
    const int left = kseg - this->k0;
    r.m.template load<WHOLE, kLive>(bm, ldm, this->mrows, left, kLive ? live + this->k0 : nullptr);
    r.n.template load<WHOLE, false>(bn, ldn, this->nrows, left, nullptr);
    this->k0 += 32;
    bm += incm;
    bn += incn;
    if (left <= 32 && this->seg + 1 < l.n) {
      ++this->seg;
      this->k0 = 0;
      enter(l);
    }
  }
  static __device__ __forceinline__ void store(const Regs& r, char* om, char* on, uint32_t sign) {
    r.m.template store<kLive, true>(om, sign);
    r.n.template store<false, false>(on, 0u);
  }
  static __device__ __forceinline__ void negate(f32x4 (&acc)[MI][NI]) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = -acc[i][j];
  }

  __device__ __forceinline__ void multiply(f32x4 (&acc)[MI][NI], const char* sm, const char* sn) const {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int at = c * 64 + 16 * (g ^ ((c >> 1) & 3));
    const char* pm = sm + this->wm * MI * 1024 + at;
    const char* pn = sn + this->wn * NI * 1024 + at;
    bf16x8 fm[3][MI], fn[3][NI];
    // part products, the smallest first: (m part, n part)
    const auto part = [&](int a, int b) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = Elem<__bf16>::mma(acc[i][j], fm[a][i], fn[b][j]);
    };
    // the reads in the order of their products
    const auto read_m = [&](int a) {
#pragma unroll
      for (int i = 0; i < MI; ++i) fm[a][i] = *(const bf16x8*)(pm + a * (BM * 64) + i * 1024);
    };
    const auto read_n = [&](int a) {
#pragma unroll
      for (int j = 0; j < NI; ++j) fn[a][j] = *(const bf16x8*)(pn + a * (BN * 64) + j * 1024);
    };
    read_m(2);
    read_n(0);
    read_m(0);
    read_n(2);
    read_m(1);
    read_n(1);
    part(2, 0);
    part(0, 2);
    part(1, 1);
    part(1, 0);
    part(0, 1);
    part(0, 0);
  }

  // The products of the step in (sm, sn), while the values of the next, in r
  // (MORE > 0), are split and stored to (om, on) and those of the one after
  // (MORE > 1) are on their way to q.
  template <bool WHOLE, int MORE>
  __device__ __forceinline__ void step(f32x4 (&acc)[MI][NI], const SegList& l, const char* sm, const char* sn,
                                       char* om, char* on, const Regs& r, Regs& q, uint32_t sign) {
    if constexpr (MORE > 1) {
      load<WHOLE>(l, q);
      __builtin_amdgcn_sched_barrier(0);
    }
    multiply(acc, sm, sn);
    if constexpr (MORE > 0) {
      store(r, om, on, sign);
      // all reads, some of the split's operations while the first arrive, then a few behind every product
      __builtin_amdgcn_sched_group_barrier(0x100, 3 * (MI + NI), 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 16, 0);
#pragma unroll
      for (int i = 0; i < 6 * MI * NI; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
      }
    }
    __syncthreads();
  }

  // The matrix instructions round their sums down, so that sums over many of
  // their results (a bias' gradient) would gather it.  The M operand's values
  // of every other two steps (+ - - + + - - ...) are stored with the opposite
  // sign, and the sums negated between: what is taken from the one is given to
  // the other.  (5567 x 103 x 1683: a mean error of -0.10 to -0.19 of its root
  // mean square without, under 0.003 with; the sum of gX's rows off by 2.7e-6
  // of it and 7.4e-7; 1 to 3 % of the time.)
  //
  // WHOLE: without a test, the number of loads on their way is known where the
  // values of the step before are waited for, and only those are.
  template <bool WHOLE>
  __device__ __forceinline__ void walk(f32x4 (&acc)[MI][NI], const SegList& l, int steps, const Lds& s) {
    Regs a, b;
    uint32_t sign = 0x80000000u;  // of the two steps after the next
    load<WHOLE>(l, a);
    store(a, s.m0, s.n0, 0u);
    if (steps > 1) load<WHOLE>(l, b);
    __syncthreads();
    for (; steps > 3; steps -= 2) {
      step<WHOLE, 2>(acc, l, s.m0, s.n0, s.m1, s.n1, b, a, sign);
      negate(acc);
      step<WHOLE, 2>(acc, l, s.m1, s.n1, s.m0, s.n0, a, b, sign);
      sign ^= 0x80000000u;
    }
    if (steps == 3) {
      step<WHOLE, 2>(acc, l, s.m0, s.n0, s.m1, s.n1, b, a, sign);
      negate(acc);
      step<WHOLE, 1>(acc, l, s.m1, s.n1, s.m0, s.n0, a, b, sign);
      step<WHOLE, 0>(acc, l, s.m0, s.n0, s.m1, s.n1, a, b, sign);
    } else if (steps == 2) {
      step<WHOLE, 1>(acc, l, s.m0, s.n0, s.m1, s.n1, b, a, sign);
      negate(acc);
      step<WHOLE, 0>(acc, l, s.m1, s.n1, s.m0, s.n0, a, b, sign);
    } else {
      step<WHOLE, 0>(acc, l, s.m0, s.n0, s.m1, s.n1, a, b, sign);
      sign ^= 0x80000000u;
    }
    if (sign) negate(acc);  // uniform
  }

  __device__ __forceinline__ void run(f32x4 (&acc)[MI][NI], const SegList& l, int lo, int hi, const Lds& s) {
    if (lo >= hi) return;  // uniform
    this->seek(l, lo);
    enter(l);
    bool whole = this->mrows >= BM && this->nrows >= BN;
    for (int i = 0; i < l.n; ++i) whole = whole && l.s[i].k % 32 == 0;
    if (whole) walk<true>(acc, l, hi - lo, s);
    else walk<false>(acc, l, hi - lo, s);
  }
};

// Small products: 32 x 32 tiles of operands that are k-contiguous, for few
// tokens or few tiles, where what counts is the way of one load after another.
// Four waves take every fourth 32 k each and load their fragments straight
// from global memory, kAhead steps at a time (no LDS, no barrier); their sums
// meet in LDS at the end, where each wave gets one 16 x 16 quarter.  fp32: the
// part products of three magnitudes are summed apart.
template <typename T>
struct DirectProduct : TileBase<32, 32, 2, 2, 32> {
  typedef TileBase<32, 32, 2, 2, 32> B;
  static constexpr bool kSplit = sizeof(T) == 4;
  static constexpr int kSums = kSplit ? 3 : 1;
  static constexpr int kAhead = kSplit ? 2 : 4;
  static constexpr int kBytesM = 4 * 4096, kBytesN = 16;

  struct Lds {
    char *m, *n;
  };
  struct Raw {
    T v[8];
  };

  __device__ __forceinline__ DirectProduct(int m0, int n0, int M, int N) : B(m0, n0, M, N) {}

  // Eight values at p; those past `left` (or of a row that does not exist) are zeros.
  static __device__ __forceinline__ Raw fetch(const T* p, bool in, int left) {
    Raw r;
    if (in && left >= 8) {
      __builtin_memcpy(r.v, p, sizeof(r.v));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) r.v[j] = in && j < left ? p[j] : (T)0.f;
    }
    return r;
  }

  __device__ __forceinline__ void run(f32x4 (&out)[1][1], const SegList& l, int, int, const Lds& s) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    f32x4 acc[kSums][2][2];
#pragma unroll
    for (int a = 0; a < kSums; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[a][i >> 1][i & 1] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int sg = 0; sg < l.n; ++sg) {
      const Seg& q = l.s[sg];
      const T *pm[2], *pn[2];
      bool im[2], in[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        im[i] = 16 * i + c < this->mrows;
        in[i] = 16 * i + c < this->nrows;
        pm[i] = (const T*)q.m + (int64_t)(this->m0 + 16 * i + c) * q.ldm;
        pn[i] = (const T*)q.n + (int64_t)(this->n0 + 16 * i + c) * q.ldn;
      }
      for (int k0 = 32 * this->wave; k0 < q.k; k0 += 128 * kAhead) {
        Raw rm[kAhead][2], rn[kAhead][2];
#pragma unroll
        for (int t = 0; t < kAhead; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int k = k0 + 128 * t + 8 * g;
            rm[t][i] = fetch(pm[i] + k, im[i], q.k - k);
            rn[t][i] = fetch(pn[i] + k, in[i], q.k - k);
          }
#pragma unroll
        for (int t = 0; t < kAhead; ++t) {
          if constexpr (!kSplit) {
            typename Elem<T>::frag fm[2], fn[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              __builtin_memcpy(&fm[i], rm[t][i].v, 16);
              __builtin_memcpy(&fn[i], rn[t][i].v, 16);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[0][i >> 1][i & 1] = Elem<T>::mma(acc[0][i >> 1][i & 1], fm[i >> 1], fn[i & 1]);
          } else {
            SplitFrag fm[2], fn[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              fm[i] = split8(rm[t][i].v);
              fn[i] = split8(rn[t][i].v);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const SplitFrag &x = fm[i >> 1], &y = fn[i & 1];
              f32x4 &lo = acc[2][i >> 1][i & 1], &mid = acc[1][i >> 1][i & 1], &hi = acc[0][i >> 1][i & 1];
              lo = Elem<__bf16>::mma(lo, x.l, y.h);
              lo = Elem<__bf16>::mma(lo, x.h, y.l);
              lo = Elem<__bf16>::mma(lo, x.m, y.m);
              mid = Elem<__bf16>::mma(mid, x.m, y.h);
              mid = Elem<__bf16>::mma(mid, x.h, y.m);
              hi = Elem<__bf16>::mma(hi, x.h, y.h);
            }
          }
        }
      }
    }
    // wave w keeps quarter (w % 2, w / 2): the four waves' sums of it, in wave order
    f32x4* p = (f32x4*)s.m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 v = acc[0][i & 1][i >> 1];
      if constexpr (kSplit) v += acc[1][i & 1][i >> 1] + acc[2][i & 1][i >> 1];
      p[(i * 4 + this->wave) * 64 + lane] = v;
    }
    __syncthreads();
    out[0][0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) out[0][0] += p[(this->wave * 4 + w) * 64 + lane];
    __syncthreads();
  }
};

// Tile (tm, tn) of workgroup `id` among tm_count x tn_count.  Workgroups go to
// the eight XCDs in turn, each with an L2 of its own: an XCD gets a run of
// neighbouring tiles, walked in blocks of kGroup tn, so that the tiles in
// flight on it share operand rows.  (kGroup 4, 2, 8: 8192 x 4096 x 65536 bf16
// forward 3290, 3313, 3316 us; 4096 x 1024 x 16384 134, 135, 131.)
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
